"""The language-model operators of maidenx_amd on work of real shape: causal attention over packed sequences with grouped
heads, the learned relative position bias inside it, and the clipped policy loss with a KL term over a vocabulary.

`own` False computes each operator from elementary torch operations in 32 bits; `own` True calls libmaidenx_hip.so."""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def attention_case(kind, dtype, lengths, heads, kv_heads, dim, buckets=0, max_distance=0):
    return {"op": "attention", "kind": kind, "dtype": dtype, "lengths": ",".join(map(str, lengths)), "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "buckets": buckets, "max_distance": max_distance}


def policy_case(kind, dtype, rows, vocab, share):
    return {"op": "policy", "kind": kind, "dtype": dtype, "rows": rows, "vocab": vocab, "share": share}


def listed():
    return [
        # three prompts of a few tokens: one wave of work, the time of a launch
        {"name": "attn fwd f32 96 tokens", **attention_case("forward", "f32", [1, 40, 55], 4, 4, 32)},
        # the prompts of a batch as a server or an evaluation meets them, shared key heads
        {"name": "attn fwd bf16 4k ragged", **attention_case("forward", "bf16", [700, 33, 512, 1, 1291, 64, 255, 840, 400], 16, 4, 64)},
        # long documents, forward only: the largest call
        {"name": "attn fwd bf16 8k long", **attention_case("forward", "bf16", [5000, 2500, 692], 32, 8, 128)},
        # one training step's attention (forward, then all gradients), whole heads
        {"name": "attn step bf16 4k", **attention_case("step", "bf16", [1024, 1000, 1048, 1024], 16, 16, 64)},
        # a head size that is no power of two, and f16
        {"name": "attn step f16 d80", **attention_case("step", "f16", [1000, 24, 777, 1], 12, 2, 80)},
        # the step with the learned bias: long sequences, where most pairs share the last bucket
        {"name": "bias step bf16 8k", **attention_case("step", "bf16", [4096, 3000, 1096], 16, 4, 128, 32, 128)},
        # ... and in f32 with buckets of 16 exact distances and borders that fall on whole distances (32, 64, 128)
        {"name": "bias step f32 1k", **attention_case("step", "f32", [512, 300, 211, 1], 8, 2, 64, 32, 256)},
        # a small batch and vocabulary: launches count
        {"name": "policy step f32 37x1000", **policy_case("step", "f32", 37, 1000, 0.8)},
        # a step of ordinary size: two fifths of the rows are prompt tokens, which the loss leaves out
        {"name": "policy step bf16 2kx32000", **policy_case("step", "bf16", 2048, 32000, 0.6)},
        # the largest: an odd vocabulary, so that rows are aligned to their elements only
        {"name": "policy step bf16 8kx50001", **policy_case("step", "bf16", 8192, 50001, 0.9)},
        # a few long rows, forward only (scoring an answer)
        {"name": "policy fwd f16 16x128000", **policy_case("forward", "f16", 16, 128000, 1.0)},
        # evaluation of a batch
        {"name": "policy fwd f32 3kx32000", **policy_case("forward", "f32", 3000, 32000, 0.7)},
    ]


def log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    kind = rng.choice(["forward", "step"])
    if rng.random() < 0.4:
        vocab = log_uniform(rng, 500, 128000)
        rows = log_uniform(rng, 1, max(2, min(8192, 150_000_000 // vocab)))
        return policy_case(kind, dtype, rows, vocab, round(rng.uniform(0.3, 1.0), 2))
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4])
    dim = rng.choice([16, 32, 40, 64, 64, 72, 96, 128, 128])
    left = log_uniform(rng, 20, 2500 if dtype == "f32" else 6000)
    lengths = []
    while left > 0 and len(lengths) < 12:
        n = min(left, log_uniform(rng, 1, 5000))
        lengths.append(n)
        left -= n
    buckets = rng.choice([0, 0, 16, 32, 64])
    return attention_case(kind, dtype, lengths, heads, kv_heads, dim, buckets, rng.choice([64, 128, 256, 500]) if buckets else 0)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return (prepare_attention if case["op"] == "attention" else prepare_policy)(case, g)


def normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEVICE).to(dtype)


def prepare_attention(case, g):
    dtype = DTYPES[case["dtype"]]
    lengths = [int(n) for n in case["lengths"].split(",")]
    tokens, heads, kv, dim = sum(lengths), case["heads"], case["kv_heads"], case["dim"]
    # query, key and value are what one projection wrote: views of a single [tokens, (heads + 2 kv) * dim] buffer
    qkv = normal(g, (tokens, heads + 2 * kv, dim), dtype)
    offsets = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=DEVICE)
    views = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    # tokens, heads, kv heads, head size, sequences, buckets, largest distance | strides of query, key, value | their offsets
    metadata = np.array([tokens, heads, kv, dim, len(lengths), case["buckets"], case["max_distance"],
                         *views[0].stride(), *views[1].stride(), *views[2].stride(), 0, 0, 0], dtype=np.uint64)
    return {"case": case, "offsets": offsets, "longest": max(lengths), "scale": dim ** -0.5, "metadata": metadata,
            "query": views[0], "key": views[1], "value": views[2],
            "bias": normal(g, (case["buckets"], heads), dtype) if case["buckets"] else None,
            "grad_output": normal(g, (tokens, heads, dim), dtype) if case["kind"] == "step" else None}


CLIP_LOW, CLIP_HIGH, KL_WEIGHT = 0.2, 0.25, 0.05


def prepare_policy(case, g):
    dtype = DTYPES[case["dtype"]]
    rows, vocab = case["rows"], case["vocab"]
    logits = (2.0 * normal(g, (rows, vocab))).to(dtype)
    # actions drawn from the policy itself
    noise = torch.empty((rows, vocab), device=DEVICE).exponential_(generator=g)
    x = logits.float()
    target = (x - noise.log_()).argmax(1)
    logp = x.gather(1, target[:, None])[:, 0] - torch.logsumexp(x, 1)
    del x, noise
    # the policy has moved since the answers were sampled, some of it beyond the clip range.  A ratio that lies on the
    # border to within rounding has no one gradient: such rows are moved off it.
    step = 0.2 * normal(g, (rows,))
    for border in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
        step = torch.where((step - border).abs() < 1e-3, step + 0.01, step)
    active = torch.zeros(rows, device=DEVICE)
    active[torch.randperm(rows, generator=g, device=DEVICE)[:active_rows(case)]] = 1.0
    return {"case": case, "logits": logits, "target": target, "old_logp": logp - step, "ref_logp": logp + 0.2 * normal(g, (rows,)),
            "advantage": normal(g, (rows,)), "weight": active / active_rows(case),
            # rows, vocabulary | strides of the logits | their offset
            "metadata": np.array([rows, vocab, *logits.stride(), 0], dtype=np.uint64)}


def active_rows(case):
    return max(1, round(case["rows"] * case["share"]))


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    if s["case"]["op"] == "attention":
        return attention_own(s) if own else attention_plain(s)
    return policy_own(s) if own else policy_plain(s)


def use_current_stream():
    from maidenx_amd import lib
    lib.load().hip_set_stream(torch.cuda.current_stream().cuda_stream)
    return lib


def attention_own(s):
    lib = use_current_stream()
    q, k, v, bias, dtype = s["query"], s["key"], s["value"], s["bias"], s["case"]["dtype"]
    table = bias.data_ptr() if bias is not None else None
    output = torch.empty(q.shape, dtype=q.dtype, device=DEVICE)
    lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=DEVICE)
    common = (s["metadata"], s["offsets"].data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), table, s["scale"])
    lib.call("attention_" + dtype, *common, output.data_ptr(), lse.data_ptr())
    if s["grad_output"] is None:
        return {"output": output, "lse": lse}
    gq, gk, gv = (torch.empty(t.shape, dtype=t.dtype, device=DEVICE) for t in (q, k, v))
    gb = torch.empty_like(bias) if bias is not None else None
    lib.call("attention_backward_" + dtype, *common, output.data_ptr(), lse.data_ptr(), s["grad_output"].data_ptr(),
             gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), gb.data_ptr() if gb is not None else None)
    return {"output": output, "grad_query": gq, "grad_key": gk, "grad_value": gv, "grad_bias": gb}


def policy_own(s):
    lib = use_current_stream()
    x, suffix = s["logits"], s["case"]["dtype"] + "_i64"
    loss = torch.empty(1, device=DEVICE)
    logp = torch.empty(x.shape[0], device=DEVICE)
    lse = torch.empty(x.shape[0], device=DEVICE)
    common = (s["metadata"], s["target"].data_ptr(), x.data_ptr(), s["old_logp"].data_ptr(), s["ref_logp"].data_ptr(),
              s["advantage"].data_ptr(), s["weight"].data_ptr(), CLIP_LOW, CLIP_HIGH, KL_WEIGHT)
    if s["case"]["kind"] == "forward":
        lib.call("policy_loss_" + suffix, *common, loss.data_ptr(), logp.data_ptr(), lse.data_ptr())
        return {"loss": loss, "logp": logp, "lse": lse}
    grad = torch.empty_like(x)
    lib.call("policy_loss_step_" + suffix, *common, None, loss.data_ptr(), logp.data_ptr(), lse.data_ptr(), grad.data_ptr())
    return {"loss": loss, "logp": logp, "grad_logits": grad}


# ---- plain forms ----------------------------------------------------------------------------------------------------
def bucket_of(distance, buckets, max_distance):
    """Distances below buckets / 2 have a bucket each, the others share the rest by their logarithm.  In 64 bits; the
    small term keeps a distance that lies on a border (where the quotient is a whole number) in the bucket it opens."""
    exact_to = buckets // 2
    far = (distance.clamp(min=exact_to).double() / exact_to).log() / math.log(max_distance / exact_to) * (buckets - exact_to)
    return torch.where(distance < exact_to, distance, (exact_to + (far + 1e-9).floor().long()).clamp(max=buckets - 1))


def attention_plain(s):
    c, tokens, longest = s["case"], s["query"].shape[0], s["longest"]
    heads, kv, dim = c["heads"], c["kv_heads"], c["dim"]
    starts, ends = s["offsets"][:-1].long(), s["offsets"][1:].long()
    place = torch.arange(longest, device=DEVICE)
    padded = (starts[:, None] + place).clamp(max=tokens - 1)                       # [sequences, longest] -> token
    inside = place < (ends - starts)[:, None]
    token = torch.arange(tokens, device=DEVICE)
    sequence = torch.searchsorted(ends, token, right=True)
    back = (sequence, slice(None), token - starts[sequence])                       # token -> [sequence, :, place]

    def lay_out(t):                                                                # [tokens, n, dim] -> [sequences, heads, longest, dim]
        t = t.float()[padded].transpose(1, 2)
        return t.repeat_interleave(heads // t.shape[1], 1).contiguous()

    def gather(t, n):                                                              # the inverse; shared heads are summed
        return t.unflatten(1, (n, heads // n)).sum(2)[back]

    q, k, v = lay_out(s["query"]), lay_out(s["key"]), lay_out(s["value"])
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s["scale"])
    distance = place[:, None] - place
    if c["buckets"]:
        bucket = bucket_of(distance.clamp(min=0), c["buckets"], c["max_distance"])
        scores += s["bias"].float().t()[:, bucket]
    hidden = (distance < 0) | ~inside[:, None, None, :]
    scores.masked_fill_(hidden, -math.inf)
    top = scores.amax(3, keepdim=True)
    p = scores.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    p /= total
    o = torch.matmul(p, v)
    output = gather(o, heads).to(s["query"].dtype)
    if s["grad_output"] is None:
        lse = (top + total.log())[back[0], :, back[2], 0].t().contiguous()
        return {"output": output, "lse": lse}
    do = lay_out(s["grad_output"]) * inside[:, None, :, None]
    gv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds -= (do * o).sum(3, keepdim=True)
    ds *= p
    gq = torch.matmul(ds, k).mul_(s["scale"])
    gk = torch.matmul(ds.transpose(2, 3).contiguous(), q).mul_(s["scale"])
    gb = None
    if c["buckets"]:
        # row i of [longest, 2 longest] starts i places later in rows that are one place shorter: distances become columns.
        # Summed in 64 bits.
        by_pair = ds.sum(0, dtype=torch.float64).masked_fill_(distance < 0, 0.0).flip(2)
        skewed = torch.nn.functional.pad(by_pair, (0, longest)).flatten(1)[:, :longest * (2 * longest - 1)]
        by_distance = skewed.unflatten(1, (longest, 2 * longest - 1)).sum(1)[:, longest - 1:]
        gb = torch.zeros((heads, c["buckets"]), dtype=torch.float64, device=DEVICE)
        gb = gb.index_add_(1, bucket[:, 0], by_distance).t().to(s["bias"].dtype).contiguous()
    dtype = s["query"].dtype
    return {"output": output, "grad_query": gather(gq, heads).to(dtype), "grad_key": gather(gk, kv).to(dtype),
            "grad_value": gather(gv, kv).to(dtype), "grad_bias": gb}


def policy_plain(s):
    x = s["logits"].float()
    on = s["weight"] != 0
    at = s["target"][:, None]
    top = x.amax(1, keepdim=True)
    p = (x - top).exp_()
    total = p.sum(1, keepdim=True)
    logp = (x.gather(1, at) - top - total.log())[:, 0]
    ratio = (logp - s["old_logp"]).exp()
    plain, clipped = ratio * s["advantage"], ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * s["advantage"]
    away = s["ref_logp"] - logp
    loss = (s["weight"] * (KL_WEIGHT * (torch.expm1(away) - away) - torch.minimum(plain, clipped))).sum().reshape(1)
    logp = torch.where(on, logp, torch.zeros_like(logp))
    if s["case"]["kind"] == "forward":
        lse = torch.where(on, (top + total.log())[:, 0], torch.zeros_like(logp))
        return {"loss": loss, "logp": logp, "lse": lse}
    g = s["weight"] * (-KL_WEIGHT * torch.expm1(away) - torch.where(plain <= clipped, plain, torch.zeros_like(plain)))
    grad = p.mul_(-g[:, None] / total)
    grad.scatter_add_(1, at, g[:, None])
    return {"loss": loss, "logp": logp, "grad_logits": grad.to(s["logits"].dtype)}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    step = case["kind"] == "step"
    if case["op"] == "policy":
        moved = active_rows(case) * case["vocab"] * size + (case["rows"] * case["vocab"] * size if step else 0)
        return {"bytes": moved + case["rows"] * (8 + 4 * 5) + 4, "flops": (7 if step else 4) * active_rows(case) * case["vocab"]}
    lengths = [int(n) for n in case["lengths"].split(",")]
    tokens, heads, kv, dim = sum(lengths), case["heads"], case["kv_heads"], case["dim"]
    pairs = sum(n * (n + 1) // 2 for n in lengths)
    table = case["buckets"] * heads * size
    forward = tokens * (heads + 2 * kv) * dim * size + tokens * heads * dim * size + table
    if not step:
        return {"bytes": forward + tokens * heads * 4, "flops": 4 * pairs * heads * dim}
    # q, k, v, the gradient of the output and the table read once; output and all gradients written once
    return {"bytes": forward + tokens * heads * dim * size + tokens * (heads + 2 * kv) * dim * size + table, "flops": 14 * pairs * heads * dim}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------
def exact(case, seed):
    def bucket_of(distance, buckets, max_distance):
        """Counts the bucket borders that a distance has reached: border m is the least n with (n/E)^M >= (X/E)^m, found
        in whole numbers."""
        exact_to = buckets // 2
        spread = buckets - exact_to
        borders, n = [], exact_to
        for m in range(1, spread):
            while n ** spread < max_distance ** m * exact_to ** (spread - m):
                n += 1
            borders.append(n)
        borders = torch.tensor(borders, device=distance.device, dtype=torch.long)
        return torch.where(distance < exact_to, distance, exact_to + torch.searchsorted(borders, distance, right=True))

    def attention(s):
        """Sequence by sequence and head by head of the keys, softmax and gradients from torch's own derivation in 64 bits."""
        c = s["case"]
        group = c["heads"] // c["kv_heads"]
        step = s["grad_output"] is not None
        names = ("query", "key", "value")
        full = {n: s[n].double().detach() for n in names}
        table = s["bias"].double() if c["buckets"] else None
        out = torch.zeros_like(full["query"])
        lse = torch.zeros((c["heads"], out.shape[0]), dtype=torch.float64, device=out.device)
        grads = {n: torch.zeros_like(full[n]) for n in names}
        table_grad = torch.zeros_like(table) if table is not None else None
        bounds = s["offsets"].tolist()
        for a, b in zip(bounds, bounds[1:]):
            if a == b:
                continue
            i = torch.arange(b - a, device=out.device)
            distance = i[:, None] - i
            bucket = bucket_of(distance.clamp(min=0), c["buckets"], c["max_distance"]) if table is not None else None
            for h in range(c["heads"]):
                with torch.enable_grad():
                    q, k, v = (full[n][a:b, h if n == "query" else h // group].clone().requires_grad_(step) for n in names)
                    scores = (q @ k.t()) * s["scale"]
                    if table is not None:
                        column = table[:, h].clone().requires_grad_(step)
                        scores = scores + column[bucket]
                    scores = scores.masked_fill(distance < 0, -math.inf)
                    o = torch.softmax(scores, 1) @ v
                    if step:
                        wanted = [q, k, v] + ([column] if table is not None else [])
                        got = torch.autograd.grad(o, wanted, s["grad_output"][a:b, h].double())
                        for n, d in zip(names, got):
                            grads[n][a:b, h if n == "query" else h // group] += d
                        if table is not None:
                            table_grad[:, h] += got[3]
                out[a:b, h] = o.detach()
                lse[h, a:b] = torch.logsumexp(scores.detach(), 1)
        if not step:
            return {"output": out, "lse": lse}
        return {"output": out, "grad_query": grads["query"], "grad_key": grads["key"], "grad_value": grads["value"], "grad_bias": table_grad}

    def policy(s):
        step = s["case"]["kind"] == "step"
        on = (s["weight"] != 0).nonzero()[:, 0]
        with torch.enable_grad():
            x = s["logits"][on].double().requires_grad_(step)
            logp = torch.log_softmax(x, 1).gather(1, s["target"][on][:, None])[:, 0]
            old, ref, advantage, weight = (s[n][on].double() for n in ("old_logp", "ref_logp", "advantage", "weight"))
            ratio = torch.exp(logp - old)
            gain = torch.minimum(ratio * advantage, torch.clamp(ratio, 1 - CLIP_LOW, 1 + CLIP_HIGH) * advantage)
            kl = torch.exp(ref - logp) - (ref - logp) - 1
            loss = (weight * (KL_WEIGHT * kl - gain)).sum()
            grad = torch.autograd.grad(loss, x)[0] if step else None
        every = torch.zeros(s["logits"].shape[0], dtype=torch.float64, device=x.device)
        every[on] = logp.detach()
        found = {"loss": loss.detach().reshape(1), "logp": every}
        if not step:
            found["lse"] = torch.zeros_like(every)
            found["lse"][on] = torch.logsumexp(x, 1)
        if step:
            found["grad_logits"] = torch.zeros(s["logits"].shape, dtype=torch.float64, device=x.device)
            found["grad_logits"][on] = grad
        return found

    s = prepare(case, seed)
    return attention(s) if case["op"] == "attention" else policy(s)
