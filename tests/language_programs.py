"""A small policy model on any host-layer library (maidenx_amd.tensor.Host) - projections, attention over packed sequences with a
learned position bias, a head, the clipped policy loss - and the same in 64-bit numpy."""
import math

import numpy as np

OFFSETS = [0, 7, 7, 19, 28]                 # an empty sequence, two tokens behind the last one
T, C, H, HK, D, V = 30, 12, 4, 2, 8, 17
BUCKETS, MAX_DISTANCE = 8, 16
CLIP, KL = (0.2, 0.25), 0.1
NAMES = ["wq", "bq", "wk", "wv", "table", "wo", "bo"]


def bucket(n, buckets=BUCKETS, far=MAX_DISTANCE):
    exact = buckets // 2
    return n if n < exact else min(buckets - 1, exact + int((buckets - exact) * math.log(n / exact) / math.log(far / exact) + 1e-12))


def plain_attention(q, k, v, offsets, bias=None, scale=None, far=MAX_DISTANCE):
    """q [T, H, D], k and v [T, Hk, D] in 64 bits; tokens of no sequence give zeros.  Returns the output and the largest |score|."""
    group, scale = q.shape[1] // k.shape[1], q.shape[2] ** -0.5 if scale is None else scale
    out, top = np.zeros(q.shape), 0.0
    for a, b in zip(offsets[:-1], offsets[1:]):
        for h in range(q.shape[1]):
            for i in range(a, b):
                s = scale * (k[a:i + 1, h // group] @ q[i, h])
                if bias is not None:
                    s = s + np.array([bias[bucket(i - j, len(bias), far), h] for j in range(a, i + 1)])
                top = max(top, np.abs(s).max())
                p = np.exp(s - s.max())
                out[i, h] = (p / p.sum()) @ v[a:i + 1, h // group]
    return out, top


def plain_policy(x, target, old, ref, adv, w, clip=CLIP, kl=KL):
    loss, logp = 0.0, np.zeros(len(x))
    x, old, ref, adv, w = (np.asarray(a, np.float64) for a in (x, old, ref, adv, w))
    for t in np.flatnonzero(w):
        lp = x[t, target[t]] - x[t].max() - math.log(np.exp(x[t] - x[t].max()).sum())
        r = math.exp(lp - old[t])
        loss += w[t] * (-min(r * adv[t], min(max(r, 1 - clip[0]), 1 + clip[1]) * adv[t]) + kl * (math.exp(ref[t] - lp) - (ref[t] - lp) - 1))
        logp[t] = lp
    return loss, logp


class Case:
    def __init__(self, seed=5):
        g = np.random.default_rng(seed)
        r = lambda *s: g.standard_normal(s).astype(np.float32)
        self.x = r(T, C)
        self.p = {"wq": r(H * D, C) / 4, "bq": r(H * D) / 4, "wk": r(HK * D, C) / 4, "wv": r(HK * D, C) / 2, "table": r(BUCKETS, H),
                  "wo": r(H * D, V) / 8, "bo": r(V) / 4}
        self.target = g.integers(0, V, T)
        self.weight = np.where(g.random(T) < 0.7, g.random(T), 0).astype(np.float32)
        self.weight[OFFSETS[-1]:] = 0
        self.target[self.weight == 0] = 99                     # (not read)
        self.old = self.ref = self.adv = np.zeros(T, np.float32)
        lp = plain_policy(self.logits(), self.target, self.old, self.ref, self.adv, self.weight)[1]
        self.old = (lp + 0.3 * r(T)).astype(np.float32)
        self.ref = (lp + 0.3 * r(T)).astype(np.float32)
        self.adv = r(T)
        ratio = np.exp(lp - self.old)[self.weight != 0]
        assert (np.abs(ratio - (1 - CLIP[0])) > 1e-3).all() and (np.abs(ratio - (1 + CLIP[1])) > 1e-3).all()     # away from the corners

    def logits(self, p=None, tops=None):
        p = {n: a.astype(np.float64) for n, a in (p or self.p).items()}
        x = self.x.astype(np.float64)
        o, top = plain_attention((x @ p["wq"].T + p["bq"]).reshape(T, H, D), (x @ p["wk"].T).reshape(T, HK, D), (x @ p["wv"].T).reshape(T, HK, D),
                                 OFFSETS, p["table"])
        y = o.reshape(T, H * D) @ p["wo"] + p["bo"]
        if tops is not None:
            tops += [top, np.abs(y).max()]
        return y

    def loss(self, p=None):
        return plain_policy(self.logits(p), self.target, self.old, self.ref, self.adv, self.weight)[0]

    def differences(self, name, entries, h=1e-5):
        """d loss / d p[name][entry] by central differences in 64 bits: off by about 1e-16 |loss| / h + h^2 |third derivative|, under 1e-8
        of the parameters' scale here."""
        out = []
        for e in entries:
            d = []
            for s in (h, -h):
                p = {n: a.astype(np.float64) for n, a in self.p.items()}
                p[name][e] += s
                d.append(self.loss(p))
            out.append((d[0] - d[1]) / (2 * h))
        return np.array(out)


class Model:
    """The case on a host library.  dtype is the parameters' and activations'."""

    def __init__(self, mx, case, dtype="f32"):
        self.mx, self.case = mx, case
        t = lambda a, g=False: mx.tensor(a, dtype=dtype).with_grad() if g else mx.tensor(a, dtype=dtype)
        self.x = t(case.x)
        self.q = mx.Linear(t(case.p["wq"]), t(case.p["bq"]))
        self.k, self.v = mx.Linear(t(case.p["wk"])), mx.Linear(t(case.p["wv"]))
        # (not a Linear: the reference's backward product reads a transposed weight as if it were not, so nothing flows back through one)
        self.wo, self.bo, self.table = (t(case.p[n], True) for n in ("wo", "bo", "table"))
        self.offsets, self.target = mx.indices(OFFSETS), mx.indices(case.target)
        self.old, self.ref, self.adv, self.weight = (mx.tensor(a) for a in (case.old, case.ref, case.adv, case.weight))
        self.modules, self.leaves = [self.q, self.k, self.v], [self.wo, self.bo, self.table]

    def logits(self):
        y = self.mx.attention(self.q.forward(self.x), self.k.forward(self.x), self.v.forward(self.x), self.offsets, bias=self.table,
                              max_distance=MAX_DISTANCE, heads=H, kv_heads=HK)
        return y.matmul(self.wo).add(self.bo)

    def loss(self, **kw):
        return self.mx.policy_loss(self.logits(), self.target, self.old, self.adv, self.weight, ref_logp=self.ref, clip_low=CLIP[0],
                                   clip_high=CLIP[1], kl_weight=KL, **kw)

    def parameters(self):
        return dict(wq=self.q.weight, bq=self.q.bias, wk=self.k.weight, wv=self.v.weight, table=self.table, wo=self.wo, bo=self.bo)

    def gradients(self):
        return {n: p.grad().numpy() for n, p in self.parameters().items()}

    def step(self, adams=None):
        self.loss().backward()
        for i, m in enumerate(self.modules):
            if adams:
                adams[i].step(m)
            else:
                m.sgd_step(0.05)
            m.zero_grad()
        for p in self.leaves:
            p.sub_(p.grad().mul_scalar(0.05))
            p.zero_grad()


def check_gradients(mx):
    """Loss, log-probabilities and the gradients of every parameter against 64 bits and its differences.

    f32: a rounding is 2^-24 of its value.  The longest path to a gradient goes through sums of C, D, 2 L, H D and V terms, forward and
    back, and some 50 roundings besides: n = 2 (C + D + 2 * 12 + H D + V + 50).  An error in an exponent counts as the exponent's value
    does: times 1 + the largest score and logit.  The bound is that share of the largest gradient of the parameter and of the largest
    logit's gradient, max weight * (|adv| r + KL |1 - exp(ref - lp)|), passed on by the head."""
    case = Case()
    m = Model(mx, case)
    loss, logp = m.loss(return_logp=True)
    tops = []
    want, want_logp = plain_policy(case.logits(tops=tops), case.target, case.old, case.ref, case.adv, case.weight)
    share = 2 * (C + D + 24 + H * D + V + 50) * 2.0 ** -24 * (1 + tops[0] + tops[1])
    ratio = np.exp(want_logp - case.old)
    each = case.weight * (np.abs(case.adv) * np.maximum(ratio, 2) + KL * (np.exp(case.ref - want_logp) + 1 + np.abs(case.ref - want_logp)))
    assert abs(loss.item() - want) <= share * each.sum()
    assert (np.abs(logp.numpy() - want_logp) <= share * (1 + np.abs(want_logp))).all()
    loss.backward()
    got = m.gradients()
    scale = {"wo": 1.0, "bo": 1.0}
    rng = np.random.default_rng(1)
    for name, g in got.items():
        flat = [tuple(i) for i in np.argwhere(np.ones(g.shape, bool))]
        entries = [flat[i] for i in rng.permutation(len(flat))[:24]]
        d = case.differences(name, entries)
        size = np.abs(g).max() + scale.get(name, np.abs(case.p["wo"]).sum(1).max()) * each.max()
        assert size > 0 and np.abs(g).max() > 1e-3, name
        off = np.abs(np.array([g[e] for e in entries]) - d)
        assert (off <= share * size + 1e-7).all(), (name, off.max(), share * size)


def check_seeds(mx):
    """The gradient of a scaled loss is the scaled gradient (one product more), a second backward pass adds the same again."""
    case = Case()
    a, b, c = Model(mx, case), Model(mx, case), Model(mx, case)
    a.loss().backward()
    b.loss().mul_scalar(4.0).backward()
    loss = c.loss()
    loss.backward()
    loss.backward()
    one, four, two = a.gradients(), b.gradients(), c.gradients()
    for n in one:
        size = np.abs(one[n]).max()
        np.testing.assert_allclose(four[n], 4 * one[n], rtol=0, atol=4 * 400 * 2.0 ** -24 * size, err_msg=n)
        if n in ("wo", "bo"):      # (the inner tensors' own gradients add up as well, and are not passed on twice)
            np.testing.assert_allclose(two[n], 2 * one[n], rtol=0, atol=2 * 400 * 2.0 ** -24 * size, err_msg=n)


def check_layouts(mx):
    """[tokens, heads * dim], [tokens, heads, dim] and a transposed view of [heads, tokens, dim] are the same call, bit for bit; tokens of no
    sequence are zeros."""
    g = np.random.default_rng(2)
    for dtype in ("f32", "bf16"):
        q, k, v = (g.standard_normal((T, h, D)).astype(np.float32) for h in (H, HK, HK))
        off = mx.indices([2, 9, 25])
        a = mx.attention(*(mx.tensor(x, dtype=dtype) for x in (q, k, v)), off)
        b = mx.attention(*(mx.tensor(x.reshape(T, -1), dtype=dtype) for x in (q, k, v)), off, heads=H, kv_heads=HK)
        c = mx.attention(*(mx.tensor(x.transpose(1, 0, 2), dtype=dtype).transpose(0, 1) for x in (q, k, v)), off)
        assert a.shape == c.shape == (T, H, D) and b.shape == (T, H * D) and a.dtype == dtype
        np.testing.assert_array_equal(a.numpy(), b.numpy().reshape(T, H, D))
        np.testing.assert_array_equal(a.numpy(), c.numpy())
        rounded = [mx.tensor(x, dtype=dtype).numpy().astype(np.float64) for x in (q, k, v)]
        want, top = plain_attention(*rounded, [2, 9, 25])
        # P and the output are rounded to the tensors' type (2^-8 for bf16, 2^-24), the rest in f32 over D and 16 terms
        eps = 2.0 ** (-8 if dtype == "bf16" else -24)
        tol = (2 * eps + 2 * (D + 16 + 8) * 2.0 ** -24 * (1 + top)) * np.abs(rounded[2]).max()
        assert np.abs(a.numpy() - want).max() <= tol
        assert (a.numpy()[:2] == 0).all() and (a.numpy()[25:] == 0).all()


def check_gradient_layouts(mx):
    """Gradients reach leaves through transposed views, rows of no sequence get zeros, and an operand without a gradient gets none."""
    g = np.random.default_rng(3)
    q, k, v = (g.standard_normal((T, h, D)).astype(np.float32) for h in (H, HK, HK))
    w = mx.tensor(g.standard_normal((T, H, D)).astype(np.float32))
    off = mx.indices([2, 9, 25])
    a = [mx.tensor(x).with_grad() for x in (q, k, v)]
    mx.attention(*a, off).mul(w).sum_all().backward()
    b = [mx.tensor(x.transpose(1, 0, 2)).with_grad() for x in (q, k, v)]
    mx.attention(*(x.transpose(0, 1) for x in b), off).mul(w).sum_all().backward()
    for x, y in zip(a, b):
        np.testing.assert_array_equal(x.grad().numpy(), y.grad().numpy().transpose(1, 0, 2))
        assert (x.grad().numpy()[:2] == 0).all() and (x.grad().numpy()[25:] == 0).all() and np.abs(x.grad().numpy()).max() > 0
    c = [mx.tensor(q), mx.tensor(k).with_grad(), mx.tensor(v)]
    mx.attention(*c, off).mul(w).sum_all().backward()
    np.testing.assert_array_equal(c[1].grad().numpy(), a[1].grad().numpy())
    assert c[0].grad() is None and c[2].grad() is None


def check_bf16_model(mx):
    """The model in bf16 runs, its loss is near the f32 one (activations are rounded to 2^-8 some ten times on the way to a logit) and its
    gradients are finite and of their parameters' type."""
    case = Case()
    m = Model(mx, case, "bf16")
    tops = []
    case.logits(tops=tops)
    loss = m.loss()
    assert loss.dtype == "f32"
    each = case.weight * (np.abs(case.adv) * 3 + KL * 3)
    assert abs(loss.item() - case.loss()) <= 10 * 2.0 ** -8 * (1 + tops[0] + tops[1]) * each.sum()
    loss.backward()
    for n, p in m.parameters().items():
        assert p.grad().dtype == "bf16" and np.isfinite(p.grad().numpy()).all() and np.abs(p.grad().numpy()).max() > 0, n


def refusals(mx):
    """(call, kind of the error)"""
    z = lambda *s, **k: mx.zeros(s, **k)
    off, ten = mx.indices([0, 10]), z(10)
    at = mx.attention
    shared = mx.tensor(np.zeros((10, 2, 8), np.float32)).with_grad()
    tgt = mx.indices(list(range(10)))
    pl = lambda x=None, t=tgt, o=ten, a=ten, w=ten, **k: mx.policy_loss(z(10, 11) if x is None else x, t, o, a, w, **k)
    return [
        (lambda: at(z(10, 2, 8), z(9, 2, 8), z(10, 2, 8), off), "InvalidShape"),
        (lambda: at(z(10), z(10), z(10), off), "InvalidShape"),
        (lambda: at(z(10, 16), z(10, 16), z(10, 16), off), "InvalidShape"),
        (lambda: at(z(10, 16), z(10, 16), z(10, 16), off, heads=3, kv_heads=3), "InvalidShape"),
        (lambda: at(z(10, 2, 8), z(10, 2, 8), z(10, 2, 8), off, heads=4), "InvalidShape"),
        (lambda: at(z(10, 3, 8), z(10, 2, 8), z(10, 2, 8), off), "ShapeMismatch"),
        (lambda: at(z(10, 2, 8), z(10, 2, 8), z(10, 1, 8), off), "ShapeMismatch"),
        (lambda: at(z(10, 2, 8), z(10, 2, 4), z(10, 2, 8), off), "ShapeMismatch"),
        (lambda: at(z(10, 2, 130), z(10, 2, 130), z(10, 2, 130), off), "ShapeMismatch"),
        (lambda: at(z(10, 2, 8), z(10, 2, 8), z(10, 2, 8, dtype="bf16"), off), "UnsupportedDType"),
        (lambda: at(z(10, 2, 8), z(10, 2, 8), z(10, 2, 8), off, bias=z(8, 3), max_distance=16), "ShapeMismatch"),
        (lambda: at(z(10, 2, 8), z(10, 2, 8), z(10, 2, 8), off, bias=z(1, 2), max_distance=16), "ShapeMismatch"),
        (lambda: at(z(10, 2, 8), z(10, 2, 8), z(10, 2, 8), off, bias=z(8, 2), max_distance=4), "InvalidArgument"),
        (lambda: at(z(10, 2, 8), z(10, 2, 8), z(10, 2, 8), off, bias=z(8, 2), max_distance=5000), "InvalidArgument"),
        (lambda: at(z(10, 2, 8), z(10, 2, 8), z(10, 2, 8), off, bias=z(8, 2, dtype="bf16"), max_distance=16), "UnsupportedDType"),
        (lambda: at(z(10, 2, 8), z(10, 2, 8), z(10, 2, 8), mx.indices([0, 11])), "InvalidArgument"),
        (lambda: at(z(10, 2, 8), z(10, 2, 8), z(10, 2, 8), mx.indices([0, 5, 3])), "InvalidArgument"),
        (lambda: at(z(10, 2, 8), z(10, 2, 8), z(10, 2, 8), mx.indices([-1, 5])), "InvalidArgument"),
        (lambda: at(z(10, 2, 8), z(10, 2, 8), z(10, 2, 8), mx.indices([])), "InvalidArgument"),
        (lambda: at(shared, shared, z(10, 2, 8), off), "InvalidOperation"),
        (lambda: mx.indices([0.5]), "InvalidArgument"),
        (lambda: mx.indices([2**31]), "InvalidArgument"),
        (lambda: pl(z(10)), "InvalidShape"),
        (lambda: pl(t=mx.indices([1, 2])), "ShapeMismatch"),
        (lambda: pl(o=z(9)), "ShapeMismatch"),
        (lambda: pl(w=z(10, 1)), "ShapeMismatch"),
        (lambda: pl(a=z(10, dtype="bf16")), "UnsupportedDType"),
        (lambda: pl(o=z(10).with_grad()), "InvalidOperation"),
        (lambda: pl(clip_low=-0.1), "InvalidArgument"),
        (lambda: pl(clip_high=float("nan")), "InvalidArgument"),
        (lambda: pl(kl_weight=0.1), "InvalidArgument"),
    ]


def check_nothing(mx):
    """No tokens, no sequences, no rows."""
    q = mx.zeros((0, 2, 8)).with_grad()
    y = mx.attention(q, mx.zeros((0, 2, 8)), mx.zeros((0, 2, 8)), mx.indices([0]))
    assert y.shape == (0, 2, 8)
    y = mx.attention(mx.ones((3, 2, 8)), mx.ones((3, 2, 8)), mx.ones((3, 2, 8)), mx.indices([1]))
    assert (y.numpy() == 0).all()
    assert mx.policy_loss(mx.zeros((0, 5)), mx.indices([]), *(mx.zeros((0,)) for _ in range(3))).item() == 0.0
