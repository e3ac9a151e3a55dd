"""CPU: the oracle's attention and policy loss against plain numpy in 64 bits and against differences, and the refusals of the
library's entry points (which are decided on the host)."""

import numpy as np
import pytest

import maidenx_amd.lib as L
from language import Attention, Policy, bind, borders, bucket_of, meta_attention
from helpers import Runner, u64


@pytest.fixture(scope="module")
def orc():
    return bind(Runner("oracle"))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", [
    dict(lengths=[5, 1, 0, 9], heads=2, kv=1, dim=8), dict(lengths=[17], heads=3, kv=3, dim=5, buckets=8, distance=12, lead=2, tail=3),
    dict(lengths=[40, 3], heads=4, kv=2, dim=4, buckets=7, distance=20, layout="fused"), dict(lengths=[6, 6], heads=2, kv=2, dim=3, layout="elements first", scale=-0.7)])
def test_oracle_attention_is_the_formula(orc, dt, case):
    Attention(dt, **case).check(orc)


@pytest.mark.parametrize("dt,rows,vocab,layout", [("f32", 7, 33, "packed"), ("bf16", 5, 20, "rows apart"), ("f16", 6, 9, "transposed"), ("f32", 1, 1, "packed")])
def test_oracle_policy_loss_is_the_formula(orc, dt, rows, vocab, layout):
    Policy(dt, rows, vocab, layout=layout, seed=3).check(orc)


def test_oracle_attention_gradients_are_the_differences(orc):
    """d/dx of sum(output * go), by central differences in f64 through numpy's forward pass."""
    a = Attention("f32", [6, 3], 2, 1, 4, buckets=4, distance=5, seed=8)
    want, _ = a.exact()

    def value():
        return float((a.exact()[0]["o"] * a.go).sum())
    step = 1e-5
    for tensor, grad in ((a.q, "gq"), (a.k, "gk"), (a.v, "gv"), (a.table, "gt")):
        flat = tensor.reshape(-1)
        for i in range(0, flat.size, 3):
            kept = flat[i]
            flat[i] = kept + step
            up = value()
            flat[i] = kept - step
            down = value()
            flat[i] = kept
            assert abs((up - down) / (2 * step) - want[grad].reshape(-1)[i]) < 1e-7


def test_oracle_policy_gradient_is_the_differences(orc):
    p = Policy("f32", 6, 5, seed=9, share=1.0)
    want = p.exact()[0]["grad"]
    for r in range(p.rows):
        for v in range(p.vocab):
            kept, sides = p.x[r, v], []
            for d in (1e-5, -1e-5):
                p.x[r, v] = kept + d
                sides.append(p.exact()[0]["loss"][0])
            p.x[r, v] = kept
            assert abs((sides[0] - sides[1]) / 2e-5 - want[r, v]) < 1e-7


def test_bucket_borders():
    """32 buckets to 256: the quotient of the logarithms is a whole number at 32, 64 and 128, which begin their buckets."""
    assert borders(32, 256)[16:] == [16, 20, 23, 27, 32, 39, 46, 54, 64, 77, 91, 108, 128, 153, 182, 216]
    assert [int(b) for b in bucket_of(np.array([0, 15, 16, 31, 32, 127, 128, 255, 256, 10 ** 6]), 32, 256)] == [0, 15, 16, 19, 20, 27, 28, 31, 31, 31]


def status(name, *args):
    L.load().hip_get_last_status()                   # what earlier tests left
    L.call(name, *args)
    return L.load().hip_get_last_status(), L.load().hip_status_string().decode()


def attention_args(dt="f32", heads=4, kv=2, dim=8, tokens=16, sequences=1, buckets=0, distance=0, **over):
    """Pointers that are never read: every refusal comes before anything is queued."""
    md = meta_attention(tokens, heads, kv, dim, sequences, buckets, distance, [heads * dim, dim, 1], [kv * dim, dim, 1], [kv * dim, dim, 1])
    a = {"md": md, "offsets": 256, "q": 512, "k": 1024, "v": 2048, "table": 4096 if buckets else None, "scale": 1.0, "out": 8192, "lse": 16384}
    a.update(over)
    return [a[n] for n in ("md", "offsets", "q", "k", "v", "table", "scale", "out", "lse")]


INVALID, TOO_LARGE, UNSUPPORTED = 1, 3, 5


@pytest.mark.parametrize("over,code,text", [
    ({"md": None}, INVALID, "null"), ({"offsets": None}, INVALID, "null"), ({"q": None}, INVALID, "null"), ({"k": None}, INVALID, "null"),
    ({"v": None}, INVALID, "null"), ({"out": None}, INVALID, "null"), ({"lse": None}, INVALID, "null"),
    ({"heads": 5}, INVALID, "multiple"), ({"kv": 0}, INVALID, "multiple"), ({"dim": 0}, INVALID, "dim"), ({"heads": 0}, INVALID, "multiple"),
    ({"dim": 129}, UNSUPPORTED, "128"), ({"tokens": 2 ** 31}, TOO_LARGE, "tokens"), ({"sequences": 2 ** 31}, TOO_LARGE, "sequences"),
    ({"buckets": 1, "distance": 8}, UNSUPPORTED, "buckets"), ({"buckets": 257, "distance": 1000}, UNSUPPORTED, "buckets"),
    ({"buckets": 32, "distance": 16}, UNSUPPORTED, "max_distance"), ({"buckets": 32, "distance": 4097}, UNSUPPORTED, "max_distance"),
])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_attention_refuses(dt, over, code, text):
    got, said = status("attention_" + dt, *attention_args(dt, **over))
    assert got == code and text in said, (got, said)
    if not {"out", "lse"} & set(over):
        md, off, q, k, v, table, scale, out, lse = attention_args(dt, **over)
        got, said = status("attention_backward_" + dt, md, off, q, k, v, table, scale, out, lse, 100, 200, 300, 400, None)
        assert got == code and text in said, (got, said)


def test_attention_backward_refuses():
    args = attention_args()
    for at in (0, 1, 2):                                    # output, lse, grad_output
        rest = [8192, 16384, 100, 200, 300, 400, None]
        rest[at] = None
        got, said = status("attention_backward_f32", *args[:7], *rest)
        assert got == INVALID and "null" in said
    got, said = status("attention_backward_f32", *args[:7], 8192, 16384, 100, 200, 300, 400, 500)
    assert got == INVALID and "bias that was not given" in said


def policy_args(rows=4, vocab=10, low=0.2, high=0.2, beta=0.1, **over):
    a = {"md": u64(rows, vocab, vocab, 1, 0), "target": 256, "x": 512, "old": 1024, "ref": 2048, "adv": 4096, "w": 8192}
    a.update(over)
    return [a[n] for n in ("md", "target", "x", "old", "ref", "adv", "w")] + [low, high, beta]


@pytest.mark.parametrize("over,code,text", [
    ({"md": None}, INVALID, "null"), ({"target": None}, INVALID, "null"), ({"x": None}, INVALID, "null"), ({"old": None}, INVALID, "null"),
    ({"adv": None}, INVALID, "null"), ({"w": None}, INVALID, "null"), ({"ref": None}, INVALID, "ref_logp"), ({"low": -0.1}, INVALID, "clip"),
    ({"high": float("nan")}, INVALID, "clip"), ({"vocab": 0}, INVALID, "vocabulary"), ({"rows": 2 ** 31}, TOO_LARGE, "rows"), ({"vocab": 2 ** 31}, TOO_LARGE, "rows"),
])
@pytest.mark.parametrize("suffix", ["f32_i32", "bf16_i64", "f16_i32"])
def test_policy_loss_refuses(suffix, over, code, text):
    args = policy_args(**over)
    for name, rest in (("policy_loss_", [10, 20, 30]), ("policy_loss_step_", [None, 10, 20, 30, 40]), ("policy_loss_backward_", [20, 30, None, 40])):
        got, said = status(name + suffix, *args, *rest)
        assert got == code and text in said, (name, got, said)


def test_policy_loss_refuses_null_outputs():
    for name, rest in (("policy_loss_f32_i32", [10, 20, 30]), ("policy_loss_step_f32_i32", [10, 20, 30, 40]), ("policy_loss_backward_f32_i32", [20, 30, 40])):
        for at in range(len(rest)):
            args = list(rest)
            args[at] = None
            if "step" in name:
                args = [None] + args
            if "backward" in name:
                args = args[:2] + [None] + args[2:]
            got, said = status(name, *policy_args(), *args)
            assert got == INVALID and "null" in said, (name, at)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_attention_refuses_more_threads_than_a_launch_takes(dt):
    for tokens, heads in ((2 ** 27, 16), (33000, 65028), (128 * 257, 65535), (2 ** 31 - 2048, 2)):
        got, said = status("attention_" + dt, *attention_args(dt, tokens=tokens, heads=heads, kv=heads))
        assert got == TOO_LARGE and "tiles" in said, (tokens, heads, got, said)


@pytest.mark.parametrize("suffix,size", [("f32_i32", 4), ("bf16_i64", 2), ("f16_i32", 2)])
@pytest.mark.parametrize("strides", [(10, 1), (12, 1), (1, 4), (2 ** 64 - 10, 1), (10, 2 ** 64 - 1)])
def test_policy_loss_refuses_a_gradient_in_place(suffix, size, strides):
    """Rows and elements in either direction; the gradient begins at the logits' first byte, at their last, or ends in them."""
    low, high = 0, 0
    for n, s in ((4, strides[0]), (10, strides[1])):
        end = (n - 1) * (s if s < 2 ** 63 else s - 2 ** 64)
        low, high = low + min(end, 0), high + max(end, 0)
    at = 2 ** 20
    args = policy_args(x=at, md=u64(4, 10, list(strides), 0))
    for grad in (at + low * size, at + high * size, at + (low - 39) * size):
        for name, rest in (("policy_loss_step_", [None, 10, 20, 30, grad]), ("policy_loss_backward_", [20, 30, None, grad])):
            got, said = status(name + suffix, *args, *rest)
            assert got == INVALID and "overlaps" in said, (name, grad - at, got, said)
