"""The clipped policy loss on the GPU against plain numpy in 64 bits; every bound is derived in language.py."""
import ctypes as C

import numpy as np
import pytest

import maidenx_amd.lib as L
from helpers import In, Null, Out, to_float, u64
from language import Policy

pytestmark = pytest.mark.gpu
ALL = ["f32", "bf16", "f16"]


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 7), (37, 1000), (300, 33), (1, 5000), (5, 4099), (260, 4097), (3, 40001), (17, 16384), (300, 12289)])
def test_sizes(hip, dt, rows, vocab):
    Policy(dt, rows, vocab, seed=vocab).check(hip)


# one size at least for each form a row can take: held in registers by 256, 512 and 1024 threads, read twice, cut in parts
@pytest.mark.parametrize("dt,rows,vocab", [("f32", 256, 2040), ("f32", 256, 2049), ("f32", 256, 8190), ("f32", 256, 16390), ("f32", 256, 33001), ("bf16", 256, 66001), ("f16", 257, 33000),
                                           ("f32", 2, 300001), ("bf16", 1, 1000003), ("f16", 255, 9001)])
def test_forms(hip, dt, rows, vocab):
    Policy(dt, rows, vocab, seed=rows, share=0.5).check(hip)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("layout", ["rows apart", "transposed"])
@pytest.mark.parametrize("rows,vocab", [(5, 70), (300, 65), (4, 9001), (260, 4500)])
def test_layouts(hip, dt, layout, rows, vocab):
    Policy(dt, rows, vocab, layout=layout, it="i32", seed=1).check(hip)


@pytest.mark.parametrize("grad_loss", [0.0, 1.0, -2.5, 1e-4])
def test_the_gradient_of_the_loss(hip, grad_loss):
    for rows, vocab in ((40, 300), (3, 20000)):
        p = Policy("f32", rows, vocab, seed=2)
        p.grad_loss = grad_loss
        p.check(hip)


@pytest.mark.parametrize("beta,low,high", [(0.0, 0.2, 0.2), (0.3, 0.0, 0.0), (0.01, 0.9, 5.0), (1.0, 0.2, 0.28)])
def test_coefficients(hip, beta, low, high):
    Policy("bf16", 60, 500, beta=beta, low=low, high=high, seed=3).check(hip)


@pytest.mark.parametrize("rows,vocab", [(50, 64), (7, 30000)])
def test_rows_that_do_not_count_are_not_read(hip, rows, vocab):
    """Weight zero: NaN logits and targets out of range are nothing to the loss, and their gradient is zero."""
    p = Policy("f32", rows, vocab, seed=4)
    off = p.weight == 0
    assert off.any() and not off.all()
    want, bound = p.exact()
    p.x[off] = np.nan
    p.target[off] = -100
    loss, logp, lse, grad = p.step(hip)
    for name, got in (("loss", loss), ("logp", logp), ("lse", lse)):
        p.close(got, want[name], bound[name], name)
    assert (grad[off] == 0).all() and not np.signbit(grad[off]).any()
    p.close(grad[~off], want["grad"][~off], bound["grad"][~off], "grad")
    assert p.backward(hip, logp, lse).tobytes() == p.backward(hip, logp, lse).tobytes()
    assert (p.backward(hip, logp, lse)[off] == 0).all()


@pytest.mark.parametrize("rows,vocab", [(20, 50), (3, 20000)])
def test_no_row_counts(hip, rows, vocab):
    p = Policy("bf16", rows, vocab, share=0.0, seed=5)
    loss, logp, lse, grad = p.step(hip)
    assert loss[0] == 0 and (logp == 0).all() and (lse == 0).all() and (to_float(grad, "bf16") == 0).all()


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("rows,vocab", [(30, 200), (3, 9000)])
def test_logits_taken_out(hip, dt, rows, vocab):
    """-inf (or the type's lowest value) in most places, also in whole 16-byte pieces: their probability and gradient are zero."""
    p = Policy(dt, rows, vocab, seed=6)
    lowest = {"f32": np.float64(np.finfo(np.float32).min), "bf16": -3.3895313892515355e38, "f16": -65504.0}[dt]
    r = np.random.default_rng(6)
    keep = np.zeros((rows, vocab), bool)
    keep[:, r.integers(0, vocab, 40)] = True
    keep[np.arange(rows), p.target] = True
    q = Policy(dt, rows, vocab, seed=6)
    q.x = np.where(keep, p.x, np.where(r.random((rows, vocab)) < 0.5, -np.inf, lowest))
    lp = q.x[np.arange(rows), q.target] - q.log_sum(q.x)
    q.old = (lp - 0.1).astype(np.float32)
    q.ref = (lp + 0.1).astype(np.float32)
    want, bound = q.exact()
    # the bound of lse goes by the largest finite logit that matters, not by the lowest value
    small = np.abs(p.x).max(1)
    q2 = Policy(dt, rows, vocab, seed=6)
    q2.x, q2.old, q2.ref = np.where(keep, p.x, -50.0 - small[:, None]), q.old, q.ref
    _, bound = q2.exact()
    loss, logp, lse, grad = q.step(hip)
    for name, got in (("loss", loss), ("logp", logp), ("lse", lse)):
        q.close(got, want[name], bound[name], name)
    q.close(grad, want["grad"], np.where(keep, bound["grad"], 0.0), "grad")


def test_targets_out_of_range_are_reported(hip):
    for rows, vocab in ((30, 100), (4, 20000)):
        for bad in (-1, vocab, 2 ** 40):
            p = Policy("f32", rows, vocab, share=1.0, seed=7)
            p.weight[:] = 1.0
            p.target[2] = bad
            for call in (lambda: p.forward(hip), lambda: p.step(hip), lambda: p.backward(hip, np.zeros(rows, np.float32), np.zeros(rows, np.float32))):
                with pytest.raises(L.HipError, match="targets of policy_loss"):
                    call()


def test_no_rows(hip):
    """The loss of no rows is zero (as after a step whose every prompt was dropped); nothing else is written."""
    p = Policy("f32", 1, 5, seed=8)
    args = p.arguments()
    args[0] = u64(0, 5, 5, 1, 0)
    loss, logp, lse, grad = hip.call(p.name("_step"), *args, Null(), Out(1, "f32"), Out(1, "f32"), Out(1, "f32"), Out(5, "f32"))
    assert loss[0] == 0
    assert all((a.view(np.uint8) == 0xCD).all() for a in (logp, lse, grad))


def test_the_same_bits_on_every_call(hip):
    for rows, vocab in ((300, 5001), (3, 50001)):
        p = Policy("bf16", rows, vocab, seed=9)
        first = [a.tobytes() for a in p.step(hip)]
        for _ in range(3):
            assert [a.tobytes() for a in p.step(hip)] == first
        assert [a.tobytes() for a in p.forward(hip)] == first[:3]


def test_capture_replays_with_new_data(hip):
    lib = L.load()
    for rows, vocab in ((40, 700), (3, 20000)):
        problems = [Policy("bf16", rows, vocab, seed=10 + i) for i in range(3)]

        def inputs(x):
            return [a.arr for a in x.arguments()[1:7]]
        md = problems[0].arguments()[0]
        bufs = [L.DeviceBuffer.from_numpy(a) for a in inputs(problems[0])]
        outs = [L.DeviceBuffer(n) for n in (4, 4 * rows, 4 * rows, 2 * rows * vocab, 2 * rows * vocab)]
        coef = problems[0].arguments()[7:]

        def calls():
            L.call("policy_loss_step_bf16_i64", md, *bufs, *coef, None, *outs[:4])
            L.call("policy_loss_backward_bf16_i64", md, *bufs, *coef, outs[1], outs[2], None, outs[4])
        calls()
        L.synchronize()
        graph = C.c_void_p()
        assert lib.hip_graph_begin_capture() == 0
        calls()
        assert lib.hip_graph_end_capture(C.byref(graph)) == 0
        try:
            for x in problems + problems[:1]:
                want = x.step(hip)
                want = [*want, x.backward(hip, want[1], want[2])]
                for b, a in zip(bufs, inputs(x)):
                    assert lib.hip_memcpy_h2d(b.ptr, np.ascontiguousarray(a).ctypes.data, a.nbytes) == 0
                assert lib.hip_graph_launch(graph) == 0
                L.synchronize()
                for o, w in zip(outs, want):
                    assert o.to_numpy(w.dtype).tobytes() == w.tobytes()
        finally:
            lib.hip_graph_destroy(graph)


def test_gradient_is_the_differences(hip):
    """Central differences of size 2^-7 of the f32 loss; rows lie 1e-3 off the clip borders at least, and a step moves lp by less
    than 2^-7 ... so rows within 0.02 of a border are given an advantage of zero."""
    p = Policy("f32", 5, 6, seed=12, share=1.0)
    p.weight[:] = 1.0
    lp = p.exact()[0]["logp"]
    near = np.minimum(np.abs(lp - p.old - np.log(1 - p.low)), np.abs(lp - p.old - np.log(1 + p.high))) < 0.02
    p.advantage[near] = 0.0
    grad = p.step(hip)[3]
    for r in range(p.rows):
        for v in range(p.vocab):
            kept, sides = p.x[r, v], []
            for d in (2.0 ** -7, -2.0 ** -7):
                p.x[r, v] = kept + d
                sides.append(float(p.forward(hip)[0][0]))
            p.x[r, v] = kept
            assert abs((sides[0] - sides[1]) * 2.0 ** 6 - grad[r, v]) < 2e-3


@pytest.mark.parametrize("suffix", ["f32_i64", "bf16_i32", "f16_i64"])
def test_no_rows_and_no_addresses(hip, suffix):
    """Tensors of no rows may have no address; the loss is zero, a separate backward call has nothing to write."""
    md, none = u64(0, 5, 5, 1, 0), [Null()] * 6
    for name, rest in (("policy_loss_", []), ("policy_loss_step_", [Null()])):
        loss = hip.call(name + suffix, md, *none, 0.2, 0.2, 0.1, *rest, Out(1, "f32"), Null(), Null(), *([Null()] if rest else []))[0]
        assert loss[0] == 0
    hip.call("policy_loss_backward_" + suffix, md, *none, 0.2, 0.2, 0.1, Null(), Null(), Null(), Null())


TOP = {"f32": float(np.finfo(np.float32).max), "bf16": 3.3895313892515355e38, "f16": 65504.0}


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("rows,vocab", [(30, 7), (30, 200), (3, 9000), (260, 33001), (258, 70000)])
@pytest.mark.parametrize("what", ["lowest", "highest", "both", "one"])
def test_logits_at_the_limits(hip, dt, rows, vocab, what):
    """Rows of nothing but the type's lowest value or its highest, with the lowest in between, or with a single highest one.  What is
    left of x - max is 0 or beyond any exponent: the bounds are those of the same rows with 0 and -200 in their place (whose
    exponentials are zero in f32); lse is the row's largest logit more, to a rounding of its own."""
    p, q = Policy(dt, rows, vocab, seed=14, share=1.0, spread=0.0), Policy(dt, rows, vocab, seed=14, share=1.0, spread=0.0)
    r, top = np.random.default_rng(14), TOP[dt]
    low = np.zeros((rows, vocab), bool)
    if what == "both":
        low = r.random((rows, vocab)) < 0.5
    if what == "one":
        low[:] = True
    low[np.arange(rows), p.target] = False
    q.x = np.where(low, -200.0, 0.0)
    p.x = np.where(low, -top, -top if what == "lowest" else top)
    lp = -q.log_sum(q.x)
    p.old = q.old = (lp - 0.1).astype(np.float32)
    p.ref = q.ref = (lp + 0.1).astype(np.float32)
    want, bound = q.exact()
    bound["lse"] = bound["lse"] + np.abs(p.x).max() * 2.0 ** -23
    want["lse"] = want["lse"] + p.x.max(1)
    loss, logp, lse = p.forward(hip)
    for name, got in (("loss", loss), ("logp", logp), ("lse", lse)):
        p.close(got, want[name], bound[name], "forward " + name)
    p.close(p.backward(hip, logp, lse), want["grad"], bound["grad"], "backward")
    for name, got in zip(("loss", "logp", "lse", "grad"), p.step(hip)):
        p.close(got, want[name], bound[name], "step " + name)


def test_more_rows_than_a_launch_has_threads_for(hip):
    """2^24 rows and some: one block of 256 threads each would be more than 2^32 threads.  Two logits a row; every row is checked by a
    plain sum in 64 bits (a f32 logarithm, exponential and product each: 2^-21 of values below 16 is generous)."""
    rows = 2 ** 24 + 300
    r = np.random.default_rng(15)
    x = r.standard_normal((rows, 2), dtype=np.float32)
    target = r.integers(0, 2, rows).astype(np.int32)
    weight = np.full(rows, 1.0, np.float32)
    adv, zero = r.standard_normal(rows, dtype=np.float32), np.zeros(rows, np.float32)
    d = (x[np.arange(rows), 1 - target].astype(np.float64) - x[np.arange(rows), target])
    lp = -np.log1p(np.exp(d))
    args = [u64(rows, 2, 2, 1, 0), In(target), In(x), In(lp.astype(np.float32)), Null(), In(adv), In(weight), 0.2, 0.2, 0.0]
    loss, logp, lse, grad = hip.call("policy_loss_step_f32_i32", *args, Null(), Out(1, "f32"), Out(rows, "f32"), Out(rows, "f32"), Out(2 * rows, "f32"))
    assert np.abs(logp - lp).max() < 2.0 ** -21 * 16
    assert np.abs(lse - (x[np.arange(rows), target] - lp)).max() < 2.0 ** -21 * 16
    g = -adv * -np.expm1(lp)                                  # the ratio is one to within a rounding, inside the clip range
    assert np.abs(grad.reshape(rows, 2)[np.arange(rows), target] - g).max() < 2.0 ** -21 * 16
    assert abs(loss[0] + adv.astype(np.float64).sum()) < rows * 2.0 ** -21
    again = hip.call("policy_loss_backward_f32_i32", *args, In(logp), In(lse), Null(), Out(2 * rows, "f32"))[0]
    assert np.abs(again - grad).max() < 2.0 ** -21 * 16


@pytest.mark.parametrize("rows,vocab", [(300, 1001), (3, 9001)])
def test_rows_beyond_32_bits(hip, rows, vocab):
    """Rows so far apart that the last lies beyond 2^31 elements.  (Not the bits of rows that lie together: how a row is cut into
    16-byte pieces goes by its alignment, and the order of its sum by that.)"""
    lib = L.load()
    p = Policy("bf16", rows, vocab, seed=16)
    want, bound = p.exact()
    args = p.arguments()
    stride = 2 ** 31 // (rows - 1) + 9
    big = L.DeviceBuffer(((rows - 1) * stride + vocab) * 2)
    x = args[2].arr.reshape(rows, vocab)
    for t in range(rows):
        assert lib.hip_memcpy_h2d(big.ptr + t * stride * 2, np.ascontiguousarray(x[t]).ctypes.data, 2 * vocab) == 0
    dev = [L.DeviceBuffer.from_numpy(a.arr) for a in (args[1], *args[3:7])]
    outs = [L.DeviceBuffer(n) for n in (4, 4 * rows, 4 * rows, 2 * rows * vocab)]
    L.call("policy_loss_step_bf16_i64", u64(rows, vocab, stride, 1, 0), dev[0], big, *dev[1:], *args[7:], None, *outs)
    L.synchronize()
    for name, got in zip(("loss", "logp", "lse", "grad"), outs):
        p.close(got.to_numpy(np.uint16 if name == "grad" else np.float32).reshape(want[name].shape), want[name], bound[name], name)
