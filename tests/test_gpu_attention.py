"""Attention over packed sequences on the GPU against plain numpy in 64 bits; every bound is derived in language.py."""
import numpy as np
import pytest

import maidenx_amd.lib as L
from helpers import to_float, to_storage
from language import E32, TINY, UNIT, Attention, borders, bucket_of

pytestmark = pytest.mark.gpu
ALL = ["f32", "bf16", "f16"]


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("lengths,lead,tail", [([1], 0, 0), ([2], 0, 0), ([31], 0, 0), ([32, 33], 0, 0), ([64, 1, 65], 0, 0), ([129], 0, 0), ([300, 0, 0, 211, 1, 1, 77], 3, 9),
                                               ([0, 0, 5, 0], 0, 2), ([17] * 40, 1, 0)])
def test_lengths(hip, dt, lengths, lead, tail):
    Attention(dt, lengths, 4, 2, 64, lead=lead, tail=tail, seed=len(lengths)).check(hip)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("dim", [1, 5, 8, 16, 31, 32, 40, 64, 72, 80, 96, 100, 128])
def test_head_sizes(hip, dt, dim):
    Attention(dt, [90, 50], 2, 1, dim, seed=dim).check(hip)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,kv,buckets", [(2, 1, 0), (2, 2, 16), (90, 90, 0), (96, 8, 32)])
def test_long_walks(hip, dt, dim, heads, kv, buckets):
    """Many tiles to a block, with few blocks and with more than two for every CU (other numbers of waves and places)."""
    Attention(dt, [790, 11], heads, kv, dim, buckets=buckets, distance=100 if buckets else 0, seed=dim + heads).check(hip)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (6, 2), (8, 8), (8, 1), (16, 4), (5, 5)])
def test_grouped_heads(hip, heads, kv):
    Attention("bf16", [70, 150], heads, kv, 32, seed=heads).check(hip)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("layout", ["fused", "heads first", "elements first", "odd", "shared"])
@pytest.mark.parametrize("dim", [64, 24])
def test_layouts(hip, dt, layout, dim):
    Attention(dt, [100, 41], 4, 2, dim, layout=layout, seed=5).check(hip)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0, 1e-6])
def test_scales(hip, dt, scale):
    Attention(dt, [70, 20], 2, 2, 32, scale=scale, seed=6).check(hip)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("buckets,distance,dim", [(32, 128, 64), (32, 256, 128), (2, 2, 32), (7, 20, 32), (16, 64, 96), (64, 1000, 64), (256, 4096, 32), (3, 4096, 32)])
def test_bias(hip, dt, buckets, distance, dim):
    Attention(dt, [333, 1, 160], 4, 2, dim, buckets=buckets, distance=distance, seed=buckets).check(hip)


@pytest.mark.parametrize("lengths", [[1], [40], [200, 0, 64], [17] * 30, [700]])
def test_bias_lengths(hip, lengths):
    Attention("bf16", lengths, 3, 1, 64, buckets=32, distance=128, lead=2, tail=5, seed=7).check(hip)


@pytest.mark.parametrize("buckets,distance", [(32, 256), (32, 128), (20, 640), (256, 4096), (5, 100)])
def test_buckets_begin_where_the_definition_says(hip, buckets, distance):
    """q . k is zero, one bucket's bias is 40 above the others: a row's output is the mean of the values in that bucket, and a
    distance too many or too few moves it by a half.  (Rounding: at most 2^-24 (1500 + 12) of values up to 1500.)"""
    first = borders(buckets, distance)
    n = min(first[-1] + 40, 1500)
    for b in sorted({0, buckets // 2 - 1, buckets // 2, buckets // 2 + 1, max(x for x in range(buckets) if first[x] < n - 1), buckets - 2, buckets - 1}):
        if first[b] >= n:
            continue
        a = Attention("f32", [n], 1, 1, 1, buckets=buckets, distance=distance, seed=b)
        a.q[:] = 0
        a.table[:] = 0
        a.table[b] = 40
        a.v[:, 0, 0] = np.arange(n)
        upto = first[b + 1] if b + 1 < buckets else n + 1
        out, _ = a.forward(hip)
        rows = np.arange(n)
        want = rows - (first[b] + np.minimum(upto - 1, rows)) / 2
        seen = rows >= first[b]
        assert np.abs(out[seen, 0, 0] - want[seen]).max() < 0.25


@pytest.mark.parametrize("dt", ALL)
def test_large_scores(hip, dt):
    """Scores of some hundreds: one key takes all, sums that a softmax without the running maximum would overflow."""
    Attention(dt, [150], 2, 1, 64, spread=8.0, scale=0.5, seed=11).check(hip, gradients=dt != "f16")


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("what", ["first", "far", "all"])
def test_rows_that_a_bias_leaves_empty(hip, dt, what):
    """A table with -inf: rows whose every pair is out have zeros, lse -inf and no gradient."""
    a = Attention(dt, [70, 1, 40], 2, 1, 32, buckets=8, distance=16, seed=12)
    a.table[{"first": slice(0, 1), "far": slice(3, 8), "all": slice(0, 8)}[what]] = -np.inf
    a.check(hip)


@pytest.mark.parametrize("dt", ALL)
def test_the_lowest_value_is_a_value(hip, dt):
    """A bias of the type's lowest value on every bucket but those from 4 on: rows near the start have nothing else and are
    the mean over their keys, since q . k is lost beside it."""
    a = Attention(dt, [40], 2, 2, 16, buckets=8, distance=16, seed=13)
    lowest = float(to_float(np.array([{"f32": np.float32(-3.4028234663852886e38).view(np.uint32), "bf16": 0xFF7F, "f16": 0xFBFF}[dt]],
                                     dtype=np.uint32 if dt == "f32" else np.uint16).view(np.float32 if dt == "f32" else np.uint16), dt)[0])
    a.table[:4] = lowest
    out, lse = a.forward(hip)
    got = to_float(out, dt).astype(np.float64)
    if dt != "f16":                                          # (-65504 does not drown q . k in f32)
        for i in range(4):
            want = a.v[: i + 1].mean(0)
            assert np.abs(got[i] - want).max() <= 2.0 ** -7 * np.abs(a.v[: i + 1]).max()
    assert np.isfinite(got).all() and np.isfinite(lse).all()
    for g in a.backward(hip, out, lse):
        assert np.isfinite(to_float(g, dt)).all()


def test_each_gradient_can_be_left_out(hip):
    a = Attention("bf16", [100, 60], 4, 2, 64, buckets=16, distance=64, seed=14)
    out, lse = a.forward(hip)
    every = a.backward(hip, out, lse)
    for mask in range(1, 15):
        want = tuple(bool(mask >> n & 1) for n in range(4))
        for w, g, e in zip(want, a.backward(hip, out, lse, want), every):
            assert (g is None) == (not w)
            if w:
                assert g.tobytes() == e.tobytes()
    plain = Attention("f32", [100, 60], 4, 2, 64, seed=14)
    out, lse = plain.forward(hip)
    every = plain.backward(hip, out, lse)
    for mask in range(1, 8):
        want = tuple(bool(mask >> n & 1) for n in range(3)) + (False,)
        for w, g, e in zip(want, plain.backward(hip, out, lse, want), every):
            assert not w or g.tobytes() == e.tobytes()


def test_the_same_bits_on_every_call(hip):
    a = Attention("bf16", [500, 300, 9], 8, 2, 64, buckets=32, distance=128, seed=15)
    out, lse = a.forward(hip)
    grads = a.backward(hip, out, lse)
    for _ in range(3):
        o, ls = a.forward(hip)
        assert o.tobytes() == out.tobytes() and ls.tobytes() == lse.tobytes()
        assert all(x.tobytes() == y.tobytes() for x, y in zip(a.backward(hip, o, ls), grads))


@pytest.mark.parametrize("dt", ALL)
def test_a_sequence_does_not_depend_on_its_neighbours(hip, dt):
    """NaN and infinities all over one sequence and in the rows that belong to none reach no other sequence."""
    a = Attention(dt, [45, 40, 70], 2, 1, 32, lead=4, tail=7, seed=16)
    want, bound = a.exact()
    dirty = np.r_[0:4, 49:89, a.tokens - 7:a.tokens]
    for t in (a.q, a.k, a.v, a.go):
        t[dirty[::2]] = np.nan
        t[dirty[1::2]] = np.inf
    out, lse = a.forward(hip)
    gq, gk, gv, _ = a.backward(hip, out, lse)
    clean = np.r_[4:49, 89:159]
    for name, got in (("o", out), ("gq", gq), ("gk", gk), ("gv", gv)):
        a.close(got[clean], want[name][clean], bound[name][clean], name)
    a.close(lse[:, clean], want["lse"][:, clean], bound["lse"][:, clean], "lse")


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_comes_later_does_not_reach_back(hip, dt, bad):
    """Non-finite keys and values at the end of a sequence (a padded batch) leave the rows before them as they were."""
    a = Attention(dt, [200, 30], 2, 1, 64, seed=17)
    want, bound = a.exact()
    a.v[150:200] = bad
    a.k[170:200] = bad
    out, lse = a.forward(hip)
    rows = np.r_[0:150, 200:230]
    a.close(out[rows], want["o"][rows], bound["o"][rows], "output")
    a.close(lse[:, rows], want["lse"][:, rows], bound["lse"][:, rows], "lse")


def test_infinite_values_in_view(hip):
    """An infinite value that a row sees is in its output, as the sum says."""
    a = Attention("f32", [100], 1, 1, 32, seed=18)
    a.v[40, 0, 3] = np.inf
    a.v[60, 0, 4] = -np.inf
    a.v[70, 0, 5] = np.nan
    out, _ = a.forward(hip)
    assert np.isfinite(out[:, 0, :3]).all() and np.isfinite(out[:, 0, 6:]).all()
    assert np.isfinite(out[:40, 0, 3]).all() and (out[40:, 0, 3] == np.inf).all()
    assert np.isfinite(out[:60, 0, 4]).all() and (out[60:, 0, 4] == -np.inf).all()
    assert np.isfinite(out[:70, 0, 5]).all() and np.isnan(out[70:, 0, 5]).all()


@pytest.mark.parametrize("offsets", [[0, 50, 40, 90], [-3, 90], [0, 91], [90, 0], [2 ** 31 - 1, 2 ** 31 - 1], [-2 ** 31, 5, 90, 2 ** 31 - 1]] + [[0] + [95] * 70])
def test_bad_offsets_are_reported(hip, offsets):
    """Nothing outside the tensors is touched: the kernels keep every bound that they make of offsets within the tokens."""
    a = Attention("f32", [90], 2, 1, 32, buckets=8, distance=16, seed=19)
    out, lse = a.forward(hip)
    a.offsets = np.array(offsets, dtype=np.int32)
    with pytest.raises(L.HipError, match="offsets of attention"):
        a.forward(hip)
    with pytest.raises(L.HipError, match="offsets of attention"):
        a.backward(hip, out, lse)


def test_nothing_to_do(hip):
    a = Attention("f32", [4], 2, 1, 8, buckets=4, distance=8, seed=20)
    a.offsets = np.array([0], dtype=np.int32)                # no sequence
    out, lse = a.forward(hip)
    assert (out.view(np.uint8) == 0xCD).all() and (lse.view(np.uint8) == 0xCD).all()
    gq, gk, gv, gt = a.backward(hip, np.zeros_like(out), np.zeros_like(lse))
    assert all((g.view(np.uint8) == 0xCD).all() for g in (gq, gk, gv)) and (gt == 0).all()


def test_many_sequences(hip):
    """More sequences than a wave has lanes (the search by halves), empty ones among them."""
    r = np.random.default_rng(21)
    Attention("bf16", [int(n) for n in r.integers(0, 9, 150)], 2, 1, 32, lead=1, tail=3, seed=21).check(hip)


def test_capture_replays_with_new_data(hip):
    """Forward and backward in a captured graph, replayed over new inputs and other sequence lengths between eager calls."""
    lib = L.load()
    problems = [Attention("bf16", lengths, 4, 2, 64, buckets=16, distance=64, seed=22 + i) for i, lengths in enumerate(([150, 50], [20, 100, 80], [200, 0]))]
    for p in problems:                                        # one number of sequences for all
        p.offsets = np.concatenate([p.offsets, [200] * (4 - len(p.offsets))]).astype(np.int32)
    p = problems[0]
    md, off, q, k, v, table, scale = p.arguments()
    names = ["off", "q", "k", "v", "table", "go"]

    def inputs(x):
        a = x.arguments()
        return dict(zip(names, [a[1].arr, a[2].arr, a[3].arr, a[4].arr, a[5].arr, to_storage(x.go, x.dt).ravel()]))
    bufs = {n: L.DeviceBuffer.from_numpy(a) for n, a in inputs(p).items()}
    outs = {n: L.DeviceBuffer(2 * c) for n, c in (("out", 200 * 4 * 64), ("gq", 200 * 4 * 64), ("gk", 200 * 2 * 64), ("gv", 200 * 2 * 64), ("gt", 64))}
    lse = L.DeviceBuffer(4 * 4 * 200)

    def calls():
        common = [md, bufs["off"], bufs["q"], bufs["k"], bufs["v"], bufs["table"], scale]
        L.call("attention_bf16", *common, outs["out"], lse)
        L.call("attention_backward_bf16", *common, outs["out"], lse, bufs["go"], outs["gq"], outs["gk"], outs["gv"], outs["gt"])
    calls()
    L.synchronize()
    import ctypes as C
    graph = C.c_void_p()
    assert lib.hip_graph_begin_capture() == 0
    calls()
    assert lib.hip_graph_end_capture(C.byref(graph)) == 0
    try:
        for x in problems + problems[:1]:
            o, ls = x.forward(hip)                            # eager, over the library's own scratch
            want = [o, *x.backward(hip, o, ls)]
            for n, a in inputs(x).items():
                assert lib.hip_memcpy_h2d(bufs[n].ptr, np.ascontiguousarray(a).ctypes.data, a.nbytes) == 0
            assert lib.hip_graph_launch(graph) == 0
            L.synchronize()
            for n, w in zip(("out", "gq", "gk", "gv", "gt"), want):
                assert outs[n].to_numpy(np.uint16).tobytes() == w.tobytes(), n
    finally:
        lib.hip_graph_destroy(graph)


def test_on_a_stream_of_the_callers(hip):
    import ctypes as C
    lib = L.load()
    a = Attention("f32", [80, 30], 2, 1, 32, seed=30)
    out, lse = a.forward(hip)
    s = C.c_void_p()
    assert lib.hip_stream_create(C.byref(s)) == 0
    try:
        assert lib.hip_set_stream(s) == 0
        o, ls = a.forward(hip)
        assert o.tobytes() == out.tobytes() and ls.tobytes() == lse.tobytes()
    finally:
        lib.hip_set_stream(None)
        lib.hip_stream_destroy(s)


def test_gradients_are_the_differences(hip):
    """sum(output * go) in f32, by central differences of size 2^-6: the truncation is below (2^-6)^2 / 6 times the third
    derivative (for inputs of order one, 1e-3 is generous), the roundings 2^-24 |sum| / 2^-6 are below it."""
    a = Attention("f32", [12, 5], 2, 1, 8, buckets=4, distance=6, seed=31)
    out, lse = a.forward(hip)
    grads = a.backward(hip, out, lse)

    def value():
        return float((a.forward(hip)[0].astype(np.float64) * a.go).sum())
    for tensor, grad in ((a.q, grads[0]), (a.k, grads[1]), (a.v, grads[2]), (a.table, grads[3])):
        flat = tensor.reshape(-1)
        for i in range(0, flat.size, max(1, flat.size // 9)):
            kept = flat[i]
            flat[i] = kept + 2.0 ** -6
            up = value()
            flat[i] = kept - 2.0 ** -6
            down = value()
            flat[i] = kept
            assert abs((up - down) * 2.0 ** 5 - grad.reshape(-1)[i]) < 3e-3


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_the_longest_table(hip, dt, dim):
    """256 buckets up to a distance of 4096: the most shared memory that a call asks for, with few blocks and with many."""
    Attention(dt, [300, 45], 2, 1, dim, buckets=256, distance=4096, seed=dim).check(hip)
    Attention(dt, [150] * 4, 70, 35, dim, buckets=256, distance=4096, seed=dim + 1).check(hip)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("buckets", [0, 16])
def test_walks_of_every_number_of_groups(hip, dt, dim, buckets):
    """Blocks for about a quarter of the CUs, for all of them, and for more than two each: the walks are shared differently."""
    for heads in (4, 40, 90):
        Attention(dt, [650, 3, 140], heads, heads // 2, dim, buckets=buckets, distance=100 if buckets else 0, seed=dim + heads).check(hip)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [16, 32])
@pytest.mark.parametrize("layout", ["packed", "odd"])
@pytest.mark.parametrize("heads,kv,buckets", [(4, 2, 0), (4, 2, 16), (96, 48, 16)])
def test_small_heads_wait_for_their_rows(hip, dt, dim, layout, heads, kv, buckets):
    """Tiles of 64-byte rows are fewer loads than a block has waves.  Walks of many tiles, with few blocks and with many: the keys' and
    values' gradients against 64 bits, and the same bits from call to call."""
    a = Attention(dt, [900, 130], heads, kv, dim, buckets=buckets, distance=100 if buckets else 0, layout=layout, seed=dim + heads)
    a.check(hip)
    out, lse = a.forward(hip)
    first = [g.tobytes() for g in a.backward(hip, out, lse) if g is not None]
    for _ in range(4):
        assert [g.tobytes() for g in a.backward(hip, out, lse) if g is not None] == first


@pytest.mark.parametrize("dt,dim", [("f32", 80), ("bf16", 24), ("f16", 96), ("bf16", 64)])
def test_bad_offsets_of_many_sequences_are_reported(hip, dt, dim):
    """Among 64 sequences and more a row's sequence is found by halves: where offsets do not ascend, an early row may see further than
    a late one.  Every access stays within the tokens (the walk's own test goes through them all), and the call is reported."""
    a = Attention(dt, [1500], 2, 1, dim, buckets=8, distance=16, seed=32)
    out, lse = a.forward(hip)
    a.offsets = np.array([0] + [1500] * 31 + [20] + [30] * 32, dtype=np.int32)
    with pytest.raises(L.HipError, match="offsets of attention"):
        a.forward(hip)
    with pytest.raises(L.HipError, match="offsets of attention"):
        a.backward(hip, out, lse)


FIRST_CALL = """
import sys
sys.path[:0] = {paths!r}
import numpy as np
import maidenx_amd.lib as L
from language import meta_attention
md = meta_attention(0, 2, 1, 8, {sequences}, 4, 8, [16, 8, 1], [8, 8, 1], [8, 8, 1])
offsets = L.DeviceBuffer.from_numpy(np.zeros({sequences} + 1, np.int32))
table = L.DeviceBuffer.from_numpy(np.ones(8, np.{np}))
grad = L.DeviceBuffer.from_numpy(np.ones(8, np.{np}))
L.call("attention_{dt}", md, offsets, None, None, None, table, 1.0, None, None)
L.synchronize()
L.call("attention_backward_{dt}", md, offsets, None, None, None, table, 1.0, None, None, None, None, None, None, grad)
L.synchronize()
assert (grad.to_numpy(np.{np}) == 0).all()
print("zeros")
"""


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("sequences", [0, 3])
def test_no_tokens(dt, sequences):
    """The first calls of a process, when the library has no workspace yet: no tokens, tensors without an address, and a table whose
    gradient is zero."""
    import subprocess
    import sys
    from helpers import ROOT
    code = FIRST_CALL.format(paths=[ROOT, ROOT + "/tests"], sequences=sequences, dt=dt, np="float32" if dt == "f32" else "uint16")
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert p.returncode == 0 and "zeros" in p.stdout, p.stderr[-2000:]


def uniform_rows(a, rows_of, u, e):
    """Gradients of rows whose scores are all equal (P = 1 / n), for the rows of a sequence that rows_of(n) names, with bounds: P comes
    from an exponential of zero and a sum of ones (a few e), dP and D are sums of dim and n terms, D with o as it was rounded (u), dS is
    rounded to the tensors' type (u), and so is each result."""
    t, h, g, d = a.tokens, a.heads, a.kv, a.dim
    group, s = h // g, abs(a.scale)
    out, lse = np.full((t, h, d), np.nan), np.full((h, t), np.nan)
    r = {"gq": np.zeros((t, h, d)), "gk": np.zeros((t, g, d)), "gv": np.zeros((t, g, d)), "gt": np.zeros((a.buckets, h))}
    b = {n: np.zeros_like(x) for n, x in r.items()}
    ob = np.zeros((t, h, d))
    for first, last in zip(a.offsets[:-1], a.offsets[1:]):
        for n in rows_of(last - first):                      # keys that the row sees
            i, r_ = first + n - 1, slice(first, first + n)
            bucket = bucket_of(np.arange(n)[::-1], a.buckets, a.distance)
            for x in range(h):
                k, v, q, go = a.k[r_, x // group], a.v[r_, x // group], a.q[i, x], a.go[i, x]
                o, dp = v.mean(0), v @ go
                ds = (dp - dp.mean()) / n
                out[i, x], lse[x, i] = o, np.log(n)
                ob[i, x] = (2 * u + e * (n + 16)) * np.abs(v).mean(0)
                off = ((np.abs(v) @ np.abs(go)) * (u + e * (n + d + 16)) * 2 + (2 * u + e * (n + d + 16)) * (np.abs(v) @ np.abs(go)).mean()) / n
                r["gq"][i, x] = a.scale * (ds @ k)
                b["gq"][i, x] = s * (off @ np.abs(k)) + u * np.abs(r["gq"][i, x])
                r["gk"][r_, x // group] += a.scale * ds[:, None] * q
                b["gk"][r_, x // group] += s * off[:, None] * np.abs(q)
                r["gv"][r_, x // group] += go / n
                b["gv"][r_, x // group] += (u + e * (n + 16)) * np.abs(go) / n
                np.add.at(r["gt"][:, x], bucket, ds)
                np.add.at(b["gt"][:, x], bucket, off)
    return out, ob, lse, r, b


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("heads,dim", [(4, 32), (4, 128), (40, 64), (90, 128), (90, 96)])
@pytest.mark.parametrize("which,value", [("near", -2.0 ** 31), ("near", "lowest"), ("all", -2.0 ** 31), ("all", "lowest"), ("all", 2.0 ** 40)])
def test_rows_of_one_large_bias(hip, dt, value, heads, dim, which):
    """A bias so large that q . k is lost beside it, on the first four distances or on all of them: rows with nothing else in view spread
    evenly, forward and backward; the others see the rest as if those pairs were out."""
    value = {"f32": -float(np.finfo(np.float32).max), "bf16": -3.3895313892515355e38}[dt] if value == "lowest" else value
    u, e = UNIT[dt], E32
    a = Attention(dt, [330, 3, 90], heads, heads // 2, dim, buckets=8, distance=16, seed=33)
    near = slice(0, 4) if which == "near" else slice(0, 8)
    a.table[near] = -np.inf
    want, bound = a.exact()                                  # of the rows that see more (none where all are masked)
    a.table[near] = value
    rows_of = (lambda n: range(1, min(4, n) + 1)) if which == "near" else (lambda n: range(1, n + 1))
    o, ob, lse_n, r, b = uniform_rows(a, rows_of, u, e)
    even = ~np.isnan(o[:, 0, 0])
    want["o"][even], bound["o"][even] = o[even], ob[even]
    want["lse"][:, even], bound["lse"][:, even] = value + lse_n[:, even], abs(value) * 2.0 ** -23
    for n in r:
        want[n] = want[n] + r[n]
        bound[n] = bound[n] + b[n] + 2 * u * np.abs(r[n])
    out, lse = a.forward(hip)
    a.close(out, want["o"], bound["o"], "output")
    a.close(lse, want["lse"], bound["lse"], "lse")
    for name, got in zip(("gq", "gk", "gv", "gt"), a.backward(hip, out, lse)):
        a.close(got, want[name], bound[name], name)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("size", [300.0, 2.0e4])
@pytest.mark.parametrize("heads,dim", [(4, 64), (40, 128), (90, 32)])
def test_large_biases(hip, dt, size, heads, dim):
    """Biases of some hundreds to the reach of f16, of either sign, beside each other."""
    a = Attention(dt, [400, 90], heads, heads // 2, dim, buckets=16, distance=64, seed=34)
    a.table[:] = to_float(to_storage(size * a.table, dt), dt)
    a.check(hip)


@pytest.mark.parametrize("dim,heads,lengths,buckets", [(32, 2, [90, 33], 0), (128, 2, [150, 20], 0), (64, 40, [330], 16), (128, 90, [200, 150], 16), (80, 12, [700], 0), (96, 4, [64, 64], 8)])
@pytest.mark.parametrize("power", [-14, -8, 6, 11])
def test_f16_gradients_of_any_size(hip, dim, heads, lengths, buckets, power):
    """Output gradients times 2^power: all gradients are as many times larger, and so are their bounds (what is held in f16 on the way is
    scaled to the type's middle: 2^-35 of the largest dS is lost, where the bound counts 2^-25); what leaves f16 is infinite, below its
    normal numbers a result is off by half of the last subnormal."""
    a = Attention("f16", lengths, heads, heads // 2, dim, buckets=buckets, distance=40 if buckets else 0, seed=35)
    go = to_float(to_storage(a.go * 2.0 ** power, "f16"), "f16").astype(np.float64)
    a.go = go * 2.0 ** -power
    want, bound = a.exact()
    a.go = go
    out, lse = a.forward(hip)
    for name, got in zip(("gq", "gk", "gv", "gt"), a.backward(hip, out, lse)):
        if got is None:
            continue
        w, b = want[name] * 2.0 ** power, bound[name] * 2.0 ** power + 2.0 ** -25
        x = to_float(got, "f16").astype(np.float64)
        fits = np.abs(w) + b < 65504
        assert fits.mean() > 0.9
        a.close(np.where(fits, x, 0), np.where(fits, w, 0), b, name)
        assert not np.isnan(x).any()
        beyond = np.abs(w) - b > 65520
        assert (x[beyond] == np.sign(w[beyond]) * np.inf).all()


def test_f16_gradients_beside_large_scores(hip):
    Attention("f16", [150], 2, 1, 64, spread=8.0, scale=0.5, seed=11).check(hip)


@pytest.mark.parametrize("dim,heads", [(64, 2), (128, 40), (96, 90)])
def test_f16_gradients_whose_inner_ones_leave_the_type(hip, dim, heads):
    """dS above 65504 on the way to gradients that f16 holds."""
    a = Attention("f16", [30, 41], heads, heads // 2, dim, scale=2.0 ** -8, seed=36)
    a.v = to_float(to_storage(a.v * 64.0, "f16"), "f16").astype(np.float64)
    a.go = to_float(to_storage(a.go * 1024.0, "f16"), "f16").astype(np.float64)
    dp = a.v[:30, 0] @ a.go[:30, 0].T                        # [keys, queries]; P is about 1 / (query + 1)
    assert max(abs(dp[:i + 1, i] - dp[:i + 1, i].mean()).max() / (i + 1) for i in range(1, 30)) > 70000
    a.check(hip)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("buckets", [0, 16])
@pytest.mark.parametrize("large", [False, True])
def test_one_gradient_alone_finds_nothing_of_an_earlier_call(hip, dt, buckets, large):
    """Each gradient by itself, after a call of another problem of the same sizes has left its numbers in the workspace."""
    a, other = (Attention(dt, [150, 60], 4, 2, 64, buckets=buckets, distance=64 if buckets else 0, seed=s, spread=f) for s, f in ((37, 1.0), (38, 3.0)))
    if large and buckets:
        a.table[:3] = to_float(to_storage(np.full((3, 4), -60000.0), dt), dt)
    out, lse = a.forward(hip)
    every = a.backward(hip, out, lse)
    for n in range(4 if buckets else 3):
        other.backward(hip, *other.forward(hip))
        got = a.backward(hip, out, lse, tuple(m == n for m in range(4)))
        assert got[n].tobytes() == every[n].tobytes(), n


class Mixed(Attention):
    """Query, key and value each packed or on no 16-byte boundary."""

    def stored(self):
        kinds, out = self.layout, []
        for n, kind in enumerate(kinds):
            self.layout = kind
            out.append(super().stored()[n])
        self.layout = kinds
        return out


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("dim", [24, 32, 64, 128])
@pytest.mark.parametrize("kinds", [("odd", "packed", "packed"), ("packed", "odd", "packed"), ("packed", "packed", "odd"), ("odd", "odd", "packed")])
def test_operands_that_lie_differently(hip, dt, dim, kinds):
    """One operand of a tile straight to shared memory, the other through registers."""
    Mixed(dt, [410, 60], 4, 2, dim, layout=kinds, buckets=8, distance=30, seed=39).check(hip)
    Mixed(dt, [300], 40, 20, dim, layout=kinds, seed=40).check(hip)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("stride", [2 ** 23 - 8, 2 ** 23 + 8])
def test_offsets_beyond_32_bits(hip, dt, stride):
    """Tokens 2^23 elements apart, on either side of the longest row that goes straight to shared memory: a sequence of 400 reaches
    over 2^31 elements and more."""
    lib, size = L.load(), 4 if dt == "f32" else 2
    a = Attention(dt, [380, 20], 2, 1, 32, buckets=8, distance=30, seed=41)
    want = [a.forward(hip)]
    want += [a.backward(hip, *want[0])]
    rows = to_storage(np.concatenate([a.q, a.k, a.v], axis=1), dt).reshape(400, -1)
    big = L.DeviceBuffer((399 * stride + rows.shape[1]) * size)
    for t in range(400):
        assert lib.hip_memcpy_h2d(big.ptr + t * stride * size, rows[t].ctypes.data, rows[t].nbytes) == 0
    md = a.arguments()[0].copy()
    for n, offset in enumerate((0, 64, 96)):
        md[7 + 3 * n], md[16 + n] = stride, offset
    dev = [L.DeviceBuffer.from_numpy(x) for x in (a.offsets, to_storage(a.table, dt).ravel(), to_storage(a.go, dt).ravel())]
    out, lse, gq, gk, gv, gt = (L.DeviceBuffer(x.nbytes) for x in (*want[0], *want[1]))
    common = [md, dev[0], big, big, big, dev[1], float(a.scale)]
    L.call("attention_" + dt, *common, out, lse)
    L.call("attention_backward_" + dt, *common, out, lse, dev[2], gq, gk, gv, gt)
    L.synchronize()
    for got, w in zip((out, lse, gq, gk, gv, gt), (*want[0], *want[1])):
        assert got.to_numpy(w.dtype).tobytes() == w.tobytes()


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("power", [-14, 0, 11])
def test_gradients_of_any_size_beside_infinite_ones(hip, dt, power):
    """Sequences that share the tiles of a wave, one full of infinities and NaN: the other's gradients keep their bounds, for output gradients of
    any size (times a power of two, as all of them then are)."""
    a = Attention(dt, [45, 40, 70], 2, 1, 64, lead=4, tail=7, seed=42)
    go = to_float(to_storage(a.go * 2.0 ** power, dt), dt).astype(np.float64)
    a.go = go * 2.0 ** -power
    want, bound = a.exact()
    a.go = go
    clean, dirty = np.r_[4:49, 89:159], np.r_[0:4, 49:89, a.tokens - 7:a.tokens]
    for t in (a.q, a.k, a.v, a.go):
        t[dirty[::2]] = np.nan
        t[dirty[1::2]] = np.inf
    out, lse = a.forward(hip)
    for name, g in zip(("gq", "gk", "gv"), a.backward(hip, out, lse)):
        a.close(g[clean], want[name][clean] * 2.0 ** power, bound[name][clean] * 2.0 ** power + TINY[dt], name)


@pytest.mark.parametrize("dt", ALL)
def test_rows_that_are_summed_once_more_leave_others_as_they_are(hip, dt):
    """Large scores in one sequence: the gradients of another in the same waves keep their bits."""
    a = Attention(dt, [45, 40, 70], 2, 1, 64, buckets=8, distance=16, seed=42)
    clean, large = np.r_[0:45, 85:155], np.r_[45:85]
    a.go[large] = 0
    want = a.backward(hip, *a.forward(hip))
    a.q[large], a.k[large] = a.q[large] * 16, a.k[large] * 16
    out, lse = a.forward(hip)
    assert np.abs(lse[:, large]).max() > 256
    for w, g in zip(want[:3], a.backward(hip, out, lse)):
        assert g[clean].tobytes() == w[clean].tobytes()
