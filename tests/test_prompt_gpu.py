"""lpp_prompt_attention against 64 bits: ragged and empty sequences, every number of query heads to a KV head, both types, strides, rows that
belong to no sequence, and what K and V hold outside a row's own positions."""
import ctypes as C

import numpy as np
import pytest

import kv4_oracle as ko
from lighterpp_amd import capi
from lighterpp_amd.capi import DeviceBuffer as DB
from test_kv4_gpu import Hip

pytestmark = pytest.mark.gpu
F, H = np.float32, np.float16


@pytest.fixture(scope="module")
def lib():
    lib = capi.load()
    assert capi.device_count() >= 1, "no HIP device visible"
    capi.check(lib.lpp_init(0))
    return lib


def run(lib, q, k, v, offsets, n_tokens=None, pad=0, seqs=None):
    """q [rows, heads, hs], k and v [rows, kv_heads, hs] binary16.  `pad`: groups of 8 elements behind every row, which must not change."""
    rows, heads, hs = q.shape
    kv = k.shape[1]
    typ = q.dtype.type
    extra = 8 * pad

    def padded(x, fill):
        return np.concatenate([x.reshape(rows, -1), np.full((rows, extra), fill, x.dtype)], 1)

    dq, dk, dv = DB.from_numpy(padded(q, np.nan)), DB.from_numpy(padded(k, np.nan)), DB.from_numpy(padded(v, np.inf))
    out = np.full((rows, heads * hs + extra), 7.25, typ)
    dout = DB.from_numpy(out)
    doff = None if offsets is None else DB.from_numpy(np.array(offsets, np.int32))
    seqs = (1 if offsets is None else len(offsets) - 1) if seqs is None else seqs
    capi.check(lib.lpp_prompt_attention(dout.ptr, dq.ptr, dk.ptr, dv.ptr, capi.F32 if typ is F else capi.F16, doff.ptr if doff else None, seqs,
                                        rows if n_tokens is None else n_tokens, heads, kv, hs, heads * hs + extra, kv * hs + extra, heads * hs + extra))
    got = dout.to_numpy(typ, out.size).reshape(out.shape)
    assert np.all(got[:, heads * hs:] == typ(7.25)), "the space between the rows was written"
    return got[:, :heads * hs].reshape(rows, heads, hs)


def inputs(seed, rows, heads, kv, hs, typ, spread=1.0):
    rng = np.random.default_rng(seed)
    return ((rng.standard_normal((rows, heads, hs)) * spread).astype(typ), rng.standard_normal((rows, kv, hs)).astype(H),
            rng.standard_normal((rows, kv, hs)).astype(H))


def against(got, q, k, v, spans):
    """Every sequence's rows against the oracle, the others untouched."""
    mine = np.zeros(q.shape[0], bool)
    worst = 0.0
    for a, b in spans:
        mine[a:b] = True
        if a == b:
            continue
        want, _, tol = ko.attend_tolerance(q[a:b], k[a:b].transpose(1, 0, 2), v[a:b].transpose(1, 0, 2), [j + 1 for j in range(b - a)],
                                           binary16=q.dtype.type is H)
        off = np.abs(got[a:b].astype(np.float64) - want)
        worst = max(worst, float((off / tol).max()))
        assert np.all(off <= tol), (a, b, float((off / tol).max()))
    assert np.all(got[~mine] == q.dtype.type(7.25))
    return worst


LENGTHS = [[1], [2, 0, 1], [31, 32, 33], [63, 65, 1, 0, 128], [257], [5, 0, 0, 300, 130]]


@pytest.mark.parametrize("heads,kv,hs", [(2, 2, 64), (8, 2, 64), (8, 1, 64), (16, 1, 128), (6, 2, 128), (3, 3, 128)])
@pytest.mark.parametrize("typ", [F, H])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_lengths(lib, lengths, typ, heads, kv, hs):
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    q, k, v = inputs(sum(lengths) * heads + hs, int(offsets[-1]), heads, kv, hs, typ)
    got = run(lib, q, k, v, offsets)
    against(got, q, k, v, list(zip(offsets[:-1], offsets[1:])))


@pytest.mark.parametrize("typ", [F, H])
@pytest.mark.parametrize("heads,kv,hs,length", [(4, 1, 64, 1100), (5, 1, 128, 700), (4, 4, 128, 1025)])
def test_one_long_prompt_without_offsets(lib, heads, kv, hs, length, typ):
    q, k, v = inputs(length, length, heads, kv, hs, typ)
    against(run(lib, q, k, v, None, pad=1), q, k, v, [(0, length)])


@pytest.mark.parametrize("typ", [F, H])
def test_many_short_sequences(lib, typ):
    """More sequences than a wavefront looks at in one go, empty ones among them, also first and last."""
    rng = np.random.default_rng(5)
    lengths = rng.integers(0, 9, 200)
    lengths[:3] = lengths[-2:] = 0
    lengths[64:130] = 0
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    q, k, v = inputs(6, int(offsets[-1]), 4, 2, 64, typ)
    against(run(lib, q, k, v, offsets), q, k, v, list(zip(offsets[:-1], offsets[1:])))


def test_thousands_of_sequences(lib):
    """More than a wavefront finds in two looks; a long one among them, empty stretches, rows of no sequence before, between none and behind."""
    rng = np.random.default_rng(15)
    lengths = rng.integers(0, 3, 5000)
    lengths[1000:1100] = 0
    lengths[2500], lengths[4999] = 300, 40
    offsets = 7 + np.concatenate([[0], np.cumsum(lengths)])
    rows = int(offsets[-1]) + 9
    q, k, v = inputs(16, rows, 2, 1, 64, F)
    got = run(lib, q, k, v, offsets)
    assert np.all(got[:7] == F(7.25)) and np.all(got[-9:] == F(7.25))
    check = [(a, b) for i, (a, b) in enumerate(zip(offsets[:-1], offsets[1:])) if b - a > 2 or i % 50 == 0]
    for a, b in check:
        if a < b:
            want, _, tol = ko.attend_tolerance(q[a:b], k[a:b].transpose(1, 0, 2), v[a:b].transpose(1, 0, 2), [j + 1 for j in range(b - a)])
            assert np.all(np.abs(got[a:b] - want) <= tol), (a, b)
    single = offsets[:-1][lengths >= 1]  # a sequence's first row is its V row
    assert np.all(np.abs(got[single] - v[single].astype(np.float64)) <= np.abs(v[single].astype(np.float64)) * 2.0 ** -20 + 1e-12)


@pytest.mark.parametrize("typ", [F, H])
def test_rows_outside_every_sequence_and_strides(lib, typ):
    """The first offset is not 0, the last is not the end; rows have space behind them."""
    q, k, v = inputs(7, 150, 6, 2, 64, typ)
    against(run(lib, q, k, v, [3, 40, 40, 141], pad=3), q, k, v, [(3, 40), (40, 141)])


@pytest.mark.parametrize("offsets,spans", [([-5, 20, 1000], [(0, 20), (20, 50)]), ([0, 2 ** 31 - 1], [(0, 50)]), ([50, 50, 50], []),
                                           ([-2 ** 31, -7, 50], [(0, 50)])])
def test_offsets_outside_are_cut(lib, offsets, spans):
    q, k, v = inputs(8, 50, 4, 2, 64, F)
    against(run(lib, q, k, v, offsets), q, k, v, spans)


@pytest.mark.parametrize("typ", [F, H])
@pytest.mark.parametrize("hs", [64, 128])
def test_large_scores(lib, typ, hs):
    """Scores of some hundreds, growing and falling along the sequence: the running maximum moves by a lot."""
    q, k, v = inputs(9, 300, 4, 1, hs, typ, spread=4.0)
    k = (k * np.linspace(0.2, 6.0, 300)[:, None, None]).astype(H)
    k[200:] = (k[200:] * 0.1).astype(H)
    against(run(lib, q, k, v, [0, 300]), q, k, v, [(0, 300)])


@pytest.mark.parametrize("typ", [F, H])
@pytest.mark.parametrize("heads,kv,hs", [(4, 4, 64), (8, 1, 64), (6, 2, 128)])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("where", ["k", "v"])
def test_nothing_comes_from_positions_a_row_does_not_attend_to(lib, where, bad, heads, kv, hs, typ):
    """A K or V row of infinities or NaN in the middle of a tile and one at a sequence's end: rows before it and other sequences are as if
    it were not there, bit for bit; the row's own output and all behind it show it."""
    offsets = [0, 37, 150, 181]
    q, k, v = inputs(10, 190, heads, kv, hs, typ)
    clean = run(lib, q, k, v, offsets)
    at = {36: 0, 90: 1, 149: 1}
    x = {"k": k.copy(), "v": v.copy()}
    for p in at:
        x[where][p, :, 3] = bad
    x[where][181:] = bad  # rows of no sequence
    got = run(lib, q, x["k"], x["v"], offsets)
    seen = np.zeros(190, bool)
    for p, s in at.items():
        seen[p:offsets[s + 1]] = True
    assert np.array_equal(got[~seen], clean[~seen])
    if where == "v":
        assert not np.isfinite(got[seen][:, :, 3]).any()
        other = np.ones(hs, bool)
        other[3] = False
        assert np.array_equal(got[seen][:, :, other], clean[seen][:, :, other])
    elif np.isnan(bad):
        assert np.isnan(got[seen]).all()


@pytest.mark.parametrize("hs", [64, 128])
def test_small_weights_alone(lib, hs):
    """Nearly all of the weight lies where V is zero: what is left is the share of weights of 2^-12 to 2^-18, with their own accuracy."""
    rng = np.random.default_rng(hs)
    rows, heads = 40, 4
    q = np.full((rows, heads, hs), 8 / np.sqrt(hs), F) * (1 + rng.random((rows, heads, 1)).astype(F) * F(0.05))
    k = np.full((rows, heads, hs), -0.6, H) - rng.random((rows, heads, 1)).astype(H) * H(0.15)
    k[0] = H(0.75) * H(8 / np.sqrt(hs))
    k[1:] = k[1:] * H(8 / np.sqrt(hs))
    v = rng.standard_normal((rows, heads, hs)).astype(H)
    v[0] = 0
    with np.errstate(invalid="ignore"):  # (row 0 is zero, and so is its tolerance)
        against(run(lib, q, k, v, [0, rows]), q, k, v, [(0, rows)])


def test_same_bits_twice(lib):
    q, k, v = inputs(11, 700, 8, 2, 64, F)
    a, b = run(lib, q, k, v, [0, 100, 700]), run(lib, q, k, v, [0, 100, 700])
    assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


def test_rows_far_apart(lib):
    """Row offsets beyond 2^31 elements: rows of q and out 2^21 elements apart."""
    rows, heads, kv, hs, stride = 1100, 2, 1, 64, 1 << 21
    q, k, v = inputs(12, rows, heads, kv, hs, H)
    dq, dout = DB(rows * stride * 2), DB(rows * stride * 2)
    dk, dv = DB.from_numpy(k), DB.from_numpy(v)
    keep = [0, 1, 500, rows - 30, rows - 1]
    for r in range(rows):
        dq.upload(q[r], r * stride * 2)
    capi.check(lib.lpp_prompt_attention(dout.ptr, dq.ptr, dk.ptr, dv.ptr, capi.F16, None, 1, rows, heads, kv, hs, stride, kv * hs, stride))
    ends = [j + 1 for j in keep]
    want, _, tol = ko.attend_tolerance(q[keep], k.transpose(1, 0, 2), v.transpose(1, 0, 2), ends, binary16=True)
    got = np.stack([dout.to_numpy(H, heads * hs, r * stride * 2).reshape(heads, hs) for r in keep]).astype(np.float64)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("heads,kv,hs,typ", [(8, 2, 64, F), (8, 8, 64, H), (4, 1, 128, F), (8, 2, 128, H)])
def test_captured_in_a_graph(lib, heads, kv, hs, typ):
    """Captured once, replayed with other rows and offsets in place and eager calls of the library between: the bits of the eager calls."""
    hip = Hip()
    rng = np.random.default_rng(heads + hs)
    rows = 900
    size = 4 if typ is F else 2
    q, k, v, offsets = DB(rows * heads * hs * size), DB(rows * kv * hs * 2), DB(rows * kv * hs * 2), DB(16)
    out = [DB.from_numpy(np.zeros(rows * heads * hs, typ)) for _ in range(2)]
    side, graph, ready = hip.stream(), C.c_void_p(), C.c_void_p()

    def call(into):
        capi.check(lib.lpp_prompt_attention(into.ptr, q.ptr, k.ptr, v.ptr, capi.F32 if typ is F else capi.F16, offsets.ptr, 3, rows, heads, kv, hs,
                                            heads * hs, kv * hs, heads * hs))

    capi.synchronize()
    try:
        capi.check(lib.lpp_set_stream(side))
        hip("hipStreamBeginCapture", side, 2)
        try:
            call(out[0])
        finally:
            hip("hipStreamEndCapture", side, C.byref(graph))
        capi.check(lib.lpp_set_stream(None))
        hip("hipGraphInstantiate", C.byref(ready), graph, None, None, C.c_size_t(0))
        for at in ([0, 1, 300, 900], [0, 0, 0, 0], [5, 400, 401, 899], [0, 900, 900, 900]):
            for buffer, n, t in ((q, heads, typ), (k, kv, H), (v, kv, H)):
                buffer.upload(rng.standard_normal((rows, n * hs)).astype(t))
            offsets.upload(np.array(at, np.int32))
            call(out[1])
            capi.synchronize()
            hip("hipGraphLaunch", ready, side)
            hip("hipStreamSynchronize", side)
            assert np.array_equal(out[0].to_numpy(np.uint8), out[1].to_numpy(np.uint8)), at
        hip("hipGraphExecDestroy", ready)
        hip("hipGraphDestroy", graph)
    finally:
        capi.check(lib.lpp_set_stream(None))
        hip("hipStreamDestroy", side)


@pytest.mark.parametrize("typ", [F, H])
@pytest.mark.parametrize("heads,kv,hs", [(8, 2, 64), (3, 3, 128), (16, 1, 64)])
@pytest.mark.parametrize("lengths", [
    {65: {64: 1}}, {128: {99: 30, 120: 20}}, {128: {s: 1 for s in range(0, 128, 3)}}, {100: {s: 1 for s in range(90, 100)}}, {71: {70: 50}},
    {5000: {0: 3, 2500: 300, 4998: 1, 4999: 40}}, {300: {0: 40}}],
    ids=["one_row_last", "two_of_128", "every_third", "ten_last", "one_prompt_last", "four_of_5000", "one_first"])
def test_fewer_rows_than_sequences(lib, lengths, heads, kv, hs, typ):
    """A table of slots, most of them without a prompt: the rows of every sequence that has some."""
    (seqs, there), = lengths.items()
    lengths = np.zeros(seqs, int)
    for s, n in there.items():
        lengths[s] = n
    assert lengths.sum() < seqs
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    q, k, v = inputs(seqs + heads, int(offsets[-1]), heads, kv, hs, typ)
    against(run(lib, q, k, v, offsets), q, k, v, list(zip(offsets[:-1], offsets[1:])))


@pytest.mark.parametrize("heads,kv,hs,lengths", [(8, 2, 64, [1, 45, 130, 300]), (6, 2, 128, [257, 90]), (32, 8, 64, [700]), (16, 8, 128, [900])])
def test_binary16_is_rounded_once(lib, heads, kv, hs, lengths):
    """Binary16 queries and output: the error of fp32 ones, and the one rounding of the output (half a step: 2^-11 of the value, 2^-25 where it is
    subnormal).  A weight's remainder is kept to 2^-33 of its row's largest."""
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    q, k, v = inputs(sum(lengths) + heads, int(offsets[-1]), heads, kv, hs, H, spread=0.25)
    got = run(lib, q, k, v, offsets).astype(np.float64)
    for a, b in zip(offsets[:-1], offsets[1:]):
        rows = np.unique(np.linspace(0, b - a - 1, 40).astype(int))
        args = q[a:b][rows], k[a:b].transpose(1, 0, 2), v[a:b].transpose(1, 0, 2), [int(j) + 1 for j in rows]
        want, weights, tol = ko.attend_tolerance(*args)
        for h in range(heads):
            tol[:, h] += weights[:, h].max(-1, keepdims=True) * 2.0 ** -33 * np.abs(v[a:b, h * kv // heads].astype(np.float64)).sum(0)
        tol += (np.abs(want) + tol) * 2.0 ** -11 + 2.0 ** -25
        off = np.abs(got[a:b][rows] - want)
        assert np.all(off <= tol), (a, b, float((off / tol).max()))


def rows_of_shape(lib, shape, heads, kv, hs):
    """Rows in all for which the library takes workgroups of 1 x 4, 2 x 2 or 4 x 1 wavefronts (by the tiles of 32 rows there are)."""
    units = C.c_int()
    capi.check(lib.lpp_device_info(None, 0, C.byref(units), None))
    few, many = (2 if hs == 64 else 1) * units.value, 6 * units.value
    tiles = {"1x4": few // 2, "2x2": few + units.value // 2, "4x1": many + units.value // 2}[shape]
    rows = tiles // kv * 32 // (heads // kv)
    assert {"1x4": lambda t: t <= few, "2x2": lambda t: few < t <= many, "4x1": lambda t: t > many}[shape]((rows * (heads // kv) + 31) // 32 * kv)
    return rows


def ragged(rows):
    """Ends inside a tile, a single row, an empty sequence, and a long one."""
    lengths = [1, 37, 0, rows // 5, rows // 7 + 3]
    return lengths + [rows - sum(lengths)]


SHAPES = [(24, 8, 64), (32, 8, 64), (30, 6, 128), (32, 8, 128)]


@pytest.mark.parametrize("typ", [F, H])
@pytest.mark.parametrize("heads,kv,hs", SHAPES)
@pytest.mark.parametrize("shape", ["2x2", "4x1"])
def test_workgroups_of_every_shape(lib, shape, heads, kv, hs, typ):
    """Rows enough for the workgroups that several rows of wavefronts share: a sample of every sequence's rows against the oracle."""
    lengths = ragged(rows_of_shape(lib, shape, heads, kv, hs))
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    q, k, v = inputs(heads * hs + len(shape), int(offsets[-1]), heads, kv, hs, typ)
    got = run(lib, q, k, v, offsets, pad=1)
    for a, b in zip(offsets[:-1], offsets[1:]):
        rows = np.unique(np.clip([0, 1, 31, 32, 62, 63, 64, 127, 128, b - a - 33, b - a - 2, b - a - 1] + list(np.linspace(0, b - a - 1, 9).astype(int)), 0, b - a - 1))
        if a == b:
            continue
        want, _, tol = ko.attend_tolerance(q[a:b][rows], k[a:b].transpose(1, 0, 2), v[a:b].transpose(1, 0, 2), [int(j) + 1 for j in rows],
                                           binary16=typ is H)
        off = np.abs(got[a:b][rows].astype(np.float64) - want)
        assert np.all(off <= tol), (a, b, float((off / tol).max()))


@pytest.mark.parametrize("typ", [F, H])
@pytest.mark.parametrize("heads,kv,hs", SHAPES)
@pytest.mark.parametrize("shape", ["2x2", "4x1"])
@pytest.mark.parametrize("where", ["k", "v"])
def test_nothing_from_other_rows_in_every_shape(lib, where, shape, heads, kv, hs, typ):
    """As above with few rows: NaN rows in the middle and at ends do not reach the rows before them or other sequences, bit for bit."""
    lengths = ragged(rows_of_shape(lib, shape, heads, kv, hs))
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    total = int(offsets[-1])
    q, k, v = inputs(heads + hs, total, heads, kv, hs, typ)
    clean = run(lib, q, k, v, offsets)
    x = {"k": k.copy(), "v": v.copy()}
    seen = np.zeros(total, bool)
    for s, at in ((1, 36), (3, lengths[3] - 1), (4, lengths[4] // 2), (5, lengths[5] * 2 // 3)):
        x[where][offsets[s] + at, :, 3] = np.nan
        seen[offsets[s] + at:offsets[s + 1]] = True
    got = run(lib, q, x["k"], x["v"], offsets)
    assert np.array_equal(got[~seen], clean[~seen])
    if where == "k":
        assert np.isnan(got[seen]).all()
    else:
        assert np.isnan(got[seen][:, :, 3]).all()
        other = np.arange(hs) != 3
        assert np.array_equal(got[seen][:, :, other], clean[seen][:, :, other])
