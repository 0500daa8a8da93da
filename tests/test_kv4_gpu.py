"""The cache of 4 bits (section E of include/lpp.h) on the GPU against 64 bits: rows into it and out of it, attention over it with the weights'
account, its reduction, and all of it together as a serving loop uses it."""
import ctypes as C

import numpy as np
import pytest

import kv4_oracle as ko
from lighterpp_amd import capi
from lighterpp_amd.capi import DeviceBuffer as DB
from lighterpp_amd.capi import LppKv4Shape as Shape

pytestmark = pytest.mark.gpu
F, H, I = np.float32, np.float16, np.int32
EPS32 = 2.0 ** -24


@pytest.fixture(scope="module")
def lib():
    lib = capi.load()
    assert capi.device_count() >= 1, "no HIP device visible"
    capi.check(lib.lpp_init(0))
    return lib


def ints(values):
    return DB.from_numpy(np.array(values, I))


def store(lib, dcache, shape, layer, k, v, offsets, starts, pad=0):
    """k, v [rows, kv_heads, hs]"""
    rows, extra = k.shape[0], 8 * pad
    wide = [np.concatenate([x.reshape(rows, -1), np.full((rows, extra), np.nan, x.dtype)], 1) for x in (k, v)]
    dk, dv = DB.from_numpy(wide[0]), DB.from_numpy(wide[1])
    doff, dst = None if offsets is None else ints(offsets), None if starts is None else ints(starts)
    capi.check(lib.lpp_kv4_store(dcache.ptr, shape, layer, dk.ptr, dv.ptr, capi.F32 if k.dtype == F else capi.F16, wide[0].shape[1],
                                 doff.ptr if doff else None, rows, dst.ptr if dst else None))
    capi.synchronize()


def host_store(cache, layer, k, v, offsets, starts):
    seqs, room = cache.dims[1], cache.dims[3]
    if offsets is None:
        each = k.shape[0] // seqs
        offsets = [s * each for s in range(seqs + 1)]
    for s in range(seqs):
        for j, row in enumerate(range(max(offsets[s], 0), min(offsets[s + 1], k.shape[0]))):
            pos = (0 if starts is None else starts[s]) + j
            if 0 <= pos < room:
                cache.put(0, layer, s, pos, k[row])
                cache.put(1, layer, s, pos, v[row])


def same_bytes(dcache, cache):
    got = dcache.to_numpy(np.uint8)
    mine = ko.Cache(*cache.dims, cache.hs).attach(got)
    for w in range(2):
        assert np.array_equal(mine.codes[w], cache.codes[w]), np.argwhere(mine.codes[w] != cache.codes[w])[:5]
        assert np.array_equal(mine.scales[w], cache.scales[w]), np.argwhere(mine.scales[w] != cache.scales[w])[:5]


# ---- rows into the cache ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("typ", [F, H])
@pytest.mark.parametrize("hs,kv", [(64, 1), (64, 3), (128, 2), (128, 8)])
@pytest.mark.parametrize("rows,offsets,starts", [
    (3, None, [0, 5, 11]),                       # a token each
    (9, None, None),                             # three each, fresh
    (20, [0, 7, 7, 20], [4, 0, 0]),              # ragged, one empty
    (20, [2, 7, 12, 18], None),                  # rows before the first and behind the last sequence
    (12, None, [10, -2, -4]),                    # the end of the room, rows dropped before 0, a sequence skipped
    (12, [0, 4, 8, 12], [2 ** 31 - 1, -2 ** 31, 3]),
    (5, [-3, 2, 90, 2 ** 31 - 1], None),         # offsets outside
])
def test_store_byte_for_byte(lib, rows, offsets, starts, hs, kv, typ):
    rng = np.random.default_rng(rows * hs + kv)
    shape, cache = Shape(2, 3, kv, 13, hs), ko.Cache(2, 3, kv, 13, hs, fill=0xA5)
    dcache = DB.from_numpy(cache.buffer)
    k = (rng.standard_normal((rows, kv, hs)) * np.exp(rng.standard_normal((rows, kv, 1)) * 2)).astype(typ)
    v = (rng.standard_normal((rows, kv, hs)) + 3 * rng.standard_normal((rows, kv, 1))).astype(typ)
    store(lib, dcache, shape, 1, k, v, offsets, starts, pad=2)
    host_store(cache, 1, k, v, offsets, starts)
    same_bytes(dcache, cache)


@pytest.mark.parametrize("n_seqs", [64, 65, 300, 5000])
def test_store_many_sequences(lib, n_seqs):
    rng = np.random.default_rng(n_seqs)
    lengths = rng.integers(0, 4, n_seqs)
    lengths[:3] = lengths[n_seqs // 2:n_seqs // 2 + 20] = 0
    offsets = 2 + np.concatenate([[0], np.cumsum(lengths)])
    rows = int(offsets[-1]) + 3
    starts = rng.integers(-1, 4, n_seqs)
    shape, cache = Shape(1, n_seqs, 1, 5, 64), ko.Cache(1, n_seqs, 1, 5, 64, fill=0x3C)
    dcache = DB.from_numpy(cache.buffer)
    k, v = rng.standard_normal((rows, 1, 64)).astype(F), rng.standard_normal((rows, 1, 64)).astype(F)
    store(lib, dcache, shape, 0, k, v, offsets, starts)
    host_store(cache, 0, k, v, offsets, starts)
    same_bytes(dcache, cache)


def test_store_values_on_borders_and_extreme_groups(lib):
    """Values exactly between two codes (ties go to the even one), one step either side of them, constant groups, subnormal scales, the
    ends of the range, and everything beyond."""
    hs, room = 64, 64
    rng = np.random.default_rng(3)
    rows = []
    for low, scale in [(0.0, 1.0), (-2.0, 0.25), (0.5, 2.0 ** -10), (-7.0, 3.0), (1000.0, 1.0), (-0.1, 0.0123)]:
        low, scale = F(H(low)), F(H(scale))
        at = low + scale * (np.arange(15, dtype=F) + F(0.5))
        g = np.concatenate([[low], at, [low + 15 * scale]] + [np.nextafter(at, F(np.inf))[:8], np.nextafter(at, F(-np.inf))[:7]])
        rows.append(np.concatenate([g, g[::-1]]))
    rows.append(np.concatenate([np.full(32, 0.3), np.full(32, -1e-7)]))
    rows.append(np.concatenate([rng.random(32) * 1e-6, 1.0 + rng.random(32) * 1e-6]))
    rows.append(np.concatenate([np.linspace(-32768, 32768, 32), np.linspace(0, 6e-5, 32)]))
    for bad in (np.nan, np.inf, -np.inf, 32769.0, -4e4, 1e30):
        r = rng.standard_normal(64)
        r[17] = bad
        rows.append(r)
    rows.append(np.concatenate([np.full(32, 1e-40), np.zeros(32)]))
    x = np.array(rows, F)[:, None, :]
    shape, cache = Shape(1, 1, 1, room, hs), ko.Cache(1, 1, 1, room, hs)
    dcache = DB.from_numpy(cache.buffer)
    store(lib, dcache, shape, 0, x, x[::-1].copy(), None, None)
    host_store(cache, 0, x, x[::-1], None, None)
    same_bytes(dcache, cache)
    # a value is off by half a step of its group at most, and by the roundings of lowest, scale (fifteen times) and sum
    n = x.shape[0] - 7
    dk, dv = DB(room * hs * 2), DB(room * hs * 2)
    capi.check(lib.lpp_kv4_load(dk.ptr, dv.ptr, dcache.ptr, shape, 0, 0, room))
    got = dk.to_numpy(H).reshape(room, hs)[:n].astype(np.float64)
    g = x[:n, 0].astype(np.float64).reshape(n, 2, 32)
    span, size = g.max(-1) - g.min(-1), np.abs(g).max(-1)
    bound = span / 30 + span * 2.0 ** -11 + 2 * size * 2.0 ** -11 + 17 * 2.0 ** -25
    assert np.all(np.abs(got.reshape(n, 2, 32) - g) <= bound[..., None])


def test_store_many_rows_against_the_oracle(lib):
    """A million values of one distribution: every code, those next to a border included."""
    rng = np.random.default_rng(9)
    rows, kv, hs = 1000, 8, 128
    shape, cache = Shape(1, 1, kv, rows, hs), ko.Cache(1, 1, kv, rows, hs)
    dcache = DB.from_numpy(cache.buffer)
    k, v = rng.standard_normal((rows, kv, hs)).astype(F), rng.standard_normal((rows, kv, hs)).astype(F)
    store(lib, dcache, shape, 0, k, v, [0, rows], [0])
    host_store(cache, 0, k, v, [0, rows], [0])
    same_bytes(dcache, cache)


@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("first,count", [(0, 37), (5, 1), (36, 1), (3, 30)])
def test_load(lib, hs, first, count):
    rng = np.random.default_rng(hs + first)
    cache = ko.Cache(3, 2, 5, 37, hs)
    cache.buffer[:] = rng.integers(0, 256, cache.buffer.size, dtype=np.uint8)
    for s in cache.scales:  # (any binary16 but NaN, whose bits need not survive)
        for part in (0, 16):
            exponent = (s >> part) & 0x7C00
            s[exponent == 0x7C00] ^= np.uint32(0x4000 << part)
    dcache = DB.from_numpy(cache.buffer)
    n = 2 * 5 * count * hs
    dk, dv = DB.from_numpy(np.full(n + 8, 3.0, H)), DB.from_numpy(np.full(n + 8, 3.0, H))
    capi.check(lib.lpp_kv4_load(dk.ptr, dv.ptr, dcache.ptr, Shape(3, 2, 5, 37, hs), 2, first, count))
    for which, d in enumerate((dk, dv)):
        got = d.to_numpy(H)
        want = cache.values(which, 2)[:, :, first:first + count]
        assert np.array_equal(got[:n].view(np.uint16), np.ascontiguousarray(want).reshape(-1).view(np.uint16))
        assert np.all(got[n:] == 3.0)


# ---- attention over it --------------------------------------------------------------------------------------------------------------

def random_cache(rng, layers, seqs, kv, room, hs):
    cache = ko.Cache(layers, seqs, kv, room, hs)
    for c in cache.codes:
        c[...] = rng.integers(0, 2 ** 32, c.shape, dtype=np.uint32)
    for s in cache.scales:
        scale = rng.uniform(0.1, 0.4, s.shape)
        low = scale * rng.uniform(-8.5, -6.5, s.shape)
        s[...] = scale.astype(H).view(np.uint16).astype(np.uint32) | (low.astype(H).view(np.uint16).astype(np.uint32) << 16)
    return cache


def attend(lib, dcache, cache, layer, q, starts, mass=None, workspace=None):
    """q [seqs, n_q, heads, hs] -> out, mass (all layers)"""
    seqs, n_q, heads, hs = q.shape
    shape = Shape(*cache.dims, hs)
    need = C.c_size_t()
    capi.check(lib.lpp_kv4_attention_workspace(shape, heads, n_q, C.byref(need)))
    # (filled with NaN: nothing may be taken from it)
    work = workspace or DB.from_numpy(np.full(need.value // 4 + 64, np.nan, F))
    dq, dout, dst = DB.from_numpy(q), DB.from_numpy(np.full(q.size + 4, 7.25, F)), ints(starts)
    dmass = None if mass is None else DB.from_numpy(mass)
    capi.check(lib.lpp_kv4_attention(dout.ptr, dq.ptr, dcache.ptr, shape, layer, heads, n_q, dst.ptr, dmass.ptr if dmass else None, work.ptr, need.value))
    got = dout.to_numpy(F)
    assert np.all(got[q.size:] == 7.25)
    if workspace is None:
        assert np.all(np.isnan(work.to_numpy(F)[need.value // 4:]))
    return got[:q.size].reshape(q.shape), None if dmass is None else dmass.to_numpy(F).reshape(mass.shape)


def check_attention(got, got_mass, cache, layer, q, starts, mass):
    seqs, n_q, heads, hs = q.shape
    kv, room = cache.dims[2], cache.dims[3]
    k, v = cache.values(0, layer), cache.values(1, layer)
    for s in range(seqs):
        ends = [int(np.clip(int(starts[s]) + j + 1, 0, room)) for j in range(n_q)]
        want, weights, tol = ko.attend_tolerance(q[s], k[s], v[s], ends)
        off = np.abs(got[s] - want)
        assert np.all(off <= tol), (s, float((off / np.maximum(tol, 1e-30)).max()))
        if mass is None:
            continue
        d = ko.score_error(q[s], k[s], ends).max()
        add = weights.reshape(n_q, kv, heads // kv, room).sum((0, 2))
        # relative to what is added (its weights' error as above, the sum of n_q * shared terms), and the rounding of the new total
        bound = add * (2 * d + 2.0 ** -20 + (n_q * heads // kv + 2 * max(ends)) * EPS32) + np.abs(mass[layer, s] + add) * EPS32 + 1e-37
        off = np.abs(got_mass[layer, s].astype(np.float64) - (mass[layer, s].astype(np.float64) + add))
        assert np.all(off <= bound), (s, float((off / bound).max()))
    if mass is not None:
        others = [i for i in range(cache.dims[0]) if i != layer]
        assert np.array_equal(got_mass[others], mass[others])


GROUPS = [(1, 1, 64), (4, 2, 64), (8, 2, 64), (8, 1, 64), (3, 1, 128), (16, 1, 128), (4, 4, 128), (15, 1, 64)]


@pytest.mark.parametrize("heads,kv,hs", GROUPS)
@pytest.mark.parametrize("lengths", [[1], [2, 31, 32], [33, 0, 64], [127, 128, 129, 1], [300, 257, 512, 511]], ids=str)
@pytest.mark.parametrize("with_mass", [False, True])
def test_decode_step(lib, lengths, heads, kv, hs, with_mass):
    rng = np.random.default_rng(sum(lengths) + heads * hs)
    seqs = len(lengths)
    cache = random_cache(rng, 2, seqs, kv, max(lengths), hs)
    dcache = DB.from_numpy(cache.buffer)
    q = rng.standard_normal((seqs, 1, heads, hs)).astype(F)
    mass = rng.random((2, seqs, kv, max(lengths))).astype(F) if with_mass else None
    starts = [n - 1 for n in lengths]
    got, got_mass = attend(lib, dcache, cache, 1, q, starts, mass)
    check_attention(got, got_mass, cache, 1, q, starts, mass)


@pytest.mark.parametrize("heads,kv,hs", GROUPS)
@pytest.mark.parametrize("n_q", [2, 3, 7, 16, 33])
def test_several_rows(lib, n_q, heads, kv, hs):
    """Draft tokens or a prompt's last rows: ends inside a tile, rows that attend to nothing, rows past the room."""
    rng = np.random.default_rng(n_q * 100 + heads)
    starts = [0, 90, -2, 200 - n_q, -n_q - 3, 198]
    cache = random_cache(rng, 1, len(starts), kv, 200, hs)
    dcache = DB.from_numpy(cache.buffer)
    q = rng.standard_normal((len(starts), n_q, heads, hs)).astype(F)
    mass = rng.random((1, len(starts), kv, 200)).astype(F)
    got, got_mass = attend(lib, dcache, cache, 0, q, starts, mass)
    check_attention(got, got_mass, cache, 0, q, starts, mass)
    plain, _ = attend(lib, dcache, cache, 0, q, starts)
    assert np.array_equal(plain, got)


@pytest.mark.parametrize("heads,kv,hs,length", [(4, 1, 64, 9001), (2, 1, 128, 20000), (8, 8, 64, 4099), (8, 1, 128, 5000)])
def test_long_context(lib, heads, kv, hs, length):
    rng = np.random.default_rng(length)
    cache = random_cache(rng, 1, 1, kv, length + 7, hs)
    dcache = DB.from_numpy(cache.buffer)
    q = rng.standard_normal((1, 1, heads, hs)).astype(F)
    mass = rng.random((1, 1, kv, length + 7)).astype(F)
    got, got_mass = attend(lib, dcache, cache, 0, q, [length - 1], mass)
    check_attention(got, got_mass, cache, 0, q, [length - 1], mass)


@pytest.mark.parametrize("heads,kv,hs,n_q,lengths", [(16, 1, 64, 1, [4001]), (8, 2, 64, 1, [20011, 33]), (12, 1, 128, 1, [12001]), (4, 1, 64, 4, [3001, 900, 2])])
def test_account_of_long_contexts(lib, heads, kv, hs, n_q, lengths):
    """So many scores for each position that they are made again from K rather than kept."""
    rng = np.random.default_rng(lengths[0])
    room = lengths[0] + 2
    cache = random_cache(rng, 1, len(lengths), kv, room, hs)
    q = rng.standard_normal((len(lengths), n_q, heads, hs)).astype(F)
    mass = rng.random((1, len(lengths), kv, room)).astype(F)
    starts = [n - n_q for n in lengths]
    got, got_mass = attend(lib, DB.from_numpy(cache.buffer), cache, 0, q, starts, mass)
    check_attention(got, got_mass, cache, 0, q, starts, mass)


def test_more_sequences_than_compute_units(lib):
    """Work enough without splitting anything."""
    rng = np.random.default_rng(77)
    seqs, kv, hs = 90, 4, 64
    lengths = rng.integers(0, 150, seqs)
    cache = random_cache(rng, 1, seqs, kv, 150, hs)
    dcache = DB.from_numpy(cache.buffer)
    q = rng.standard_normal((seqs, 1, 8, hs)).astype(F)
    mass = np.zeros((1, seqs, kv, 150), F)
    got, got_mass = attend(lib, dcache, cache, 0, q, lengths - 1, mass)
    check_attention(got, got_mass, cache, 0, q, lengths - 1, mass)


@pytest.mark.parametrize("n_seqs,n_q", [(300, 1), (300, 5), (2000, 1)])
def test_very_many_sequences(lib, n_seqs, n_q):
    rng = np.random.default_rng(n_seqs + n_q)
    room = 40 if n_seqs > 1000 else 700
    lengths = rng.integers(0, 30, n_seqs)
    lengths[7], lengths[n_seqs - 1] = room, room - 1
    cache = random_cache(rng, 1, n_seqs, 1, room, 64)
    q = rng.standard_normal((n_seqs, n_q, 2, 64)).astype(F)
    mass = np.zeros((1, n_seqs, 1, room), F)
    got, got_mass = attend(lib, DB.from_numpy(cache.buffer), cache, 0, q, lengths - n_q, mass)
    check_attention(got, got_mass, cache, 0, q, lengths - n_q, mass)


@pytest.mark.parametrize("hs", [64, 128])
def test_large_scores(lib, hs):
    """Scores of hundreds that grow along the cache, and a row whose every score is far below zero."""
    rng = np.random.default_rng(4)
    room = 700
    cache = random_cache(rng, 1, 2, 1, room, hs)
    k = rng.standard_normal((room, 1, hs)) * np.linspace(0.1, 8.0, room)[:, None, None]
    for p in range(room):
        cache.put(0, 0, 0, p, k[p].astype(F))
        cache.put(0, 0, 1, p, np.full((1, hs), 2.0, F) + rng.random((1, hs)).astype(F))
    dcache = DB.from_numpy(cache.buffer)
    q = (rng.standard_normal((2, 1, 4, hs)) * 5).astype(F)
    q[1] = -np.abs(q[1])
    mass = np.zeros((1, 2, 1, room), F)
    got, got_mass = attend(lib, dcache, cache, 0, q, [room - 1, room - 1], mass)
    check_attention(got, got_mass, cache, 0, q, [room - 1, room - 1], mass)


@pytest.mark.parametrize("hs", [64, 128])
def test_small_weights_alone(lib, hs):
    """Nearly all of the weight lies where V is zero: what is left is the share of weights of 2^-12 to 2^-18, with their own accuracy."""
    rng = np.random.default_rng(hs)
    room, heads, scale = 40, 4, 8 / np.sqrt(hs)
    cache = random_cache(rng, 1, 1, heads, room, hs)
    for p in range(room):
        k = np.full((heads, hs), 0.75 if p == 0 else -0.6, F) - (0 if p == 0 else rng.random((heads, 1)).astype(F) * F(0.15))
        cache.put(0, 0, 0, p, (k * scale).astype(F))
        cache.put(1, 0, 0, p, np.zeros((heads, hs), F) if p == 0 else rng.standard_normal((heads, hs)).astype(F))
    q = np.full((1, 3, heads, hs), scale, F) * (1 + rng.random((1, 3, heads, 1)).astype(F) * F(0.05))
    got, _ = attend(lib, DB.from_numpy(cache.buffer), cache, 0, q, [room - 3])
    check_attention(got, None, cache, 0, q, [room - 3], None)


@pytest.mark.parametrize("heads,kv,hs", [(4, 4, 64), (8, 1, 64), (6, 2, 128)])
@pytest.mark.parametrize("n_q", [1, 5])
@pytest.mark.parametrize("where", [0, 1])
def test_nothing_comes_from_positions_a_row_does_not_attend_to(lib, where, n_q, heads, kv, hs):
    """Groups that stand for NaN at positions behind a row's end, also those of the rows after it, and everywhere in the room behind."""
    rng = np.random.default_rng(hs + n_q)
    starts, room = [40, 95, 0], 130
    cache = random_cache(rng, 1, 3, kv, room, hs)
    q = rng.standard_normal((3, n_q, heads, hs)).astype(F)
    mass = np.zeros((1, 3, kv, room), F)
    clean, clean_mass = attend(lib, DB.from_numpy(cache.buffer), cache, 0, q, starts, mass)
    row = min(3, n_q)  # rows `row` and later attend to it
    for s, start in enumerate(starts):
        cache.scales[where][0, s, :, start + row:] = 0x7E000000
        cache.codes[where][0, s, :, start + row:] = 0
    got, got_mass = attend(lib, DB.from_numpy(cache.buffer), cache, 0, q, starts, mass)
    assert np.array_equal(got[:, :row], clean[:, :row])
    assert np.isnan(got[:, row:]).all()
    if n_q == 1 or where == 1:
        assert np.array_equal(got_mass, clean_mass)
    for s, start in enumerate(starts):
        assert np.all(got_mass[0, s, :, start + n_q:] == 0)


def test_infinite_values_show(lib):
    """l + code * c beyond binary16 is an infinity; with weights of zero elsewhere the others stay as they are."""
    rng = np.random.default_rng(8)
    cache = random_cache(rng, 1, 1, 1, 50, 64)
    q = rng.standard_normal((1, 1, 2, 64)).astype(F)
    clean, _ = attend(lib, DB.from_numpy(cache.buffer), cache, 0, q, [49])
    cache.scales[1][0, 0, 0, 20, 1] = 0x7BFF7BFF  # 65504 + code * 65504
    cache.codes[1][0, 0, 0, 20, 4:] = 0x11111111
    got, _ = attend(lib, DB.from_numpy(cache.buffer), cache, 0, q, [49])
    assert np.all(got[..., 32:] == np.inf) and np.array_equal(got[..., :32], clean[..., :32])


def test_same_bits_twice(lib):
    rng = np.random.default_rng(12)
    cache = random_cache(rng, 1, 2, 2, 3000, 64)
    dcache = DB.from_numpy(cache.buffer)
    q = rng.standard_normal((2, 3, 8, 64)).astype(F)
    mass = rng.random((1, 2, 2, 3000)).astype(F)
    runs = [attend(lib, dcache, cache, 0, q, [2000, 2996], mass) for _ in range(3)]
    for out, m in runs[1:]:
        assert np.array_equal(out.view(np.uint32), runs[0][0].view(np.uint32)) and np.array_equal(m.view(np.uint32), runs[0][1].view(np.uint32))


def test_offsets_beyond_32_bits(lib):
    """A cache of 20 GB: the last sequence's last KV head lies beyond 2^32 bytes and 2^31 words of every part."""
    layers, seqs, kv, room, hs = 2, 16, 8, 1 << 19, 128
    shape = Shape(layers, seqs, kv, room, hs)
    need = C.c_size_t()
    capi.check(lib.lpp_kv4_bytes(shape, C.byref(need)))
    assert need.value > 20e9
    dcache = DB(need.value)
    rng = np.random.default_rng(1)
    small = ko.Cache(1, seqs, kv, 40, hs)
    k, v = rng.standard_normal((40 * seqs, kv, hs)).astype(H), rng.standard_normal((40 * seqs, kv, hs)).astype(H)
    store(lib, dcache, shape, 1, k, v, None, None)
    host_store(small, 0, k, v, None, None)
    q = rng.standard_normal((seqs, 2, 16, hs)).astype(F)
    capi.check(lib.lpp_kv4_attention_workspace(shape, 16, 2, C.byref(need)))
    work, dq, dout, dst = DB(need.value), DB.from_numpy(q), DB(q.nbytes), ints([38] * seqs)
    dmass = DB(layers * seqs * kv * room * 4)
    capi.check(lib.lpp_memset(dmass.ptr, 0, dmass.nbytes))
    capi.check(lib.lpp_kv4_attention(dout.ptr, dq.ptr, dcache.ptr, shape, 1, 16, 2, dst.ptr, dmass.ptr, work.ptr, need.value))
    got_mass = np.stack([dmass.to_numpy(F, 40, 4 * ((layers // 2 * seqs * kv + p) * room)) for p in range(seqs * kv)]).reshape(1, seqs, kv, 40)
    check_attention(dout.to_numpy(F).reshape(q.shape), got_mass, small, 0, q, [38] * seqs, np.zeros((1, seqs, kv, 40), F))
    dk, dv = DB(seqs * kv * 40 * hs * 2), DB(seqs * kv * 40 * hs * 2)
    capi.check(lib.lpp_kv4_load(dk.ptr, dv.ptr, dcache.ptr, shape, 1, 0, 40))
    assert np.array_equal(dv.to_numpy(H), small.values(1).reshape(-1))
    # reduced into a small cache
    less = Shape(1, seqs, kv, 10, hs)
    capi.check(lib.lpp_kv4_bytes(less, C.byref(need)))
    dless, dless_mass, dlen, dkept = DB(need.value), DB(seqs * kv * 10 * 4), ints([0] * seqs), DB(seqs * kv * 10 * 4)
    capi.check(lib.lpp_kv4_evict(dless.ptr, less, 0, dless_mass.ptr, dlen.ptr, dkept.ptr, dcache.ptr, shape, 1, dmass.ptr, ints([40] * seqs).ptr, 10, 3))
    kept = dkept.to_numpy(I).reshape(seqs, kv, 10)
    for s in range(seqs):
        for h in range(kv):
            assert np.array_equal(kept[s, h], ko.keep_positions(got_mass[0, s, h], 40, 10, 3))
    dk, dv = DB(seqs * kv * 10 * hs * 2), DB(seqs * kv * 10 * hs * 2)
    capi.check(lib.lpp_kv4_load(dk.ptr, dv.ptr, dless.ptr, less, 0, 0, 10))
    want = np.take_along_axis(small.values(0), kept[..., None].astype(np.int64), 2)
    assert np.array_equal(dk.to_numpy(H), want.reshape(-1))


# ---- its reduction ----------------------------------------------------------------------------------------------------------------------

def evict(lib, cache, mass, lengths, keep, recent, room, layer=0, dst_layers=1, dst_layer=0):
    seqs, kv = cache.dims[1], cache.dims[2]
    less = ko.Cache(dst_layers, seqs, kv, room, cache.hs, fill=0x5A)
    before = ko.Cache(dst_layers, seqs, kv, room, cache.hs, fill=0x5A)
    dsrc, ddst = DB.from_numpy(cache.buffer), DB.from_numpy(less.buffer)
    dmass, dless_mass = DB.from_numpy(mass), DB.from_numpy(np.full((dst_layers, seqs, kv, room), -9.0, F))
    dlen, dless_len, dkept = ints(lengths), ints([-1] * seqs), DB.from_numpy(np.full(seqs * kv * keep + 3, 77, I))
    capi.check(lib.lpp_kv4_evict(ddst.ptr, Shape(dst_layers, seqs, kv, room, cache.hs), dst_layer, dless_mass.ptr, dless_len.ptr, dkept.ptr, dsrc.ptr,
                                 Shape(*cache.dims, cache.hs), layer, dmass.ptr, dlen.ptr, keep, recent))
    less.attach(ddst.to_numpy(np.uint8))
    kept = dkept.to_numpy(I)
    assert np.all(kept[-3:] == 77)
    kept = kept[:-3].reshape(seqs, kv, keep)
    got_mass = dless_mass.to_numpy(F).reshape(dst_layers, seqs, kv, room)
    assert np.array_equal(dsrc.to_numpy(np.uint8), cache.buffer) and np.array_equal(dlen.to_numpy(I), np.array(lengths, I))
    full = cache.dims[3]
    for s in range(seqs):
        n = int(np.clip(lengths[s], 0, full))
        assert dless_len.to_numpy(I)[s] == min(n, keep)
        for h in range(kv):
            want = ko.keep_positions(mass[layer, s, h], n, keep, recent)
            m = len(want)
            assert np.array_equal(kept[s, h, :m], want), (s, h)
            assert np.all(kept[s, h, m:] == -1)
            assert np.array_equal(got_mass[dst_layer, s, h, :m], mass[layer, s, h, want], equal_nan=True)
            assert np.all(got_mass[dst_layer, s, h, m:] == 0)
            for w in range(2):
                assert np.array_equal(less.codes[w][dst_layer, s, h, :m], cache.codes[w][layer, s, h, want])
                assert np.array_equal(less.scales[w][dst_layer, s, h, :m], cache.scales[w][layer, s, h, want])
                assert np.array_equal(less.codes[w][dst_layer, s, h, m:], before.codes[w][dst_layer, s, h, m:])
                assert np.array_equal(less.scales[w][dst_layer, s, h, m:], before.scales[w][dst_layer, s, h, m:])
    for other in range(dst_layers):
        if other != dst_layer:
            assert np.all(got_mass[other] == -9.0)
            for w in range(2):
                assert np.array_equal(less.codes[w][other], before.codes[w][other])
    return kept


@pytest.mark.parametrize("hs,kv", [(64, 2), (128, 3)])
@pytest.mark.parametrize("lengths,keep,recent,room", [
    ([1], 1, 0, 1), ([5, 0, 9], 4, 2, 4), ([100, 64, 3], 64, 64, 70), ([1024, 1025, 2047], 300, 0, 300), ([1500, -4, 9999], 1, 1, 5),
    ([1500, 1499, 700], 1499, 10, 1499), ([3000], 999, 33, 1200), ([5000], 4000, 17, 4001), ([20000], 77, 5, 80), ([40000, 70000], 36000, 100, 36000)], ids=str)
def test_evict(lib, lengths, keep, recent, room, hs, kv):
    rng = np.random.default_rng(keep + hs)
    full = max(max(lengths), 1) if 9999 not in lengths else 1500
    cache = random_cache(rng, 2, len(lengths), kv, full, hs)
    mass = np.exp(2 * rng.standard_normal((2, len(lengths), kv, full))).astype(F)
    mass = np.round(mass * 16) / F(16)  # (many equal ones)
    evict(lib, cache, mass.astype(F), lengths, keep, recent, room, layer=1, dst_layers=3, dst_layer=2)


@pytest.mark.parametrize("kind", ["equal", "zero", "signs", "nan", "close", "one"])
def test_evict_weights_of_all_sorts(lib, kind):
    rng = np.random.default_rng(2)
    n = 2500
    mass = {"equal": np.full(n, 0.7), "zero": np.where(np.arange(n) % 2, 0.0, -0.0), "signs": rng.standard_normal(n) * 10.0 ** rng.integers(-40, 30, n),
            "nan": np.where(rng.random(n) < 0.01, np.nan, rng.random(n)), "close": 1.0 + rng.integers(0, 5, n) * 2.0 ** -23,
            "one": np.where(np.arange(n) == 1234, np.inf, 0.0)}[kind].astype(F).reshape(1, 1, 1, n)
    cache = random_cache(rng, 1, 1, 1, n, 64)
    for keep, recent in [(1, 0), (700, 100), (2499, 0), (2499, 2499)]:
        evict(lib, cache, mass, [n], keep, recent, keep)


# ---- together ---------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv,hs", [(8, 2, 64), (6, 2, 128)])
def test_serving_loop(lib, heads, kv, hs):
    """Two layers, three prompts: attention of the packed prompts, their rows stored, their last rows asked once more for the weights, decode
    steps with the account, the cache reduced into a smaller one, and decode steps from there; every output against 64 bits on what the
    cache holds, the cache byte for byte."""
    rng = np.random.default_rng(hs)
    layers, lengths, steps, keep, recent, window = 2, [70, 9, 41], 3, 24, 6, 4
    seqs, room, less_room = 3, 80, 32
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(I)
    total = int(offsets[-1])
    big, small = Shape(layers, seqs, kv, room, hs), Shape(layers, seqs, kv, less_room, hs)
    need = C.c_size_t()
    capi.check(lib.lpp_kv4_attention_workspace(big, heads, window, C.byref(need)))
    work = DB(need.value)
    host = ko.Cache(layers, seqs, kv, room, hs)
    dbig = DB.from_numpy(host.buffer)
    mass = np.zeros((layers, seqs, kv, room), F)
    last_q = []
    for layer in range(layers):
        q = rng.standard_normal((total, heads, hs)).astype(F)
        k32, v32 = (rng.standard_normal((total, kv, hs)).astype(F) for _ in range(2))
        d32, d16, dq, dout, doff = [DB.from_numpy(x) for x in (k32, v32)], [DB(k32.size * 2) for _ in range(2)], DB.from_numpy(q), DB(q.nbytes), DB.from_numpy(offsets)
        for a, b in zip(d16, d32):
            capi.check(lib.lpp_convert_f32_to_f16(a.ptr, b.ptr, k32.size))
        capi.check(lib.lpp_prompt_attention(dout.ptr, dq.ptr, d16[0].ptr, d16[1].ptr, capi.F32, doff.ptr, seqs, total, heads, kv, hs, heads * hs, kv * hs, heads * hs))
        capi.check(lib.lpp_kv4_store(dbig.ptr, big, layer, d16[0].ptr, d16[1].ptr, capi.F16, kv * hs, doff.ptr, total, None))
        got = dout.to_numpy(F).reshape(q.shape)
        k, v = k32.astype(H), v32.astype(H)
        for s in range(seqs):
            a, b = offsets[s], offsets[s + 1]
            want, _, tol = ko.attend_tolerance(q[a:b], k[a:b].transpose(1, 0, 2), v[a:b].transpose(1, 0, 2), list(range(1, b - a + 1)))
            assert np.all(np.abs(got[a:b] - want) <= tol)
        host_store(host, layer, k, v, offsets, None)
        last_q.append(np.stack([q[offsets[s + 1] - window:offsets[s + 1]] for s in range(seqs)]))
    same_bytes(dbig, host)
    for layer in range(layers):
        starts = [n - window for n in lengths]
        got, after = attend(lib, dbig, host, layer, last_q[layer], starts, mass, work)
        check_attention(got, after, host, layer, last_q[layer], starts, mass)
        mass = after

    def decode(dcache, cache, lengths, mass):
        for _ in range(steps):
            for layer in range(layers):
                k, v = (rng.standard_normal((seqs, kv, hs)).astype(F) for _ in range(2))
                q = rng.standard_normal((seqs, 1, heads, hs)).astype(F)
                store(lib, dcache, Shape(*cache.dims, hs), layer, k, v, None, lengths)
                host_store(cache, layer, k, v, None, lengths)
                got, after = attend(lib, dcache, cache, layer, q, lengths, mass, work)
                check_attention(got, after, cache, layer, q, lengths, mass)
                mass = after
            lengths = [n + 1 for n in lengths]
        same_bytes(dcache, cache)
        return lengths, mass

    lengths, mass = decode(dbig, host, lengths, mass)
    less = ko.Cache(layers, seqs, kv, less_room, hs)
    dsmall, dmass, dless_mass = DB.from_numpy(less.buffer), DB.from_numpy(mass), DB.from_numpy(np.full((layers, seqs, kv, less_room), 5.0, F))
    dlen, dnew, dkept = ints(lengths), ints([0] * seqs), DB(seqs * kv * keep * 4)
    for layer in range(layers):
        capi.check(lib.lpp_kv4_evict(dsmall.ptr, small, layer, dless_mass.ptr, dnew.ptr, dkept.ptr, dbig.ptr, big, layer, dmass.ptr, dlen.ptr, keep, recent))
        for s in range(seqs):
            for h in range(kv):
                at = ko.keep_positions(mass[layer, s, h], lengths[s], keep, recent)
                for w in range(2):
                    less.codes[w][layer, s, h, :len(at)] = host.codes[w][layer, s, h, at]
                    less.scales[w][layer, s, h, :len(at)] = host.scales[w][layer, s, h, at]
    same_bytes(dsmall, less)
    lengths = [min(n, keep) for n in lengths]
    assert dnew.to_numpy(I).tolist() == lengths
    decode(dsmall, less, lengths, dless_mass.to_numpy(F).reshape(layers, seqs, kv, less_room))


class Hip:
    """Streams and graphs of the HIP runtime the library itself is linked against."""

    def __init__(self):
        self.lib = C.CDLL("libamdhip64.so")

    def __call__(self, name, *args):
        status = getattr(self.lib, name)(*args)
        assert status == 0, (name, status)

    def stream(self):
        s = C.c_void_p()
        self("hipStreamCreateWithFlags", C.byref(s), 1)  # non-blocking
        return s


def test_steps_captured_in_a_graph(lib):
    """Store, attention with the account and eviction captured once on a caller's stream, replayed with new rows and lengths in place and
    eager calls of the library between: every replay gives the bits of the eager calls."""
    rng = np.random.default_rng(31)
    hip = Hip()
    seqs, heads, kv, hs, room, keep = 2, 8, 2, 64, 700, 100
    shape, less = Shape(1, seqs, kv, room, hs), Shape(1, seqs, kv, keep, hs)
    need = C.c_size_t()
    capi.check(lib.lpp_kv4_attention_workspace(shape, heads, 1, C.byref(need)))
    cache = random_cache(rng, 1, seqs, kv, room, hs)
    sizes = {"mass": seqs * kv * room * 4, "out": seqs * heads * hs * 4, "less": seqs * kv * keep * hs * 5 // 4, "less_mass": seqs * kv * keep * 4, "less_len": seqs * 4,
             "kept": seqs * kv * keep * 4}

    def state():
        return {"cache": DB.from_numpy(cache.buffer), "work": DB(need.value)} | {name: DB.from_numpy(np.zeros(n, np.uint8)) for name, n in sizes.items()}

    q, k, v, starts, lengths = DB(seqs * heads * hs * 4), DB(seqs * kv * hs * 4), DB(seqs * kv * hs * 4), DB(4 * seqs), DB(4 * seqs)

    def step(s):
        p = {name: x.ptr for name, x in s.items()}
        capi.check(lib.lpp_kv4_store(p["cache"], shape, 0, k.ptr, v.ptr, capi.F32, kv * hs, None, seqs, starts.ptr))
        capi.check(lib.lpp_kv4_attention(p["out"], q.ptr, p["cache"], shape, 0, heads, 1, starts.ptr, p["mass"], p["work"], need.value))
        capi.check(lib.lpp_kv4_evict(p["less"], less, 0, p["less_mass"], p["less_len"], p["kept"], p["cache"], shape, 0, p["mass"], lengths.ptr, keep, 8))

    eager, captured = state(), state()
    side, graph, ready = hip.stream(), C.c_void_p(), C.c_void_p()
    capi.synchronize()
    try:
        capi.check(lib.lpp_set_stream(side))
        hip("hipStreamBeginCapture", side, 2)
        try:
            step(captured)
        finally:
            hip("hipStreamEndCapture", side, C.byref(graph))
        capi.check(lib.lpp_set_stream(None))
        hip("hipGraphInstantiate", C.byref(ready), graph, None, None, C.c_size_t(0))
        for at in (300, 301, 10, 698, 0):
            q.upload(rng.standard_normal((seqs, heads * hs)).astype(F))
            k.upload(rng.standard_normal((seqs, kv * hs)).astype(F))
            v.upload(rng.standard_normal((seqs, kv * hs)).astype(F))
            starts.upload(np.array([at, at // 2], I))
            lengths.upload(np.array([at + 1, at // 2 + 1], I))
            step(eager)
            capi.synchronize()
            hip("hipGraphLaunch", ready, side)
            hip("hipStreamSynchronize", side)
            for name in eager:
                if name != "work":
                    assert np.array_equal(eager[name].to_numpy(np.uint8), captured[name].to_numpy(np.uint8)), (at, name)
        hip("hipGraphExecDestroy", ready)
        hip("hipGraphDestroy", graph)
    finally:
        capi.check(lib.lpp_set_stream(None))
        hip("hipStreamDestroy", side)


def test_two_streams_at_once(lib):
    """Calls on two streams that may overlap, a workspace each: the bits of the calls one after the other."""
    rng = np.random.default_rng(32)
    hip = Hip()
    heads, kv, hs, room = 8, 2, 64, 4000
    cache = random_cache(rng, 1, 1, kv, room, hs)
    shape = Shape(1, 1, kv, room, hs)
    need = C.c_size_t()
    capi.check(lib.lpp_kv4_attention_workspace(shape, heads, 4, C.byref(need)))
    dcache, start = DB.from_numpy(cache.buffer), ints([3990])
    q = [DB.from_numpy(rng.standard_normal((4, heads * hs)).astype(F)) for _ in range(2)]
    out = [DB(4 * 4 * heads * hs) for _ in range(4)]
    mass = [DB.from_numpy(np.zeros((kv, room), F)) for _ in range(4)]
    work = [DB(need.value) for _ in range(2)]
    capi.synchronize()
    streams = [hip.stream(), hip.stream()]

    def call(i, into):
        capi.check(lib.lpp_kv4_attention(out[into].ptr, q[i].ptr, dcache.ptr, shape, 0, heads, 4, start.ptr, mass[into].ptr, work[i].ptr, need.value))

    try:
        for _ in range(20):
            for i in range(2):
                capi.check(lib.lpp_set_stream(streams[i]))
                call(i, i)
        for s in streams:
            hip("hipStreamSynchronize", s)
    finally:
        capi.check(lib.lpp_set_stream(None))
    for _ in range(20):
        for i in range(2):
            call(i, 2 + i)
    for i in range(2):
        assert np.array_equal(out[i].to_numpy(np.uint8), out[2 + i].to_numpy(np.uint8))
        assert np.array_equal(mass[i].to_numpy(np.uint8), mass[2 + i].to_numpy(np.uint8))
    for s in streams:
        hip("hipStreamDestroy", s)


@pytest.mark.parametrize("heads,kv,hs,room", [(32, 4, 64, 3000), (8, 2, 128, 7000)])
def test_one_workspace_for_all_calls(lib, heads, kv, hs, room):
    """Sized for the most rows a sequence and the whole room, given with its real size to calls of fewer rows and of a smaller cache; nothing behind it
    is written."""
    rng = np.random.default_rng(room)
    need = C.c_size_t()
    capi.check(lib.lpp_kv4_attention_workspace(Shape(1, 2, kv, room, hs), heads, 16, C.byref(need)))
    guard = 1 << 16
    work = DB.from_numpy(np.full(need.value // 4 + guard, np.nan, F))
    for n_q, positions in ((16, room), (3, room), (2, room), (1, room), (1, 2000), (5, 600), (2, 40)):
        cache = random_cache(rng, 1, 2, kv, positions, hs)
        dcache, q = DB.from_numpy(cache.buffer), rng.standard_normal((2, n_q, heads, hs)).astype(F)
        starts, mass = [positions - n_q, positions // 3], rng.random((1, 2, kv, positions)).astype(F)
        dq, dout, dst, dmass = DB.from_numpy(q), DB.from_numpy(np.full(q.size, 7.25, F)), ints(starts), DB.from_numpy(mass)
        capi.check(lib.lpp_kv4_attention(dout.ptr, dq.ptr, dcache.ptr, Shape(1, 2, kv, positions, hs), 0, heads, n_q, dst.ptr, dmass.ptr, work.ptr,
                                         need.value))
        check_attention(dout.to_numpy(F).reshape(q.shape), dmass.to_numpy(F).reshape(mass.shape), cache, 0, q, starts, mass)
    assert np.all(np.isnan(work.to_numpy(F, guard, need.value)))


def part_of(cache, seqs):
    """Some of a cache's sequences."""
    part = ko.Cache(cache.dims[0], len(seqs), *cache.dims[2:], cache.hs)
    for w in range(2):
        part.codes[w][:], part.scales[w][:] = cache.codes[w][:, seqs], cache.scales[w][:, seqs]
    return part


@pytest.mark.parametrize("seqs,heads,kv,hs,room,n_q", [(9, 16, 8, 128, 5000, 1), (9, 32, 4, 128, 3001, 5), (17, 8, 4, 64, 2500, 1)])
def test_many_heads_and_several_shares(lib, seqs, heads, kv, hs, room, n_q):
    """Four wavefronts to a share, positions enough for several, with and without the account, whose scores are kept (one tile of rows) or made again."""
    rng = np.random.default_rng(room)
    lengths = np.concatenate([[room, n_q, 0], rng.integers(room // 6, room, seqs - 3)])
    cache = random_cache(rng, 1, seqs, kv, room, hs)
    dcache, q = DB.from_numpy(cache.buffer), rng.standard_normal((seqs, n_q, heads, hs)).astype(F)
    mass, starts = rng.random((1, seqs, kv, room)).astype(F), lengths - n_q
    got, got_mass = attend(lib, dcache, cache, 0, q, starts, mass)
    check_attention(got, got_mass, cache, 0, q, starts, mass)
    assert np.array_equal(attend(lib, dcache, cache, 0, q, starts)[0], got)


def test_account_of_many_heads_from_kept_scores(lib):
    """So many sequences that a block of the account takes several rounds of 1024 positions: a sample of them."""
    rng = np.random.default_rng(21)
    seqs, heads, kv, hs, room = 128, 16, 8, 64, 1100
    cache = random_cache(rng, 1, seqs, kv, room, hs)
    q, mass = rng.standard_normal((seqs, 1, heads, hs)).astype(F), rng.random((1, seqs, kv, room)).astype(F)
    starts = rng.integers(0, room, seqs)
    starts[[0, 1, 50, 127]] = [room - 1, 1023, 1024, 1026]
    got, got_mass = attend(lib, DB.from_numpy(cache.buffer), cache, 0, q, starts, mass)
    some = [0, 1, 2, 3, 50, 90, 126, 127]
    check_attention(got[some], got_mass[:, some], part_of(cache, some), 0, q[some], starts[some], mass[:, some])
    for s in range(seqs):
        assert np.array_equal(got_mass[0, s, :, starts[s] + 1:], mass[0, s, :, starts[s] + 1:])
        added = got_mass[0, s].astype(np.float64).sum(-1) - mass[0, s].astype(np.float64).sum(-1)
        # (the weights of two heads; every position's total is below 4, so its rounding is 2^-23 at most, and its weights' errors are far below 2^-16)
        assert np.all(np.abs(added - 2) <= room * 2.0 ** -23 + 2 * 2.0 ** -16)


@pytest.mark.parametrize("heads,hs,room", [(4, 64, 5001), (4, 128, 8000)])
def test_account_made_again_for_several_rows_of_one_tile(lib, heads, hs, room):
    """Four rows of four heads, one tile, of more positions than whose scores are kept (16 rows: 4 bytes each of all positions and the partial results of a
    share for every 512 of them are more than those of 64 shares)."""
    assert 16 * room + -(-room // 512) * 16 * (hs + 2) > 64 * 16 * (hs + 2)
    rng = np.random.default_rng(room)
    lengths = [room - 1, 900, 4, 2]
    cache = random_cache(rng, 1, len(lengths), 1, room, hs)
    q, mass = rng.standard_normal((len(lengths), 4, heads, hs)).astype(F), rng.random((1, len(lengths), 1, room)).astype(F)
    starts = [n - 4 for n in lengths]
    got, got_mass = attend(lib, DB.from_numpy(cache.buffer), cache, 0, q, starts, mass)
    check_attention(got, got_mass, cache, 0, q, starts, mass)
