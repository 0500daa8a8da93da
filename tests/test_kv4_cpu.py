"""Section E of include/lpp.h without a GPU: sizes, and every refusal (a call that is refused does no device work)."""
import ctypes as C

import numpy as np
import pytest

import kv4_oracle as ko
from lighterpp_amd import capi
from lighterpp_amd.capi import LppKv4Shape as Shape

P = 1 << 20  # an address that is never touched


@pytest.fixture(scope="module")
def lib():
    return capi.load()


def refused(lib, status, word):
    assert status == capi.LPP_ERR_INVALID_ARG
    assert word in lib.lpp_last_error(), lib.lpp_last_error()


def test_bytes(lib):
    n = C.c_size_t()
    for dims in [(1, 1, 1, 1, 64), (3, 2, 8, 100, 128), (32, 64, 8, 131072, 128)]:
        capi.check(lib.lpp_kv4_bytes(Shape(*dims), C.byref(n)))
        assert n.value == int(np.prod(dims, dtype=np.int64)) * 5 // 4
    assert ko.Cache(3, 2, 8, 100, 128).buffer.nbytes == 3 * 2 * 8 * 100 * 128 * 5 // 4


@pytest.mark.parametrize("dims", [(0, 1, 1, 1, 64), (1, 0, 1, 1, 64), (1, 1, 0, 1, 64), (1, 1, 1, 0, 64), (1, 1, 1, -5, 64), (1, 1, 1, 8, 48),
                                  (1, 1, 1, 8, 256), (1, 1, 1, (1 << 24) + 1, 64), (1 << 20, 1 << 20, 1, 8, 64)])
def test_shapes_refused(lib, dims):
    n = C.c_size_t()
    refused(lib, lib.lpp_kv4_bytes(Shape(*dims), C.byref(n)), b"lpp_kv4_bytes")
    refused(lib, lib.lpp_kv4_store(P, Shape(*dims), 0, P, P, 0, 1 << 20, None, 0, None), b"lpp_kv4_store")
    refused(lib, lib.lpp_kv4_load(P, P, P, Shape(*dims), 0, 0, 0), b"lpp_kv4_load")
    refused(lib, lib.lpp_kv4_attention(P, 2 * P, 3 * P, Shape(*dims), 0, 1, 1, P, None, P, 1 << 30), b"lpp_kv4_attention")
    refused(lib, lib.lpp_kv4_evict(P, Shape(*dims), 0, P, P, P, 3 * P, Shape(*dims), 0, P, P, 1, 0), b"lpp_kv4_evict")
    refused(lib, lib.lpp_kv4_bytes(None, C.byref(n)), b"null shape")
    refused(lib, lib.lpp_kv4_bytes(Shape(1, 1, 1, 1, 64), None), b"null output")


def test_store_refused(lib):
    s = Shape(2, 3, 2, 10, 64)
    call = lambda cache=P, layer=0, k=2 * P, v=3 * P, type=0, stride=128, offsets=None, n=6, starts=None: \
        lib.lpp_kv4_store(cache, s, layer, k, v, type, stride, offsets, n, starts)  # noqa: E731
    assert call(n=0) == capi.LPP_OK and call(n=0, k=None, v=None) == capi.LPP_OK
    refused(lib, call(cache=None), b"null cache")
    refused(lib, call(cache=P + 4), b"aligned")
    refused(lib, call(layer=2), b"layer")
    refused(lib, call(layer=-1), b"layer")
    refused(lib, call(k=None), b"null pointer")
    refused(lib, call(v=None), b"null pointer")
    refused(lib, call(type=2), b"type")
    refused(lib, call(n=-1), b"n_tokens")
    refused(lib, call(n=7), b"n_tokens")
    refused(lib, call(stride=127), b"kv_stride")
    refused(lib, call(stride=130), b"16 bytes")
    refused(lib, call(type=1, stride=132), b"16 bytes")
    refused(lib, call(k=4 * P + 8), b"16 bytes")
    refused(lib, call(v=P + 1024), b"overlap")


def test_load_refused(lib):
    s = Shape(1, 1, 2, 10, 64)
    call = lambda k=P, v=2 * P, cache=3 * P, layer=0, first=0, count=10: lib.lpp_kv4_load(k, v, cache, s, layer, first, count)  # noqa: E731
    assert call(count=0) == capi.LPP_OK and call(first=10, count=0) == capi.LPP_OK
    for bad in [dict(first=-1), dict(count=-1), dict(count=11), dict(first=1), dict(first=11, count=0), dict(first=2 ** 31 - 1, count=2 ** 31 - 1)]:
        refused(lib, call(**bad), b"positions")
    refused(lib, call(k=None), b"null pointer")
    refused(lib, call(v=None), b"null pointer")
    refused(lib, call(v=2 * P + 2), b"16 bytes")
    refused(lib, call(k=3 * P + 16), b"overlap")
    refused(lib, call(k=2 * P), b"overlap")
    refused(lib, call(cache=None), b"null cache")


def test_attention_refused(lib):
    s = Shape(1, 3, 2, 10, 64)
    need = C.c_size_t()
    capi.check(lib.lpp_kv4_attention_workspace(s, 8, 2, C.byref(need)))
    assert need.value > 0
    call = lambda out=P, q=2 * P, cache=3 * P, layer=0, heads=8, n_q=2, starts=P, work=4 * P, size=need.value, mass=None: \
        lib.lpp_kv4_attention(out, q, cache, s, layer, heads, n_q, starts, mass, work, size)  # noqa: E731
    refused(lib, call(out=None), b"null pointer")
    refused(lib, call(q=None), b"null pointer")
    refused(lib, call(starts=None), b"null pointer")
    refused(lib, call(work=None), b"null pointer")
    refused(lib, call(cache=None), b"null cache")
    refused(lib, call(layer=1), b"layer")
    refused(lib, call(heads=7), b"n_heads")
    refused(lib, call(heads=0), b"n_heads")
    refused(lib, call(heads=34), b"query heads")
    refused(lib, call(n_q=0), b"n_q")
    refused(lib, call(n_q=11), b"n_q")
    refused(lib, call(size=need.value - 1), b"workspace")
    refused(lib, call(out=2 * P + 16), b"overlap")
    refused(lib, call(work=2 * P + 64), b"workspace")
    refused(lib, call(work=P - 64), b"workspace")
    refused(lib, call(work=3 * P + 64), b"workspace")
    for base in (P, 2 * P, 3 * P, 4 * P):
        refused(lib, call(mass=base + 64), b"d_mass overlaps")
    for name in ("out", "q", "work"):
        refused(lib, call(**{name: 5 * P + 4}), b"16 bytes")
    refused(lib, lib.lpp_kv4_attention_workspace(s, 8, 2, None), b"null output")
    refused(lib, lib.lpp_kv4_attention_workspace(s, 5, 2, C.byref(need)), b"n_heads")


def test_evict_refused(lib):
    src, dst = Shape(1, 3, 2, 100, 64), Shape(2, 3, 2, 20, 64)
    call = lambda cache=P, to=dst, to_layer=0, to_mass=2 * P, to_len=3 * P, kept=4 * P, other=5 * P, layer=0, mass=6 * P, length=7 * P, keep=20, recent=5: \
        lib.lpp_kv4_evict(cache, to, to_layer, to_mass, to_len, kept, other, src, layer, mass, length, keep, recent)  # noqa: E731
    for name in ("to_mass", "to_len", "kept", "mass", "length"):
        refused(lib, call(**{name: None}), b"null pointer")
    for name in ("cache", "other"):
        refused(lib, call(**{name: None}), b"null cache")
        refused(lib, call(**{name: 8 * P + 8}), b"aligned")
    refused(lib, call(to_layer=2), b"layer")
    refused(lib, call(layer=1), b"layer")
    refused(lib, call(keep=21), b"keep")
    refused(lib, call(keep=0, recent=0), b"keep")
    refused(lib, call(keep=5, recent=6), b"keep")
    refused(lib, call(recent=-1), b"keep")
    for other in (Shape(1, 2, 2, 20, 64), Shape(1, 3, 1, 20, 64), Shape(1, 3, 2, 20, 128)):
        refused(lib, call(to=other), b"caches are of")
    refused(lib, call(cache=5 * P + 64), b"overlap")
    refused(lib, call(to_mass=6 * P + 4), b"overlap")
    refused(lib, call(to_len=7 * P), b"overlap")


def test_prompt_refused(lib):
    call = lambda out=P, q=2 * P, k=3 * P, v=4 * P, type=0, offsets=5 * P, seqs=2, n=8, heads=4, kv=2, hs=64, sq=256, sk=128, so=256: \
        lib.lpp_prompt_attention(out, q, k, v, type, offsets, seqs, n, heads, kv, hs, sq, sk, so)  # noqa: E731
    assert call(n=0) == capi.LPP_OK
    for name in ("out", "q", "k", "v"):
        refused(lib, call(**{name: None}), b"null pointer")
        refused(lib, call(**{name: 6 * P + 8}), b"16 bytes")
    refused(lib, call(type=3), b"type")
    refused(lib, call(heads=5), b"n_heads")
    refused(lib, call(kv=0), b"n_heads")
    refused(lib, call(heads=34, sq=34 * 64, so=34 * 64), b"query heads")
    refused(lib, call(hs=48), b"head_size")
    refused(lib, call(n=-1), b"n_tokens")
    refused(lib, call(seqs=0), b"n_seqs")
    refused(lib, call(offsets=None), b"n_seqs")
    for name in ("sq", "so"):
        refused(lib, call(**{name: 255}), b"strides")
        refused(lib, call(**{name: 258}), b"16 bytes")
    refused(lib, call(sk=127), b"strides")
    refused(lib, call(sk=132), b"16 bytes")
    refused(lib, call(sk=(1 << 24) + 8), b"kv_stride")
    refused(lib, call(out=2 * P + 1024), b"overlap")
    refused(lib, call(out=4 * P - 16), b"overlap")


def test_oracle_groups():
    """The oracle's own rules: ends of the range, constant groups, overflow."""
    x = np.zeros((1, 64), np.float32)
    x[0, :32] = np.linspace(-1, 2, 32)
    x[0, 40] = 3.0
    codes, scale, low = ko.quantise(x)
    assert codes[0, 0, 0] == 0 and codes[0, 0, 31] == 15 and codes[0, 1].max() == 15 and codes[0, 1, 0] == 0
    v = ko.rounded(x).astype(np.float64)
    assert np.abs(v - x).max() <= 0.5 * 0.2 * (1 + 2.0 ** -10) + 2 * 2.0 ** -10
    assert np.array_equal(ko.rounded(np.full((1, 32), 0.3, np.float32)), np.full((1, 32), 0.3, np.float16))
    for bad in (np.inf, -np.inf, np.nan, 32769.0):
        y = x.copy()
        y[0, 3] = bad
        assert np.isnan(ko.rounded(y)[0, :32]).all() and not np.isnan(ko.rounded(y)[0, 32:]).any()
    assert not np.isnan(ko.rounded(np.array([[32768.0, -32768.0] * 16], np.float32))).any()


def test_a_workspace_of_the_largest_call_serves_smaller_ones(lib):
    """Bytes do not shrink with sequences, positions, query heads or rows, and stay within partial results of 64 shares of 16 rows."""
    def need(seqs, kv, room, hs, shared, n_q):
        n = C.c_size_t()
        capi.check(lib.lpp_kv4_attention_workspace(Shape(1, seqs, kv, room, hs), kv * shared, n_q, C.byref(n)))
        tiles = -(-n_q // (16 // shared))
        assert n.value <= seqs * kv * tiles * 64 * 16 * (hs + 2) * 4
        return n.value

    rooms = [1, 40, 512, 513, 2000, 3000, 3680, 3681, 6624, 6625, 14000, 14912, 14913, 16000, 27000, 40000, 200000, 1 << 24]
    rows = [1, 2, 3, 4, 5, 8, 15, 16, 17, 33, 64, 100, 256, 1000, 5000]
    for hs in (64, 128):
        for kv in (1, 4, 8):
            for seqs in (1, 4, 33, 300):
                table = np.array([[[need(seqs, kv, room, hs, shared, n_q) for n_q in rows if n_q <= room] + [0] * sum(n_q > room for n_q in rows)
                                   for room in rooms] for shared in range(1, 17)])
                there = table > 0
                assert np.all(np.diff(table, axis=0)[there[1:]] >= 0), "query heads"
                assert np.all(np.diff(table, axis=1)[there[:, :-1]] >= 0), "positions"
                assert np.all(np.diff(table, axis=2)[there[:, :, 1:]] >= 0), "rows"
                if seqs > 1:
                    assert np.all(table >= before), "sequences"
                before = table


def test_attention_too_large_for_a_launch_is_refused_before_any(lib):
    """Positions of so many KV heads that the account's blocks pass a launch: nothing is launched, the attention included."""
    far = [(i + 1) << 40 for i in range(6)]
    shape, need = Shape(1, 128, 8, 1 << 20, 64), C.c_size_t()
    capi.check(lib.lpp_kv4_attention_workspace(shape, 128, 2, C.byref(need)))
    refused(lib, lib.lpp_kv4_attention(far[0], far[1], far[2], shape, 0, 128, 2, far[3], far[4], far[5], need.value), b"too many for a launch")


def test_evict_refuses_every_overlap(lib):
    """Each of the four buffers that are written with each other and with each of the three that are read."""
    src, dst = Shape(2, 3, 2, 100, 64), Shape(2, 3, 2, 20, 64)
    sizes = [2 * 3 * 2 * 20 * 80, 2 * 3 * 2 * 20 * 4, 3 * 4, 3 * 2 * 20 * 4, 2 * 3 * 2 * 100 * 80, 2 * 3 * 2 * 100 * 4, 3 * 4]
    for a in range(4):
        for b in range(7):
            if a == b:
                continue
            at = [(i + 1) * P for i in range(7)]
            at[a] = (at[b] + sizes[b] - 1) // 16 * 16  # begins in b's last bytes
            refused(lib, lib.lpp_kv4_evict(at[0], dst, 1, at[1], at[2], at[3], at[4], src, 1, at[5], at[6], 20, 5), b"overlaps")


def test_outputs_over_the_cache_or_the_ints_are_refused(lib):
    s, need = Shape(1, 3, 2, 10, 64), C.c_size_t()
    capi.check(lib.lpp_kv4_attention_workspace(s, 8, 2, C.byref(need)))
    attend = lambda out=P, cache=3 * P, starts=6 * P, mass=5 * P: \
        lib.lpp_kv4_attention(out, 2 * P, cache, s, 0, 8, 2, starts, mass, 4 * P, need.value)  # noqa: E731
    refused(lib, attend(out=3 * P + 4784), b"d_out overlaps the cache")
    for base in (P, 4 * P, 5 * P):
        refused(lib, attend(starts=base + 8), b"d_starts overlaps")
    refused(lib, attend(starts=P - 8), b"d_starts overlaps")
    store = lambda offsets=None, starts=None: lib.lpp_kv4_store(P, s, 0, 2 * P, 3 * P, 0, 128, offsets, 6, starts)  # noqa: E731
    refused(lib, store(offsets=P - 12), b"overlaps the cache")
    refused(lib, store(starts=P + 4796), b"overlaps the cache")
    refused(lib, lib.lpp_prompt_attention(P, 2 * P, 3 * P, 4 * P, 0, P - 8, 2, 8, 4, 2, 64, 256, 128, 256), b"overlaps")


def test_store_too_large_for_a_launch(lib):
    s, far = Shape(1, 1, 1, 1 << 24, 64), [(i + 1) << 40 for i in range(3)]
    for n in (1 << 26, (1 << 26) - 3, 2 ** 31 - 1):
        refused(lib, lib.lpp_kv4_store(far[0], s, 0, far[1], far[2], capi.F16, 64, None, n, None), b"too many for a launch")


def test_scale_against_the_quotient_in_64_bits():
    """The format's scale, the range times the fp32 number 1/15, is the fifteenth of the range to its own rounding (2^-11, or 2^-25 where it is subnormal) and three
    of fp32: the difference, 1/15, the product.  Every value stands for one within half a step of it."""
    rng = np.random.default_rng(13)
    x = (rng.standard_normal((20000, 32)) * np.exp(3 * rng.standard_normal((20000, 1)))).astype(np.float32)
    x[:2000] *= np.float32(1e-6)
    x = np.clip(x, -32768, 32768)
    _, scale, low = ko.quantise(x)
    g = x.astype(np.float64)
    span = g.max(-1) - g.min(-1)
    assert np.all(np.abs(scale[:, 0].astype(np.float64) - span / 15) <= span / 15 * (2.0 ** -11 + 3.01 * 2.0 ** -24) + 2.0 ** -25)
    got = ko.rounded(x).astype(np.float64)
    # half a step, fifteen times the scale's rounding, and the roundings of lowest and value
    bound = span / 30 + span * 2.0 ** -11 * 1.01 + 2 * np.abs(g).max(-1) * 2.0 ** -11 * 1.01 + 17 * 2.0 ** -25
    assert np.all(np.abs(got - g) <= bound[:, None])
