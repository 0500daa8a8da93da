"""What section E of include/lpp.h computes, in 64 bits (numpy): the groups of the 4-bit cache, attention of rows over a
range of positions, and the choice of positions to keep.  Also how far a correct fp32 / binary16 kernel can be off."""
import numpy as np

GROUP = 32
F16, F32, F64 = np.float16, np.float32, np.float64
SHIFT = np.array([4 * (e // 2) + 16 * (e % 2) for e in range(8)], dtype=np.uint32)


def quantise(x):
    """(codes, scale, lowest) of rows [..., hs]: codes [..., hs / 32, 32], the others binary16 [..., hs / 32]."""
    x = np.asarray(x)
    g = x.astype(F32).reshape(*x.shape[:-1], -1, GROUP)
    bad = ~(np.abs(g) <= 32768).all(-1)
    g = np.where(bad[..., None], F32(0), g)
    low, high = g.min(-1), g.max(-1)
    scale = ((high - low) * (F32(1) / F32(15))).astype(F16)
    low = low.astype(F16)
    with np.errstate(divide="ignore", invalid="ignore"):
        t = np.rint((g.astype(F64) - low.astype(F64)[..., None]) / scale.astype(F64)[..., None])
    codes = np.where(scale[..., None] > 0, np.clip(np.nan_to_num(t), 0, 15), 0).astype(np.uint32)
    codes[bad] = 0
    return codes, np.where(bad, F16(0), scale), np.where(bad, F16(np.nan), low)


def stands_for(codes, scale, low):
    """binary16 [..., hs].  (The sum is exact in 64 bits, so this rounds once.)"""
    v = low.astype(F64)[..., None] + codes.astype(F64) * scale.astype(F64)[..., None]
    with np.errstate(over="ignore"):
        return v.astype(F16).reshape(*codes.shape[:-2], -1)


def rounded(x):
    return stands_for(*quantise(x))


class Cache:
    """One buffer as the library lays it out, filled and read on the host."""

    def __init__(self, n_layers, n_seqs, n_kv_heads, seq_len, head_size, fill=0):
        self.dims = (n_layers, n_seqs, n_kv_heads, seq_len)
        self.hs = head_size
        rows = int(np.prod(self.dims))
        self.buffer = np.full(rows * head_size * 5 // 4, fill, np.uint8)
        self.attach(self.buffer)

    def attach(self, buffer):
        rows = int(np.prod(self.dims))
        words = buffer.view(np.uint32)
        cut = np.split(words, [rows * self.hs // 8, rows * self.hs // 4, rows * self.hs // 4 + rows * self.hs // 32])
        self.buffer = buffer
        self.codes = [c.reshape(*self.dims, self.hs // 8) for c in cut[:2]]
        self.scales = [c.reshape(*self.dims, self.hs // GROUP) for c in cut[2:]]
        return self

    def put(self, which, layer, seq, pos, rows):
        """rows [n_kv_heads, hs] at one position."""
        codes, scale, low = quantise(rows)
        words = (codes.reshape(*codes.shape[:-2], -1, 8) << SHIFT).sum(-1, dtype=np.uint32)
        self.codes[which][layer, seq, :, pos] = words
        self.scales[which][layer, seq, :, pos] = scale.view(np.uint16).astype(np.uint32) | (low.view(np.uint16).astype(np.uint32) << 16)

    def values(self, which, layer=0):
        """binary16 [n_seqs, n_kv_heads, seq_len, hs]."""
        words, pair = self.codes[which][layer], self.scales[which][layer]
        codes = ((words[..., None] >> SHIFT) & 15).reshape(*words.shape[:-1], -1, GROUP)
        scale = (pair & 0xFFFF).astype(np.uint16).view(F16)
        low = (pair >> 16).astype(np.uint16).view(F16)
        with np.errstate(invalid="ignore"):
            return stands_for(codes, scale, low)


def attend(q, k, v, ends):
    """q [rows, heads, hs], k and v [kv_heads, positions, hs]; row j attends to the first ends[j] positions.  Returns (out [rows, heads, hs],
    weights [rows, heads, positions]) in 64 bits."""
    rows, heads, hs = q.shape
    kv_heads, n, _ = k.shape
    out, weights = np.zeros((rows, heads, hs)), np.zeros((rows, heads, n))
    for j in range(rows):
        e = ends[j]
        if e <= 0:
            continue
        for h in range(heads):
            g = h * kv_heads // heads
            s = k[g, :e].astype(F64) @ q[j, h].astype(F64) / np.sqrt(hs)
            w = np.exp(s - s.max())
            weights[j, h, :e] = w / w.sum()
            out[j, h] = weights[j, h, :e] @ v[g, :e].astype(F64)
    return out, weights


def score_error(q, k, ends):
    """[rows, heads]: how far any of a row's scores may be off, in fp32 with q as binary16 head and remainder.  A head and a remainder are
    within 2^-22 of the value, or 2^-25 where the remainder is a subnormal binary16; hs products are added in fp32, twice (heads, remainders);
    the scaled score is rounded twice more, once after its reference is taken off."""
    rows, heads, hs = q.shape
    kv_heads = k.shape[0]
    d = np.zeros((rows, heads))
    for j in range(rows):
        if ends[j] <= 0:
            continue
        for h in range(heads):
            a = np.abs(k[h * kv_heads // heads, :ends[j]].astype(F64))
            size = np.abs(q[j, h].astype(F64))
            worst = (a @ size).max()
            d[j, h] = (worst * (2.0 ** -22 + (2 * hs + 4) * 2.0 ** -24) + a.sum(-1).max() * 2.0 ** -25) / np.sqrt(hs)
    return d


def attend_tolerance(q, k, v, ends, binary16=False):
    """[rows, heads, hs]: a weight's relative error is twice the scores' (its own and that of the sum it is divided by), and 2^-20 for the
    exponential, the remainder's rounding (2^-22) and the quotient; the sums of n terms in fp32 add n 2^-24 at most, twice.
    binary16: the output is rounded (2^-11, or 2^-25 where it is subnormal), and there is room for weights of as many bits."""
    rows, heads, hs = q.shape
    kv_heads = k.shape[0]
    d = score_error(q, k, ends)
    tol = np.zeros((rows, heads, hs))
    out, weights = attend(q, k, v, ends)
    for j in range(rows):
        e = ends[j]
        if e <= 0:
            continue
        for h in range(heads):
            a = np.abs(v[h * kv_heads // heads, :e].astype(F64))
            part = weights[j, h, :e] @ a
            tol[j, h] = part * (2 * d[j, h] + 2.0 ** -20 + 2 * e * 2.0 ** -24)
            if binary16:
                # (of weights of 11 bits and a sum of unrounded ones; the kernels keep the remainders, and test_prompt_gpu.py has the bound for that)
                tol[j, h] += part * 2.0 ** -11 + a.sum(0) * 2.0 ** -25 * weights[j, h].max() + np.abs(out[j, h]) * 2.0 ** -11 + 2.0 ** -25
    return out, weights, tol


def keep_positions(mass, n, keep, recent):
    """Positions kept of the first n, ascending."""
    if n <= keep:
        return np.arange(n)
    others = np.asarray(mass[:n - recent], F32)
    order = sorted(range(n - recent), key=lambda i: (0 if np.isnan(others[i]) else 1, 0.0 if np.isnan(others[i]) else -float(others[i]), i))
    return np.sort(np.array(order[:keep - recent] + list(range(n - recent, n)), dtype=np.int64))
