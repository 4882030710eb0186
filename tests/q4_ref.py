"""4-bit weights in numpy, from their definition: a row's elements in groups
along K, element = (q - 8) * s with q of 0..15 and the group's bf16 scale s."""
import numpy as np

import herbert_hip as hb

U = 2.0 ** -23  # an f32 operation's rounding, a whole step: MFMA sums may truncate


def values(codes, scales, group):
    """The weights in 64 bits: codes [n][k] of 0..15, scales [n][groups] bf16 bits."""
    s = hb.bf16_to_f32(scales).astype(np.float64)
    return (codes.astype(np.float64) - 8) * np.repeat(s, group, axis=1)[:, :codes.shape[1]]


def nibbles(codes):
    """Codes [n][k] as bytes [n][k / 2], the even element in the low half."""
    return (codes[:, 0::2] | codes[:, 1::2] << 4).astype(np.uint8)


def quantize(w, group):
    """(codes, scales) of bf16 bits w [n][k]: s = bf16(the group's element of
    largest size, the positive one of two, / -8), q = round(w / s) within
    -8..7, ties to even; a group with a NaN or an infinity stands for NaN."""
    n, k = w.shape
    groups = -(-k // group)
    v = np.zeros((n, groups * group))
    v[:, :k] = hb.bf16_to_f32(w)
    v = v.reshape(n, groups, group)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[..., None], 0.0, v)
    hi, lo = v.max(-1), v.min(-1)
    far = np.where(hi >= -lo, hi, lo)
    scales = hb.f32_to_bf16((far / -8).astype(np.float32))
    s = hb.bf16_to_f32(scales).astype(np.float64)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(s == 0, 0, np.clip(np.rint(v / s), -8, 7)) + 8
    scales = np.where(bad, np.uint16(0x7FC0), scales).astype(np.uint16)
    return q.reshape(n, -1)[:, :k].astype(np.uint8), scales


def random_codes(rng, n, k, group):
    codes = np.clip(np.rint(rng.normal(8, 3.2, (n, k))), 0, 15).astype(np.uint8)
    s = rng.uniform(0.004, 0.009, (n, -(-k // group))) * rng.choice([-1, 1], (n, -(-k // group)))
    return codes, hb.f32_to_bf16(s.astype(np.float32))


def exact_codes(rng, n, k, group):
    """Any codes under scales that are powers of two: with small whole x every
    sum is exact in f32, whatever its order."""
    codes = rng.integers(0, 16, (n, k)).astype(np.uint8)
    s = np.exp2(rng.integers(-2, 3, (n, -(-k // group)))) * rng.choice([-1, 1], (n, -(-k // group)))
    return codes, hb.f32_to_bf16(s.astype(np.float32))


def pack(gpu, codes, scales, k, n, group, count=1):
    """A buffer with the packed matrices (codes [count * n][k])."""
    c, s = gpu.alloc_with(nibbles(codes)), gpu.alloc_with(scales)
    w = gpu.alloc(count * hb.q4_bytes(k, n, group))
    gpu.launch(gpu.pipeline(hb.q4_pack(k, n, group)), [hb.r(c), hb.r(s), hb.r(w)], count)
    gpu.sync()
    gpu.free(c)
    gpu.free(s)
    return w


def sum_bound(x, codes, scales, group):
    """What the f32 sums of matvec_q4 may be off by, [m][n].  A group's sum of
    (16 + q) x over one of -24 x takes at most two roundings a product, of
    partial sums no larger than 55 sum |x|; then a product and an addition a
    group, and an addition a part of K (at most 16)."""
    k = codes.shape[1]
    s = np.abs(np.repeat(hb.bf16_to_f32(scales).astype(np.float64), group, axis=1)[:, :k])
    a = np.abs(x).astype(np.float64) @ (55 * s).T
    return (2 * group + 2 * -(-k // group) + 16) * U * a


def silu(g):
    return g / (1 + np.exp(-g))


def swiglu_bound(g, u, eg, eu):
    """|silu(g) u| off by what its f32 sums are off by (|silu'| <= 1.1), and 16
    roundings of the arithmetic itself."""
    return 1.1 * eg * (np.abs(u) + eu) + np.abs(silu(g)) * eu + 16 * U * np.abs(silu(g) * u)


HALF_BF16 = 2.0 ** -8  # one rounding to bf16, relative to the value


def close(got, want, bound, what):
    """got (bf16 bits or f32) within `bound` of want, and one rounding if bf16."""
    if got.dtype == np.uint16:
        got = hb.bf16_to_f32(got)
        bound = bound + HALF_BF16 * (np.abs(want) + bound) + 2.0 ** -134
    off = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all(), what
    worst = float((off - bound).max()) if off.size else 0.0
    assert (off <= bound).all(), "%s: %g over, off %g at %s" % (what, worst, off.max(), np.unravel_index((off - bound).argmax(), off.shape))
