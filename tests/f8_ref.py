"""8-bit operands in numpy, from their definition (OCP e4m3: four bits of
exponent with a bias of 7, three of mantissa, 448 the largest, 0x7f and 0xff
NaN), and the products of them in 64 bits."""
import numpy as np

import herbert_hip as hb

U = 2.0 ** -23  # an f32 operation's rounding, a whole step: MFMA sums may truncate
TINY = 2.0 ** -100


def _table():
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * np.exp2(e - 10.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b >> 7, -v, v)


VALUES = _table()
_POSITIVE = VALUES[:127]


def encode(v):
    """The codes nearest to v (|v| <= 464), ties to the even code; NaN 0x7f."""
    v = np.asarray(v, np.float64)
    a = np.abs(v)
    hi = np.clip(np.searchsorted(_POSITIVE, np.where(np.isnan(a), 0, a)), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(a >= 448, 126, code) | (np.signbit(v) << 7)
    return np.where(np.isnan(v), 0x7F, code).astype(np.uint8)


def blocks(n):
    return -(-n // 128)


def _groups(x, axis):
    """f64 values padded with zeros to whole groups of 128 along `axis`."""
    pad = [(0, 0)] * x.ndim
    pad[axis] = (0, -x.shape[axis] % 128)
    return np.pad(x, pad)


def f64(bits):
    return hb.bf16_to_f32(bits).astype(np.float64)


def _codes_of(v, a):
    """Codes of 448 v / a, a the sizes that f32 holds; a NaN or infinite a gives scales that are not finite."""
    with np.errstate(invalid="ignore"):
        q = np.where(np.isfinite(a), 448.0 * v / np.where(np.isfinite(a), a, 1.0), np.where(np.isfinite(v), 0.0, np.nan))
        q = np.where(np.isnan(a), np.nan, q)
    return encode(q), (a / 448.0).astype(np.float32)


def _largest(v, axis):
    with np.errstate(invalid="ignore"):
        a = np.abs(v)
    top = np.where(np.isnan(a).any(axis=axis, keepdims=True), np.nan, np.max(np.where(np.isnan(a), 0, a), axis=axis, keepdims=True))
    return np.maximum(top, TINY)  # NaN stays


def quantize_rows(x):
    """(codes [m][k], scales f32 [m][blocks]) of bf16 bits."""
    m, k = x.shape
    v = _groups(f64(x), 1).reshape(m, -1, 128)
    c, s = _codes_of(v, _largest(v, 2))
    return c.reshape(m, -1)[:, :k], s[:, :, 0]


def quantize(w):
    """(codes [n][k], scales f32 [blocks][blocks]) of bf16 bits."""
    n, k = w.shape
    v = _groups(_groups(f64(w), 0), 1).reshape(blocks(n), 128, blocks(k), 128)
    c, s = _codes_of(v, _largest(v, (1, 3)))
    return c.reshape(blocks(n) * 128, -1)[:n, :k], s[:, 0, :, 0]


def row_values(codes, scales):
    return VALUES[codes] * np.repeat(scales.astype(np.float64), 128, 1)[:, :codes.shape[1]]


def values(codes, scales):
    s = np.repeat(np.repeat(scales.astype(np.float64), 128, 0)[:codes.shape[0]], 128, 1)[:, :codes.shape[1]]
    return VALUES[codes] * s


def pack_rows(codes, scales):
    m, k = codes.shape
    out = np.zeros((m, hb.f8_row_bytes(k)), np.uint8)
    out[:, :k] = codes
    out[:, k:k + 4 * scales.shape[1]] = np.ascontiguousarray(scales, np.float32).view(np.uint8)
    return out


def unpack_rows(raw, m, k):
    raw = raw.reshape(m, hb.f8_row_bytes(k))
    return raw[:, :k], np.ascontiguousarray(raw[:, k:k + 4 * blocks(k)]).view(np.float32)


def pack(codes, scales):
    n, k = codes.shape
    out = np.zeros(hb.f8_bytes(k, n), np.uint8)
    out[:n * k] = codes.reshape(-1)
    out[n * k:n * k + 4 * scales.size] = np.ascontiguousarray(scales, np.float32).view(np.uint8).reshape(-1)
    return out


def random_weights(rng, n, k):
    """Codes of normal weights and scales of either size."""
    codes = encode(np.clip(rng.normal(0, 96, (n, k)), -448, 448))
    return codes, rng.uniform(1e-4, 3e-4, (blocks(n), blocks(k))).astype(np.float32)


def exact_weights(rng, n, k):
    """Codes of whole numbers up to 8 under scales of powers of two."""
    return encode(rng.integers(-8, 9, (n, k))), np.exp2(rng.integers(-2, 2, (blocks(n), blocks(k)))).astype(np.float32)


def wide_weights(rng, n, k):
    """The same under scales of 1, four of each 128 in a row +-256: beside x's 448
    the products of a group span 17 bits, and every sum over 1152 is whole and
    below 2^23."""
    w = rng.integers(-8, 9, (n, k))
    for b in range(blocks(k)):
        for i in range(n):
            at = rng.choice(np.arange(128 * b, min(128 * (b + 1), k)), 4, replace=False)
            w[i, at] = rng.choice([-256, 256], 4)
    return encode(w), np.ones((blocks(n), blocks(k)), np.float32)


def exact_x(rng, m, k, powers=(-2, 2)):
    """bf16 bits of whole multiples of a power of two, each group's largest 448
    times it, so that its codes are the whole numbers and its scale the power."""
    x = rng.integers(-8, 9, (m, k)).astype(np.float64)
    for b in range(blocks(k)):
        end = min(128 * (b + 1), k)
        x[np.arange(m), rng.integers(128 * b, end, m)] = rng.choice([-448, 448], m)
        x[:, 128 * b:end] *= np.exp2(rng.integers(*powers, m))[:, None]
    return hb.f32_to_bf16(x.astype(np.float32))


def sum_bound(xv, wv):
    """What the f32 sums may be off by, [m][n]: within a block at most two
    roundings a product; then a product of scales, one with the sum and an
    addition a block, and an addition a part of K (at most 16)."""
    k = xv.shape[1]
    return (2 * 128 + 3 + blocks(k) + 16) * U * (np.abs(xv) @ np.abs(wv).T)


def mfma_bound(xv, wv):
    """The same for the GEMM's outputs of two bytes and its SwiGLU, whose f8 MFMA
    adds products in eights along k, each cut at 2^-13 of the power of two that
    the largest of its eight reaches: seven of them lose less than that (one is
    the largest and loses nothing)."""
    eights = [np.abs(t).reshape(len(t), -1, 8).max(2) for t in (xv, wv)]
    return sum_bound(xv, wv) + 7 * 2.0 ** -13 * (eights[0] @ eights[1].T)


def silu(g):
    return g / (1 + np.exp(-g))


def swiglu_bound(g, u, eg, eu):
    """|silu(g) u| off by what its f32 sums are off by (|silu'| <= 1.1), 16
    roundings of the arithmetic itself, and the exponent: -log2(e) g takes one
    rounding beside the constant's own, half a step each, which moves e^-g, and
    the sigmoid by no more, by 1.5 |g| 2^-24 of itself."""
    return 1.1 * eg * (np.abs(u) + eu) + np.abs(silu(g)) * eu + (16 + np.abs(g)) * U * np.abs(silu(g) * u)


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
