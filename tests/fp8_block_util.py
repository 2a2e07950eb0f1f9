"""The FP8 format with one scale per block of 128, restated in numpy from its definition: E4M3 decoding and rounding, the
block quantiser in the library's FP32 arithmetic, and the scaled product in float64."""
import numpy as np

BLOCK = 128
TOP = np.float32(448.0)
SMALLEST = np.float32(2.0 ** -126)


def decode_table():
    """Value of every E4M3 code: 1.mmm * 2^(e - 7), subnormals m * 2^-9, S.1111.111 = NaN, no infinities."""
    codes = np.arange(256)
    e, m = (codes >> 3) & 15, codes & 7
    value = np.where(e == 0, m * 2.0 ** -9, (1.0 + m / 8.0) * 2.0 ** (e - 7.0))
    value[(codes & 0x7F) == 0x7F] = np.nan
    return np.where(codes >= 128, -value, value)


TABLE = decode_table()


def decode(codes):
    return TABLE[np.asarray(codes)]


def round_e4m3(x):
    """The E4M3 value nearest to x, ties to the even code, saturating at 448 (float64 in and out; NaN stays)."""
    x = np.asarray(x, dtype=np.float64)
    size = np.minimum(np.abs(x), 448.0)
    exponent = np.floor(np.log2(np.maximum(size, 2.0 ** -6)))
    step = 2.0 ** (exponent - 3.0)
    return np.copysign(np.minimum(np.rint(size / step) * step, 448.0), x)


def half_step(q):
    """Largest distance of a value in E4M3's range from its rounding: half a step, 2^-4 of the value or half the
    subnormal step 2^-9."""
    return np.maximum(2.0 ** -4 * np.abs(q), 2.0 ** -10)


def blocks_of(cols):
    return (cols + BLOCK - 1) // BLOCK


def block_scales(y):
    """FP32 scales [blocks, rows] of FP32 y [rows, cols], in the library's arithmetic."""
    y = np.asarray(y, dtype=np.float32)
    scales = np.empty((blocks_of(y.shape[1]), y.shape[0]), dtype=np.float32)
    for b in range(scales.shape[0]):
        size = np.abs(y[:, b * BLOCK:(b + 1) * BLOCK])
        amax = np.where(np.isfinite(size), size, np.float32(0)).max(axis=1)
        scales[b] = np.where(amax == 0, np.float32(1), np.maximum(amax / TOP, SMALLEST))
    return scales


def per_column(scales, cols):
    """[blocks, rows] scales spread over [rows, cols]."""
    return np.repeat(scales.T, BLOCK, axis=1)[:, :cols]


def quantize(y):
    """(E4M3 values, scales) of FP32 y: what the codes of the block quantiser decode to, bit for bit."""
    y = np.asarray(y, dtype=np.float32)
    scales = block_scales(y)
    with np.errstate(over="ignore", invalid="ignore"):
        scaled = y * per_column(np.float32(1) / scales, y.shape[1])
    return round_e4m3(scaled), scales


def product(a_codes, sa, w_codes, sw):
    """(out, magnitude) in float64: the scaled product and the sum of its terms' magnitudes."""
    a = decode(a_codes) * per_column(sa.astype(np.float64), a_codes.shape[1])
    n, k = w_codes.shape
    w = decode(w_codes) * np.repeat(np.repeat(sw.astype(np.float64), BLOCK, axis=0)[:n], BLOCK, axis=1)[:, :k]
    return a @ w.T, np.abs(a) @ np.abs(w).T


def product_tolerance(want, magnitude, k):
    """Half a bf16 step of the result, and for the FP32 sums the classical bound of a sum of m terms, (m - 1) 2^-24 of the
    terms' magnitudes: at most 128 terms within a block, one per block after it, three roundings for the two scales and
    the product with the block's sum."""
    terms = min(k, BLOCK) + blocks_of(k) + 3
    return 2.0 ** -8 * np.abs(want) + terms * 2.0 ** -24 * (1.0 + 2.0 ** -8) * magnitude + 2.0 ** -133


def random_codes(rng, shape):
    """E4M3 codes of every size, no NaN."""
    codes = rng.integers(0, 256, size=shape, dtype=np.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x3C
    return codes


def operands(rng, tokens, n, k):
    """Codes of all sizes and scales over a few binades: (a, sa, w, sw)."""
    sa = np.exp2(rng.uniform(-9, -4, size=(blocks_of(k), tokens))).astype(np.float32)
    sw = np.exp2(rng.uniform(-12, -8, size=(blocks_of(n), blocks_of(k)))).astype(np.float32)
    return random_codes(rng, (tokens, k)), sa, random_codes(rng, (n, k)), sw
