"""GPU tests of the FP8 operators with a scale per block of 128, through the C ABI, against their definition in 64 bits
(tests/fp8_block_util.py): sizes around whole blocks and tiles, blocks of zeros, subnormals, NaN and infinities, strides,
streams, captured graphs, and the operators in a row as a layer uses them."""
import importlib
import os
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

from oracle import oracle as orc
from tests import fixtures as fx
from tests import fp8_block_util as f8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from tests import gpu_util

    orc.build()
    gpu_util.capi.load()
    return gpu_util


def bf16_values(bits):
    return orc.bf16_decode(np.asarray(bits)).astype(np.float32)


def rows_with_extremes(rng, rows, cols):
    """Normal rows, and in the first blocks what a quantiser can get wrong."""
    x = bf16_values(fx.normal_bf16(rng, (rows, cols)))
    special = [np.zeros(16), np.full(16, np.nan), np.full(16, np.inf), np.r_[np.full(8, -np.inf), np.full(8, 3.0)],
               np.full(16, 1e-40), np.r_[np.full(15, 1e-38), np.nan], np.full(16, 3.3e38), np.r_[np.zeros(15), 1e-45],
               np.r_[np.full(15, -1.0), -448.0]]
    for i, block in enumerate(special):
        row, at = i % rows, (i // rows) * f8.BLOCK
        if at < cols:
            width = min(f8.BLOCK, cols - at)
            x[row, at:at + width] = np.tile(block, 8)[:width]
    return orc.bf16_encode(x.astype(np.float32))


def assert_codes(got_codes, got_scales, y, relative, what=""):
    """Codes and scales of a result y known in float64, when the kernel's own y is within `relative` of it: a scale moves
    by that much and its one rounding, a code by half a step more."""
    want = f8.block_scales(y.astype(np.float32)).astype(np.float64)
    assert np.all(np.abs(got_scales - want) <= (relative + 2.0 ** -22) * want), what
    q = y / f8.per_column(got_scales.astype(np.float64), y.shape[1])
    got = f8.decode(got_codes)
    assert np.array_equal(np.isnan(got), np.isnan(y)), what
    fine = np.isfinite(y)
    # (2^-22: the rounding of 1 / scale and of the product; 448 (1 + relative) saturates to 448)
    slack = f8.half_step(q[fine]) + (relative + 2.0 ** -22) * np.abs(q[fine])
    worst = np.max(np.abs(got[fine] - q[fine]) - slack) if fine.any() else 0.0
    assert worst <= 0, f"{what}: a code is {worst} past half a step"


# ---------------------------------------------------------------------------------------------------- quantiser


@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 128), (1, 144), (3, 112), (9, 272), (5, 2048), (2, 2064), (300, 640),
                                       (1, 17408), (700, 6144)])
def test_quantize_is_bit_exact(g, rows, cols):
    rng = np.random.default_rng([rows, cols, 7])
    x = rows_with_extremes(rng, rows, cols)
    codes, scales = g.empty_like_dev((rows, cols), dtype=np.uint8), g.empty_like_dev((f8.blocks_of(cols), rows), dtype=np.float32)
    g.capi.check("q3x_b200_fp8_block_quantize", g.Dev(x), rows, cols, codes, scales, None)
    g.sync()
    want, want_scales = f8.quantize(bf16_values(x))
    assert np.array_equal(scales.get(), want_scales)
    assert np.array_equal(f8.decode(codes.get()), want, equal_nan=True)
    assert codes.guards_intact() and scales.guards_intact()


def test_quantize_scales_of_every_bf16_amax(g):
    """One block per positive finite bf16 value, subnormals included: its scale is fl(amax / 448), its codes are exact."""
    amax = np.arange(1, 0x7F80, dtype=np.uint16)
    x = np.zeros((amax.size, f8.BLOCK), dtype=np.uint16)
    x[:, 77] = amax | 0x8000
    x[:, 5] = np.maximum(amax, 0x100) - 0x80  # half of it
    codes, scales = g.empty_like_dev(x.shape, dtype=np.uint8), g.empty_like_dev((1, amax.size), dtype=np.float32)
    g.capi.check("q3x_b200_fp8_block_quantize", g.Dev(x), amax.size, f8.BLOCK, codes, scales, None)
    g.sync()
    want, want_scales = f8.quantize(bf16_values(x))
    assert np.array_equal(scales.get(), want_scales)
    assert np.array_equal(f8.decode(codes.get()), want)


# ---------------------------------------------------------------------------------------------------- residual + norm


@pytest.mark.parametrize("rows,cols,with_normalized", [(1, 16, True), (1, 5120, False), (3, 144, True), (37, 2064, True),
                                                       (5, 8192, False), (3, 8208, True), (2, 16384, False), (2, 32768, True),
                                                       (260, 5120, True)])
def test_residual_norm(g, rows, cols, with_normalized):
    rng = np.random.default_rng([rows, cols, 11])
    left, right = fx.normal_bf16(rng, (rows, cols)), fx.normal_bf16(rng, (rows, cols))
    weight = orc.bf16_encode((0.2 * rng.standard_normal(cols)).astype(np.float32))
    residual, normalized = g.empty_like_dev((rows, cols)), g.empty_like_dev((rows, cols))
    codes, scales = g.empty_like_dev((rows, cols), dtype=np.uint8), g.empty_like_dev((f8.blocks_of(cols), rows), dtype=np.float32)
    g.capi.check("q3x_b200_residual_add_rms_norm_fp8_block", g.Dev(left), g.Dev(right), g.Dev(weight), rows, cols, 1e-6, residual,
                 normalized if with_normalized else None, codes, scales, None)
    g.sync()
    want_residual = orc.bf16_encode(bf16_values(left) + bf16_values(right))
    g.assert_bits_equal(residual.get(), want_residual, "residual")
    r = bf16_values(want_residual).astype(np.float64)
    y = r / np.sqrt((r * r).mean(axis=1, keepdims=True) + np.float64(np.float32(1e-6))) * (1.0 + bf16_values(weight).astype(np.float64))
    # the FP32 y: at most 64 squares in a row and ten levels of a tree (half their error through the root), the
    # reciprocal root's 2^-22, and three roundings -- below 2^-18
    assert_codes(codes.get(), scales.get(), y, 2.0 ** -18, f"{rows} x {cols}")
    if with_normalized:
        # half a bf16 step and the FP32 error
        got = bf16_values(normalized.get()).astype(np.float64)
        assert np.all(np.abs(got - y) <= (2.0 ** -8 + 2.0 ** -18) * np.abs(y))
    for d in (residual, normalized, codes, scales):
        assert d.guards_intact()


def test_residual_norm_in_place_of_right_and_odd_rows(g):
    """normalized_out may be exactly `right`; a row with a NaN and one of zeros stay their own affair."""
    rng = np.random.default_rng(13)
    rows, cols = 4, 640
    left, right = fx.normal_bf16(rng, (rows, cols)), fx.normal_bf16(rng, (rows, cols))
    left[1, 5] = 0x7FC0
    left[2], right[2] = 0, 0
    left[3, 130] = 0x7F80
    weight = fx.normal_bf16(rng, (cols,))
    d_right = g.Dev(right)
    residual, apart = g.empty_like_dev((rows, cols)), g.empty_like_dev((rows, cols))
    blocks = f8.blocks_of(cols)
    out = [(g.empty_like_dev((rows, cols), dtype=np.uint8), g.empty_like_dev((blocks, rows), dtype=np.float32)) for _ in range(2)]
    args = (weight_d := g.Dev(weight), rows, cols, 1e-6, residual)
    g.capi.check("q3x_b200_residual_add_rms_norm_fp8_block", g.Dev(left), d_right, *args, apart, *out[0], None)
    g.capi.check("q3x_b200_residual_add_rms_norm_fp8_block", g.Dev(left), d_right, *args, d_right, *out[1], None)
    g.sync()
    assert weight_d is not None
    g.assert_bits_equal(d_right.get(), apart.get(), "normalized in place")
    for a, b in zip(out[0], out[1]):
        assert np.array_equal(a.get(), b.get())
    values, scales = f8.decode(out[0][0].get()), out[0][1].get()
    assert np.isnan(values[1]).all() and np.all(scales[:, 1] == 1.0)
    assert np.all(values[2] == 0) and np.all(scales[:, 2] == 1.0)
    # an infinite sum normalises by 0: the finite elements vanish, the infinite one is NaN
    assert np.isnan(values[3, 130]) and np.all(np.delete(values[3], 130) == 0)
    # the other row is what it is alone
    alone = g.empty_like_dev((1, cols), dtype=np.uint8), g.empty_like_dev((blocks, 1), dtype=np.float32)
    g.capi.check("q3x_b200_residual_add_rms_norm_fp8_block", g.Dev(left[:1]), g.Dev(right[:1]), g.Dev(weight), 1, cols, 1e-6,
                 g.empty_like_dev((1, cols)), None, *alone, None)
    g.sync()
    assert np.array_equal(alone[0].get()[0], out[0][0].get()[0]) and np.array_equal(alone[1].get()[:, 0], scales[:, 0])


# ---------------------------------------------------------------------------------------------------- SwiGLU


@pytest.mark.parametrize("rows,cols,merged", [(1, 16, False), (1, 17408, True), (7, 144, True), (33, 2064, False), (300, 1280, True),
                                              (513, 640, False)])
def test_silu_mul(g, rows, cols, merged):
    rng = np.random.default_rng([rows, cols, 17])
    both = orc.bf16_encode((3.0 * rng.standard_normal((rows, 2 * cols))).astype(np.float32))
    both[0, 0], both[0, 1] = 0xC2C8, 0x42C8  # gates of -100 and 100
    gate, up = both[:, :cols], both[:, cols:]
    codes, scales = g.empty_like_dev((rows, cols), dtype=np.uint8), g.empty_like_dev((f8.blocks_of(cols), rows), dtype=np.float32)
    if merged:
        d = g.Dev(both)
        g.capi.check("q3x_b200_silu_mul_fp8_block", d, d.ptr_at(cols), 2 * cols, rows, cols, codes, scales, None)
    else:
        g.capi.check("q3x_b200_silu_mul_fp8_block", g.Dev(gate), g.Dev(up), cols, rows, cols, codes, scales, None)
    g.sync()
    gv, uv = bf16_values(gate).astype(np.float64), bf16_values(up).astype(np.float64)
    y = gv / (1.0 + np.exp(-gv)) * uv
    # silu's FP32 error is bounded by 1e-5 (tests/test_gpu_chain_oracle.py); the product rounds once more
    assert_codes(codes.get(), scales.get(), y, 1.1e-5, f"{rows} x {cols}")
    assert codes.guards_intact() and scales.guards_intact()


def test_silu_mul_non_finite(g):
    rng = np.random.default_rng(19)
    gate, up = fx.normal_bf16(rng, (2, 256)), fx.normal_bf16(rng, (2, 256))
    gate[0, 3], up[1, 200], gate[1, 7], up[1, 7] = 0x7FC0, 0x7F80, 0x3F80, 0xFF80
    codes, scales = g.empty_like_dev((2, 256), dtype=np.uint8), g.empty_like_dev((2, 2), dtype=np.float32)
    g.capi.check("q3x_b200_silu_mul_fp8_block", g.Dev(gate), g.Dev(up), 256, 2, 256, codes, scales, None)
    g.sync()
    gv, uv = bf16_values(gate).astype(np.float64), bf16_values(up).astype(np.float64)
    y = gv / (1.0 + np.exp(-gv)) * uv
    assert_codes(codes.get(), scales.get(), y, 1.1e-5)
    values = f8.decode(codes.get())
    assert np.array_equal(values[np.isinf(y)], np.sign(y[np.isinf(y)]) * 448.0)


# ---------------------------------------------------------------------------------------------------- product

SHAPES = [(1, 8, 16), (1, 128, 128), (1, 5120, 5120), (2, 256, 1024), (3, 136, 2064), (16, 264, 144), (17, 128, 272), (31, 5120, 640),
          (33, 1000, 400), (48, 640, 17408), (64, 1024, 5120), (65, 384, 1296), (100, 24, 2048), (127, 520, 640), (128, 5120, 5120),
          (129, 256, 384), (255, 776, 1040), (256, 2048, 512), (300, 640, 6144), (512, 1288, 5120), (513, 136, 2064), (1000, 4104, 528),
          (2049, 1032, 656), (9000, 1032, 272), (2049, 2040, 2064), (5000, 2600, 400), (4097, 4104, 656), (256, 10232, 912),
          (500, 10072, 1040), (8193, 1000, 1168), (2000, 2600, 1296)]


def run_gemm(g, a, sa, w, sw, stream=None):
    tokens, (n, k) = a.shape[0], w.shape
    out = g.empty_like_dev((tokens, n), fill=0x7FC1)
    held = [g.Dev(w), g.Dev(sw), g.Dev(a), g.Dev(sa)]
    g.capi.check("q3x_b200_fp8_block_gemm_bf16", *held, tokens, n, k, out, stream)
    g.sync()
    assert out.guards_intact()
    return out.get()


@pytest.mark.parametrize("tokens,n,k", SHAPES)
def test_gemm(g, tokens, n, k):
    rng = np.random.default_rng([tokens, n, k, 23])
    a, sa, w, sw = f8.operands(rng, tokens, n, k)
    got = bf16_values(run_gemm(g, a, sa, w, sw)).astype(np.float64)
    want, magnitude = f8.product(a, sa, w, sw)
    over = np.abs(got - want) - f8.product_tolerance(want, magnitude, k)
    assert np.max(over) <= 0, f"{np.max(over)} past the tolerance at {np.unravel_index(np.argmax(over), over.shape)}"


@pytest.mark.parametrize("tokens,n,k", [(1, 136, 272), (16, 256, 1040), (40, 264, 640), (100, 136, 2064), (130, 392, 528), (600, 520, 400),
                                        (2049, 2040, 2064), (2000, 2600, 1296)])
def test_gemm_keeps_non_finite_values_to_their_rows_and_columns(g, tokens, n, k):
    """A NaN code, an infinite scale and scales of zero touch the outputs they belong to and no others."""
    rng = np.random.default_rng([tokens, n, k, 29])
    a, sa, w, sw = f8.operands(rng, tokens, n, k)
    a[(a & 0x7F) < 0x10] |= 0x30  # no zeros or subnormals: an infinite scale gives infinities and NaN alike everywhere
    w[(w & 0x7F) < 0x10] |= 0x30
    clean = run_gemm(g, a, sa, w, sw)
    row, col = tokens // 2, n // 2 + 3
    a2, w2, sa2 = a.copy(), w.copy(), sa.copy()
    a2[row, k - 1] = 0x7F
    w2[col, 0] = 0xFF
    sa2[:, tokens - 1] = 0.0
    if tokens > 2:
        sa2[0, 0] = np.inf
    got = run_gemm(g, a2, sa2, w2, sw)
    values = bf16_values(got)
    bad = np.zeros((tokens, n), dtype=bool)
    bad[row, :], bad[:, col] = True, True
    assert np.isnan(values[row]).all() and np.isnan(values[:, col]).all()
    if tokens > 2:
        assert not np.isfinite(values[0]).any()
        bad[0, :] = True
    if tokens - 1 != row:
        assert np.all(values[tokens - 1][~bad[tokens - 1]] == 0)
        bad[tokens - 1, :] = True
    assert np.array_equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("tokens,n,k", [(6, 264, 400), (30, 264, 400), (60, 392, 528), (128, 5120, 5120), (200, 264, 400), (500, 10072, 1040),
                                        (2049, 2040, 2064)])
def test_gemm_multiplies_the_scales_first(g, tokens, n, k):
    """Scales whose product is small, subnormal, 0, large or infinite in FP32: that product is what the sum is multiplied by."""
    rng = np.random.default_rng([tokens, n, k, 67])
    # (codes of 1/4 to 15/8, so that no block's sum is 0 and the products stay in range wherever the factor does)
    a, w = (rng.integers(0x28, 0x40, size=shape, dtype=np.uint8) for shape in ((tokens, k), (n, k)))
    row = np.resize(np.exp2([-126.0, -100, 0, 90, 119, -120]).astype(np.float32) * np.float32(1.25), tokens)
    col = np.resize(np.exp2([-30.0, -12, 20]).astype(np.float32) * np.float32(1.375), f8.blocks_of(n))
    sa, sw = np.tile(row, (f8.blocks_of(k), 1)), np.tile(col[:, None], (1, f8.blocks_of(k)))
    got = bf16_values(run_gemm(g, a, sa, w, sw)).astype(np.float64)
    with np.errstate(over="ignore", under="ignore"):
        factor = (row[:, None] * np.repeat(col, f8.BLOCK)[None, :n]).astype(np.float64)
    assert factor.min() == 0 and np.isinf(factor.max())
    want = factor * (f8.decode(a) @ f8.decode(w).T)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine])
    assert np.all(got[factor == 0] == 0)
    # (all terms are positive: their sum is their magnitude)
    got, want = got[fine], want[fine]
    assert np.all(np.abs(got - want) <= f8.product_tolerance(want, want, k))


@pytest.mark.parametrize("tokens,n,k", [(1, 520, 5136), (5, 520, 5136), (16, 520, 5136), (40, 520, 5136), (100, 520, 5136), (129, 520, 5136),
                                        (700, 520, 5136), (2049, 2040, 2064), (2000, 2600, 1296)])
def test_gemm_repeats_bit_for_bit(g, tokens, n, k):
    """Sums are joined in one order, whatever the launch: equal inputs give equal bytes."""
    rng = np.random.default_rng([tokens, 31])
    a, sa, w, sw = f8.operands(rng, tokens, n, k)
    first = run_gemm(g, a, sa, w, sw)
    for _ in range(3):
        assert np.array_equal(run_gemm(g, a, sa, w, sw), first)


# Strips whose clusters of two to five CTAs share K and walk two to five tiles each, with ranks that own no group of four tokens and
# with ranks that all own one; and, in the last line, clusters of one CTA that walk two tiles.
ROUNDS = [(1, 24576, 1024), (4, 24568, 1024), (1, 10240, 1040), (4, 10240, 1536), (8, 10240, 1536), (8, 20480, 1152), (5, 10248, 1168),
          (16, 10240, 1536), (12, 13312, 5120), (7, 12288, 5120), (2, 34816, 912), (30, 10240, 1536), (24, 19456, 912), (50, 10240, 2064),
          (64, 19464, 1168),
          (1, 34816, 640), (48, 34816, 640)]


@pytest.mark.parametrize("tokens,n,k", ROUNDS)
def test_gemm_strips_of_several_tiles_per_cluster(g, tokens, n, k):
    """Against the definition, and again and again: the barriers of a tile's end come round from tile to tile."""
    rng = np.random.default_rng([tokens, n, k, 59])
    a, sa, w, sw = f8.operands(rng, tokens, n, k)
    held = [g.Dev(w), g.Dev(sw), g.Dev(a), g.Dev(sa)]
    out = g.empty_like_dev((tokens, n), fill=0x7FC1)
    g.capi.check("q3x_b200_fp8_block_gemm_bf16", *held, tokens, n, k, out, None)
    g.sync()
    first = out.get()
    want, magnitude = f8.product(a, sa, w, sw)
    over = np.abs(bf16_values(first).astype(np.float64) - want) - f8.product_tolerance(want, magnitude, k)
    assert np.max(over) <= 0, f"{np.max(over)} past the tolerance at {np.unravel_index(np.argmax(over), over.shape)}"
    expected, wrong = out.t.clone(), torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(200):
        out.t.zero_()
        g.capi.check("q3x_b200_fp8_block_gemm_bf16", *held, tokens, n, k, out, None)
        wrong += (out.t != expected).sum()
    g.sync()
    assert int(wrong) == 0
    assert out.guards_intact()
    assert g.capi.lib().q3x_b200_fp8_block_gemm_error() == 0


@pytest.mark.parametrize("tokens", [1, 24, 100, 300])
def test_gemm_on_streams_and_in_graphs(g, tokens):
    """Two calls at once on two streams, and a captured pair replayed on new inputs."""
    rng = np.random.default_rng([tokens, 37])
    n, k = 1032, 2576
    sets = [f8.operands(rng, tokens, n, k) for _ in range(2)]
    want = [run_gemm(g, *s) for s in sets]
    held = [[g.Dev(s[2]), g.Dev(s[3]), g.Dev(s[0]), g.Dev(s[1])] for s in sets]
    outs = [g.empty_like_dev((tokens, n)) for _ in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    g.sync()
    for _ in range(5):
        for h, o, s in zip(held, outs, streams):
            g.capi.check("q3x_b200_fp8_block_gemm_bf16", *h, tokens, n, k, o, s.cuda_stream)
    g.sync()
    for o, w in zip(outs, want):
        assert np.array_equal(o.get(), w)
    graph = torch.cuda.CUDAGraph()
    for o in outs:
        o.t.zero_()
    with torch.cuda.graph(graph):
        s = torch.cuda.current_stream().cuda_stream
        for h, o in zip(held, outs):
            g.capi.check("q3x_b200_fp8_block_gemm_bf16", *h, tokens, n, k, o, s)
    graph.replay()
    g.sync()
    for o, w in zip(outs, want):
        assert np.array_equal(o.get(), w)
    for i in range(4):  # the first call's operands become the second's
        held[0][i].t.copy_(held[1][i].t)
    graph.replay()
    g.sync()
    assert np.array_equal(outs[0].get(), want[1]) and np.array_equal(outs[1].get(), want[1])


def test_calls_from_two_threads_and_graphs_of_all_kernels_at_once(g):
    """Two threads enqueue products of every kernel on streams of their own; then two captured graphs of the same
    products are replayed at once, again and again.  Nothing is shared between them but their inputs."""
    rng = np.random.default_rng(47)
    shapes = [(1, 2056, 2576), (30, 1032, 1296), (60, 520, 2064), (100, 136, 2064), (200, 1032, 1296), (500, 10072, 1040), (2049, 2040, 2064)]
    work = []
    for shape in shapes:
        a, sa, w, sw = f8.operands(rng, *shape)
        work.append((shape, [g.Dev(w), g.Dev(sw), g.Dev(a), g.Dev(sa)], run_gemm(g, a, sa, w, sw)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[g.empty_like_dev(want.shape) for _, _, want in work] for _ in streams]
    g.sync()

    def enqueue(outs, stream, order):
        for i in order:
            (tokens, n, k), held, _ = work[i]
            g.capi.check("q3x_b200_fp8_block_gemm_bf16", *held, tokens, n, k, outs[i], stream)

    def verify():
        g.sync()
        for mine in outs:
            for out, (shape, _, want) in zip(mine, work):
                assert np.array_equal(out.get(), want), shape
                assert out.guards_intact()
                out.t.zero_()
        assert g.capi.lib().q3x_b200_fp8_block_gemm_error() == 0

    orders = [list(range(len(work))), list(reversed(range(len(work))))]
    threads = [threading.Thread(target=lambda o=o, s=s, r=r: [enqueue(o, s.cuda_stream, r) for _ in range(10)])
               for o, s, r in zip(outs, streams, orders)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    verify()
    graphs = []
    for o, r in zip(outs, orders):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            enqueue(o, torch.cuda.current_stream().cuda_stream, r)
        graphs.append(graph)
    for _ in range(10):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    verify()


def test_gemm_error_waits_for_streams_that_the_default_one_does_not(g):
    """The word answers for every call enqueued before, on a non-blocking stream too."""
    rng = np.random.default_rng(61)
    a, sa, w, sw = f8.operands(rng, 3, 264, 400)
    want = run_gemm(g, a, sa, w, sw)
    held, out, side = [g.Dev(w), g.Dev(sw), g.Dev(a), g.Dev(sa)], g.empty_like_dev((3, 264)), torch.cuda.Stream()
    g.sync()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)  # some 50 ms
    g.capi.check("q3x_b200_fp8_block_gemm_bf16", *held, 3, 264, 400, out, side.cuda_stream)
    assert not side.query()
    assert g.capi.lib().q3x_b200_fp8_block_gemm_error() == 0
    assert side.query()
    assert np.array_equal(out.get(), want)


def test_gemm_captured_from_a_thread_that_made_no_call_before(g):
    rng = np.random.default_rng(53)
    shapes = [(3, 264, 400), (600, 520, 400), (2049, 2040, 2064)]
    work = []
    for shape in shapes:
        a, sa, w, sw = f8.operands(rng, *shape)
        work.append((shape, [g.Dev(w), g.Dev(sw), g.Dev(a), g.Dev(sa)], run_gemm(g, a, sa, w, sw), g.empty_like_dev(shape[:2])))
    graph, failed = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        stream = torch.cuda.current_stream().cuda_stream
        for (tokens, n, k), held, _, out in work:
            call = lambda: failed.append(g.capi.call("q3x_b200_fp8_block_gemm_bf16", *held, tokens, n, k, out, stream))
            thread = threading.Thread(target=call)
            thread.start()
            thread.join()
    assert failed == [0, 0, 0]
    graph.replay()
    g.sync()
    for shape, _, want, out in work:
        assert np.array_equal(out.get(), want), shape


def test_gemm_reads_scales_from_any_float_address(g):
    rng = np.random.default_rng(43)
    for tokens in (3, 50, 150):
        a, sa, w, sw = f8.operands(rng, tokens, 264, 656)
        out = g.empty_like_dev((tokens, 264))
        g.capi.check("q3x_b200_fp8_block_gemm_bf16", g.Dev(w), g.Dev(sw, misalign=1), g.Dev(a), g.Dev(sa, misalign=3), tokens, 264, 656,
                     out, None)
        g.sync()
        assert np.array_equal(out.get(), run_gemm(g, a, sa, w, sw))


FIRST_CALL = """
import importlib, sys
import torch
capi = importlib.import_module("qwen3x-orin_b200").capi
capi.load()
for tokens, n, k in ((1, 520, 1040), (100, 136, 2064), (200, 264, 400), (2049, 2040, 2064), (500, 10072, 1040)):
    blocks = (k + 127) // 128
    w, a = torch.full((n, k), 0x38, dtype=torch.uint8, device="cuda"), torch.full((tokens, k), 0x38, dtype=torch.uint8, device="cuda")
    sw, sa = torch.ones((n + 127) // 128, blocks, device="cuda"), torch.ones(blocks, tokens, device="cuda")
    out = torch.zeros(tokens, n, dtype=torch.bfloat16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.check("q3x_b200_fp8_block_gemm_bf16", w, sw, a, sa, tokens, n, k, out, torch.cuda.current_stream().cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((out == torch.tensor(float(k)).bfloat16().item()).all()), (tokens, n, k)
assert capi.lib().q3x_b200_fp8_block_gemm_error() == 0
"""


def test_gemm_can_be_captured_by_the_first_call_of_a_process(g):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=240)
    assert done.returncode == 0, done.stdout[-2000:] + done.stderr[-2000:]


# ---------------------------------------------------------------------------------------------------- long tensors


def random_codes_on_device(rows, cols, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (rows, cols), generator=gen, device="cuda", dtype=torch.uint8)
    return torch.where((codes & 0x7F) == 0x7F, torch.full_like(codes, 0x3C), codes)


@pytest.mark.parametrize("tokens,n,k", [(70001, 34816, 144), (140001, 136, 17408)])
def test_gemm_beyond_32_bit_offsets(g, tokens, n, k):
    """More than 2^31 outputs, and more than 2^31 codes: a few rows from every part against their definition."""
    a, w = random_codes_on_device(tokens, k, 1), random_codes_on_device(n, k, 2)
    gen = torch.Generator(device="cuda").manual_seed(3)
    sa = torch.rand((f8.blocks_of(k), tokens), generator=gen, device="cuda") * 0.01 + 0.001
    sw = torch.rand((f8.blocks_of(n), f8.blocks_of(k)), generator=gen, device="cuda") * 0.001 + 0.0001
    out = torch.zeros((tokens, n), dtype=torch.bfloat16, device="cuda")
    g.capi.check("q3x_b200_fp8_block_gemm_bf16", w, sw, a, sa, tokens, n, k, out, None)
    g.sync()
    rows = torch.tensor([0, 127, 128, tokens // 2, 61681, 61682, tokens - 129, tokens - 2, tokens - 1], device="cuda")
    host = lambda t: t.cpu().numpy()
    want, magnitude = f8.product(host(a[rows]), host(sa[:, rows]), host(w), host(sw))
    got = host(out[rows].double())
    assert np.all(np.abs(got - want) <= f8.product_tolerance(want, magnitude, k))
    assert bool((out != 0).any(dim=1).all())  # no row was left out


def test_quantisers_beyond_32_bit_offsets(g):
    rows, cols = 131073, 17408
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    for first in range(0, rows, 16384):
        part = x[first:first + 16384]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda"))
    codes = torch.zeros((rows, cols), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((f8.blocks_of(cols), rows), device="cuda")
    picked = torch.tensor([0, 1, 61680, 61681, 123361, 123362, rows - 2, rows - 1], device="cuda")
    values = x[picked].float().cpu().numpy()
    g.capi.check("q3x_b200_fp8_block_quantize", x, rows, cols, codes, scales, None)
    g.sync()
    want, want_scales = f8.quantize(values)
    assert np.array_equal(scales[:, picked].cpu().numpy(), want_scales)
    assert np.array_equal(f8.decode(codes[picked].cpu().numpy()), want)
    # SwiGLU of the two halves of each row: the second half starts at an odd number of blocks
    half = cols // 2
    codes, scales = codes[:, :half].contiguous(), torch.zeros((f8.blocks_of(half), rows), device="cuda")
    g.capi.check("q3x_b200_silu_mul_fp8_block", x, x.data_ptr() + 2 * half, cols, rows, half, codes, scales, None)
    g.sync()
    gate, up = values[:, :half].astype(np.float64), values[:, half:].astype(np.float64)
    assert_codes(codes[picked].cpu().numpy(), scales[:, picked].cpu().numpy(), gate / (1.0 + np.exp(-gate)) * up, 1.1e-5)


# ---------------------------------------------------------------------------------------------------- in a row


@pytest.mark.parametrize("tokens", [1, 19, 200])
def test_mlp_block_in_a_row(g, tokens):
    """Residual + norm -> merged gate | up product -> SwiGLU -> down product, captured and replayed, each stage against
    its definition on the previous stage's own bytes."""
    rng = np.random.default_rng([tokens, 41])
    hidden, inter, eps = 640, 1296, 1e-6
    left, right = fx.normal_bf16(rng, (tokens, hidden)), fx.normal_bf16(rng, (tokens, hidden))
    weight = orc.bf16_encode((0.1 * rng.standard_normal(hidden)).astype(np.float32))
    w1, w2 = f8.random_codes(rng, (2 * inter, hidden)), f8.random_codes(rng, (hidden, inter))
    s1 = np.exp2(rng.uniform(-13, -11, size=(f8.blocks_of(2 * inter), f8.blocks_of(hidden)))).astype(np.float32)
    s2 = np.exp2(rng.uniform(-13, -11, size=(f8.blocks_of(hidden), f8.blocks_of(inter)))).astype(np.float32)
    d = {n: g.Dev(v) for n, v in dict(left=left, right=right, weight=weight, w1=w1, s1=s1, w2=w2, s2=s2).items()}
    residual, merged, down = g.empty_like_dev((tokens, hidden)), g.empty_like_dev((tokens, 2 * inter)), g.empty_like_dev((tokens, hidden))
    x_codes, x_scales = g.empty_like_dev((tokens, hidden), dtype=np.uint8), g.empty_like_dev((f8.blocks_of(hidden), tokens), dtype=np.float32)
    h_codes, h_scales = g.empty_like_dev((tokens, inter), dtype=np.uint8), g.empty_like_dev((f8.blocks_of(inter), tokens), dtype=np.float32)

    def enqueue(s):
        g.capi.check("q3x_b200_residual_add_rms_norm_fp8_block", d["left"], d["right"], d["weight"], tokens, hidden, eps, residual, None,
                     x_codes, x_scales, s)
        g.capi.check("q3x_b200_fp8_block_gemm_bf16", d["w1"], d["s1"], x_codes, x_scales, tokens, 2 * inter, hidden, merged, s)
        g.capi.check("q3x_b200_silu_mul_fp8_block", merged, merged.ptr_at(inter), 2 * inter, tokens, inter, h_codes, h_scales, s)
        g.capi.check("q3x_b200_fp8_block_gemm_bf16", d["w2"], d["s2"], h_codes, h_scales, tokens, hidden, inter, down, s)

    enqueue(None)
    g.sync()
    eager = [b.get() for b in (residual, x_codes, x_scales, merged, h_codes, h_scales, down)]
    r = bf16_values(residual.get()).astype(np.float64)
    y = r / np.sqrt((r * r).mean(axis=1, keepdims=True) + np.float64(np.float32(eps))) * (1.0 + bf16_values(weight).astype(np.float64))
    assert_codes(x_codes.get(), x_scales.get(), y, 2.0 ** -18, "norm")
    want, mag = f8.product(x_codes.get(), x_scales.get(), w1, s1)
    assert np.all(np.abs(bf16_values(merged.get()) - want) <= f8.product_tolerance(want, mag, hidden))
    m = bf16_values(merged.get()).astype(np.float64)
    h = m[:, :inter] / (1.0 + np.exp(-m[:, :inter])) * m[:, inter:]
    assert_codes(h_codes.get(), h_scales.get(), h, 1.1e-5, "SwiGLU")
    want, mag = f8.product(h_codes.get(), h_scales.get(), w2, s2)
    assert np.all(np.abs(bf16_values(down.get()) - want) <= f8.product_tolerance(want, mag, inter))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        enqueue(torch.cuda.current_stream().cuda_stream)
    for b in (residual, x_codes, x_scales, merged, h_codes, h_scales, down):
        b.t.zero_()
    graph.replay()
    g.sync()
    for b, e in zip((residual, x_codes, x_scales, merged, h_codes, h_scales, down), eager):
        assert np.array_equal(b.get(), e) and b.guards_intact()


@pytest.mark.parametrize("tokens", [1, 300])
def test_projected_mlp_fp8_block(g, tokens):
    """chain.ProjectedMlpFp8Block, stage by stage on its own buffers."""
    chain = importlib.import_module("qwen3x-orin_b200.chain")
    block = chain.ProjectedMlpFp8Block(tokens, torch.device("cuda", 0), hidden=1280, intermediate=1040, seed=5)
    block.enqueue(None)
    g.sync()
    block.check_error()
    bits = lambda t: t.view(torch.int16).cpu().numpy().view(np.uint16)
    host = lambda t: t.cpu().numpy()
    r = bf16_values(orc.bf16_encode(bf16_values(bits(block.left)) + bf16_values(bits(block.right))))
    assert np.array_equal(bf16_values(bits(block.residual)), r)
    r = r.astype(np.float64)
    y = r / np.sqrt((r * r).mean(axis=1, keepdims=True) + np.float64(np.float32(chain.EPS))) * (1.0 + bf16_values(bits(block.norm_w)).astype(np.float64))
    assert_codes(host(block.x_codes), host(block.x_scales), y, 2.0 ** -18, "norm")
    want, mag = f8.product(host(block.x_codes), host(block.x_scales), host(block.w_gate_up["codes"]), host(block.w_gate_up["scales"]))
    assert np.all(np.abs(bf16_values(bits(block.gate_up)) - want) <= f8.product_tolerance(want, mag, 1280))
    m = bf16_values(bits(block.gate_up)).astype(np.float64)
    h = m[:, :1040] / (1.0 + np.exp(-m[:, :1040])) * m[:, 1040:]
    assert_codes(host(block.h_codes), host(block.h_scales), h, 1.1e-5, "SwiGLU")
    want, mag = f8.product(host(block.h_codes), host(block.h_scales), host(block.w_down["codes"]), host(block.w_down["scales"]))
    assert np.all(np.abs(bf16_values(bits(block.down)) - want) <= f8.product_tolerance(want, mag, 1040))
