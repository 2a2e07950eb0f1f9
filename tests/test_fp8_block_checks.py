"""Refusals of the FP8 operators with a scale per block of 128 (they happen on the host, before any device work, so they
run without a GPU), and the numpy restatement of the format against torch's own E4M3 type."""
import importlib
import os
import re

import numpy as np
import pytest
import torch

from tests import fp8_block_util as f8

INVALID, UNSUPPORTED, OK = 1, 801, 0
A, STEP = 1 << 40, 1 << 32  # fake device addresses, never dereferenced, far enough apart for every shape below


@pytest.fixture(scope="module")
def capi():
    pkg = importlib.import_module("qwen3x-orin_b200")
    importlib.import_module("qwen3x-orin_b200.build").build_all()
    pkg.capi.load()
    return pkg.capi


def test_restatement_matches_torch_e4m3():
    codes = np.arange(256, dtype=np.uint8)
    torch_values = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(f8.decode(codes), torch_values, equal_nan=True)
    rng = np.random.default_rng(1)
    x = np.concatenate([rng.normal(size=20000) * 100, rng.normal(size=20000) * 2.0 ** -7, [448, -448, 2.0 ** -10, 3 * 2.0 ** -10]])
    x = np.clip(x.astype(np.float32), -448, 448)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(f8.round_e4m3(x), want)
    grid = np.sort(f8.TABLE[:127])
    middles = (grid[1:] + grid[:-1]) / 2  # exact midpoints go to the even code
    want = torch.from_numpy(middles).float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(f8.round_e4m3(middles), want)
    assert np.all(np.abs(f8.round_e4m3(x) - x) <= f8.half_step(x))


def test_quantize_refusals(capi):
    def call(**kw):
        a = dict(x=A, rows=4, cols=256, codes=A + STEP, scales=A + 2 * STEP)
        a.update(kw)
        return capi.call("q3x_b200_fp8_block_quantize", a["x"], a["rows"], a["cols"], a["codes"], a["scales"], None)

    assert call(cols=24) == INVALID and call(cols=8) == INVALID
    assert call(x=None) == INVALID and call(codes=None) == INVALID and call(scales=None) == INVALID
    assert call(codes=A + 16) == INVALID and call(scales=A + 2044) == INVALID and call(scales=A + STEP + 1020) == INVALID
    assert call(rows=1 << 62) == INVALID and call(x=(1 << 64) - 1024) == INVALID
    assert call(x=A + 2) == UNSUPPORTED and call(codes=A + STEP + 8) == UNSUPPORTED and call(scales=A + 2 * STEP + 2) == UNSUPPORTED
    assert call(rows=1 << 31, cols=16, codes=A + 64 * STEP, scales=A + 128 * STEP) == UNSUPPORTED
    assert call(rows=0, x=None, codes=None, scales=None) == OK and call(cols=0, x=None, codes=None, scales=None) == OK


def test_residual_norm_refusals(capi):
    def call(**kw):
        a = dict(left=A, right=A + STEP, w=A + 2 * STEP, t=4, h=256, eps=1e-6, res=A + 3 * STEP, norm=A + 4 * STEP,
                 codes=A + 5 * STEP, scales=A + 6 * STEP)
        a.update(kw)
        return capi.call("q3x_b200_residual_add_rms_norm_fp8_block", a["left"], a["right"], a["w"], a["t"], a["h"], a["eps"],
                         a["res"], a["norm"], a["codes"], a["scales"], None)

    assert call(eps=0.0) == INVALID and call(eps=float("nan")) == INVALID and call(eps=float("inf")) == INVALID
    assert call(h=24) == INVALID and call(h=0) == OK and call(t=0, left=None, codes=None) == OK
    for name in ("left", "right", "w", "res", "codes", "scales"):
        assert call(**{name: None}) == INVALID, name
    assert call(res=A) == INVALID and call(right=A + 2) == INVALID and call(norm=A) == INVALID
    for other in ("left", "right", "w", "res", "norm"):
        at = dict(left=A, right=A + STEP, w=A + 2 * STEP, res=A + 3 * STEP, norm=A + 4 * STEP)[other]
        assert call(codes=at) == INVALID and call(scales=at + 16) == INVALID, other
    assert call(codes=A + 5 * STEP, scales=A + 5 * STEP + 1020) == INVALID
    for name in ("left", "right", "w", "res", "norm"):
        at = dict(left=A, right=A + STEP, w=A + 2 * STEP, res=A + 3 * STEP, norm=A + 4 * STEP)[name]
        assert call(**{name: at + 2}) == UNSUPPORTED, name
    assert call(h=32768 + 16) == UNSUPPORTED and call(codes=A + 5 * STEP + 4) == UNSUPPORTED
    assert call(t=1 << 62) == INVALID


def test_silu_mul_refusals(capi):
    def call(**kw):
        a = dict(gate=A, up=A + STEP, stride=256, t=4, i=256, codes=A + 2 * STEP, scales=A + 3 * STEP)
        a.update(kw)
        return capi.call("q3x_b200_silu_mul_fp8_block", a["gate"], a["up"], a["stride"], a["t"], a["i"], a["codes"], a["scales"],
                         None)

    assert call(i=24, stride=32) == INVALID and call(stride=240) == INVALID
    for name in ("gate", "up", "codes", "scales"):
        assert call(**{name: None}) == INVALID, name
    assert call(codes=A + 2032) == INVALID and call(scales=A + STEP) == INVALID and call(scales=A + 2 * STEP) == INVALID
    # the gap between the rows of a strided operand belongs to it
    assert call(stride=512, codes=A + 512) == INVALID
    assert call(stride=260) == UNSUPPORTED and call(gate=A + 8) == UNSUPPORTED and call(up=A + STEP + 2) == UNSUPPORTED
    assert call(codes=A + 2 * STEP + 1) == UNSUPPORTED and call(scales=A + 3 * STEP + 1) == UNSUPPORTED
    assert call(t=1 << 60) == INVALID and call(t=0, gate=None) == OK and call(i=0, stride=0, gate=None) == OK


def test_gemm_refusals(capi):
    def call(**kw):
        a = dict(w=A, sw=A + STEP, x=A + 2 * STEP, sx=A + 3 * STEP, t=4, n=64, k=256, out=A + 4 * STEP)
        a.update(kw)
        return capi.call("q3x_b200_fp8_block_gemm_bf16", a["w"], a["sw"], a["x"], a["sx"], a["t"], a["n"], a["k"], a["out"], None)

    assert call(k=0) == INVALID and call(k=24) == INVALID and call(n=12) == INVALID
    for name in ("w", "sw", "x", "sx", "out"):
        assert call(**{name: None}) == INVALID, name
    assert call(t=1 << 31) == INVALID and call(n=1 << 31) == INVALID and call(k=1 << 31) == INVALID
    assert call(out=A) == INVALID and call(out=A + 2 * STEP + 16) == INVALID
    assert call(sw=A + 4 * STEP) == INVALID and call(sx=A + 4 * STEP + 508) == INVALID
    assert call(w=A + 8) == UNSUPPORTED and call(x=A + 2 * STEP + 8) == UNSUPPORTED and call(out=A + 4 * STEP + 8) == UNSUPPORTED
    assert call(sw=A + STEP + 2) == UNSUPPORTED and call(sx=A + 3 * STEP + 1) == UNSUPPORTED
    assert call(t=0, w=None) == OK and call(n=0, w=None) == OK


def test_corrected_quotient_is_the_rounded_one():
    """amax / 448 as the kernels form it -- a product with the rounded reciprocal and one correction by the exact
    remainder -- for every mantissa of one binade (the others are its multiples by powers of two)."""
    a = np.arange(1 << 23, 1 << 24, dtype=np.int64).astype(np.float32)
    reciprocal = np.float32(1) / np.float32(448)
    q = a * reciprocal
    rest = a.astype(np.float64) - q.astype(np.float64) * 448.0  # 27 bits: exact
    assert np.all(rest.astype(np.float32).astype(np.float64) == rest)
    # (the sum has to be rounded once; the quotient is at least 1/14 step away from a midpoint, 64 bits of it decide)
    corrected = (q.astype(np.longdouble) + rest.astype(np.longdouble) * np.longdouble(reciprocal)).astype(np.float32)
    assert np.array_equal(corrected, a / np.float32(448))


def test_aligned_cluster_barriers_follow_a_convergence_of_their_warp():
    """barrier.cluster.*.aligned wants all lanes of a warp at the instruction together; its callers come from branches that
    one lane takes (an arrival, a copy).  So each helper that issues one brings its warp together first, and nothing issues
    one past the helpers."""
    source = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3x-orin_b200", "csrc", "fp8_block_gemm.cu")
    with open(source) as f:
        text = f.read()
    found = [m.start() for m in re.finditer(r"barrier\.cluster\.\w+[\w.]*\.aligned", text)]
    helpers = [re.search(r"void cluster_%s\(\) \{(.*?)\n?\}" % what, text, re.S) for what in ("arrive", "wait")]
    assert len(found) == 2
    for helper, at in zip(helpers, found):
        assert helper.start() < at < helper.end()
        assert "__syncwarp();" in text[helper.start():at]
