"""Rotary plans and the 4-bit cache without a GPU: the layout's host walk, the scaled frequencies, refusals."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

from powerinfer_x64_amd import _abi, runtime as rt
from tests import q4_ref as ref

EXE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build", "test_q4_layout")


def test_layout_walk():
    assert os.path.exists(EXE), "tests/cpp not built (python -m powerinfer_x64_amd.build)"
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and " 0 failures" in r.stdout, r.stdout


@pytest.mark.parametrize("dim", [2, 18, 64, 128, 256, 512])
@pytest.mark.parametrize("base", [1e4, 1e7])
def test_frequencies(dim, base):
    plain, m = rt.rope_freqs(dim, base)
    want = np.array([base ** (-2.0 * i / dim) for i in range(dim // 2)])
    np.testing.assert_allclose(plain, want, rtol=1e-14)
    assert m == 1.0
    f, m = rt.rope_freqs(dim, base, "linear", factor=3.0)
    np.testing.assert_allclose(f, want / 3, rtol=1e-14)
    if dim > 2:
        f, m = rt.rope_freqs(dim, base, "ntk", factor=4.0)
        assert m == 1.0 and f[0] == 1.0
        np.testing.assert_allclose(f[-1], want[-1] / 4, rtol=1e-13)  # the slowest pair slows down by the factor
    # yarn: every pair lies between scaled and unscaled, fast pairs keep their speed, and the slowest are scaled
    f, m = rt.rope_freqs(dim, base, "yarn", factor=8.0, orig_ctx=4096)
    assert m == 0.1 * math.log(8.0) + 1.0
    assert (f <= want * (1 + 1e-14)).all() and (f >= want / 8 * (1 - 1e-14)).all()
    # the band's edges, as whole pair indices at which a pair turns 32 times and once in 4096 tokens
    lo, hi = (dim * math.log(4096 / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (32.0, 1.0))
    for i in range(dim // 2):
        if i <= math.floor(lo):
            assert math.isclose(f[i], want[i], rel_tol=1e-13)
        if i >= math.ceil(hi):
            assert math.isclose(f[i], want[i] / 8, rel_tol=1e-13)
    f, m = rt.rope_freqs(dim, base, "bands", factor=8.0, orig_ctx=8192, params=(1.0, 4.0))
    for i in range(dim // 2):
        turns = 8192 * want[i] / (2 * math.pi)
        share = min(1.0, max(0.0, (turns - 1) / 3))
        assert math.isclose(f[i], want[i] * (share + (1 - share) / 8), rel_tol=1e-13)


@pytest.mark.parametrize("args", [
    dict(rope_dim=3), dict(rope_dim=0), dict(rope_dim=-2), dict(rope_dim=64, base=0.0), dict(rope_dim=64, base=math.nan),
    dict(rope_dim=64, base=math.inf), dict(rope_dim=64, scaling="linear", factor=0.0),
    dict(rope_dim=64, scaling="linear", factor=-1.0), dict(rope_dim=64, scaling="ntk", factor=math.inf),
    dict(rope_dim=2, scaling="ntk", factor=2.0), dict(rope_dim=64, base=1.0, scaling="yarn", factor=2.0),
    dict(rope_dim=64, scaling="bands", factor=2.0, params=(4.0, 4.0)), dict(rope_dim=64, scaling="yarn", factor=2.0, orig_ctx=0),
    dict(rope_dim=64, scaling="yarn", factor=2.0, params=(32.0,)), dict(rope_dim=64, scaling="other"),
    dict(rope_dim=64, scaling="linear", factor=2.0, params=(1.0, 2.0))])
def test_frequency_refusals(args):
    with pytest.raises(rt.InvalidArg):
        rt.rope_freqs(**args)


def test_null_handles_and_arguments_are_refused():
    lib = _abi.load()
    x = (ctypes.c_double * 4)()
    p = ctypes.c_void_p()
    n = ctypes.c_size_t()
    assert lib.pi_rope_scaled_freqs(8, 1e4, 0, None, 0, None, None) == 1
    assert lib.pi_rope_scaled_freqs(8, 1e4, 7, None, 0, x, x) == 1
    assert lib.pi_rope_plan_create(None, 8, 0, x, 1.0, ctypes.byref(p)) == 1
    assert lib.pi_rope_apply(None, None, 0, 1, 8, None, None, 8, 8, 1, None, 8, 8, None, 0, 0, 0, None, 0, 0, None) == 1
    assert lib.pi_q4_pool_create(None, 1, 16, 1, 64, ctypes.byref(p)) == 1
    assert lib.pi_q4_append(None, None, None, 0, 1, None, None, 1, None, 1, None, 0, 0, 0, None, 0, 0, None, 0, 0, None, 0, 0,
                            None, None, 0.0, None, None, None) == 1
    assert lib.pi_q4_read(None, None, None, 1, 0, 0, 1, None, None, None, None, None) == 1
    assert lib.pi_q4_write(None, None, None, 1, 0, 0, 1, None, None, None, None, None) == 1
    assert lib.pi_q4_attn_ws_bytes(None, None, 0, 1, 1, 1, 1, 0, 1, 0, ctypes.byref(n)) == 1
    assert lib.pi_q4_attn_decode(None, None, None, 0, None, 1, 0, None, 1, 1, 0, 1.0, None, None, None, 0, None) == 1
    assert lib.pi_q4_attn_prefill(None, None, None, 0, 1, None, None, 1, 1, None, 1, 0, 1, 0, 1.0, None, None, None, 0, None) == 1
    assert b"null pi_handle" in lib.pi_last_error(None)
    lib.pi_rope_plan_destroy(None)
    lib.pi_q4_pool_destroy(None)
    assert lib.pi_q4_pool_bytes(None) == 0


def test_reference_quantiser_keeps_its_own_rules():
    """The formulas that the GPU tests hold the cache to: exact extremes, half a step elsewhere, ties, saturation."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((500, 64))
    c, s = ref.quantise(x)
    y = ref.values(c, s)
    assert np.array_equal(y.astype(np.float16).astype(np.float64), y)  # exact in f16
    g, gy, st = x.reshape(500, 2, 32), y.reshape(500, 2, 32), np.abs(s)[..., None]
    inside = np.abs(g) <= 7.5 * st
    assert (np.abs(g - gy)[inside] <= (0.5 * st * np.ones_like(g))[inside] * (1 + 1e-12)).all()
    assert (np.abs(g - gy) <= st * (1 + 2.0 ** -3)).all()
    one = np.zeros(32)
    one[3], one[9] = -2.0, 2.0  # a tie: the positive one sets the scale
    c, s = ref.quantise(one)
    assert s[0] == -0.25 and ref.values(c, s)[9] == 2.0 and ref.values(c, s)[3] == -1.75
    assert np.array_equal(ref.unpack(ref.pack(c)), c)
    one[:] = [np.nan, np.inf, -np.inf] + [1.0] * 29
    assert np.array_equal(ref.values(*ref.quantise(one))[:4], [0.0, 7232.0, -6328.0, 0.0])
