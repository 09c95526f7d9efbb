"""CPU checks of the 8-bit row makers: the refusals of the C ABI (nothing is launched for any of
them, so they run without a GPU) and the oracle the GPU tests compare against."""
import ctypes as C

import numpy as np
import pytest

from frisk_b200 import runtime as R
from frisk_b200 import workloads as W
from oracle import ref

INVALID, UNSUPPORTED, MISALIGNED, TOO_LARGE = -1, -2, -3, -9


def run(desc, x=0x10000, q=0x20000, scale=0x30000, **kw):
    """A launch on made-up addresses: only calls that are refused before the launch come here."""
    R.quant_run(desc, x, q, scale, **kw)


def refused(code, desc, *a, **kw):
    with pytest.raises(R.FriskError) as e:
        run(desc, *a, **kw)
    assert e.value.code == code, e.value


def test_descriptions_that_are_refused():
    d = R.quant_desc
    refused(INVALID, d(-1, 8, W.BF16, W.I8))
    refused(INVALID, d(4, 0, W.BF16, W.I8))
    refused(INVALID, d(4, -8, W.BF16, W.I8))
    refused(UNSUPPORTED, d(4, 8, W.E4M3, W.I8))
    refused(UNSUPPORTED, d(4, 8, W.I8, W.I8))
    refused(UNSUPPORTED, d(4, 8, W.BF16, W.BF16))
    refused(UNSUPPORTED, d(4, 8, W.BF16, W.F32))
    refused(UNSUPPORTED, d(4, 8, 17, W.I8))
    refused(UNSUPPORTED, d(4, 8, W.BF16, W.I8, "rmsnorm", weight_type=W.F16))
    refused(UNSUPPORTED, d(4, 8, W.F32, W.I8, "rmsnorm", weight_type=W.BF16))
    for eps in (-1e-6, float("nan"), float("inf")):
        refused(INVALID, d(4, 8, W.BF16, W.I8, "rmsnorm", eps=eps))
    for ld in ("ldx", "ldo", "lds", "ldq"):
        refused(INVALID, d(4, 8, W.BF16, W.I8, "rmsnorm", **{ld: 7}))
        refused(INVALID, d(4, 8, W.BF16, W.I8, "rmsnorm", **{ld: -8}))
        refused(TOO_LARGE, d(4, 8, W.BF16, W.I8, "rmsnorm", **{ld: 1 << 60}))
        refused(TOO_LARGE, d(1 << 39, 8, W.BF16, W.I8, "rmsnorm", **{ld: 1 << 39}))
    refused(TOO_LARGE, d(4, 1 << 31, W.BF16, W.I8))
    refused(TOO_LARGE, d(1 << 58, 8, W.BF16, W.I8))
    bad = d(4, 8, W.BF16, W.I8)
    bad.kind = 3
    refused(INVALID, bad)
    with pytest.raises(ValueError):
        d(4, 8, W.BF16, W.I8, "layernorm")


def test_operands_that_are_refused():
    d = R.quant_desc
    plain, norm, gate = (d(4, 8, W.BF16, W.I8, k) for k in ("plain", "rmsnorm", "silu_mul"))
    assert R.lib().frisk_b200_quant_run(None, None) == INVALID
    assert R.lib().frisk_b200_quant_run(C.byref(plain), None) == INVALID
    refused(INVALID, plain, None)
    refused(INVALID, plain, 0x10000, None)
    refused(INVALID, plain, 0x10000, 0x20000, None)
    for name in ("weight", "residual", "up", "sum_out"):      # not an operand of this kind
        refused(INVALID, plain, **{name: 0x40000})
    for name in ("weight", "residual", "sum_out"):
        refused(INVALID, gate, **{name: 0x40000})
    refused(INVALID, norm, up=0x40000)
    refused(INVALID, norm, sum_out=0x40000)                   # a sum of x alone
    refused(MISALIGNED, plain, 0x10001)
    refused(MISALIGNED, plain, scale=0x30002)
    refused(MISALIGNED, norm, weight=0x40001)
    refused(MISALIGNED, norm, residual=0x40001)
    refused(MISALIGNED, norm, residual=0x40000, sum_out=0x50001)
    refused(MISALIGNED, gate, up=0x40001)
    refused(MISALIGNED, d(4, 8, W.BF16, W.I8, "rmsnorm", weight_type=W.F32), weight=0x40002)
    # in place of x or the residual only at the same pitch
    wide = d(4, 8, W.BF16, W.I8, "rmsnorm", ldx=16)
    refused(INVALID, wide, residual=0x40000, sum_out=0x10000)
    wide = d(4, 8, W.BF16, W.I8, "rmsnorm", lds=16)
    refused(INVALID, wide, residual=0x40000, sum_out=0x40000)
    # the outputs lie by themselves
    refused(INVALID, plain, 0x10000, 0x10000)
    refused(INVALID, plain, 0x10000, 0x20000, 0x10000)
    refused(INVALID, plain, 0x10000, 0x20000, 0x20000)
    refused(INVALID, norm, residual=0x20000)
    refused(INVALID, norm, weight=0x30000)
    refused(INVALID, norm, residual=0x40000, sum_out=0x20000)
    # gate and up side by side need rows of twice the width
    refused(INVALID, d(4, 8, W.BF16, W.I8, "silu_mul", ldx=15))


def test_no_rows_is_nothing_to_do():
    R.quant_run(R.quant_desc(0, 8, W.BF16, W.I8), None, None, None)
    q, s = R.quant_host(np.zeros((0, 8), np.uint16), W.BF16, W.E4M3)
    assert q.shape == (0, 8) and s.shape == (0,)


def test_host_form_refuses_wrong_shapes_and_types():
    x = np.zeros((4, 8), np.uint16)
    with pytest.raises(ValueError):
        R.quant_host(x[0], W.BF16, W.I8)
    with pytest.raises(ValueError):
        R.quant_host(x, W.F16, W.I8)
    with pytest.raises(ValueError):
        R.quant_host(x[:, :7], W.BF16, W.I8, "silu_mul")
    with pytest.raises(ValueError):
        R.quant_host(x, W.BF16, W.I8, "rmsnorm", weight=np.zeros(7, np.uint16))
    with pytest.raises(ValueError):
        R.quant_host(x, W.BF16, W.I8, "rmsnorm", residual=np.zeros((4, 9), np.uint16))
    with pytest.raises(ValueError):
        R.quant_host(x, W.BF16, W.I8, "rmsnorm", weight=np.zeros(8, np.uint16), weight_type=W.F32)


@pytest.mark.parametrize("q_type", [W.I8, W.E4M3, W.E5M2])
def test_oracle_rounding_is_the_nearest_stored_number(q_type):
    grid = W.decode(np.arange(256, dtype=np.uint8).view(W.storage_numpy_dtype(q_type)), q_type)
    grid = np.where(np.isfinite(grid), grid, 0).astype(np.float64)
    grid = np.unique(grid[np.abs(grid) <= W.QUANT_MAX[q_type]])
    rng = np.random.default_rng(0)
    v = np.concatenate([rng.uniform(-1.1, 1.1, 4000) * W.QUANT_MAX[q_type], np.exp(rng.uniform(-14, 10, 4000)), grid,
                        (grid[1:] + grid[:-1]) / 2])
    r = ref.round8(v, q_type)
    assert np.isin(r, grid).all()
    near = np.abs(grid[None, :] - v[:, None]).min(axis=1)
    assert np.array_equal(np.abs(r - v), near)
    mid = ref.round8((grid[1:] + grid[:-1]) / 2, q_type)     # ties: the neighbour with the even last bit
    bits = W.encode(mid.astype(np.float32), q_type).view(np.uint8)
    assert (bits & 1 == 0).all()
    assert np.array_equal(W.decode(W.encode(grid.astype(np.float32), q_type), q_type), grid)


def test_oracle_against_a_row_worked_by_hand():
    x = np.array([[3.0, -4.0, 0.0, 0.0]], np.float32)
    v, h = ref.ref_quant(x, W.F32, "rmsnorm", eps=0.0, residual=np.array([[0.0, 0.0, 0.0, 5.0]], np.float32),
                         weight=np.array([1.0, 2.0, 1.0, 0.5], np.float32))
    assert np.array_equal(h, [[3.0, -4.0, 0.0, 5.0]])
    rms = np.sqrt(50.0 / 4.0)
    np.testing.assert_allclose(v, np.array([[3.0, -8.0, 0.0, 2.5]]) / rms, rtol=1e-15)
    s = ref.quant_scale(v, W.I8)
    np.testing.assert_allclose(s, [8.0 / rms / 127.0], rtol=1e-15)
    assert np.array_equal(ref.round8(v / s[:, None], W.I8), [[48.0, -127.0, 0.0, 40.0]])  # 47.625, 39.6875
    v, _ = ref.ref_quant(np.array([[0.0, np.log(3.0), 2.0, 8.0]], np.float64).astype(np.float32), W.F32, "silu_mul")
    np.testing.assert_allclose(v, [[0.0, np.log(3.0) * 0.75 * 8.0]], rtol=1e-6)
    assert ref.quant_scale(np.zeros((1, 3)), W.E4M3)[0] == 2.0 ** -126
