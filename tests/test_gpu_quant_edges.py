"""GPU checks of the 8-bit row makers where their arithmetic is at its limits: rows of the smallest
numbers, ties, sums that leave fp32, gates far out.  Every case runs through each kernel that a width
and an alignment choose; inputs are fp32 unless the case needs another type.  Tolerances are those of
test_gpu_quant.py (u = 2^-24) unless a test derives its own."""
import numpy as np
import pytest

from frisk_b200 import runtime as R
from frisk_b200 import workloads as W
from oracle import ref
from test_gpu_quant import IN_TYPES, Q_TYPES, check_q, ids

pytestmark = pytest.mark.gpu

# in registers; off the 16-byte grid; two passes over aligned rows; element by element
WIDTHS = [64, 1024, 1001, 40000, 40001]
STEP = 2.0 ** -149   # fp32's smallest number


@pytest.mark.parametrize("q_type", Q_TYPES, ids=ids)
@pytest.mark.parametrize("cols", WIDTHS)
def test_norms_of_the_smallest_numbers(cols, q_type):
    """Rows of a few thousand of fp32's smallest steps, whose 8-bit scale is still a regular number:
    with eps = 1e-10 a norm multiplies them by 1e5.  Nothing is rounded on the way to max |g| (no
    weight), so q and the scale keep the tolerances of ordinary rows."""
    top = {W.I8: 10710, W.E4M3: 37800, W.E5M2: 4838300}[q_type]   # the scale is about 1.18e-38, 2^-126 = 1.175e-38
    rng = np.random.default_rng(cols)
    n = rng.integers(-top, top + 1, (4, cols))
    n[:, cols // 2] = top
    n[1, cols // 3] = -top
    x = (n.astype(np.float64) * STEP).astype(np.float32)
    v, _ = ref.ref_quant(x, W.F32, "rmsnorm", eps=1e-10)
    assert (ref.quant_scale(v, q_type) > 2.0 ** -126).all()
    q, s = R.quant_host(x, W.F32, q_type, "rmsnorm", eps=1e-10)
    check_q(q, s, v, "rmsnorm", q_type)
    assert (W.decode(q, q_type)[:, cols // 2] == W.QUANT_MAX[q_type]).all()


@pytest.mark.parametrize("q_type", Q_TYPES, ids=ids)
@pytest.mark.parametrize("in_type", [W.F16, W.BF16], ids=ids)
@pytest.mark.parametrize("rows,cols", [(64, 64), (700, 1024), (700, 1001), (40, 3001), (3, 40000), (3, 40001)])
def test_ties_of_16_bit_rows_fall_as_defined(rows, cols, in_type, q_type):
    """q is the rounding of v Q / max |v|, ties to even, for 16-bit rows WITHOUT any allowance: with v = a 2^i
    and max = b 2^j, a and b whole numbers below 2^11, and Q = 127, 7 * 2^6 or 7 * 2^13, the quotient and a
    border between two 8-bit numbers, an odd number below 2^8 times a power of two, differ by a whole number
    over 255 * 2047 of the larger at least, if they differ: 2^-19, and the quotient is good to 2^-23.  The
    values are multiples of a few steps, so that many quotients are borders."""
    rng = np.random.default_rng([7, rows, cols, in_type])
    x = (rng.integers(-64, 65, (rows, cols)) * 2.0 ** rng.integers(-6, 7, (rows, 1))).astype(np.float32)
    x[rows // 2:] = (rng.standard_normal((rows - rows // 2, cols)) * 3).astype(np.float32)
    x = W.encode(x, in_type)
    v, _ = ref.ref_quant(x, in_type, "plain")
    want = ref.quant_scale(v, q_type)
    q, s = R.quant_host(x, in_type, q_type)
    got = W.decode(q, q_type).astype(np.float64)
    t = v * W.QUANT_MAX[q_type] / np.abs(v).max(axis=1)[:, None]   # one rounding of a short product's quotient
    bad = got != ref.round8(t, q_type)
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} values, first at {tuple(np.argwhere(bad)[0])}"
    assert (np.abs(s - want) <= 2.0 ** -24 * want).all()


def borders(q_type):
    """The numbers half way between two neighbours of an 8-bit type (positive)."""
    codes = np.arange(256, dtype=np.uint8).view(W.storage_numpy_dtype(q_type))
    with np.errstate(invalid="ignore"):
        grid = W.decode(codes, q_type).astype(np.float64)
    grid = np.unique(grid[np.isfinite(grid) & (grid >= 0) & (grid <= W.QUANT_MAX[q_type])])
    return (grid[1:] + grid[:-1]) / 2


@pytest.mark.parametrize("q_type", Q_TYPES, ids=ids)
@pytest.mark.parametrize("rows,cols", [(64, 64), (700, 1024), (700, 1001), (40, 3001), (3, 40000), (3, 40001)])
def test_fp32_rows_next_to_borders_round_exactly(rows, cols, q_type):
    """fp32 rows as they are, with most elements within a few of fp32's steps of a border between two 8-bit
    numbers: q is the rounding of the exact v Q / max |v|, without any allowance.  float64 decides that
    exactly too: v Q is exact in it, and a quotient that is not a border differs from one by 2^-32 at least."""
    rng = np.random.default_rng([8, rows, cols])
    top = rng.uniform(1, 2, (rows, 1)).astype(np.float32) * np.exp2(rng.integers(-60, 60, (rows, 1))).astype(np.float32)
    at = rng.choice(borders(q_type), (rows, cols)) * top.astype(np.float64) / W.QUANT_MAX[q_type]
    x = at.astype(np.float32)
    x = (x.view(np.int32) + rng.integers(-2, 3, x.shape)).astype(np.int32).view(np.float32)
    x = np.clip(x * rng.choice([-1, 1], x.shape).astype(np.float32), -top, top)
    x[:, cols // 2] = top[:, 0]
    t = x.astype(np.float64) * W.QUANT_MAX[q_type] / top.astype(np.float64)
    q, s = R.quant_host(x, W.F32, q_type)
    got = W.decode(q, q_type).astype(np.float64)
    bad = got != ref.round8(t, q_type)
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} values, first at {tuple(np.argwhere(bad)[0])}"


@pytest.mark.parametrize("q_type", Q_TYPES, ids=ids)
@pytest.mark.parametrize("cols", [512] + WIDTHS)
def test_rows_whose_squares_overflow_have_zeros_beside_their_scale(cols, q_type):
    """A norm past fp32: NaN for the scale, zeros for q (also where the weight takes the row to zero)."""
    x = np.random.default_rng(cols).uniform(1, 2, (4, cols)).astype(np.float32)
    x[0] *= 1e25
    x[1, cols - 1] = 3e38
    x[2, 0] = -1e20
    w = np.ones(cols, np.float32)
    for weight in (None, w, 0 * w):
        q, s = R.quant_host(x, W.F32, q_type, "rmsnorm", weight=weight)
        assert np.isnan(s[:3]).all() and not q[:3].any()
        assert np.isfinite(s[3]) and bool(q[3].any()) == (weight is None or bool(weight.any()))


@pytest.mark.parametrize("cols", [1, 17, 64, 1000])
def test_eps_as_large_as_fp32_allows(cols):
    """mean + eps may leave fp32's range although neither does: the factor 1 / rms is that of the sum."""
    eps = 3.4e38
    x = np.random.default_rng(cols).uniform(0.5, 1, (3, cols)).astype(np.float32)
    x *= np.float32(1.8e19 / np.sqrt(cols))
    v, _ = ref.ref_quant(x, W.F32, "rmsnorm", eps=eps)
    for q_type in Q_TYPES:
        q, s = R.quant_host(x, W.F32, q_type, "rmsnorm", eps=eps)
        check_q(q, s, v, "rmsnorm", q_type)


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-13, 1e-10])
@pytest.mark.parametrize("cols", [1] + WIDTHS)
def test_norms_of_rows_whose_squares_fp32_does_not_hold(cols, eps):
    """eps down to zero with rows from 1e-44 to 1e15 times a normal one: the norm is that of the row,
    and a row of zeros has q = 0 and the scale 2^-126."""
    rng = np.random.default_rng([cols, 3])
    tops = [0.0, 1e-44, 1e-39, 1e-30, 1e-24, 1e-22, 1e-19, 1e-14, 1e-8, 1e-6, 1e-5, 1e-3, 1.0, 1e6, 1e15]
    x = (rng.standard_normal((len(tops), cols)) * np.array(tops)[:, None]).astype(np.float32)
    x[:, 0] = np.where(x[:, 0] == 0, np.array(tops, np.float32), x[:, 0])
    r = (rng.standard_normal(x.shape) * np.array(tops)[:, None]).astype(np.float32)
    w = (1 + 0.2 * rng.standard_normal(cols)).astype(np.float32)
    for q_type in (W.I8, W.E4M3):
        v, h = ref.ref_quant(x, W.F32, "rmsnorm", eps=eps, residual=r, weight=w)
        q, s, total = R.quant_host(x, W.F32, q_type, "rmsnorm", eps=eps, residual=r, weight=w, want_sum=True)
        h32 = x + r
        assert np.array_equal(total, h32)
        assert s[0] == np.float32(2.0 ** -126) and not W.decode(q[0], q_type).any()   # (-0 stays -0)
        # h is rounded once; below 2^-126 by up to half a step of 2^-149, like h * weight where the rows'
        # factor 1 / rms is at most 2^20 (beyond that the product is not rounded)
        h64 = h32.astype(np.float64)
        live = h64.any(axis=1)
        rstd = np.where(live, 1 / np.sqrt(np.where(live, np.mean(h64 * h64, axis=1) + np.float64(np.float32(eps)), 1)), 0)
        v = h64 * rstd[:, None] * w
        want = ref.quant_scale(v, q_type)
        terms = cols / 32 + 1 + 37
        slack = np.where(rstd <= 2.0 ** 20, 2.0 ** -150 * rstd, 0.0)
        err = np.abs(s.astype(np.float64) - want)
        assert (err <= (terms / 2 + 9) * 2.0 ** -24 * want + slack / W.QUANT_MAX[q_type])[live].all(), (err / want)[live]
        t = v / want[:, None]
        a = np.abs(t) * 7 * 2.0 ** -24 + 2 * (slack / want)[:, None]
        lo, hi = ref.round8(t - a, q_type), ref.round8(t + a, q_type)
        clamped = want <= 2.0 ** -126 * (1 + 2.0 ** -20)   # the stored scale is the least one: v's own error shows
        got = W.decode(q, q_type).astype(np.float64)
        bad = ~((got >= lo) & (got <= hi)) & (live & ~clamped)[:, None]
        assert not bad.any(), np.unique(np.argwhere(bad)[:, 0])
        step = np.where(np.abs(t) < 1, 1, np.abs(t)) * (terms / 2 + 16) * 2.0 ** -24 + a
        lo, hi = ref.round8(t - step, q_type), ref.round8(t + step, q_type)
        assert (((got >= lo) & (got <= hi)) | ~(live & clamped)[:, None]).all()


@pytest.mark.parametrize("in_type", IN_TYPES, ids=ids)
@pytest.mark.parametrize("cols", WIDTHS)
def test_eps_zero_with_the_sum_in_place(cols, in_type):
    """Without eps, rows of ordinary and of very small numbers side by side; the sum over x or the residual."""
    import torch
    dev = torch.device("cuda:0")
    rng = np.random.default_rng([cols, 4])
    tops = np.array([1.0, 3e-7, 0.0, 2e-4, 6e-8, 40.0])[:, None]   # (6e-8: fp16's smallest numbers)
    x, r = (W.encode((rng.standard_normal((6, cols)) * tops).astype(np.float32), in_type) for _ in range(2))
    wt = W.encode((1 + 0.2 * rng.standard_normal(cols)).astype(np.float32), in_type)
    v, h = ref.ref_quant(x, in_type, "rmsnorm", eps=0.0, residual=r, weight=wt)
    on = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.uint8)).to(dev)  # noqa: E731
    desc, weight = R.quant_desc(6, cols, in_type, W.I8, "rmsnorm", eps=0.0), on(wt)
    got = []
    for where in ("apart", "x", "residual"):
        bx, br = on(x), on(r)
        total = torch.zeros_like(bx) if where == "apart" else bx if where == "x" else br
        q, s = torch.zeros((6, cols), dtype=torch.int8, device=dev), torch.zeros(6, device=dev)
        R.quant_run(desc, bx, q, s, weight=weight, residual=br, sum_out=total)
        torch.cuda.synchronize()
        got.append((q.cpu().numpy(), s.cpu().numpy(), total.cpu().numpy()))
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert np.array_equal(a, b)
    q, s, _ = got[0]
    live = h.any(axis=1)
    check_q(q[live], s[live], v[live], "rmsnorm", W.I8)
    assert not q[~live].any() and (s[~live] == np.float32(2.0 ** -126)).all()


def far_gates(rows_of, cols, in_type, rng):
    """Rows of gate and up with gates in bands from both ends: (values as stored, names)."""
    bands = [(-88.7, -87.1), (-104.0, -88.8), (-140.0, -100.0), (-90.0, 90.0), (87.0, 300.0), (-190.0, -185.0)]
    gate = np.stack([rng.uniform(*bands[i % len(bands)], cols) for i in range(rows_of)])
    size = 1e4 if in_type == W.F16 else 1e35
    up = rng.uniform(-size, size, (rows_of, cols))
    return W.encode(np.concatenate([gate, up], axis=1).astype(np.float32), in_type), len(bands)


def check_gates(q, s, x, in_type, q_type):
    """As for ordinary gates (v carries 7 u); what leaves fp32's regular numbers on the way is rounded to
    its smallest step once more, half a step of 2^-149."""
    v, _ = ref.ref_quant(x, in_type, "silu_mul")
    want = ref.quant_scale(v, q_type)
    least = 2.0 ** -150
    assert (np.abs(s - want) <= 9 * 2.0 ** -24 * want + least).all(), (s / want)
    t = v / want[:, None]
    a = np.abs(t) * 17 * 2.0 ** -24 + 2 * least / want[:, None]
    lo, hi = ref.round8(t - a, q_type), ref.round8(t + a, q_type)
    got = W.decode(q, q_type).astype(np.float64)
    bad = ~((got >= lo) & (got <= hi))
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} values, first at {tuple(np.argwhere(bad)[0])}"


@pytest.mark.parametrize("q_type", Q_TYPES, ids=ids)
@pytest.mark.parametrize("in_type", IN_TYPES, ids=ids)
@pytest.mark.parametrize("cols", WIDTHS)
def test_gates_far_from_zero(cols, in_type, q_type):
    """exp(-gate) leaves fp32 below -88.7, and its reciprocal the regular numbers below -87.3; the product
    with a large up does not."""
    x, _ = far_gates(12, cols, in_type, np.random.default_rng([cols, 5]))
    q, s = R.quant_host(x, in_type, q_type, "silu_mul")
    check_gates(q, s, x, in_type, q_type)


def test_gates_far_from_zero_in_streamed_rows():
    x, _ = far_gates(4500, 4096, W.BF16, np.random.default_rng(6))
    q, s = R.quant_host(x, W.BF16, W.E4M3, "silu_mul")
    check_gates(q, s, x, W.BF16, W.E4M3)


@pytest.mark.parametrize("q_type", Q_TYPES, ids=ids)
@pytest.mark.parametrize("cols", WIDTHS)
def test_infinite_gates(cols, q_type):
    """gate = infinity times up is an infinity, and so is the row's scale; -infinity * 0 is NaN."""
    x = np.random.default_rng(cols).standard_normal((4, 2 * cols)).astype(np.float32)
    x[0, cols // 2], x[0, cols + cols // 2] = np.inf, 2.0
    x[1, 0] = -np.inf
    x[2, cols - 1] = np.nan
    q, s = R.quant_host(x, W.F32, q_type, "silu_mul")
    assert np.isposinf(s[0]) and np.isnan(s[1:3]).all() and not q[:3].any()
    v, _ = ref.ref_quant(x[3:], W.F32, "silu_mul")
    check_q(q[3:], s[3:], v, "silu_mul", q_type)


@pytest.mark.parametrize("rows,cols,in_type", [(4500, 4096, W.BF16), (1100, 16384, W.BF16), (1500, 12008, W.F16), (800, 28672, W.BF16)],
                         ids=["4500x4096", "1100x16384", "1500x12008", "800x28672"])
def test_streamed_rows_report_a_wait_that_runs_out(rows, cols, in_type):
    """With no time to wait the teams give up on rows whose copies have not landed: the status word says
    so, those rows have NaN scales and zeros, and the launches after it are as ever."""
    import ctypes
    import torch
    dev = torch.device("cuda:0")
    limit = R.lib().frisk_internal_quant_wait_cycles
    limit.argtypes, limit.restype = [ctypes.c_int64], ctypes.c_int64
    dt = torch.bfloat16 if in_type == W.BF16 else torch.float16
    x = torch.randn((rows, 2 * cols), generator=torch.Generator(device=dev).manual_seed(cols), device=dev).to(dt)
    desc = R.quant_desc(rows, cols, in_type, W.I8, "silu_mul")
    status = torch.zeros(1, dtype=torch.int32, device=dev)

    def run():
        q = torch.full((rows, cols), 0x5A, dtype=torch.int8, device=dev)
        s = torch.full((rows,), 7.0, device=dev)
        torch.cuda.synchronize()
        R.quant_run(desc, x, q, s, stream=torch.cuda.current_stream().cuda_stream, status=status)
        torch.cuda.synchronize()
        return q, s

    want_q, want_s = run()
    R.check_status(status)
    before = limit(0)
    try:
        q, s = run()
        with pytest.raises(R.FriskError) as e:
            R.quant_host(x.view(torch.int16).cpu().numpy().view(W.storage_numpy_dtype(in_type)), in_type, W.I8, "silu_mul")
        assert e.value.code == -6
    finally:
        limit(before)
    assert before == 1 << 29
    with pytest.raises(R.FriskError) as e:
        R.check_status(status)
    assert e.value.code == -6 and "0x10" in str(e.value)
    lost = torch.isnan(s)
    assert bool(lost.any()) and not bool(q[lost].any())
    assert torch.equal(q[~lost], want_q[~lost]) and torch.equal(s[~lost], want_s[~lost])
    status.zero_()
    again_q, again_s = run()
    R.check_status(status)
    assert torch.equal(again_q, want_q) and torch.equal(again_s, want_s)
