"""GPU parity of the 8-bit row makers, through the C ABI, against the float64 restatement in
oracle/ref.py on the same seeded inputs.

Tolerances, with u = 2^-24 (half a step of fp32, relative).  The kernel rounds to nearest at every
step, so
  * plain: the scale carries one rounding (1 u); v / scale carries that one and its own (2 u);
  * silu_mul: exp is good to 2 units in the last place (4 u), 1 + exp, the division and the product
    add 1 u each: v carries 7 u, the scale 8 u, v / scale 16 u;
  * rmsnorm: h = x + residual carries 1 u, h * weight 2 u, its maximum over Q 3 u, their quotient 6 u.
    A sum of squares whose terms pass through at most L additions carries (L + 2) u (every term is
    positive), the division by the width, eps, the root (which halves what came before) and the
    reciprocal bring the factor 1 / rms to (L / 2 + 4) u, and the scale to (L / 2 + 8) u.  No thread
    adds more than width / 32 + 1 squares, the tree over at most 32 lanes and 32 warps at most 37 more.
  * sum_out: h is rounded twice, to fp32 and to the stored type: half a step of that type plus 1 u.
Products of the roundings (second order in u) are covered by 1 u on top of each figure.  The 8-bit
value has to be the rounding of SOME number that close to the exact quotient: rounding is monotonic, so
it has to lie between the roundings of the two ends.  The stored scale has to be the row's, and the
scale 2^-126 of a row whose exact scale is smaller."""
import numpy as np
import pytest

from frisk_b200 import runtime as R
from frisk_b200 import workloads as W
from oracle import ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {W.F32: 2.0 ** -24, W.F16: 2.0 ** -11, W.BF16: 2.0 ** -8}
NAMES = {W.F32: "f32", W.F16: "f16", W.BF16: "bf16", W.I8: "i8", W.E4M3: "e4m3", W.E5M2: "e5m2"}
IN_TYPES, Q_TYPES = [W.F32, W.F16, W.BF16], [W.I8, W.E4M3, W.E5M2]
ids = NAMES.get


def inputs(rows, cols, in_type, kind, seed, weight_type=None):
    rng = np.random.default_rng([seed, rows, cols, in_type])
    spread = np.exp(0.5 * rng.standard_normal((1, cols)))

    def values(n=cols):
        return W.encode((rng.standard_normal((rows, n)) * np.resize(spread, (1, n))).astype(np.float32), in_type)

    if kind == "plain":
        return values(), {}
    if kind == "silu_mul":
        return values(2 * cols), {}
    wt = in_type if weight_type is None else weight_type
    return values(), {"residual": values(), "weight": W.encode((1 + 0.2 * rng.standard_normal(cols)).astype(np.float32), wt),
                      "weight_type": wt}


def check_q(q, scale, v, kind, q_type):
    cols = v.shape[1]
    terms = cols / 32 + 1 + 37
    e_scale = {"plain": 1, "silu_mul": 8, "rmsnorm": terms / 2 + 8}[kind] + 1
    e_q = {"plain": 2, "silu_mul": 16, "rmsnorm": 6}[kind] + 1
    want = ref.quant_scale(v, q_type)
    err = np.abs(scale.astype(np.float64) - want)
    assert (err <= e_scale * U * want).all(), f"scale off by {(err / want).max() / U:.1f} u"
    t = v / want[:, None]
    lo, hi = ref.round8(t - np.abs(t) * e_q * U, q_type), ref.round8(t + np.abs(t) * e_q * U, q_type)
    got = W.decode(q, q_type).astype(np.float64)
    bad = ~((got >= lo) & (got <= hi))
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} values, first at {tuple(np.argwhere(bad)[0])}"


def check_sum(total, h, in_type):
    got = W.decode(total, in_type).astype(np.float64)
    least = {W.F32: 2.0 ** -150, W.F16: 2.0 ** -25, W.BF16: 2.0 ** -134}[in_type]   # half of the smallest step
    assert (np.abs(got - h) <= (HALF_STEP[in_type] + 2 * U) * np.abs(h) + least).all()


SHAPES = [(1, 1), (2, 3), (3, 8), (5, 31), (4, 128), (7, 257), (3, 1000), (33, 1024), (2, 4096), (3, 5001), (2, 8192),
          (2, 16384), (1, 20008), (1, 33000), (1, 70000)]


@pytest.mark.parametrize("q_type", Q_TYPES, ids=ids)
@pytest.mark.parametrize("in_type", IN_TYPES, ids=ids)
@pytest.mark.parametrize("kind", ["plain", "rmsnorm", "silu_mul"])
@pytest.mark.parametrize("rows,cols", SHAPES, ids=[f"{r}x{c}" for r, c in SHAPES])
def test_rows_match_the_oracle(rows, cols, kind, in_type, q_type):
    x, kw = inputs(rows, cols, in_type, kind, 1)
    v, h = ref.ref_quant(x, in_type, kind, **kw)
    got = R.quant_host(x, in_type, q_type, kind, want_sum=kind == "rmsnorm", **kw)
    check_q(got[0], got[1], v, kind, q_type)
    if kind == "rmsnorm":
        check_sum(got[2], h, in_type)


@pytest.mark.parametrize("rows,cols", [(3, 7), (2, 1024), (2, 4100), (1, 40000)])
@pytest.mark.parametrize("in_type", IN_TYPES, ids=ids)
def test_norm_without_residual_or_weight_and_with_an_fp32_weight(rows, cols, in_type):
    x, kw = inputs(rows, cols, in_type, "rmsnorm", 2, W.F32)
    for drop in ((), ("residual",), ("weight",), ("residual", "weight")):
        k = {n: a for n, a in kw.items() if n not in drop}
        v, _ = ref.ref_quant(x, in_type, "rmsnorm", eps=1e-3, **k)
        q, s = R.quant_host(x, in_type, W.E4M3, "rmsnorm", eps=1e-3, **k)
        check_q(q, s, v, "rmsnorm", W.E4M3)


@pytest.mark.parametrize("cols", [5, 1024, 3001])
def test_up_as_a_matrix_of_its_own(cols):
    x, _ = inputs(3, cols, W.BF16, "plain", 3)
    up, _ = inputs(3, cols, W.BF16, "plain", 4)
    v, _ = ref.ref_quant(x, W.BF16, "silu_mul", up=up)
    q, s = R.quant_host(x, W.BF16, W.I8, "silu_mul", up=up)
    check_q(q, s, v, "silu_mul", W.I8)
    both = R.quant_host(np.concatenate([x, up], axis=1), W.BF16, W.I8, "silu_mul")
    assert np.array_equal(q, both[0]) and np.array_equal(s, both[1])


@pytest.mark.parametrize("q_type", Q_TYPES, ids=ids)
@pytest.mark.parametrize("cols", [9, 1024, 9000])
@pytest.mark.parametrize("kind", ["plain", "rmsnorm", "silu_mul"])
def test_rows_of_zeros_tiny_rows_and_rows_that_are_not_finite(kind, cols, q_type):
    x, kw = inputs(8, cols, W.F32, kind, 5)
    kw.pop("residual", None)
    width = x.shape[1]
    x[0] = 0.0
    x[1] *= 1e-30 if kind == "rmsnorm" else 1e-38 if kind == "plain" else 1e-20
    x[2] *= 1e-18 if kind == "silu_mul" else 1e-44
    x[3] = np.where(np.arange(width) % 2, 1.0, -1.0)
    x[4, width - 1] = np.inf
    x[5, 0] = np.nan
    x[6, cols // 2] = -np.inf
    v, _ = ref.ref_quant(x, W.F32, kind, **kw)
    q, s = R.quant_host(x, W.F32, q_type, kind, **kw)
    check_rows = [0, 3, 7] + ([1] if kind != "silu_mul" else [])
    check_q(q[check_rows], s[check_rows], v[check_rows], kind, q_type)
    with np.errstate(invalid="ignore"):
        got = W.decode(q, q_type).astype(np.float64) * s.astype(np.float64)[:, None]
    # row 2 is below what a scale of 2^-126 resolves (or close to it): within one step of that scale
    assert np.isfinite(s[:4]).all() and (s[:4] >= np.float32(2.0 ** -126)).all()
    assert (np.abs(got[2] - v[2]) <= np.maximum(s[2] * 0.5, np.abs(v[2]) * 2.0 ** -2) + 2.0 ** -140).all()
    assert not got[0].any()
    for r in (4, 5, 6):
        assert not np.isfinite(s[r]) and not q[r].any(), r


def test_squares_past_fp32_give_no_silent_scale():
    x = np.full((2, 512), 1e25, np.float32)
    x[1] = 1e15
    q, s = R.quant_host(x, W.F32, W.I8, "rmsnorm")
    assert np.isnan(s[0]) and abs(float(s[1]) * 127 - 1) < 1e-5 and (q[1] == 127).all()


def test_nan_and_infinity_in_sum_weight_and_gate():
    x, kw = inputs(4, 64, W.F16, "rmsnorm", 6)
    kw["residual"][1, 3] = np.inf
    kw["weight"][5] = 0
    q, s, h = R.quant_host(x, W.F16, W.E4M3, "rmsnorm", want_sum=True, **kw)
    assert np.isfinite(s[[0, 2, 3]]).all() and not np.isfinite(s[1])
    assert np.isinf(h[1, 3]) and (W.decode(q[[0, 2, 3]], W.E4M3)[:, 5] == 0).all()
    x, _ = inputs(2, 64, W.BF16, "silu_mul", 7)
    vals = W.decode(x, W.BF16)
    vals[0, 3] = -300.0    # exp overflows: silu is -0, not NaN
    vals[0, 7] = 300.0
    x = W.encode(vals, W.BF16)
    v, _ = ref.ref_quant(x, W.BF16, "silu_mul")
    q, s = R.quant_host(x, W.BF16, W.I8, "silu_mul")
    check_q(q, s, v, "silu_mul", W.I8)


@pytest.mark.parametrize("cols", [1, 40, 1023, 2048, 4097])
@pytest.mark.parametrize("in_type", IN_TYPES, ids=ids)
@pytest.mark.parametrize("kind", ["plain", "rmsnorm", "silu_mul"])
def test_pitches_offsets_and_untouched_padding(kind, in_type, cols):
    """Device buffers at any alignment and pitch; everything around the rows stays as it was."""
    import torch
    dev = torch.device("cuda:0")
    rows, es = 5, W.ELEM_SIZE[in_type]
    x, kw = inputs(rows, cols, in_type, kind, 8)
    v, h = ref.ref_quant(x, in_type, kind, **kw)

    def place(a, ld, shift, size):
        """`a` at element offset `shift` and pitch `ld` of a buffer of 0x5a bytes."""
        n = (rows - 1) * ld + a.shape[1]
        host = np.full((n + shift + 16) * size, 0x5A, np.uint8)
        view = host[shift * size:(shift + n) * size]
        for r in range(rows):
            view[r * ld * size:(r * ld + a.shape[1]) * size] = np.ascontiguousarray(a[r]).view(np.uint8)
        return torch.from_numpy(host).to(dev)

    def rows_of(buf, ld, shift, size, width):
        host = buf.cpu().numpy()
        out = np.stack([host[(shift + r * ld) * size:(shift + r * ld + width) * size] for r in range(rows)])
        for r in range(rows):
            host[(shift + r * ld) * size:(shift + r * ld + width) * size] = 0x5A
        assert (host == 0x5A).all(), "bytes outside the rows were written"
        return out

    for pad, shift in ((0, 0), (1, 1), (8, 8), (16, 3), (5, 2)):
        ldx, ldo, lds, ldq = x.shape[1] + pad, cols + 2 * pad, cols + pad, cols + pad
        desc = R.quant_desc(rows, cols, in_type, W.I8, kind, ldx=ldx, ldo=ldo if kind == "rmsnorm" else 0,
                            lds=lds if kind == "rmsnorm" else 0, ldq=ldq)
        bx = place(x, ldx, shift, es)
        bq = torch.full(((rows - 1) * ldq + cols + shift + 16,), 0x5A, dtype=torch.uint8, device=dev)
        bs = torch.full((rows + 2,), 7.0, device=dev)
        extra = {}
        if kind == "rmsnorm":
            br = place(kw["residual"], ldo, shift, es)
            bw = torch.from_numpy(np.ascontiguousarray(kw["weight"]).view(np.uint8)).to(dev)
            bh = torch.full((((rows - 1) * lds + cols + shift + 16) * es,), 0x5A, dtype=torch.uint8, device=dev)
            extra = dict(residual=br.data_ptr() + shift * es, weight=bw, sum_out=bh.data_ptr() + shift * es)
        R.quant_run(desc, bx.data_ptr() + shift * es, bq.data_ptr() + shift, bs[1:], stream=torch.cuda.current_stream().cuda_stream, **extra)
        torch.cuda.synchronize()
        s = bs.cpu().numpy()
        assert s[0] == 7.0 and s[-1] == 7.0
        q = rows_of(bq, ldq, shift, 1, cols).view(np.int8)
        check_q(q, s[1:-1], v, kind, W.I8)
        if kind == "rmsnorm":
            check_sum(rows_of(bh, lds, shift, es, cols).view(x.dtype), h, in_type)
            for place_ in ("x", "residual"):     # the sum in place of an addend: same bits
                at, ld = (bx.data_ptr(), ldx) if place_ == "x" else (br.data_ptr(), ldo)
                keep = (bx if place_ == "x" else br).clone()
                q2, s2 = torch.full_like(bq, 0x5A), torch.zeros(rows, device=dev)
                desc2 = R.quant_desc(rows, cols, in_type, W.I8, kind, ldx=ldx, ldo=ldo, lds=ld, ldq=ldq)
                R.quant_run(desc2, bx.data_ptr() + shift * es, q2.data_ptr() + shift, s2, **dict(extra, sum_out=at + shift * es))
                torch.cuda.synchronize()
                assert np.array_equal(s2.cpu().numpy(), s[1:-1])
                assert np.array_equal(rows_of(q2, ldq, shift, 1, cols).view(np.int8), q)
                buf = bx if place_ == "x" else br
                check_sum(rows_of(buf, ld, shift, es, cols).view(x.dtype), h, in_type)
                buf.copy_(keep)


def test_many_short_rows_and_repeatable_bits():
    x, kw = inputs(5000, 24, W.BF16, "rmsnorm", 9)
    v, h = ref.ref_quant(x, W.BF16, "rmsnorm", **kw)
    a = R.quant_host(x, W.BF16, W.E4M3, "rmsnorm", want_sum=True, **kw)
    b = R.quant_host(x, W.BF16, W.E4M3, "rmsnorm", want_sum=True, **kw)
    for p, q in zip(a, b):
        assert np.array_equal(p, q)
    check_q(a[0], a[1], v, "rmsnorm", W.E4M3)
    check_sum(a[2], h, W.BF16)


def test_captured_into_a_graph_and_on_another_stream():
    import torch
    dev = torch.device("cuda:0")
    rows, cols = 16, 2048
    desc = R.quant_desc(rows, cols, W.BF16, W.I8, "silu_mul")
    x = torch.zeros((rows, 2 * cols), dtype=torch.int16, device=dev)
    q = torch.zeros((rows, cols), dtype=torch.int8, device=dev)
    s = torch.zeros((rows,), device=dev)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        R.quant_run(desc, x, q, s, stream=side.cuda_stream)
    for seed in (10, 11):
        host, _ = inputs(rows, cols, W.BF16, "silu_mul", seed)
        x.copy_(torch.from_numpy(host.view(np.int16)))
        graph.replay()
        torch.cuda.synchronize()
        v, _ = ref.ref_quant(host, W.BF16, "silu_mul")
        check_q(q.cpu().numpy(), s.cpu().numpy(), v, "silu_mul", W.I8)


@pytest.mark.parametrize("q_type", [W.I8, W.E4M3], ids=ids)
@pytest.mark.parametrize("rows,cols,in_type", [(600, 3080, W.BF16), (1500, 4096, W.F32), (1201, 3336, W.F16), (640, 8192, W.BF16),
                                               (601, 16384, W.F32), (700, 16384, W.BF16),
                                               (400, 40000, W.BF16), (5, 53248, W.F32), (3, 40001, W.F16)],
                         ids=["600x3080", "1500x4096", "1201x3336", "640x8192", "601x16384", "700x16384", "400x40000", "5x53248", "3x40001"])
@pytest.mark.parametrize("kind", ["plain", "rmsnorm", "silu_mul"])
def test_many_wide_rows(kind, rows, cols, in_type, q_type):
    many_rows(kind, rows, cols, in_type, q_type)


@pytest.mark.parametrize("rows,cols,in_type,q_type", [(1100, 16384, W.BF16, W.E4M3), (1500, 12008, W.F16, W.I8), (1101, 8192, W.F32, W.E5M2),
                                                      (4500, 4096, W.BF16, W.I8)],
                         ids=["1100x16384", "1500x12008", "1101x8192", "4500x4096"])
def test_gated_rows_streamed_through_shared_memory(rows, cols, in_type, q_type):
    many_rows("silu_mul", rows, cols, in_type, q_type)


def many_rows(kind, rows, cols, in_type, q_type):
    """More rows than the device holds at once, run three times: the same bits each time."""
    import torch
    dev = torch.device("cuda:0")
    x, kw = inputs(rows, cols, in_type, kind, 12)
    kw.pop("weight_type", None)
    on = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.uint8)).to(dev)  # noqa: E731
    bx, extra = on(x), {n: on(a) for n, a in kw.items()}
    runs = []
    for _ in range(3):
        q = torch.zeros((rows, cols), dtype=torch.uint8, device=dev)
        s = torch.zeros(rows, device=dev)
        h = torch.zeros((rows, cols * W.ELEM_SIZE[in_type]), dtype=torch.uint8, device=dev) if kind == "rmsnorm" else None
        R.quant_run(R.quant_desc(rows, cols, in_type, q_type, kind), bx, q, s, sum_out=h, **extra)
        runs.append((q, s, h))
    torch.cuda.synchronize()
    for q, s, h in runs[1:]:
        assert torch.equal(q, runs[0][0]) and torch.equal(s, runs[0][1]) and (h is None or torch.equal(h, runs[0][2]))
    v, hw = ref.ref_quant(x, in_type, kind, **kw)
    q, s, h = runs[0]
    check_q(q.cpu().numpy().view(W.storage_numpy_dtype(q_type)), s.cpu().numpy(), v, kind, q_type)
    if kind == "rmsnorm":
        check_sum(h.cpu().numpy().view(x.dtype), hw, in_type)


@pytest.mark.parametrize("cols", [1000, 1001, 4096, 40000])
@pytest.mark.parametrize("in_type", [W.F32, W.BF16], ids=ids)
def test_many_rows_with_the_sum_in_place(in_type, cols):
    """The sum over x, then over the residual, of many packed rows: what separate buffers give."""
    import torch
    dev = torch.device("cuda:0")
    rows = 700 if cols < 40000 else 40
    x, kw = inputs(rows, cols, in_type, "rmsnorm", 15)
    on = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.uint8)).to(dev)  # noqa: E731
    weight, desc = on(kw["weight"]), R.quant_desc(rows, cols, in_type, W.E4M3, "rmsnorm")
    got = []
    for where in ("apart", "x", "residual"):
        bx, br = on(x), on(kw["residual"])
        h = torch.zeros_like(bx) if where == "apart" else bx if where == "x" else br
        q, s = torch.zeros((rows, cols), dtype=torch.uint8, device=dev), torch.zeros(rows, device=dev)
        R.quant_run(desc, bx, q, s, weight=weight, residual=br, sum_out=h)
        torch.cuda.synchronize()
        got.append((q, s, h))
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)
    v, h = ref.ref_quant(x, in_type, "rmsnorm", **kw)
    check_q(got[0][0].cpu().numpy(), got[0][1].cpu().numpy(), v, "rmsnorm", W.E4M3)
    check_sum(got[0][2].cpu().numpy().view(x.dtype).reshape(h.shape), h, in_type)


def test_streamed_rows_captured_into_a_graph():
    import torch
    dev = torch.device("cuda:0")
    rows, cols = 1200, 16384
    desc = R.quant_desc(rows, cols, W.BF16, W.E4M3, "silu_mul")
    x = torch.zeros((rows, 2 * cols), dtype=torch.bfloat16, device=dev)
    q, s = torch.zeros((rows, cols), dtype=torch.uint8, device=dev), torch.zeros(rows, device=dev)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        R.quant_run(desc, x, q, s, stream=side.cuda_stream)
    for seed in (1, 2):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev))
        q2, s2 = torch.zeros_like(q), torch.zeros_like(s)
        R.quant_run(desc, x, q2, s2, stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, q2) and torch.equal(s, s2) and bool((s > 0).all())


@pytest.mark.parametrize("cols", [32768, 32761])
def test_offsets_past_32_bits(cols):
    """More than 2^31 elements (and 2^32 bytes) in x and more than 2^31 bytes in q: the last rows."""
    import torch
    dev = torch.device("cuda:0")
    rows = 66000
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device=dev)
    q = torch.full((rows, cols), 0x5A, dtype=torch.uint8, device=dev)
    s = torch.zeros(rows, device=dev)
    pick = [0, 1, 65535, 65536, rows - 2, rows - 1]
    host, _ = inputs(len(pick), cols, W.BF16, "plain", 16)
    x[pick] = torch.from_numpy(host.view(np.int16)).view(torch.bfloat16).to(dev)
    R.quant_run(R.quant_desc(rows, cols, W.BF16, W.I8), x, q, s)
    torch.cuda.synchronize()
    v, _ = ref.ref_quant(host, W.BF16, "plain")
    check_q(q[pick].cpu().numpy().view(np.int8), s[pick].cpu().numpy(), v, "plain", W.I8)
    q[pick] = 0
    assert not bool(q.any()) and int((s == 2.0 ** -126).sum()) == rows - len(pick)
