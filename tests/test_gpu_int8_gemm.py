"""GPU parity of the 8-bit integer gemm, through the C ABI, against the exact product.

The sums are exact in the kernels (32-bit integers) and in the reference (float64: every partial sum
is below 2^31).  With u = 2^-24: the conversion of the sum to fp32 and the products with the two scales
round once each (3 u of the product), adding the old C once more (1 u of the result), and storing
rounds to half a step of C's type.  So |got - want| <= 4 u (|product| + |want|) + half a step at want,
and an fp32 C without scales is off by the conversion alone."""
import numpy as np
import pytest

from frisk_b200 import runtime as R
from frisk_b200 import workloads as W
from oracle import ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {W.F32: 2.0 ** -24, W.F16: 2.0 ** -11, W.BF16: 2.0 ** -8}
LEAST = {W.F32: 2.0 ** -150, W.F16: 2.0 ** -25, W.BF16: 2.0 ** -134}


def make(M, N, K, seed=0, full=False):
    rng = np.random.default_rng([seed, M, N, K])
    if full:   # the whole range of the type, -128 too
        a, b = (rng.integers(-128, 128, s, dtype=np.int8) for s in ((M, K), (K, N)))
    else:
        a, b = (np.clip(np.rint(rng.standard_normal(s) * 30), -127, 127).astype(np.int8) for s in ((M, K), (K, N)))
    sa = (rng.uniform(0.5, 2.0, M) / 127).astype(np.float32)
    sb = (rng.uniform(0.5, 2.0, N) / 127).astype(np.float32)
    return a, b, sa, sb


def stored(a, trans, pitch_pad=0):
    """The matrix in its memory order, rows `pitch_pad` elements apart from packed; (buffer, pitch)."""
    m = np.ascontiguousarray(a.T if trans else a)
    if pitch_pad:
        m = np.concatenate([m, np.full((m.shape[0], pitch_pad), 99, np.int8)], axis=1)
    return np.ascontiguousarray(m), m.shape[1]


def expect(a, b, sa=None, sb=None, c0=None):
    prod = a.astype(np.float64) @ b.astype(np.float64)
    if sa is not None:
        prod = prod * sa.astype(np.float64)[:, None] * sb.astype(np.float64)[None, :]
    return prod, prod if c0 is None else prod + c0


def check(got, prod, want, ct, scaled=True):
    g = W.decode(got, ct).astype(np.float64)
    tol = 4 * U * (np.abs(prod) + np.abs(want)) + HALF_STEP[ct] * np.abs(want) + LEAST[ct]
    bad = ~(np.abs(g - want) <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} off, first at {tuple(np.argwhere(bad)[0])}: {g[bad][0]} for {want[bad][0]}"


def run(M, N, K, ct=W.BF16, ta=False, tb=True, clear=True, scales=True, pad=(0, 0), seed=0, full=False, kernel=None, **kw):
    a, b, sa, sb = make(M, N, K, seed, full)
    A, lda = stored(a, ta, pad[0])
    B, ldb = stored(b, tb, pad[1])
    c = np.zeros((M, N), W.storage_numpy_dtype(ct))
    c0 = None
    if not clear:
        c[...] = W.encode(np.random.default_rng(seed + 1).standard_normal((M, N)).astype(np.float32), ct)
        c0 = W.decode(c, ct).astype(np.float64)
    plan = R.GemmPlan(M, N, K, W.I8, ct, transA=ta, transB=tb, clear_accum=clear, scales=scales, lda=lda, ldb=ldb, **kw)
    info = plan.info
    plan.run_host(A, B, c, sa if scales else None, sb if scales else None)
    plan.close()
    prod, want = expect(a, b, sa if scales else None, sb if scales else None, c0)
    check(c, prod, want, ct)
    if kernel:
        assert info["kernel_name"] == kernel, info
    return info


SIZES = [(1, 1, 1), (1, 1, 300), (3, 5, 7), (17, 33, 100), (64, 64, 64), (1, 300, 130), (130, 257, 129), (300, 520, 272)]


@pytest.mark.parametrize("ct", [W.F32, W.F16, W.BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("ta,tb", [(False, True), (False, False), (True, True), (True, False)], ids=["nt", "nn", "tt", "tn"])
@pytest.mark.parametrize("M,N,K", SIZES, ids=["x".join(map(str, s)) for s in SIZES])
def test_every_order_and_result_type(M, N, K, ta, tb, ct):
    run(M, N, K, ct, ta, tb, seed=1)
    run(M, N, K, ct, ta, tb, clear=False, pad=(3, 5), seed=2)


@pytest.mark.parametrize("M,N,K", [(5, 70, 200), (40, 300, 512), (200, 300, 1000)])
def test_without_scales_and_over_the_whole_range(M, N, K):
    a, b, _, _ = make(M, N, K, 3, full=True)
    c = np.zeros((M, N), np.float32)
    plan = R.GemmPlan(M, N, K, W.I8, W.F32, transB=True)
    plan.run_host(a, np.ascontiguousarray(b.T), c)
    plan.close()
    want = a.astype(np.int64) @ b.astype(np.int64)
    assert np.array_equal(c, want.astype(np.float32))     # one rounding to fp32, of the exact sum
    run(M, N, K, W.F16, seed=4, full=True, clear=False)


def test_the_longest_sums_do_not_overflow():
    M, N, K = 3, 260, 131071
    a = np.full((M, K), -128, np.int8)
    b = np.full((K, N), -128, np.int8)
    a[1], b[:, 7] = 127, 127
    c = np.zeros((M, N), np.float32)
    plan = R.GemmPlan(M, N, K, W.I8, W.F32, transB=True)
    plan.run_host(a, np.ascontiguousarray(b.T), c)
    plan.close()
    assert np.array_equal(c, (a.astype(np.int64) @ b.astype(np.int64)).astype(np.float32))


def test_through_the_ir_builder():
    import frisk as F
    M, N, K = 200, 300, 160
    a, b, sa, sb = make(M, N, K, 5)
    h = F.create_session()
    f32 = h.builder.get_f32_ty()
    tys = [h.memref_type((M, K), "int8"), h.memref_type((K, N), "int8"), h.memref_type((M, N), "bf16"),
           h.memref_type((M,), f32), h.memref_type((N,), f32)]
    _, entry = h.new_kernel("k", tys)
    v = [entry.get_argument(i) for i in range(5)]
    h.builder.create_gemm_op(v[0], v[1], v[2], False, True, True, v[3], v[4])
    assert h.module.verify(), h.module.verify_message()
    out = np.zeros((M, N), np.uint16)
    F.run(str(h.module), "k", [a, np.ascontiguousarray(b.T), out, sa, sb])     # through the textual form
    check(out, *expect(a, b, sa, sb), W.BF16)


def test_oracle_agrees_with_the_exact_product():
    a, b, sa, sb = make(33, 50, 200, 6)
    w = W.GemmWorkload("i8", 33, 50, 200, W.I8, W.F32, transB=True, A=a, B=np.ascontiguousarray(b.T), scale_a=sa, scale_b=sb)
    prod, want = expect(a, b, sa, sb)
    check(ref.ref_gemm(w, acc64=True), prod, want, W.F32)
    check(R.gemm_host(w), prod, want, W.F32)
