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


@pytest.mark.parametrize("M,N", [(64, 256), (128, 128), (20, 64), (200, 300), (640, 640)])
def test_the_longest_sums_split_over_clusters(M, N):
    K = 131071
    a, b, _, _ = make(M, N, K, 16, full=True)
    a[0], b[:, 0] = -128, -128
    a[-1], b[:, -1] = 127, -128
    c = np.zeros((M, N), np.float32)
    plan = R.GemmPlan(M, N, K, W.I8, W.F32, transB=True)
    plan.run_host(a, np.ascontiguousarray(b.T), c)
    plan.close()
    assert np.array_equal(c, np.rint(a.astype(np.float64) @ b.astype(np.float64)).astype(np.float32))


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


# ----------------------------------------------------------------------------- tensor-core plans
# Every plan family, over the whole range of the type: without scales an fp32 C is the exact sum
# rounded once, whatever the tiles and the split of K.
PLANS = [
    # (M, N, K, kernel, plan options)
    (256, 512, 256, "tcgen05_pair", {}),
    (300, 520, 272, "tcgen05_pair", {}),                                 # ragged rows, columns and K
    (700, 1000, 4112, "tcgen05_pair", {"k_split": -1}),                  # many k-blocks, narrow last wave
    (300, 521, 272, "tcgen05_pair", {}),                                 # rows of C at any element
    (520, 1029, 300, "tcgen05_pair", {}),
    (290, 518, 272, "tcgen05_pair", {"epilogue": 3}),
    (333, 201, 400, "tcgen05", {"force_kernel": "tcgen05"}),
    (333, 390, 400, "tcgen05", {"force_kernel": "tcgen05"}),
    (512, 768, 640, "tcgen05_pair", {"epilogue": 1}),
    (512, 768, 640, "tcgen05_pair", {"epilogue": 2}),
    (512, 768, 640, "tcgen05_pair", {"epilogue": 3}),
    (512, 768, 640, "tcgen05_pair", {"epilogue": 4}),
    (128, 256, 256, "tcgen05", {"force_kernel": "tcgen05"}),
    (333, 200, 400, "tcgen05", {"force_kernel": "tcgen05", "tile_n": 64}),
    (1, 4096, 4096, "i8_rows", {}),                                      # one token
    (1, 256, 16, "i8_rows", {}),
    (1, 1, 16, "i8_rows", {}),
    (3, 37, 100, "i8_rows", {}),                                         # repacked, less than a chunk of K
    (8, 100, 528, "i8_rows", {}),
    (8, 4100, 528, "i8_rows", {}),
    (5, 8192, 8192, "i8_rows", {}),                                      # two tiles of weight rows per CTA
    (2, 300, 28672, "i8_rows", {}),
    (9, 4100, 528, "i8_rows", {}),                                       # two tiles of tokens
    (16, 8192, 1024, "i8_rows", {}),
    (16, 512, 4096, "i8_rows", {}),
    (13, 1000, 4099, "i8_rows", {}),
    (16, 2048, 28672, "skinny", {}),
    (1, 4096, 4096, "skinny", {"force_kernel": "skinny"}),
    (1, 256, 16, "skinny", {"force_kernel": "skinny"}),
    (16, 8192, 1024, "skinny", {"force_kernel": "skinny"}),
    (16, 512, 4096, "skinny", {"force_kernel": "skinny"}),
    (33, 4100, 528, "skinny", {}),
    (64, 2048, 2048, "skinny", {}),
    (31, 20000, 272, "skinny", {}),                                      # more columns than the SMs' tiles:
    (32, 20000, 272, "tcgen05", {}),                                     # whole tiles from 32 rows on
    (47, 19001, 528, "tcgen05", {}),
    (32, 20000, 272, "skinny", {"num_ctas": 148}),
    (100, 8192, 512, "skinny", {}),
    (128, 8192, 1040, "skinny", {}),
    (16, 8192, 1024, "skinny", {"num_ctas": 97}),                        # stream-K: partials in slots
    (24, 512, 8192, "skinny", {"num_ctas": 148}),                        # more partials of a tile than its list holds
    (17, 256, 144, "skinny", {}),                                        # one or two tiles: a cluster all the same,
    (64, 256, 1168, "skinny", {}),                                       # with a part of K that is shorter or empty
    (32, 512, 8192, "skinny", {}),
    (128, 300, 1040, "skinny", {}),
    (128, 128, 1152, "tcgen05", {}),                                     # small C: K over clusters of eight
    (128, 128, 16384, "tcgen05", {}),
    (40, 64, 2064, "tcgen05", {}),
    (100, 200, 1100, "tcgen05", {}),
    (130, 60, 2200, "tcgen05", {}),
    (384, 320, 1024, "tcgen05", {}),
    (160, 512, 4112, "tcgen05", {}),
    (500, 500, 4112, "tcgen05", {}),
    (499, 501, 1040, "tcgen05", {}),
    (2048, 64, 4112, "tcgen05", {}),
    (300, 640, 16400, "tcgen05", {}),
    (1280, 256, 6160, "tcgen05_pair", {}),                               # four pairs to a cluster
    (640, 640, 6144, "tcgen05_pair", {}),
    (333, 1000, 6200, "tcgen05_pair", {}),
    (600, 2008, 272, "tcgen05_pair", {"epilogue": 2}),                   # the last columns' chunk: on the 16-byte grid,
    (600, 2004, 272, "tcgen05_pair", {}),                                # words, elements
    (600, 2001, 272, "tcgen05_pair", {}),
    (47, 19010, 144, "tcgen05", {}),
    (512, 512, 4096, "tcgen05_pair", {"k_split": 3}),                    # K over the pairs of a cluster
    (260, 128, 8192, "tcgen05_pair", {"k_split": 3}),
    (512, 500, 4096, "tcgen05_pair", {"k_split": 2}),                    # K planes
    (520, 264, 2320, "tcgen05_pair", {"k_split": 2}),
    (129, 1000, 8192, "tcgen05", {"k_split": 1}),                        # K over a cluster, not swapped
    (512, 512, 65536, "tcgen05_pair", {}),
]


@pytest.mark.parametrize("M,N,K,kernel,kw", PLANS, ids=["-".join(map(str, [*p[:3], *p[4].values()])) for p in PLANS])
def test_sums_are_exact_on_every_plan(M, N, K, kernel, kw):
    a, b, _, _ = make(M, N, K, 7, full=True)
    c = np.zeros((M, N), np.float32)
    plan = R.GemmPlan(M, N, K, W.I8, W.F32, transB=True, **kw)
    assert plan.info["kernel_name"] == kernel, plan.info
    plan.run_host(a, np.ascontiguousarray(b.T), c)
    plan.close()
    want = np.rint(a.astype(np.float64) @ b.astype(np.float64))
    assert np.array_equal(c, want.astype(np.float32))


@pytest.mark.parametrize("clear", [True, False], ids=["set", "add"])
@pytest.mark.parametrize("ct", [W.F32, W.F16, W.BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N,K,kernel,kw", PLANS, ids=["-".join(map(str, [*p[:3], *p[4].values()])) for p in PLANS])
def test_scales_and_result_types_on_every_plan(M, N, K, kernel, kw, ct, clear):
    run(M, N, K, ct, clear=clear, seed=8, kernel=kernel, **kw)


@pytest.mark.parametrize("kind", ["max", "add", "min"])
@pytest.mark.parametrize("M,N,K", [(300, 520, 272), (512, 768, 640), (300, 521, 272), (130, 1030, 300)])
def test_row_reduce_folded_into_the_epilogue(M, N, K, kind):
    a, b, sa, sb = make(M, N, K, 9)
    c, dst = np.zeros((M, N), np.uint16), np.zeros(M, np.uint16)
    plan = R.GemmPlan(M, N, K, W.I8, W.BF16, transB=True, scales=True, row_reduce=kind)
    plan.run_host(a, np.ascontiguousarray(b.T), c, sa, sb, dst)
    plan.close()
    check(c, *expect(a, b, sa, sb), W.BF16)
    want, mag = ref.ref_reduce(c, 1, W.BF16, kind)
    err = np.abs(W.decode(dst, W.BF16).astype(np.float64) - want)
    assert (err <= (0 if kind != "add" else N * U * mag + 2.0 ** -8 * np.abs(want))).all()


def test_stays_inside_c_and_the_workspace():
    """Device buffers with guards around C, the rows' padding and the workspace."""
    import torch
    dev = torch.device("cuda:0")
    for M, N, K, kw in ((1, 300, 144, {}), (16, 8192, 1024, {"num_ctas": 97}), (130, 257, 272, {}), (512, 500, 4096, {"k_split": 2}),
                        (300, 520, 4099, {}), (600, 2037, 176, {}), (300, 1025, 144, {}), (300, 1983, 144, {}), (47, 19010, 144, {}),
                        (32, 512, 1168, {}), (100, 200, 1100, {})):
        a, b, sa, sb = make(M, N, K, 10)
        for ct, ldc, shift in ((W.BF16, N + 3, 0), (W.BF16, N + 1, 2), (W.F16, N + 2, 6), (W.BF16, N + 8, 16), (W.F32, N + 4, 0),
                               (W.F32, N + 1, 4)):
            es = W.ELEM_SIZE[ct]
            plan = R.GemmPlan(M, N, K, W.I8, ct, transB=True, scales=True, ldc=ldc, **kw)
            guard = 256 + shift
            cbuf = torch.full((M * ldc * es + 2 * guard,), 0x5A, dtype=torch.uint8, device=dev)
            wbuf = torch.full((plan.workspace_bytes + 512,), 0x5A, dtype=torch.uint8, device=dev)
            A, B = torch.from_numpy(a).to(dev), torch.from_numpy(np.ascontiguousarray(b.T)).to(dev)
            dsa, dsb = torch.from_numpy(sa).to(dev), torch.from_numpy(sb).to(dev)
            plan.run(A, B, cbuf.data_ptr() + guard, dsa, dsb, wbuf[256:256 + plan.workspace_bytes] if plan.workspace_bytes else None,
                     stream=torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            host, ws = cbuf.cpu().numpy(), wbuf.cpu().numpy()
            assert (host[:guard] == 0x5A).all() and (host[guard + M * ldc * es:] == 0x5A).all()
            assert (ws[:256] == 0x5A).all() and (ws[256 + plan.workspace_bytes:] == 0x5A).all()
            rows = host[guard:guard + M * ldc * es].reshape(M, ldc * es)
            assert (rows[:, N * es:] == 0x5A).all()
            check(np.ascontiguousarray(rows[:, :N * es]).view(W.storage_numpy_dtype(ct)), *expect(a, b, sa, sb), ct)
            plan.close()


def test_captured_into_a_graph():
    import torch
    dev = torch.device("cuda:0")
    M, N, K = 16, 1024, 2048
    plan = R.GemmPlan(M, N, K, W.I8, W.BF16, transB=True, scales=True)
    A, B = torch.zeros((M, K), dtype=torch.int8, device=dev), torch.zeros((N, K), dtype=torch.int8, device=dev)
    sa, sb = torch.zeros(M, device=dev), torch.zeros(N, device=dev)
    c = torch.zeros((M, N), dtype=torch.bfloat16, device=dev)
    ws = torch.zeros(max(plan.workspace_bytes, 16), dtype=torch.uint8, device=dev)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        plan.run(A, B, c, sa, sb, ws, stream=side.cuda_stream)
    for seed in (11, 12):
        a, b, ha, hb = make(M, N, K, seed)
        A.copy_(torch.from_numpy(a))
        B.copy_(torch.from_numpy(np.ascontiguousarray(b.T)))
        sa.copy_(torch.from_numpy(ha))
        sb.copy_(torch.from_numpy(hb))
        graph.replay()
        torch.cuda.synchronize()
        check(c.view(torch.int16).cpu().numpy().view(np.uint16), *expect(a, b, ha, hb), W.BF16)
    plan.close()


def test_the_tensor_pipes_rate_can_be_measured():
    got = R.measure_mma_peak(W.I8, pair=True, k_blocks=1024, reps=5)
    assert got["tflops"] > 1000.0, got
    print(got)


@pytest.mark.parametrize("M,N,K", [(200, 300, 1000), (16, 4096, 520), (1, 300, 130), (513, 257, 129)])
def test_orders_through_the_workspace_and_the_cuda_core_kernel_agree(M, N, K):
    """The transposed and copied operands' plans against the kernel that takes any order, bit for bit."""
    for ta, tb, pad in ((False, False, (0, 0)), (True, True, (0, 0)), (True, False, (1, 3)), (False, True, (5, 0))):
        a, b, _, _ = make(M, N, K, 13, full=True)
        A, lda = stored(a, ta, pad[0])
        B, ldb = stored(b, tb, pad[1])
        out = []
        for kw in ({}, {"force_kernel": "simt"}):
            c = np.zeros((M, N), np.float32)
            plan = R.GemmPlan(M, N, K, W.I8, W.F32, transA=ta, transB=tb, lda=lda, ldb=ldb, **kw)
            plan.run_host(A, B, c)
            plan.close()
            out.append(c)
        assert np.array_equal(out[0], out[1])
        assert np.array_equal(out[0], (a.astype(np.int64) @ b.astype(np.int64)).astype(np.float32))


def test_misaligned_bases_still_give_the_right_answer():
    import torch
    dev = torch.device("cuda:0")
    M, N, K = 40, 300, 256
    a, b, sa, sb = make(M, N, K, 14)
    A, B = torch.zeros(M * K + 16, dtype=torch.int8, device=dev), torch.zeros(N * K + 16, dtype=torch.int8, device=dev)
    A[3:3 + M * K] = torch.from_numpy(a.reshape(-1)).to(dev)
    B[5:5 + N * K] = torch.from_numpy(np.ascontiguousarray(b.T).reshape(-1)).to(dev)
    c = torch.zeros((M, N), dtype=torch.float32, device=dev)
    plan = R.GemmPlan(M, N, K, W.I8, W.F32, transB=True, scales=True)
    plan.run(A.data_ptr() + 3, B.data_ptr() + 5, c, torch.from_numpy(sa).to(dev), torch.from_numpy(sb).to(dev),
             stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert plan.refresh_info()["cuda_core_runs"] == 1
    plan.close()
    check(c.cpu().numpy(), *expect(a, b, sa, sb), W.F32)


@pytest.mark.parametrize("N", [32768, 32761])
def test_offsets_past_32_bits(N):
    """More than 2^31 elements of C: the last rows."""
    import torch
    dev = torch.device("cuda:0")
    M, K = 66000, 64
    A = torch.zeros((M, K), dtype=torch.int8, device=dev)
    pick = [0, 65535, 65536, M - 1]
    a, b, sa, sb = make(len(pick), N, K, 15)
    A[pick] = torch.from_numpy(a).to(dev)
    B = torch.from_numpy(np.ascontiguousarray(b.T)).to(dev)
    scale = torch.ones(M, device=dev)
    scale[pick] = torch.from_numpy(sa).to(dev)
    c = torch.full((M, N), 7.0, dtype=torch.bfloat16, device=dev)
    plan = R.GemmPlan(M, N, K, W.I8, W.BF16, transB=True, scales=True)
    ws = torch.zeros(max(plan.workspace_bytes, 16), dtype=torch.uint8, device=dev)
    plan.run(A, B, c, scale, torch.from_numpy(sb).to(dev), ws, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    plan.close()
    check(c[pick].view(torch.int16).cpu().numpy().view(np.uint16), *expect(a, b, sa, sb), W.BF16)
    c[pick] = 0
    assert not bool(c.any())
