"""GEMM into a C whose rows start on 16-byte boundaries and end off them, by tensor stores: the whole units
of a row, and the elements behind the last one, which keep the padding as it is."""
import pytest

from frisk_b200 import runtime as R
from frisk_b200 import workloads as W

pytestmark = pytest.mark.gpu

TYPES = {W.BF16: "bfloat16", W.F16: "float16", W.E4M3: "float8_e4m3fn", W.I8: "int8", W.F32: "float32"}


def case(torch, M, N, K, ldc, ab, ct, clear=True, peers=0, scales=False, **kw):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(N)
    types = {k: getattr(torch, v) for k, v in TYPES.items()}
    lda = -(-K // 16) * 16
    # small whole numbers: every product sum is exact in fp32, and so are sums with scales that are powers of two
    a, b = (torch.randint(-4, 5, (n, lda), generator=gen, device=dev).to(types[ab]) for n in (M, N))
    c = torch.randint(-9, 10, (M + 1, ldc), generator=gen, device=dev).to(types[ct])
    before = c.clone()
    copies = [before.clone() for _ in range(peers)]
    sa, sb = (torch.exp2(torch.randint(-2, 3, (n,), generator=gen, device=dev).float()) for n in (M, N))
    plan = R.GemmPlan(M, N, K, ab, ct, transB=True, lda=lda, ldb=lda, ldc=ldc, clear_accum=clear, scales=scales, epilogue=4, **kw)
    assert plan.info["kernel_name"] == "tcgen05_pair"
    ws = torch.empty(max(16, plan.workspace_bytes), dtype=torch.uint8, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    plan.run_ex(a, b, c, scale_a=sa if scales else None, scale_b=sb if scales else None, workspace=ws, status=status,
                peers=copies, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    R.check_status(status)
    plan.close()
    prod = a[:, :K].double() @ b[:, :K].double().T
    if scales:
        prod = prod * sa.double()[:, None] * sb.double()
    want = before.clone()
    want[:M, :N] = (prod if clear else prod + before[:M, :N].double()).to(types[ct])
    for got in [c, *copies]:
        assert torch.equal(got, want)


@pytest.mark.parametrize("clear", [True, False], ids=["set", "add"])
@pytest.mark.parametrize("N", list(range(1017, 1025)) + [130, 1027])
@pytest.mark.parametrize("ct", [W.BF16, W.F16], ids=["bf16", "f16"])
def test_every_end_of_a_16_bit_row(ct, N, clear):
    import torch
    case(torch, 600, N, 64, 1032, W.BF16 if ct == W.BF16 else W.F16, ct, clear)


@pytest.mark.parametrize("clear", [True, False], ids=["set", "add"])
@pytest.mark.parametrize("N", [1021, 1022, 1023, 1024, 131])
@pytest.mark.parametrize("ab", [W.BF16, W.E4M3, W.I8], ids=["bf16", "e4m3", "i8"])
def test_every_end_of_a_32_bit_row(ab, N, clear):
    import torch
    case(torch, 520, N, 96, 1028, ab, W.F32, clear, scales=ab != W.BF16)


@pytest.mark.parametrize("M,N", [(257, 2037), (300, 261), (2048, 2047)])
@pytest.mark.parametrize("ct", [W.BF16, W.F32], ids=["bf16", "f32"])
def test_copies_get_the_same_rows(ct, M, N):
    import torch
    case(torch, M, N, 80, 2048, W.BF16, ct, peers=2)


@pytest.mark.parametrize("kind", ["max", "add"])
@pytest.mark.parametrize("ab,ct,N", [(W.BF16, W.BF16, 1021), (W.I8, W.F32, 1022), (W.I8, W.BF16, 133)], ids=["bf16", "i8-f32", "i8-bf16"])
def test_row_reduce_of_such_rows(ab, ct, N, kind):
    import torch
    dev = torch.device("cuda:0")
    M, K, ldc = 520, 64, 1024
    types = {k: getattr(torch, v) for k, v in TYPES.items()}
    gen = torch.Generator(device=dev).manual_seed(N)
    a, b = (torch.randint(-1, 2, (n, K), generator=gen, device=dev).to(types[ab]) for n in (M, N))
    c, dst = torch.full((M, ldc), 7.0, dtype=types[ct], device=dev), torch.zeros(M, dtype=types[ct], device=dev)
    plan = R.GemmPlan(M, N, K, ab, ct, transB=True, ldc=ldc, epilogue=4, row_reduce=kind)
    assert plan.info["kernel_name"] == "tcgen05_pair"
    ws = torch.empty(max(16, plan.workspace_bytes), dtype=torch.uint8, device=dev)
    plan.run_ex(a, b, c, workspace=ws, stream=torch.cuda.current_stream().cuda_stream, row_reduce_dst=dst)
    torch.cuda.synchronize()
    plan.close()
    prod = a.double() @ b.double().T   # whole numbers up to 64: exact in every type, and so is a row's sum before its rounding
    assert torch.equal(c[:, :N].double(), prod) and bool((c[:, N:] == 7).all())
    assert torch.equal(dst, (prod.amax(1) if kind == "max" else prod.sum(1)).to(types[ct]))
