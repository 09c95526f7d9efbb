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
