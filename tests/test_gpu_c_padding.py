"""GEMM into a C with padded rows: the padding belongs to the caller and keeps its bits, whichever
epilogue stores the rows."""
import pytest

from frisk_b200 import runtime as R
from frisk_b200 import workloads as W

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("epilogue", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("ct", [W.F32, W.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("ab", [W.BF16, W.E4M3, W.I8], ids=["bf16", "e4m3", "i8"])
def test_padding_between_rows_is_kept(ab, ct, epilogue):
    import torch
    dev = torch.device("cuda:0")
    M, N, K, lda, ldc = 600, 2037, 170, 176, 2040       # rows start on 16-byte boundaries and end off them
    types = {W.BF16: torch.bfloat16, W.E4M3: torch.float8_e4m3fn, W.I8: torch.int8, W.F32: torch.float32}
    gen = torch.Generator(device=dev).manual_seed(3)
    # small whole numbers: every product sum is exact in fp32
    a, b = (torch.randint(-4, 5, (n, lda), generator=gen, device=dev).to(types[ab]) for n in (M, N))
    c = torch.full((M, ldc), 7.0, dtype=types[ct], device=dev)
    plan = R.GemmPlan(M, N, K, ab, ct, transB=True, lda=lda, ldb=lda, ldc=ldc, epilogue=epilogue)
    assert plan.info["kernel_name"] == "tcgen05_pair"
    ws = torch.empty(max(16, plan.workspace_bytes), dtype=torch.uint8, device=dev)
    plan.run(a, b, c, None, None, ws, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    plan.close()
    want = (a[:, :K].double() @ b[:, :K].double().T).to(types[ct])
    assert torch.equal(c[:, :N], want) and bool((c[:, N:] == 7).all())
