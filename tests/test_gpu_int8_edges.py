"""GPU checks of gemm runs whose operands lie off the 16-byte grid next to operands that a plan copies."""
import numpy as np
import pytest

from frisk_b200 import runtime as R
from frisk_b200 import workloads as W

pytestmark = pytest.mark.gpu


def operand(torch, rows, cols, ld, shift, dtype, seed):
    """rows x cols small whole numbers at a pitch and `shift` elements behind a 256-byte boundary."""
    gen = torch.Generator(device="cuda:0").manual_seed(seed)
    flat = torch.randint(-3, 4, (rows * ld + 64,), generator=gen, device="cuda:0").to(dtype)
    return flat, flat[shift:shift + rows * ld].view(rows, ld)[:, :cols], flat.data_ptr() + shift * flat.element_size()


@pytest.mark.parametrize("ab,shift", [(W.I8, 3), (W.E4M3, 5), (W.BF16, 1)], ids=["i8", "e4m3", "bf16"])
@pytest.mark.parametrize("moved", ["A", "B"])
@pytest.mark.parametrize("M", [8, 300])
def test_nothing_is_copied_for_a_run_on_the_cuda_cores(M, moved, ab, shift):
    """One operand has an odd pitch, so the plan copies it; the other starts off the 16-byte grid, so the run
    goes to the CUDA cores, which read both where they are: the workspace keeps its bits."""
    import torch
    types = {W.I8: torch.int8, W.E4M3: torch.float8_e4m3fn, W.BF16: torch.bfloat16}
    N, K, odd, even = 520, 250, 251, 256
    fa, a, pa = operand(torch, M, K, even if moved == "A" else odd, shift if moved == "A" else 0, types[ab], 1)
    fb, b, pb = operand(torch, N, K, even if moved == "B" else odd, shift if moved == "B" else 0, types[ab], 2)
    c = torch.zeros((M, N), device="cuda:0")
    plan = R.GemmPlan(M, N, K, ab, W.F32, transB=True, lda=a.stride(0), ldb=b.stride(0))
    assert plan.workspace_bytes > 0 and plan.info["kernel_name"] != "simt"
    ws = torch.full((plan.workspace_bytes,), 0x5A, dtype=torch.uint8, device="cuda:0")
    plan.run(pa, pb, c, None, None, ws, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert plan.refresh_info()["cuda_core_runs"] == 1
    want = a.double() @ b.double().T   # sums of whole numbers: exact in fp32
    assert torch.equal(c, want.float()) and bool((ws == 0x5A).all())
    # the operand that is copied may start anywhere
    fb2, b2, pb2 = operand(torch, N, K, odd, shift, types[ab], 3)
    fa2, a2, pa2 = operand(torch, M, K, even, 0, types[ab], 4)
    plan2 = R.GemmPlan(M, N, K, ab, W.F32, transB=True, lda=even, ldb=odd)
    ws2 = torch.empty(max(16, plan2.workspace_bytes), dtype=torch.uint8, device="cuda:0")
    plan2.run(pa2, pb2, c, None, None, ws2, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert plan2.refresh_info()["cuda_core_runs"] == 0 and torch.equal(c, (a2.double() @ b2.double().T).float())
    plan.close()
    plan2.close()


def test_a_refused_run_launches_nothing():
    """A fused row reduce with an operand off the grid is refused, before the other one is copied."""
    import torch
    M, N, K = 300, 520, 250
    fa, a, pa = operand(torch, M, K, 256, 3, torch.int8, 1)
    fb, b, pb = operand(torch, N, K, 251, 0, torch.int8, 2)
    c, dst = torch.zeros((M, N), device="cuda:0"), torch.zeros(M, device="cuda:0")
    plan = R.GemmPlan(M, N, K, W.I8, W.F32, transB=True, lda=256, ldb=251, row_reduce="max")
    ws = torch.full((plan.workspace_bytes,), 0x5A, dtype=torch.uint8, device="cuda:0")
    with pytest.raises(R.FriskError) as e:
        plan.run_ex(pa, pb, c, workspace=ws, stream=torch.cuda.current_stream().cuda_stream, row_reduce_dst=dst)
    assert e.value.code == -2
    torch.cuda.synchronize()
    assert bool((ws == 0x5A).all()) and not bool(c.any())
    plan.run_ex(fa.data_ptr(), pb, c, workspace=ws, stream=torch.cuda.current_stream().cuda_stream, row_reduce_dst=dst)
    torch.cuda.synchronize()
    plan.close()
    want = (fa[:M * 256].view(M, 256)[:, :K].double() @ b.double().T).float()
    assert torch.equal(c, want) and torch.equal(dst, want.amax(1))
