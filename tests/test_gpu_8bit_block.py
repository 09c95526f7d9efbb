"""The 8-bit operators together, as a program uses them: a gated feed-forward block in 8 bits,

    q, s, h = rows of rmsnorm(x + residual) * weight          (8-bit rows and scales, the new residual)
    y       = (q . W1^T) with scales                           (gate and up side by side)
    p, t    = rows of silu(gate) * up                          (8-bit rows and scales)
    z       = (p . W2^T) with scales

with weights quantised on the device first, every step on one stream.  Each step is compared with the
float64 restatement of that step on the inputs it really had, at the tolerances that the operators'
own tests derive; then the block is captured into a graph and replayed on other inputs, where it has to
give the bits of the plain launches."""
import numpy as np
import pytest

from frisk_b200 import runtime as R
from frisk_b200 import workloads as W
from oracle import ref
from test_gpu_quant import check_q, check_sum

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


class Block:
    def __init__(self, torch, rows, width, hidden, q_type, seed):
        self.torch, self.dims, self.q_type = torch, (rows, width, hidden), q_type
        dev = torch.device("cuda:0")
        g = torch.Generator(device=dev).manual_seed(seed)
        q8 = torch.int8 if q_type == W.I8 else torch.float8_e4m3fn if q_type == W.E4M3 else torch.float8_e5m2
        bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=dev)  # noqa: E731
        f32 = lambda *s: torch.zeros(s, device=dev)  # noqa: E731
        self.x, self.residual, self.h = bf(rows, width), bf(rows, width), bf(rows, width)
        self.weight = (1 + 0.2 * torch.randn(width, generator=g, device=dev)).to(torch.bfloat16)
        self.q, self.s = torch.zeros((rows, width), dtype=q8, device=dev), f32(rows)
        self.y, self.z = bf(rows, 2 * hidden), bf(rows, width)
        self.p, self.t = torch.zeros((rows, hidden), dtype=q8, device=dev), f32(rows)
        stream = torch.cuda.current_stream().cuda_stream
        self.mats = []   # quantised weights: (master, q, scale)
        for n, k in ((2 * hidden, width), (width, hidden)):
            m = (torch.randn((n, k), generator=g, device=dev) / k ** 0.5).float()
            q, s = torch.zeros((n, k), dtype=q8, device=dev), f32(n)
            R.quant_run(R.quant_desc(n, k, W.F32, q_type), m, q, s, stream=stream)
            self.mats.append((m, q, s))
        self.norm = R.quant_desc(rows, width, W.BF16, q_type, "rmsnorm", eps=1e-5)
        self.gate = R.quant_desc(rows, hidden, W.BF16, q_type, "silu_mul")
        self.up = R.GemmPlan(rows, 2 * hidden, width, q_type, W.BF16, transB=True, scales=True)
        self.down = R.GemmPlan(rows, width, hidden, q_type, W.BF16, transB=True, scales=True)
        self.ws = torch.zeros(max(self.up.workspace_bytes, self.down.workspace_bytes, 16), dtype=torch.uint8, device=dev)

    def set_inputs(self, seed):
        g = self.torch.Generator(device="cuda:0").manual_seed(seed)
        for t in (self.x, self.residual):
            t.copy_(self.torch.randn(t.shape, generator=g, device="cuda:0"))

    def run(self, stream):
        (_, q1, s1), (_, q2, s2) = self.mats
        R.quant_run(self.norm, self.x, self.q, self.s, weight=self.weight, residual=self.residual, sum_out=self.h, stream=stream)
        self.up.run(self.q, q1, self.y, self.s, s1, workspace=self.ws, stream=stream)
        R.quant_run(self.gate, self.y, self.p, self.t, stream=stream)
        self.down.run(self.p, q2, self.z, self.t, s2, workspace=self.ws, stream=stream)

    def results(self):
        self.torch.cuda.synchronize()
        return [t.contiguous().view(self.torch.uint8).cpu().numpy() for t in (self.q, self.s, self.h, self.y, self.p, self.t, self.z)]

    def close(self):
        self.up.close()
        self.down.close()


def bits(t, dtype):
    import torch
    return t.contiguous().view(torch.uint8).cpu().numpy().view(W.storage_numpy_dtype(dtype)).reshape(t.shape)


def check_gemm(got, q, s, qw, sw, q_type):
    """bf16 result of an 8-bit product: integer sums are exact; fp8 products are exact in fp32 and summed
    in fp32 (k roundings of the partial sums at worst); scales and the stored type round as ever."""
    a, b = W.decode(q, q_type).astype(np.float64), W.decode(qw, q_type).astype(np.float64)
    scale = s.astype(np.float64)[:, None] * sw.astype(np.float64)[None, :]
    want = (a @ b.T) * scale
    mag = (np.abs(a) @ np.abs(b).T) * scale if q_type != W.I8 else np.abs(want)
    k = a.shape[1] if q_type != W.I8 else 0
    tol = (k + 4) * U * mag + 2.0 ** -8 * np.abs(want) + 1e-30
    err = np.abs(W.decode(got, W.BF16).astype(np.float64) - want)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("q_type", [W.I8, W.E4M3], ids=["i8", "e4m3"])
@pytest.mark.parametrize("rows,width,hidden", [(1, 512, 1024), (16, 1024, 2816), (200, 768, 1000), (700, 1024, 2048)])
def test_feed_forward_block(rows, width, hidden, q_type):
    import torch
    blk = Block(torch, rows, width, hidden, q_type, 21)
    blk.set_inputs(22)
    stream = torch.cuda.current_stream().cuda_stream
    blk.run(stream)
    torch.cuda.synchronize()
    for m, q, s in blk.mats:
        check_q(bits(q, q_type), s.cpu().numpy(), m.cpu().numpy().astype(np.float64), "plain", q_type)
    v, h = ref.ref_quant(bits(blk.x, W.BF16), W.BF16, "rmsnorm", weight=bits(blk.weight, W.BF16),
                         residual=bits(blk.residual, W.BF16), eps=1e-5)
    check_q(bits(blk.q, q_type), blk.s.cpu().numpy(), v, "rmsnorm", q_type)
    check_sum(bits(blk.h, W.BF16), h, W.BF16)
    check_gemm(bits(blk.y, W.BF16), bits(blk.q, q_type), blk.s.cpu().numpy(), bits(blk.mats[0][1], q_type), blk.mats[0][2].cpu().numpy(), q_type)
    v, _ = ref.ref_quant(bits(blk.y, W.BF16), W.BF16, "silu_mul")
    check_q(bits(blk.p, q_type), blk.t.cpu().numpy(), v, "silu_mul", q_type)
    check_gemm(bits(blk.z, W.BF16), bits(blk.p, q_type), blk.t.cpu().numpy(), bits(blk.mats[1][1], q_type), blk.mats[1][2].cpu().numpy(), q_type)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        blk.run(side.cuda_stream)
    for seed in (23, 24):
        blk.set_inputs(seed)
        blk.run(stream)
        plain = blk.results()
        for t in (blk.q, blk.p):
            t.view(torch.uint8).zero_()
        blk.z.zero_()
        torch.cuda.synchronize()
        graph.replay()
        for a, b in zip(plain, blk.results()):
            assert np.array_equal(a, b)
    del graph
    blk.close()


def test_two_blocks_on_two_streams_at_once():
    """Separate plans, workspaces and buffers, launches interleaved: each gives what it gives alone."""
    import torch
    blks = [Block(torch, 64, 1024, 2048, W.I8, 31), Block(torch, 300, 768, 1536, W.I8, 32)]
    alone = []
    for i, b in enumerate(blks):
        b.set_inputs(40 + i)
        b.run(torch.cuda.current_stream().cuda_stream)
        alone.append(b.results())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for b, st in zip(blks, streams):
            b.run(st.cuda_stream)
    torch.cuda.synchronize()
    for b, want in zip(blks, alone):
        for x, y in zip(b.results(), want):
            assert np.array_equal(x, y)
        b.close()
