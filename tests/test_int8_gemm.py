"""CPU checks of the 8-bit integer gemm: plans, refusals, the IR surface, the codec."""
import numpy as np
import pytest

from frisk_b200 import runtime as R
from frisk_b200 import workloads as W


def refused(code, *a, **kw):
    with pytest.raises(R.FriskError) as e:
        R.GemmPlan(*a, **kw)
    assert e.value.code == code, e.value


def test_plans_that_are_refused():
    refused(-2, 64, 64, 64, W.I8, W.I8, transB=True)           # inputs only
    refused(-2, 64, 64, 64, W.I8, W.E4M3, transB=True)
    refused(-9, 64, 64, 131072, W.I8, W.F32, transB=True)      # the sum could pass 2^31
    refused(-1, 64, 64, 0, W.I8, W.F32, transB=True)
    refused(-1, 64, 64, 64, W.I8, W.F32, transB=True, lda=63)
    refused(-2, 64, 64, 64, W.I8, W.F32, transB=True, force_kernel="tf32x3")
    R.GemmPlan(64, 64, 131071, W.I8, W.F32, transB=True).close()


def test_run_refuses_missing_scales():
    plan = R.GemmPlan(64, 64, 64, W.I8, W.BF16, transB=True, scales=True)
    with pytest.raises(R.FriskError) as e:
        plan.run(0x10000, 0x20000, 0x30000)
    assert e.value.code == -1
    plan.close()


def test_the_codec_rounds_to_even_and_leaves_out_minus_128():
    x = np.array([0.5, 1.5, -0.5, -2.5, 126.5, 200.0, -200.0, -127.6, np.nan, np.inf], np.float32)
    assert W.encode(x, W.I8).tolist() == [0, 2, 0, -2, 126, 127, -127, -127, 0, 127]
    every = np.arange(-127, 128).astype(np.float32)
    assert np.array_equal(W.decode(W.encode(every, W.I8), W.I8), every)


def test_builder_and_parser_take_8_bit_integers():
    import frisk as F
    h = F.create_session()
    f32 = h.builder.get_f32_ty()
    assert str(h.builder.get_int8_ty()) == "i8"
    tys = [h.memref_type((8, 4), "int8"), h.memref_type((4, 16), "int8"), h.memref_type((8, 16), "bf16"),
           h.memref_type((8,), f32), h.memref_type((16,), f32)]
    _, entry = h.new_kernel("k", tys)
    a = [entry.get_argument(i) for i in range(5)]
    h.builder.create_gemm_op(a[0], a[1], a[2], False, True, True, a[3], a[4])
    assert h.module.verify(), h.module.verify_message()
    (call,) = F.find_gemms(h.module, "k")
    assert (call.ab_type, call.c_type, call.arg_scale_a, call.arg_scale_b) == (W.I8, W.BF16, 3, 4)
    (again,) = F.find_gemms(F.parse_module(str(h.module)), "k")
    assert again == call
    with pytest.raises(ValueError, match="matching element types"):
        h64 = F.create_session()
        tys = [h64.memref_type((8, 4), "int64"), h64.memref_type((4, 16), "int64"), h64.memref_type((8, 16), "bf16")]
        _, e = h64.new_kernel("k", tys)
        h64.builder.create_gemm_op(*[e.get_argument(i) for i in range(3)])


def test_kernel_families_and_the_fixed_scratch_entry_point():
    for (M, N, K), kernel in (((8192, 8192, 8192), "tcgen05_pair"), ((16, 8192, 8192), "i8_rows"), ((1, 4096, 4096), "i8_rows"),
                              ((8, 8192, 8192), "i8_rows"), ((17, 8192, 8192), "skinny"),
                              ((31, 28672, 4096), "skinny"), ((32, 28672, 4096), "tcgen05"), ((64, 8192, 8192), "skinny"),
                              ((128, 192, 256), "tcgen05")):
        p = R.GemmPlan(M, N, K, W.I8, W.BF16, transB=True, scales=True)
        assert p.info["kernel_name"] == kernel and p.info["tile_k"] == 128, p.info
        p.close()
    refused(-2, 17, 4096, 4096, W.I8, W.BF16, transB=True, force_kernel="i8_rows")      # at most 16 tokens
    refused(-2, 8, 4096, 4096, W.BF16, W.BF16, transB=True, force_kernel="i8_rows")
    d = R.GemmDesc()     # its scratch adds fp32 partial sums: not for an exact product
    d.M, d.N, d.K, d.a_type, d.b_type, d.c_type, d.transB, d.clear_accum = 16, 512, 512, W.I8, W.I8, W.BF16, 1, 1
    assert R.lib().frisk_b200_gemm_skinny_static(d, 0x10000, 0x20000, 0x30000, None, None, None, None) == -2


def test_other_orders_and_odd_pitches_are_brought_into_the_tensor_cores_order():
    base = R.GemmPlan(512, 520, 256, W.I8, W.BF16, transB=True)
    assert base.info["kernel_name"] == "tcgen05_pair" and base.workspace_bytes == 0 and base.info["launches"] == 1
    base.close()
    for kw, launches, ws in ((dict(transB=False), 2, 520 * 256), (dict(transA=True, transB=False), 3, (512 + 520) * 256),
                             (dict(transA=True, transB=True), 2, 512 * 256),
                             (dict(transB=True, lda=257, ldb=259), 2, (512 + 520) * 256),      # both copied by one launch
                             (dict(transB=True, ldb=259), 2, 520 * 256)):
        p = R.GemmPlan(512, 520, 256, W.I8, W.BF16, **kw)
        assert p.info["kernel_name"] == "tcgen05_pair" and p.info["launches"] == launches and p.workspace_bytes == ws, (kw, p.info)
        p.close()
    p = R.GemmPlan(512, 520, 250, W.I8, W.BF16, transB=False, force_kernel="simt")
    assert p.info["kernel_name"] == "simt" and p.workspace_bytes == 0 and p.info["launches"] == 1
    p.close()
