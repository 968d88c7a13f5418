"""Refusals of the layer-level operators, without a GPU: argument mistakes must come back as status codes or
exceptions before anything is launched.  Pointers in these calls are never read."""
import ctypes as C

import pytest
import torch

import gemmkernels_b200 as GK
from gemmkernels_b200 import _lib as L
from gemmkernels_b200 import Epilogue, Layout, Operator, Transform

FAKE = C.c_void_p(0x1000)


def desc(**kw):
    base = dict(number=L.GK_REAL, m=64, n=64, k=64, dtype_a=L.GK_F16, dtype_b=L.GK_F16, dtype_c=L.GK_F32, dtype_d=L.GK_F32,
                compute=L.GK_F16, op=L.GK_OP_TCGEN05, lda=64, ldb=64, ldc=64, ldd=64, alpha=1.0)
    base.update(kw)
    return L.GemmDesc(**base)


def groups(**kw):
    base = dict(ragged=L.GK_RAGGED_COLUMNS, groups=4, offsets_dtype=L.GK_I32, offsets=0x1000, stride_a=4096, stride_d=4096)
    base.update(kw)
    return L.GroupDesc(**base)


def call(d, fu=None, gr=None, a=FAKE, b=FAKE, c=None, dd=FAKE, ws=None, ws_bytes=0):
    fu = fu or L.FusedDesc()
    return L.lib.gk_gemm_fused(None, C.byref(d), C.byref(fu), C.byref(gr) if gr is not None else None, a, b, c, dd, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,fu,gr,status,needle", [
    (dict(number=L.GK_COMPLEX), {}, None, L.GK_ERR_INVALID_CONFIG, "real"),
    (dict(batch=2, batch_stride_d=4096), {}, None, L.GK_ERR_INVALID_CONFIG, "single"),
    (dict(debug=8), {}, None, L.GK_ERR_INVALID_CONFIG, "diagnostic"),
    (dict(op=L.GK_OP_FPU), {}, None, L.GK_ERR_INVALID_CONFIG, "TCGen05Operator"),
    (dict(layout_a=L.GK_LAYOUT_DIAGONAL), {}, None, L.GK_ERR_INVALID_CONFIG, "dense"),
    (dict(dtype_a=L.GK_F32, dtype_b=L.GK_F32, compute=L.GK_TF32), {}, None, L.GK_ERR_INVALID_CONFIG, "Float16 or BFloat16"),
    (dict(dtype_b=L.GK_BF16), {}, None, L.GK_ERR_INVALID_CONFIG, "Float16 or BFloat16"),
    (dict(dtype_d=L.GK_F64), {}, None, L.GK_ERR_INVALID_CONFIG, "D must be"),
    (dict(beta=1.0, dtype_c=L.GK_F16), {}, None, L.GK_ERR_INVALID_CONFIG, "element type of D"),
    (dict(ldd=63), {}, None, L.GK_ERR_DIMENSION_MISMATCH, "ldd"),
    (dict(), dict(form=7), None, L.GK_ERR_UNSUPPORTED, "form"),
    (dict(), dict(activation=9), None, L.GK_ERR_UNSUPPORTED, "activation"),
    (dict(), dict(bias_axis=5), None, L.GK_ERR_UNSUPPORTED, "bias axis"),
    (dict(), dict(form=L.GK_FUSED_GRADIENT, bias_axis=L.GK_BIAS_ROW, z=0x2000, ldz=64), None, L.GK_ERR_INVALID_CONFIG, "no bias"),
    (dict(), dict(z=0x2000, ldz=63), None, L.GK_ERR_DIMENSION_MISMATCH, "ldz"),
    (dict(), {}, dict(ragged=3), L.GK_ERR_UNSUPPORTED, "ragged"),
    (dict(), {}, dict(groups=0), L.GK_ERR_INVALID_CONFIG, "groups"),
    (dict(), {}, dict(groups=L.GK_MAX_GROUPS + 1), L.GK_ERR_INVALID_CONFIG, "groups"),
    (dict(), {}, dict(offsets=None), L.GK_ERR_INVALID_ARGUMENT, "offsets is NULL"),
    (dict(), {}, dict(offsets=0x1002), L.GK_ERR_INVALID_ARGUMENT, "aligned"),
    (dict(), {}, dict(offsets_dtype=L.GK_F32), L.GK_ERR_UNSUPPORTED, "offsets"),
    (dict(), {}, dict(stride_a=-8), L.GK_ERR_DIMENSION_MISMATCH, "negative"),
    (dict(), dict(bias_axis=L.GK_BIAS_COL, bias=0x2000), {}, L.GK_ERR_INVALID_CONFIG, "per row"),
    (dict(), {}, dict(ragged=L.GK_RAGGED_DEPTH, stride_d=64 * 32), L.GK_ERR_DIMENSION_MISMATCH, "overlap"),
    (dict(), dict(activation=L.GK_ACT_RELU), dict(ragged=L.GK_RAGGED_DEPTH), L.GK_ERR_INVALID_CONFIG, "ragged depth"),
    (dict(), dict(z=0x2000, ldz=64), dict(ragged=L.GK_RAGGED_DEPTH), L.GK_ERR_INVALID_CONFIG, "ragged depth"),
])
def test_fused_descriptor_refusals(kw, fu, gr, status, needle):
    st = call(desc(**kw), L.FusedDesc(**fu), groups(**gr) if gr is not None else None, c=FAKE)
    assert st == status and needle in L.last_error(), (st, L.last_error())


@pytest.mark.parametrize("kw,fu,ptrs,needle", [
    (dict(), {}, dict(a=None), "A is NULL"),
    (dict(), {}, dict(b=None), "B is NULL"),
    (dict(), {}, dict(dd=None), "D is NULL"),
    (dict(beta=1.0), {}, dict(c=None), "C is NULL"),
    (dict(), dict(bias_axis=L.GK_BIAS_ROW), {}, "bias pointer is NULL"),
    (dict(), dict(form=L.GK_FUSED_GRADIENT), {}, "needs Z"),
    (dict(), dict(form=L.GK_FUSED_RESIDUAL, z=0x1000, ldz=64), {}, "share memory"),
    (dict(), {}, dict(ws_bytes=64), "workspace_bytes"),
    (dict(), {}, dict(a=C.c_void_p(0x1001)), "aligned"),
    (dict(), {}, dict(dd=C.c_void_p(0x1002)), "aligned"),
    (dict(), dict(form=L.GK_FUSED_RESIDUAL, z=0x2002, ldz=64), {}, "aligned"),
    (dict(), dict(bias_axis=L.GK_BIAS_ROW, bias=0x2002), {}, "aligned"),
    (dict(beta=1.0, ldc=72), {}, dict(c=FAKE), "leading dimension"),
    (dict(), dict(form=L.GK_FUSED_GRADIENT, z=0x1000, ldz=72), {}, "leading dimension"),
    (dict(), {}, {}, "handle is NULL"),
])
def test_fused_pointer_refusals(kw, fu, ptrs, needle):
    assert call(desc(**kw), L.FusedDesc(**fu), **ptrs) == L.GK_ERR_INVALID_ARGUMENT
    assert needle in L.last_error(), L.last_error()


def test_in_place_gradients_need_equal_strides():
    gr = groups(ragged=L.GK_RAGGED_DEPTH, stride_d=4096, stride_c=8192)
    assert call(desc(beta=1.0, trans_b=1), gr=gr, c=FAKE) == L.GK_ERR_INVALID_ARGUMENT and "strides" in L.last_error()


def test_struct_sizes_are_checked():
    for which in ("fused", "groups"):
        fu, gr = L.FusedDesc(), groups()
        (fu if which == "fused" else gr).struct_size = 8
        assert call(desc(), fu, gr) == L.GK_ERR_INVALID_ARGUMENT and "struct_size" in L.last_error()
    assert L.lib.gk_gemm_fused(None, C.byref(desc()), None, None, FAKE, FAKE, None, FAKE, None, 0, None) == L.GK_ERR_INVALID_ARGUMENT
    assert (C.sizeof(L.FusedDesc), C.sizeof(L.GroupDesc), C.sizeof(L.ActivationGradientDesc)) == (48, 56, 80)


@pytest.mark.parametrize("kw,ptrs,status,needle", [
    (dict(m=-1), {}, L.GK_ERR_DIMENSION_MISMATCH, "negative"),
    (dict(dtype=L.GK_I32), {}, L.GK_ERR_UNSUPPORTED, "Float16"),
    (dict(activation=4), {}, L.GK_ERR_UNSUPPORTED, "activation"),
    (dict(ld_dz=63), {}, L.GK_ERR_DIMENSION_MISMATCH, "leading dimension"),
    (dict(ld_z=63), {}, L.GK_ERR_DIMENSION_MISMATCH, "leading dimension"),
    (dict(groups=2), {}, L.GK_ERR_INVALID_ARGUMENT, "offsets is NULL"),
    (dict(groups=0), {}, L.GK_ERR_INVALID_CONFIG, "groups"),
    (dict(groups=2, offsets=0x1000, offsets_dtype=L.GK_F16), {}, L.GK_ERR_UNSUPPORTED, "offsets"),
    (dict(), dict(dz=None, db=None), L.GK_ERR_INVALID_ARGUMENT, "neither"),
    (dict(), dict(dd=None), L.GK_ERR_INVALID_ARGUMENT, "dD is NULL"),
    (dict(), dict(z=None), L.GK_ERR_INVALID_ARGUMENT, "Z is NULL"),
    (dict(), dict(z=C.c_void_p(0x1001)), L.GK_ERR_INVALID_ARGUMENT, "aligned"),
    (dict(), dict(db=C.c_void_p(0x1002)), L.GK_ERR_INVALID_ARGUMENT, "aligned"),
    (dict(ld_dz=72), {}, L.GK_ERR_INVALID_ARGUMENT, "leading dimension"),
    (dict(), {}, L.GK_ERR_INVALID_ARGUMENT, "handle is NULL"),
])
def test_activation_gradient_refusals(kw, ptrs, status, needle):
    base = dict(dtype=L.GK_F16, m=64, n=64, ld_dd=64, ld_z=64, ld_dz=64, ld_db=64, activation=L.GK_ACT_GELU, groups=1)
    base.update(kw)
    p = dict(dd=FAKE, z=FAKE, dz=FAKE, db=FAKE)
    p.update(ptrs)
    st = L.lib.gk_activation_gradient(None, C.byref(L.ActivationGradientDesc(**base)), p["dd"], p["z"], p["dz"], p["db"], None, 0, None)
    assert st == status and needle in L.last_error(), (st, L.last_error())


# ------------------------------------------------------------------------------------------------
# the Python layer
# ------------------------------------------------------------------------------------------------
F16, F32 = GK.Float16, GK.Float32


def cm(*shape, dtype=torch.float16):
    return torch.zeros(tuple(reversed(shape)), dtype=dtype).permute(*reversed(range(len(shape))))


def conf(m, n, k, out=F32, residual=False, b_row_major=False, op=None):
    return GK.get_config(gemm_shape=(m, n, k), operator=op or Operator.TCGen05Operator[F16, F32], global_a_layout=Layout.ColMajor[F16],
                         global_b_layout=(Layout.RowMajor if b_row_major else Layout.ColMajor)[F16],
                         global_c_layout=(Layout.ColMajor if residual else Layout.Zero)[out], global_d_layout=Layout.ColMajor[out],
                         is_b_col_major=not b_row_major)


def refused(exc, needle, fn):
    with pytest.raises(exc) as e:
        fn()
    assert needle in str(e.value), str(e.value)


def test_fused_epilogue_arguments_are_checked():
    a, b, d = cm(64, 32), cm(32, 40), cm(64, 40, dtype=torch.float32)

    def run(epilogue, **kw):
        return lambda: GK.matmul(conf(64, 40, 32), a, b, None, d, epilogue=epilogue, **kw)

    R = Epilogue.BiasActivationResidual
    refused(Transform.UnsupportedFunctor, "activation", run(R(activation=Transform.Scale(2.0))))
    refused(Transform.UnsupportedFunctor, "activation hooks", run(R(), transform_shared_to_global_d=Transform.Elementwise(Transform.ReLU())))
    refused(Transform.UnsupportedFunctor, "Float32", run(R(torch.zeros(64, dtype=torch.float16))))
    refused(GK.DimensionMismatch, "bias", run(R(torch.zeros(63))))
    scale = Transform.Elementwise(Transform.Scale(2.0))
    refused(Transform.UnsupportedFunctor, "not fused", run(R(torch.zeros(64)), transform_shared_to_global_d=scale))
    refused(Transform.UnsupportedFunctor, "before the bias", run(R(torch.zeros(64)), transform_regs_to_shared_d=Transform.Elementwise(Transform.ReLU())))
    refused(GK.DimensionMismatch, "bias", run(R(torch.zeros(64), axis="col")))
    refused(GK.GemmKernelsError, "consecutive", run(R(torch.zeros(128)[::2])))
    refused(GK.GemmKernelsError, "address", run(R(0x1000)))
    refused(GK.DimensionMismatch, "pre-activation", run(R(preactivation=cm(64, 39, dtype=torch.float32))))
    refused(GK.ConfigError, "pre-activation", run(R(preactivation=cm(64, 40))))
    refused(GK.GemmKernelsError, "column-major", run(R(preactivation=torch.zeros(64, 40))))
    refused(GK.GemmKernelsError, "pre-activation", run(Epilogue.ActivationGradient(None)))
    refused(GK.GemmKernelsError, "CUDA", run(R()))
    with pytest.raises(ValueError):
        R(axis="diag")


def test_grouped_arguments_are_checked():
    a, b, d = cm(64, 32, 4), cm(32, 40), cm(64, 40, dtype=torch.float32)
    offsets = torch.zeros(5, dtype=torch.int32)

    def run(a=a, b=b, d=d, offsets=offsets, c=None, **kw):
        return lambda: GK.matmul_grouped(conf(64, 40, 32), a, b, c, d, offsets, **kw)

    refused(GK.DimensionMismatch, "one matrix per group", run(a=a[:, :, 0]))
    refused(GK.DimensionMismatch, "one matrix per group", run(a=a[:, :, :0]))
    refused(GK.DimensionMismatch, "offsets", run(offsets=offsets[:4]))
    refused(GK.DimensionMismatch, "offsets", run(offsets=torch.zeros(10, dtype=torch.int32)[::2]))
    refused(GK.ConfigError, "offsets", run(offsets=offsets.float()))
    refused(GK.DimensionMismatch, "bias", run(epilogue=Epilogue.Bias(torch.zeros(64), axis="row")))
    refused(GK.GemmKernelsError, "consecutive", run(epilogue=Epilogue.Bias(torch.zeros(64, 4), axis="row")))
    refused(Transform.UnsupportedFunctor, "before the bias", run(epilogue=Epilogue.Bias(cm(64, 4, dtype=torch.float32), axis="row"),
                                                                 transform_regs_to_shared_d=Transform.Elementwise(Transform.ReLU())))
    refused(GK.GemmKernelsError, "column-major", run(a=torch.zeros(64, 32, 4, dtype=torch.float16)))
    refused(GK.GemmKernelsError, "overlapping", run(b=cm(32, 40).as_strided((32, 40), (1, 16))))
    refused(GK.GemmKernelsError, "CUDA", run())


def test_grouped_outer_arguments_are_checked():
    a, b, d = cm(64, 32), cm(40, 32), cm(64, 40, 4, dtype=torch.float32)
    offsets = torch.zeros(5, dtype=torch.int64)
    cf = conf(64, 40, 32, b_row_major=True)

    def run(d=d, offsets=offsets, c=None, cf=cf, **kw):
        return lambda: GK.matmul_grouped_outer(cf, a, b, c, d, offsets, **kw)

    refused(GK.DimensionMismatch, "one matrix per group", run(d=d[:, :, 0]))
    refused(GK.DimensionMismatch, "offsets", run(offsets=offsets[:3]))
    refused(GK.DimensionMismatch, "last extent", run(c=d[:, :, :3], cf=conf(64, 40, 32, residual=True, b_row_major=True)))
    refused(Transform.UnsupportedFunctor, "alpha, beta", run(transform_shared_to_global_d=Transform.Elementwise(Transform.ReLU())))
    refused(GK.GemmKernelsError, "CUDA", run())


def test_activation_gradient_arguments_are_checked():
    x = cm(64, 40)
    db = torch.zeros(64)
    f = GK.activation_gradient_
    refused(GK.GemmKernelsError, "neither", lambda: f(None, x, x, Transform.GELU()))
    refused(GK.GemmKernelsError, "needs the pre-activation", lambda: f(x, x, None, Transform.GELU()))
    refused(GK.DimensionMismatch, "dZ", lambda: f(cm(64, 39), x, x))
    refused(GK.ConfigError, "Z holds", lambda: f(x, x, cm(64, 40, dtype=torch.bfloat16), Transform.ReLU()))
    refused(GK.ConfigError, "Float32", lambda: f(x, x, x, bias_gradient=db.half()))
    refused(GK.DimensionMismatch, "bias gradient", lambda: f(x, x, x, bias_gradient=torch.zeros(63)))
    refused(GK.DimensionMismatch, "bias gradient", lambda: f(x, x, x, bias_gradient=db, offsets=torch.zeros(3, dtype=torch.int32)))
    refused(GK.DimensionMismatch, "offsets", lambda: f(x, x, x, offsets=torch.zeros(1, dtype=torch.int32)))
    refused(GK.GemmKernelsError, "CUDA", lambda: f(x, x, x, Transform.SiLU(), bias_gradient=db))


def test_other_entry_points_refuse_the_fused_epilogues():
    a, b, d = cm(64, 32), cm(32, 40), cm(64, 40, dtype=torch.float32)
    with pytest.raises(Transform.UnsupportedFunctor):
        GK.matmul_host(conf(64, 40, 32), a, b, None, d, epilogue=Epilogue.BiasActivationResidual())
    with pytest.raises(Transform.UnsupportedFunctor):
        GK.matmul_batched(conf(64, 40, 32), a, b, None, cm(64, 40, 2, dtype=torch.float32), epilogue=Epilogue.BiasActivationResidual())
    with pytest.raises(Transform.UnsupportedFunctor):
        GK.matmul(conf(64, 40, 32), a, b, None, d, transform_shared_to_global_d=Transform.Elementwise(Transform.SiLU()))
