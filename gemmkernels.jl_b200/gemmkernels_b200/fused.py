"""Layer-level operators over gk_gemm_fused and gk_activation_gradient: products with a fused bias, activation and
residual (reached through `matmul` and `bind` with an Epilogue.Fused), products grouped by expert, and the
gradients of both.  The reference has no counterpart.

Everything is column-major and tokens are columns.  A group (an expert) owns the columns offsets[g] ..
offsets[g + 1] - 1; `offsets` stays on the device, so a router's output is used without a host synchronisation.
Its values are clamped to the matrix and made non-decreasing by a running maximum; columns outside every group are
neither computed nor written.
"""
from __future__ import annotations

import ctypes as C

from . import _lib as L
from . import arrays
from . import epilogue as Epilogue
from . import kernel as Kernel
from . import transform as Transform
from .config import Config, ConfigError, DimensionMismatch
from .matmul import BoundScratch, GemmKernelsError, _fold_transforms, _raise, _workspace_bytes, handle, lent_workspace, lower

_ACT = {Transform.Identity: L.GK_ACT_NONE, Transform.ReLU: L.GK_ACT_RELU, Transform.GELU: L.GK_ACT_GELU,
        Transform.SiLU: L.GK_ACT_SILU}


def _activation(f) -> int:
    if isinstance(f, Transform.Elementwise):
        f = f.f
    act = L.GK_ACT_NONE if f is None else _ACT.get(type(f))
    if act is None:
        raise Transform.UnsupportedFunctor(f"activation {f!r} is not None, ReLU, GELU or SiLU")
    return act


def _matrix(t, rows: int, cols: int, name: str, eltype=None):
    """Checks a column-major (rows, cols) array; returns its leading dimension."""
    if t.dim() != 2 or tuple(t.shape) != (rows, cols):
        raise DimensionMismatch(f"Dimensions do not match: {name} is {tuple(t.shape)}, expected ({rows}, {cols})")
    if eltype is not None and arrays.eltype_of(t) != eltype:
        raise ConfigError(f"{name} holds {arrays.eltype_of(t)}, expected {eltype}")
    if not arrays.is_col_major(t) or (cols > 1 and t.stride(1) < rows):
        raise GemmKernelsError(f"{name} must be stored column-major without overlapping columns")
    return arrays.leading_dimension(t)


def _offsets(t, groups: int):
    import torch
    if t.dtype not in (torch.int32, torch.int64):
        raise ConfigError(f"offsets must be Int32 or Int64, not {t.dtype}")
    if t.dim() != 1 or t.numel() != groups + 1 or not t.is_contiguous():
        raise DimensionMismatch(f"offsets has shape {tuple(t.shape)}, expected {groups + 1} consecutive values")
    return t.data_ptr(), L.GK_I32 if t.dtype == torch.int32 else L.GK_I64


def _one_device(*tensors):
    """The device all arrays are on (None entries are skipped)."""
    present = [t for t in tensors if t is not None]
    dev = present[0].device
    for t in present:
        if not t.is_cuda or t.device != dev:
            raise GemmKernelsError(f"all arrays must be on one CUDA device (found {t.device} beside {dev})")
    return dev


def _stack(t, groups: int, name: str):
    """(first matrix, elements between matrices) of a (rows, cols, groups) array."""
    if t.dim() != 3 or t.shape[2] != groups:
        raise DimensionMismatch(f"{name} has shape {tuple(t.shape)}, expected a last extent of {groups}")
    first = t[:, :, 0]
    if not arrays.is_col_major(first) or (first.shape[1] > 1 and first.stride(1) < first.shape[0]):
        raise GemmKernelsError(f"{name} must be stored column-major without overlapping columns")
    return first, (t.stride(2) if groups > 1 else 0)


class _Call:
    """A lowered call: descriptors, pointers and the arrays they point into."""

    def __init__(self, desc, fused, groups, ptrs, device, keep):
        self.desc, self.fused, self.groups, self.ptrs, self.device, self.keep = desc, fused, groups, ptrs, device, keep

    def _group_ref(self):
        return C.byref(self.groups) if self.groups is not None else None

    def _off_16_bytes(self):
        return (self.ptrs[0] or 0) % 16, (self.ptrs[1] or 0) % 16

    def query(self, h) -> L.GemmPlan:
        # The query has no addresses and takes them to be 16-byte aligned.  An operand that is not is planned (and its copy
        # sized) like one whose leading dimension is no multiple of 8.
        desc = L.GemmDesc.from_buffer_copy(self.desc)
        off_a, off_b = self._off_16_bytes()
        desc.lda += off_a != 0 and desc.lda % 8 == 0
        desc.ldb += off_b != 0 and desc.ldb % 8 == 0
        plan = L.GemmPlan()
        st = L.lib.gk_gemm_fused_query(h, C.byref(desc), C.byref(self.fused), self._group_ref(), C.byref(plan))
        if st != L.GK_OK:
            _raise(st)
        return plan

    def plan(self) -> L.GemmPlan:
        """`query` for the arrays' device, made current: planning sets attributes of its kernels."""
        import torch
        with torch.cuda.device(self.device):
            return self.query(handle(self.device.index))

    def workspace_bytes(self, h) -> int:
        d, gr = self.desc, self.groups
        ragged = gr.ragged if gr is not None else 0
        aligned = d.lda % 8 == 0 and d.ldb % 8 == 0 and (gr is None or gr.stride_a % 8 == 0) and self._off_16_bytes() == (0, 0)
        if aligned and ragged == L.GK_RAGGED_COLUMNS:
            return 0
        if aligned and ragged == 0 and not (d.m * d.n <= (1 << 22) and d.k >= 2048):
            return 0          # many output tiles, or a short K: nothing is cut along K
        return self.query(h).workspace_bytes

    function = L.lib.gk_gemm_fused

    def arguments(self, h, ws, ws_bytes):
        """Everything `function` takes but the stream."""
        return (h, C.byref(self.desc), C.byref(self.fused), self._group_ref(), *(C.c_void_p(p) for p in self.ptrs), ws, ws_bytes)


class _GradientCall:
    def __init__(self, desc, ptrs, device, keep):
        self.desc, self.ptrs, self.device, self.keep = desc, ptrs, device, keep

    def workspace_bytes(self, h) -> int:
        if self.ptrs[3] is None:
            return 0
        n = C.c_int64(0)
        st = L.lib.gk_activation_gradient_query(h, C.byref(self.desc), C.byref(n))
        if st != L.GK_OK:
            _raise(st)
        return n.value

    function = L.lib.gk_activation_gradient

    def arguments(self, h, ws, ws_bytes):
        return (h, C.byref(self.desc), *(C.c_void_p(p) for p in self.ptrs), ws, ws_bytes)


def _run(call, stream, workspace=None):
    import torch
    dev = call.device
    with torch.cuda.device(dev):
        h = handle(dev.index)
        s = stream if stream is not None else torch.cuda.current_stream(dev).cuda_stream
        with lent_workspace(dev, s, call.workspace_bytes(h) if workspace is None else 0) as lent:
            ws = workspace if workspace is not None else lent
            st = call.function(*call.arguments(h, ws.data_ptr() if ws is not None else None, _workspace_bytes(ws)), s)
    if st != L.GK_OK:
        _raise(st)


class BoundFused:
    """A layer-level operator with its arguments lowered once: calling the object enqueues it again on the same
    arrays for the cost of one FFI call.  It keeps the arrays alive and has a workspace on every stream it is
    called on (unless one was given); calls of one object write the same results and must not overlap on the GPU."""

    def __init__(self, call, workspace=None):
        import torch
        self._call, self._torch = call, torch
        self.device = call.device.index if call.device.index is not None else torch.cuda.current_device()
        with torch.cuda.device(self.device):
            self.handle = handle(self.device)
            need = call.workspace_bytes(self.handle) if workspace is None else 0
            self._scratch = BoundScratch(call.device, need) if need else None
        self._keep = workspace
        # converted once: ctypes would do it again for every argument of every call (8.8 -> 7 us of host time)
        self._arguments = call.arguments(self.handle, C.c_void_p(workspace.data_ptr() if workspace is not None else None),
                                         C.c_int64(_workspace_bytes(workspace)))
        self._without_scratch = self._arguments[:-2]
        self._function = call.function

    def __call__(self, stream=None):
        """Enqueues on `stream` (a raw CUDA stream handle) or on torch's current stream of the arrays' device."""
        cuda = self._torch.cuda
        if cuda.current_device() != self.device:
            with cuda.device(self.device):
                return self(stream)
        s = stream if stream is not None else cuda.current_stream(self.device).cuda_stream
        if self._scratch is None:
            st = self._function(*self._arguments, s)
        else:
            address, buffer = self._scratch.on(s, stream is None)
            st = self._function(*self._without_scratch, address, self._scratch.nbytes, s)
        if st != L.GK_OK:
            _raise(st)


# ------------------------------------------------------------------------------------------------
# lowering
# ------------------------------------------------------------------------------------------------
def _lower_epilogue(epilogue, hooks: dict, act_hook: int, d, m: int, n: int, groups: int):
    """-> (FusedDesc, bias group stride, arrays to keep alive).  groups == 0: a plain product."""
    import torch
    fu = L.FusedDesc()
    if not isinstance(epilogue, Epilogue.Default):
        _fold_transforms(hooks, True)      # refuses what would have to run between the product and the bias, or scale both
    if isinstance(epilogue, Epilogue.Fused) and act_hook != L.GK_ACT_NONE:
        raise Transform.UnsupportedFunctor("the fused epilogues carry their own activation: leave the activation hooks empty")
    bias, axis, z = None, "row", None
    if isinstance(epilogue, Epilogue.BiasActivationResidual):
        fu.form, fu.activation = L.GK_FUSED_RESIDUAL, _activation(epilogue.activation)
        bias, axis, z = epilogue.bias, epilogue.axis, epilogue.preactivation
    elif isinstance(epilogue, Epilogue.ActivationGradient):
        fu.form, fu.activation, z = L.GK_FUSED_GRADIENT, _activation(epilogue.activation), epilogue.preactivation
        if z is None:
            raise GemmKernelsError("Epilogue.ActivationGradient needs the pre-activation")
    elif isinstance(epilogue, Epilogue.Bias):
        fu.form, fu.activation, bias, axis = L.GK_FUSED_STANDARD, act_hook, epilogue.bias, epilogue.axis
    elif isinstance(epilogue, Epilogue.Default):
        fu.form, fu.activation = L.GK_FUSED_STANDARD, act_hook
    else:
        raise Transform.UnsupportedFunctor(f"epilogue {epilogue!r} is not one of Epilogue's")
    stride = 0
    if bias is not None:
        if isinstance(bias, int):
            raise GemmKernelsError("the layer-level operators take the bias as an array, not as an address")
        if bias.dtype != torch.float32:
            raise Transform.UnsupportedFunctor("the bias must be Float32")
        if groups and axis == "row":
            if bias.dim() != 2 or tuple(bias.shape) != (m, groups):
                raise DimensionMismatch(f"bias has shape {tuple(bias.shape)}, expected ({m}, {groups})")
            stride = bias.stride(1) if groups > 1 else 0
        elif bias.dim() != 1 or bias.numel() != (m if axis == "row" else n):
            raise DimensionMismatch(f"bias has shape {tuple(bias.shape)}, expected ({m if axis == 'row' else n},)")
        if bias.numel() and bias.shape[0] > 1 and bias.stride(0) != 1:
            raise GemmKernelsError("the values of a bias must be consecutive")
        fu.bias, fu.bias_axis = bias.data_ptr(), L.GK_BIAS_ROW if axis == "row" else L.GK_BIAS_COL
    if z is not None:
        fu.ldz = _matrix(z, m, n, "the pre-activation", arrays.eltype_of(d))
        fu.z = z.data_ptr()
    return fu, stride, (bias, z)


def _check_matrices(**arrays_by_name):
    for name, t in arrays_by_name.items():
        if t is not None and t.dim() == 2 and t.shape[1] > 1 and t.stride(1) < t.shape[0]:
            raise GemmKernelsError(f"{name} must be stored column-major without overlapping columns")


def lower_fused(conf: Config, a, b, c, d, hooks: dict, epilogue, kernel) -> _Call:
    """One product with a fused epilogue.  Pure host logic."""
    desc, epi, ptrs = lower(conf, a, b, c, d, hooks, Epilogue.Default(), kernel)
    m, n = desc.m, desc.n
    _check_matrices(A=a, B=b, C=c, D=d)
    fu, _, keep = _lower_epilogue(epilogue, hooks, epi.activation, d, m, n, 0)
    dev = _one_device(d, a, b, c, *keep)
    return _Call(desc, fu, None, ptrs, dev, (a, b, c, d, epilogue) + keep)


def lower_grouped(conf: Config, a, b, c, d, offsets, hooks: dict, epilogue, kernel) -> _Call:
    """D[:, J_g] = epilogue(A_g * B[:, J_g]).  Pure host logic."""
    if a.dim() != 3 or a.shape[2] < 1:
        raise DimensionMismatch(f"matmul_grouped: A has shape {tuple(a.shape)}, expected one matrix per group in the last extent")
    groups = a.shape[2]
    a0, stride_a = _stack(a, groups, "A")
    desc, epi, ptrs = lower(conf, a0, b, c, d, hooks, Epilogue.Default(), kernel)
    m, n = desc.m, desc.n
    _check_matrices(B=b, C=c, D=d)
    fu, stride_bias, keep = _lower_epilogue(epilogue, hooks, epi.activation, d, m, n, groups)
    gr = L.GroupDesc(ragged=L.GK_RAGGED_COLUMNS, groups=groups, stride_a=stride_a, stride_bias=stride_bias)
    gr.offsets, gr.offsets_dtype = _offsets(offsets, groups)
    dev = _one_device(d, a, b, c, offsets, *keep)
    return _Call(desc, fu, gr, ptrs, dev, (a, b, c, d, offsets, epilogue) + keep)


def lower_grouped_outer(conf: Config, a, b, c, d, offsets, hooks: dict, kernel) -> _Call:
    """D_g = A[:, J_g] * B[J_g, :] + C_g.  Pure host logic."""
    if d.dim() != 3 or d.shape[2] < 1:
        raise DimensionMismatch(f"matmul_grouped_outer: D has shape {tuple(d.shape)}, expected one matrix per group in the last extent")
    groups = d.shape[2]
    d0, stride_d = _stack(d, groups, "D")
    c0, stride_c = (None, 0) if c is None else _stack(c, groups, "C")
    desc, epi, ptrs = lower(conf, a, b, c0, d0, hooks, Epilogue.Default(), kernel)
    if epi.activation != L.GK_ACT_NONE:
        raise Transform.UnsupportedFunctor("matmul_grouped_outer applies alpha, beta and C only")
    _check_matrices(A=a, B=b)
    gr = L.GroupDesc(ragged=L.GK_RAGGED_DEPTH, groups=groups, stride_c=stride_c, stride_d=stride_d)
    gr.offsets, gr.offsets_dtype = _offsets(offsets, groups)
    dev = _one_device(d, a, b, c, offsets)
    return _Call(desc, L.FusedDesc(), gr, ptrs, dev, (a, b, c, d, offsets))


def _hooks(transforms: dict) -> dict:
    return {k.replace("transform_", ""): v for k, v in transforms.items()}


# ------------------------------------------------------------------------------------------------
# products grouped by expert
# ------------------------------------------------------------------------------------------------
def matmul_grouped(conf: Config, a, b, c, d, offsets, *, epilogue=None, kernel=Kernel.matmul_singlestage, stream=None,
                   workspace=None, **transforms):
    """D[:, J_g] = epilogue(A[:, :, g] * B[:, J_g] + C[:, J_g]) for every group g, in one launch.

    `a` is (M, K, groups) - or (K, M, groups) with a RowMajor layout, which makes this the input gradient of the same
    layer; its groups may lie any distance apart.  `b`, `c` and `d` are as for `matmul` with N = all columns there are
    (`conf.matmul_shape`); `offsets` is a device array of groups + 1 Int32 or Int64 values, of which group g takes the
    columns offsets[g] .. offsets[g + 1] - 1.  `epilogue` is Epilogue.Default, Epilogue.Bias with a bias of (M, groups)
    and axis="row", or one of the fused ones.  Columns outside every group are left as they were.  Operands
    whose columns are not 16-byte aligned are copied into the workspace first (`grouped_query` reports its size; the
    package lends one when it is None); when it is too small, slower bounds-checked loads read them."""
    _run(lower_grouped(conf, a, b, c, d, offsets, _hooks(transforms), epilogue or Epilogue.Default(), kernel), stream, workspace)


def bind_grouped(conf: Config, a, b, c, d, offsets, *, epilogue=None, kernel=Kernel.matmul_singlestage, workspace=None,
                 **transforms) -> BoundFused:
    """`matmul_grouped` with its arguments lowered once (and a workspace of its own, where it uses one)."""
    return BoundFused(lower_grouped(conf, a, b, c, d, offsets, _hooks(transforms), epilogue or Epilogue.Default(), kernel), workspace)


def matmul_grouped_outer(conf: Config, a, b, c, d, offsets, *, kernel=Kernel.matmul_singlestage, stream=None, workspace=None,
                         **transforms):
    """D[:, :, g] = A[:, J_g] * B[J_g, :] + C[:, :, g] for every group g: products whose contracted index is ragged,
    such as the weight gradients dW_g = dY[:, J_g] * X[:, J_g]'.

    `conf.matmul_shape` is (M, N, K = all columns there are); `a` is (M, K), `b` with a RowMajor layout is (N, K) - the
    layouts in which both run through TMA; the others read one column at a time and are slower.  `c` may be None or
    `d` itself (accumulation).  A group without columns gets beta * C.  `workspace`: uint8, what `grouped_query`
    reports; the package lends one when it is None."""
    _run(lower_grouped_outer(conf, a, b, c, d, offsets, _hooks(transforms), kernel), stream, workspace)


def bind_grouped_outer(conf: Config, a, b, c, d, offsets, *, kernel=Kernel.matmul_singlestage, workspace=None,
                       **transforms) -> BoundFused:
    """`matmul_grouped_outer` with its arguments lowered once (and a workspace of its own)."""
    return BoundFused(lower_grouped_outer(conf, a, b, c, d, offsets, _hooks(transforms), kernel), workspace)


def grouped_query(conf: Config, a, b, c, d, offsets, *, epilogue=None, kernel=Kernel.matmul_singlestage, **transforms) -> L.GemmPlan:
    """What `matmul_grouped` (a 3-D `a`) or `matmul_grouped_outer` (a 3-D `d`) would launch; launches nothing."""
    call = lower_grouped_outer(conf, a, b, c, d, offsets, _hooks(transforms), kernel) if d.dim() == 3 else \
        lower_grouped(conf, a, b, c, d, offsets, _hooks(transforms), epilogue or Epilogue.Default(), kernel)
    return call.plan()


# ------------------------------------------------------------------------------------------------
# activation gradient
# ------------------------------------------------------------------------------------------------
def lower_activation_gradient(dz, dd, z, activation, bias_gradient, offsets) -> _GradientCall:
    import torch
    if dd.dim() != 2:
        raise DimensionMismatch(f"dD has shape {tuple(dd.shape)}, expected a matrix")
    m, n = dd.shape
    et = arrays.eltype_of(dd)
    if dz is None and bias_gradient is None:
        raise GemmKernelsError("neither dZ nor the bias gradient is wanted")
    act = _activation(activation)
    if z is None and act != L.GK_ACT_NONE:
        raise GemmKernelsError("an activation needs the pre-activation Z")
    d = L.ActivationGradientDesc(dtype=et.gk, m=m, n=n, activation=act, groups=1)
    d.ld_dd = _matrix(dd, m, n, "dD")
    d.ld_z = _matrix(z, m, n, "Z", et) if z is not None else max(m, 1)
    d.ld_dz = _matrix(dz, m, n, "dZ", et) if dz is not None else max(m, 1)
    d.ld_db = max(m, 1)
    if offsets is not None:
        if offsets.dim() != 1 or offsets.numel() < 2:
            raise DimensionMismatch(f"offsets has shape {tuple(offsets.shape)}, expected one value more than there are groups")
        d.groups = offsets.numel() - 1
        d.offsets, d.offsets_dtype = _offsets(offsets, d.groups)
    if bias_gradient is not None:
        if bias_gradient.dtype != torch.float32:
            raise ConfigError("the bias gradient is Float32")
        bg = bias_gradient[:, None] if bias_gradient.dim() == 1 else bias_gradient
        d.ld_db = _matrix(bg, m, d.groups, "the bias gradient")
    dev = _one_device(dd, z, dz, bias_gradient, offsets)
    ptr = [t.data_ptr() if t is not None else None for t in (dd, z, dz, bias_gradient)]
    return _GradientCall(d, ptr, dev, (dd, z, dz, bias_gradient, offsets))


def activation_gradient_(dz, dd, z, activation=None, *, bias_gradient=None, offsets=None, stream=None):
    """dZ = dD * act'(Z) and, with `bias_gradient`, the sums of dZ over the columns (of each group): the backward pass
    of D = act(Z), Z = A*B + bias.

    All matrices are column-major M x N of one type; `dz` may be `dd` or `z` itself, or None when only the sums are
    wanted.  `bias_gradient` is Float32, (M,) - or (M, groups) with `offsets`, the device array of `matmul_grouped`;
    columns outside every group are then left alone, and a group without columns gets zero.  Returns `dz`."""
    _run(lower_activation_gradient(dz, dd, z, activation, bias_gradient, offsets), stream)
    return dz


def bind_activation_gradient(dz, dd, z, activation=None, *, bias_gradient=None, offsets=None) -> BoundFused:
    """`activation_gradient_` with its arguments lowered once (and a workspace of its own)."""
    return BoundFused(lower_activation_gradient(dz, dd, z, activation, bias_gradient, offsets))
