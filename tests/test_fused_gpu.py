"""Layer-level operators on the GPU against their formulas in 64 bits.

Tolerances.  Where the inputs are small integers every product and every partial sum is an integer below 2^24, FP32
arithmetic is exact and the result must be equal.  Elsewhere, with u the half step of D's type (eps / 2), an element
may be off by
    u * |D|  +  (1 + u) * e  +  tiny,    e = 1.13 * ((K + 4) * 2^-23 * (|A| |B| + |bias|) + 8 * 2^-23 * (|x| + 1)),
the rounding of D, and in FP32 before it: K products that are exact in FP32, added with at most one ulp (2^-23) per
addition, then the activation, whose slope is at most 1.13 and which is evaluated in FP32 (a few ulp of its argument
and of its value; 2^-21 for the hardware exponential, inside the factor 8).  tiny is the type's smallest subnormal.
"""
import math

import pytest
import torch

import gemmkernels_b200 as GK
from gemmkernels_b200 import Epilogue, Layout, Operator, Transform

pytestmark = pytest.mark.gpu

F16, BF16, F32 = GK.Float16, GK.BFloat16, GK.Float32
ET = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32}
ACT = {None: None, "relu": Transform.ReLU(), "gelu": Transform.GELU(), "silu": Transform.SiLU()}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def cm(t):
    """The same values in column-major storage."""
    return t.permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim())))


def ints(g, *shape, dtype=torch.float16, lo=-2, hi=2):
    return cm(torch.randint(lo, hi + 1, shape, generator=g, device="cuda").to(dtype))


def normal(g, *shape, dtype=torch.float16, scale=1.0):
    return cm((torch.randn(shape, generator=g, device="cuda") * scale).to(dtype))


def padded(t, extra):
    """The same matrix with `extra` rows between its columns."""
    buf = torch.full((t.shape[1], t.shape[0] + extra), float("nan"), dtype=t.dtype, device=t.device)
    view = buf.T[: t.shape[0]]
    view.copy_(t)
    return view


def conf(m, n, k, dt, out, ta=False, tb=False, residual=False, **kw):
    t, o = ET[dt], ET[out]
    return GK.get_config(gemm_shape=(m, n, k), operator=Operator.TCGen05Operator[t, F32], is_a_col_major=not ta, is_b_col_major=not tb,
                         global_a_layout=(Layout.RowMajor if ta else Layout.ColMajor)[t],
                         global_b_layout=(Layout.RowMajor if tb else Layout.ColMajor)[t],
                         global_c_layout=(Layout.ColMajor if residual else Layout.Zero)[o], global_d_layout=Layout.ColMajor[o], **kw)


def act64(x, name):
    if name == "relu":
        return x.clamp(min=0)
    if name == "gelu":
        return 0.5 * x * torch.special.erfc(-x / math.sqrt(2))
    if name == "silu":
        return x * torch.sigmoid(x)
    return x


def grad64(x, name):
    if name == "relu":
        return (x > 0).double()
    if name == "gelu":
        return 0.5 * torch.special.erfc(-x / math.sqrt(2)) + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(x)
        return s * (1 + x * (1 - s))
    return torch.ones_like(x)


def close(got, want, e, what="D"):
    fi = torch.finfo(got.dtype)
    u = fi.eps / 2
    tol = u * want.abs() + (1 + u) * e + fi.smallest_normal * fi.eps
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got.double() - want).abs().max()):.3e} " \
        f"at tolerance {float(tol[bad].min()):.3e}, first {bad.nonzero()[0].tolist()}"


def err(k, mag, x, slope=1.13):
    return slope * ((k + 4) * 2.0 ** -23 * mag + 8 * 2.0 ** -23 * (x.abs() + 1))


def done():
    torch.cuda.synchronize()
    GK.poll_status()


def offsets_of(counts, first=0, dtype=torch.int32):
    o = [first]
    for c in counts:
        o.append(o[-1] + c)
    return torch.tensor(o, dtype=dtype, device="cuda"), o


# ------------------------------------------------------------------------------------------------
# one product, fused epilogue
# ------------------------------------------------------------------------------------------------
SHAPES = [(128, 256, 64), (256, 512, 128), (1, 1, 1), (3, 2, 5), (64, 1, 512), (72, 2, 264), (136, 4, 1000), (130, 3, 96), (520, 5, 304),
          (1000, 77, 111), (264, 300, 72), (511, 513, 129), (2048, 640, 256), (128, 32, 4096)]


@pytest.mark.parametrize("ta,tb", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_fused_product_of_integers_is_exact(m, n, k, ta, tb, dt):
    g = gen(m * 7 + n * 3 + k)
    a, b, r = ints(g, m, k, dtype=dt), ints(g, k, n, dtype=dt), ints(g, m, n, dtype=torch.float32, hi=50)
    for axis in ("row", "col"):
        bias = ints(g, m if axis == "row" else n, dtype=torch.float32, hi=9)
        d, z = torch.full_like(r, -7.0), torch.full_like(r, -7.0)
        GK.matmul(conf(m, n, k, dt, torch.float32, ta, tb, True), cm(a.T) if ta else a, cm(b.T) if tb else b, r, d,
                  epilogue=Epilogue.BiasActivationResidual(bias, axis, ACT["relu"], z))
        done()
        x = a.double() @ b.double() + (bias.double()[:, None] if axis == "row" else bias.double()[None, :])
        assert torch.equal(z.double(), x)
        assert torch.equal(d.double(), x.clamp(min=0) + r.double())


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 2, 3, 7, 33, 257])
def test_fused_epilogue_values(n, out, act):
    dt = torch.float16 if out == torch.float16 else torch.bfloat16
    m, k = 328, 520
    g = gen(n)
    a, b, r = normal(g, m, k, dtype=dt, scale=2 * k ** -0.5), normal(g, k, n, dtype=dt), padded(normal(g, m, n, dtype=out), 5)
    bias = normal(g, m, dtype=torch.float32)
    mag = a.double().abs() @ b.double().abs() + bias.double().abs()[:, None]
    x = 1.5 * (a.double() @ b.double()) + bias.double()[:, None]
    for keep in (False, True):
        d = padded(torch.zeros_like(r), 3)
        z = padded(torch.zeros_like(r), 8) if keep else None
        GK.matmul(conf(m, n, k, dt, out, residual=True), a, b, r, d, transform_shared_to_regs_a=Transform.Elementwise(Transform.Scale(1.5)),
                  transform_shared_to_regs_c=Transform.Elementwise(Transform.Scale(-0.5)),
                  epilogue=Epilogue.BiasActivationResidual(bias, "row", ACT[act], z))
        done()
        close(d, act64(x, act) - 0.5 * r.double(), err(k, 1.5 * mag, x) + 2.0 ** -23 * r.double().abs())
        if keep:
            close(z, x, err(k, 1.5 * mag, x), "Z")


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(264, 1, 512), (264, 130, 96), (77, 45, 33), (512, 600, 256)])
def test_gradient_epilogue(m, n, k, dt, act):
    g = gen(m + n)
    w, dy, z = normal(g, k, m, dtype=dt, scale=k ** -0.5), normal(g, k, n, dtype=dt), normal(g, m, n, dtype=dt, scale=2.0)
    if act == "relu":
        z[::3, ::2] = 0.0
    want = (w.double().T @ dy.double()) * grad64(z.double(), act)
    mag = w.double().abs().T @ dy.double().abs()
    for inplace in (False, True):
        d = z if inplace else torch.zeros_like(z)       # D may be Z itself
        GK.matmul(conf(m, n, k, dt, dt, ta=True), w, dy, None, d, epilogue=Epilogue.ActivationGradient(z, ACT[act]))
        done()
        # act' is evaluated in FP32 to a few ulp of 1 (its value is below 1.13)
        close(d, want, err(k, mag, want) + 16 * 2.0 ** -23 * mag)


def test_gradient_epilogue_adds_c_before_the_slope():
    g = gen(3)
    m, n, k = 200, 70, 64
    a, b, c, z = ints(g, m, k), ints(g, k, n), ints(g, m, n, dtype=torch.float32), ints(g, m, n, dtype=torch.float32)
    GK.matmul(conf(m, n, k, torch.float16, torch.float32, residual=True), a, b, c, c, epilogue=Epilogue.ActivationGradient(z, ACT["relu"]),
              transform_shared_to_regs_c=Transform.Elementwise(Transform.Scale(2.0)))
    done()
    g = gen(3)
    a, b, c0 = ints(g, m, k), ints(g, k, n), ints(g, m, n, dtype=torch.float32)
    assert torch.equal(c.double(), (a.double() @ b.double() + 2 * c0.double()) * (z > 0))


def test_infinite_preactivations_have_the_limit_slope():
    m, n, k = 64, 32, 64
    a, b = torch.ones(m, k, dtype=torch.float16, device="cuda").T.contiguous().T, cm(torch.ones(k, n, dtype=torch.float16, device="cuda"))
    z = cm(torch.full((m, n), float("inf"), dtype=torch.float16, device="cuda"))
    z[:, ::2] = float("-inf")
    for act in ("relu", "gelu", "silu"):
        d = torch.zeros_like(z)
        GK.matmul(conf(m, n, k, torch.float16, torch.float16), a, b, None, d, epilogue=Epilogue.ActivationGradient(z, ACT[act]))
        dz = torch.zeros_like(z)
        GK.activation_gradient_(dz, torch.ones_like(z), z, ACT[act])
        done()
        assert torch.equal(d[:, 1::2], torch.full_like(d[:, 1::2], k)) and not d[:, ::2].any(), act
        assert torch.equal(dz[:, 1::2], torch.ones_like(dz[:, 1::2])) and not dz[:, ::2].any(), act


def test_nan_reaches_its_own_column_and_no_other():
    g = gen(5)
    m, n, k = 256, 40, 128
    for cols in (1, 3, n):
        a, b = normal(g, m, k, scale=0.1), normal(g, k, cols)
        b[3, cols - 1] = float("nan")
        d = torch.zeros((cols, m), dtype=torch.float16, device="cuda").T
        GK.matmul(conf(m, cols, k, torch.float16, torch.float16), a, b, None, d, epilogue=Epilogue.BiasActivationResidual(activation=ACT["relu"]))
        done()
        assert d[:, cols - 1].isnan().all() and not d[:, : cols - 1].isnan().any()


def test_nothing_to_multiply():
    g = gen(6)
    m, n = 200, 50
    bias, r = ints(g, m, dtype=torch.float32), ints(g, m, n, dtype=torch.float32)
    bad = cm(torch.full((m, 64), float("nan"), dtype=torch.float16, device="cuda"))
    badb = cm(torch.full((64, n), float("nan"), dtype=torch.float16, device="cuda"))
    want = bias.double()[:, None].clamp(min=0) + r.double()
    for k, alpha in ((64, 0.0), (0, 1.0)):
        d, z = torch.zeros_like(r), torch.zeros_like(r)
        cf = conf(m, n, k, torch.float16, torch.float32, residual=True)
        GK.matmul(cf, bad[:, :k], badb[:k], r, d, transform_shared_to_regs_a=Transform.Elementwise(Transform.Scale(alpha)),
                  epilogue=Epilogue.BiasActivationResidual(bias, "row", ACT["relu"], z))
        done()
        assert torch.equal(d.double(), want) and torch.equal(z.double(), bias.double()[:, None].expand(m, n))
    for shape in ((0, n), (m, 0)):
        d = torch.zeros((shape[1], shape[0]), dtype=torch.float32, device="cuda").T
        GK.matmul(conf(*shape, 64, torch.float16, torch.float32), bad[: shape[0]], badb[:, : shape[1]], None, d,
                  epilogue=Epilogue.BiasActivationResidual())
    done()


@pytest.mark.parametrize("m,n,k", [(256, 256, 16384), (512, 96, 8192), (1024, 7, 4096)])
@pytest.mark.parametrize("form", ["residual", "gradient"])
def test_fused_split_along_k(m, n, k, form):
    """Few output tiles and a long K: partial sums in the workspace, the epilogue in the reduction."""
    g = gen(k)
    a, b = ints(g, m, k, lo=-1, hi=1), ints(g, k, n, lo=-1, hi=1)
    r, z = ints(g, m, n, dtype=torch.float32), ints(g, m, n, dtype=torch.float32)
    bias = ints(g, m, dtype=torch.float32)
    x = a.double() @ b.double()
    d = torch.zeros_like(r)
    if form == "residual":
        epi, cc, want = Epilogue.BiasActivationResidual(bias, "row", ACT["relu"], z), r, (x + bias.double()[:, None]).clamp(min=0) + r.double()
    else:
        epi, cc, want = Epilogue.ActivationGradient(z, ACT["relu"]), None, x * (z > 0)
    cf = conf(m, n, k, torch.float16, torch.float32, residual=cc is not None)
    plan = GK.query(cf, a, b, cc, d, epilogue=epi)
    assert plan.workspace_bytes > 0 or plan.kernel == 6
    GK.bind(cf, a, b, cc, d, epilogue=epi)()
    done()
    assert torch.equal(d.double(), want)
    if form == "residual":
        assert torch.equal(z.double(), x + bias.double()[:, None])
    d2 = torch.zeros_like(r)
    small = torch.zeros(256, dtype=torch.uint8, device="cuda")       # too small to split: the same product, unsplit
    GK.matmul(cf, a, b, cc, d2, epilogue=epi, workspace=small)
    done()
    assert torch.equal(d2.double(), want) and not small.any()


@pytest.mark.parametrize("tile_n,cg", [(32, 1), (64, 1), (128, 1), (256, 1), (128, 2), (256, 2), (512, 2)])
@pytest.mark.parametrize("m", [700, 704])
def test_fused_tile_shapes(tile_n, cg, m):
    g = gen(tile_n)
    n, k = 1100, 1088
    a, b, r = ints(g, m, k), ints(g, k, n), ints(g, m, n, dtype=torch.float32)
    d, z = torch.zeros_like(r), torch.zeros_like(r)

    GK.matmul(conf(m, n, k, torch.float16, torch.float32, residual=True, tile_n=tile_n, cta_group=cg), a, b, r, d,
              epilogue=Epilogue.BiasActivationResidual(None, "row", ACT["relu"], z))
    done()
    x = a.double() @ b.double()
    assert torch.equal(z.double(), x) and torch.equal(d.double(), x.clamp(min=0) + r.double())


@pytest.mark.parametrize("ta,tb", [(False, False), (True, True)])
@pytest.mark.parametrize("m,n,k", [(77, 45, 33), (300, 257, 1111), (130, 70, 6)])
def test_unaligned_operands_with_and_without_room_for_their_copies(m, n, k, ta, tb):
    g = gen(m)
    a, b, r = ints(g, m, k), ints(g, k, n), ints(g, m, n, dtype=torch.float32)
    aw, bw = cm(a.T) if ta else a, cm(b.T) if tb else b
    cf = conf(m, n, k, torch.float16, torch.float32, ta, tb, True)
    epi = Epilogue.BiasActivationResidual(activation=ACT["relu"])
    want = (a.double() @ b.double()).clamp(min=0) + r.double()
    need = GK.query(cf, aw, bw, r, torch.zeros_like(r), epilogue=epi).workspace_bytes
    assert need > 0
    for room in (need, 256):
        ws = torch.full((need + 256,), 5, dtype=torch.uint8, device="cuda")
        d = torch.zeros_like(r)
        GK.matmul(cf, aw, bw, r, d, epilogue=epi, workspace=ws[:room])
        done()
        assert torch.equal(d.double(), want) and (ws[room:] == 5).all()
    # operands that start in the middle of an allocation, two bytes past a 16-byte boundary
    big = torch.zeros(a.numel() + 64, dtype=torch.float16, device="cuda")
    shifted = big[1: 1 + a.numel()].view(aw.shape[1], aw.shape[0]).T
    shifted.copy_(aw)
    d = torch.zeros_like(r)
    GK.matmul(cf, shifted, bw, r, d, epilogue=epi)
    done()
    assert torch.equal(d.double(), want)


@pytest.mark.parametrize("n", [1, 2, 3, 4])
@pytest.mark.parametrize("ta,tb", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("m,k", [(1, 1), (7, 9), (65, 1023), (200, 257), (129, 2055), (64, 300)])
def test_few_columns_of_any_size_and_order(m, k, n, ta, tb):
    g = gen(m + k + n)
    a, b, r = ints(g, m, k), ints(g, k, n), ints(g, m, n, dtype=torch.float32)
    bias = ints(g, m, dtype=torch.float32)
    poison = torch.full((a.numel() + 40,), float("nan"), dtype=torch.float16, device="cuda")     # NaN around A
    aw = cm(a.T) if ta else a
    view = poison[11: 11 + a.numel()].view(aw.shape[1], aw.shape[0]).T
    view.copy_(aw)
    for src in (aw, view):
        d = torch.full_like(r, -9.0)
        cf = conf(m, n, k, torch.float16, torch.float32, ta, tb, True)
        epi = Epilogue.BiasActivationResidual(bias, activation=ACT["relu"])
        assert GK.query(cf, src, cm(b.T) if tb else b, r, d, epilogue=epi).kernel == 6
        GK.matmul(cf, src, cm(b.T) if tb else b, r, d, epilogue=epi)
        done()
        assert torch.equal(d.double(), (a.double() @ b.double() + bias.double()[:, None]).clamp(min=0) + r.double())


# ------------------------------------------------------------------------------------------------
# products grouped by expert
# ------------------------------------------------------------------------------------------------
COUNTS = [[5], [0, 0, 0], [1, 0, 2, 1], [3, 9, 1, 0, 4], [1] * 40, [0, 31, 32, 33, 0, 0, 129, 64, 1], [300, 0, 17, 256], [7, 700, 2, 0, 513, 1]]


def run_grouped(counts, m, k, dt, ta, tb, first=0, tail=0, offdt=torch.int32, out=torch.float32, seed=0, epilogue="residual", **kw):
    g = gen(seed + len(counts))
    offsets, o = offsets_of(counts, first, offdt)
    G, total = len(counts), o[-1] + tail
    w, x = ints(g, m, k, G, dtype=dt), ints(g, k, total, dtype=dt)
    bias, r = ints(g, m, G, dtype=torch.float32, hi=9), ints(g, m, total, dtype=out, hi=20)
    d, z = torch.full_like(r, -99.0), torch.full_like(r, -99.0)
    aw = cm(w.permute(1, 0, 2)) if ta else w
    GK.matmul_grouped(conf(m, total, k, dt, out, ta, tb, True, **kw), aw, cm(x.T) if tb else x, r, d, offsets,
                      epilogue=Epilogue.BiasActivationResidual(bias, "row", ACT["relu"], z))
    done()
    wd, wz = torch.full_like(r, -99.0).double(), torch.full_like(r, -99.0).double()
    for i in range(G):
        c = slice(o[i], o[i + 1])
        wz[:, c] = w[:, :, i].double() @ x[:, c].double() + bias[:, i:i + 1].double()
        wd[:, c] = wz[:, c].clamp(min=0) + r[:, c].double()
    assert torch.equal(z.double(), wz), f"Z: first wrong column {(z.double() != wz).any(0).nonzero()[0].item()}"
    assert torch.equal(d.double(), wd), f"D: first wrong column {(d.double() != wd).any(0).nonzero()[0].item()}"


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("ta,tb", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("m,k", [(128, 64), (264, 520), (77, 45)])
def test_grouped_product_of_integers_is_exact(counts, m, k, ta, tb):
    dt = torch.bfloat16 if m == 264 else torch.float16
    run_grouped(counts, m, k, dt, ta, tb)
    run_grouped(counts, m, k, dt, ta, tb, first=3, tail=13, offdt=torch.int64)


@pytest.mark.parametrize("ta,tb", [(False, False), (True, True)])
@pytest.mark.parametrize("counts", [[40, 0, 300, 1], [2, 0, 3, 1]])
def test_grouped_unaligned_with_and_without_room(counts, ta, tb):
    g = gen(51)
    m, k, G = 77, 45, 4
    offsets, o = offsets_of(counts, first=1)
    total = o[-1] + 2
    w, x = ints(g, m, k, G), ints(g, k, total)
    want = cm(torch.full((m, total), -9.0, device="cuda")).double()
    for i in range(G):
        want[:, o[i]:o[i + 1]] = w[:, :, i].double() @ x[:, o[i]:o[i + 1]].double()
    aw, xw = cm(w.permute(1, 0, 2)) if ta else w, cm(x.T) if tb else x
    cf = conf(m, total, k, torch.float16, torch.float32, ta, tb)
    for room in (None, 256):
        d = cm(torch.full((m, total), -9.0, device="cuda"))
        GK.matmul_grouped(cf, aw, xw, None, d, offsets, workspace=None if room is None else torch.zeros(room, dtype=torch.uint8, device="cuda"))
        done()
        assert torch.equal(d.double(), want)


@pytest.mark.parametrize("tile_n,cg", [(32, 1), (64, 1), (128, 1), (256, 1), (128, 2), (256, 2)])
@pytest.mark.parametrize("tb", [False, True])
def test_grouped_tile_shapes(tile_n, cg, tb):
    if tb and (tile_n // cg) % 64:
        pytest.skip("a transposed B is loaded 64 columns at a time")
    run_grouped([40, 0, 300, 1, 129, 77, 0, 5], 392, 328, torch.float16, False, tb, first=5, tail=9, tile_n=tile_n, cta_group=cg)


def test_grouped_many_groups():
    counts = [(i * 7) % 5 for i in range(1024)]
    run_grouped(counts, 72, 64, torch.float16, True, False, tail=1)


def test_grouped_standard_epilogues_and_shared_weights():
    g = gen(11)
    m, k, counts = 200, 96, [4, 0, 60, 130]
    offsets, o = offsets_of(counts)
    w, x, bias = ints(g, m, k), ints(g, k, o[-1]), ints(g, m, 4, dtype=torch.float32)
    c = ints(g, m, o[-1], dtype=torch.float32)
    shared = w[:, :, None].expand(m, k, 4)             # one matrix for all groups: stride 0
    want = (2 * (w.double() @ x.double()) + 3 * c.double())
    owner = torch.repeat_interleave(torch.arange(4, device="cuda"), torch.tensor(counts, device="cuda"))
    want = (want + bias.double()[:, owner]).clamp(min=0)
    GK.matmul_grouped(conf(m, o[-1], k, torch.float16, torch.float32, residual=True), shared, x, c, c, offsets,
                      epilogue=Epilogue.Bias(bias, axis="row"), transform_shared_to_global_d=Transform.Elementwise(Transform.ReLU()),
                      transform_shared_to_regs_a=Transform.Elementwise(Transform.Scale(2.0)),
                      transform_shared_to_regs_c=Transform.Elementwise(Transform.Scale(3.0)))
    done()
    assert torch.equal(c.double(), want)


@pytest.mark.parametrize("counts", [[2, 0, 1, 5], [90, 0, 260, 33]])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_grouped_input_gradient(counts, act):
    g = gen(12)
    m, k = 264, 328
    offsets, o = offsets_of(counts)
    w, dy, z = normal(g, k, m, 4, dtype=torch.bfloat16, scale=k ** -0.5), normal(g, k, o[-1], dtype=torch.bfloat16), normal(g, m, o[-1], dtype=torch.bfloat16)
    d = torch.zeros_like(z)
    GK.matmul_grouped(conf(m, o[-1], k, torch.bfloat16, torch.bfloat16, ta=True), w, dy, None, d, offsets,
                      epilogue=Epilogue.ActivationGradient(z, ACT[act]))
    done()
    for i in range(4):
        c = slice(o[i], o[i + 1])
        mag = w[:, :, i].double().abs().T @ dy[:, c].double().abs()
        want = (w[:, :, i].double().T @ dy[:, c].double()) * grad64(z[:, c].double(), act)
        close(d[:, c], want, err(k, mag, want) + 16 * 2.0 ** -23 * mag, f"group {i}")


BAD_OFFSETS = [[0, 30, 10, 50, 60], [-5, 20, 20, 1000, 2000], [2 ** 31 - 1] * 5, [-2 ** 31] * 5, [60, 50, 40, 30, 20], [0, 0, 0, 0, 60]]


@pytest.mark.parametrize("values", BAD_OFFSETS)
@pytest.mark.parametrize("tokens", [60, 8])
def test_any_offsets_stay_inside_the_matrix(values, tokens):
    """Clamped to [0, columns], then the running maximum."""
    g = gen(13)
    m, k = 136, 72
    offsets = torch.tensor(values, dtype=torch.int32, device="cuda")
    o, top = [], 0
    for v in values:
        top = max(top, min(max(v, 0), tokens))
        o.append(top)
    w, x = ints(g, m, k, 4), ints(g, k, tokens)
    d = cm(torch.full((m, tokens), -9.0, device="cuda"))
    GK.matmul_grouped(conf(m, tokens, k, torch.float16, torch.float32), w, x, None, d, offsets)
    dw = cm(torch.full((m, k, 4), -9.0, device="cuda"))
    dy = ints(g, m, tokens)
    GK.matmul_grouped_outer(conf(m, k, tokens, torch.float16, torch.float32, tb=True), dy, x, None, dw, offsets)
    dz, db = torch.full_like(dy, -9.0), cm(torch.full((m, 4), -9.0, device="cuda"))
    GK.activation_gradient_(dz, dy, None, None, bias_gradient=db, offsets=offsets)
    done()
    want, wz = torch.full_like(d, -9.0).double(), torch.full_like(dz, -9.0)
    for i in range(4):
        c = slice(o[i], o[i + 1])
        want[:, c] = w[:, :, i].double() @ x[:, c].double()
        wz[:, c] = dy[:, c]
        assert torch.equal(dw[:, :, i].double(), dy[:, c].double() @ x[:, c].double().T)
        assert torch.equal(db[:, i].double(), dy[:, c].double().sum(1))
    assert torch.equal(d.double(), want) and torch.equal(dz, wz)


@pytest.mark.parametrize("tb", [False, True])
def test_poison_outside_the_groups_is_not_seen(tb):
    g = gen(14)
    m, k, counts = 264, 136, [70, 0, 5, 200]
    offsets, o = offsets_of(counts, first=4)
    total = o[-1] + 40
    w, x = ints(g, m, k, 4), ints(g, k, total)
    dy = ints(g, m, total)
    clean = x.clone()
    for t, bad in ((x, float("nan")), (dy, float("inf"))):
        t[:, : o[0]] = bad
        t[:, o[-1]:] = bad
    # and a NaN token of group 0 stays in its column / its group
    x[5, o[1] - 1] = float("nan")
    d = cm(torch.zeros(m, total, device="cuda"))
    GK.matmul_grouped(conf(m, total, k, torch.float16, torch.float32, tb=tb), w, cm(x.T) if tb else x, None, d, offsets)
    dw = cm(torch.zeros(m, k, 4, device="cuda"))
    GK.matmul_grouped_outer(conf(m, k, total, torch.float16, torch.float32, tb=True), dy, x, None, dw, offsets)
    done()
    assert d[:, o[1] - 1].isnan().all()
    for i in range(4):
        hi = o[i + 1] - (1 if i == 0 else 0)
        assert torch.equal(d[:, o[i]:hi].double(), w[:, :, i].double() @ clean[:, o[i]:hi].double())
        want = dy[:, o[i]:o[i + 1]].double() @ clean[:, o[i]:o[i + 1]].double().T
        if i:
            assert torch.equal(dw[:, :, i].double(), want)
        else:
            rows = [j for j in range(k) if j != 5]
            assert torch.equal(dw[:, rows, 0].double(), want[:, rows])
    assert not d[:, : o[0]].any() and not d[:, o[-1]:].any()


@pytest.mark.parametrize("counts", COUNTS + [[64, 128, 65, 63, 1, 0, 200]])
@pytest.mark.parametrize("ta,tb", [(False, True), (False, False), (True, True), (True, False)])
@pytest.mark.parametrize("m,n", [(128, 256), (264, 136), (77, 45)])
def test_grouped_outer_of_integers_is_exact(counts, m, n, ta, tb):
    g = gen(len(counts))
    offsets, o = offsets_of(counts, first=2)
    G, total = len(counts), o[-1] + 5
    dy, x = ints(g, m, total), ints(g, n, total)
    prod = torch.stack([dy[:, o[i]:o[i + 1]].double() @ x[:, o[i]:o[i + 1]].double().T for i in range(G)], dim=2)
    a, b = cm(dy.T) if ta else dy, x if tb else cm(x.T)
    d = cm(torch.full((m, n, G), -9.0, device="cuda"))
    GK.matmul_grouped_outer(conf(m, n, total, torch.float16, torch.float32, ta, tb), a, b, None, d, offsets)
    done()
    assert torch.equal(d.double(), prod)
    c = ints(g, m, n, G, dtype=torch.float32)
    want = 2 * prod + 3 * c.double()
    GK.matmul_grouped_outer(conf(m, n, total, torch.float16, torch.float32, ta, tb, True), a, b, c, c, offsets,
                            transform_shared_to_regs_a=Transform.Elementwise(Transform.Scale(2.0)),
                            transform_shared_to_regs_c=Transform.Elementwise(Transform.Scale(3.0)))
    done()
    assert torch.equal(c.double(), want)


@pytest.mark.parametrize("tile_n,cg", [(64, 1), (128, 1), (256, 1), (128, 2), (256, 2)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_grouped_outer_tile_shapes(tile_n, cg, out):
    g = gen(tile_n)
    m, n, counts = 392, 584, [40, 0, 300, 1, 129, 64]
    offsets, o = offsets_of(counts)
    dy, x = ints(g, m, o[-1], dtype=torch.bfloat16, lo=-1, hi=1), ints(g, n, o[-1], dtype=torch.bfloat16, lo=0, hi=1)
    d = cm(torch.zeros(m, n, 6, dtype=out, device="cuda"))
    GK.bind_grouped_outer(conf(m, n, o[-1], torch.bfloat16, out, tb=True, tile_n=tile_n, cta_group=cg), dy, x, None, d, offsets)()
    done()
    for i in range(6):
        want = dy[:, o[i]:o[i + 1]].double() @ x[:, o[i]:o[i + 1]].double().T
        assert torch.equal(d[:, :, i], want.to(out))


def test_no_tokens_at_all():
    m, k, G = 136, 72, 3
    offsets = torch.zeros(G + 1, dtype=torch.int32, device="cuda")
    w, x = cm(torch.zeros(m, k, G, dtype=torch.float16, device="cuda")), torch.zeros(0, k, dtype=torch.float16, device="cuda").T
    dy = torch.zeros(0, m, dtype=torch.float16, device="cuda").T
    d = torch.zeros(0, m, device="cuda").T
    GK.matmul_grouped(conf(m, 0, k, torch.float16, torch.float32), w, x, None, d, offsets)
    dw = cm(torch.ones(m, k, G, device="cuda"))
    GK.matmul_grouped_outer(conf(m, k, 0, torch.float16, torch.float32, tb=True, residual=True), dy, x, dw, dw, offsets,
                            transform_shared_to_regs_c=Transform.Elementwise(Transform.Scale(5.0)))
    db = cm(torch.ones(m, G, device="cuda"))
    GK.activation_gradient_(None, dy, None, bias_gradient=db, offsets=offsets)
    done()
    assert torch.equal(dw, torch.full_like(dw, 5.0)) and not db.any()


def test_outputs_beyond_32_bit_offsets():
    """D and Z of more than 2^31 elements: the last columns are where they belong."""
    m, k, total = 8192, 64, 270000
    g = gen(15)
    w, x = ints(g, m, k, 2, dtype=torch.bfloat16, lo=-1, hi=1), ints(g, k, total, dtype=torch.bfloat16, lo=-1, hi=1)
    d = torch.zeros((total, m), dtype=torch.bfloat16, device="cuda").T
    offsets = torch.tensor([0, total - 5000, total - 3], dtype=torch.int32, device="cuda")
    GK.matmul_grouped(conf(m, total, k, torch.bfloat16, torch.bfloat16), w, x, None, d, offsets)
    done()
    for i, c in ((0, slice(total - 5100, total - 5000)), (1, slice(total - 5000, total - 4900)), (1, slice(total - 100, total - 3))):
        assert torch.equal(d[:, c].double(), w[:, :, i].double() @ x[:, c].double())
    assert not d[:, total - 3:].any()
    db = torch.zeros(m, device="cuda")
    GK.activation_gradient_(d, d, None, bias_gradient=db)
    done()
    want = w[:, :, 0].double() @ x[:, : total - 5000].double().sum(1) + w[:, :, 1].double() @ x[:, total - 5000: total - 3].double().sum(1)
    assert torch.equal(db.double(), want)


# ------------------------------------------------------------------------------------------------
# activation gradient
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("m,counts", [(64, [1]), (72, [5, 0, 200, 31]), (333, [40, 3]), (520, [700, 0, 1300]), (136, [0, 0])])
def test_activation_gradient(m, counts, act, dt):
    g = gen(m)
    offsets, o = offsets_of(counts, first=1)
    total = o[-1] + 6
    dd, z = normal(g, m, total, dtype=dt), normal(g, m, total, dtype=dt, scale=2.0)
    if m == 520:
        dd, z = padded(dd, 8), padded(z, 16)
    dz, db = cm(torch.full((m, total), -9.0, dtype=dt, device="cuda")), cm(torch.full((m, len(counts)), -9.0, device="cuda"))
    GK.activation_gradient_(dz, dd, None if act is None else z, ACT[act], bias_gradient=db, offsets=offsets)
    done()
    want = dd.double() * grad64(z.double(), act)
    slop = 16 * 2.0 ** -23 * dd.double().abs()            # act' in FP32: a few ulp of 1
    assert (dz[:, : o[0]] == -9).all() and (dz[:, o[-1]:] == -9).all()
    close(dz[:, o[0]:o[-1]], want[:, o[0]:o[-1]], slop[:, o[0]:o[-1]], "dZ")
    for i, n in enumerate(counts):
        c = slice(o[i], o[i + 1])
        tol = (n + 4) * 2.0 ** -23 * want[:, c].abs().sum(1) + slop[:, c].sum(1) + 1e-37
        assert ((db[:, i].double() - want[:, c].sum(1)).abs() <= tol).all(), i
    only = torch.full_like(db, 3.0)
    GK.activation_gradient_(None, dd, None if act is None else z, ACT[act], bias_gradient=only, offsets=offsets)
    again = dd.clone(memory_format=torch.preserve_format)
    GK.activation_gradient_(again, again, None if act is None else z, ACT[act], offsets=offsets)      # in place, no sums
    done()
    assert torch.equal(only, db)                           # a fixed order: the same bits
    assert torch.equal(again[:, o[0]:o[-1]], dz[:, o[0]:o[-1]])


def test_activation_gradient_without_groups():
    g = gen(21)
    dd = ints(g, 256, 3000, dtype=torch.bfloat16)
    db, dz = torch.zeros(256, device="cuda"), torch.zeros_like(dd)
    GK.activation_gradient_(dz, dd, None, bias_gradient=db)
    done()
    assert torch.equal(dz, dd) and torch.equal(db.double(), dd.double().sum(1))


# ------------------------------------------------------------------------------------------------
# together, and around them: an expert layer, streams, graphs
# ------------------------------------------------------------------------------------------------
def expert_layer(w1, b1, w2, b2, x, r, offsets, act, dt):
    """y[:, J_g] = W2_g act(W1_g x + b1_g) + b2_g + r, and a function that takes dy to all gradients."""
    f, h, G = w1.shape
    h, f = w1.shape[0], w1.shape[1]
    total = x.shape[1]

    def new(rows, cols, *more, dtype=dt):
        return torch.zeros(tuple(reversed((rows, cols, *more))), dtype=dtype, device="cuda").permute(*reversed(range(2 + len(more))))

    z, hid, y = new(h, total), new(h, total), new(f, total)
    GK.matmul_grouped(conf(h, total, f, dt, dt), w1, x, None, hid, offsets,
                      epilogue=Epilogue.BiasActivationResidual(b1, activation=ACT[act], preactivation=z))
    GK.matmul_grouped(conf(f, total, h, dt, dt, residual=True), w2, hid, r, y, offsets, epilogue=Epilogue.BiasActivationResidual(b2))

    def backward(dy):
        dz, dx = new(h, total), new(f, total)
        dw1, dw2 = new(h, f, G, dtype=torch.float32), new(f, h, G, dtype=torch.float32)
        db1, db2 = new(h, G, dtype=torch.float32), new(f, G, dtype=torch.float32)
        GK.activation_gradient_(None, dy, None, bias_gradient=db2, offsets=offsets)
        GK.matmul_grouped_outer(conf(f, h, total, dt, torch.float32, tb=True), dy, hid, None, dw2, offsets)
        GK.matmul_grouped(conf(h, total, f, dt, dt, ta=True), w2, dy, None, dz, offsets, epilogue=Epilogue.ActivationGradient(z, ACT[act]))
        GK.activation_gradient_(None, dz, None, bias_gradient=db1, offsets=offsets)
        GK.matmul_grouped_outer(conf(h, f, total, dt, torch.float32, tb=True), dz, x, None, dw1, offsets)
        GK.matmul_grouped(conf(f, total, h, dt, dt, ta=True), w1, dz, None, dx, offsets)
        return dx, dw1, db1, dw2, db2
    return y, backward


@pytest.mark.parametrize("counts", [[3, 0, 1, 2], [150, 0, 40, 301]])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_expert_layer_forward_and_backward(counts, act):
    """Against the same layer in 64 bits and its derivatives, by autograd and by differences.

    Each stored BF16 array (hidden, dz) carries a relative rounding of 2^-8 at most, so a sum over them is off by at most
    2^-8 of the sum of magnitudes for each array on the way (three: z, hidden or dz, and the result), plus FP32 terms that
    are smaller by orders; z's rounding moves act' by at most 2^-8 |z| max|act''|, max|act''| < 0.8."""
    g = gen(31)
    dt, f, h, G = torch.bfloat16, 136, 264, 4
    offsets, o = offsets_of(counts)
    T = o[-1]
    w1, w2 = normal(g, h, f, G, dtype=dt, scale=f ** -0.5), normal(g, f, h, G, dtype=dt, scale=h ** -0.5)
    b1, b2 = normal(g, h, G, dtype=torch.float32, scale=0.1), normal(g, f, G, dtype=torch.float32, scale=0.1)
    x, r, dy = normal(g, f, T, dtype=dt), normal(g, f, T, dtype=dt), normal(g, f, T, dtype=dt)
    y, backward = expert_layer(w1, b1, w2, b2, x, r, offsets, act, dt)
    grads = backward(dy)
    done()
    leaves = [t.double().requires_grad_() for t in (x, w1, b1, w2, b2)]

    def layer64(x, w1, b1, w2, b2):
        parts = []
        for i in range(G):
            c = slice(o[i], o[i + 1])
            hid = act64(w1[:, :, i] @ x[:, c] + b1[:, i:i + 1], act)
            parts.append(w2[:, :, i] @ hid + b2[:, i:i + 1])
        return torch.cat(parts, dim=1) + r.double()

    want = layer64(*leaves)
    exact = torch.autograd.grad(want, leaves, dy.double())
    # magnitudes: the same sums of absolute values
    u = 2.0 ** -8
    A = [t.double().abs() for t in (x, w1, w2, dy)]
    owner = torch.repeat_interleave(torch.arange(G, device="cuda"), torch.tensor(counts, device="cuda"))
    hid_mag, dz_mag, z_mag = torch.zeros(h, T, device="cuda").double(), torch.zeros(h, T, device="cuda").double(), torch.zeros(h, T, device="cuda").double()
    y_tol, dx_tol = torch.zeros(f, T, device="cuda").double(), torch.zeros(f, T, device="cuda").double()
    for i in range(G):
        c = slice(o[i], o[i + 1])
        z_mag[:, c] = A[1][:, :, i] @ A[0][:, c] + b1[:, i:i + 1].double().abs()
        zz = w1[:, :, i].double() @ x[:, c].double() + b1[:, i:i + 1].double()
        hid_mag[:, c] = act64(zz, act).abs()
        down = A[2][:, :, i].T @ A[3][:, c]
        dz_mag[:, c] = down * (1.13 + 0.8 * zz.abs())
        y_tol[:, c] = A[2][:, :, i] @ hid_mag[:, c]
        dx_tol[:, c] = A[1][:, :, i].T @ dz_mag[:, c]
    slack = 1e-4
    close(y, want.detach(), u * y_tol + slack, "y")
    close(grads[0], exact[0], 2 * u * dx_tol + slack, "dx")
    for i in range(G):
        c = slice(o[i], o[i + 1])
        close(grads[1][:, :, i], exact[1][:, :, i], 2 * u * dz_mag[:, c] @ A[0][:, c].T + slack, f"dW1 {i}")
        close(grads[2][:, i], exact[2][:, i], 2 * u * dz_mag[:, c].sum(1) + slack, f"db1 {i}")
        close(grads[3][:, :, i], exact[3][:, :, i], u * A[3][:, c] @ hid_mag[:, c].T + slack, f"dW2 {i}")
        close(grads[4][:, i], exact[4][:, i], u * A[3][:, c].sum(1) * 0 + slack, f"db2 {i}")
    # differences: the derivative of <y, dy> along a direction of every leaf, in 64 bits, against the kernels' gradients
    for leaf, (name, got) in enumerate(zip(("x", "w1", "b1", "w2", "b2"), grads)):
        base = [t.detach() for t in leaves]
        direction = torch.randn(base[leaf].shape, generator=g, device="cuda").double()
        step = 1e-5
        up, down = list(base), list(base)
        up[leaf], down[leaf] = base[leaf] + step * direction, base[leaf] - step * direction
        slope = ((layer64(*up) - layer64(*down)) * dy.double()).sum() / (2 * step)
        bound = (exact[leaf].abs() * direction.abs()).sum()
        mine = (got.double() * direction).sum()
        # independent roundings: far inside the sum of the elementwise tolerances; 4 u of the magnitudes covers them
        assert abs(float(mine - slope)) <= float(4 * u * bound) + 1e-2, name


def test_grouped_products_on_another_stream_and_back_to_back():
    """Dependent calls on one stream without synchronising: each kernel may start early, none may read early."""
    g = gen(41)
    m, counts = 256, [30, 0, 100, 126]
    offsets, o = offsets_of(counts)
    w, x = ints(g, m, m, 4, lo=0, hi=0), ints(g, m, 256, hi=3)
    for i in range(4):
        w[:, :, i] = torch.eye(m, device="cuda").roll(i + 1, 0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    bufs = [x] + [torch.zeros_like(x) for _ in range(8)]
    dws = [cm(torch.zeros(m, m, 4, device="cuda")) for _ in range(8)]
    with torch.cuda.stream(s):
        for src, dst, dw in zip(bufs, bufs[1:], dws):
            GK.matmul_grouped(conf(m, 256, m, torch.float16, torch.float16), w, src, None, dst, offsets)
            GK.matmul_grouped_outer(conf(m, m, 256, torch.float16, torch.float32, tb=True), dst, src, None, dw, offsets)
    s.synchronize()
    GK.poll_status()
    cur = x.double()
    for dst, dw in zip(bufs[1:], dws):
        nxt = torch.cat([cur[:, o[i]:o[i + 1]].roll(i + 1, 0) for i in range(4)], dim=1)
        assert torch.equal(dst.double(), nxt)
        for i in range(4):
            assert torch.equal(dw[:, :, i].double(), nxt[:, o[i]:o[i + 1]] @ cur[:, o[i]:o[i + 1]].T)
        cur = nxt


def test_captured_graphs_follow_the_offsets():
    """Two graphs captured on one stream (their workspaces are their own), replayed with other tokens and offsets."""
    g = gen(42)
    m, k, G, T = 136, 264, 4, 300
    w = ints(g, m, k, G)
    state, graphs = [], []
    side = torch.cuda.Stream()
    for _ in range(2):
        x, dy = ints(g, k, T), ints(g, m, T)
        offsets = torch.tensor([0, 50, 50, 170, T], dtype=torch.int32, device="cuda")
        d, dw = cm(torch.zeros(m, T, device="cuda")), cm(torch.zeros(m, k, G, device="cuda"))
        db, dz = cm(torch.zeros(m, G, device="cuda")), torch.zeros_like(dy)

        def step():
            GK.matmul_grouped(conf(m, T, k, torch.float16, torch.float32), w, x, None, d, offsets)
            GK.matmul_grouped_outer(conf(m, k, T, torch.float16, torch.float32, tb=True), dy, x, None, dw, offsets)
            GK.activation_gradient_(dz, dy, None, bias_gradient=db, offsets=offsets)

        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        state.append((x, dy, offsets, d, dw, db))
        graphs.append(graph)
    # a larger product in between makes the package replace its lent workspace
    big = torch.zeros(1025, dtype=torch.int64, device="cuda")
    with torch.cuda.stream(side):
        GK.matmul_grouped_outer(conf(8, 8, 16, torch.float16, torch.float32, tb=True), ints(g, 8, 16), ints(g, 8, 16), None,
                                cm(torch.zeros(8, 8, 1024, device="cuda")), big)
    side.synchronize()
    for values in ([0, 1, 2, 3, 4], [10, 10, 200, 290, 299], [0, 300, 300, 300, 300]):
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (x, dy, offsets, *_), graph, s in zip(state, graphs, streams):
            x.copy_(ints(g, k, T))
            offsets.copy_(torch.tensor(values, dtype=torch.int32))
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    graph.replay()
        done()
        for x, dy, offsets, d, dw, db in state:
            for i in range(G):
                c = slice(values[i], values[i + 1])
                assert torch.equal(d[:, c].double(), w[:, :, i].double() @ x[:, c].double())
                assert torch.equal(dw[:, :, i].double(), dy[:, c].double() @ x[:, c].double().T)
                assert torch.equal(db[:, i].double(), dy[:, c].double().sum(1))


def test_bound_operators_replay_on_new_values():
    g = gen(43)
    m, n, k = 520, 3, 1032
    a, b, d = ints(g, m, k), ints(g, k, n), cm(torch.zeros(m, n, device="cuda"))
    call = GK.bind(conf(m, n, k, torch.float16, torch.float32), a, b, None, d, epilogue=Epilogue.BiasActivationResidual())
    for _ in range(3):
        b.copy_(ints(g, k, n))
        call()
        done()
        assert torch.equal(d.double(), a.double() @ b.double())


def test_ragged_depth_refuses_a_missing_workspace():
    g = gen(44)
    offsets, o = offsets_of([64, 64])
    dy, x = ints(g, 128, 128), ints(g, 128, 128)
    d = cm(torch.zeros(128, 128, 2, device="cuda"))
    cf = conf(128, 128, 128, torch.float16, torch.float32, tb=True)
    plan = GK.grouped_query(cf, dy, x, None, d, offsets)
    assert plan.kernel == 1 and plan.workspace_bytes == 2 * 2 * 128
    with pytest.raises(GK.GemmKernelsError, match="workspace"):
        GK.matmul_grouped_outer(cf, dy, x, None, d, offsets, workspace=torch.zeros(256, dtype=torch.uint8, device="cuda"))
    guard = torch.full((1024,), 7, dtype=torch.uint8, device="cuda")
    GK.matmul_grouped_outer(cf, dy, x, None, d, offsets, workspace=guard)
    done()
    assert (guard[512:] == 7).all()
    for i in range(2):
        c = slice(o[i], o[i + 1])
        assert torch.equal(d[:, :, i].double(), dy[:, c].double() @ x[:, c].double().T)


# ------------------------------------------------------------------------------------------------
# combinations: types, leading dimensions, group strides, in-place C, epilogues - small integers, exact
# ------------------------------------------------------------------------------------------------
def roomy(t, pad, gap=0):
    """The same (rows, cols[, groups]) array with `pad` elements between columns and `gap` more between groups, NaN there."""
    rows, cols, groups = (*t.shape, 1)[:3]
    ld = rows + pad
    size = groups * (ld * cols + gap) + 8
    buf = torch.full((size,), float("nan"), dtype=t.dtype, device=t.device)
    view = buf.as_strided((rows, cols, groups), (1, ld, ld * cols + gap))
    view.copy_(t if t.dim() == 3 else t[:, :, None])
    return view if t.dim() == 3 else view[:, :, 0]


@pytest.mark.parametrize("seed", range(60))
def test_randomised_fused_and_grouped_combinations(seed):
    import random
    r = random.Random(seed)
    g = gen(1000 + seed)
    dt = r.choice([torch.float16, torch.bfloat16])
    out = r.choice([torch.float32, dt])
    step = r.choice([1, 8, 8, 16])
    size = lambda lo, hi: max(step, r.randint(lo, hi) // step * step)
    m, k, G = size(1, 600), size(1, 400), r.choice([1, 2, 5, 33])
    counts = [r.choice([0, 0, 1, 3, 20, 70, 150]) for _ in range(G)]
    grouped = r.random() < 0.6
    n = sum(counts) + r.choice([0, 7]) if grouped else r.choice([1, 3, 9, 64, 130, 333])
    ta, tb = r.random() < 0.5, r.random() < 0.3
    pad, gap = r.choice([0, 8, 3]), r.choice([0, 16, 5])
    form = r.choice(["standard", "residual", "gradient"])
    act = r.choice([None, "relu"])
    bits16 = out != torch.float32
    lim = 1 if bits16 else 2
    w = ints(g, m, k, G, dtype=dt, lo=-lim, hi=lim)
    x = ints(g, k, n, dtype=dt, lo=0, hi=1)
    if bits16:                       # at most 60 products of -1 .. 1 and small addends: every value is exact in 8 bits
        x[:, :] = 0
        x[: min(k, 60)] = ints(g, min(k, 60), n, dtype=dt, lo=0, hi=1)
    has_c, keep = r.random() < 0.6, r.random() < 0.5
    beta = r.choice([1.0, -2.0]) if has_c else 0.0
    c, z0 = ints(g, m, n, dtype=out, lo=-9, hi=9), ints(g, m, n, dtype=out, lo=-2, hi=2)
    bias = ints(g, m, G, dtype=torch.float32, lo=-5, hi=5)
    owner = torch.full((n,), -1, device="cuda")
    offsets, o = offsets_of(counts, dtype=r.choice([torch.int32, torch.int64]))
    prod = torch.zeros(m, n, device="cuda", dtype=torch.float64)
    if grouped:
        for i in range(G):
            prod[:, o[i]:o[i + 1]] = w[:, :, i].double() @ x[:, o[i]:o[i + 1]].double()
            owner[o[i]:o[i + 1]] = i
    else:
        prod, owner[:] = w[:, :, 0].double() @ x.double(), 0
    live = owner >= 0
    add = bias.double()[:, owner.clamp(min=0)] if form != "gradient" else 0.0
    pre = prod + add + (beta * c.double() if form != "residual" else 0.0)
    f = (lambda t: t.clamp(min=0)) if act else (lambda t: t)
    want = pre * (grad64(z0.double(), act)) if form == "gradient" else f(pre) + (beta * c.double() if form == "residual" else 0.0)
    wd = roomy(torch.full((m, n), -77.0, dtype=out, device="cuda"), pad)
    wz = roomy(z0, pad)
    aw = roomy(w.permute(1, 0, 2) if ta else w, pad, gap)
    xw = roomy(x.T if tb else x, pad)
    cw = roomy(c, pad) if has_c else None
    inplace = has_c and r.random() < 0.4 and not grouped
    d = cw if inplace else wd
    if form == "standard":
        epi, keep = Epilogue.Bias(bias if grouped else bias[:, 0].contiguous(), axis="row"), False
    elif form == "residual":
        epi = Epilogue.BiasActivationResidual(bias if grouped else bias[:, 0].contiguous(), activation=ACT[act], preactivation=wz if keep else None)
    else:
        epi = Epilogue.ActivationGradient(wz, ACT[act])
    kw = {}
    if beta != 1.0 and has_c:
        kw["transform_shared_to_regs_c"] = Transform.Elementwise(Transform.Scale(beta))
    if form == "standard" and act:
        kw["transform_shared_to_global_d"] = Transform.Elementwise(ACT[act])
    cf = conf(m, n, k, dt, out, ta, tb, has_c)
    if grouped:
        GK.matmul_grouped(cf, aw, xw, cw, d, offsets, epilogue=epi, **kw)
    else:
        GK.matmul(cf, aw[:, :, 0], xw, cw, d, epilogue=epi, **kw)
    done()
    assert torch.equal(d[:, live].double(), want[:, live])
    assert (d[:, ~live] == -77).all()
    if form == "residual" and keep:
        assert torch.equal(wz[:, live].double(), pre[:, live]) and torch.equal(wz[:, ~live], z0[:, ~live])


@pytest.mark.parametrize("seed", range(24))
def test_randomised_outer_combinations(seed):
    import random
    r = random.Random(seed)
    g = gen(2000 + seed)
    dt = r.choice([torch.float16, torch.bfloat16])
    out = r.choice([torch.float32, dt])
    step = r.choice([1, 8, 8])
    m, n, G = max(step, r.randint(1, 500) // step * step), max(step, r.randint(1, 500) // step * step), r.choice([1, 3, 20])
    counts = [r.choice([0, 1, 5, 63, 64, 65, 130]) for _ in range(G)]
    offsets, o = offsets_of(counts, first=r.choice([0, 5]))
    total = o[-1] + r.choice([0, 9])
    dy, x = ints(g, m, total, dtype=dt, lo=-1, hi=1), ints(g, n, total, dtype=dt, lo=0, hi=1)
    dy[:, r.randrange(0, 2)::3] = 0                                   # |sums| stay below 256: exact in BF16
    c = ints(g, m, n, G, dtype=out, lo=-20, hi=20)
    pad, gap = r.choice([0, 8, 3]), r.choice([0, 16, 5])
    has_c, inplace = r.random() < 0.6, r.random() < 0.5
    alpha = r.choice([1.0, 0.0, -1.0])
    cw = roomy(c, pad, gap) if has_c else None
    d = cw if has_c and inplace else roomy(torch.full((m, n, G), -77.0, dtype=out, device="cuda"), pad, gap)
    ta, tb = r.random() < 0.2, r.random() < 0.8
    GK.matmul_grouped_outer(conf(m, n, total, dt, out, ta, tb, has_c), roomy(dy.T if ta else dy, pad), roomy(x if tb else x.T, pad), cw, d, offsets,
                            transform_shared_to_regs_a=Transform.Elementwise(Transform.Scale(alpha)))
    done()
    for i in range(G):
        want = alpha * (dy[:, o[i]:o[i + 1]].double() @ x[:, o[i]:o[i + 1]].double().T) + (c[:, :, i].double() if has_c else 0.0)
        assert torch.equal(d[:, :, i].double(), want), i


def test_grouped_with_nothing_to_multiply():
    g = gen(61)
    m, counts = 136, [30, 0, 5]
    offsets, o = offsets_of(counts, first=2)
    total = o[-1] + 3
    bias, c = ints(g, m, 3, dtype=torch.float32), ints(g, m, total, dtype=torch.float32)
    nan = lambda *s: cm(torch.full(s, float("nan"), dtype=torch.float16, device="cuda"))
    for k, alpha in ((64, 0.0), (0, 1.0)):
        d = cm(torch.full((m, total), -9.0, device="cuda"))
        w = nan(m, max(k, 1), 3)[:, :k]
        GK.matmul_grouped(conf(m, total, k, torch.float16, torch.float32, residual=True), w, nan(max(k, 1), total)[:k], c, d, offsets,
                          epilogue=Epilogue.BiasActivationResidual(bias), transform_shared_to_regs_a=Transform.Elementwise(Transform.Scale(alpha)))
        done()
        for i in range(3):
            assert torch.equal(d[:, o[i]:o[i + 1]], bias[:, i:i + 1] + c[:, o[i]:o[i + 1]])
        assert (d[:, : o[0]] == -9).all() and (d[:, o[-1]:] == -9).all()
    with pytest.raises(GK.ConfigError, match="per row"):
        GK.matmul_grouped(conf(m, total, 64, torch.float16, torch.float32), nan(m, 64, 3), nan(64, total), None, d, offsets,
                          epilogue=Epilogue.Bias(torch.zeros(total, device="cuda"), axis="col"))


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("counts", [[5000, 2048, 0, 2049], [4096, 100], [2047, 6145]])
@pytest.mark.parametrize("m", [264, 131])
def test_long_runs_are_added_up_in_parts(counts, accumulate, m):
    """FP32 sums over more than 2048 columns: exact on integers, and the error does not grow with the length any more."""
    g = gen(71)
    offsets, o = offsets_of(counts, first=1)
    n, G, total = 520, len(counts), o[-1] + 5
    dy, x, c = ints(g, m, total), ints(g, n, total), ints(g, m, n, G, dtype=torch.float32, lo=-50, hi=50)
    d = c.clone(memory_format=torch.preserve_format) if accumulate else cm(torch.full((m, n, G), float("nan"), device="cuda"))
    call = GK.bind_grouped_outer(conf(m, n, total, torch.float16, torch.float32, tb=True, residual=accumulate), dy, x, d if accumulate else None, d,
                                 offsets, transform_shared_to_regs_a=Transform.Elementwise(Transform.Scale(2.0)))
    call()
    done()
    for i in range(G):
        want = 2 * (dy[:, o[i]:o[i + 1]].double() @ x[:, o[i]:o[i + 1]].double().T) + (c[:, :, i].double() if accumulate else 0.0)
        assert torch.equal(d[:, :, i].double(), want), i
    dy, x = normal(g, m, total, dtype=torch.bfloat16), normal(g, n, total, dtype=torch.bfloat16)
    d = cm(torch.zeros(m, n, G, device="cuda"))
    GK.matmul_grouped_outer(conf(m, n, total, torch.bfloat16, torch.float32, tb=True), dy, x, None, d, offsets)
    done()
    for i, count in enumerate(counts):
        want = dy[:, o[i]:o[i + 1]].double() @ x[:, o[i]:o[i + 1]].double().T
        mag = dy[:, o[i]:o[i + 1]].double().abs() @ x[:, o[i]:o[i + 1]].double().abs().T
        # within a part at most one ulp of the running sum per 16 products (128 additions of 2^-23), then one rounding a part
        assert ((d[:, :, i].double() - want).abs() <= (128 + 4) * 2.0 ** -23 * mag + 1e-30).all(), i


@pytest.mark.parametrize("n", [2, 5, 8, 9, 15, 16])
@pytest.mark.parametrize("ta", [False, True])
@pytest.mark.parametrize("m,k", [(8, 8), (64, 64), (72, 136), (200, 2048), (1000, 520), (4096, 264)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_several_columns_stream(m, k, n, ta, dt):
    g = gen(m + n)
    a, b, r = ints(g, m, k, dtype=dt), ints(g, k, n, dtype=dt), ints(g, m, n, dtype=torch.float32)
    bias = ints(g, m, dtype=torch.float32)
    aw, bw = roomy(cm(a.T) if ta else a, 8), roomy(b, 16)
    d, z = torch.full_like(r, -9.0), torch.full_like(r, -9.0)
    cf, epi = conf(m, n, k, dt, torch.float32, ta, residual=True), Epilogue.BiasActivationResidual(bias, activation=ACT["relu"], preactivation=z)
    assert GK.query(cf, aw, bw, r, d, epilogue=epi).kernel == (6 if ta or n <= 8 else 1)
    GK.matmul(cf, aw, bw, r, d, epilogue=epi)
    done()
    x = a.double() @ b.double() + bias.double()[:, None]
    assert torch.equal(z.double(), x) and torch.equal(d.double(), x.clamp(min=0) + r.double())


@pytest.mark.parametrize("counts", [[3, 0, 2, 7], [16, 1, 0, 15], [17, 0, 0, 0], [1, 33, 2, 0], [4] * 9])
@pytest.mark.parametrize("ta", [False, True])
def test_several_columns_per_group_stream(counts, ta):
    run_grouped(counts, 136, 264, torch.bfloat16, ta, False, tail=1)
    run_grouped(counts, 520, 1032, torch.float16, ta, False, first=2, tail=1)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("n", [3, 200])
def test_gradient_epilogue_in_32_bits(n, act):
    g = gen(81)
    m, k = 200, 96
    a, b, z = normal(g, m, k, scale=k ** -0.5), normal(g, k, n), normal(g, m, n, dtype=torch.float32, scale=2.0)
    d = torch.zeros_like(z)
    GK.matmul(conf(m, n, k, torch.float16, torch.float32), a, b, None, d, epilogue=Epilogue.ActivationGradient(z, ACT[act]))
    done()
    want = (a.double() @ b.double()) * grad64(z.double(), act)
    mag = a.double().abs() @ b.double().abs()
    close(d, want, err(k, mag, want) + 16 * 2.0 ** -23 * mag)


def test_offsets_of_64_bits_far_outside():
    g = gen(82)
    w, x = ints(g, 136, 72, 3), ints(g, 72, 100)
    offsets = torch.tensor([-2 ** 60, 40, 2 ** 33 + 50, 2 ** 62], device="cuda")      # 2^33 + 50 is 50 in its low 32 bits
    d = cm(torch.full((136, 100), -9.0, device="cuda"))
    GK.matmul_grouped(conf(136, 100, 72, torch.float16, torch.float32), w, x, None, d, offsets)
    done()
    assert torch.equal(d[:, :40].double(), w[:, :, 0].double() @ x[:, :40].double())
    assert torch.equal(d[:, 40:].double(), w[:, :, 1].double() @ x[:, 40:].double())


@pytest.mark.parametrize("m,n,k,ta", [(300, 257, 1111, False), (520, 1, 1032, True), (520, 7, 1032, True), (77, 2, 45, False), (256, 96, 8192, False)])
def test_captured_single_products(m, n, k, ta):
    """Every route of a single product - copies, both streaming kernels, split K - in a graph of its own workspace."""
    g = gen(83)
    side = torch.cuda.Stream()
    made = []
    for _ in range(2):
        a, b, r = ints(g, m, k, lo=-1, hi=1), ints(g, k, n, lo=-1, hi=1), ints(g, m, n, dtype=torch.float32)
        aw = cm(a.T) if ta else a
        d = torch.zeros_like(r)
        cf = conf(m, n, k, torch.float16, torch.float32, ta, residual=True)
        epi = Epilogue.BiasActivationResidual(activation=ACT["relu"])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            GK.matmul(cf, aw, b, r, d, epilogue=epi)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            GK.matmul(cf, aw, b, r, d, epilogue=epi)
        made.append((graph, aw, b, r, d))
    for _ in range(3):
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for graph, aw, b, r, d in made:
            aw.copy_(ints(g, *aw.shape, lo=-1, hi=1))
            b.copy_(ints(g, k, n, lo=-1, hi=1))
            d.zero_()
        torch.cuda.synchronize()
        for s, (graph, *_) in zip(streams, made):
            with torch.cuda.stream(s):
                graph.replay()
                graph.replay()
        done()
        for graph, aw, b, r, d in made:
            a = aw.T if ta else aw
            assert torch.equal(d.double(), (a.double() @ b.double()).clamp(min=0) + r.double())


@pytest.mark.parametrize("which", ["a", "b", "both"])
@pytest.mark.parametrize("ta", [False, True])
@pytest.mark.parametrize("n", [2, 6, 8, 16])
def test_few_columns_that_start_off_16_bytes(n, ta, which):
    """Aligned leading dimensions and a base one element off: the plan made without the pointers may not hold."""
    g = gen(84)
    m, k = 136, 264
    a, b = ints(g, m, k), ints(g, k, n)

    def off(t):
        big = torch.zeros(t.numel() + 8, dtype=t.dtype, device="cuda")
        view = big[1: 1 + t.numel()].view(t.shape[1], t.shape[0]).T
        view.copy_(t)
        return view

    aw = cm(a.T) if ta else a
    if which != "b":
        aw = off(aw)
    bw = off(b) if which != "a" else b
    d, z = cm(torch.full((m, n), -9.0, device="cuda")), cm(torch.full((m, n), -9.0, device="cuda"))
    GK.matmul(conf(m, n, k, torch.float16, torch.float32, ta), aw, bw, None, d,
              epilogue=Epilogue.BiasActivationResidual(activation=ACT["relu"], preactivation=z))
    done()
    x = a.double() @ b.double()
    assert torch.equal(z.double(), x) and torch.equal(d.double(), x.clamp(min=0))


@pytest.mark.parametrize("ta", [False, True])
@pytest.mark.parametrize("n", [5, 7, 8])
def test_streamed_columns_do_not_mix(n, ta):
    """A NaN in a column of B, an infinity in a row of A, NaN in the padding of both: each stays where it belongs."""
    g = gen(85)
    m, k = 200, 520
    a, b = ints(g, m, k, lo=1, hi=2), ints(g, k, n, lo=1, hi=2)
    a[77, 515] = math.inf
    b[333, 3] = math.nan
    want = a.double() @ b.double()
    d = cm(torch.full((m, n), -9.0, device="cuda"))
    GK.matmul(conf(m, n, k, torch.float16, torch.float32, ta), padded(cm(a.T) if ta else a, 8), padded(b, 16), None, d,
              epilogue=Epilogue.BiasActivationResidual())
    done()
    assert want[77, 0] == math.inf and want[:, 3].isnan().all() and want.isnan().sum() == m
    assert torch.equal(d.isnan(), want.isnan())
    assert torch.equal(d.double().nan_to_num(nan=-1.0, posinf=-2.0), want.nan_to_num(nan=-1.0, posinf=-2.0))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [5, 8])
@pytest.mark.parametrize("form", ["gradient", "residual"])
def test_streamed_columns_of_any_value(form, n, dt):
    g = gen(86)
    m, k = 264, 1032
    a, b, r = normal(g, m, k, dtype=dt, scale=k ** -0.5), normal(g, k, n, dtype=dt), normal(g, m, n, dtype=dt)
    d = torch.zeros_like(r)
    x = a.double() @ b.double()
    mag = a.double().abs() @ b.double().abs()
    if form == "gradient":
        GK.matmul(conf(m, n, k, dt, dt), a, b, None, d, epilogue=Epilogue.ActivationGradient(r, ACT["silu"]))
        want, more = x * grad64(r.double(), "silu"), 16 * 2.0 ** -23 * mag
    else:
        GK.matmul(conf(m, n, k, dt, dt, residual=True), a, b, r, d, epilogue=Epilogue.BiasActivationResidual(activation=ACT["gelu"]))
        want, more = act64(x, "gelu") + r.double(), 4 * 2.0 ** -23 * (x.abs() + r.double().abs())
    done()
    close(d, want, err(k, mag, x) + more)


def test_captured_product_of_seven_columns():
    g = gen(87)
    m, n, k = 520, 7, 1032
    a, b = ints(g, m, k), ints(g, k, n)
    d = cm(torch.zeros(m, n, device="cuda"))
    cf, epi = conf(m, n, k, torch.float16, torch.float32), Epilogue.BiasActivationResidual(activation=ACT["relu"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        GK.matmul(cf, a, b, None, d, epilogue=epi)
    for _ in range(2):
        a.copy_(ints(g, m, k))
        d.zero_()
        graph.replay()
        graph.replay()
        done()
        assert torch.equal(d.double(), (a.double() @ b.double()).clamp(min=0))
