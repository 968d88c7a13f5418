"""Layer-level operators on the GPU where they are used out of the ordinary: from two threads, on operands and results that
start anywhere, at the ends of the activations' range.  Integers are exact, other tolerances stand beside their tests."""
import math
import threading

import pytest
import torch

import gemmkernels_b200 as GK
from gemmkernels_b200 import Epilogue, Transform
from test_fused_gpu import ACT, cm, conf, done, gen, ints, normal, offsets_of

pytestmark = pytest.mark.gpu


def test_threads_that_share_a_stream():
    """Both enqueue products of a ragged depth (tensor maps, then the product) and split products (partial sums, then their
    addition) on the default stream, with scratch lent by the package."""
    g = gen(301)
    m, n, counts = 128, 256, [100, 0, 65, 3]
    offsets, o = offsets_of(counts)
    cf = conf(m, n, o[-1], torch.float16, torch.float32, False, True)
    cs = conf(256, 64, 8192, torch.float16, torch.float32)
    sets = []
    for _ in range(2):
        a, b = ints(g, m, o[-1]), ints(g, n, o[-1])
        x, y = ints(g, 256, 8192, lo=-1, hi=1), ints(g, 8192, 64, lo=-1, hi=1)
        sets.append((a, b, x, y, [(cm(torch.full((m, n, 4), -9.0, device="cuda")), cm(torch.full((256, 64), -9.0, device="cuda"))) for _ in range(40)]))
    torch.cuda.synchronize()
    errors = []

    def work(a, b, x, y, outs):
        try:
            for d, p in outs:
                GK.matmul_grouped_outer(cf, a, b, None, d, offsets)
                GK.matmul(cs, x, y, None, p, epilogue=Epilogue.BiasActivationResidual())
        except Exception as e:      # noqa: BLE001 - reported by the assertion below
            errors.append(e)

    threads = [threading.Thread(target=work, args=s) for s in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    done()
    assert not errors, errors
    for a, b, x, y, outs in sets:
        want = torch.stack([a[:, o[i]:o[i + 1]].double() @ b[:, o[i]:o[i + 1]].double().T for i in range(4)], 2)
        prod = x.double() @ y.double()
        for d, p in outs:
            assert torch.equal(d.double(), want) and torch.equal(p.double(), prod)


def test_two_graphs_of_split_products_replayed_at_once():
    """Plain products whose K is split, captured into two graphs on one stream and replayed on two."""
    g = gen(302)
    m, n, k = 256, 64, 16384
    cf = conf(m, n, k, torch.float16, torch.float32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    made = []
    for _ in range(2):
        a, b = ints(g, m, k, lo=-1, hi=1), ints(g, k, n, lo=-1, hi=1)
        d = cm(torch.full((m, n), -9.0, device="cuda"))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            for _ in range(20):
                GK.matmul(cf, a, b, None, d)
        made.append((graph, a, b, d))
    other = torch.cuda.Stream()
    for (graph, *_), s in zip(made, (side, other)):
        with torch.cuda.stream(s):
            graph.replay()
    done()
    for _, a, b, d in made:
        assert torch.equal(d.double(), a.double() @ b.double())


def shifted(t, by=1, extra=0):
    """The same matrix (rows, cols[, groups]) `by` elements behind a 16-byte boundary, `extra` elements between its columns."""
    rows, cols, groups = (*t.shape, 1)[:3]
    ld = rows + extra
    buf = torch.full((groups * ld * cols + by + 8,), float("nan"), dtype=t.dtype, device="cuda")
    view = buf[by:].as_strided((rows, cols, groups), (1, ld, ld * cols))
    view.copy_(t if t.dim() == 3 else t[:, :, None])
    return view if t.dim() == 3 else view[:, :, 0]


@pytest.mark.parametrize("by", [1, 2, 3])
@pytest.mark.parametrize("m,n", [(132, 40), (300, 129), (512, 257)])
@pytest.mark.parametrize("kind", ["residual", "standard", "grouped"])
def test_results_in_32_bits_that_start_off_16_bytes(kind, m, n, by):
    """C aligned, D not: C is copied 16 bytes at a time, D is stored element by element."""
    g = gen(303 + by)
    k = 72
    a, b, c = ints(g, m, k), ints(g, k, n), ints(g, m, n, dtype=torch.float32, hi=50)
    d = shifted(torch.full((m, n), -9.0, device="cuda"), by)
    cf = conf(m, n, k, torch.float16, torch.float32, residual=True)
    if kind == "grouped":
        offsets, _ = offsets_of([n])
        GK.matmul_grouped(cf, a[:, :, None], b, c, d, offsets)
    else:
        GK.matmul(cf, a, b, c, d, epilogue=Epilogue.BiasActivationResidual() if kind == "residual" else Epilogue.Default())
    done()
    assert torch.equal(d.double(), a.double() @ b.double() + c.double())


@pytest.mark.parametrize("m,n", [(264, 72), (100, 40), (1032, 200)])
def test_accumulation_in_tiles_that_end_early(m, n):
    """Many tiles per CTA whose last chunks of 32 columns, and whose last warps, have nothing to add: each buffer of C is
    filled again by the next tile."""
    g = gen(310)
    counts = [(7 * i) % 23 for i in range(300)]
    offsets, o = offsets_of(counts)
    a, b = ints(g, m, o[-1]), ints(g, n, o[-1])
    c = ints(g, m, n, 300, dtype=torch.float32, lo=-50, hi=50)
    want = c.double() + torch.stack([a[:, o[i]:o[i + 1]].double() @ b[:, o[i]:o[i + 1]].double().T for i in range(300)], 2)
    GK.matmul_grouped_outer(conf(m, n, o[-1], torch.float16, torch.float32, False, True, True), a, b, c, c, offsets)
    done()
    assert torch.equal(c.double(), want)


@pytest.mark.parametrize("room", ["query", "copies - 256", "copies", "copies + 256", "copies + maps - 256", "copies + maps", "lent"])
@pytest.mark.parametrize("which", ["a", "b", "both"])
def test_ragged_depth_of_operands_off_16_bytes(which, room):
    """Many groups of small matrices, whose tensor maps are larger than the padded copies: whatever room there is, the call
    computes the product (the bounds-checked loads need none)."""
    g = gen(311)
    groups, m, n = 64, 64, 64
    offsets, o = offsets_of([1] * groups)
    a, b = ints(g, m, o[-1]), ints(g, n, o[-1])
    want = torch.stack([torch.outer(a[:, i].double(), b[:, i].double()) for i in range(groups)], 2)
    aw, bw = shifted(a) if which != "b" else a, shifted(b) if which != "a" else b
    cf = conf(m, n, o[-1], torch.float16, torch.float32, False, True)
    maps, copies = groups * 256, 64 * 64 * 2 * (2 if which == "both" else 1)
    for out in (torch.float32, torch.float16):
        cf = conf(m, n, o[-1], torch.float16, out, False, True)
        d = cm(torch.full((m, n, groups), -9.0, device="cuda", dtype=out))
        size = GK.grouped_query(cf, aw, bw, None, d, offsets).workspace_bytes if room == "query" else \
            None if room == "lent" else eval(room, dict(copies=copies, maps=maps))
        ws = None if size is None else torch.empty(size, dtype=torch.uint8, device="cuda")
        GK.matmul_grouped_outer(cf, aw, bw, None, d, offsets, workspace=ws)
        done()
        assert torch.equal(d.double(), want)


@pytest.mark.parametrize("which", ["a", "b", "both"])
@pytest.mark.parametrize("kind", ["fused", "grouped", "outer"])
def test_operands_off_16_bytes_are_given_room_for_their_copies(kind, which):
    """Views such as x[1:] whose columns are a multiple of 16 bytes apart."""
    g = gen(312)
    m, k, n = 136, 264, 96
    a, b = ints(g, m, k), ints(g, k, n)
    if kind == "outer":
        b = ints(g, n, k)
    aw, bw = shifted(a) if which != "b" else a, shifted(b) if which != "a" else b
    room = (m * k * 2 + 255) // 256 * 256 * (which != "b") + (n * k * 2 + 255) // 256 * 256 * (which != "a")
    if kind == "fused":
        d = cm(torch.full((m, n), -9.0, device="cuda"))
        cf, epi = conf(m, n, k, torch.float16, torch.float32), Epilogue.BiasActivationResidual()
        assert GK.query(cf, aw, bw, None, d, epilogue=epi).workspace_bytes == room
        for run in (lambda: GK.matmul(cf, aw, bw, None, d, epilogue=epi), GK.bind(cf, aw, bw, None, d, epilogue=epi)):
            d.fill_(-9)
            run()
            done()
            assert torch.equal(d.double(), a.double() @ b.double())
    elif kind == "grouped":
        d = cm(torch.full((m, n), -9.0, device="cuda"))
        offsets, _ = offsets_of([n])
        cf = conf(m, n, k, torch.float16, torch.float32)
        assert GK.grouped_query(cf, aw[:, :, None], bw, None, d, offsets).workspace_bytes == room
        GK.matmul_grouped(cf, aw[:, :, None], bw, None, d, offsets)
        done()
        assert torch.equal(d.double(), a.double() @ b.double())
    else:
        d = cm(torch.full((m, n, 2), -9.0, device="cuda"))
        offsets, o = offsets_of([100, 164])
        cf = conf(m, n, k, torch.float16, torch.float32, False, True)
        assert GK.grouped_query(cf, aw, bw, None, d, offsets).workspace_bytes == room + 2 * 256
        GK.matmul_grouped_outer(cf, aw, bw, None, d, offsets)
        done()
        assert torch.equal(d.double(), torch.stack([a[:, i:j].double() @ b[:, i:j].double().T for i, j in ((0, 100), (100, 264))], 2))


def test_bound_operators_on_another_stream_than_they_were_made_on():
    """Called on a busy stream and dropped at once, while the stream they were made on allocates and writes memory."""
    g = gen(313)
    m, n, counts = 128, 256, [100, 0, 65, 3]
    offsets, o = offsets_of(counts)
    a, b = ints(g, m, o[-1]), ints(g, n, o[-1])
    x, y = ints(g, 256, 8192, lo=-1, hi=1), ints(g, 8192, 64, lo=-1, hi=1)
    want = torch.stack([a[:, o[i]:o[i + 1]].double() @ b[:, o[i]:o[i + 1]].double().T for i in range(4)], 2)
    prod = x.double() @ y.double()
    d, p, q = cm(torch.empty(m, n, 4, device="cuda")), cm(torch.empty(256, 64, device="cuda")), cm(torch.empty(256, 64, device="cuda"))
    cf, cs = conf(m, n, o[-1], torch.float16, torch.float32, False, True), conf(256, 64, 8192, torch.float16, torch.float32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        calls = [GK.bind_grouped_outer(cf, a, b, None, d, offsets), GK.bind(cs, x, y, None, p),
                 GK.bind(cs, x, y, None, q, epilogue=Epilogue.BiasActivationResidual())]
        with torch.cuda.stream(side):
            torch.cuda._sleep(200000)
            for call in calls:
                call()
        del calls, call
        for size in (1024, 1 << 16, 1 << 18, 1 << 20):
            torch.empty(size, dtype=torch.uint8, device="cuda").fill_(255)
    done()
    assert torch.equal(d.double(), want) and torch.equal(p.double(), prod) and torch.equal(q.double(), prod)


# ------------------------------------------------------------------------------------------------
# activations over their whole range
# ------------------------------------------------------------------------------------------------
ROUTES = {"words": (128, 96, 128), "elements": (130, 96, 128), "streamed": (128, 1, 128), "several": (128, 8, 128), "split": (128, 96, 16384)}


def through_a_product(x, route, dt, out, act, z=None):
    """act(x) - or with z x * act'(z) - as the fused epilogue computes it on one of its routes: x, exact in `dt`, behind a product
    with the identity.  x and z have n columns of m values."""
    m, n, k = ROUTES[route]
    a = cm(torch.zeros(m, k, device="cuda", dtype=dt))
    a[:, :min(m, k)] = torch.eye(m, min(m, k), device="cuda", dtype=dt)
    b = cm(torch.zeros(k, n, device="cuda", dtype=dt))
    b[: min(m, k)] = x[: min(m, k)].to(dt)
    d = cm(torch.full((m, n), -9.0, device="cuda", dtype=out))
    epi = Epilogue.ActivationGradient(z, ACT[act]) if z is not None else Epilogue.BiasActivationResidual(activation=ACT[act])
    cf = conf(m, n, k, dt, out)
    plan = GK.query(cf, a, b, None, d, epilogue=epi)
    assert (plan.kernel == 6) == (route in ("streamed", "several")) and (route != "split" or plan.workspace_bytes >= 2 * m * n * 4)
    GK.matmul(cf, a, b, None, d, epilogue=epi)
    done()
    return d


def span(route, dt, lo=-12.0, hi=12.0):
    m, n, k = ROUTES[route]
    x = torch.linspace(lo, hi, m * n, device="cuda", dtype=torch.float64).reshape(n, m).T.to(dt)
    x[min(m, k):] = 0                       # (rows that the identity does not reach)
    return x


def gelu64(x):
    return 0.5 * x * torch.special.erfc(-x / math.sqrt(2))


def within(got, want, rel, slack):
    """One rounding to the type of `got`, behind a relative error `rel` and an absolute error `slack` before it."""
    fi = torch.finfo(got.dtype)
    tol = want.abs() * (fi.eps / 2 + rel * (1 + fi.eps)) + slack + fi.smallest_normal * fi.eps
    off = (got.double() - want).abs() / tol
    assert (off <= 1).all(), f"{int((~(off <= 1)).sum())} off, worst {float(off.max()):.2f} times the tolerance"


# The tail's polynomial is off by 8.0e-7, the FP32 arithmetic around it rounds about 16 times (2^-24 each; two units of the last
# place for the hardware's exponential and one for its reciprocal among them), and the exponent a^2 / 2 by three roundings of
# 2^-24: a relative error of 8.0e-7 + (16 + 1.5 a^2) 2^-24 in Phi(-a); 1 - Phi(-a) and the sums with it round once more.
def tail_error(x):
    return 8.0e-7 + (16 + 1.5 * x * x) * 2.0 ** -24


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_gelu_keeps_its_relative_accuracy_in_16_bits(dt):
    x = span("words", dt)
    want = gelu64(x.double())
    got = through_a_product(x, "words", dt, dt, "gelu")
    within(got, want, tail_error(x.double()), 0.0)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_gelu_gradient_keeps_its_accuracy_in_16_bits(dt):
    z = cm(span("words", dt))
    zd = z.double()
    phi = zd.abs() * torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi)
    tail = 0.5 * torch.special.erfc(zd.abs() / math.sqrt(2))
    want = 0.5 * torch.special.erfc(-zd / math.sqrt(2)) + zd * torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi)
    got = through_a_product(torch.ones_like(z), "words", dt, dt, "gelu", z)
    slack = (tail + phi) * tail_error(zd) + 2.0 ** -23 * torch.maximum(phi, 0.5 * torch.special.erfc(-zd / math.sqrt(2)))
    within(got, want, 0.0, slack * (1 + torch.finfo(dt).eps))


# In 32 bits, what x / 2 * erfc(-x / sqrt(2)) costs when it is evaluated as it stands: the argument is off by two half steps
# (2^-23), which its exponential exp(-x^2 / 2) multiplies by x^2; the function by 4 units of the last place (2^-21 at
# most), the products around it by two half steps.  (The kernels carry the exponent's roundings along.)  The split sum,
# alpha and the bias add zeros to x and leave it exact.
def gelu32_error(x):
    return (x * x + 4 + 2) * 2.0 ** -23


@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("route", ["elements", "streamed", "several", "split"])
def test_gelu_keeps_its_relative_accuracy_in_32_bits(route, out):
    x = span(route, torch.float16)
    got = through_a_product(x, route, torch.float16, out, "gelu")
    within(got, gelu64(x.double()), gelu32_error(x.double()), 0.0)


@pytest.mark.parametrize("out", [torch.float32, torch.float16])
@pytest.mark.parametrize("route", ["elements", "streamed", "several", "split"])
def test_gelu_gradient_keeps_its_accuracy_in_32_bits(route, out):
    """Phi(z) and z phi(z), each to its own relative error (the exponential: its exponent rounded twice, two units of the last
    place), and their sum's rounding."""
    z = cm(span(route, out))
    zd = z.double()
    phi, tail = zd.abs() * torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi), 0.5 * torch.special.erfc(-zd / math.sqrt(2))
    got = through_a_product(torch.ones_like(z), route, torch.float16, out, "gelu", z)
    x = torch.zeros_like(zd)
    x[: min(ROUTES[route][0], ROUTES[route][2])] = 1
    slack = x * (tail * gelu32_error(zd) + phi * (zd * zd / 2 + 4 + 3) * 2.0 ** -23 + 2.0 ** -24 * (tail + phi))
    within(got, x * (tail + zd * torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi)), 0.0, slack * (1 + torch.finfo(out).eps))


@pytest.mark.parametrize("m,dt", [(128, torch.float32), (131, torch.float32), (131, torch.bfloat16)])
def test_activation_gradient_of_gelu_keeps_its_accuracy(m, dt):
    """The kernel of its own: in 32 bits, and element by element in 16."""
    z = cm(torch.linspace(-12, 12, m * 200, device="cuda", dtype=torch.float64).reshape(200, m).T.to(dt))
    zd = z.double()
    phi, tail = zd.abs() * torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi), 0.5 * torch.special.erfc(-zd / math.sqrt(2))
    dz = cm(torch.full((m, 200), -9.0, device="cuda", dtype=dt))
    GK.activation_gradient_(dz, cm(torch.ones(m, 200, device="cuda", dtype=dt)), z, ACT["gelu"])
    done()
    slack = tail * gelu32_error(zd) + phi * (zd * zd / 2 + 4 + 3) * 2.0 ** -23 + 2.0 ** -24 * (tail + phi)
    within(dz, tail + zd * torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi), 0.0, slack * (1 + torch.finfo(dt).eps))


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("route", list(ROUTES))
def test_activations_of_infinities_are_their_limits(route, out, act):
    """On every route alike: 0 and infinity (x itself without an activation), and a NaN stays one."""
    m, n, k = ROUTES[route]
    a, b = cm(torch.zeros(m, k, device="cuda", dtype=torch.float16)), cm(torch.zeros(k, n, device="cuda", dtype=torch.float16))
    bias = torch.zeros(m, device="cuda")
    bias[0], bias[3], bias[m - 1], bias[64] = -math.inf, math.inf, math.nan, -200.0
    d = cm(torch.full((m, n), -9.0, device="cuda", dtype=out))
    GK.matmul(conf(m, n, k, torch.float16, out), a, b, None, d, epilogue=Epilogue.BiasActivationResidual(bias, activation=ACT[act]))
    done()
    want = torch.zeros(m, n, device="cuda", dtype=torch.float64)
    want[3], want[m - 1] = math.inf, math.nan
    if act is None:
        want[0], want[64] = -math.inf, -200.0
    assert torch.equal(d.double().nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0))


@pytest.mark.parametrize("m,k,groups,n,streams", [(2048, 2048, 64, 8, True), (2048, 2048, 64, 64, False), (256, 128, 64, 64, True),
                                                   (4096, 4096, 8, 8, False), (8192, 16384, 2, 1, True), (8192, 16384, 2, 2, False)])
def test_grouped_columns_stream_while_the_worst_routing_allows(m, k, groups, n, streams):
    """All tokens may fall on one group, whose weights the streaming kernel would read once for each of them; the choice is made
    without knowing, and either kernel is right for any routing."""
    g = gen(314)
    w = ints(g, k, m, lo=-1, hi=1)
    a = w[:, :, None].expand(k, m, groups)                 # one matrix for all groups (row-major weights)
    b = cm(torch.zeros(k, n, device="cuda", dtype=torch.float16))
    b[: 64] = ints(g, 64, n)
    want = w.double().T @ b.double()
    cf = conf(m, n, k, torch.float16, torch.float32, True)
    for counts in ([1] * n + [0] * (groups - n), [0] * (groups - 1) + [n]):
        offsets, _ = offsets_of(counts)
        d = cm(torch.full((m, n), -9.0, device="cuda"))
        assert (GK.grouped_query(cf, a, b, None, d, offsets).kernel == 6) == streams
        GK.matmul_grouped(cf, a, b, None, d, offsets)
        done()
        assert torch.equal(d.double(), want)


@pytest.mark.parametrize("ta", [False, True])
def test_grouped_columns_of_unaligned_operands_without_room(ta):
    """More columns than the routing rule lets stream, and no workspace for the copies that the tensor cores would need: the
    streaming kernel takes them after all."""
    g = gen(315)
    m, k, groups, n = 1023, 2049, 64, 48
    w = ints(g, *((k, m) if ta else (m, k)), lo=-1, hi=1)
    a = w[:, :, None].expand(*w.shape, groups)
    b = ints(g, k, n, lo=-1, hi=1)
    cf = conf(m, n, k, torch.float16, torch.float32, ta)
    want = (w.double().T if ta else w.double()) @ b.double()
    for counts in ([1] * n + [0] * (groups - n), [0] * (groups - 1) + [n]):
        offsets, _ = offsets_of(counts)
        for room in (256, None):
            d = cm(torch.full((m, n), -9.0, device="cuda"))
            GK.matmul_grouped(cf, a, b, None, d, offsets, workspace=room and torch.empty(room, dtype=torch.uint8, device="cuda"))
            done()
            assert torch.equal(d.double(), want)
