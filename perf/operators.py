"""The layer-level operators on real sizes: products with a fused bias, activation and residual, the gradients behind
them, and products grouped by expert - in plain torch, and through the package.

All matrices are column-major, as everywhere in the package: a torch tensor of shape (rows, columns) with stride 1
along the rows.  Tokens are columns (features x tokens).  The operators:

  fused           D = act(W X + bias) + R, keeping Z = W X + bias when a backward pass will need it
  gradient        D = (W^T dY) * act'(Z), the gradient handed to the layer below, activation included
  activation      dZ = dD * act'(Z) and the bias gradient, dZ summed over the tokens (of each expert)
  grouped         D[:, J_g] = act(W_g X[:, J_g] + bias_g), J_g the columns of expert g
  grouped_dgrad   D[:, J_g] = (W_g^T dY[:, J_g]) * act'(Z[:, J_g])
  grouped_outer   D_g = dY[:, J_g] X[:, J_g]^T (+ D_g), the weight gradient of expert g

Expert g owns the columns offsets[g] .. offsets[g + 1]; columns behind offsets[-1] are padding and stay as they were.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of one request through a dense layer (weights stored as torch.nn.Linear does): latency
        dict(name="fused_token", op="fused", m=4096, k=4096, n=1, dtype="bf16", act="gelu", wt=True, z=False),
        # a handful of requests decoding together
        dict(name="fused_few", op="fused", m=8192, k=2048, n=7, dtype="fp16", act="silu", wt=False, z=False),
        # sizes that no tile divides and no 16-byte row holds
        dict(name="fused_odd", op="fused", m=1000, k=1111, n=777, dtype="fp16", act="relu", wt=False, z=True),
        # the up-projection of a dense layer over a long batch, in training
        dict(name="fused_train", op="fused", m=8192, k=8192, n=4096, dtype="bf16", act="gelu", wt=True, z=True),
        # the gradient through the down-projection and the activation before it
        dict(name="gradient_train", op="gradient", m=8192, k=2048, n=4096, dtype="bf16", act="gelu", wt=False),
        # last layer's activation gradient on a short ragged batch of experts
        dict(name="activation_small", op="activation", m=2048, n=333, groups=8, skew=1.0, pad=21, dtype="fp16", act="silu"),
        # the same over a whole training batch, one bias
        dict(name="activation_large", op="activation", m=8192, n=16384, groups=1, skew=0.0, pad=0, dtype="bf16", act="gelu"),
        # eight tokens, two experts each, decoding over 64 experts
        dict(name="grouped_decode", op="grouped", m=2048, k=2048, n=16, groups=64, skew=0.5, pad=0, dtype="bf16",
             act="silu", wt=True, z=False),
        # a prompt batch over 32 experts
        dict(name="grouped_prefill", op="grouped", m=2048, k=2048, n=8192, groups=32, skew=0.7, pad=100, dtype="bf16",
             act="gelu", wt=True, z=True),
        # the input gradient of the same layer
        dict(name="grouped_dgrad", op="grouped_dgrad", m=2048, k=1024, n=8192, groups=32, skew=0.7, pad=100, dtype="fp16",
             act="gelu", wt=False),
        # weight gradients of a small layer: few tokens per expert, some without any
        dict(name="outer_ragged", op="grouped_outer", m=1032, k=520, n=1500, groups=16, skew=1.5, pad=33, dtype="fp16",
             out="fp16", accumulate=False),
        # weight gradients accumulated in 32 bits over a training batch
        dict(name="outer_train", op="grouped_outer", m=4096, k=2048, n=16384, groups=16, skew=0.7, pad=0, dtype="bf16",
             out="fp32", accumulate=True),
    ]


def draw(rng):
    def size(lo, hi, step=1):
        return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)

    while True:
        op = rng.choice(["fused", "fused", "gradient", "activation", "grouped", "grouped", "grouped_dgrad", "grouped_outer"])
        step = rng.choice([1, 8, 8, 64])
        c = dict(op=op, m=size(64, 8192, step), n=size(1, 16384), dtype=rng.choice(["bf16", "fp16"]),
                 act=rng.choice(["relu", "gelu", "silu"]))
        if op != "activation":
            c["k"] = size(64, 8192, step)
        if op in ("fused", "gradient", "grouped", "grouped_dgrad"):
            c["wt"] = rng.random() < 0.5
        if op in ("fused", "grouped"):
            c["z"] = rng.random() < 0.5
        if op in ("activation", "grouped", "grouped_dgrad", "grouped_outer"):
            c["groups"] = size(1, 128)
            c["skew"] = rng.choice([0.0, 0.5, 1.0, 1.5])
            c["pad"] = rng.choice([0, 0, size(1, 64)])
        if op == "grouped_outer":
            c["accumulate"] = rng.random() < 0.5
            c["out"] = "fp32" if c["accumulate"] else rng.choice(["fp32", c["dtype"]])
            del c["act"]
        w = work(c)
        if w["flops"] <= 5.0e11 and w["bytes"] <= 8.0e8 and c.get("groups", 1) * c["m"] * c.get("k", 1) <= 5.0e8:
            return c


def _counts(c):
    """Columns per expert, falling like a power of the rank; the largest remainders get the columns left over."""
    share = [(g + 1.0) ** -c["skew"] for g in range(c["groups"])]
    want = [c["n"] * s / sum(share) for s in share]
    have = [int(w) for w in want]
    order = sorted(range(c["groups"]), key=lambda g: (have[g] - want[g], g))
    for g in order[: c["n"] - sum(have)]:
        have[g] += 1
    return have


def work(c):
    es = 2
    m, n = c["m"], c["n"]
    if c["op"] == "activation":
        return {"bytes": 3 * m * n * es + 4 * m * c["groups"], "flops": 20 * m * n}
    k = c["k"]
    if c["op"] == "fused":
        return {"bytes": es * (m * k + k * n + 2 * m * n + (m * n if c["z"] else 0)) + 4 * m, "flops": 2 * m * n * k}
    if c["op"] == "gradient":
        return {"bytes": es * (m * k + k * n + 2 * m * n), "flops": 2 * m * n * k}
    active = sum(1 for x in _counts(c) if x)
    if c["op"] == "grouped":
        return {"bytes": es * (active * m * k + k * n + m * n + (m * n if c["z"] else 0)) + 4 * m * active, "flops": 2 * m * n * k}
    if c["op"] == "grouped_dgrad":
        return {"bytes": es * (active * m * k + k * n + 2 * m * n), "flops": 2 * m * n * k}
    ob = 4 if c["out"] == "fp32" else es
    return {"bytes": es * (m + k) * n + c["groups"] * m * k * ob * (2 if c["accumulate"] else 1), "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[c["dtype"]]

    def mat(*shape, scale=1.0, dtype=dt):
        """A column-major array of normal values: (rows, columns[, experts])."""
        t = torch.randn(tuple(reversed(shape)), generator=gen, device="cuda", dtype=torch.float32)
        return (t * scale).to(dtype).permute(*reversed(range(len(shape))))

    m, n, op = c["m"], c["n"], c["op"]
    s = {"case": c}
    groups = c.get("groups", 0)
    total = n + c.get("pad", 0)
    if groups:
        perm = torch.randperm(groups, generator=torch.Generator().manual_seed(seed)).tolist()
        have = _counts(c)
        offs = [0]
        for g in perm:
            offs.append(offs[-1] + have[g])
        s["bounds"] = offs
        s["offsets"] = torch.tensor(offs, dtype=torch.int32, device="cuda")
    if op == "activation":
        s["dd"], s["z"] = mat(m, total), mat(m, total)
        s["dz"] = torch.zeros((total, m), dtype=dt, device="cuda").T
        s["db"] = torch.zeros((groups, m), dtype=torch.float32, device="cuda").T
        return s
    k = c["k"]
    if op == "grouped_outer":
        s["dy"], s["x"] = mat(m, total), mat(k, total)
        s["d"] = mat(m, k, groups, dtype=_TYPES[c["out"]]) if c["accumulate"] \
            else torch.zeros((groups, k, m), dtype=_TYPES[c["out"]], device="cuda").permute(2, 1, 0)
        if c["accumulate"]:
            s["c"] = s["d"].clone()
        return s
    w_shape = (k, m) if c["wt"] else (m, k)          # wt: each output row's weights are consecutive
    s["w"] = mat(*w_shape, *([groups] if groups else []), scale=k ** -0.5)
    s["x"] = mat(k, total)
    s["d"] = torch.zeros((total, m), dtype=dt, device="cuda").T
    if op in ("fused", "grouped"):
        s["bias"] = mat(m, *([groups] if groups else []), scale=0.1, dtype=torch.float32)
        if c["z"]:
            s["z"] = torch.zeros((total, m), dtype=dt, device="cuda").T
        if op == "fused":
            s["r"] = mat(m, total)
    else:
        s["z"] = mat(m, total)
    return s


def _package():
    root = Path(__file__).resolve().parents[1] / "gemmkernels.jl_b200"
    if str(root) not in sys.path:
        sys.path.insert(0, str(root))
    import gemmkernels_b200
    return gemmkernels_b200


def _bound(s):
    """The package's operator with its arguments lowered once, as a program that runs it every step keeps it."""
    GK = _package()
    c, op = s["case"], s["case"]["op"]
    act = {"relu": GK.Transform.ReLU, "gelu": GK.Transform.GELU, "silu": GK.Transform.SiLU, None: lambda: None}[c.get("act")]()
    if op == "activation":
        offsets = s["offsets"] if c["groups"] > 1 or c["pad"] else None
        return GK.bind_activation_gradient(s["dz"], s["dd"], s["z"], act, bias_gradient=s["db"], offsets=offsets)
    et = {"bf16": GK.BFloat16, "fp16": GK.Float16, "fp32": GK.Float32}
    t = et[c["dtype"]]
    out = et[c.get("out", c["dtype"])]
    L, operator = GK.Layout, GK.Operator.TCGen05Operator[t, GK.Float32]
    m, k, total = c["m"], c["k"], c["n"] + c.get("pad", 0)
    if op == "grouped_outer":
        conf = GK.get_config(gemm_shape=(m, k, total), operator=operator, global_a_layout=L.ColMajor[t],
                             global_b_layout=L.RowMajor[t], global_d_layout=L.ColMajor[out], is_b_col_major=False,
                             global_c_layout=L.ColMajor[out] if c["accumulate"] else L.Zero[out])
        return GK.bind_grouped_outer(conf, s["dy"], s["x"], s.get("c"), s["d"], s["offsets"])
    conf = GK.get_config(gemm_shape=(m, total, k), operator=operator, is_a_col_major=not c["wt"],
                         global_a_layout=(L.RowMajor if c["wt"] else L.ColMajor)[t], global_b_layout=L.ColMajor[t],
                         global_c_layout=L.ColMajor[out] if op == "fused" else L.Zero[out],
                         global_d_layout=L.ColMajor[out])
    if op in ("fused", "grouped"):
        epilogue = GK.Epilogue.BiasActivationResidual(s["bias"], activation=act, preactivation=s.get("z"))
    else:
        epilogue = GK.Epilogue.ActivationGradient(s["z"], act)
    if op in ("grouped", "grouped_dgrad"):
        return GK.bind_grouped(conf, s["w"], s["x"], None, s["d"], s["offsets"], epilogue=epilogue)
    return GK.bind(conf, s["w"], s["x"], s.get("r"), s["d"], epilogue=epilogue)


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        s["call"] = _bound(s)
    return s


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def _act(x, name):
    if name == "relu":
        return x.clamp(min=0)
    if name == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * 0.5 ** 0.5))
    return x / (1.0 + torch.exp(-x))


def _act_gradient(x, name):
    if name == "relu":
        return (x > 0).to(x.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(x * 0.5 ** 0.5)) + x * torch.exp(-0.5 * x * x) * (2.0 * math.pi) ** -0.5
    sig = 1.0 / (1.0 + torch.exp(-x))
    return sig * (1.0 + x * (1.0 - sig))


def _outputs(s):
    c = s["case"]
    if c["op"] == "activation":
        return {"dz": s["dz"], "db": s["db"]}
    return {"d": s["d"], "z": s["z"]} if c.get("z") else {"d": s["d"]}


def run(s):
    if own:
        s["call"]()
        return _outputs(s)
    c, op = s["case"], s["case"]["op"]
    if op in ("fused", "gradient"):
        w = s["w"].T.float() if c["wt"] else s["w"].float()
        p = w @ s["x"].float()
        if op == "gradient":
            s["d"].copy_(p * _act_gradient(s["z"].float(), c["act"]))
            return _outputs(s)
        p += s["bias"][:, None]
        if c["z"]:
            s["z"].copy_(p)
        s["d"].copy_(_act(p, c["act"]) + s["r"].float())
        return _outputs(s)
    for g in range(c["groups"]):
        lo, hi = s["bounds"][g], s["bounds"][g + 1]
        if op == "activation":
            dz = s["dd"][:, lo:hi].float() * _act_gradient(s["z"][:, lo:hi].float(), c["act"])
            s["dz"][:, lo:hi] = dz
            s["db"][:, g] = dz.sum(1)
        elif op == "grouped_outer":
            p = s["dy"][:, lo:hi].float() @ s["x"][:, lo:hi].float().T
            s["d"][:, :, g] = p + s["c"][:, :, g].float() if c["accumulate"] else p
        elif hi > lo:
            w = s["w"][:, :, g].T.float() if c["wt"] else s["w"][:, :, g].float()
            p = w @ s["x"][:, lo:hi].float()
            if op == "grouped_dgrad":
                s["d"][:, lo:hi] = p * _act_gradient(s["z"][:, lo:hi].float(), c["act"])
                continue
            p += s["bias"][:, g:g + 1]
            if c["z"]:
                s["z"][:, lo:hi] = p
            s["d"][:, lo:hi] = _act(p, c["act"])
    return _outputs(s)


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _phi64(x):
    """Value and slope of the activation at x: {name: (f, f')}."""
    cdf = torch.special.erfc(-x / math.sqrt(2.0)) / 2.0
    pdf = torch.exp(-x.square() / 2.0) / math.sqrt(2.0 * math.pi)
    sig = torch.sigmoid(x)
    pos = torch.heaviside(x, torch.zeros((), dtype=x.dtype, device=x.device))
    return {"relu": (x * pos, pos), "gelu": (x * cdf, cdf + x * pdf), "silu": (x * sig, sig + x * sig * (1.0 - sig))}


def exact(case, seed):
    s = _inputs(case, seed)
    op, name = case["op"], case.get("act")
    cuts = s.get("bounds", [0, case["n"]])
    total = case["n"] + case.get("pad", 0)

    def blank(*shape):
        return torch.zeros(shape, dtype=torch.float64, device="cuda")

    if op == "activation":
        dz, db = blank(case["m"], total), blank(case["m"], case["groups"])
        for g, (a, b) in enumerate(zip(cuts, cuts[1:])):
            dz[:, a:b] = torch.mul(s["dd"][:, a:b].double(), _phi64(s["z"][:, a:b].double())[name][1])
            db[:, g] = dz[:, a:b].sum(dim=1)
        return {"dz": dz, "db": db}
    if op == "grouped_outer":
        d = blank(case["m"], case["k"], case["groups"])
        for g, (a, b) in enumerate(zip(cuts, cuts[1:])):
            d[:, :, g] = torch.einsum("mt,kt->mk", s["dy"][:, a:b].double(), s["x"][:, a:b].double())
        return {"d": d + s["c"].double() if case["accumulate"] else d}
    d, z = blank(case["m"], total), blank(case["m"], total)
    for g, (a, b) in enumerate(zip(cuts, cuts[1:])):
        w = (s["w"] if s["w"].dim() == 2 else s["w"][:, :, g]).double()
        z[:, a:b] = torch.einsum("km,kt->mt" if case["wt"] else "mk,kt->mt", w, s["x"][:, a:b].double())
        if op in ("fused", "grouped"):
            z[:, a:b] += (s["bias"] if s["bias"].dim() == 1 else s["bias"][:, g]).double().unsqueeze(1)
            d[:, a:b] = _phi64(z[:, a:b])[name][0]
        else:
            d[:, a:b] = z[:, a:b] * _phi64(s["z"][:, a:b].double())[name][1]
    if op == "fused":
        d += s["r"].double()
    return {"d": d, "z": z} if case.get("z") else {"d": d}
