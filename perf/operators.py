"""Group norm with an activation, the dense layer with bias, activation and residual, and the orthogonalised update of weight
matrices, as cases that can be timed and compared: `run` computes them by elementary torch operations, or by this package's
entry points where `own` is set.

Kinds:
  norm    y = act(group norm(x)) with the groups' statistics
  normg   its gradient: of x, of scale and bias
  dense   y = act(x w^T + bias) + residual, with what the activation was applied to where a training step keeps it
  denseg  its gradient: of x, w and bias (the residual's is dy itself)
  muon    one update of a set of weight matrices and their momenta
"""
import math

import torch

own = False

ACTS = ("none", "relu", "gelu", "silu")
EPS = 1e-5
MUON = {"lr": 0.02, "mu": 0.95, "decay": 0.01}
NS = (3.4445, -4.7750, 2.0315)   # coefficients of the five steps
NS_STEPS, NS_EPS = 5, 1e-7


def listed():
    return [
        # one small image in the last layers of a network that answers single requests: latency and nothing else
        {"name": "norm b1", "kind": "norm", "n": 1, "c": 64, "h": 8, "w": 8, "groups": 8, "last": False, "act": "silu"},
        # the first stage of the wide residual network at batch 128
        {"name": "norm wrn stage 1", "kind": "norm", "n": 128, "c": 160, "h": 32, "w": 32, "groups": 32, "last": False, "act": "relu"},
        # a training batch of odd images, channels last, as a layer of dense products reads them
        {"name": "norm last ragged", "kind": "norm", "n": 37, "c": 200, "h": 29, "w": 33, "groups": 25, "last": True, "act": "gelu"},
        # the way back through the second stage
        {"name": "normg wrn stage 2", "kind": "normg", "n": 128, "c": 320, "h": 16, "w": 16, "groups": 32, "last": False, "act": "silu"},
        # ... and through channels-last images
        {"name": "normg last", "kind": "normg", "n": 64, "c": 128, "h": 32, "w": 32, "groups": 16, "last": True, "act": "gelu"},
        # a single image in the dense layers of VGG-16: one row, the weights' bytes
        {"name": "dense b1", "kind": "dense", "m": 1, "n": 4096, "k": 4096, "act": "gelu", "residual": True, "keep": False},
        # the 784-512-512-10 network's first layer at batch 256
        {"name": "dense mlp b256", "kind": "dense", "m": 256, "n": 512, "k": 784, "act": "gelu", "residual": False, "keep": True},
        # a large layer of a residual network of dense layers
        {"name": "dense large", "kind": "dense", "m": 8192, "n": 4096, "k": 4096, "act": "silu", "residual": True, "keep": True},
        # a training step's way back through a layer of odd sizes
        {"name": "denseg ragged", "kind": "denseg", "m": 1000, "n": 1777, "k": 1111, "act": "gelu"},
        # the first 3 x 3 filters of a small network, one matrix: latency
        {"name": "muon one 64x576", "kind": "muon", "shapes": "64x576", "nesterov": True},
        # every matrix of VGG-16 with the dense layers 512-512-10
        {"name": "muon vgg16", "kind": "muon", "nesterov": True,
         "shapes": "64x27,64x576,128x576,128x1152,256x1152,256x2304,256x2304,512x2304,512x4608,512x4608,512x4608,512x4608,"
                   "512x4608,512x512,512x512,10x512"},
        # the last stage of the wide residual network
        {"name": "muon wrn stage 3", "kind": "muon", "nesterov": True,
         "shapes": "640x2880,640x5760,640x5760,640x5760,640x5760,640x5760,640x5760,640x5760"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ones' ranges, at most as costly as the largest of them.  Two kinds of norm are left out: the gradient
    through a relu, where either answer is one if z lies within a rounding of zero, and groups of a handful of values, whose
    gradient is what remains after its leading digits have cancelled."""
    while True:
        case = _draw(rng)
        w = work(case)
        small = case["kind"] in ("norm", "normg") and case["c"] // case["groups"] * case["h"] * case["w"] < 32
        if w["flops"] <= 2.7e11 and w["bytes"] <= 4.1e8 and not small:
            return case


def _draw(rng):
    kind = rng.choice(["norm", "normg", "dense", "dense", "denseg", "muon", "muon"])
    if kind in ("norm", "normg"):
        groups = rng.choice([1, 2, 4, 8, 16, 32])
        return {"kind": kind, "n": _log_int(rng, 1, 256), "c": groups * _log_int(rng, 1, 40), "h": _log_int(rng, 1, 64),
                "w": _log_int(rng, 1, 64), "groups": groups, "last": rng.random() < 0.5,
                "act": rng.choice(ACTS if kind == "norm" else ("none", "gelu", "silu"))}
    if kind in ("dense", "denseg"):
        case = {"kind": kind, "m": _log_int(rng, 1, 8192), "n": _log_int(rng, 10, 8192), "k": _log_int(rng, 16, 8192),
                "act": rng.choice(ACTS)}
        if kind == "dense":
            case["residual"], case["keep"] = rng.random() < 0.5, case["act"] != "none" and rng.random() < 0.5
        return case
    count = rng.randint(1, 16)
    return {"kind": kind, "nesterov": rng.random() < 0.7,
            "shapes": ",".join("%dx%d" % (_log_int(rng, 8, 2048), _log_int(rng, 8, 8192)) for _ in range(count))}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _xshape(case):
    return (case["n"], case["h"], case["w"], case["c"]) if case["last"] else (case["n"], case["c"], case["h"], case["w"])


def work(case):
    if case["kind"] in ("norm", "normg"):
        v, back = case["n"] * case["c"] * case["h"] * case["w"], case["kind"] == "normg"
        return {"bytes": 4 * ((3 if back else 2) * v + 2 * case["n"] * case["groups"] + (4 if back else 2) * case["c"]),
                "flops": (20 if back else 10) * v}
    if case["kind"] in ("dense", "denseg"):
        m, n, k = case["m"], case["n"], case["k"]
        if case["kind"] == "dense":
            return {"bytes": 4 * (m * k + n * k + n + m * n * (1 + case["residual"] + case["keep"])), "flops": 2 * m * n * k}
        return {"bytes": 4 * (m * n * (1 if case["act"] == "none" else 2) + 2 * m * k + 2 * n * k + n), "flops": 4 * m * n * k}
    # A = X X^T and A A are symmetric: half of each is all there is to compute
    flops = sum(NS_STEPS * (3 * min(s) ** 2 * max(s) + min(s) ** 3) for s in _shapes(case))
    return {"bytes": 20 * sum(r * c for r, c in _shapes(case)), "flops": flops}


# ------------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda") * scale


def _inputs(case, seed):
    """What the operator reads, made from the seed alone."""
    g = _gen(seed)
    if case["kind"] in ("norm", "normg"):
        c, shape = case["c"], _xshape(case)
        per = (1, 1, 1, c) if case["last"] else (1, c, 1, 1)
        # activations whose channels differ in level and spread, as a convolution's do
        x = _randn(g, *shape) * (0.5 + torch.rand(per, generator=g, device="cuda")) + 0.5 * _randn(g, *per)
        t = {"x": x, "scale": 1.0 + 0.1 * _randn(g, c), "bias": 0.1 * _randn(g, c)}
        if case["kind"] == "normg":
            t["dy"] = _randn(g, *shape, scale=0.01)
            d, dims = _grouped(case, x).double(), (1, 3) if case["last"] else (2, 3)
            rstd = (d.var(dims, unbiased=False) + EPS).rsqrt()
            t["stats"] = torch.cat([d.mean(dims).reshape(-1), rstd.reshape(-1)]).float()   # as the forward pass left them
        return t
    if case["kind"] in ("dense", "denseg"):
        m, n, k = case["m"], case["n"], case["k"]
        t = {"x": _randn(g, m, k), "w": _randn(g, n, k, scale=math.sqrt(2.0 / k))}
        if case["kind"] == "dense":
            t["bias"] = _randn(g, n, scale=0.1)
            if case["residual"]:
                t["residual"] = _randn(g, m, n)
        else:
            t["dy"] = _randn(g, m, n, scale=0.01)
            if case["act"] != "none":
                t["pre"] = _randn(g, m, n, scale=1.4)
        return t
    t = {"w": [], "g": [], "m": []}
    for r, c in _shapes(case):
        t["w"].append(_randn(g, r, c, scale=math.sqrt(2.0 / c)))
        # a gradient's few strong directions over many weak ones
        rank = max(1, min(r, c) // 16)
        strong = _randn(g, r, rank) @ _randn(g, rank, c)
        t["g"].append(1e-3 * (_randn(g, r, c) + strong / math.sqrt(rank)))
        t["m"].append(1e-3 * _randn(g, r, c))
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, "t": t}
    if own:
        _plan(state)
    return state


# ------------------------------------------------------------------------------------------------ the plain forms

def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * torch.erfc(z * -math.sqrt(0.5))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(dy, z, act):
    if act == "relu":
        return torch.where(z > 0, dy, torch.zeros_like(dy))
    if act == "gelu":
        return dy * (0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return dy * (s * (1 + z * (1 - s)))
    return dy


def _grouped(case, x):
    """x as [n, groups, channels of a group, pixels], or [n, pixels, groups, channels of a group] where channels are last."""
    n, g, p = case["n"], case["groups"], case["h"] * case["w"]
    return x.reshape(n, p, g, case["c"] // g) if case["last"] else x.reshape(n, g, case["c"] // g, p)


def _spread(case, s):
    """One value per (sample, group) against what _grouped gives."""
    s = s.reshape(case["n"], case["groups"])
    return s[:, None, :, None] if case["last"] else s[:, :, None, None]


def _per_channel(case, v):
    v = v.reshape(case["groups"], -1)
    return v[None, None] if case["last"] else v[None, :, :, None]


def _norm(case, t):
    x, dims = _grouped(case, t["x"]), (1, 3) if case["last"] else (2, 3)
    mean = x.mean(dims)
    d = x - _spread(case, mean)
    rstd = (d.square().mean(dims) + EPS).rsqrt()
    z = d * _spread(case, rstd) * _per_channel(case, t["scale"]) + _per_channel(case, t["bias"])
    return {"y": _act(z, case["act"]).reshape(t["x"].shape), "mean": mean.reshape(-1), "rstd": rstd.reshape(-1)}


def _norm_grad(case, t):
    x, dy = _grouped(case, t["x"]), _grouped(case, t["dy"])
    dims, over = ((1, 3), (0, 1)) if case["last"] else ((2, 3), (0, 3))
    mean, rstd = (_spread(case, s) for s in t["stats"].chunk(2))
    xhat, scale = (x - mean) * rstd, _per_channel(case, t["scale"])
    dz = _act_grad(dy, xhat * scale + _per_channel(case, t["bias"]), case["act"])
    ds = dz * scale
    s1, s2 = ds.mean(dims, keepdim=True), (ds * xhat).mean(dims, keepdim=True)
    return {"dx": (rstd * (ds - s1 - xhat * s2)).reshape(t["x"].shape), "dscale": (dz * xhat).sum(over).reshape(-1),
            "dbias": dz.sum(over).reshape(-1)}


def _dense(case, t):
    pre = t["x"] @ t["w"].t() + t["bias"]
    y = _act(pre, case["act"])
    out = {"y": y + t["residual"] if case["residual"] else y}
    if case["keep"]:
        out["pre"] = pre
    return out


def _dense_grad(case, t):
    dz = _act_grad(t["dy"], t["pre"], case["act"]) if case["act"] != "none" else t["dy"]
    return {"dx": dz @ t["w"], "dw": dz.t() @ t["x"], "dbias": dz.sum(0)}


def _orthogonal(u):
    x = u / (torch.linalg.vector_norm(u) + NS_EPS)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    for _ in range(NS_STEPS):
        a = x @ x.t()
        x = NS[0] * x + (NS[1] * a + NS[2] * (a @ a)) @ x
    return x.t() if tall else x


def _muon(case, t):
    lr, mu, decay = MUON["lr"], MUON["mu"], MUON["decay"]
    for w, g, m in zip(t["w"], t["g"], t["m"]):
        m.mul_(mu).add_(g)
        o = _orthogonal(g + mu * m if case["nesterov"] else m)
        w.mul_(1 - lr * decay).sub_(o * (lr * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))))
    return {"w": t["w"], "m": t["m"]}


_PLAIN = {"norm": _norm, "normg": _norm_grad, "dense": _dense, "denseg": _dense_grad, "muon": _muon}


# ------------------------------------------------------------------------------------------------ this package's entry points

def _ref(t):
    """A torch tensor as an operand of the entry points; it stays the tensor's memory."""
    from dopt_amd import ops
    return None if t is None else ops.Tensor(tuple(t.shape), "float32", _ptr=t.data_ptr(), _owner=t)


def _plan(state):
    """What a program keeps between calls: its operands as the entry points take them, result buffers, the optimizer's handle."""
    from dopt_amd import ops
    case, t = state["case"], state["t"]
    if case["kind"] == "muon":
        refs = {k: [_ref(x) for x in v] for k, v in t.items()}
        state["opt"] = ops.MuonOptimizer(refs["w"], refs["g"], refs["m"])
        return
    state["r"] = {k: _ref(v) for k, v in t.items()}
    if case["kind"] in ("norm", "normg"):
        v, c, ng = t["x"].numel(), case["c"], case["n"] * case["groups"]
        packed = torch.empty(v + 2 * (ng if case["kind"] == "norm" else c), device="cuda")
        state["o"] = {"out": _ref(packed)}
        a, b = ("mean", "rstd") if case["kind"] == "norm" else ("dscale", "dbias")
        tail = packed[v:].chunk(2)
        state["outs"] = {"y" if case["kind"] == "norm" else "dx": packed[:v].view(t["x"].shape), a: tail[0], b: tail[1]}
        return
    m, n, k = case["m"], case["n"], case["k"]
    shapes = {"dx": (m, k), "dw": (n, k), "dbias": (n,)}
    if case["kind"] == "dense":
        shapes = {"y": (m, n), "pre": (m, n)} if case["keep"] else {"y": (m, n)}
    state["outs"] = {name: torch.empty(s, device="cuda") for name, s in shapes.items()}
    state["o"] = {name: _ref(v) for name, v in state["outs"].items()}


def _call(state):
    from dopt_amd import ops
    case = state["case"]
    if case["kind"] == "muon":
        state["opt"].step(MUON["lr"], MUON["mu"], case["nesterov"], MUON["decay"])
        return {"w": state["t"]["w"], "m": state["t"]["m"]}
    r, o = state["r"], state["o"]
    if case["kind"] == "norm":
        ops.group_norm(r["x"], r["scale"], r["bias"], case["groups"], EPS, case["act"], case["last"], out=o["out"])
    elif case["kind"] == "normg":
        ops.group_norm_grad(r["dy"], r["x"], r["scale"], r["bias"], r["stats"], case["groups"], case["act"], case["last"], out=o["out"])
    elif case["kind"] == "dense":
        ops.dense_act(r["x"], r["w"], r["bias"], r.get("residual"), case["act"], out=o["y"], pre=o.get("pre"))
    else:
        ops.dense_act_grad(r["dy"], r["x"], r["w"], r.get("pre"), case["act"], dx=o["dx"], dw=o["dw"], dbias=o["dbias"])
    return state["outs"]


def run(state):
    if own:
        return _call(state)
    return _PLAIN[state["case"]["kind"]](state["case"], state["t"])


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits

def _phi(z):
    return torch.special.ndtr(z)


def _sigma(z):
    return torch.sigmoid(z)


def _exact_act(z, act):
    return {"none": lambda: z, "relu": lambda: z * (z > 0), "gelu": lambda: z * _phi(z), "silu": lambda: z * _sigma(z)}[act]()


def _exact_slope(z, act):
    if act == "gelu":
        return _phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        return _sigma(z) + z * _sigma(z) * _sigma(-z)
    return torch.ones_like(z) if act == "none" else (z > 0).double()


def _exact_norm(case, t):
    # channels first: one row per sample and group
    n, g, c, p = case["n"], case["groups"], case["c"], case["h"] * case["w"]
    flat = (lambda x: x.reshape(n, p, c).transpose(1, 2)) if case["last"] else (lambda x: x.reshape(n, c, p))
    back = (lambda x: x.reshape(n, c, p).transpose(1, 2)) if case["last"] else (lambda x: x.reshape(n, c, p))
    shape = t["x"].shape
    x = flat(t["x"]).reshape(n * g, -1)
    ch = lambda v: v.reshape(1, c, 1).expand(n, c, p).reshape(n * g, -1)  # noqa: E731
    if case["kind"] == "norm":
        mean, rstd = x.mean(1), 1 / torch.sqrt(x.var(1, unbiased=False) + EPS)
        z = (x - mean[:, None]) * rstd[:, None] * ch(t["scale"]) + ch(t["bias"])
        return {"y": back(_exact_act(z, case["act"])).reshape(shape), "mean": mean, "rstd": rstd}
    mean, rstd = t["stats"].reshape(2, n * g, 1)
    xhat = (x - mean) * rstd
    dz = flat(t["dy"]).reshape(n * g, -1) * _exact_slope(xhat * ch(t["scale"]) + ch(t["bias"]), case["act"])
    dxhat = dz * ch(t["scale"])
    dx = rstd * (dxhat - dxhat.mean(1, keepdim=True) - xhat * (dxhat * xhat).mean(1, keepdim=True))
    return {"dx": back(dx).reshape(shape), "dscale": (dz * xhat).reshape(n, c, p).sum((0, 2)),
            "dbias": dz.reshape(n, c, p).sum((0, 2))}


def _exact_dense(case, t):
    if case["kind"] == "dense":
        pre = torch.addmm(t["bias"], t["x"], t["w"].t())
        y = _exact_act(pre, case["act"])
        out = {"y": y if not case["residual"] else y + t["residual"]}
        return dict(out, pre=pre) if case["keep"] else out
    dz = t["dy"] if case["act"] == "none" else t["dy"] * _exact_slope(t["pre"], case["act"])
    return {"dx": torch.mm(dz, t["w"]), "dw": torch.mm(dz.t(), t["x"]), "dbias": dz.sum(0)}


def _exact_muon(case, t):
    lr, mu, decay = MUON["lr"], MUON["mu"], MUON["decay"]
    out = {"w": [], "m": []}
    for w, g, m in zip(t["w"], t["g"], t["m"]):
        m = g + m * mu
        u = g + m * mu if case["nesterov"] else m
        x = u / (u.square().sum().sqrt() + NS_EPS)
        # the polynomial a + b s + c s^2 of s = X X^T (or X^T X), whichever is the smaller
        for _ in range(NS_STEPS):
            s = x @ x.T if x.shape[0] <= x.shape[1] else x.T @ x
            p = NS[0] * torch.eye(len(s), dtype=s.dtype, device=s.device) + NS[1] * s + NS[2] * (s @ s)
            x = p @ x if x.shape[0] <= x.shape[1] else x @ p
        out["w"].append(w - lr * decay * w - lr * max(1.0, w.shape[0] / w.shape[1]) ** 0.5 * x)
        out["m"].append(m)
    return out


def exact(case, seed):
    t = {k: [x.double() for x in v] if isinstance(v, list) else v.double() for k, v in _inputs(case, seed).items()}
    if case["kind"] in ("norm", "normg"):
        return _exact_norm(case, t)
    return _exact_dense(case, t) if case["kind"] in ("dense", "denseg") else _exact_muon(case, t)
