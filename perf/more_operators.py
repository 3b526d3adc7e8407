"""The norms around a block with its gate and residual scale, dense layers of groups of rows, and the norm of all gradients with
clipping, as cases that can be timed and compared: `run` computes them by elementary torch operations, or by this package's entry
points where `own` is set.

Kinds:
  join     y = scale x + gate norm(branch), h = norm(y): what lies between two blocks of a residual network
  joing    its gradient: of x, the branch, the gate and the norms' scales and biases
  groups   y = act(x w^T + bias) with a w and a bias for each group of consecutive rows; rows of no group give zeros
  groupsg  its gradient: of x, w and bias
  clip     gradients times min(1, max / their norm), and the norm
  step     one ADAM update with the gradients so scaled, and the norm
"""
import math

import torch

own = False

EPS = 1e-5
ADAM = {"alpha": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8}


def _text(sizes):
    return ",".join(str(s) for s in sizes)


def _ints(text):
    return [int(v) for v in text.split(",")]


def _vgg16():
    """The tensors of VGG-16 with batch norm and the dense layers 512-512-10: filters, biases, scales, shifts."""
    sizes, c = [], 3
    for k in (64, 64, 128, 128, 256, 256, 256, 512, 512, 512, 512, 512, 512):
        sizes += [k * c * 9, k, k, k]
        c = k
    return sizes + [512 * 512, 512, 512 * 512, 512, 10 * 512, 10]


def _wrn():
    """The tensors of the wide residual network of 28 layers, ten times as wide."""
    sizes, c = [16 * 27], 16
    for k in (160, 320, 640):
        for block in range(4):
            sizes += [c, c, k * c * 9, k, k, k * k * 9] + ([k * c] if block == 0 else [])
            c = k
    return sizes + [c, c, 10 * c, 10]


def listed():
    return [
        # one row between two blocks of a network that answers single requests: latency and nothing else
        {"name": "join b1", "kind": "join", "rows": 1, "cols": 512, "gates": 1, "post": "layer", "pre": "layer", "scale": 1.0},
        # a training batch of wide rows
        {"name": "join wide", "kind": "join", "rows": 8192, "cols": 4096, "gates": 1, "post": "rms", "pre": "rms", "scale": 1.0},
        # the way back, 37 samples of 111 rows, each with a gate of its own, rows of an odd length
        {"name": "joing ragged", "kind": "joing", "rows": 4107, "cols": 1111, "gates": 37, "post": "layer", "pre": "layer", "scale": 0.8},
        # ... through a large batch with one gate for all rows
        {"name": "joing large", "kind": "joing", "rows": 16384, "cols": 1024, "gates": 1, "post": "rms", "pre": "layer", "scale": 1.0},
        # a handful of requests at eight groups: the bytes of w
        {"name": "groups b64", "kind": "groups", "rows": 64, "sizes": "9,0,17,3,11,8,14,2", "n": 512, "k": 512, "act": "silu", "keep": False},
        # a training batch that falls unevenly on eight groups
        {"name": "groups train", "kind": "groups", "rows": 4096, "sizes": "512,311,905,77,640,388,1001,262", "n": 2048, "k": 512, "act": "gelu",
         "keep": True},
        # a large one on sixteen
        {"name": "groups large", "kind": "groups", "rows": 16384, "n": 4096, "k": 2048, "act": "silu", "keep": False,
         "sizes": "1024,2049,333,1500,801,1190,64,1777,950,1024,700,1303,512,2000,157,1000"},
        # the way back through such a layer
        {"name": "groupsg train", "kind": "groupsg", "rows": 8192, "sizes": "1024,777,1540,300,1200,1333,1018,1000", "n": 4096, "k": 1024, "act": "gelu"},
        # ... of odd sizes, with groups without rows and rows without a group
        {"name": "groupsg ragged", "kind": "groupsg", "rows": 1000, "sizes": "131,0,77,200,1,64,0,45,150,33,9,120,101", "n": 1111, "k": 777, "act": "silu"},
        # the gradients of the 784-512-512-10 network: launches
        {"name": "clip mlp", "kind": "clip", "sizes": "401408,512,262144,512,5120,10", "max": 0.5},
        # a training step's end: all gradients of VGG-16
        {"name": "step vgg16", "kind": "step", "sizes": _text(_vgg16()), "max": 1.0},
        # the gradients of the wide residual network, 36.5 million values
        {"name": "clip wrn", "kind": "clip", "sizes": _text(_wrn()), "max": 1.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ones' ranges, at most as costly as the largest of them.  Rows of a handful of values are left out: what
    remains of their gradient is what its leading digits leave when they cancel."""
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= 2.7e11 and w["bytes"] <= 5.3e8:
            return case


def _draw(rng):
    kind = rng.choice(["join", "joing", "groups", "groups", "groupsg", "clip", "step"])
    if kind in ("join", "joing"):
        gates = rng.choice([0, 1, _log_int(rng, 1, 64)])
        rows = max(1, gates) * max(1, _log_int(rng, 1, 16384) // max(1, gates))
        if rng.random() < 0.1 and gates:
            gates = rows   # a gate for every value
        norms = rng.choice([("layer", "layer"), ("rms", "rms"), ("rms", "layer"), ("none", "layer"), ("none", "rms"), ("layer", "none")])
        return {"kind": kind, "rows": rows, "cols": _log_int(rng, 32, 8192), "gates": gates, "post": norms[0], "pre": norms[1],
                "scale": rng.choice([1.0, 1.0, round(rng.uniform(0.3, 2.0), 3)])}
    if kind in ("groups", "groupsg"):
        groups, used = _log_int(rng, 1, 64), _log_int(rng, 1, 16384)
        cuts = sorted(rng.randint(0, used) for _ in range(groups - 1))
        sizes = [b - a for a, b in zip([0] + cuts, cuts + [used])]
        case = {"kind": kind, "rows": used + rng.choice([0, 0, used // 8]), "sizes": _text(sizes), "n": _log_int(rng, 10, 4096),
                "k": _log_int(rng, 16, 4096), "act": rng.choice(["none", "relu", "gelu", "silu"])}
        if kind == "groups":
            case["keep"] = case["act"] != "none" and rng.random() < 0.5
        return case
    sizes = [_log_int(rng, 1, 4000000) for _ in range(rng.randint(1, 60))]
    return {"kind": kind, "sizes": _text(sizes), "max": round(math.exp(rng.uniform(-2.0, 2.0)), 4)}


def work(case):
    kind = case["kind"]
    if kind in ("join", "joing"):
        v, c = case["rows"] * case["cols"], case["cols"]
        norms = [n for n in (case["post"], case["pre"]) if n != "none"]
        params = c * sum(2 if n == "layer" else 1 for n in norms) + case["gates"] * c
        stats = case["rows"] * sum(2 if n == "layer" else 1 for n in norms)
        after = case["pre"] != "none"
        if kind == "join":
            return {"bytes": 4 * ((4 if after else 3) * v + params + stats), "flops": 16 * v}
        # dy, the branch, dx and its gradient; y and dh where there is a norm of y
        return {"bytes": 4 * ((6 if after else 4) * v + 2 * params + stats), "flops": 32 * v}
    if kind in ("groups", "groupsg"):
        sizes, m, n, k = _ints(case["sizes"]), case["rows"], case["n"], case["k"]
        used, live = sum(sizes), sum(s > 0 for s in sizes)
        if kind == "groups":
            return {"bytes": 4 * (used * k + live * (n * k + n) + m * n * (1 + case["keep"])), "flops": 2 * used * n * k}
        return {"bytes": 4 * (used * n * (1 if case["act"] == "none" else 2) + used * k + m * k + (live + len(sizes)) * n * k + len(sizes) * n),
                "flops": 4 * used * n * k}
    v = sum(_ints(case["sizes"]))
    return {"bytes": 4 * v * (2 if kind == "clip" else 7), "flops": v * (3 if kind == "clip" else 16)}


# ------------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda") * scale


def _offsets(case):
    at = [0]
    for s in _ints(case["sizes"]):
        at.append(at[-1] + s)
    return at


def _places(case):
    """Where the tensors of a set lie in its buffer, each from a multiple of 256 bytes on as an allocation does: (begin, next begin)."""
    at = [0]
    for s in _ints(case["sizes"]):
        at.append(at[-1] + (s + 63) // 64 * 64)
    return list(zip(at, at[1:]))


def _tensors(case, flat):
    return [flat[a:a + s] for (a, _), s in zip(_places(case), _ints(case["sizes"]))]


def _stats64(u, norm):
    """The mean (of a layer norm) and 1 / deviation of every row, as the forward pass leaves them."""
    u = u.double()
    if norm == "layer":
        return [u.mean(1).float(), (u.var(1, unbiased=False) + EPS).rsqrt().float()]
    return [(u.square().mean(1) + EPS).rsqrt().float()] if norm == "rms" else []


def _inputs(case, seed):
    """What the operator reads, made from the seed alone."""
    g, kind = _gen(seed), case["kind"]
    if kind in ("join", "joing"):
        m, c = case["rows"], case["cols"]
        # rows of a residual stream and of a branch, whose levels and spreads differ from row to row and column to column
        t = {"branch": _randn(g, m, c) * (0.3 + torch.rand((m, 1), generator=g, device="cuda")) + 0.2 * _randn(g, 1, c)}
        if case["gates"]:
            t["gate"] = _randn(g, case["gates"], c, scale=0.5)
        for norm in ("post", "pre"):
            if case[norm] != "none":
                t[norm + "_scale"] = 1.0 + 0.1 * _randn(g, c)
            if case[norm] == "layer":
                t[norm + "_bias"] = 0.1 * _randn(g, c)
        stream = 2.0 * _randn(g, m, c) + _randn(g, m, 1)
        if kind == "join":
            return dict(t, x=stream)
        t["dy"] = _randn(g, m, c, scale=0.01)
        if case["pre"] != "none":
            t["y"], t["dh"] = stream, _randn(g, m, c, scale=0.01)
        stats = _stats64(t["branch"], case["post"]) + (_stats64(t["y"], case["pre"]) if "y" in t else [])
        return dict(t, stats=torch.cat(stats))
    if kind in ("groups", "groupsg"):
        m, n, k = case["rows"], case["n"], case["k"]
        count = len(_ints(case["sizes"]))
        t = {"x": _randn(g, m, k), "w": _randn(g, count, n, k, scale=math.sqrt(2.0 / k))}
        t["offsets"] = torch.tensor(_offsets(case), dtype=torch.int32, device="cuda")
        if kind == "groups":
            t["bias"] = _randn(g, count, n, scale=0.1)
        else:
            t["dy"] = _randn(g, m, n, scale=0.01)
            if case["act"] != "none":
                t["pre"] = _randn(g, m, n, scale=1.4)
        return t
    # gradients of tensors whose sizes and magnitudes differ, one after the other in a buffer
    size = _places(case)[-1][1]
    t = {"g": torch.zeros(size, device="cuda")}
    for i, v in enumerate(_tensors(case, t["g"])):
        v.copy_(_randn(g, len(v), scale=10.0 ** (-3 + i % 3)))
    if kind == "step":
        live = torch.zeros_like(t["g"])   # no state of what lies between two tensors
        for v in _tensors(case, live):
            v.fill_(1.0)
        t.update(w=_randn(g, size, scale=0.05) * live, m=_randn(g, size, scale=1e-3) * live, v=_randn(g, size, scale=1e-3).square() * live)
    return t


def prepare(case, seed):
    state = {"case": case, "t": _inputs(case, seed)}
    if case["kind"] in ("groups", "groupsg"):
        state["at"] = _offsets(case)   # where groups begin, on the host as well: the plain form slices by it
    if case["kind"] in ("clip", "step"):
        state.update(set={k: _tensors(case, v) for k, v in state["t"].items()}, powers=[1.0, 1.0])
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


def _normed(u, norm):
    """(u normed, its rows' statistics)"""
    if norm == "none":
        return u, []
    mean = u.mean(1, keepdim=True) if norm == "layer" else None
    d = u - mean if norm == "layer" else u
    rstd = (d.square().mean(1, keepdim=True) + EPS).rsqrt()
    return d * rstd, ([mean.reshape(-1)] if norm == "layer" else []) + [rstd.reshape(-1)]


def _affine(z, t, norm):
    z = z * t[norm + "_scale"] if norm + "_scale" in t else z
    return z + t[norm + "_bias"] if norm + "_bias" in t else z


def _gated(case, t, v):
    """v times the gate of its row's sample."""
    if not case["gates"]:
        return v
    return (v.reshape(case["gates"], -1, case["cols"]) * t["gate"][:, None]).reshape(v.shape)


def _join(case, t):
    z, stats = _normed(t["branch"], case["post"])
    y = case["scale"] * t["x"] + _gated(case, t, _affine(z, t, "post"))
    out = {"y": y}
    if case["pre"] != "none":
        z, more = _normed(y, case["pre"])
        out["h"], stats = _affine(z, t, "pre"), stats + more
    return dict(out, stats=torch.cat(stats))


def _take_stats(case, t):
    """The norms' (mean, rstd) from the packed statistics, a mean of none where there is none."""
    parts, out = list(t["stats"].reshape(-1, case["rows"], 1)), {}
    for norm in ("post", "pre"):
        if case[norm] != "none":
            mean = parts.pop(0) if case[norm] == "layer" else None
            out[norm] = (mean, parts.pop(0))
    return out


def _standard(u, stats):
    mean, rstd = stats
    return (u if mean is None else u - mean) * rstd


def _norm_back(dz, z, rstd, norm):
    """The gradient of a norm's operand from that of its result z."""
    d = dz - z * (dz * z).mean(1, keepdim=True)
    return rstd * (d - dz.mean(1, keepdim=True) if norm == "layer" else d)


def _join_grad(case, t):
    out, stats, total = {}, _take_stats(case, t), t["dy"]
    if case["pre"] != "none":
        z = _standard(t["y"], stats["pre"])
        out["dpre_scale"] = (t["dh"] * z).sum(0)
        if case["pre"] == "layer":
            out["dpre_bias"] = t["dh"].sum(0)
        total = total + _norm_back(t["dh"] * t["pre_scale"], z, stats["pre"][1], case["pre"])
    out["dx"] = case["scale"] * total
    z = _standard(t["branch"], stats["post"]) if case["post"] != "none" else t["branch"]
    if case["gates"]:
        out["dgate"] = (total * _affine(z, t, "post")).reshape(case["gates"], -1, case["cols"]).sum(1)
    du = _gated(case, t, total)
    if case["post"] != "none":
        out["dpost_scale"] = (du * z).sum(0)
        if case["post"] == "layer":
            out["dpost_bias"] = du.sum(0)
        du = _norm_back(du * t["post_scale"], z, stats["post"][1], case["post"])
    return dict(out, dbranch=du)


def _spans(state):
    return [(i, slice(a, b)) for i, (a, b) in enumerate(zip(state["at"], state["at"][1:])) if b > a]


def _groups(state):
    case, t = state["case"], state["t"]
    pre = torch.zeros((case["rows"], case["n"]), device="cuda")
    for i, span in _spans(state):
        pre[span] = t["x"][span] @ t["w"][i].t() + t["bias"][i]
    out = {"y": _act(pre, case["act"])}
    return dict(out, pre=pre) if case["keep"] else out


def _groups_grad(state):
    case, t = state["case"], state["t"]
    dz = _act_grad(t["dy"], t["pre"], case["act"]) if case["act"] != "none" else t["dy"]
    dx, dw = torch.zeros_like(t["x"]), torch.zeros_like(t["w"])
    dbias = torch.zeros((len(state["at"]) - 1, case["n"]), device="cuda")
    for i, span in _spans(state):
        dx[span] = dz[span] @ t["w"][i]
        dw[i] = dz[span].t() @ t["x"][span]
        dbias[i] = dz[span].sum(0)
    return {"dx": dx, "dw": dw, "dbias": dbias}


def _gradient_norm(grads):
    return torch.stack([g.square().sum() for g in grads]).sum().sqrt()


def _factor(norm, most):
    return (most / norm).clamp_max(1.0)


def _clip(state):
    case, out = state["case"], torch.zeros_like(state["t"]["g"])
    norm = _gradient_norm(state["set"]["g"])
    factor = _factor(norm, case["max"])
    for g, to in zip(state["set"]["g"], _tensors(case, out)):
        torch.mul(g, factor, out=to)
    return {"norm": norm.reshape(1), "g": out}


def _step(state):
    t = state["set"]
    norm = _gradient_norm(t["g"])
    factor = _factor(norm, state["case"]["max"])
    b1, b2 = state["powers"] = [p * ADAM[k] for p, k in zip(state["powers"], ("beta1", "beta2"))]
    eta = ADAM["alpha"] * math.sqrt(1.0 - b2) / (1.0 - b1)
    for w, g, m, v in zip(t["w"], t["g"], t["m"], t["v"]):
        g = g * factor
        m.mul_(ADAM["beta1"]).add_(g * (1.0 - ADAM["beta1"]))
        v.mul_(ADAM["beta2"]).add_(g.square() * (1.0 - ADAM["beta2"]))
        w.sub_(m / (v.sqrt() + ADAM["eps"]) * eta)
    return dict({k: state["t"][k] for k in ("w", "m", "v")}, norm=norm.reshape(1))


# ------------------------------------------------------------------------------------------------ this package's entry points

def _ref(t):
    """A torch tensor as an operand of the entry points; it stays the tensor's memory."""
    from dopt_amd import ops
    kind = "int32" if t.dtype == torch.int32 else "float32"
    return ops.Tensor(tuple(t.shape), kind, _ptr=t.data_ptr(), _owner=t)


def _plan(state):
    """What a program keeps between calls: its operands as the entry points take them, result buffers, the optimizer's handles."""
    from dopt_amd import ops
    case, t = state["case"], state["t"]
    kind = case["kind"]
    if kind in ("clip", "step"):
        refs = {k: [_ref(x) for x in v] for k, v in state["set"].items()}
        result = torch.empty(2, device="cuda")   # the norm, and what the gradients are multiplied by
        state["result"] = _ref(result)
        state["outs"] = {"norm": result[:1]}
        if kind == "clip":
            state["outs"]["g"] = torch.zeros_like(t["g"])
            state["norm"] = ops.GradientNorm(refs["g"], [_ref(g) for g in _tensors(case, state["outs"]["g"])])
        else:
            state["outs"].update({k: t[k] for k in ("w", "m", "v")})
            state["norm"] = ops.GradientNorm(refs["g"])
            state["opt"] = ops.FusedOptimizer(refs["w"], refs["g"], refs["m"], refs["v"])
        return
    state["r"] = {k: _ref(v) for k, v in t.items()}
    if kind in ("groups", "groupsg"):
        m, n, k = case["rows"], case["n"], case["k"]
        shapes = {"dx": (m, k), "dw": tuple(t["w"].shape), "dbias": (len(t["w"]), n)}
        if kind == "groups":
            shapes = {"y": (m, n), "pre": (m, n)} if case["keep"] else {"y": (m, n)}
    else:
        m, c = case["rows"], case["cols"]
        shapes = {"y": (m, c), "stats": (sum({"layer": 2, "rms": 1, "none": 0}[case[p]] for p in ("post", "pre")) * m,)}
        if case["pre"] != "none":
            shapes["h"] = (m, c)
        if kind == "joing":
            shapes = {"d" + k: tuple(t[k].shape) for k in ("gate", "post_scale", "post_bias", "pre_scale", "pre_bias", "branch") if k in t}
            shapes["dx"] = (m, c)
    state["outs"] = {name: torch.empty(s, device="cuda") for name, s in shapes.items()}
    state["o"] = {name: _ref(v) for name, v in state["outs"].items()}


def _call(state):
    from dopt_amd import ops
    case, r, kind = state["case"], state.get("r"), state["case"]["kind"]
    if kind == "clip":
        state["norm"].clip(case["max"], out=state["result"])
    elif kind == "step":
        state["norm"].norm(case["max"], out=state["result"])
        state["opt"].adam(ADAM["alpha"], ADAM["beta1"], ADAM["beta2"], ADAM["eps"], factor=state["result"].view(1, (1,)))
    elif kind == "groups":
        o = state["o"]
        ops.dense_groups(r["x"], r["w"], r["offsets"], r["bias"], case["act"], out=o["y"], pre=o.get("pre"))
    elif kind == "groupsg":
        o = state["o"]
        ops.dense_groups_grad(r["dy"], r["x"], r["w"], r["offsets"], r.get("pre"), case["act"], dx=o["dx"], dw=o["dw"], dbias=o["dbias"])
    else:
        norms = {k: r.get(k) for k in ("gate", "post_scale", "post_bias", "pre_scale", "pre_bias")}
        norms.update(post=case["post"], pre=case["pre"], residual_scale=case["scale"])
        if kind == "join":
            ops.residual_norm(r["x"], r["branch"], eps=EPS, **norms, **state["o"])
        else:
            ops.residual_norm_grad(r["dy"], r.get("dh"), r.get("y"), r["branch"], r["stats"], out=state["o"], **norms)
    return state["outs"]


def run(state):
    if own:
        return _call(state)
    kind = state["case"]["kind"]
    if kind in ("join", "joing"):
        return {"join": _join, "joing": _join_grad}[kind](state["case"], state["t"])
    return {"groups": _groups, "groupsg": _groups_grad, "clip": _clip, "step": _step}[kind](state)


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits

def _phi(z):
    return torch.special.ndtr(z)


def _exact_act(z, act):
    return {"none": lambda: z, "relu": lambda: z * (z > 0), "gelu": lambda: z * _phi(z), "silu": lambda: z * torch.sigmoid(z)}[act]()


def _exact_slope(z, act):
    if act == "gelu":
        return _phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return s + z * s * torch.sigmoid(-z)
    return torch.ones_like(z) if act == "none" else (z > 0).double()


def _moments(u, norm):
    if norm == "rms":
        return torch.zeros_like(u[:, :1]), 1 / torch.sqrt((u * u).sum(1, keepdim=True) / u.shape[1] + EPS)
    return u.mean(1, keepdim=True), 1 / torch.sqrt(u.var(1, keepdim=True, unbiased=False) + EPS)


def _exact_join(case, t):
    rows, cols = case["rows"], case["cols"]
    zero, one = torch.zeros(cols, dtype=torch.double, device="cuda"), torch.ones(cols, dtype=torch.double, device="cuda")
    gate = t["gate"].repeat_interleave(rows // case["gates"], 0) if case["gates"] else one.expand(rows, cols)
    ps, pb, qs, qb = t.get("post_scale", one), t.get("post_bias", zero), t.get("pre_scale", one), t.get("pre_bias", zero)
    post, pre = case["post"], case["pre"]
    if case["kind"] == "join":
        u, stats = t["branch"], []
        if post != "none":
            mean, rstd = _moments(u, post)
            u, stats = (u - mean) * rstd * ps + pb, ([mean] if post == "layer" else []) + [rstd]
        out = {"y": t["x"] * case["scale"] + gate * u}
        if pre != "none":
            mean, rstd = _moments(out["y"], pre)
            out["h"] = (out["y"] - mean) * rstd * qs + qb
            stats = stats + ([mean] if pre == "layer" else []) + [rstd]
        return dict(out, stats=torch.cat(stats).reshape(-1))
    at = {"post": 0, "pre": 0 if post == "none" else 1 + (post == "layer")}
    s = t["stats"].reshape(-1, rows, 1)

    def standard(u, which):   # the normed rows, 1 / deviation, and whether their mean was taken out
        kind = case[which]
        if kind == "none":
            return u, torch.ones_like(u[:, :1]), 0.0
        mean = s[at[which]] if kind == "layer" else 0.0
        rstd = s[at[which] + (kind == "layer")]
        return (u - mean) * rstd, rstd, float(kind == "layer")

    def through(dz, z, rstd, centred):
        return rstd * (dz - centred * dz.sum(1, keepdim=True) / cols - z * ((dz * z).sum(1, keepdim=True) / cols))

    out, dy = {}, t["dy"]
    if pre != "none":
        z, rstd, centred = standard(t["y"], "pre")
        dy = dy + through(t["dh"] * qs, z, rstd, centred)
        out["dpre_scale"] = (t["dh"] * z).sum(0)
        if pre == "layer":
            out["dpre_bias"] = t["dh"].sum(0)
    out["dx"] = dy * case["scale"]
    z, rstd, centred = standard(t["branch"], "post")
    if case["gates"]:
        out["dgate"] = (dy * (z * ps + pb)).reshape(case["gates"], -1, cols).sum(1)
    du = dy * gate
    if post == "none":
        return dict(out, dbranch=du)
    out["dpost_scale"] = (du * z).sum(0)
    if post == "layer":
        out["dpost_bias"] = du.sum(0)
    return dict(out, dbranch=through(du * ps, z, rstd, centred))


def _exact_groups(case, t):
    sizes, m = _ints(case["sizes"]), case["rows"]
    pieces = lambda v: torch.split(v[:sum(sizes)], sizes)  # noqa: E731
    rest = lambda v: torch.cat([v, torch.zeros((m - len(v),) + v.shape[1:], dtype=v.dtype, device=v.device)])  # noqa: E731
    if case["kind"] == "groups":
        pre = rest(torch.cat([torch.addmm(b, x, w.t()) for x, w, b in zip(pieces(t["x"]), t["w"], t["bias"])]))
        out = {"y": _exact_act(pre, case["act"])}
        return dict(out, pre=pre) if case["keep"] else out
    dz = pieces(t["dy"] * _exact_slope(t["pre"], case["act"]) if "pre" in t else t["dy"])
    return {"dx": rest(torch.cat([torch.mm(d, w) for d, w in zip(dz, t["w"])])),
            "dw": torch.stack([torch.mm(d.t(), x) for d, x in zip(dz, pieces(t["x"]))]), "dbias": torch.stack([d.sum(0) for d in dz])}


def exact(case, seed):
    t = {k: v.double() for k, v in _inputs(case, seed).items()}
    kind = case["kind"]
    if kind in ("join", "joing"):
        return _exact_join(case, t)
    if kind in ("groups", "groupsg"):
        return _exact_groups(case, t)
    norm = math.sqrt(float(torch.dot(t["g"], t["g"])))
    x = t["g"] * min(1.0, case["max"] / norm)
    out = {"norm": torch.tensor([norm], dtype=torch.double, device="cuda")}
    if kind == "clip":
        return dict(out, g=x)
    b1, b2 = ADAM["beta1"], ADAM["beta2"]
    m, v = b1 * t["m"] + (1 - b1) * x, b2 * t["v"] + (1 - b2) * x * x
    w = t["w"] - ADAM["alpha"] * math.sqrt(1 - b2) / (1 - b1) * m / (v.sqrt() + ADAM["eps"])
    return dict(out, w=w, m=m, v=v)
