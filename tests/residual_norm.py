"""The residual norm and its gradient in float64, with bounds on how far a float32 computation may be from them.

As norm_dense_muon counts them: E is a rounding, a sum of n terms over a row is off by (n / 64 + 32) E times the sum of the terms' sizes,
since at least 64 lanes or a tree are on it.  A column's sum goes by runs of at most 128 rows, whose sums are added by sixteen lanes in pieces of 64: at most
128 + 128 additions follow each other."""
import numpy as np

from norm_dense_muon import E, chain, group_norm

NORMS = ("none", "layer", "rms")
NAMES = ("post_scale", "post_bias", "pre_scale", "pre_bias")


def norm(v, kind, eps):
    """((z, its bound), [(mean, bound)] or [], [(rstd, bound)]) of rows."""
    v = np.asarray(v, np.float64)
    n = v.shape[1]
    if kind == "layer":
        one, zero = np.ones(n), np.zeros(n)
        z, mean, rstd = group_norm(v, one, zero, 1, eps, "none", False)
        return z, [mean], [rstd]
    ms = (v * v).mean(1)
    e = (chain(n) + 8) * E * ms
    rstd = 1 / np.sqrt(ms + eps)
    e_rstd = rstd * (0.5 * e / (ms + eps) + 4 * E)
    z = v * rstd[:, None]
    return (z, np.abs(v) * e_rstd[:, None] + 4 * E * np.abs(z)), [], [(rstd, e_rstd)]


def per_row(gate, rows):
    return 1.0 if gate is None else np.repeat(np.asarray(gate, np.float64).reshape(-1, gate.shape[-1]), rows // (gate.size // gate.shape[-1]), 0)


def affine(z_and_bound, scale, bias):
    z, e = z_and_bound
    a = 1.0 if scale is None else np.asarray(scale, np.float64)
    b = 0.0 if bias is None else np.asarray(bias, np.float64)
    return z * a + b, e * np.abs(a) + 4 * E * (np.abs(z * a) + np.abs(b))


def forward(x, branch, gate, post, pre, v, scale, eps, y=None):
    """{y, h, stats}, each with its bound.  `v`: the norms' scales and biases by name, None where there is none.  `y`: what the device
    wrote, from which h and its statistics are formed."""
    rows = len(x if x is not None else branch)
    u, e_u, stats = 0.0, 0.0, []
    if branch is not None:
        u = np.asarray(branch, np.float64)
        if post != "none":
            z, means, rstds = norm(u, post, eps)
            u, e_u = affine(z, v["post_scale"], v["post_bias"])
            stats += means + rstds
    g = per_row(gate, rows)
    sx = 0.0 if x is None else scale * np.asarray(x, np.float64)
    want = sx + g * u
    out = {"y": (want, np.abs(g) * e_u + 4 * E * (np.abs(sx) + np.abs(g * u)))}
    if pre != "none":
        z, means, rstds = norm(want if y is None else y, pre, eps)
        out["h"] = affine(z, v["pre_scale"], v["pre_bias"])
        stats += means + rstds
    out["stats"] = tuple(np.concatenate([s[i] for s in stats]) if stats else np.zeros(0) for i in (0, 1))
    return out


def _back(dz, e_dz, z, e_z, rstd, kind):
    """rstd (dz - mean(dz) - z mean(dz z)), with its bound."""
    n = dz.shape[1]
    deep = chain(n) + 8
    m = lambda t: t.mean(1, keepdims=True)  # noqa: E731
    q, e_q = dz * z, e_dz * np.abs(z) + np.abs(dz) * e_z + 2 * E * np.abs(dz * z)
    s2, e_s2 = m(q), m(e_q + deep * E * np.abs(q))
    s1, e_s1 = (m(dz), m(e_dz + deep * E * np.abs(dz))) if kind == "layer" else (0.0, 0.0)
    e = e_dz + e_s1 + np.abs(z) * e_s2 + e_z * np.abs(s2) + 4 * E * (np.abs(dz) + np.abs(s1) + np.abs(z * s2))
    return rstd * (dz - s1 - z * s2), rstd * e


def backward(dy, dh, y, branch, gate, stats, post, pre, v, scale):
    """{dx, dbranch, dgate, dpost_scale, ..}, each with its bound; statistics as the device is given them."""
    rows = len(dy if dy is not None else dh)
    s = [np.asarray(r, np.float64).reshape(-1, 1) for r in np.asarray(stats).reshape(-1, rows)]
    take = {}
    for which, kind in (("post", post), ("pre", pre)):
        if kind != "none":
            take[which] = (s.pop(0) if kind == "layer" else 0.0, s.pop(0))
    f = lambda a: np.asarray(a, np.float64)  # noqa: E731
    t, e_t = (0.0, 0.0) if dy is None else (f(dy), 0.0)
    deep = min(rows, 128) + 128
    fold = lambda a, e: (a.sum(0), e.sum(0) + deep * E * np.abs(a).sum(0))  # noqa: E731
    out = {}
    if pre != "none":
        mean, rstd = take["pre"]
        z = (f(y) - mean) * rstd
        e_z = 4 * E * np.abs(z)
        out["dpre_scale"] = fold(f(dh) * z, np.abs(f(dh)) * e_z + 2 * E * np.abs(f(dh) * z))
        out["dpre_bias"] = fold(f(dh), 0 * f(dh))
        e = f(dh) * (1.0 if v["pre_scale"] is None else f(v["pre_scale"]))
        b, e_b = _back(e, 2 * E * np.abs(e), z, e_z, rstd, pre)
        t, e_t = t + b, e_b + 2 * E * (np.abs(t) + np.abs(b))
    out["dx"] = (scale * t, abs(scale) * e_t + 2 * E * np.abs(scale * t))
    if branch is None:
        return out
    z, e_z = f(branch), 0.0
    if post != "none":
        mean, rstd = take["post"]
        z = (z - mean) * rstd
        e_z = 4 * E * np.abs(z)
    g = per_row(gate, rows)
    if gate is not None:
        u, e_u = affine((z, e_z), v["post_scale"], v["post_bias"]) if post != "none" else (z, 0.0)
        q, e_q = t * u, e_t * np.abs(u) + np.abs(t) * e_u + 2 * E * np.abs(t * u)
        c = gate.shape[-1]
        q, e_q = (a.reshape(gate.size // c, -1, c) for a in (q, e_q))
        out["dgate"] = (q.sum(1).reshape(gate.shape), (e_q.sum(1) + deep * E * np.abs(q).sum(1)).reshape(gate.shape))
    du, e_du = t * g, e_t * np.abs(g) + 2 * E * np.abs(t * g)
    if post != "none":
        out["dpost_scale"] = fold(du * z, e_du * np.abs(z) + np.abs(du) * e_z + 2 * E * np.abs(du * z))
        out["dpost_bias"] = fold(du, e_du)
        a = 1.0 if v["post_scale"] is None else f(v["post_scale"])
        du, e_du = _back(du * a, e_du * np.abs(a) + 2 * E * np.abs(du * a), z, e_z, rstd, post)
    out["dbranch"] = (du, e_du)
    return out
