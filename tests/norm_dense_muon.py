"""Group norm, the dense layer with its activation, and the orthogonalised update in float64, with bounds on how far a float32
computation may be from them.

The bounds count roundings.  E = 2^-24 is what one rounding is off by, relative to its result.  A sum of n terms that is formed
by chains of at most d additions is off by d E times the sum of the terms' sizes; d is taken as n / 64 + 32, since the kernels have
at least 64 lanes on every sum and join those in trees.
"""
import numpy as np
from scipy.special import ndtr

E = 2.0 ** -24
ACTS = ("none", "relu", "gelu", "silu")


def act(z, name):
    if name == "relu":
        return np.where(z < 0, 0.0, z)
    if name == "gelu":
        return z * ndtr(z)
    if name == "silu":
        return z / (1 + np.exp(-z))
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).astype(np.float64)
    if name == "gelu":
        return ndtr(z) + z * np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    if name == "silu":
        s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    return np.ones_like(z)


def act_error(z, ez, name):
    """Of act(z) in float32 where z is off by ez: slopes are at most 1.13; a handful of roundings and a function good to a few units
    of its result, whose argument's rounding moves z Phi(z) and z sigmoid(z) by at most z^2 E of themselves, under E in all."""
    return 1.13 * ez + (16 * np.abs(act(z, name)) + 4) * E


def slope_error(z, ez, name):
    """Of dy act'(z) / dy: the slopes' own slopes are at most 0.8 (none for relu and none, away from relu's border)."""
    return (0.8 * ez if name in ("gelu", "silu") else 0.0) + 24 * E


def chain(n):
    return n / 64 + 32


def grouped(x, groups, last):
    """[N, groups, C / groups, inner] in float64."""
    n = x.shape[0]
    c = x.shape[-1] if last else x.shape[1]
    x = np.asarray(x, np.float64)
    x = np.moveaxis(x.reshape(n, -1, c), 2, 1) if last else x.reshape(n, c, -1)
    return x.reshape(n, groups, c // groups, -1)


def ungrouped(v, shape, last):
    n = shape[0]
    c = shape[-1] if last else shape[1]
    v = v.reshape(n, c, -1)
    return (np.moveaxis(v, 1, 2) if last else v).reshape(shape)


def group_norm(x, scale, bias, groups, eps, name, last):
    """((y, its bound), (mean, bound), (rstd, bound))."""
    v = grouped(x, groups, last)
    ch = lambda p: np.asarray(p, np.float64).reshape(1, groups, -1, 1)  # noqa: E731
    n = v.shape[2] * v.shape[3]
    size = np.abs(v).mean((2, 3), keepdims=True)
    mean, var = v.mean((2, 3), keepdims=True), v.var((2, 3), keepdims=True)
    e_mean = chain(n) * E * size
    # of the mean of (x - m')^2 where m' and each difference are off: the first order of m' - mean cancels in the sum
    spread = np.abs(v - mean).max((2, 3), keepdims=True)
    e_var = (chain(n) + 8) * E * var + 2 * E * np.abs(mean) * np.sqrt(var) + e_mean ** 2 + 4 * E * E * (spread + np.abs(mean)) ** 2
    rstd = 1 / np.sqrt(var + eps)
    e_rstd = rstd * (0.5 * e_var / (var + eps) + 4 * E)
    xhat = (v - mean) * rstd
    z = xhat * ch(scale) + ch(bias)
    e_xhat = rstd * (e_mean + E * np.abs(v - mean)) + np.abs(xhat) * (e_rstd / rstd + 4 * E)
    e_z = np.abs(ch(scale)) * e_xhat + 4 * E * (np.abs(xhat * ch(scale)) + np.abs(ch(bias)))
    return ((ungrouped(act(z, name), x.shape, last), ungrouped(act_error(z, e_z, name), x.shape, last)),
            (mean.ravel(), e_mean.ravel() + 2 * E * np.abs(mean.ravel())), (rstd.ravel(), e_rstd.ravel()))


def group_norm_grad(dy, x, scale, bias, mean, rstd, groups, name, last):
    """((dx, bound), (dscale, bound), (dbias, bound)); mean and rstd as the kernel is given them."""
    v, g = grouped(x, groups, last), grouped(dy, groups, last)
    ch = lambda p: np.asarray(p, np.float64).reshape(1, groups, -1, 1)  # noqa: E731
    st = lambda p: np.asarray(p, np.float64).reshape(v.shape[0], groups, 1, 1)  # noqa: E731
    mean, rstd, a = st(mean), st(rstd), ch(scale)
    n, inner = v.shape[2] * v.shape[3], v.shape[3]
    xhat = (v - mean) * rstd
    z = xhat * a + ch(bias)
    e_xhat = 4 * E * np.abs(xhat)
    e_z = np.abs(a) * e_xhat + 4 * E * (np.abs(xhat * a) + np.abs(ch(bias)))
    dz = g * slope(z, name)
    e_dz = np.abs(g) * slope_error(z, e_z, name)
    q, e_q = dz * xhat, e_dz * np.abs(xhat) + np.abs(dz) * e_xhat + 2 * E * np.abs(dz * xhat)
    rows = v.shape[0]
    fold = lambda t: t.sum((0, 3)).ravel()  # noqa: E731
    # a channel's sum: along the pixels, then over the samples
    deep = chain(inner) + chain(rows) + rows / 8
    db = (fold(dz), fold(e_dz) + deep * E * fold(np.abs(dz)))
    ds = (fold(q), fold(e_q) + deep * E * fold(np.abs(q)))
    m = lambda t: t.mean((2, 3), keepdims=True)  # noqa: E731
    s1, s2 = m(dz * a), m(q * a)
    deep = chain(n) + v.shape[2] + 8
    e_s1 = m((e_dz + deep * E * np.abs(dz)) * np.abs(a))
    e_s2 = m((e_q + deep * E * np.abs(q)) * np.abs(a))
    parts = dz * a - s1 - xhat * s2
    e = (e_dz + 2 * E * np.abs(dz)) * np.abs(a) + e_s1 + np.abs(xhat) * e_s2 + e_xhat * np.abs(s2)
    e += 4 * E * (np.abs(dz * a) + np.abs(s1) + np.abs(xhat * s2))
    return ((ungrouped(rstd * parts, x.shape, last), ungrouped(rstd * e, x.shape, last)), ds, db)


def product(a, b):
    """a b^T and a bound: K products whose partial sums, of mixed signs, stay within four times the root of their squares' sum; each of
    K additions rounds one of those, and no worse than that adds up."""
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return a @ b.T, 4 * E * np.sqrt(max(1, a.shape[1])) * np.sqrt((a * a) @ (b * b).T)


def dense_act(x, w, bias, residual, name):
    """((y, bound), (pre, bound))."""
    pre, e = product(x, w)
    if bias is not None:
        pre = pre + np.asarray(bias, np.float64)
        e = e + E * np.abs(pre)
    y, e_y = act(pre, name), act_error(pre, e, name) if name != "none" else e
    if residual is not None:
        y = y + np.asarray(residual, np.float64)
        e_y = e_y + E * np.abs(y)
    return (y, e_y + E * np.abs(y)), (pre, e + E * np.abs(pre))


def dense_act_grad(dy, x, w, pre, name):
    """((dx, bound), (dw, bound), (dbias, bound))."""
    dy, x, w = (np.asarray(t, np.float64) for t in (dy, x, w))
    dz = dy if name == "none" else dy * slope(np.asarray(pre, np.float64), name)
    e_dz = np.abs(dy) * (0.0 if name == "none" else 24 * E)
    dx, e_dx = product(dz, w.T)
    dw, e_dw = product(dz.T, x.T)
    return ((dx, e_dx + e_dz @ np.abs(w)), (dw, e_dw + e_dz.T @ np.abs(x)),
            (dz.sum(0), e_dz.sum(0) + (chain(len(dz)) + len(dz) / 8) * E * np.abs(dz).sum(0)))


def muon(w, g, m, lr, mu, nesterov, decay, iterations):
    """(w', m', the orthogonalised matrix with its scale) in float64."""
    w, g, m = (np.asarray(t, np.float64) for t in (w, g, m))
    m = mu * m + g
    u = g + mu * m if nesterov else m
    x = u.reshape(u.shape[0], -1)
    x = x / (np.sqrt((x * x).sum()) + 1e-7)
    rows, cols = x.shape
    x = x.T if rows > cols else x
    for _ in range(iterations):
        a = x @ x.T
        x = 3.4445 * x + (-4.7750 * a + 2.0315 * a @ a) @ x
    x = (x.T if rows > cols else x).reshape(w.shape) * np.sqrt(max(1.0, rows / cols))
    return (1 - lr * decay) * w - lr * x, m, x


def muon_bound(iterations):
    """How far the orthogonalised matrix may be off, in the 2-norm of all values relative to its own.  An iteration forms three products
    and two sums; a product's error is that of `product` in this norm, under 16 E of the factors' norms here, and |X|, |A| and |b A +
    c A A| are at most 1.3, 1.6 and 3 as operators: 100 E in all.  What came before grows at most fourfold, the largest slope of
    3.4445 s - 4.775 s^3 + 2.0315 s^5 on [0, 1.2]."""
    return 100 * E * sum(4.0 ** k for k in range(iterations)) + 8 * E * 4.0 ** iterations


def close(got, want_and_bound, what):
    want, bound = want_and_bound
    got = np.asarray(got, np.float64).reshape(np.shape(want))
    off = np.abs(got - want)
    bad = ~(off <= bound)
    if bad.any():
        i = np.unravel_index(np.nanargmax(np.where(bad, off / np.maximum(bound, 1e-300), 0)), off.shape)
        raise AssertionError("%s: %d of %d values off by more than their bound; at %s %r instead of %r, bound %.3g" % (
            what, bad.sum(), bad.size, i, got[i], want[i], np.broadcast_to(bound, off.shape)[i]))
