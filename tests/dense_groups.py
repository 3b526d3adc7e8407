"""Dense layers of groups of rows in float64, one group after the other, with norm_dense_muon's bounds.

Products that are not small are formed from two fp16 parts of each value, scaled by its row: a value keeps 22 bits, or 2^-38 of its row's largest (a
scaled row's largest value so far is at least 2^13, and a low part is off by at most half of fp16's last place, 2^-25), and the product of two
low parts is left out.  Three errors of 2^-22 of |a| |b| are under 2^-20 of it, and of the largest ones' 2 2^-38: `parts`
adds those, which matter where a group has few rows (norm_dense_muon's bound shrinks with them)."""
import numpy as np

import norm_dense_muon as R


def bounds(offsets, rows):
    """The boundaries as a kernel sees them: within the rows, none below the one before."""
    return np.minimum(np.maximum.accumulate(np.maximum(np.asarray(offsets, np.int64), 0)), rows)


def _of_parts(a, b):
    """What two fp16 parts add to the bound of a b^T."""
    if not a.shape[1]:
        return 0.0
    a, b = np.abs(np.asarray(a, np.float64)), np.abs(np.asarray(b, np.float64))
    return 2.0 ** -20 * (a @ b.T) + 2.0 ** -37 * a.shape[1] * np.outer(a.max(1), b.max(1))


def forward(x, w, bias, offsets, name, parts=False):
    """((y, bound), (pre, bound))."""
    m, n = len(x), w.shape[1]
    out = [np.zeros((m, n)) for _ in range(4)]
    at = bounds(offsets, m)
    for g in range(len(w)):
        s = slice(at[g], at[g + 1])
        if at[g + 1] > at[g]:
            (y, ey), (pre, ep) = R.dense_act(x[s], w[g], None if bias is None else bias[g], None, name)
            more = _of_parts(x[s], w[g]) if parts else 0.0
            for o, v in zip(out, (y, ey + 1.13 * more, pre, ep + more)):   # (activations' slopes are at most 1.13)
                o[s] = v
    return (out[0], out[1]), (out[2], out[3])


def backward(dy, x, w, pre, offsets, name, parts=False):
    """((dx, bound), (dw, bound), (dbias, bound))."""
    out = [np.zeros(s) for s in (x.shape, x.shape, w.shape, w.shape, w.shape[:2], w.shape[:2])]
    at = bounds(offsets, len(x))
    for g in range(len(w)):
        s = slice(at[g], at[g + 1])
        if at[g + 1] > at[g]:
            (dx, ex), (dw, ew), (db, eb) = R.dense_act_grad(dy[s], x[s], w[g], None if pre is None else pre[s], name)
            if parts:
                dz = dy[s] if name == "none" else dy[s] * R.slope(np.asarray(pre[s], np.float64), name)
                ex, ew = ex + _of_parts(dz, w[g].T), ew + _of_parts(dz.T, x[s].T)
            out[0][s], out[1][s], out[2][g], out[3][g], out[4][g], out[5][g] = dx, ex, dw, ew, db, eb
    return (out[0], out[1]), (out[2], out[3]), (out[4], out[5])
