"""Dense layers of groups of rows in float64, one group after the other, with norm_dense_muon's bounds."""
import numpy as np

import norm_dense_muon as R


def bounds(offsets, rows):
    """The boundaries as a kernel sees them: within the rows, none below the one before."""
    return np.minimum(np.maximum.accumulate(np.maximum(np.asarray(offsets, np.int64), 0)), rows)


def forward(x, w, bias, offsets, name):
    """((y, bound), (pre, bound))."""
    m, n = len(x), w.shape[1]
    out = [np.zeros((m, n)) for _ in range(4)]
    at = bounds(offsets, m)
    for g in range(len(w)):
        s = slice(at[g], at[g + 1])
        if at[g + 1] > at[g]:
            (y, ey), (pre, ep) = R.dense_act(x[s], w[g], None if bias is None else bias[g], None, name)
            for o, v in zip(out, (y, ey, pre, ep)):
                o[s] = v
    return (out[0], out[1]), (out[2], out[3])


def backward(dy, x, w, pre, offsets, name):
    """((dx, bound), (dw, bound), (dbias, bound))."""
    out = [np.zeros(s) for s in (x.shape, x.shape, w.shape, w.shape, w.shape[:2], w.shape[:2])]
    at = bounds(offsets, len(x))
    for g in range(len(w)):
        s = slice(at[g], at[g + 1])
        if at[g + 1] > at[g]:
            (dx, ex), (dw, ew), (db, eb) = R.dense_act_grad(dy[s], x[s], w[g], None if pre is None else pre[s], name)
            out[0][s], out[1][s], out[2][g], out[3][g], out[4][g], out[5][g] = dx, ex, dw, ew, db, eb
    return (out[0], out[1]), (out[2], out[3]), (out[4], out[5])
