"""Optimizers, in two forms.

`sgd`, `adam`, `amsgrad` restate online/source/dopt/online/{sgd,adam,amsgrad}.d: the update
rule is built as a graph of pointwise operations (scalars broadcast through products with ones
vectors) and compiled into one plan whose outputs are written back over the variables.  This is
the reference's own formulation; it runs on the HIP backend kernel by kernel and serves as the
un-fused ground truth.

`fused_sgd`, `fused_adam`, `fused_amsgrad` are what a `dopt.hip` build substitutes: the plan
computes only the outputs and the gradients (plus projections that do not depend on the updated
value, i.e. batch-norm's running statistics), and ONE multi-tensor kernel applies the rule in
place with the same per-node fp32 rounding, so parameters and optimizer state match the un-fused
form bit for bit.  Projections of the updated value itself (operator-norm constraints) run as a
second small plan after the kernel.
"""
import numpy as np

from . import capi, core, ops
from .core import float32, grad, sqrt


def _newbufs(variables):
    return [v.device_ptr()[0] for v in variables]


def _check_norm(maxNorm):
    if maxNorm is not None and not maxNorm >= 0:
        raise ValueError("The largest norm is %r" % (maxNorm,))


def clipped(grads, maxNorm):
    """The gradients times min(1, maxNorm / norm), norm the square root of the sum of all their squares; as they are where maxNorm
    is None.  A gradient that stands for several parameters counts for each.  Of any size: the squares are those of the gradients over the
    largest magnitude, so that none overflows and what vanishes is too small to count.  NaN for a norm that is NaN, zero for an infinite one.  No counterpart in
    the reference."""
    _check_norm(maxNorm)
    low, high = float(np.finfo(np.float32).tiny), float(np.finfo(np.float32).max)
    most = np.inf if maxNorm is None or maxNorm > high else float(maxNorm)
    if np.isinf(most) or not grads:
        return list(grads)
    top = total = None
    for g in grads:
        t = core.maxElement(core.abs(g))   # (passes over NaN, which the squares keep)
        top = t if top is None else core.max(top, t)
    top = core.min(core.max(top, float32([], [low])), float32([], [high]))
    for g in grads:
        v = g / top
        s = core.sum(v * v)
        total = s if total is None else total + s
    # Norm and bound over the largest magnitude; the bound is cut where no norm comes near, so that the quotient is one within bounds and
    # its divisor never zero.
    norm, bound = sqrt(total), core.min(float32([], [most]) / top, float32([], [1e30]))
    factor = bound / core.max(norm, core.max(bound, float32([], [low])))
    return [g * factor for g in grads]


class _GraphUpdater:
    def __init__(self, outputs, plan_outputs, targets, flags):
        self.outputs = outputs
        self.plan = core.compile(plan_outputs, flags)
        self._targets = targets
        self._out_bufs = [ops.Tensor(o.shape, o.dtype) for o in outputs]
        self._rets = [t.ptr for t in self._out_bufs] + _newbufs(targets)

    def __call__(self, args=None):
        self.plan.execute(args, self._rets)
        return [t.numpy() for t in self._out_bufs]

    def step_async(self, args=None):
        """Enqueues one update without reading the outputs back."""
        self.plan.execute(args, self._rets)


def sgd(outputs, wrt, projs=None, learningRate=None, momentumRate=None, nesterov=False, flags=0, maxNorm=None):
    """online/sgd.d:28-94.  maxNorm (here and below; no counterpart there): the gradients are clipped to that norm of them all."""
    projs = projs or {}
    learningRate = learningRate if learningRate is not None else float32([], [0.01])
    momentumRate = momentumRate if momentumRate is not None else float32([], [0.0])
    grads = clipped(grad(outputs[0], wrt), maxNorm)
    momentum = [float32(g.shape) for g in grads]
    if nesterov:
        new_momentum = [m * momentumRate - learningRate * g for g, m in zip(grads, momentum)]
        newvals = [w + momentumRate * nm - learningRate * g for w, nm, g in zip(wrt, new_momentum, grads)]
    else:
        new_momentum = [m * momentumRate + learningRate * g for g, m in zip(grads, momentum)]
        newvals = [w - nm for w, nm in zip(wrt, new_momentum)]
    for i, w in enumerate(wrt):
        if w in projs:
            newvals[i] = projs[w](newvals[i])
    up = _GraphUpdater(outputs, list(outputs) + newvals + new_momentum, list(wrt) + momentum, flags)
    up.momentum = momentum
    return up


def _adam_graph(outputs, wrt, projs, alpha, beta1, beta2, eps, with_varhat, flags, maxNorm):
    projs = projs or {}
    alpha = alpha if alpha is not None else float32([], [0.001])
    beta1 = beta1 if beta1 is not None else float32([], [0.9])
    beta2 = beta2 if beta2 is not None else float32([], [0.999])
    eps = eps if eps is not None else float32([], [1e-8])
    grads = clipped(grad(outputs[0], wrt), maxNorm)
    means = [float32(w.shape) for w in wrt]
    vars_ = [float32(w.shape) for w in wrt]
    varhats = [float32(w.shape) for w in wrt] if with_varhat else []
    b1, b2 = float32([], [1.0]), float32([], [1.0])
    nb1, nb2 = b1 * beta1, b2 * beta2
    eta = alpha * sqrt(1.0 - nb2) / (1.0 - nb1)
    new_means = [beta1 * m + (1.0 - beta1) * g for g, m in zip(grads, means)]
    new_vars = [beta2 * v + (1.0 - beta2) * g * g for g, v in zip(grads, vars_)]
    new_varhats = [core.max(vh, v) for vh, v in zip(varhats, vars_)]
    newvals = [w - eta * (m / (sqrt(v) + eps)) for w, m, v in zip(wrt, new_means, new_vars)]
    for i, w in enumerate(wrt):
        if w in projs:
            newvals[i] = projs[w](newvals[i])
    up = _GraphUpdater(outputs, list(outputs) + newvals + new_means + new_vars + new_varhats + [nb1, nb2],
                       list(wrt) + means + vars_ + varhats + [b1, b2], flags)
    up.means, up.vars, up.varhats, up.b1, up.b2 = means, vars_, varhats, b1, b2
    return up


def adam(outputs, wrt, projs=None, alpha=None, beta1=None, beta2=None, eps=None, flags=0, maxNorm=None):
    """online/adam.d:32-93."""
    return _adam_graph(outputs, wrt, projs, alpha, beta1, beta2, eps, False, flags, maxNorm)


def amsgrad(outputs, wrt, projs=None, alpha=None, beta1=None, beta2=None, eps=None, flags=0, maxNorm=None):
    """online/amsgrad.d:32-99."""
    return _adam_graph(outputs, wrt, projs, alpha, beta1, beta2, eps, True, flags, maxNorm)


def _is_matrix(w):
    """Whether a weight is updated as the matrix of its first dimension against the others."""
    return w.rank >= 2 and w.shape[0] > 1 and w.volume > w.shape[0]


def _orthogonalised(u, iterations):
    rows, cols = u.shape[0], u.volume // u.shape[0]
    x = u.reshape([rows, cols])
    x = x / (sqrt(core.sum(x * x)) + 1e-7)
    if rows > cols:
        x = core.transpose(x, [1, 0])
    for _ in range(iterations):
        a = core.matmul(x, core.transpose(x, [1, 0]))
        x = 3.4445 * x + core.matmul(-4.7750 * a + 2.0315 * core.matmul(a, a), x)
    return (core.transpose(x, [1, 0]) if rows > cols else x).reshape(u.shape)


def _wide(w):
    return float(np.sqrt(np.maximum(1.0, w.shape[0] / (w.volume // w.shape[0]))))


def muon(outputs, wrt, projs=None, learningRate=0.02, momentumRate=0.95, nesterov=True, decay=0.0, restRate=0.01, iterations=5,
         flags=0, maxNorm=None):
    """Weight matrices move along their momentum's orthogonalised form (see dopt_hip_muon_step), all other parameters as `sgd` moves
    them with restRate and momentumRate.  No counterpart in the reference."""
    projs = projs or {}
    grads = clipped(grad(outputs[0], wrt), maxNorm)
    momentum = [float32(g.shape) for g in grads]
    newvals, new_momentum = [], []
    for w, g, m in zip(wrt, grads, momentum):
        if _is_matrix(w):
            nm = momentumRate * m + g
            o = _orthogonalised(g + momentumRate * nm if nesterov else nm, iterations)
            newvals.append((1.0 - learningRate * decay) * w - (learningRate * _wide(w)) * o)
        else:
            nm = m * momentumRate + restRate * g
            newvals.append(w - nm)
        new_momentum.append(nm)
    for i, w in enumerate(wrt):
        if w in projs:
            newvals[i] = projs[w](newvals[i])
    up = _GraphUpdater(outputs, list(outputs) + newvals + new_momentum, list(wrt) + momentum, flags)
    up.momentum = momentum
    return up


# ------------------------------------------------------------------------------- fused

class _Placeholder:
    pass


class _FusedUpdater:
    def __init__(self, rule, outputs, wrt, projs, hyper, flags, maxNorm=None):
        _check_norm(maxNorm)
        projs = projs or {}
        self.rule, self.hyper, self.outputs, self.wrt = rule, hyper, list(outputs), list(wrt)
        grads = grad(outputs[0], wrt)
        # Three kinds of projection (online/sgd.d:75-85 applies them to the updated value inside
        # the one plan):
        #  - it ignores the updated value (batch-norm replaces its running statistics by graph
        #    outputs, nnet/layers/batchnorm.d:140-154): computed by the step's plan, the kernel skips
        #    the parameter;
        #  - it depends on the updated value and otherwise on nothing the step reads (the
        #    operator-norm projections of nnet/lipschitz.d: constants, their own scalar variables,
        #    fresh random draws): a second plan, run after the fused kernel, reads the updated
        #    parameter and writes the projected one over it;
        #  - it also reads other variables (the max-gain projections read this batch's
        #    activations, computed from the OLD parameters): only the op-graph optimizers can
        #    reproduce that ordering.
        proj_ops, skip, post = [], [], []
        step_nodes = {id(o) for o in core.topological_sort(list(outputs))}   # what the step itself reads
        for w in wrt:
            skip.append(False)
            if w not in projs:
                continue
            probe = float32(w.shape)
            p = projs[w](probe)
            nodes = core.topological_sort([p])
            if not any(o is probe for o in nodes):
                proj_ops.append((w, p))
                skip[-1] = True
            elif all(o is probe or o.opType != "variable" or id(o) not in step_nodes for o in nodes):
                post.append((w, projs[w](w)))
            else:
                raise NotImplementedError("fused updaters cannot order a projection that reads both the updated "
                                          "value and other variables; use dopt_amd.online.%s for this model" % rule)
        self._post_plan = core.compile([p for _, p in post], flags) if post else None
        self._post_rets = [w.device_ptr()[0] for w, _ in post]
        self._proj = proj_ops
        self.plan = core.compile(list(outputs) + grads + [p for _, p in proj_ops], flags)
        self._out_bufs = [ops.Tensor(o.shape, o.dtype) for o in outputs]
        self._rets = [t.ptr for t in self._out_bufs] + [None] * len(grads) + [w.device_ptr()[0] for w, _ in proj_ops]

        def view(op_or_var, ptr):
            return ops.Tensor(op_or_var.shape, np.float32, _ptr=ptr, _owner=self)

        params = [view(w, w.device_ptr()[0]) for w in wrt]
        gviews = [view(g, self.plan.result_ptr(g)[0]) for g in grads]
        self.maxNorm, self._factor, self.norm = maxNorm, None, None
        if maxNorm is not None:
            self._gradientNorm = ops.GradientNorm(gviews)
            self.norm = ops.Tensor((2,))   # of the last step's gradients; what they were multiplied by
            self._factor = self.norm.view(1, (1,))
        self.state = {"m": [ops.Tensor(w.shape) for w in wrt]}
        if rule in ("adam", "amsgrad"):
            self.state["v"] = [ops.Tensor(w.shape) for w in wrt]
        if rule == "amsgrad":
            self.state["vhat"] = [ops.Tensor(w.shape) for w in wrt]
        rest = list(range(len(wrt)))
        self.muon = None
        if rule == "muon":   # matrices are updated by a set of launches of their own, the rest as sgd
            mats = [i for i in rest if _is_matrix(wrt[i]) and not skip[i]]
            rest = [i for i in rest if i not in set(mats)]
            self.muon = ops.MuonOptimizer(*[[v[i] for i in mats] for v in (params, gviews, self.state["m"])])

        def of(name):
            return [self.state[name][i] for i in rest] if name in self.state else None
        self.opt = ops.FusedOptimizer([params[i] for i in rest], [gviews[i] for i in rest], of("m"), of("v"), of("vhat"),
                                      [skip[i] for i in rest])

    def step_async(self, args=None):
        # The plan reads the OLD parameters; the fused kernel then updates them in place; projected
        # parameters were written by the plan's return copies (they are skipped by the kernel).
        self.plan.execute(args, self._rets)
        h, f = self.hyper, self._factor
        if f is not None:
            self._gradientNorm.norm(self.maxNorm, out=self.norm)
        if self.rule == "sgd":
            self.opt.sgd(h["lr"], h["mu"], h["nesterov"], f)
        elif self.rule == "adam":
            self.opt.adam(h["alpha"], h["beta1"], h["beta2"], h["eps"], f)
        elif self.rule == "muon":
            self.muon.step(h["lr"], h["mu"], h["nesterov"], h["decay"], h["iterations"], f)
            self.opt.sgd(h["rest"], h["mu"], False, f)
        else:
            self.opt.amsgrad(h["alpha"], h["beta1"], h["beta2"], h["eps"], f)
        if self._post_plan is not None:
            self._post_plan.execute(None, self._post_rets)

    def __call__(self, args=None):
        self.step_async(args)
        return [t.numpy() for t in self._out_bufs]


def fused_sgd(outputs, wrt, projs=None, learningRate=0.01, momentumRate=0.0, nesterov=False, flags=0, maxNorm=None):
    return _FusedUpdater("sgd", outputs, wrt, projs,
                         {"lr": float(learningRate), "mu": float(momentumRate), "nesterov": bool(nesterov)}, flags, maxNorm)


def fused_adam(outputs, wrt, projs=None, alpha=0.001, beta1=0.9, beta2=0.999, eps=1e-8, flags=0, maxNorm=None):
    return _FusedUpdater("adam", outputs, wrt, projs,
                         {"alpha": float(alpha), "beta1": float(beta1), "beta2": float(beta2), "eps": float(eps)},
                         flags, maxNorm)


def fused_amsgrad(outputs, wrt, projs=None, alpha=0.001, beta1=0.9, beta2=0.999, eps=1e-8, flags=0, maxNorm=None):
    return _FusedUpdater("amsgrad", outputs, wrt, projs,
                         {"alpha": float(alpha), "beta1": float(beta1), "beta2": float(beta2), "eps": float(eps)},
                         flags, maxNorm)


def fused_muon(outputs, wrt, projs=None, learningRate=0.02, momentumRate=0.95, nesterov=True, decay=0.0, restRate=0.01, iterations=5,
               flags=0, maxNorm=None):
    return _FusedUpdater("muon", outputs, wrt, projs,
                         {"lr": float(learningRate), "mu": float(momentumRate), "nesterov": bool(nesterov), "decay": float(decay),
                          "rest": float(restRate), "iterations": int(iterations)}, flags, maxNorm)
