"""Muon: momentum whose update is orthogonalised, for the weight matrices of the segmentation networks; Adam for everything else.

For a matrix parameter W (a convolution weight is the matrix [out, in * kh * kw]) with gradient G:
    M <- momentum M + (1 - momentum) G          U = (1 - momentum) G + momentum M   (Nesterov)
    W <- (1 - lr wd) W - lr 0.2 sqrt(max(rows, cols)) orthogonalize(U)
The factor gives the update the root mean square of an Adam update (an orthogonal [m, n] matrix has 1 / sqrt(max(m, n))), so that one learning
rate and its schedule serve both kinds of parameters.  The orthogonalisation of all matrices is one call (`_lib.orthogonalize`,
csrc/orthogonalize.hip).  The reference trains with Adam only (scheduler.py:5-34); this is `run.py --optimizer muon`.
"""
import torch

from . import _lib


def _takes(p):
    """a matrix of a size that `_lib.orthogonalize` takes"""
    return p.dim() >= 2 and 0 < p.numel() <= 1 << 28 and max(p.shape[0], p.numel() // p.shape[0]) <= 1 << 16


def is_matrix(p):
    """Parameters the orthogonalised update is for: two or more axes, a filter over more than one input channel (depthwise filters are
    vectors per channel), at least 16 values along the shorter side (classifier rows and the like stay with Adam), and a size that
    `_lib.orthogonalize` takes."""
    return _takes(p) and p.shape[1] > 1 and min(p.shape[0], p.numel() // p.shape[0]) >= 16


class Muon(torch.optim.Optimizer):
    """`params`: parameters on one GPU, or groups of them as torch's optimisers take them.  Every group, one added later too, becomes a Muon and an
    Adam group, split by `is_matrix` (one learning rate, one decay); `matrices=True / False` in a group puts all of it on one side.  Parameters that
    require no gradient are left out.  `weight_decay` is decoupled for the matrices and added to the gradient for the others, as in Adam.
    Float32 parameters only."""

    def __init__(self, params, lr=1e-3, weight_decay=0.0, momentum=0.95, betas=(0.9, 0.999), eps=1e-8, steps=5):
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, betas=betas, eps=eps, steps=steps))

    def add_param_group(self, param_group):
        group = {**self.defaults, **param_group}
        lr, wd, momentum, betas, eps, steps = (group[k] for k in ("lr", "weight_decay", "momentum", "betas", "eps", "steps"))
        if (not lr >= 0.0 or not wd >= 0.0 or not 0.0 <= momentum < 1.0 or not all(0.0 <= b < 1.0 for b in betas) or not eps > 0.0 or
                not (1 <= steps <= 64 and int(steps) == steps)):
            raise ValueError("Muon: lr %r, weight_decay %r, momentum %r, betas %r, eps %r, steps %r" % (lr, wd, momentum, betas, eps, steps))
        params = [group["params"]] if torch.is_tensor(group["params"]) else list(group["params"])
        tensor = lambda p: p[1] if isinstance(p, tuple) else p                                  # noqa: E731  (name, parameter)
        if isinstance(group["params"], set) or not all(torch.is_tensor(tensor(p)) for p in params):
            raise TypeError("Muon: parameters must be tensors, in an order")
        params = [p for p in params if tensor(p).requires_grad]
        if not params:
            raise ValueError("Muon: no parameter of the group requires a gradient")
        device = next((p.device for g in self.param_groups for p in g["params"]), tensor(params[0]).device)
        for p in map(tensor, params):
            if not p.is_cuda or p.device != device:
                raise _lib.AadgError("Muon: parameters must be on one GPU (got %s, %s); there is no CPU path" % (p.device, device))
            if p.dtype != torch.float32:
                raise _lib.AadgError("Muon: float32 parameters only, got %s" % p.dtype)
            if group.get("matrices") and not _takes(p):
                raise ValueError("Muon: a parameter of shape %s has no orthogonalised update" % (tuple(p.shape),))
        known = {id(p) for g in self.param_groups for p in g["params"]}      # (what torch refuses, before half of the group is in)
        if any(id(p) in known or not (p.is_leaf or p.retains_grad) for p in map(tensor, params)):
            raise ValueError("Muon: a parameter is in another group already, or no leaf")
        side = lambda p: group["matrices"] if group.get("matrices") is not None else is_matrix(tensor(p))       # noqa: E731
        for matrices in (True, False):
            part = [p for p in params if bool(side(p)) == matrices]
            if part:
                super().add_param_group({**group, "params": part, "matrices": matrices})

    @torch.no_grad()
    def step(self, closure=None):
        if torch.cuda.is_current_stream_capturing():
            raise _lib.AadgError("Muon: step() cannot be captured into a graph (learning rate and step count are host values)")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if params:
                (self._matrices if group["matrices"] else self._others)(group, params, [p.grad for p in params])
        return loss

    def _matrices(self, group, params, grads):
        for p in params:
            if not self.state[p]:
                self.state[p]["momentum"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
        bufs, mu, lr = [self.state[p]["momentum"] for p in params], group["momentum"], group["lr"]
        torch._foreach_lerp_(bufs, grads, 1.0 - mu)
        updates = torch._foreach_lerp(grads, bufs, mu)
        flat = []
        for i in range(0, len(updates), 4096):                               # (matrices per call of the library)
            flat += _lib.orthogonalize([u.reshape(u.shape[0], -1) for u in updates[i:i + 4096]], steps=group["steps"])
        out = [o.view(p.shape) for o, p in zip(flat, params)]
        torch._foreach_mul_(out, [-0.2 * lr * max(o.shape) ** 0.5 for o in flat])
        if group["weight_decay"] != 0.0:
            torch._foreach_mul_(params, 1.0 - lr * group["weight_decay"])
        torch._foreach_add_(params, out)

    def _others(self, group, params, grads):
        (b1, b2), lr, eps = group["betas"], group["lr"], group["eps"]
        for p in params:
            if not self.state[p]:
                self.state[p].update(step=0, exp_avg=torch.zeros_like(p), exp_avg_sq=torch.zeros_like(p))
        steps = []
        for p in params:
            self.state[p]["step"] += 1
            steps.append(self.state[p]["step"])
        m, v = [self.state[p]["exp_avg"] for p in params], [self.state[p]["exp_avg_sq"] for p in params]
        if group["weight_decay"] != 0.0:
            grads = torch._foreach_add(grads, params, alpha=group["weight_decay"])
        torch._foreach_lerp_(m, grads, 1.0 - b1)
        torch._foreach_mul_(v, b2)
        torch._foreach_addcmul_(v, grads, grads, 1.0 - b2)
        denom = torch._foreach_sqrt(v)
        torch._foreach_div_(denom, [(1.0 - b2 ** s) ** 0.5 for s in steps])
        torch._foreach_add_(denom, eps)
        torch._foreach_addcdiv_(params, m, denom, [-lr / (1.0 - b1 ** s) for s in steps])
