"""Muon: momentum whose update is orthogonalised, for the weight matrices of the encoder stack; and ``orthogonalize``, the
operation itself (GPU: the kernels of libenc_hip.so; CPU tensors: an elementary PyTorch path, by device)."""
import torch

from . import layer_checks, layer_ext

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


@torch.no_grad()
def orthogonalize(update, steps=5, coefficients=COEFFICIENTS, eps=1e-7, dtype=None):
    """The nearly orthogonal matrix that `steps` Newton-Schulz steps X <- a X + (b A + c A A) X, A = X X^T, make of
    update / max(|update|, eps) (Frobenius norm).  update [..., rows, cols], a batch of matrices of any shape, fp32, bf16
    or fp16; the result has its shape and type, or `dtype`: of an fp32 update bf16 or fp16 too (what the type does not reach
    keeps its direction that way).  Not differentiable.  A zero update gives zeros."""
    a, b, c = coefficients
    if update.is_cuda:
        return layer_ext.bind().orthogonalize(update, steps, a, b, c, eps, dtype)
    layer_checks.orthogonalize(update, steps, dtype)
    x = update.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()        # squares of 32-bit values leave 32 bits
    x = (x / norm.clamp(min=eps)).float()
    with torch.autocast("cpu", enabled=False):
        for _ in range(steps):
            gram = x @ x.mT
            x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.mT if tall else x).to(dtype or update.dtype).contiguous()


class Muon(torch.optim.Optimizer):
    """For parameters of two dimensions (others: another optimiser).  v = momentum * v + g;  u = g + momentum * v (nesterov)
    or v;  w <- w (1 - lr * weight_decay) - lr * sqrt(max(1, rows / cols)) * orthogonalize(u).  Matrices of one shape,
    type and device are orthogonalised in one batch.  v and u are fp32 whatever the type of w (in 16 bits a gradient below
    2^-9 of v would leave it as it is, and u, up to 20 gradients, leaves fp16's range at either end); the orthogonal matrix
    has w's type."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS,
                 eps=1e-7):
        if lr < 0 or not 0 <= momentum < 1 or weight_decay < 0:
            raise ValueError("Muon: lr and weight_decay must not be negative, momentum must be in [0, 1)")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)          # (the constructor's groups come this way too)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2:
                del self.param_groups[-1]
                raise ValueError("Muon takes parameters of two dimensions, got one of shape %s" % (tuple(p.shape),))

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)           # casts to the parameters' types
        new = [p for group in self.param_groups for p in group["params"]]
        old = [i for group in state_dict["param_groups"] for i in group["params"]]
        for p, i in zip(new, old):
            v = state_dict["state"].get(i, {}).get("momentum_buffer")
            if v is not None:
                self.state[p]["momentum_buffer"] = v.to(p.device, torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            alike = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon does not take sparse gradients")
                state = self.state[p]
                if "momentum_buffer" not in state:
                    state["momentum_buffer"] = torch.zeros_like(p.grad, dtype=torch.float32)
                v = state["momentum_buffer"]
                v.mul_(group["momentum"]).add_(p.grad)
                u = p.grad.float().add(v, alpha=group["momentum"]) if group["nesterov"] else v
                alike.setdefault((p.shape, p.dtype, p.device), []).append((p, u))
            for (shape, dtype, _), members in alike.items():
                batch = orthogonalize(torch.stack([u for _, u in members]), group["steps"], group["coefficients"],
                                      group["eps"], dtype)
                factor = -group["lr"] * max(1.0, shape[0] / shape[1]) ** 0.5
                for (p, _), o in zip(members, batch):
                    if group["weight_decay"]:
                        p.mul_(1 - group["lr"] * group["weight_decay"])
                    p.add_(o, alpha=factor)
        return loss
