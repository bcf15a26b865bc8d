"""Plain 64-bit forms of the layer operators (gated feed-forward block, residual norm, orthogonalised update) for the
tests, with bounds on what a kernel that sums in 32 bits and rounds as documented may be off by, value for value."""
import math

import torch

F64 = torch.float64
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a step of the type
U32 = 2.0 ** -24
# Below its smallest normal value a type's steps are all alike: fp16's are 2^-24 under 2^-14, so half a step is 2^-25 there,
# more than 2^-11 of the value.  (An exact 0.0008401 * 0.0581 = 4.88e-5 rounds to fp16 with up to 2^-25 = 2.98e-8, while
# 2^-11 of it are 2.38e-8.)  The same holds for a 16-bit value between two products.
FLOOR = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
LIPSCHITZ = 1.2             # of the activations: silu 1.10, gelu 1.13, sigmoid 0.25, relu 1
CURVATURE = 0.8             # of their derivatives: silu 0.5, gelu 0.8, sigmoid 0.1
TINY = 1e-30


def activate(b, kind):
    if kind == "relu":
        return b.clamp(min=0)
    if kind == "gelu":
        return 0.5 * b * (1 + torch.erf(b / math.sqrt(2.0)))
    s = 1 / (1 + torch.exp(-b))
    return s if kind == "sigmoid" else b * s


def slope(b, kind):
    if kind == "relu":
        return (b > 0).to(b.dtype)
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(b / math.sqrt(2.0))) + b * torch.exp(-b * b / 2) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-b))
    return s * (1 - s) if kind == "sigmoid" else s * (1 + b * (1 - s))


def _dot_error(k):
    """Relative to the sum of the products' magnitudes: k additions in 32 bits (a matrix instruction may cut instead of
    round: a whole step each), and three parts a factor for fp32 (what is left out is below a step of a product)."""
    return (k + 8) * 2 * U32


def ffn(x, w_in, b_in, w_out, b_out, kind, grad=None):
    """{name: (value, bound)} in 64 bits for inputs of one type."""
    u, floor = U[x.dtype], FLOOR.get(x.dtype, 0.0)
    u_mid = u if x.dtype != torch.float32 else 2 * U32        # h, da, db between two products
    x, w_in, w_out = x.to(F64), w_in.to(F64), w_out.to(F64)
    hidden = w_out.shape[1]
    bi = torch.zeros(2 * hidden, dtype=F64, device=x.device) if b_in is None else b_in.to(F64)
    bo = torch.zeros(w_out.shape[0], dtype=F64, device=x.device) if b_out is None else b_out.to(F64)
    p = x @ w_in.t() + bi
    dp = _dot_error(x.shape[1]) * (x.abs() @ w_in.abs().t() + bi.abs())
    a, b = p[:, :hidden], p[:, hidden:]
    da_, db_ = dp[:, :hidden], dp[:, hidden:]
    act, sl = activate(b, kind), slope(b, kind)
    e_act = LIPSCHITZ * db_ + 64 * U32 * (1 + b.abs()) * (act.abs() + sl.abs())        # exp / erf / rcp of 32 bits
    e_sl = CURVATURE * db_ + 64 * U32 * (1 + b.abs())
    if kind == "relu":                        # the kink: within the error of b either side is right
        e_sl = torch.where(b.abs() <= db_, torch.ones_like(b), torch.zeros_like(b))
    h = a * act
    e_h = da_ * act.abs() + a.abs() * e_act + da_ * e_act + (u_mid * h.abs()).clamp(min=floor)
    y = h @ w_out.t() + bo
    wa = w_out.abs()
    e_y = e_h @ wa.t() + _dot_error(hidden) * (h.abs() @ wa.t() + bo.abs()) + (u * y.abs()).clamp(min=floor)
    out = {"y": (y, e_y + TINY)}
    if grad is None:
        return out
    g = grad.to(F64)
    dh = g @ w_out
    e_dh = _dot_error(w_out.shape[0]) * (g.abs() @ wa)
    d_a, d_b = dh * act, dh * a * sl
    e_da = e_dh * act.abs() + dh.abs() * e_act + e_dh * e_act
    e_db = e_dh * (a * sl).abs() + dh.abs() * (da_ * sl.abs() + a.abs() * e_sl + da_ * e_sl) + e_dh * a.abs() * e_sl
    d_p, e_raw = torch.cat((d_a, d_b), 1), torch.cat((e_da, e_db), 1) + 8 * U32 * torch.cat((d_a, d_b), 1).abs()
    e_p = e_raw + (u_mid * d_p.abs()).clamp(min=floor)
    m = x.shape[0]
    d_x = d_p @ w_in
    out["d_x"] = (d_x, e_p @ w_in.abs() + _dot_error(2 * hidden) * (d_p.abs() @ w_in.abs()) + (u * d_x.abs()).clamp(min=floor) + TINY)
    d_wi = d_p.t() @ x
    out["d_w_in"] = (d_wi, e_p.t() @ x.abs() + _dot_error(m) * (d_p.abs().t() @ x.abs()) + (u * d_wi.abs()).clamp(min=floor) + TINY)
    d_bi = d_p.sum(0)
    out["d_b_in"] = (d_bi, e_raw.sum(0) + _dot_error(m) * d_p.abs().sum(0) + (u * d_bi.abs()).clamp(min=floor) + TINY)
    d_wo = g.t() @ h
    out["d_w_out"] = (d_wo, g.abs().t() @ e_h + _dot_error(m) * (g.abs().t() @ h.abs()) + (u * d_wo.abs()).clamp(min=floor) + TINY)
    d_bo = g.sum(0)
    out["d_b_out"] = (d_bo, _dot_error(m) * g.abs().sum(0) + (u * d_bo.abs()).clamp(min=floor) + TINY)
    return out


def residual_norm(t, inner, outer, eps, grads=None):
    """t: dict of x, y and what else the call has; grads: dict with d_residual / d_normed.  {name: value} in 64 bits, by
    autograd."""
    d = {k: v.detach().to(F64).requires_grad_(True) for k, v in t.items() if v is not None}

    def norm(v, kind, w, b):
        if kind == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
        v = v if w is None else v * w
        return v if b is None else v + b

    z = d["y"] if inner is None else norm(d["y"], inner, d.get("inner_weight"), d.get("inner_bias"))
    if "gate" in d:
        z = z * d["gate"]
    if "scale" in d:
        z = z * d["scale"]
    r = d["x"] + z
    out = {"residual": r}
    if outer is not None:
        out["normed"] = norm(r, outer, d.get("outer_weight"), d.get("outer_bias"))
    if grads:
        pairs = [(out[k], g.to(F64)) for k, g in grads.items() if g is not None]
        got = torch.autograd.grad([o for o, _ in pairs], list(d.values()), [g for _, g in pairs], allow_unused=True)
        out.update(("d_" + k, v if v is not None else torch.zeros_like(d[k])) for k, v in zip(d, got))
    return {k: v.detach() for k, v in out.items()}


def orthogonalize(u, steps, coefficients, eps):
    a, b, c = coefficients
    x = u.to(F64)
    x = x / torch.clamp(torch.sqrt((x * x).sum((-2, -1), keepdim=True)), min=eps)
    for _ in range(steps):
        if x.shape[-2] <= x.shape[-1]:
            m = x @ x.mT.contiguous()
            x = a * x + (b * m + c * (m @ m)) @ x
        else:
            m = x.mT.contiguous() @ x
            x = a * x + x @ (b * m + c * (m @ m))
    return x


def within(got, want, bound, what):
    """Every value of `got` within `bound` of `want`; the worst one is named."""
    ratio = ((got.to(F64) - want).abs() / bound)
    worst = float(ratio.max()) if ratio.numel() else 0.0
    assert worst <= 1.0, "%s: %.3g of its bound (at %s)" % (what, worst, int(ratio.argmax()))
