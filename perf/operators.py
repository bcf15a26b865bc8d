"""What is measured of the encoder layer's operators: the residual norm (norms before and after a block with its gate and
residual scale), the gated feed-forward block, and the orthogonalised update of the Muon optimiser -- each in its plain
form (elementary torch operations in 32 bits) and as the framework's own call."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)    # the quintic of the Newton-Schulz step
EPS = 1e-5


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of a served pre/post-norm block: latency
        norm("norm one token", "bf16", 1, 1, 2048, inner="rms", outer="rms", scale=True),
        # the encoder layer's norm1 / norm2 in a training step: 2 images of 1024^2 (21504 tokens each), 256 channels
        norm("norm encoder fp32 train", "fp32", 2, 21504, 256, outer="layer", affine="wb", train=True, residual=False),
        # a sandwich-normed block with a per-sample gate (conditioning) and a learned residual scale
        norm("norm sandwich bf16 train", "bf16", 4, 2048, 4096, inner="rms", outer="rms", gate="sample", scale=True,
             train=True),
        # odd sizes everywhere, a gate for each token
        norm("norm odd fp16 train", "fp16", 3, 331, 1027, inner="layer", outer="layer", affine="wb", gate="token",
             train=True),
        # one token through a served block: the weights' stream
        ffn("ffn one token", "bf16", 1, 2048, 5632, "silu"),
        # a small ragged batch of tokens, odd widths
        ffn("ffn 37 tokens odd", "fp16", 37, 1001, 2725, "gelu", bias=True),
        # the encoder layer's block, one image of 1024^2, training step in fp32
        ffn("ffn encoder fp32 train", "fp32", 21504, 256, 1024, "gelu", bias=True, train=True),
        # a wide block, training step
        ffn("ffn wide bf16 train", "bf16", 8192, 4096, 8192, "silu", train=True),
        # the 256 x 256 projections of six encoder layers, gradients in fp32
        muon("muon projections fp32", "fp32", 12, 256, 256),
        # the feed-forward weights of six encoder layers
        muon("muon ffn weights fp32", "fp32", 6, 1024, 256),
        # odd sizes, short and long side either way
        muon("muon odd fp32", "fp32", 3, 389, 515),
        # one wide weight, momentum kept in bf16
        muon("muon wide bf16", "bf16", 1, 2048, 5632),
    ]


def norm(name, dtype, batch, tokens, width, inner="none", outer="layer", affine="w", gate="none", scale=False,
         train=False, residual=True):
    c = {"op": "norm", "dtype": dtype, "batch": batch, "tokens": tokens, "width": width, "inner": inner, "outer": outer,
         "affine": affine, "gate": gate, "scale": scale, "train": train, "residual": residual}
    return dict(c, name=name) if name else c


def ffn(name, dtype, tokens, width, hidden, activation, bias=False, train=False):
    c = {"op": "ffn", "dtype": dtype, "tokens": tokens, "width": width, "hidden": hidden, "activation": activation,
         "bias": bias, "train": train}
    return dict(c, name=name) if name else c


def muon(name, dtype, batch, rows, cols):
    c = {"op": "muon", "dtype": dtype, "batch": batch, "rows": rows, "cols": cols, "steps": 5}
    return dict(c, name=name) if name else c


def _size(rng, lo, hi, step=32):
    """A size spread over the logarithm of [lo, hi]; every other one a multiple of `step`, the rest as they fall."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        n = max(step, n // step * step)
    return min(max(n, lo), hi)


def draw(rng):
    op, dtype = rng.choice(["norm", "ffn", "muon"]), rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "norm":
        batch, width = rng.randint(1, 8), _size(rng, 33, 8192)
        tokens = _size(rng, 1, max(2, min(21504, (1 << 25) // (batch * width))))
        return norm(None, dtype, batch, tokens, width, inner=rng.choice(["none", "layer", "rms"]),
                    outer=rng.choice(["layer", "rms", "none"]), affine=rng.choice(["w", "wb", "none"]),
                    gate=rng.choice(["none", "sample", "token"]), scale=rng.random() < 0.5, train=rng.random() < 0.6)
    if op == "ffn":
        width, hidden = _size(rng, 64, 4096), _size(rng, 96, 8192)
        cap = (8192 * 4096 * 8192 if dtype != "fp32" else 21504 * 256 * 8192) // (width * hidden)
        return ffn(None, dtype, _size(rng, 1, max(2, min(21504, cap))), width, hidden,
                   rng.choice(["silu", "gelu", "sigmoid", "relu"]), bias=rng.random() < 0.5, train=rng.random() < 0.5)
    rows, cols = _size(rng, 24, 2048), _size(rng, 24, 2048)
    return muon(None, dtype, max(1, min(rng.randint(1, 12), (1 << 33) // (rows * cols * min(rows, cols)))), rows, cols)


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def rand(*shape, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device=dev) * std + mean).to(dtype)

    s = {"case": dict(case)}
    if case["op"] == "norm":
        b, t, d = case["batch"], case["tokens"], case["width"]
        s["x"], s["y"] = rand(b, t, d, std=1.5, mean=0.1), rand(b, t, d, std=0.7)
        if case["gate"] != "none":
            s["gate"] = rand(b, 1 if case["gate"] == "sample" else t, d, std=0.5)
        if case["scale"]:
            s["scale"] = rand(d, std=0.05, mean=0.3)
        for which in ("inner", "outer"):
            if case[which] != "none" and "w" in case["affine"]:
                s[which + "_weight"] = rand(d, std=0.1, mean=1.0)
            if case[which] == "layer" and "b" in case["affine"]:
                s[which + "_bias"] = rand(d, std=0.1)
        if case["train"]:
            if case["outer"] != "none":
                s["grad_normed"] = rand(b, t, d)
            if case["residual"] or case["outer"] == "none":
                s["grad_residual"] = rand(b, t, d, std=0.5)
    elif case["op"] == "ffn":
        m, d, f = case["tokens"], case["width"], case["hidden"]
        s["x"] = rand(m, d)
        s["w_in"], s["w_out"] = rand(2 * f, d, std=d ** -0.5), rand(d, f, std=f ** -0.5)
        s["b_in"] = rand(2 * f, std=0.1) if case["bias"] else None
        s["b_out"] = rand(d, std=0.1) if case["bias"] else None
        if case["train"]:
            s["grad"] = rand(m, d)
    else:
        # gradients of a layer: a few strong directions over noise
        b, m, n = case["batch"], case["rows"], case["cols"]
        low = torch.randn((b, m, 8), generator=g, device=dev) @ torch.randn((b, 8, n), generator=g, device=dev)
        s["update"] = (1e-3 * (0.3 * low + torch.randn((b, m, n), generator=g, device=dev))).to(dtype)
    if case.get("train"):
        for k, v in s.items():
            if isinstance(v, torch.Tensor) and not k.startswith("grad"):
                v.requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return {"norm": _own_norm, "ffn": _own_ffn, "muon": _own_muon}[op](s)
    with torch.no_grad():
        return {"norm": _plain_norm, "ffn": _plain_ffn, "muon": _plain_muon}[op](s)


NORM_INPUTS = ("x", "y", "gate", "scale", "inner_weight", "inner_bias", "outer_weight", "outer_bias")
FFN_INPUTS = ("x", "w_in", "b_in", "w_out", "b_out")


def _own_norm(s):
    from instaorder_amd import residual_norm
    c = s["case"]
    options = {k: s[k] for k in NORM_INPUTS[2:] if k in s}
    residual, normed = residual_norm(s["x"], s["y"], inner=None if c["inner"] == "none" else c["inner"],
                                     outer=None if c["outer"] == "none" else c["outer"], eps=EPS,
                                     want_residual=c["residual"] or c["outer"] == "none", **options)
    out = {k: v for k, v in (("residual", residual), ("normed", normed)) if v is not None}
    if c["train"]:
        names = [k for k in NORM_INPUTS if k in s]
        grads = torch.autograd.grad(list(out.values()), [s[k] for k in names], [s["grad_" + k] for k in out])
        out = {k: v.detach() for k, v in out.items()}
        out.update(("d_" + k, v) for k, v in zip(names, grads))
    return out


def _own_ffn(s):
    from instaorder_amd import gated_feed_forward
    c = s["case"]
    y = gated_feed_forward(s["x"], s["w_in"], s["b_in"], s["w_out"], s["b_out"], activation=c["activation"])
    if not c["train"]:
        return {"y": y}
    names = [k for k in FFN_INPUTS if s[k] is not None]
    grads = torch.autograd.grad(y, [s[k] for k in names], s["grad"])
    return {"y": y.detach(), **{"d_" + k: v for k, v in zip(names, grads)}}


def _own_muon(s):
    from instaorder_amd import orthogonalize
    return {"update": orthogonalize(s["update"], steps=s["case"]["steps"])}


# ---- plain forms: elementary operations, 32 bits inside, one rounding at the end ----
def _normalise(v, kind):
    """(v-hat, 1 / deviation)"""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    rstd = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return v * rstd, rstd


def _normalise_backward(d_hat, hat, rstd, kind):
    d = d_hat - hat * (d_hat * hat).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - d_hat.mean(-1, keepdim=True)
    return d * rstd


def _plain_norm(s):
    c = s["case"]
    f = {k: v.float() for k, v in s.items() if isinstance(v, torch.Tensor)}
    z = f["y"]
    if c["inner"] != "none":
        y_hat, y_rstd = _normalise(z, c["inner"])
        z = y_hat * f["inner_weight"] if "inner_weight" in f else y_hat
        z = z + f["inner_bias"] if "inner_bias" in f else z
    factor = f.get("gate")
    if "scale" in f:
        factor = f["scale"] if factor is None else factor * f["scale"]
    r = f["x"] + (z if factor is None else factor * z)
    out = {"residual": r} if c["residual"] or c["outer"] == "none" else {}
    if c["outer"] != "none":
        r_hat, r_rstd = _normalise(r, c["outer"])
        n = r_hat * f["outer_weight"] if "outer_weight" in f else r_hat
        out["normed"] = n + f["outer_bias"] if "outer_bias" in f else n
    if c["train"]:
        d_r = f.get("grad_residual")
        if c["outer"] != "none":
            d_n = f["grad_normed"]
            if "outer_weight" in f:
                out["d_outer_weight"] = (d_n * r_hat).sum((0, 1))
            if "outer_bias" in f:
                out["d_outer_bias"] = d_n.sum((0, 1))
            d_hat = d_n * f["outer_weight"] if "outer_weight" in f else d_n
            through = _normalise_backward(d_hat, r_hat, r_rstd, c["outer"])
            d_r = through if d_r is None else d_r + through
        out["d_x"] = d_r
        d_z = d_r if factor is None else d_r * factor
        if "gate" in f:
            d_gate = d_r * z if "scale" not in f else d_r * z * f["scale"]
            out["d_gate"] = d_gate.sum(1, keepdim=True) if c["gate"] == "sample" else d_gate
        if "scale" in f:
            out["d_scale"] = (d_r * z if "gate" not in f else d_r * z * f["gate"]).sum((0, 1))
        if c["inner"] != "none":
            if "inner_weight" in f:
                out["d_inner_weight"] = (d_z * y_hat).sum((0, 1))
            if "inner_bias" in f:
                out["d_inner_bias"] = d_z.sum((0, 1))
            d_z = _normalise_backward(d_z * f["inner_weight"] if "inner_weight" in f else d_z, y_hat, y_rstd, c["inner"])
        out["d_y"] = d_z
    return {k: v.to(s["x"].dtype) for k, v in out.items()}


def _activate(b, kind):
    """act(b), act'(b)"""
    if kind == "relu":
        return b.clamp(min=0), (b > 0).to(b.dtype)
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(b * math.sqrt(0.5)))
        return b * cdf, cdf + b * torch.exp(-0.5 * b * b) / math.sqrt(2 * math.pi)
    sig = 1 / (1 + torch.exp(-b))
    return (sig, sig * (1 - sig)) if kind == "sigmoid" else (b * sig, sig * (1 + b * (1 - sig)))


def _plain_ffn(s):
    c = s["case"]
    f = {k: v.float() for k, v in s.items() if isinstance(v, torch.Tensor)}
    p = f["x"] @ f["w_in"].t()
    if c["bias"]:
        p = p + f["b_in"]
    a, b = p[:, :c["hidden"]], p[:, c["hidden"]:]
    act, slope = _activate(b, c["activation"])
    h = a * act
    y = h @ f["w_out"].t()
    out = {"y": y + f["b_out"] if c["bias"] else y}
    if c["train"]:
        g = f["grad"]
        d_h = g @ f["w_out"]
        d_p = torch.cat((d_h * act, d_h * a * slope), 1)
        out.update(d_x=d_p @ f["w_in"], d_w_in=d_p.t() @ f["x"], d_w_out=g.t() @ h)
        if c["bias"]:
            out.update(d_b_in=d_p.sum(0), d_b_out=g.sum(0))
    return {k: v.to(s["x"].dtype) for k, v in out.items()}


def _plain_muon(s):
    u = s["update"]
    x = u.float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    a, b, c = COEFFICIENTS
    x = x / (x * x).sum((1, 2), keepdim=True).sqrt().clamp(min=1e-7)
    for _ in range(s["case"]["steps"]):
        gram = torch.bmm(x, x.transpose(1, 2).contiguous())
        poly = b * gram + c * torch.bmm(gram, gram)
        x = a * x + torch.bmm(poly, x)
    if tall:
        x = x.transpose(1, 2)
    return {"update": x.to(u.dtype).contiguous()}


# ------------------------------------------------------------------------------------------------
# 64 bits, by the operators' definitions
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "muon":
        a, b, c = COEFFICIENTS
        outs = []
        for x in d["update"]:                       # left and right products agree: take the one on the short side
            x = x / max(float(torch.linalg.norm(x)), 1e-7)
            for _ in range(case["steps"]):
                if x.shape[0] <= x.shape[1]:
                    m = x @ x.T
                    x = a * x + (b * m + c * (m @ m)) @ x
                else:
                    m = x.T @ x
                    x = a * x + x @ (b * m + c * (m @ m))
            outs.append(x)
        return {"update": torch.stack(outs)}
    names = [k for k in (NORM_INPUTS if case["op"] == "norm" else FFN_INPUTS) if k in d]
    if case["train"]:
        for k in names:
            d[k].requires_grad_(True)
    nn = torch.nn.functional

    def normed(v, which):
        w, bias = d.get(which + "_weight"), d.get(which + "_bias")
        if case[which] == "layer":
            return nn.layer_norm(v, v.shape[-1:], w, bias, EPS)
        v = v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + EPS)
        return v if w is None else v * w

    if case["op"] == "norm":
        z = d["y"] if case["inner"] == "none" else normed(d["y"], "inner")
        r = d["x"] + z * d.get("gate", 1.0) * d.get("scale", 1.0)
        out = {"residual": r} if case["residual"] or case["outer"] == "none" else {}
        if case["outer"] != "none":
            out["normed"] = normed(r, "outer")
        grads = [d.get("grad_" + k) for k in out]
    else:
        p = nn.linear(d["x"], d["w_in"], d.get("b_in"))
        a, b = p.chunk(2, -1)
        act = {"silu": nn.silu, "gelu": nn.gelu, "relu": nn.relu, "sigmoid": torch.sigmoid}[case["activation"]]
        out = {"y": nn.linear(a * act(b), d["w_out"], d.get("b_out"))}
        grads = [d.get("grad")]
    if case["train"]:
        got = torch.autograd.grad(list(out.values()), [d[k] for k in names], grads)
        out = {k: v.detach() for k, v in out.items()}
        out.update(("d_" + k, v) for k, v in zip(names, got))
    return out


def work(case):
    es = DTYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        b, t, d = case["batch"], case["tokens"], case["width"]
        full, row = b * t * d, d
        gate = {"none": 0, "sample": b * d, "token": full}[case["gate"]]
        both = (1 if case["residual"] or case["outer"] == "none" else 0) + (case["outer"] != "none")
        params = row * (bool(case["scale"]) + sum((case[w] != "none") * ("w" in case["affine"]) +
                                                   (case[w] == "layer") * ("b" in case["affine"])
                                                   for w in ("inner", "outer")))
        values = (2 + both) * full + gate + params
        if case["train"]:                          # the gradients in, the gradients out
            values += (both + 2) * full + gate + params
        return {"bytes": es * values, "flops": (40 if case["train"] else 15) * full}
    if case["op"] == "ffn":
        m, d, f = case["tokens"], case["width"], case["hidden"]
        bias = (2 * f + d) if case["bias"] else 0
        values, flops = 2 * m * d + 3 * d * f + bias, 6 * m * d * f
        if case["train"]:
            values, flops = 2 * values, 3 * flops
        return {"bytes": es * values, "flops": flops}
    n, k = sorted((case["rows"], case["cols"]))
    # both squares are symmetric: half of each product is enough
    return {"bytes": 2 * es * case["batch"] * n * k,
            "flops": case["batch"] * case["steps"] * (n * n * k + n ** 3 + 2 * n * n * k)}
