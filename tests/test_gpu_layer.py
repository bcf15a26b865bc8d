"""GPU tests of the layer operators (gated feed-forward block, residual norm, orthogonalised update) through the public
entry points, against the 64-bit forms of layer_reference.py.

Tolerances.  Feed-forward: value for value, the bounds that layer_reference.ffn derives.  Residual norm: a row's results
pass through at most 16 + 6 + 16 sequential additions a sum and a dozen operations, 64 steps of 32 bits of the row's own
magnitude (below, per output), and one rounding to the type.  Orthogonalised update: a step's error grows by at most
p'(0) = 3.4445 in each later one, 3.4445^5 = 485 in all; with three products a step of 2^-24 (fp32) or 2^-17 (two parts)
that is 1e-4, or 485 * 2^-17 and the rounding to the type, relative in the 2-norm."""
import pytest
import torch

import layer_reference as R

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.bfloat16, torch.float16]
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def rand(gen, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std + mean).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- gated feed-forward block -----------------------------------------------------------------
def ffn_inputs(dtype, m, d, f, o, bias, seed=1):
    g = gen(seed)
    return [rand(g, m, d, dtype=dtype), rand(g, 2 * f, d, dtype=dtype, std=d ** -0.5),
            rand(g, 2 * f, dtype=dtype, std=0.3) if bias else None, rand(g, o, f, dtype=dtype, std=f ** -0.5),
            rand(g, o, dtype=dtype, std=0.3) if bias else None]


def ffn_check(args, kind, grad=None, needs=None):
    from instaorder_amd import gated_feed_forward, layer_ext
    names = ("d_x", "d_w_in", "d_b_in", "d_w_out", "d_b_out")
    want = R.ffn(*[None if a is None else a.detach() for a in args], kind, grad)
    before = layer_ext.launch_count()
    if grad is None:
        y = gated_feed_forward(*args, activation=kind)
        R.within(y, *want["y"], "y")
    else:
        leaves = [None if a is None else a.detach().requires_grad_(needs is None or needs[i]) for i, a in enumerate(args)]
        y = gated_feed_forward(*leaves, activation=kind)
        R.within(y.detach(), *want["y"], "y")
        asked = [(n, t) for n, t in zip(names, leaves) if t is not None and t.requires_grad]
        got = torch.autograd.grad(y, [t for _, t in asked], grad)
        for (n, t), v in zip(asked, got):
            assert v.shape == t.shape and v.dtype == t.dtype
            R.within(v, *want[n], n)
    assert layer_ext.launch_count() > before


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m", [1, 15, 16, 17, 32, 33, 64, 65, 130, 257])
@pytest.mark.parametrize("d, f, o", [(64, 96, 64), (33, 17, 41), (8, 1, 3), (1, 8, 1), (256, 520, 136)])
def test_feed_forward_sizes(dtype, m, d, f, o):
    kind = ("silu", "gelu", "sigmoid", "relu")[(m + d) % 4]
    args = ffn_inputs(dtype, m, d, f, o, bias=(m + f) % 2 == 0, seed=m * d)
    ffn_check(args, kind)
    ffn_check(args, kind, rand(gen(7), m, o, dtype=dtype))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("kind", ["silu", "gelu", "sigmoid", "relu"])
@pytest.mark.parametrize("m", [3, 200])
def test_feed_forward_activations_far_out(dtype, kind, m):
    """Gates from -60 to 60: exp and erf at their ends."""
    args = ffn_inputs(dtype, m, 16, 24, 16, True)
    args[2] = torch.linspace(-60, 60, 48, device="cuda").to(dtype)
    ffn_check(args, kind, rand(gen(9), m, 16, dtype=dtype))


@pytest.mark.parametrize("dtype", FLOATS)
def test_feed_forward_big_tiles_and_slices(dtype):
    """Enough rows for the large tile, a long reduction in slices for the weights, many workgroups."""
    args = ffn_inputs(dtype, 4104, 264, 3080, 248, True)
    ffn_check(args, "silu", rand(gen(3), 4104, 248, dtype=dtype))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m, d, f, o", [(130, 72, 6000, 72), (700, 40, 3000, 40), (5, 1024, 4104, 520), (16, 2048, 2056, 2048),
                                        (40, 520, 8192, 264), (300, 2048, 512, 1024), (520, 264, 4096, 1032)])
def test_feed_forward_tiles_for_few_rows(dtype, m, d, f, o):
    """Each tile that the number of rows and widths may choose, and products in many slices of k."""
    args = ffn_inputs(dtype, m, d, f, o, True, seed=m)
    ffn_check(args, "silu")
    ffn_check(args, "gelu", rand(gen(4), m, o, dtype=dtype))


@pytest.mark.parametrize("m, d, f, o", [(33, 2052, 4104, 36), (64, 2052, 4104, 37), (65, 36, 72, 7), (300, 100, 1032, 516), (1030, 68, 200, 64)])
def test_feed_forward_fp32_in_place_and_not(m, d, f, o):
    """Short fp32 forward passes read the tensors where they lie; the same call with rows that do not allow it."""
    args = ffn_inputs(torch.float32, m, d, f, o, True, seed=m)
    ffn_check(args, "silu")
    ffn_check(args, "gelu", rand(gen(4), m, o))
    wide = rand(gen(8), m, d + 5)
    ffn_check([wide[:, 1:d + 1], *args[1:]], "silu")
    shifted = torch.empty(2 * f * d + 1, device="cuda")[1:].view(2 * f, d)
    ffn_check([args[0], shifted.copy_(args[1]), *args[2:]], "relu")
    bad = args[0].clone()
    bad[m // 2, d // 2] = float("nan")
    from instaorder_amd import gated_feed_forward
    y, clean = (gated_feed_forward(x, *args[1:]) for x in (bad, args[0]))
    rest = torch.arange(m, device="cuda") != m // 2
    assert torch.equal(y[rest], clean[rest]) and not y[m // 2].isfinite().any()


@pytest.mark.parametrize("needs", [(True, False, False, False, False), (False, True, False, False, False),
                                   (False, False, True, False, True), (False, False, False, True, False),
                                   (False, False, False, False, True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_feed_forward_only_the_gradients_that_are_asked_for(dtype, needs):
    ffn_check(ffn_inputs(dtype, 70, 40, 48, 24, True), "silu", rand(gen(5), 70, 24, dtype=dtype), needs)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m", [5, 100])
def test_feed_forward_strides_and_alignment(dtype, m):
    from instaorder_amd import gated_feed_forward
    g = gen(11)
    wide = rand(g, m, 80, dtype=dtype)
    args = ffn_inputs(dtype, m, 40, 24, 32, True)
    flat = rand(g, 1 + 48 * 40, dtype=dtype)
    for x in (wide[:, :40], wide[:, 3:43], wide[:, ::2], rand(g, 40, m, dtype=dtype).t(), rand(g, 1, 40, dtype=dtype).expand(m, 40)):
        ffn_check([x, *args[1:]], "silu", rand(g, m, 32, dtype=dtype))
    odd = [args[0], flat[1:].view(48, 40), args[2], args[3].t().contiguous().t(), args[4]]        # 2-byte aligned; transposed
    ffn_check(odd, "gelu", rand(g, 32, m, dtype=dtype).t())
    ffn_check(args, "gelu", rand(g, 1, 1, dtype=dtype).expand(m, 32))                              # a sum's gradient
    y = gated_feed_forward(args[0].view(1, m, 1, 40), *args[1:])
    assert y.shape == (1, m, 1, 32) and torch.equal(y.view(m, 32), gated_feed_forward(*args))


@pytest.mark.parametrize("dtype", FLOATS)
def test_feed_forward_no_tokens(dtype):
    from instaorder_amd import gated_feed_forward
    args = [None if a is None else a.requires_grad_(True) for a in ffn_inputs(dtype, 0, 16, 24, 8, True)]
    y = gated_feed_forward(*args)
    assert y.shape == (0, 8)
    grads = torch.autograd.grad(y.sum(), args)
    assert all(g.shape == a.shape and not g.count_nonzero() for g, a in zip(grads, args))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m", [9, 150])
def test_feed_forward_a_token_that_is_not_finite_stays_alone(dtype, m):
    from instaorder_amd import gated_feed_forward
    args = ffn_inputs(dtype, m, 48, 40, 33, True)
    clean = gated_feed_forward(*args)
    for bad in (float("nan"), float("inf"), float("-inf")):
        x = args[0].clone()
        x[m // 2, 5] = bad
        y = gated_feed_forward(x, *args[1:])
        rest = torch.arange(m, device="cuda") != m // 2
        assert torch.equal(y[rest], clean[rest]) and not torch.isfinite(y[m // 2]).all()
    x = args[0].clone().requires_grad_(True)
    grad = rand(gen(2), m, 33, dtype=dtype)
    dx, = torch.autograd.grad(gated_feed_forward(x, *args[1:]), x, grad)
    grad[m // 3, 0] = float("nan")
    dx2, = torch.autograd.grad(gated_feed_forward(x, *args[1:]), x, grad)
    rest = torch.arange(m, device="cuda") != m // 3
    assert torch.equal(dx[rest], dx2[rest]) and dx2[m // 3].isnan().all()


def test_feed_forward_large_fp32_values_do_not_overflow_in_parts():
    from instaorder_amd import gated_feed_forward
    x = torch.full((80, 8), 3.4e38, device="cuda")
    x[:, 1:] = 0
    wi = torch.zeros(32, 8, device="cuda")
    wi[:16, 0] = 1e-38                                # a = 3.4
    wi[16:, 0] = 1e-38
    y = gated_feed_forward(x, wi, None, torch.ones(4, 16, device="cuda"), None, "relu")
    # 1e-38 is below the smallest normal value: its parts end at bf16's smallest step, 2^-133, so each factor is off by up
    # to 2^-134 / 1e-38 = 4.6e-3 of itself, and y = a * b by twice that
    assert torch.allclose(y, torch.full_like(y, 16 * (3.4e38 * 1e-38) ** 2), rtol=2 * 2.0 ** -134 / 1e-38 + 1e-5)
    x.mul_(2.0 ** -20)                                # away from the ends all 24 bits are there
    wi.mul_(2.0 ** 20)
    y = gated_feed_forward(x, wi, None, torch.ones(4, 16, device="cuda"), None, "relu")
    a = float(x[0, 0]) * float(wi[0, 0])
    assert torch.allclose(y, torch.full_like(y, 16 * a * a), rtol=2 * 2.0 ** -134 / float(wi[0, 0]) + 1e-5)


def test_feed_forward_offsets_beyond_32_bits():
    """Hidden values past 2^32 elements, and past 4 GiB: the first, a middle and the last rows."""
    from instaorder_amd import gated_feed_forward
    m, d, f, o = 530000, 8, 8200, 8
    args = ffn_inputs(torch.bfloat16, m, d, f, o, False)
    leaves = [None if a is None else a.requires_grad_(True) for a in args]
    y = gated_feed_forward(*leaves)
    grad = rand(gen(4), m, o, dtype=torch.bfloat16)
    dx, = torch.autograd.grad(y, leaves[0], grad)
    for rows in (slice(0, 300), slice(262000, 262300), slice(m - 300, m)):
        want = R.ffn(args[0][rows].detach(), args[1].detach(), None, args[3].detach(), None, "silu", grad[rows])
        R.within(y[rows].detach(), *want["y"], "y")
        R.within(dx[rows], *want["d_x"], "d_x")


def test_feed_forward_repeats_exactly():
    from instaorder_amd import gated_feed_forward
    for dtype in FLOATS:
        args = [None if a is None else a.requires_grad_(True) for a in ffn_inputs(dtype, 600, 72, 264, 72, True)]
        grad = rand(gen(1), 600, 72, dtype=dtype)
        runs = [torch.autograd.grad(gated_feed_forward(*args), args, grad) for _ in range(3)]
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


# ---- residual norm ----------------------------------------------------------------------------
def norm_inputs(dtype, lead, d, inner, outer, gate, scale, affine, seed=1):
    g = gen(seed)
    t = {"x": rand(g, *lead, d, dtype=dtype, std=1.5, mean=0.5), "y": rand(g, *lead, d, dtype=dtype, mean=-0.3)}
    if gate == "token":
        t["gate"] = rand(g, *lead, d, dtype=dtype)
    elif gate == "sample":
        t["gate"] = rand(g, *lead[:-1], 1, d, dtype=dtype)
    elif gate == "all":
        t["gate"] = rand(g, *[1] * len(lead), d, dtype=dtype)
    if scale:
        t["scale"] = rand(g, d, dtype=dtype, std=0.2, mean=0.5)
    for which, kind in (("inner", inner), ("outer", outer)):
        if kind and "w" in affine:
            t[which + "_weight"] = rand(g, d, dtype=dtype, std=0.3, mean=1.0)
        if kind and "b" in affine:
            t[which + "_bias"] = rand(g, d, dtype=dtype)
    return t


def norm_check(t, inner, outer, want_residual=True, eps=1e-5, grads=("residual", "normed")):
    from instaorder_amd import layer_ext, residual_norm
    dtype = t["x"].dtype
    u = R.U[dtype]
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
    g = gen(99)
    given = {}
    for k in grads:
        if (k == "normed" and outer is None) or (k == "residual" and not (want_residual or outer is None)):
            continue
        given[k] = rand(g, *t["x"].shape, dtype=dtype)
    before = layer_ext.launch_count()
    residual, normed = residual_norm(**leaves, inner=inner, outer=outer, eps=eps, want_residual=want_residual)
    assert layer_ext.launch_count() > before or not t["x"].numel()
    out = {k: v for k, v in (("residual", residual), ("normed", normed)) if v is not None}
    assert set(out) == {k for k in ("residual", "normed") if (k == "residual" and want_residual) or (k == "normed" and outer)}
    want = R.residual_norm(t, inner, outer, eps, given)
    got = dict(out)
    if given:
        vs = torch.autograd.grad([out[k] for k in given], list(leaves.values()), list(given.values()), allow_unused=True)
        got.update(("d_" + k, v) for k, v in zip(leaves, vs))
    d = t["x"].shape[-1]
    for k, v in got.items():
        if k in want and v is not None:
            w = want[k]
            assert v.shape == w.shape and v.dtype == dtype, k
            # a row's own magnitude; column sums add as many rounded values as there are rows, in at most
            # rows / workers + 64 sequential steps
            across = w.dim() == 1 or v.shape != t["x"].shape
            if not w.numel():
                continue
            size = w.abs().max() if across else w.abs().amax(-1, keepdim=True)
            rows = max(t["x"].numel() // d, 1)
            steps = 64 + (rows ** 0.5 * 4 if across else 0)
            # inputs that cancel in the mean leave steps of their own size behind, by 1 / deviation
            spread = 16 if k not in ("residual",) else 2
            R.within(v.detach(), w, (u * w.abs()).clamp(min=R.FLOOR[dtype]) + steps * spread * R.U32 * (size + 1.0) + R.TINY, k)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("d", [1, 3, 8, 33, 64, 255, 256, 257, 512, 513, 1024, 1027, 2048, 2049, 4096, 4100, 8192, 8193, 16384])
def test_norm_widths(dtype, d):
    norm_check(norm_inputs(dtype, (2, 7), d, "layer", "layer", "sample", True, "wb", d), "layer", "layer")
    norm_check(norm_inputs(dtype, (2, 7), d, None, "rms", None, False, "w", d), None, "rms", want_residual=False)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("inner", [None, "layer", "rms"])
@pytest.mark.parametrize("outer", [None, "layer", "rms"])
@pytest.mark.parametrize("gate", [None, "sample", "token", "all"])
def test_norm_forms(dtype, inner, outer, gate):
    for affine, scale in (("wb", True), ("w", False), ("", True)):
        norm_check(norm_inputs(dtype, (3, 5), 96, inner, outer, gate, scale, affine), inner, outer)


@pytest.mark.parametrize("rows", [0, 1, 2, 3, 5, 63, 1000, 20001])
@pytest.mark.parametrize("d", [48, 1500])
def test_norm_rows(rows, d):
    norm_check(norm_inputs(torch.float32, (rows,), d, "rms", "layer", "token", True, "wb"), "rms", "layer")
    norm_check(norm_inputs(torch.bfloat16, (rows, 3), d, "layer", "rms", "sample", False, "w"), "layer", "rms")


@pytest.mark.parametrize("lead", [(1, 4000), (4000, 1), (700, 6), (6, 700), (70000, 2)])
def test_norm_shared_gates(lead):
    norm_check(norm_inputs(torch.float32, lead, 40, "rms", "rms", "sample", True, "w"), "rms", "rms")


def test_norm_gradient_of_a_gate_without_rows():
    from instaorder_amd import residual_norm
    x, gate = rand(gen(1), 3, 0, 64), rand(gen(2), 3, 1, 64).requires_grad_(True)
    junk = torch.full((3, 1, 64), 7.0, device="cuda")       # what the allocator hands out next
    del junk
    r, n = residual_norm(x, x, gate=gate, outer="rms")
    grad, = torch.autograd.grad(r.sum() + n.sum(), gate)
    assert torch.equal(grad, torch.zeros_like(gate))


@pytest.mark.parametrize("grads", [("residual",), ("normed",)])
def test_norm_one_gradient_only(grads):
    norm_check(norm_inputs(torch.float32, (4, 9), 72, "rms", "layer", "token", True, "wb"), "rms", "layer", grads=grads)


def test_norm_one_gradient_for_x_and_y():
    """Plain sum under the norm: x and y have the same gradient."""
    norm_check(norm_inputs(torch.float32, (40,), 256, None, "layer", None, False, "wb"), None, "layer", want_residual=False)
    from instaorder_amd import residual_norm
    x, y = rand(gen(1), 5, 64).requires_grad_(True), rand(gen(2), 5, 64).requires_grad_(True)
    n = residual_norm(x, y.detach(), outer="rms", want_residual=False)[1]
    dx, = torch.autograd.grad(n.sum(), x)
    n = residual_norm(x.detach(), y, outer="rms", want_residual=False)[1]
    dy, = torch.autograd.grad(n.sum(), y)
    assert torch.equal(dx, dy)
    residual_norm(x, y, outer="rms")[1].square().sum().backward()         # leaves' .grad do not share memory
    x.grad.zero_()
    assert y.grad.count_nonzero()


@pytest.mark.parametrize("dtype", FLOATS)
def test_norm_strides_and_alignment(dtype):
    g = gen(21)
    d = 100
    wide = rand(g, 6, 260, dtype=dtype)
    t = norm_inputs(dtype, (6,), d, "layer", "rms", "token", True, "wb")
    for x in (wide[:, :d], wide[:, 1:d + 1], wide[:, ::2][:, :d], rand(g, d, 6, dtype=dtype).t(), rand(g, 1, d, dtype=dtype).expand(6, d)):
        norm_check({**t, "x": x, "gate": x * 0.5, "y": x.flip(0)}, "layer", "rms")
    flat = rand(g, 1 + d, dtype=dtype)
    norm_check({**t, "scale": flat[1:], "outer_weight": flat[:d], "inner_bias": wide[0, ::2][:d]}, "layer", "rms")


def test_norm_constant_rows_and_rows_that_are_not_finite():
    from instaorder_amd import residual_norm
    x = torch.full((6, 40), 3.0, device="cuda")
    n = residual_norm(x, torch.zeros_like(x), outer="layer")[1]
    assert torch.equal(n, torch.zeros_like(n))                            # no deviation: eps decides
    n = residual_norm(torch.zeros_like(x), torch.zeros_like(x), inner="rms", outer="rms")[1]
    assert torch.equal(n, torch.zeros_like(n))
    y = rand(gen(1), 6, 40)
    clean = residual_norm(x, y, inner="layer", outer="rms")
    for bad in (float("nan"), float("inf")):
        y2 = y.clone()
        y2[2, 7] = bad
        r, n = residual_norm(x, y2, inner="layer", outer="rms")
        rest = torch.arange(6, device="cuda") != 2
        assert torch.equal(r[rest], clean[0][rest]) and torch.equal(n[rest], clean[1][rest]) and not n[2].isfinite().any()


def test_norm_offsets_beyond_32_bits():
    from instaorder_amd import residual_norm
    rows, d = 530000, 8192                            # 4.3e9 elements, 8.7 GB a tensor
    base = rand(gen(1), 1000, d, dtype=torch.bfloat16)
    x = base.repeat(rows // 1000, 1).requires_grad_(True)
    y = x.detach().flip(0).contiguous()
    r, n = residual_norm(x, y, outer="rms")
    dx, = torch.autograd.grad([r, n], x, [x.detach(), y])
    for at in (slice(0, 40), slice(262100, 262200), slice(rows - 40, rows)):
        a = x[at].detach().requires_grad_(True)
        r2, n2 = residual_norm(a, y[at], outer="rms")
        d2, = torch.autograd.grad([r2, n2], a, [a.detach(), y[at]])
        assert torch.equal(r[at], r2) and torch.equal(n[at], n2) and torch.equal(dx[at], d2)


def test_norm_more_rows_than_a_grid_has_threads_for():
    from instaorder_amd import residual_norm
    rows = (1 << 26) + 7                              # a wave each: 2^32 threads and some
    x = rand(gen(1), 1 << 20, 2, dtype=torch.bfloat16).repeat(65, 1)[:rows]
    r, n = residual_norm(x, x, outer="layer")
    first = residual_norm(x[:1 << 20], x[:1 << 20], outer="layer")
    for i in range(0, rows, 1 << 20):
        end = min(i + (1 << 20), rows)
        assert torch.equal(r[i:end], first[0][:end - i]) and torch.equal(n[i:end], first[1][:end - i])


# ---- orthogonalised update --------------------------------------------------------------------
MUON = {torch.float32: 1e-4, torch.bfloat16: 2.0 ** -8 + 485 * 2.0 ** -17, torch.float16: 2.0 ** -11 + 485 * 2.0 ** -17}


def muon_check(u, steps=5):
    from instaorder_amd import orthogonalize
    o = orthogonalize(u, steps=steps)
    assert o.shape == u.shape and o.dtype == u.dtype and o.is_contiguous()
    want = R.orthogonalize(u, steps, COEFFICIENTS, 1e-7)
    flat, ref = o.double().flatten(-2), want.flatten(-2)
    off = (flat - ref).norm(dim=-1) / ref.norm(dim=-1).clamp(min=1e-20)
    assert float(off.max()) <= MUON[u.dtype], float(off.max())


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 9), (9, 1), (8, 8), (7, 33), (33, 7), (64, 64), (65, 64), (64, 130), (130, 65),
                                        (256, 96), (97, 255), (300, 300), (513, 40), (40, 1031)])
def test_orthogonalize_sizes(dtype, rows, cols):
    muon_check(rand(gen(rows * cols), 3, rows, cols, dtype=dtype))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(1, 700, 1500), (1500, 600), (2, 1024, 1024), (20, 136, 200), (3, 260, 1000), (3, 1000, 260)])
def test_orthogonalize_large_tiles_and_slices(dtype, shape):
    g = gen(5)
    low = rand(g, *shape[:-1], 4) @ rand(g, *shape[:-2], 4, shape[-1])
    muon_check((low + rand(g, *shape)).to(dtype))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(8, 1000, 1000), (8, 1001, 997), (1300, 1700), (1700, 1300), (2049, 2300)])
def test_orthogonalize_tiles(dtype, shape):
    """Each tile of the symmetric products and of the updates, whole and in slices, with odd edges."""
    g = gen(6)
    low = rand(g, *shape[:-1], 4) @ rand(g, *shape[:-2], 4, shape[-1])
    muon_check((low + rand(g, *shape)).to(dtype))


def test_orthogonalize_steps_batches_scales_and_strides():
    from instaorder_amd import orthogonalize
    u = rand(gen(1), 2, 3, 24, 40)
    for steps in (1, 2, 3, 7):
        muon_check(u, steps)
    one = torch.stack([orthogonalize(m) for m in u.flatten(0, 1)]).view_as(u)
    assert torch.equal(one, orthogonalize(u))                              # a batch is its matrices
    for factor in (2.0 ** -60, 2.0 ** 60):                                 # squares leave the range of 32 bits
        assert torch.allclose(orthogonalize(u * factor, eps=1e-30), orthogonalize(u), rtol=1e-5, atol=1e-6)
    muon_check(u.transpose(-1, -2))
    muon_check(rand(gen(2), 24, 80)[:, ::2])
    assert orthogonalize(u[:0]).shape == (0, 3, 24, 40)
    z = u.clone()
    z[0, 1] = 0
    o = orthogonalize(z)
    assert not o[0, 1].count_nonzero() and torch.equal(o[1], orthogonalize(u)[1])
    z[0, 1, 3, 3] = float("nan")
    o = orthogonalize(z)
    assert o[0, 1].isnan().all() and torch.equal(o[1], orthogonalize(u)[1])


def test_muon_on_the_gpu_follows_the_cpu():
    from instaorder_amd import Muon
    g = torch.Generator().manual_seed(3)
    start = [torch.randn(s, generator=g) for s in ((40, 24), (40, 24), (24, 96))]
    grads = [[torch.randn(w.shape, generator=g) for w in start] for _ in range(3)]
    ends = []
    for device in ("cpu", "cuda"):
        ps = [torch.nn.Parameter(w.to(device, copy=True)) for w in start]
        opt = Muon(ps, lr=0.05, weight_decay=0.1)
        for step in grads:
            for p, gr in zip(ps, step):
                p.grad = gr.to(device)
            opt.step()
        ends.append([p.detach().cpu() for p in ps])
    for a, b in zip(*ends):
        assert torch.allclose(a, b, atol=3 * 0.05 * 2 * 1e-4 * 10)         # three steps of lr * sqrt(4) * 1e-4 of values to 10


# ---- together, on streams, in graphs ----------------------------------------------------------
def block(t, kind="silu"):
    """A pre-norm feed-forward block with a gate and a residual scale, as a model strings the operators together."""
    from instaorder_amd import gated_feed_forward, residual_norm
    _, n = residual_norm(t["x"], t["attn"], outer="layer", outer_weight=t["w1"], outer_bias=t["b1"])
    h = gated_feed_forward(n, t["w_in"], t["b_in"], t["w_out"], t["b_out"], activation=kind)
    return residual_norm(n, h, gate=t["gate"], scale=t["scale"], inner="rms", inner_weight=t["w2"], outer="rms",
                         outer_weight=t["w3"])


def block_inputs(dtype, batch, tokens, d, f, seed=1):
    g = gen(seed)
    r = lambda *s, std=1.0, mean=0.0: rand(g, *s, dtype=dtype, std=std, mean=mean)      # noqa: E731
    return {"x": r(batch, tokens, d), "attn": r(batch, tokens, d), "w1": r(d, mean=1.0, std=0.1), "b1": r(d, std=0.1),
            "w_in": r(2 * f, d, std=d ** -0.5), "b_in": r(2 * f, std=0.1), "w_out": r(d, f, std=f ** -0.5),
            "b_out": r(d, std=0.1), "gate": r(batch, 1, d), "scale": r(d, std=0.1, mean=0.3), "w2": r(d, mean=1.0, std=0.1),
            "w3": r(d, mean=1.0, std=0.1)}


def plain_block(t):
    def layer(v, w=None, b=None):
        v = v - v.mean(-1, keepdim=True)
        return v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-5) * w + b

    def rms(v, w):
        return v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-5) * w

    n = layer(t["x"] + t["attn"], t["w1"], t["b1"])
    a, b = (n @ t["w_in"].t() + t["b_in"]).chunk(2, -1)
    h = a * R.activate(b, "silu") @ t["w_out"].t() + t["b_out"]
    r = n + t["gate"] * t["scale"] * rms(h, t["w2"])
    return r, rms(r, t["w3"])


@pytest.mark.parametrize("dtype, tol", [(torch.float32, 2e-5), (torch.bfloat16, 6 * 2.0 ** -8), (torch.float16, 6 * 2.0 ** -11)])
@pytest.mark.parametrize("batch, tokens", [(1, 1), (2, 37), (3, 200)])
def test_a_block_of_the_operators_together(dtype, tol, batch, tokens):
    """Values and all gradients of the run, relative in the 2-norm: six roundings of 16 bits lie on its longest way."""
    t = {k: v.requires_grad_(True) for k, v in block_inputs(dtype, batch, tokens, 72, 104).items()}
    out = block(t)
    grads = [rand(gen(8), batch, tokens, 72, dtype=dtype) for _ in out]
    got = [*[o.detach() for o in out], *torch.autograd.grad(out, list(t.values()), grads)]
    d = {k: v.detach().double().requires_grad_(True) for k, v in t.items()}
    ref = plain_block(d)
    want = [*[o.detach() for o in ref], *torch.autograd.grad(ref, list(d.values()), [g.double() for g in grads])]
    for name, a, b in zip(["r", "n", *t], got, want):
        assert float((a.double() - b).norm()) <= tol * float(b.norm()) + 1e-6, name


def test_side_stream_and_interleaved_calls():
    t = block_inputs(torch.bfloat16, 2, 90, 64, 96)
    u = block_inputs(torch.bfloat16, 2, 70, 64, 96, seed=2)
    with torch.no_grad():
        want = [block(t), block(u)]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = [None, None]
        for _ in range(5):
            for i, (s, v) in enumerate(zip(streams, (t, u))):
                with torch.cuda.stream(s):
                    got[i] = block(v)
        torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_two_threads_call_at_once():
    """Forward and backward of two blocks from two threads, each on a stream of its own; an error in one is its own."""
    import threading
    from instaorder_amd import gated_feed_forward
    cases = [block_inputs(torch.bfloat16, 2, 75, 64, 96, seed=s) for s in (1, 2)]

    def work(t):
        leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
        r, n = block(leaves)
        return [r.detach(), n.detach(), *torch.autograd.grad(r.float().sum() + n.float().sum(), list(leaves.values()))]

    want = [work(t) for t in cases]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                try:
                    gated_feed_forward(cases[i]["x"], cases[i]["w_in"][:, 1:], None, cases[i]["w_out"], None)
                except RuntimeError as e:
                    failed.append(str(e))
                got[i] = work(cases[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(failed) == 40 and all("w_in has shape" in f for f in failed)
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.parametrize("tokens", [1, 90])
def test_captured_inference_replays_with_new_inputs(tokens):
    """Two graphs over the same operators, replayed in turn with eager calls between: no workspace is shared."""
    sets = [block_inputs(torch.bfloat16, 1, tokens, 64, 96, seed=s) for s in (1, 2)]
    graphs, outs = [], []
    with torch.no_grad():
        for t in sets:
            block(t)
        torch.cuda.synchronize()
        for t in sets:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(block(t))
            graphs.append(graph)
        for turn in range(4):
            for i in (0, 1, 0):
                new = block_inputs(torch.bfloat16, 1, tokens, 64, 96, seed=10 + turn + i)
                for k, v in sets[i].items():
                    v.copy_(new[k])
                graphs[i].replay()
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(outs[i], block(new)))


def test_captured_training_step_and_update_replay():
    from instaorder_amd import orthogonalize
    t = {k: v.requires_grad_(True) for k, v in block_inputs(torch.float32, 2, 80, 64, 96).items()}
    grads = [rand(gen(5), 2, 80, 64) for _ in range(2)]
    names = list(t)

    def step():
        got = torch.autograd.grad(block(t), [t[n] for n in names], grads)
        return got, orthogonalize(got[names.index("w_in")])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for turn in range(4):
        with torch.no_grad():
            for k, v in block_inputs(torch.float32, 2, 80, 64, 96, seed=20 + turn).items():
                t[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(captured[0], eager[0])) and torch.equal(captured[1], eager[1])


# ---- the encoder layer and the harness that call them -------------------------------------------
@pytest.mark.parametrize("activation", ["relu", "swiglu", "glu"])
def test_encoder_layer_with_the_operators_agrees_with_its_plain_path(activation):
    from instaorder_amd import layer_ext
    from instaorder_amd.encoder import MSDeformAttnTransformerEncoderLayer
    torch.manual_seed(0)
    layer = MSDeformAttnTransformerEncoderLayer(256, 512, 0.0, activation, n_levels=1, n_heads=8, n_points=4,
                                                use_adapters=True).cuda()
    src = rand(gen(1), 2, 130, 256)
    shapes, start = torch.tensor([[10, 13]], device="cuda"), torch.tensor([0], device="cuda")
    ref = torch.rand(2, 130, 1, 2, device="cuda", generator=gen(2))

    pull = rand(gen(3), 2, 130, 256)

    def run(fused, loss="squares"):
        layer.fused_norm = fused
        layer.zero_grad()
        x = src.clone().requires_grad_(True)
        y = layer(x, None, ref, shapes, start)
        (y.square() if loss == "squares" else y * pull).sum().backward()
        return [y.detach(), x.grad, *[p.grad.clone() for p in layer.parameters() if p.grad is not None]]

    before = layer_ext.launch_count()
    plain = run(False)
    assert (layer_ext.launch_count() > before) == (activation != "relu")
    between = layer_ext.launch_count()
    fused = run(True)
    assert layer_ext.launch_count() > between + 2
    for a, b in zip(plain, fused):
        # 32-bit sums in another order; the attention op's own vary with the run by 1e-5 of the largest value.  The sum of
        # squares of a normed row does not change with the row (its weights are still 1), so what reaches the inputs is the
        # difference of equal terms of up to 2 |y| = 9: off by 64 steps of those, 64 * 2^-24 * 9
        assert float((a - b).abs().max()) <= 1e-4 * float(a.abs().max()) + 64 * 2.0 ** -24 * 9
    for a, b in zip(run(False, "pull"), run(True, "pull")):
        assert float((a - b).abs().max()) <= 1e-4 * float(a.abs().max())


def test_encoder_stack_trains_with_muon():
    import train_bench
    from instaorder_amd import layer_ext
    enc = train_bench.build_encoder(levels=1, freeze_base=False, activation="swiglu").cuda()
    for m in enc.modules():
        if hasattr(m, "fused_norm"):
            m.fused_norm = True
    opts = train_bench.optimisers(enc, "muon")
    feats, pos = [rand(gen(1), 1, 256, 6, 7)], [rand(gen(2), 1, 256, 6, 7)]
    weights = [p.detach().clone() for p in enc.parameters()]
    before = layer_ext.launch_count()
    for _ in range(2):
        for o in opts:
            o.zero_grad(set_to_none=True)
        enc(feats, pos)[0].square().mean().backward()
        for o in opts:
            o.step()
    assert layer_ext.launch_count() > before
    assert all(p.isfinite().all() for p in enc.parameters())
    assert all(not torch.equal(p, w) for p, w in zip(enc.parameters(), weights) if p.grad is not None and p.grad.count_nonzero())


def test_gradients_are_differentiable_once():
    """With create_graph the first gradients are there; differentiating those again is an error, not silence."""
    from instaorder_amd import gated_feed_forward, residual_norm
    args = [a.requires_grad_(True) for a in ffn_inputs(torch.float32, 5, 16, 8, 16, True)]
    for y in (gated_feed_forward(*args), residual_norm(args[0], args[0] * 2, outer="rms")[1]):
        dx, = torch.autograd.grad(y.square().sum(), args[0], create_graph=True)
        assert dx.isfinite().all()
        with pytest.raises(RuntimeError):             # nothing leads from dx back to x
            torch.autograd.grad(dx.sum(), args[0], retain_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            dx.sum().backward()


def test_inputs_changed_after_the_forward_pass_are_noticed():
    from instaorder_amd import gated_feed_forward
    args = [a.requires_grad_(True) for a in ffn_inputs(torch.float32, 5, 16, 8, 16, True)]
    y = gated_feed_forward(*args)
    with torch.no_grad():
        args[1].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
