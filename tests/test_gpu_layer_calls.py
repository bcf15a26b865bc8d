"""GPU tests of how the layer operators are called: derivatives of other kinds, broadcast gates, autocast, weights in 16 bits
with gradients out of their range, hooks; against the 64-bit forms of layer_reference.py where there are values to compare."""
import pytest
import torch

import layer_reference as R
from test_gpu_layer import COEFFICIENTS, FLOATS, MUON, ffn_inputs, gen, norm_inputs, rand

pytestmark = pytest.mark.gpu


def test_a_gradient_with_a_tangent_is_refused():
    """Forward over reverse: the kernels of the backward pass would drop it."""
    import torch.autograd.forward_ad as fwAD
    from instaorder_amd import gated_feed_forward, residual_norm
    args = [a.requires_grad_(True) for a in ffn_inputs(torch.float32, 5, 16, 8, 16, True)]
    for call in (lambda: gated_feed_forward(*args), lambda: residual_norm(args[0], args[0] * 2, outer="rms")[1]):
        y = call()
        with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, args[0], fwAD.make_dual(torch.ones_like(y), torch.ones_like(y)))
        dx, = torch.autograd.grad(call(), args[0], torch.ones_like(y))
        assert dx.isfinite().all()


def gradients(t, inner, outer):
    """Results and all gradients of a residual norm of the leaves `t`; none may be missing."""
    from instaorder_amd import residual_norm
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
    r, n = residual_norm(**leaves, inner=inner, outer=outer)
    g = gen(99)
    grads = {"residual": rand(g, *t["x"].shape, dtype=t["x"].dtype), "normed": rand(g, *t["x"].shape, dtype=t["x"].dtype)}
    got = torch.autograd.grad([r, n], list(leaves.values()), list(grads.values()))
    return {"residual": r.detach(), "normed": n.detach(), **{"d_" + k: v for k, v in zip(leaves, got)}}, grads


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("lead, gate", [((3, 1), (1, 1)), ((2, 3, 1), (2, 1, 1)), ((3, 1, 5), (1, 1, 1)), ((3, 1, 5), (3, 1, 1)),
                                        ((700, 1), (1, 1)), ((1, 1), (1, 1))])
def test_gates_shared_over_dimensions_of_one(dtype, lead, gate):
    t = norm_inputs(dtype, lead, 72, "layer", "rms", None, True, "wb")
    t["gate"] = rand(gen(3), *gate, 72, dtype=dtype)
    got, grads = gradients(t, "layer", "rms")
    want = R.residual_norm(t, "layer", "rms", 1e-5, grads)
    norm_within(got, want, dtype, t["x"].numel() // 72, 72)


def norm_within(got, want, dtype, rows, width):
    """The bounds of test_gpu_layer.py for rows and column sums; every result and gradient has to be there."""
    assert set(got) == set(want)
    for k, v in got.items():
        w = want[k]
        assert v is not None and v.shape == w.shape and v.dtype == dtype, k
        row = v.dim() and v.shape[-1] == width and v.numel() == rows * width and v.dim() > 1
        size, steps = (w.abs().amax(-1, keepdim=True), 64) if row else (w.abs().max(), 64 + 4 * rows ** 0.5)
        R.within(v, w, (R.U[dtype] * w.abs()).clamp(min=R.FLOOR[dtype]) + steps * 16 * R.U32 * (size + 1.0) + R.TINY, k)


OPTIONAL = ("gate", "scale", "inner_weight", "inner_bias", "outer_weight", "outer_bias")


@pytest.mark.parametrize("present", range(64))
def test_norm_every_gradient_is_there(present):
    """Each choice of the optional inputs: all gradients against the 64-bit form, then each input's alone (the scale's is summed
    in another order where no gate's is formed beside it)."""
    from instaorder_amd import residual_norm
    given = [k for i, k in enumerate(OPTIONAL) if present >> i & 1]
    t = {k: v for k, v in norm_inputs(torch.float32, (3, 7), 40, "layer", "rms", "sample", True, "wb").items() if k in ("x", "y", *given)}
    got, grads = gradients(t, "layer", "rms")
    want = R.residual_norm(t, "layer", "rms", 1e-5, grads)
    norm_within(got, want, torch.float32, 21, 40)
    for k in t:
        one = {n: v.detach().requires_grad_(n == k) for n, v in t.items()}
        r, n = residual_norm(**one, inner="layer", outer="rms")
        v, = torch.autograd.grad([r, n], one[k], list(grads.values()))
        norm_within({"d_" + k: v}, {"d_" + k: want["d_" + k]}, torch.float32, 21, 40)


@pytest.mark.parametrize("present", range(4))
def test_feed_forward_every_gradient_is_there(present):
    from instaorder_amd import gated_feed_forward
    args = ffn_inputs(torch.float32, 70, 40, 48, 24, True)
    args[2], args[4] = args[2] if present & 1 else None, args[4] if present & 2 else None
    grad = rand(gen(5), 70, 24)
    want = R.ffn(*args, "silu", grad)
    names = ("d_x", "d_w_in", "d_b_in", "d_w_out", "d_b_out")
    leaves = [None if a is None else a.detach().requires_grad_(True) for a in args]
    all_of = [(i, v) for i, v in enumerate(leaves) if v is not None]
    got = torch.autograd.grad(gated_feed_forward(*leaves), [v for _, v in all_of], grad)
    for (i, _), v in zip(all_of, got):
        R.within(v, *want[names[i]], names[i])
        one = [None if a is None else a.detach().requires_grad_(j == i) for j, a in enumerate(args)]
        alone, = torch.autograd.grad(gated_feed_forward(*one), one[i], grad)
        assert torch.equal(alone, v), names[i]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_feed_forward_takes_no_room_for_copies_that_it_does_not_make(dtype):
    """A training call whose tensors lie well: beside its results and what it saves (a, b in 32 bits) it holds h, its gradients,
    and sums.  The same call on rows that have to be laid out gives the same."""
    from instaorder_amd import gated_feed_forward
    m, d, f = 1024, 2048, 2048
    args = [a.requires_grad_(True) for a in ffn_inputs(dtype, m, d, f, d, True)]
    grad = rand(gen(2), m, d, dtype=dtype)
    y = gated_feed_forward(*args)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = torch.autograd.grad(y, args, grad)
    peak = torch.cuda.max_memory_allocated() - before
    results = sum(g.numel() for g in got) * 2
    hidden = 3 * m * f * 2                              # h, da, db
    # sums: slices of k in 32 bits (their number grows until the chip is full: 512 tiles of 128 x 128 at most), 64 rows of columns
    assert peak <= results + hidden + 4 * (512 * 128 * 128 + 64 * 2 * f) + (1 << 20)
    shifted = [torch.cat((torch.zeros(1, device="cuda", dtype=dtype), a.detach().flatten()))[1:].view(a.shape).requires_grad_(True) for a in args]
    y2 = gated_feed_forward(*shifted)
    again = torch.autograd.grad(y2, shifted, grad)
    assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(got, again))


# ---- how h is held ------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m, d, f, o", [(1, 2048, 5632, 2048), (16, 2048, 2056, 520), (7, 1024, 4104, 71), (3, 176, 24600, 64),
                                        (1, 8200, 520, 8), (16, 64, 96, 64), (1, 1024, 2816, 1024), (5, 33, 17, 41), (16, 2049, 2051, 36)])
def test_feed_forward_of_few_tokens_holds_the_hidden_values_in_two_parts(dtype, m, d, f, o):
    """Up to 16 tokens, whatever the weights' size and rows: the result is as good as h were never rounded.

    In the 2-norm a result is off by its own rounding and twice what it is off before (the distance to the next value of a
    type changes no faster than the value).  Before, it is off by k sums of 32 bits, whose roundings of U32 / sqrt(3) go
    either way (2.5 sqrt(k) is above four deviations) but for a cut of up to 2 U32 in each matrix instruction of 32 k, and by
    u^2 of h, what two parts leave over (fp16: or half its smallest step).  One part's rounding of h is as large as y's."""
    from instaorder_amd import gated_feed_forward
    args = ffn_inputs(dtype, m, d, f, o, True, seed=m)
    x, wi, bi, wo, bo = (a.double() for a in args)
    a, b = (x @ wi.t() + bi).chunk(2, -1)
    h, u, k = a * R.activate(b, "silu"), R.U[dtype], d + f
    want = h @ wo.t() + bo
    size = float((h.square() @ wo.square().t() + bo.square()).sum().sqrt())
    rest = float(((u * u * h.abs()).clamp(min=R.FLOOR[dtype]).square() @ wo.square().t()).sum().sqrt())
    tol = float((want.to(dtype).double() - want).norm()) + 2 * ((2.5 * k ** 0.5 + k / 16) * R.U32 * size + rest)
    leaves = [v.detach().requires_grad_(True) for v in args]                 # and where pre-activations are kept
    for y in (gated_feed_forward(*args), gated_feed_forward(*leaves).detach()):
        assert float((y.double() - want).norm()) <= tol


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [5, 100, 700])
@pytest.mark.parametrize("f", [1, 8, 17, 40])
def test_feed_forward_infinities_do_not_meet_the_padding(dtype, m, f):
    """Hidden widths that are no multiple of 8 are padded with zeros, which an Inf would turn to NaN: everything is positive
    here, so what the definition makes of an Inf is Inf."""
    from instaorder_amd import gated_feed_forward
    x, wi, bi, wo, bo = (a.abs() + 0.01 for a in ffn_inputs(dtype, m, 24, f, 16, True))
    row, rest = m // 2, torch.arange(m, device="cuda") != m // 2
    clean = gated_feed_forward(x, wi, bi, wo, bo, "relu")
    x2 = x.clone()
    x2[row, 3] = float("inf")
    y = gated_feed_forward(x2, wi, bi, wo, bo, "relu")
    assert (y[row] == float("inf")).all() and torch.equal(y[rest], clean[rest])
    leaves = [v.requires_grad_(True) for v in (x, wi, bi, wo, bo)]
    grad = torch.ones(m, 16, device="cuda", dtype=dtype)
    grad[row, 5] = float("inf")
    d_x, d_wi, d_bi, d_wo, d_bo = torch.autograd.grad(gated_feed_forward(*leaves, "relu"), leaves, grad)
    assert (d_x[row] == float("inf")).all() and d_x[rest].isfinite().all()
    assert (d_wi == float("inf")).all() and (d_bi == float("inf")).all()
    assert (d_wo[5] == float("inf")).all() and d_wo[:5].isfinite().all() and d_bo[5] == float("inf")


# ---- autocast -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_operators_under_autocast(dtype):
    from test_layer_calls_cpu import autocast_checks
    autocast_checks("cuda", dtype)


@pytest.mark.parametrize("activation", ["relu", "swiglu"])
def test_fused_norm_of_the_layer_under_autocast(activation):
    """A 16-bit block under an fp32 residual goes through the kernel, with the values of the plain path."""
    from instaorder_amd import layer_ext
    from instaorder_amd.encoder import MSDeformAttnTransformerEncoderLayer
    torch.manual_seed(0)
    layer = MSDeformAttnTransformerEncoderLayer(64, 96, 0.0, activation, n_levels=1, n_heads=2, n_points=4).cuda()
    src = rand(gen(1), 2, 130, 64)
    out = {}
    for fused in (False, True):
        layer.fused_norm = fused
        before = layer_ext.launch_count()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out[fused] = layer._add_and_norm(src, layer._feed_forward(src), layer.norm2)
        launches = layer_ext.launch_count() - before
        assert out[fused].dtype == torch.float32 and (launches > 0) == (fused or activation != "relu")
    assert launches > (activation != "relu")
    # the same 16-bit block: the norms' sums in another order
    assert float((out[True] - out[False]).abs().max()) <= 64 * R.U32 * 16 * (1 + float(out[False].abs().max()))


# ---- submodules of the layer ----------------------------------------------------------------------
def test_changed_norms_of_the_layer_are_called():
    from instaorder_amd import layer_ext
    from instaorder_amd.encoder import MSDeformAttnTransformerEncoderLayer
    torch.manual_seed(0)
    layer = MSDeformAttnTransformerEncoderLayer(64, 96, 0.0, "relu", n_levels=1, n_heads=2, n_points=4).cuda()
    layer.fused_norm = True
    src, block = rand(gen(1), 2, 30, 64), rand(gen(2), 2, 30, 64)

    def call():
        before = layer_ext.launch_count()
        out = layer._add_and_norm(src, block, layer.norm1)
        return out.detach(), layer_ext.launch_count() > before

    plain, fused = call()
    assert fused
    handle = layer.norm1.register_forward_hook(lambda m, i, o: o * 3)
    out, fused = call()
    assert not fused and torch.allclose(out, 3 * plain, atol=1e-4)
    handle.remove()
    layer.norm1 = torch.nn.LayerNorm(64, elementwise_affine=False).cuda()        # no weight: still the kernel
    out, fused = call()
    assert fused and torch.allclose(out, plain, atol=1e-4)                       # (the weights were still one and zero)
    layer.norm1 = torch.nn.LayerNorm((30, 64)).cuda()                            # over two dimensions: not the kernel's norm
    out, fused = call()
    assert not fused and torch.equal(out, layer.norm1(src + block))

    class Doubled(torch.nn.LayerNorm):
        def forward(self, x):
            return 2 * super().forward(x)

    layer.norm1 = Doubled(64).cuda()
    out, fused = call()
    assert not fused and torch.allclose(out, 2 * plain, atol=1e-4)


@pytest.mark.parametrize("activation", ["relu", "swiglu"])
def test_traced_layer_takes_its_modules(activation):
    from instaorder_amd.encoder import MSDeformAttnTransformerEncoderLayer
    torch.manual_seed(0)
    layer = MSDeformAttnTransformerEncoderLayer(64, 96, 0.0, activation, n_levels=1, n_heads=2, n_points=4).cuda()
    layer.requires_grad_(False)                          # a trace of a function takes weights as constants
    layer.fused_norm = True

    def call(x):
        return layer._add_and_norm(x, layer._feed_forward(x), layer.norm2)

    with torch.no_grad():
        traced = torch.jit.trace(call, rand(gen(1), 2, 30, 64))
        for seed in (1, 2):
            x = rand(gen(seed), 2, 30, 64)
            assert torch.allclose(traced(x), call(x), atol=1e-4)


def test_compiled_and_inference_mode_calls_are_the_eager_ones():
    """torch.compile breaks its graph at the kernels."""
    import warnings
    from instaorder_amd import gated_feed_forward, residual_norm
    x, wi, bi, wo, bo = ffn_inputs(torch.float32, 9, 16, 24, 16, True)

    def call(x):
        return gated_feed_forward(residual_norm(x, x * 2, outer="rms")[1], wi, bi, wo, bo) + 1

    want = call(x)
    with torch.inference_mode():
        assert torch.equal(call(x), want)
    y = x.clone().requires_grad_(True)
    d_want, = torch.autograd.grad(call(y).sum(), y)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        compiled = torch.compile(call, backend="aot_eager")
        assert torch.equal(compiled(x), want)
        d, = torch.autograd.grad(compiled(y).sum(), y)
    assert torch.equal(d, d_want)


# ---- Muon ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, size", [(torch.float16, 9000.0), (torch.float16, 1.0), (torch.float16, 1e-5), (torch.float16, 2e-7),
                                         (torch.bfloat16, 1e30), (torch.bfloat16, 1.0)])
def test_muon_takes_gradients_of_any_size(dtype, size):
    from test_layer_calls_cpu import MUON_16, muon_runs
    got, want = muon_runs(dtype, size, "cuda")
    assert got.isfinite().all()
    assert float((got - want).norm() / want.norm()) <= MUON_16[dtype]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (7, 33), (3, 130, 65), (2, 260, 1000), (1500, 600), (0, 4, 4)])
def test_orthogonalize_results_of_another_type(dtype, shape):
    """An fp32 update with a 16-bit result: within the bound of that type, for values that the type does not reach too."""
    from instaorder_amd import orthogonalize
    u = rand(gen(5), *shape)
    for factor in (1.0, 2.0 ** 40, 2.0 ** -10):
        o = orthogonalize(u * factor, dtype=dtype)
        assert o.shape == u.shape and o.dtype == dtype
        if u.numel():
            want = R.orthogonalize(u * factor, 5, COEFFICIENTS, 1e-7).flatten(-2)
            off = (o.double().flatten(-2) - want).norm(dim=-1) / want.norm(dim=-1)
            assert float(off.max()) <= MUON[dtype]
    assert torch.equal(orthogonalize(u, dtype=torch.float32), orthogonalize(u))
    for bad in (lambda: orthogonalize(u.to(dtype), dtype=torch.float32), lambda: orthogonalize(u, dtype=torch.float64)):
        with pytest.raises(RuntimeError, match="orthogonalize"):
            bad()
