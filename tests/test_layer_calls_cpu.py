"""CPU-only checks of how the layer operators are called: under tracing, forward-mode derivatives, autocast, hooks; with
broadcast gates, after failed launches; and of the CPU paths beside the kernels."""
import pytest
import torch


def raw_calls():
    """The kernels' entry points by name, on CPU tensors: whatever they refuse they refuse before any device is touched."""
    from instaorder_amd import layer_ext
    b = layer_ext.bind()
    w_in, w_out = torch.randn(12, 8), torch.randn(8, 6)
    return {"gated_feed_forward": lambda x: b.gated_feed_forward(x, w_in, None, w_out, None, "silu"),
            "residual_norm": lambda x: b.residual_norm(x, x, None, None, None, None, None, "layer", None, None, 1e-5, True)[1],
            "orthogonalize": lambda x: b.orthogonalize(x, 5, 1.0, 1.0, 1.0, 1e-7)}


@pytest.mark.parametrize("name", ["gated_feed_forward", "residual_norm", "orthogonalize"])
def test_tracing_is_refused(name):
    """A trace would hold the results' allocations and not the kernels that fill them."""
    from torch.fx.experimental.proxy_tensor import make_fx
    call, x = raw_calls()[name], torch.randn(4, 8)
    with pytest.raises(RuntimeError, match=name + ".*cannot be traced"):
        torch.jit.trace(call, x)
    with pytest.raises(RuntimeError, match=name + ".*cannot be traced"):
        make_fx(call)(x)
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):       # and nothing is left behind
        call(x)


@pytest.mark.parametrize("name", ["gated_feed_forward", "residual_norm", "orthogonalize"])
def test_forward_mode_derivatives_are_refused(name):
    """With and without a graph to record: the kernels have no tangents, so none may be dropped."""
    import torch.autograd.forward_ad as fwAD
    call, x = raw_calls()[name], torch.randn(4, 8)
    with fwAD.dual_level():
        dual = fwAD.make_dual(x, torch.ones_like(x))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(RuntimeError, match=name + ".*forward-mode"):
                call(dual)
        with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
            call(x)


GATES = [((3, 1), (1, 1)), ((8, 5), (1, 1)), ((3, 1), (3, 1)), ((2, 3, 1), (2, 1, 1)), ((2, 3, 1), (1, 1, 1)),
         ((3, 1, 5), (1, 1, 1)), ((3, 1, 5), (3, 1, 1)), ((1, 1), (1, 1)), ((4, 1, 1), (1, 1, 1)), ((0, 1), (1, 1)),
         ((2, 1, 0), (2, 1, 1))]


@pytest.mark.parametrize("lead, gate", GATES)
def test_gates_shared_over_dimensions_of_one(lead, gate):
    """One token of a batch: x [batch, 1, width] under a gate [1, 1, width]."""
    from instaorder_amd import residual_norm
    g = torch.Generator().manual_seed(1)
    x, y, v = (torch.randn(*s, 16, generator=g) for s in (lead, lead, gate))
    r, _ = residual_norm(x, y, gate=v, outer="rms")
    assert torch.equal(r, x + y * v)
    with pytest.raises(RuntimeError, match="gate has shape"):
        residual_norm(x, y, gate=torch.zeros(*[2 if n == 1 else n for n in gate], 16), outer="rms")


def test_gates_in_other_dimensions_are_refused():
    from instaorder_amd import residual_norm
    x = torch.zeros(3, 4, 5, 16)
    for gate in ((3, 1, 5, 16), (1, 4, 1, 16), (1, 4, 5, 16), (4, 5, 16), (5, 16), (3, 4, 5, 1), (16,)):
        with pytest.raises(RuntimeError, match="gate has shape"):
            residual_norm(x, x, gate=torch.zeros(gate))


@pytest.mark.skipif(torch.cuda.is_available(), reason="the launches have to fail: the pointers are made up")
def test_every_failed_launch_is_reported():
    """Without a device each launch fails alike: the second failure is one too, and neither is counted or left pending."""
    from test_layer_cpu import lib, norm_call
    handle = lib()
    before = handle.enc_launch_count()
    for _ in range(3):
        assert norm_call() == 2
        assert "kernel launch failed" in handle.enc_last_error().decode()
        assert handle.enc_orthogonalize(0, 256, 256, 1, 8, 8, 5, 1.0, 1.0, 1.0, 1e-7, 256, 1 << 30, None) == 2
        assert handle.enc_gated_ffn_forward(1, 0, 16, 32, 16, None, 16, None, 4, 32, 8, 32, 16, None, 256, 1 << 30, None) == 2
        assert handle.enc_gated_ffn_backward(1, 0, 16, 32, 16, 16, 16, 16, 32, 4, 32, 8, 32, 16, 16, 16, 16, 16, 256, 1 << 30, None) == 2
    assert handle.enc_launch_count() == before


@pytest.mark.skipif(torch.cuda.is_available(), reason="the launches have to fail: the pointers are made up")
def test_every_failed_launch_of_the_attention_op_is_reported():
    import ctypes
    import os
    from conftest import ROOT
    handle = ctypes.CDLL(os.path.join(ROOT, "instaorder_amd", "libmsda_hip.so"))
    handle.msda_last_error.restype, handle.msda_launch_count.restype = ctypes.c_char_p, ctypes.c_uint64
    before, made_up = handle.msda_launch_count(), [ctypes.c_void_p(256)] * 5
    for _ in range(3):
        for head in (32, 24):                           # the kernels for 32 channels a head, and those for any
            assert handle.msda_forward_f32(*made_up, 1, 6, 2, head, 1, 4, 2, ctypes.c_void_p(256), None) == 2
            assert b"kernel launch failed" in handle.msda_last_error()
    assert handle.msda_launch_count() == before


def muon_runs(dtype, size, device="cpu", steps=4):
    """The same gradients, held exactly in `dtype`, for weights of that type and for fp32 weights: the two updates."""
    from instaorder_amd import Muon
    g = torch.Generator().manual_seed(11)
    grads = [(torch.randn(24, 40, generator=g) * size).to(dtype) for _ in range(steps)]
    out = []
    for kind in (dtype, torch.float32):
        p = torch.nn.Parameter(torch.zeros(24, 40, dtype=kind, device=device))
        opt = Muon([p], lr=0.05)
        for gr in grads:
            p.data.zero_()                             # the update alone, not its sum with a rounded weight
            p.grad = gr.to(device=device, dtype=kind)
            opt.step()
        out.append(p.detach().double().cpu())
    return out


# The update of 16-bit weights is off from that of fp32 weights by three roundings to the type of values up to 0.05 * 1.3 (the
# orthogonal matrix, the product with the rate, the weight), on the GPU also by two-part iterates (485 * 2^-17, as derived
# in test_gpu_layer.py); in the 2-norm of the whole the largest a rounding can be.
MUON_16 = {torch.float16: 3 * 2.0 ** -11 + 485 * 2.0 ** -17, torch.bfloat16: 3 * 2.0 ** -8 + 485 * 2.0 ** -17}


@pytest.mark.parametrize("dtype, size", [(torch.float16, 9000.0), (torch.float16, 1.0), (torch.float16, 1e-5), (torch.float16, 2e-7),
                                         (torch.bfloat16, 1e30), (torch.bfloat16, 1.0)])
def test_muon_takes_gradients_of_any_size(dtype, size):
    """v + g grows to 20 times the gradient and leaves fp16's range at either end; its direction is all that counts."""
    got, want = muon_runs(dtype, size)
    assert got.isfinite().all()
    assert float((got - want).norm() / want.norm()) <= MUON_16[dtype]


def test_orthogonalize_results_of_another_type():
    from instaorder_amd import orthogonalize
    u = torch.randn(2, 6, 9, generator=torch.Generator().manual_seed(2)) * 1e30
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        o = orthogonalize(u, dtype=dtype)
        assert o.dtype == dtype and torch.equal(o, orthogonalize(u).to(dtype))
    for given, dtype in ((torch.float16, torch.float32), (torch.float16, torch.bfloat16), (torch.float32, torch.float64),
                         (torch.bfloat16, torch.int16)):
        with pytest.raises(RuntimeError, match="orthogonalize"):
            orthogonalize(u.to(given), dtype=dtype)


@pytest.mark.parametrize("factor", [2.0 ** -60, 2.0 ** 100])
def test_cpu_orthogonalize_of_values_whose_squares_leave_32_bits(factor):
    from instaorder_amd import orthogonalize
    u = torch.randn(2, 6, 9, generator=torch.Generator().manual_seed(2))
    want = orthogonalize(u)
    assert torch.allclose(orthogonalize(u * factor, eps=1e-30), want, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("dtype, text", [(16, "unknown dtype"), (17, "workspace"), (18, "workspace"), (19, "unknown dtype")])
def test_c_abi_types_of_an_fp32_update(dtype, text):
    from test_layer_cpu import lib
    handle = lib()
    assert handle.enc_orthogonalize(dtype, 256, 256, 2, 8, 8, 5, 1.0, 1.0, 1.0, 1e-7, None, 0, None) == 1
    assert text in handle.enc_last_error().decode()
    room = handle.enc_orthogonalize_workspace_bytes
    assert room(dtype, 2, 8, 8) == (room(dtype & 3, 2, 8, 8) if text == "workspace" else 0)


@pytest.mark.parametrize("shape", [(6,), (2, 3, 4), ()])
def test_muon_refuses_added_groups_of_other_dimensions(shape):
    """A group that is added later: biases of one shape would be taken for the rows of a matrix."""
    from instaorder_amd import Muon
    opt = Muon([torch.nn.Parameter(torch.zeros(3, 3))])
    with pytest.raises(ValueError, match="two dimensions"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(shape))]})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": torch.nn.Parameter(torch.zeros(4, 3)), "lr": 0.1})
    assert len(opt.param_groups) == 2


def autocast_checks(device, dtype):
    """Under autocast the block runs in autocast's type, as F.linear does, and the norm in fp32, as F.layer_norm does: the
    calls of tensors cast by hand; gradients arrive in the leaves' own types."""
    from instaorder_amd import gated_feed_forward, residual_norm
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).to(device)      # noqa: E731
    x, wi, bi, wo, bo = (v.requires_grad_(True) for v in (r(3, 5, 16), r(48, 16), r(48), r(16, 24), r(16)))
    for given in (x, x.to(dtype)):
        with torch.autocast(device, dtype=dtype):
            y = gated_feed_forward(given, wi, bi, wo, bo)
        want = gated_feed_forward(*[v.to(dtype) for v in (x, wi, bi, wo, bo)])
        assert y.dtype == dtype and torch.equal(y, want)
        pull = r(3, 5, 16).to(dtype)
        got = torch.autograd.grad(y, [x, wi, bi, wo, bo], pull)
        ref = torch.autograd.grad(want, [x, wi, bi, wo, bo], pull)
        assert all(a.dtype == torch.float32 and torch.equal(a, b) for a, b in zip(got, ref))
    w, b, gate = (v.requires_grad_(True) for v in (r(16), r(16), r(3, 1, 16)))
    block = y.detach().requires_grad_(True)             # a 16-bit block under an fp32 residual
    for given in (x, x.to(dtype)):
        with torch.autocast(device, dtype=dtype):
            res, n = residual_norm(given, block, gate=gate, inner="rms", outer="layer", outer_weight=w, outer_bias=b)
        want = residual_norm(given.float(), block.float(), gate=gate, inner="rms", outer="layer", outer_weight=w, outer_bias=b)
        assert all(a.dtype == torch.float32 and torch.equal(a, c) for a, c in zip((res, n), want))
        got = torch.autograd.grad([res.sum(), n.square().sum()], [x, block, gate, w, b])
        ref = torch.autograd.grad([want[0].sum(), want[1].square().sum()], [x, block, gate, w, b])
        assert all(a.dtype == c.dtype and torch.equal(a, c) for a, c in zip(got, ref)) and got[1].dtype == dtype
    with torch.autocast(device, dtype=dtype), pytest.raises(RuntimeError, match="not implemented for"):
        gated_feed_forward(x.double(), wi, bi, wo, bo)   # 64 bits stay what they are
    with torch.autocast(device, enabled=False), pytest.raises(RuntimeError, match="has dtype"):
        gated_feed_forward(x.to(dtype), wi, bi, wo, bo)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_operators_under_autocast(dtype):
    autocast_checks("cpu", dtype)


def test_cpu_orthogonalize_is_the_same_under_autocast():
    from instaorder_amd import orthogonalize
    u = torch.randn(12, 20, generator=torch.Generator().manual_seed(4))
    want = orthogonalize(u)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert torch.equal(orthogonalize(u), want)


def encoder_layer(activation, dropout=0.0):
    from instaorder_amd.encoder import MSDeformAttnTransformerEncoderLayer
    torch.manual_seed(0)
    return MSDeformAttnTransformerEncoderLayer(32, 24, dropout, activation, n_levels=1, n_heads=4, n_points=2)


def test_gated_block_of_the_layer_under_autocast():
    layer, x = encoder_layer("swiglu"), torch.randn(2, 5, 32)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        got = layer._feed_forward(x)
        a, b = layer.linear1(x).chunk(2, -1)
        plain = layer.linear2(a * torch.nn.functional.silu(b))
    assert got.dtype == plain.dtype == torch.bfloat16
    assert torch.allclose(got.float(), plain.float(), atol=4 * 2.0 ** -8 * float(plain.abs().max()))


def submodule_changes():
    """(what, change(layer)): each replaces or watches a submodule of the gated block; a call has to show it."""
    def own_forward(layer):
        inner = layer.linear1.forward
        layer.linear1.forward = lambda x: 2 * inner(x)

    class Wrapped(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner, self.weight, self.bias = inner, inner.weight, inner.bias

        def forward(self, x):
            return self.inner(x) + 1

    class Doubled(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    def subclass(layer):
        new = Doubled(24, 32)
        new.load_state_dict(layer.linear2.state_dict())
        layer.linear2 = new

    return [("hook on the output", lambda layer: layer.linear1.register_forward_hook(lambda m, i, o: o * 3)),
            ("hook on the input", lambda layer: layer.linear2.register_forward_pre_hook(lambda m, i: (i[0] + 1,))),
            ("hook on dropout", lambda layer: layer.dropout2.register_forward_hook(lambda m, i, o: o * 3)),
            ("forward of its own", own_forward), ("wrapper", lambda layer: setattr(layer, "linear2", Wrapped(layer.linear2))),
            ("subclass", subclass), ("activation", lambda layer: setattr(layer, "activation", torch.tanh)),
            ("dropout alone in training", lambda layer: (layer.eval(), setattr(layer.dropout2, "p", 0.9), layer.dropout2.train()))]


@pytest.mark.parametrize("at", range(8))
def test_changed_submodules_of_the_gated_block_are_called(at):
    what, change = submodule_changes()[at]
    layer, x = encoder_layer("swiglu"), torch.randn(2, 5, 32)
    plain = layer._feed_forward(x)
    change(layer)
    torch.manual_seed(3)
    got = layer._feed_forward(x)
    torch.manual_seed(3)
    a, b = layer.linear1(x).chunk(2, -1)
    want = layer.linear2(layer.dropout2(a * layer.activation(b)))
    assert torch.equal(got, want) and not torch.allclose(got, plain), what


def test_hooks_of_all_modules_and_of_gradients_see_the_gated_block():
    layer, x, seen = encoder_layer("swiglu"), torch.randn(2, 5, 32), []
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, i, o: seen.append(m))
    try:
        layer._feed_forward(x)
    finally:
        handle.remove()
    assert layer.linear1 in seen and layer.linear2 in seen
    layer.linear1.register_full_backward_hook(lambda m, gi, go: seen.clear())
    layer._feed_forward(x).sum().backward()
    assert not seen


def test_layers_saved_whole_before_the_gated_block_still_run():
    """A pickled layer has its attributes, not those that later ones set in their constructor."""
    layer, x = encoder_layer("relu"), torch.randn(1, 12, 32)
    args = (None, torch.rand(1, 12, 1, 2), torch.tensor([[3, 4]]), torch.tensor([0]))
    want = layer(x, *args)
    for name in ("gate", "fused_norm"):
        layer.__dict__.pop(name, None)
    assert torch.equal(layer(x, *args), want)


def test_cpu_paths_need_no_build(tmp_path):
    """Only GPU tensors need the compiled library: a copy of the package without it computes on the CPU and says what a GPU
    call would need."""
    import os
    import shutil
    import subprocess
    import sys
    from conftest import ROOT
    shutil.copytree(os.path.join(ROOT, "instaorder_amd"), tmp_path / "instaorder_amd",
                    ignore=shutil.ignore_patterns("*.so", "*.o", "__pycache__", "csrc"))
    code = """
import torch, instaorder_amd as A
x, w, v = torch.randn(3, 8), torch.randn(12, 8), torch.randn(8, 6)
assert A.gated_feed_forward(x, w, None, v, None).shape == (3, 8)
assert A.residual_norm(x, x)[1].shape == (3, 8)
assert A.orthogonalize(x).shape == (3, 8)
p = torch.nn.Parameter(x); p.grad = x.clone(); A.Muon([p]).step()
for call in (lambda: A.gated_feed_forward(x, w[1:], None, v, None), lambda: A.residual_norm(x, x[:, 1:])):
    try:
        call()
        raise SystemExit("taken")
    except RuntimeError as e:
        assert "shape" in str(e) or "expected" in str(e), e
from instaorder_amd import layer_ext
try:
    layer_ext.bind()
    raise SystemExit("bound")
except RuntimeError as e:
    assert "not built" in str(e)
print("ok")
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, capture_output=True, text=True, timeout=300,
                         env=dict(os.environ, PYTHONPATH=str(tmp_path)))
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stderr[-2000:]


def refusals():
    """Calls that both the CPU paths and the kernels' binding refuse: (operator, arguments)."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    x, wi, bi, wo, bo = r(2, 3, 8), r(12, 8), r(12), r(5, 6), r(5)
    ffn = [(x, wi, bi, wo, bo, "tanh"), (x.double(), wi, bi, wo, bo, "silu"), (x.long(), wi, bi, wo, bo, "silu"),
           (x, wi[:-1], bi, wo, bo, "silu"), (x, wi[:, 1:], bi, wo, bo, "silu"), (x, wi[0], bi, wo, bo, "silu"),
           (x, wi, bi, wo[0], bo, "silu"), (x, wi, bi[1:], wo, bo, "silu"), (x, wi, bi, wo.half(), bo, "silu"),
           (x, wi, bi, wo, bo[1:], "silu"), (x, wi.to("meta"), bi, wo, bo, "silu"), (x[..., :0], wi[:, :0], bi, wo, bo, "silu"),
           (x, wi[:0], bi[:0], wo[:, :0], bo, "silu"), (torch.tensor(1.0), wi, bi, wo, bo, "silu")]
    n = lambda x, y, gate=None, scale=None, inner=None, iw=None, ib=None, outer="layer", ow=None, ob=None, want=True: (      # noqa: E731
        x, y, gate, scale, inner, iw, ib, outer, ow, ob, 1e-5, want)
    norm = [n(x, x[..., 1:]), n(x, x, inner="batch"), n(x, x, outer="l2"), n(x, x, outer=None, want=False), n(x, x, iw=x[0, 0]),
            n(x, x, ib=x[0, 0]), n(x, x, outer=None, ob=x[0, 0]), n(x, x, outer=None, ow=x[0, 0]), n(x, x, scale=x[0]),
            n(x, x, gate=x[:1]), n(x, x, gate=x[0]), n(x.double(), x.double()), n(x, x, gate=x.half()), n(x, x.half()),
            n(torch.zeros(1, 16385), torch.zeros(1, 16385)), n(torch.zeros(3, 0), torch.zeros(3, 0)),
            n(torch.tensor(1.0), torch.tensor(1.0)), n(x, x.to("meta")), n(x, x, inner="rms", iw=x[0, 0, 1:])]
    muon = [(x[0, 0], 5), (x.double(), 5), (x, 0), (x, 101), (torch.zeros(2, 0, 3), 5), (torch.zeros(2, 3, 0), 5),
            (x, 5, torch.float64), (x.half(), 5, torch.float32)]
    return [("gated_feed_forward", a) for a in ffn] + [("residual_norm", a) for a in norm] + [("orthogonalize", a) for a in muon]


@pytest.mark.parametrize("at", range(41))
def test_the_cpu_paths_refuse_what_the_kernels_refuse(at):
    """With the same words."""
    from instaorder_amd import gated_feed_forward, layer_ext, orthogonalize, residual_norm
    name, a = refusals()[at]
    bind, text = layer_ext.bind(), []
    if name == "gated_feed_forward":
        calls = [lambda: bind.gated_feed_forward(*a), lambda: gated_feed_forward(*a)]
    elif name == "residual_norm":
        keys = ("gate", "scale", "inner", "inner_weight", "inner_bias", "outer", "outer_weight", "outer_bias", "eps", "want_residual")
        calls = [lambda: bind.residual_norm(*a), lambda: residual_norm(*a[:2], **dict(zip(keys, a[2:])))]
    else:
        calls = [lambda: bind.orthogonalize(a[0], a[1], 1.0, 1.0, 1.0, 1e-7, *a[2:]),
                 lambda: orthogonalize(a[0], steps=a[1], dtype=a[2] if len(a) > 2 else None)]
    for call in calls:
        with pytest.raises(RuntimeError, match=name) as e:
            call()
        text.append(str(e.value).split("\n")[0])
    assert text[0] == text[1] and "Not implemented on the CPU" not in text[0]


def test_refusals_are_all_run():
    assert len(refusals()) == 41


def test_the_width_limit_is_one():
    import os
    import re
    from conftest import ROOT
    from instaorder_amd import layer_ext
    header = open(os.path.join(ROOT, "include", "enc_hip.h")).read()
    assert int(re.search(r"#define ENC_NORM_MAX_WIDTH (\d+)", header).group(1)) == layer_ext.NORM_MAX_WIDTH


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_cpu_paths_round_as_documented(dtype):
    """16-bit tensors: 32 bits inside and one rounding a result, on the CPU as on the GPU."""
    import layer_reference as R
    from instaorder_amd import gated_feed_forward, residual_norm
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)      # noqa: E731
    t = [v.requires_grad_(True) for v in (r(9, 40), r(48, 40), r(48), r(33, 24), r(33))]
    grad = r(9, 33)
    y = gated_feed_forward(*t, activation="gelu")
    got = dict(zip(("d_x", "d_w_in", "d_b_in", "d_w_out", "d_b_out"), torch.autograd.grad(y, t, grad)), y=y.detach())
    want = R.ffn(*[v.detach() for v in t], "gelu", grad)
    assert set(got) == set(want)
    for k, (v, bound) in want.items():
        assert got[k].dtype == dtype
        R.within(got[k], v, bound, k)
    d = {"x": r(6, 7, 40), "y": r(6, 7, 40), "gate": r(6, 1, 40), "scale": r(40), "inner_weight": r(40), "inner_bias": r(40),
         "outer_weight": r(40), "outer_bias": r(40)}
    for inner, outer in (("layer", "rms"), ("rms", "layer")):
        leaves = {k: v.detach().requires_grad_(True) for k, v in d.items()}
        res, n = residual_norm(**leaves, inner=inner, outer=outer)
        grads = {"residual": r(6, 7, 40), "normed": r(6, 7, 40)}
        got = torch.autograd.grad([res, n], list(leaves.values()), list(grads.values()))
        got = {"residual": res.detach(), "normed": n.detach(), **{"d_" + k: v for k, v in zip(leaves, got)}}
        want = R.residual_norm(d, inner, outer, 1e-5, grads)
        assert set(got) == set(want)
        for k, w in want.items():
            # one rounding to the type, and 32-bit sums of at most 64 + 4 sqrt(42) terms of the largest size, spread 16 times
            R.within(got[k], w, (R.U[dtype] * w.abs()).clamp(min=R.FLOOR[dtype]) + 90 * 16 * R.U32 * (w.abs().max() + 1.0), k)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspace_of_calls_whose_tensors_lie_well(dtype, backward):
    """Room for copies is asked for only where copies are made: the query's flag, what a call then needs, and its refusal of a
    workspace of that size where a tensor has to be laid out after all.  (Launches fail without a device, or are not reached.)"""
    from test_layer_cpu import lib
    handle, m, d, f, o = lib(), 512, 64, 256, 72
    query = handle.enc_gated_ffn_backward_workspace_bytes if backward else handle.enc_gated_ffn_forward_workspace_bytes
    full, placed = query(dtype, m, d, f, o), query(dtype | 32, m, d, f, o)
    copies = 2 * (m * d + 2 * f * d + o * f + (m * o if backward else 0))
    assert full - placed == (copies if dtype else 0)                          # (fp32 is laid out in parts in any case)
    assert query(9 | 32, m, d, f, o) == 0
    odd = query(dtype, m, d, f + 1, o) - query(dtype | 32, m, d, f + 1, o)     # odd hidden widths: the weights are laid out
    assert odd == (2 * (m * d + (m * o if backward else 0)) if dtype else 0)

    def call(nbytes, **change):
        a = {**dict(x=256, ld=d, w_in=256, w_out=256, grad=256, grad_ld=o), **change}
        if backward:
            return handle.enc_gated_ffn_backward(dtype, 0, a["x"], a["ld"], a["w_in"], a["w_out"], 256, a["grad"], a["grad_ld"], m, d, f, o,
                                                 256, 256, 256, 256, 256, 256, nbytes, None)
        return handle.enc_gated_ffn_forward(dtype, 0, a["x"], a["ld"], a["w_in"], None, a["w_out"], None, m, d, f, o, 256, None, 256,
                                            nbytes, None)

    assert call(placed - 1) == 1 and "workspace" in handle.enc_last_error().decode()
    if dtype:
        for change in (dict(x=258), dict(ld=d + 1), dict(ld=1 << 22), dict(w_in=264), dict(w_out=266),
                       *([dict(grad=258), dict(grad_ld=o + 4)] if backward else [])):
            assert call(placed, **change) == 1 and "workspace" in handle.enc_last_error().decode(), change
    if not torch.cuda.is_available():
        assert call(placed) == 2 and call(full, x=264) == 2


@pytest.mark.parametrize("name", ["gated_feed_forward", "residual_norm", "orthogonalize"])
def test_fake_tensors_are_refused(name):
    from torch._subclasses.fake_tensor import FakeTensorMode
    call, x = raw_calls()[name], torch.randn(4, 8)
    with FakeTensorMode() as mode, pytest.raises(RuntimeError, match=name + ".*cannot be traced"):
        call(mode.from_tensor(x))


def test_cpu_paths_can_be_traced():
    """They are torch's own operators; the checks leave nothing in the trace, whatever they look at."""
    import warnings
    from instaorder_amd import gated_feed_forward, residual_norm
    wi, wo, gate, w = torch.randn(12, 8), torch.randn(8, 6), torch.randn(2, 1, 8), torch.randn(8)

    def call(x):
        r, n = residual_norm(x, 2 * x, gate=gate, outer="rms", outer_weight=w)
        return gated_feed_forward(n, wi, None, wo, None), r

    with warnings.catch_warnings():
        warnings.simplefilter("error", torch.jit.TracerWarning)
        traced = torch.jit.trace(call, torch.randn(2, 3, 8))
    x = torch.randn(2, 3, 8)
    assert all(torch.allclose(a, b) for a, b in zip(traced(x), call(x)))
    assert "aten::empty" not in str(traced.graph)
