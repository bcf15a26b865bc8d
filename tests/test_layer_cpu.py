"""CPU-only checks of the layer operators: the C ABI of libenc_hip.so (symbols, refusals before any launch), the Python
entry points' refusals, the CPU path against the 64-bit forms, the encoder layer and the optimiser that call them."""
import copy
import ctypes
import json
import os
import re
import subprocess
import sys

import pytest
import torch

import layer_reference as R
from conftest import ROOT

LIB = os.path.join(ROOT, "instaorder_amd", "libenc_hip.so")
HEADER = os.path.join(ROOT, "include", "enc_hip.h")


I, L, Z, P, F = ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_float
PROTOTYPES = {
    "enc_abi_version": ([], I), "enc_last_error": ([], ctypes.c_char_p), "enc_launch_count": ([], ctypes.c_uint64),
    "enc_gated_ffn_forward_workspace_bytes": ([I] + [L] * 4, Z), "enc_gated_ffn_backward_workspace_bytes": ([I] + [L] * 4, Z),
    "enc_gated_ffn_pre_floats": ([L, L], Z), "enc_residual_norm_backward_workspace_bytes": ([L] * 3, Z),
    "enc_orthogonalize_workspace_bytes": ([I] + [L] * 3, Z),
    "enc_gated_ffn_forward": ([I, I, P, L] + [P] * 4 + [L] * 4 + [P] * 3 + [Z, P], I),
    "enc_gated_ffn_backward": ([I, I, P, L] + [P] * 4 + [L] * 5 + [P] * 6 + [Z, P], I),
    "enc_residual_norm_forward": ([I, I, I, F, P, L, P, L, P, L, L] + [P] * 5 + [L, L] + [P] * 4, I),
    "enc_residual_norm_backward": ([I, I, I, P, L, P, L, P, L, L] + [P] * 6 + [L, P, L, L, L] + [P] * 9 + [Z, P], I),
    "enc_orthogonalize": ([I, P, P] + [L] * 3 + [I] + [F] * 4 + [P, Z, P], I)}


def lib():
    handle = ctypes.CDLL(LIB)
    for name, (args, res) in PROTOTYPES.items():
        getattr(handle, name).argtypes, getattr(handle, name).restype = args, res
    return handle


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(enc_[a-z0-9_]+)\s*\(", text)))
    assert names == sorted(PROTOTYPES)
    handle = ctypes.CDLL(LIB)
    for n in names:
        assert hasattr(handle, n), n
    assert lib().enc_abi_version() == 1


FFN = dict(dtype=1, act=0, x=16, x_stride=32, w_in=16, b_in=None, w_out=16, b_out=None, tokens=4, width=32, hidden=8,
           out_width=32, y=16, pre=None, ws=None, nbytes=0, stream=None)


@pytest.mark.parametrize("change, text", [
    (dict(dtype=7), "unknown dtype"), (dict(act=9), "unknown activation"), (dict(tokens=-1), "bad dimensions"),
    (dict(width=0), "bad dimensions"), (dict(hidden=0), "bad dimensions"), (dict(hidden=1 << 22), "bad dimensions"),
    (dict(tokens=1 << 23), "bad dimensions"), (dict(x=None), "a tensor is missing"), (dict(x_stride=31), "x_stride"),
    (dict(pre=8), "16-byte aligned"), ({}, "workspace"), (dict(ws=256, nbytes=1), "workspace"),
    (dict(ws=128, nbytes=1 << 30), "workspace")])
def test_c_abi_refuses_feed_forward_calls(change, text):
    a = {**FFN, **change}
    assert lib().enc_gated_ffn_forward(*a.values()) == 1
    assert text in lib().enc_last_error().decode()


def test_c_abi_empty_calls_launch_nothing():
    before = lib().enc_launch_count()
    assert lib().enc_gated_ffn_forward(*{**FFN, "tokens": 0}.values()) == 0
    assert lib().enc_residual_norm_forward(0, 0, 1, 1e-5, None, 8, None, 8, None, 0, 1, None, None, None, None, None, 0, 8, None,
                                           None, None, None) == 0
    assert lib().enc_orthogonalize(0, None, None, 0, 4, 4, 5, 1.0, 1.0, 1.0, 1e-7, None, 0, None) == 0
    assert lib().enc_launch_count() == before


def norm_call(dtype=0, inner=0, outer=1, x=16, x_ld=8, y=16, y_ld=8, gate=None, gate_ld=0, group=1, rows=4, width=8,
              residual=None, normed=16, stats=None):
    return lib().enc_residual_norm_forward(dtype, inner, outer, 1e-5, x, x_ld, y, y_ld, gate, gate_ld, group, None, None, None,
                                           None, None, rows, width, residual, normed, stats, None)


@pytest.mark.parametrize("change, text", [
    (dict(dtype=3), "unknown dtype"), (dict(inner=3), "unknown norm"), (dict(outer=-1), "unknown norm"),
    (dict(width=0), "bad dimensions"), (dict(width=16385, x_ld=20000, y_ld=20000), "bad dimensions"),
    (dict(rows=-1), "bad dimensions"), (dict(rows=1 << 31), "bad dimensions"), (dict(group=0), "bad dimensions"),
    (dict(group=3), "bad dimensions"), (dict(x=None), "missing"), (dict(normed=None), "missing"),
    (dict(outer=0), "missing"), (dict(x_ld=7), "stride"), (dict(gate=16, gate_ld=4), "stride"), (dict(stats=8), "misaligned")])
def test_c_abi_refuses_norm_calls(change, text):
    assert norm_call(**change) == 1
    assert text in lib().enc_last_error().decode()


def test_c_abi_refuses_norm_gradients_of_what_was_not_there():
    args = [0, 0, 1, 16, 8, 16, 8, None, 0, 1, None, None, None, None, 16, None, 0, 16, 8, 4, 8, 16, 16]
    for wrong in range(4):                              # d_gate, d_scale, d_inner_weight, d_inner_bias
        tail = [None] * 6
        tail[wrong] = 16
        assert lib().enc_residual_norm_backward(*args, *tail, None, 0, None) == 1
        assert "did not have" in lib().enc_last_error().decode()


@pytest.mark.parametrize("change, text", [
    (dict(dtype=5), "unknown dtype"), (dict(rows=0), "bad dimensions"), (dict(steps=0), "bad dimensions"),
    (dict(steps=101), "bad dimensions"), (dict(batch=65536), "bad dimensions"), (dict(batch=-1), "bad dimensions"),
    (dict(rows=65537, cols=65537), "bad dimensions"), (dict(update=None), "missing"), ({}, "workspace")])
def test_c_abi_refuses_orthogonalize_calls(change, text):
    a = {**dict(dtype=0, update=16, out=16, batch=2, rows=8, cols=8, steps=5, a=1.0, b=1.0, c=1.0, eps=1e-7, ws=None, n=0,
                st=None), **change}
    assert lib().enc_orthogonalize(*a.values()) == 1
    assert text in lib().enc_last_error().decode()


def test_workspace_queries_grow_and_refuse():
    q = lib().enc_gated_ffn_forward_workspace_bytes
    assert 0 < q(1, 8, 64, 64, 64) < q(1, 4096, 64, 64, 64) and q(9, 8, 64, 64, 64) == 0
    assert lib().enc_gated_ffn_pre_floats(17, 9) == 2 * 1 * 512 and lib().enc_gated_ffn_pre_floats(-1, 9) == 0
    assert lib().enc_residual_norm_backward_workspace_bytes(10, 8, 3) == 0       # 10 rows are no groups of 3
    assert lib().enc_orthogonalize_workspace_bytes(0, 1, 0, 4) == 0


def params(width=8, hidden=6, out=5, dtype=torch.float32):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64).to(dtype)      # noqa: E731
    return r(2, 3, width), r(2 * hidden, width), r(2 * hidden), r(out, hidden), r(out)


def test_python_refusals():
    import instaorder_amd as A
    from instaorder_amd import layer_ext
    x, wi, bi, wo, bo = params()
    bad = [lambda: A.gated_feed_forward(x, wi, bi, wo, bo, "tanh"), lambda: A.gated_feed_forward(x.double(), wi, bi, wo, bo),
           lambda: A.gated_feed_forward(x, wi[:-1], bi, wo, bo), lambda: A.gated_feed_forward(x, wi[:, 1:], bi, wo, bo),
           lambda: A.gated_feed_forward(x, wi, bi[1:], wo, bo), lambda: A.gated_feed_forward(x, wi, bi, wo.half(), bo),
           lambda: A.gated_feed_forward(x, wi, bi, wo, bo[1:]), lambda: A.gated_feed_forward(x, wi.to("meta"), bi, wo, bo),
           lambda: A.residual_norm(x, x[..., 1:]), lambda: A.residual_norm(x, x, inner="batch"),
           lambda: A.residual_norm(x, x, outer=None, want_residual=False), lambda: A.residual_norm(x, x, inner_weight=x[0, 0]),
           lambda: A.residual_norm(x, x, outer=None, outer_bias=x[0, 0]), lambda: A.residual_norm(x, x, scale=x[0]),
           lambda: A.residual_norm(x, x, gate=x[:1]), lambda: A.residual_norm(x, x, gate=x[0]),
           lambda: A.residual_norm(x.double(), x.double()), lambda: A.residual_norm(x, x, gate=x.half()),
           lambda: A.residual_norm(torch.zeros(1, 16385), torch.zeros(1, 16385)),
           lambda: A.residual_norm(torch.zeros(3, 0), torch.zeros(3, 0)),
           lambda: A.orthogonalize(x[0, 0]), lambda: A.orthogonalize(x.double()), lambda: A.orthogonalize(x, steps=0),
           lambda: A.orthogonalize(torch.zeros(2, 0, 3))]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail("call %d was taken" % i)
    b = layer_ext.bind()                               # the kernels themselves never take a CPU tensor
    for call in (lambda: b.gated_feed_forward(x, wi, bi, wo, bo, "silu"), lambda: b.orthogonalize(x, 5, 1., 1., 1., 1.),
                 lambda: b.residual_norm(x, x, None, None, None, None, None, "layer", None, None, 1e-5, True)):
        with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
            call()


@pytest.mark.parametrize("kind", ["silu", "gelu", "sigmoid", "relu"])
def test_cpu_feed_forward_matches_the_formula_and_its_gradients(kind):
    import instaorder_amd as A
    t = [v.requires_grad_(True) for v in params()]
    grad = torch.randn(2, 3, 5, generator=torch.Generator().manual_seed(2))
    y = A.gated_feed_forward(*t, activation=kind)
    got = dict(zip(("d_x", "d_w_in", "d_b_in", "d_w_out", "d_b_out"), torch.autograd.grad(y, t, grad)), y=y.detach())
    want = R.ffn(t[0].detach().reshape(-1, 8), *[v.detach() for v in t[1:]], kind, grad.reshape(-1, 5))
    for k, (v, bound) in want.items():
        R.within(got[k].reshape(v.shape), v, bound, k)


def test_reference_gradients_agree_with_differences():
    """The formulas that the kernels are held to, against central differences in 64 bits."""
    x, wi, bi, wo, bo = (v.double() for v in params())
    x = x.reshape(-1, 8)
    grad = torch.randn(6, 5, dtype=torch.float64, generator=torch.Generator().manual_seed(3))
    R.U[torch.float64], eps = 0.0, 1e-6
    try:
        for kind in ("silu", "gelu", "sigmoid"):
            args = [x, wi, bi, wo, bo]
            want = R.ffn(*args, kind, grad)
            for i, name in enumerate(("d_x", "d_w_in", "d_b_in", "d_w_out", "d_b_out")):
                flat = args[i].reshape(-1)
                for at in range(0, flat.numel(), 7):
                    def value(step):
                        moved = flat.clone()
                        moved[at] += step
                        return (R.ffn(*args[:i], moved.view_as(args[i]), *args[i + 1:], kind)["y"][0] * grad).sum()
                    assert abs((value(eps) - value(-eps)) / (2 * eps) - want[name][0].reshape(-1)[at]) < 1e-6
    finally:
        del R.U[torch.float64]


@pytest.mark.parametrize("inner, outer, gate", [(None, "layer", None), ("rms", "rms", "sample"), ("layer", "layer", "token"),
                                                ("layer", None, None), (None, "rms", "token")])
def test_cpu_residual_norm_matches_the_formula(inner, outer, gate):
    import instaorder_amd as A
    g = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(s, generator=g)      # noqa: E731
    t = {"x": r(2, 3, 8), "y": r(2, 3, 8), "scale": r(8)}
    if gate:
        t["gate"] = r(2, 1 if gate == "sample" else 3, 8)
    if inner:
        t["inner_weight"] = r(8)
    if outer == "layer":
        t["outer_weight"], t["outer_bias"] = r(8), r(8)
    grads = {"residual": r(2, 3, 8), **({"normed": r(2, 3, 8)} if outer else {})}
    for v in t.values():
        v.requires_grad_(True)
    res, normed = A.residual_norm(inner=inner, outer=outer, **t)
    out = {k: v for k, v in (("residual", res), ("normed", normed)) if v is not None}
    got = torch.autograd.grad(list(out.values()), list(t.values()), [grads[k] for k in out])
    out.update(("d_" + k, v) for k, v in zip(t, got))
    want = R.residual_norm(t, inner, outer, 1e-5, grads)
    for k, v in want.items():
        assert float((out[k].double() - v).norm() / v.norm()) < 1e-5, k


def test_cpu_orthogonalize_and_its_properties():
    from instaorder_amd import orthogonalize
    g = torch.Generator().manual_seed(5)
    for shape in ((6, 9), (9, 6), (2, 3, 5, 4), (1, 7)):
        u = torch.randn(shape, generator=g)
        o = orthogonalize(u)
        assert o.shape == u.shape and not o.requires_grad
        want = R.orthogonalize(u, 5, (3.4445, -4.7750, 2.0315), 1e-7)
        assert float((o.double() - want).norm() / want.norm()) < 1e-4
        s = torch.linalg.svdvals(o.double())
        assert float(s.max()) < 1.3                   # the quintic keeps singular values in about [0.7, 1.2]
    assert torch.equal(orthogonalize(torch.zeros(3, 4)), torch.zeros(3, 4))


def test_muon_steps_are_the_rule():
    from instaorder_amd import Muon, orthogonalize
    g = torch.Generator().manual_seed(6)
    w = [torch.nn.Parameter(torch.randn(6, 4, generator=g)) for _ in range(2)] + [torch.nn.Parameter(torch.randn(3, 5, generator=g))]
    start = [p.detach().clone() for p in w]
    opt = Muon(w, lr=0.1, momentum=0.9, weight_decay=0.01)
    v = [torch.zeros_like(p) for p in w]
    for _ in range(2):
        grads = [torch.randn(p.shape, generator=g) for p in w]
        for p, gr in zip(w, grads):
            p.grad = gr.clone()
        opt.step()
        for i, gr in enumerate(grads):
            v[i] = 0.9 * v[i] + gr
            o = orthogonalize(gr + 0.9 * v[i])
            start[i] = start[i] * (1 - 0.1 * 0.01) - 0.1 * max(1, start[i].shape[0] / start[i].shape[1]) ** 0.5 * o
    for p, s in zip(w, start):
        assert torch.allclose(p, s, rtol=1e-5, atol=1e-6)
    state = copy.deepcopy(opt.state_dict())
    opt.load_state_dict(state)
    w[0].grad = None                                  # parameters without a gradient are left as they are
    before = w[0].detach().clone()
    opt.step()
    assert torch.equal(w[0], before)
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(3, 3))], momentum=1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_muon_keeps_its_momentum_in_fp32(dtype):
    from instaorder_amd import Muon
    g = torch.Generator().manual_seed(8)
    grads = [(torch.randn(6, 4, generator=g) * s).to(dtype) for s in (1.0, 2e-3, 2e-3)]
    runs = []
    for reload in (False, True):
        p = torch.nn.Parameter(torch.zeros(6, 4, dtype=dtype))
        opt = Muon([p], lr=0.1, momentum=0.999)
        for gr in grads:
            p.grad = gr.clone()
            opt.step()
            if reload:
                state = copy.deepcopy(opt.state_dict())
                opt = Muon([p], lr=0.1, momentum=0.999)
                opt.load_state_dict(state)
        runs.append((p.detach(), opt.state[p]["momentum_buffer"]))
    want = torch.zeros(6, 4, dtype=torch.float64)
    for gr in grads:
        want = 0.999 * want + gr.double()
    for _, v in runs:
        # two roundings a step to half of 2^-23 each, of values to 2 |v|
        assert v.dtype == torch.float32 and float((v - want).abs().max()) <= 6 * 2.0 ** -24 * 2 * float(want.abs().max())
    assert torch.equal(runs[0][0], runs[1][0])
    p.grad = torch.eye(6, 4).to(dtype).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()


@pytest.mark.parametrize("activation", ["glu", "swiglu", "geglu", "reglu"])
def test_encoder_layer_with_a_gated_block(activation):
    from instaorder_amd.encoder import GATED, MSDeformAttnTransformerEncoderLayer
    torch.manual_seed(0)
    layer = MSDeformAttnTransformerEncoderLayer(32, 24, 0.0, activation, n_levels=1, n_heads=4, n_points=2)
    assert layer.linear1.weight.shape == (48, 32) and layer.linear2.weight.shape == (32, 24)
    x = torch.randn(2, 5, 32)
    want = R.ffn(x.reshape(-1, 32), layer.linear1.weight.detach(), layer.linear1.bias.detach(), layer.linear2.weight.detach(),
                 layer.linear2.bias.detach(), GATED[activation])["y"]
    R.within(layer._feed_forward(x).detach().reshape(-1, 32), *want, activation)
    if activation == "glu":                           # the order of F.glu
        a = torch.nn.functional.linear(torch.nn.functional.glu(layer.linear1(x)), layer.linear2.weight, layer.linear2.bias)
        assert torch.allclose(layer._feed_forward(x), a, atol=1e-6)
    dropping = MSDeformAttnTransformerEncoderLayer(32, 24, 0.5, activation, n_levels=1, n_heads=4, n_points=2)
    assert dropping._feed_forward(x).shape == x.shape                       # dropout inside: the plain path
    layer.double()
    assert layer._feed_forward(x.double()).dtype == torch.float64


def test_fused_norm_changes_nothing_on_the_cpu_and_keeps_the_state_dict():
    from instaorder_amd.encoder import MSDeformAttnTransformerEncoderLayer
    torch.manual_seed(0)
    layer = MSDeformAttnTransformerEncoderLayer(32, 24, 0.0, "relu", n_levels=1, n_heads=4, n_points=2)
    keys = set(layer.state_dict())
    src, shapes, start = torch.randn(1, 12, 32), torch.tensor([[3, 4]]), torch.tensor([0])
    ref = torch.rand(1, 12, 1, 2)
    plain = layer(src, None, ref, shapes, start)
    layer.fused_norm = True
    assert torch.equal(layer(src, None, ref, shapes, start), plain) and set(layer.state_dict()) == keys
    assert layer.gate is None and layer.linear1.weight.shape == (24, 32)


def test_training_harness_takes_the_new_choices():
    common = [sys.executable, os.path.join(ROOT, "train_bench.py"), "--cpu", "--image", "64", "--global-batch", "2", "--steps", "1",
              "--warmup", "0"]
    env = dict(os.environ, OMP_NUM_THREADS="2")
    for extra in (["--activation", "swiglu", "--optimizer", "muon", "--all-trainable", "--fused-norm"], ["--optimizer", "muon"]):
        run = subprocess.run(common + extra, capture_output=True, text=True, env=env, timeout=300)
        assert run.returncode == 0, run.stderr[-2000:]
        r = json.loads([line for line in run.stdout.splitlines() if line.startswith("{")][-1])
        assert r["config"]["optimizer"] == "muon" and r["value"] > 0
