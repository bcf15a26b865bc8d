"""GPU tests: captured calls of the attention op whose results are added into cleared memory, replayed several times with
eager work between."""
import pytest
import torch

from conftest import rel_err

pytestmark = pytest.mark.gpu

ORDER_TOL = {torch.float32: 2e-5, torch.bfloat16: 2.0 ** -8, torch.float64: 1e-12}       # atomic sums in another order; one rounding


@pytest.fixture(scope="module")
def msda():
    import MultiScaleDeformableAttention
    return MultiScaleDeformableAttention


@pytest.mark.parametrize("dtype, batch, channels", [(torch.float32, 2, 32), (torch.bfloat16, 2, 32), (torch.float32, 1, 24),
                                                    (torch.float64, 1, 32)])
def test_captured_backward_replays(msda, dtype, batch, channels):
    """Few images (the lists of a tile in parts that add into grad_value) and any other head width (atomics)."""
    from instaorder_amd import synthetic

    def inputs(seed):
        inp = synthetic.make_inputs(batch, synthetic.encoder_shapes(256), dist="model", seed=seed, device="cuda")
        grad = inp["grad_output"].view(batch, -1, 8, 32)[..., :channels].reshape(batch, -1, 8 * channels)
        other = torch.float32 if dtype == torch.bfloat16 else dtype
        return [inp["value"][..., :channels].contiguous().to(dtype), inp["spatial_shapes"], inp["level_start_index"],
                inp["sampling_locations"].to(other), inp["attention_weights"].to(other), grad.contiguous().to(dtype)]

    a = inputs(3)
    step = lambda: msda.ms_deform_attn_backward(*a, 128)      # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (4, 5, 6, 7):
        for t, new in zip(a, inputs(seed)):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, step()):
            assert rel_err(x.double().cpu().numpy(), y.double().cpu().numpy()) < ORDER_TOL[dtype]
