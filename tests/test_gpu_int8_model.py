"""The -shaped DiT models with their blocks' linear layers in 8 bits (ShapedDiT.quantize_linears_).

What may be expected: a step of the rows is 1/127 of a row's largest value, some 4 deviations, so a row's values are off by
4 / 127 / sqrt(12) = 0.9 % of their deviation, a weight's by about as much, and a layer's result by 1.3 %. Over the four layers in
a row of five blocks that is 1.3 % * sqrt(20) = 6 %, a cosine of 0.998."""
import pytest
import torch

from tests.test_gpu_model import DEV, _inputs, tiny_shape

pytestmark = pytest.mark.gpu


def _cosine(a, b):
    return torch.nn.functional.cosine_similarity(a.float().flatten(), b.float().flatten(), dim=0).item()


def _model(kind, seed=3):
    from hetu_dit_b200.model_executor.models.shaped_dit import ShapedDiT
    shape, grid = tiny_shape(kind)
    model = ShapedDiT(shape).to(DEV).init_weights(seed=seed, std=0.05).bfloat16()
    lat, txt, pooled, t, g = _inputs(shape, int(torch.tensor(grid).prod()), 33)
    args = (lat.to(DEV), txt.to(DEV), pooled.to(DEV) if shape.pooled_dim else None, t.to(DEV), g.to(DEV))
    return model, args, grid


@pytest.mark.parametrize("kind", ["flux", "sd3", "cogvideox", "hunyuan"])
@torch.no_grad()
def test_quantized_model_step(kind):
    from hetu_dit_b200 import _C
    from hetu_dit_b200.model_executor.layers.int8_linear import Int8Linear
    model, args, grid = _model(kind)
    want = model(*args, grid=grid)
    assert model.quantize_linears_() is model
    blocks = list(model.transformer_blocks) + list(model.single_transformer_blocks)
    assert not any(type(m) is torch.nn.Linear for b in blocks for m in b.modules())
    assert type(model.x_embedder) is torch.nn.Linear and any(type(m) is Int8Linear for m in blocks[0].modules())
    got = model(*args, grid=grid)
    assert torch.isfinite(got).all() and _cosine(got, want) >= 0.995
    assert torch.equal(got, model(*args, grid=grid))  # nothing depends on an order
    graphed = model.forward_graphed(*args, grid=grid)
    assert torch.equal(graphed, got)
    # with a hook on every layer each is called by itself: rows of 16-bit values, one tail kernel after each
    handles = [m.register_forward_hook(lambda m, i, o: None) for b in blocks for m in b.modules() if type(m) is Int8Linear]
    separate = model(*args, grid=grid)
    # half a step apart where the 16-bit rounding of a norm's result (2^-9 of it, a quarter of a step at most) crosses a border:
    # less than the 8-bit values' own error
    assert _cosine(separate, got) >= 0.998 and _cosine(separate, want) >= 0.995
    for h in handles:
        h.remove()
    torch.cuda.synchronize()
    assert _C.device_status(0, clear=True)[0] == 0


@torch.no_grad()
def test_graph_of_the_16_bit_model_is_not_replayed():
    model, args, grid = _model("sd3")
    before = model.forward_graphed(*args, grid=grid).clone()
    after = model.quantize_linears_().forward_graphed(*args, grid=grid)
    assert not torch.equal(before, after) and torch.equal(after, model(*args, grid=grid))


@torch.no_grad()
def test_int8_linear_layer_is_the_product_over_its_rows():
    from hetu_dit_b200 import kernels
    from hetu_dit_b200.model_executor.layers.int8_linear import Int8Linear
    gen = torch.Generator(device=DEV).manual_seed(1)
    for k, n, bias in ((256, 96, True), (100, 33, False), (100, 1, True)):
        linear = torch.nn.Linear(k, n, bias=bias, device=DEV, dtype=torch.bfloat16)
        layer = Int8Linear.from_linear(linear)
        x = torch.randn(2, 50, k, generator=gen, device=DEV).bfloat16()
        want = kernels.linear_int8(x, kernels.quantize_rows(linear.weight), linear.bias)
        assert torch.equal(layer(x), want) and torch.equal(layer(kernels.quantize_rows(x)), want)
        assert torch.equal(layer(x[0]), want[0])
        moved = Int8Linear.from_linear(linear).to("cpu").to(DEV)  # the rows keep their places
        assert torch.equal(moved(x), want)
        assert _cosine(want, linear(x)) >= 0.999


@pytest.mark.parametrize("through", ["model", "blocks"])
@torch.no_grad()
def test_a_pipeline_that_ran_in_16_bits_runs_the_8_bit_layers(through):
    """The pipeline keeps captured steps of its own."""
    from hetu_dit_b200 import _C
    from hetu_dit_b200.config import EngineConfig
    from hetu_dit_b200.core.distributed import parallel_state as ps
    from hetu_dit_b200.core.distributed.runtime_state import ModelGeometry, initialize_runtime_state, reset_runtime_state
    from hetu_dit_b200.core.resource_manager.cache_manager import reset_cache_manager
    from hetu_dit_b200.model_executor.layers.int8_linear import quantize_linears_
    from hetu_dit_b200.model_executor.pipelines.pipeline_flux_shaped import FluxShapedPipeline
    from tests.test_gpu_pipefusion import _tiny_flux
    _, model, *inputs = _tiny_flux()
    model, inputs = model.to(DEV), [x.to(DEV) for x in inputs]
    ps.destroy_model_parallel()
    reset_cache_manager()
    rt = initialize_runtime_state(ModelGeometry(4, 64), EngineConfig())
    rt.set_input_parameters(height=512, width=256, batch_size=1, num_inference_steps=4)
    try:
        pipe = FluxShapedPipeline(model, guidance_scale=3.5, grid=(32, 16))
        steps = lambda: pipe.diffusion_stage(*inputs, 4).clone()  # noqa: E731
        in_16_bits = steps()
        assert pipe._graphs.captures == 1 and pipe._graphs.replays == 3
        if through == "model":
            model.quantize_linears_()
        else:
            quantize_linears_(model.transformer_blocks)
            quantize_linears_(model.single_transformer_blocks)
        got = steps()
        assert pipe._graphs.captures == 2
        assert torch.equal(steps(), got)  # replays only
        pipe.use_cuda_graph = False
        assert torch.equal(steps(), got) and not torch.equal(got, in_16_bits)
        torch.cuda.synchronize()
        assert _C.device_status(0, clear=True)[0] == 0
    finally:
        reset_runtime_state()
        reset_cache_manager()
