"""CPU tests of what the wrappers of the 8-bit rows and the group norm refuse before a launch, and of what the library
refuses by itself. Nothing is launched."""
import ctypes

import pytest
import torch

from hetu_dit_b200 import _C, kernels
from tests.test_host_dispatch import OnGpu, gpu_like, lib  # noqa: F401


def rows8(*shape, dtype=torch.bfloat16):
    q = torch.zeros(*shape, dtype=torch.int8)
    pitch = -(-shape[-1] // 16) * 16
    q = torch.zeros(*shape[:-1], pitch, dtype=torch.int8)[..., :shape[-1]].as_subclass(OnGpu)
    return kernels.Int8Rows(q, torch.ones(shape[:-1]).as_subclass(OnGpu), dtype)


def test_host_tensors_are_refused(lib):  # noqa: F811
    x, w = torch.randn(1, 4, 32).bfloat16(), rows8(16, 32)
    for call in (lambda: kernels.quantize_rows(x), lambda: kernels.ln_modulate_int8(x, x[:, 0], x[:, 0]),
                 lambda: kernels.linear_int8(x, w), lambda: kernels.group_norm(x, 4), lambda: kernels.group_norm_int8(x, 4)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    assert lib.calls == []


def _linear(**change):
    a = dict(x=gpu_like(2, 40, 32), weight=rows8(24, 32), bias=gpu_like(24), epilogue="gate_residual", residual=gpu_like(2, 40, 24),
             gate=gpu_like(2, 24), out=gpu_like(2, 40, 24))
    a.update(change)
    return kernels.linear_int8(a.pop("x"), a.pop("weight"), a.pop("bias"), a.pop("epilogue"), **a)


BAD_LINEAR = {
    "type of x": dict(x=gpu_like(2, 40, 32, dtype=torch.float32)),
    "weight in 16 bits": dict(weight=gpu_like(24, 32)),
    "inner sizes": dict(x=gpu_like(2, 40, 48)),
    "epilogue": dict(epilogue="silu"),
    "bias size": dict(bias=gpu_like(23)),
    "bias type": dict(bias=gpu_like(24, dtype=torch.float16)),
    "no residual": dict(residual=None),
    "no gate": dict(gate=None),
    "residual shape": dict(residual=gpu_like(2, 40, 25)),
    "residual type": dict(residual=gpu_like(2, 40, 24, dtype=torch.float16)),
    "gate shape": dict(gate=gpu_like(1, 24)),
    "out shape": dict(out=gpu_like(2, 41, 24)),
    "out type": dict(out=gpu_like(2, 40, 24, dtype=torch.float16)),
    "x columns": dict(x=gpu_like(2, 40, 64)[..., ::2]),
    "weight scale type": dict(weight=kernels.Int8Rows(rows8(24, 32).q, torch.ones(24).half().as_subclass(OnGpu))),
    "weight scale count": dict(weight=kernels.Int8Rows(rows8(24, 32).q, torch.ones(23).as_subclass(OnGpu))),
    "weight rows": dict(weight=kernels.Int8Rows(torch.zeros(24, 40, dtype=torch.int8).as_subclass(OnGpu)[:, :32],
                                                torch.ones(24).as_subclass(OnGpu))),
    "x rows": dict(x=kernels.Int8Rows(torch.zeros(2, 40, 40, dtype=torch.int8).as_subclass(OnGpu)[..., :32],
                                      torch.ones(2, 40).as_subclass(OnGpu))),
    "x scale": dict(x=kernels.Int8Rows(rows8(2, 40, 32).q, torch.ones(2, 41).as_subclass(OnGpu))),
    "dimensions": dict(x=gpu_like(2, 2, 40, 32)),
    "another device": dict(bias=torch.empty(24, dtype=torch.bfloat16, device="meta")),
}


@pytest.mark.parametrize("what", BAD_LINEAR)
def test_linear_int8_refuses(lib, what):  # noqa: F811
    with pytest.raises((ValueError, TypeError)):
        _linear(**BAD_LINEAR[what])
    assert lib.calls == []


def test_linear_int8_takes_what_it_documents(lib, monkeypatch):  # noqa: F811
    monkeypatch.setattr(kernels, "_cuda_index", lambda device: 0)
    _linear()
    _linear(x=rows8(2, 40, 32))
    assert [c[0] for c in lib.calls] == ["hdit_int8_linear"] * 2
    first, second = (c[1][0]._obj for c in lib.calls)
    assert (first.m, first.n, first.k, first.rows_per_batch) == (80, 24, 32, 40)
    assert first.x and not second.x
    assert _linear(x=gpu_like(2, 0, 32), residual=gpu_like(2, 0, 24), out=gpu_like(2, 0, 24)).shape == (2, 0, 24)
    assert len(lib.calls) == 2
    # rows that are a slice of every entry's: a launch for each
    _linear(out=gpu_like(2, 50, 24)[:, 3:43])
    assert len(lib.calls) == 4


def test_rows_and_norms_refuse(lib):  # noqa: F811
    x = gpu_like(2, 40, 64)
    for bad in (gpu_like(64), x[..., ::2], x[..., :0]):
        with pytest.raises(ValueError):
            kernels.quantize_rows(bad)
    with pytest.raises(TypeError):
        kernels.quantize_rows(x.float())
    for sh, sc in ((gpu_like(1, 64), gpu_like(1, 64)), (gpu_like(2, 64), gpu_like(2, 128)[:, :64]), (gpu_like(2, 128)[:, ::2],) * 2):
        with pytest.raises(ValueError):
            kernels.ln_modulate_int8(x, sh, sc)
    with pytest.raises(TypeError):
        kernels.ln_modulate_int8(x, gpu_like(2, 64, dtype=torch.float16), gpu_like(2, 64))
    image = gpu_like(2, 6, 10, 64).permute(0, 3, 1, 2)
    for bad in (gpu_like(2, 64, 6, 10), image[..., ::2], image[:, ::2], gpu_like(60, 64)):
        with pytest.raises(ValueError):
            kernels.group_norm(bad, 8)
        with pytest.raises(ValueError):
            kernels.group_norm_int8(bad, 8)
    for kw in (dict(groups=7), dict(groups=0), dict(groups=8, act="gelu"), dict(groups=8, weight=gpu_like(63)),
               dict(groups=8, bias=gpu_like(64, dtype=torch.float16)), dict(groups=8, out=gpu_like(2, 64, 6, 10)),
               dict(groups=8, out=gpu_like(2, 64, 6, 11))):
        with pytest.raises(ValueError):
            kernels.group_norm(image, **kw)
    assert [c for c in lib.calls if c[0] != "hdit_group_norm_scratch"] == []


def test_the_library_refuses_by_itself():
    real = _C.lib()
    q, s = ctypes.c_void_p(4096), ctypes.c_void_p(4096)  # addresses that nothing reads
    none = ctypes.c_void_p(0)
    rows = lambda **k: real.hdit_quantize_rows(*{**dict(dtype=0, x=q, q=q, s=s, rows=4, dim=32, rpb=4, xb=0, xr=32, qr=32, st=none), **k}.values())  # noqa: E731
    for bad in (dict(dtype=2), dict(rows=-1), dict(dim=0), dict(rpb=0), dict(x=none), dict(q=none), dict(s=none), dict(qr=24), dict(qr=16),
                dict(q=ctypes.c_void_p(4104)), dict(x=ctypes.c_void_p(4097)), dict(s=ctypes.c_void_p(4098)), dict(dim=1 << 31)):
        assert rows(**bad) in (_C.HDIT_ERR_BAD_ARG, _C.HDIT_ERR_SHAPE, _C.HDIT_ERR_TOO_LARGE), bad
    assert rows(rows=0) == 0
    ln = lambda **k: real.hdit_ln_modulate_int8(*{**dict(dtype=0, x=q, sh=q, sc=q, q=q, s=s, rows=4, dim=32, rpb=4, xb=0, xr=32, qr=32, mb=32, eps=1e-6, st=none), **k}.values())  # noqa: E731
    for bad in (dict(dim=20), dict(dim=8200, qr=8208), dict(sh=none), dict(sc=ctypes.c_void_p(4097))):
        assert ln(**bad) in (_C.HDIT_ERR_BAD_ARG, _C.HDIT_ERR_SHAPE), bad
    def gn(entry=real.hdit_group_norm, **change):
        a = _C.GroupNormArgs()
        fields = dict(dtype=0, act=0, x=4096, out=4096, out_scale=4096, scratch=4096, batch=1, rows=4, channels=64, groups=8, x_row_stride=64,
                      out_row_stride=64, eps=1e-6)
        for name, v in {**fields, **change}.items():
            setattr(a, name, v)
        return entry(ctypes.byref(a))

    for entry in (real.hdit_group_norm, real.hdit_group_norm_int8):
        for bad in (dict(dtype=2), dict(batch=-1), dict(channels=60), dict(groups=7), dict(groups=0), dict(channels=4104), dict(act=2), dict(x=0),
                    dict(out=0), dict(batch=65536), dict(rows=1 << 31), dict(rows=1 << 22, scratch=4100), dict(rows=1 << 22, scratch=0)):
            assert gn(entry, **bad) in (_C.HDIT_ERR_BAD_ARG, _C.HDIT_ERR_SHAPE, _C.HDIT_ERR_TOO_LARGE), bad
        assert gn(entry, batch=0) == 0 and gn(entry, rows=0) == 0 and entry(None) == _C.HDIT_ERR_BAD_ARG
    for bad in (dict(out=4104), dict(out_row_stride=72), dict(out_row_stride=48), dict(out_scale=0)):
        assert gn(real.hdit_group_norm_int8, **bad) in (_C.HDIT_ERR_BAD_ARG, _C.HDIT_ERR_SHAPE), bad

    def linear(**change):
        a = _C.Int8LinearArgs()
        fields = dict(dtype=0, epilogue=2, m=8, n=24, k=32, a=4096, lda=32, a_scale=4096, w=4096, ldw=32, w_scale=4096, bias=4096, out=4096,
                      ldo=24, residual=4096, ldr=24, gate=4096, gate_batch_stride=24, rows_per_batch=4)
        for name, v in {**fields, **change}.items():
            setattr(a, name, v)
        return real.hdit_int8_linear(ctypes.byref(a))

    for bad in (dict(dtype=2), dict(epilogue=3), dict(m=-1), dict(n=0), dict(k=0), dict(k=131073), dict(m=1 << 31), dict(a=0), dict(w=0), dict(out=0),
                dict(a_scale=0), dict(w_scale=0), dict(lda=24), dict(ldw=16), dict(a=4104), dict(w=4104), dict(ldo=20), dict(ldr=20), dict(residual=0),
                dict(gate=0), dict(rows_per_batch=0), dict(out=4097), dict(a_scale=4098), dict(residual=4097)):
        assert linear(**bad) in (_C.HDIT_ERR_BAD_ARG, _C.HDIT_ERR_SHAPE, _C.HDIT_ERR_TOO_LARGE), bad
    assert linear(m=0) == 0
    few = dict(epilogue=0, m=2, x=1 << 20, x_rows_per_batch=2, x_row_stride=32)  # two rows need no scratch, but where they may be overwritten
    for bad in (dict(x=4096, a=0), dict(x=4096, a_scale=0), dict(m=3, a=0), dict(tile=1, a=0), dict(x_rows_per_batch=0), dict(x=(1 << 20) + 1),
                dict(tile=5, m=9), dict(tile=6), dict(tile=5, k=131072, ldw=131072, m=2)):
        assert linear(**{**few, **bad}) in (_C.HDIT_ERR_BAD_ARG, _C.HDIT_ERR_SHAPE), bad
    assert real.hdit_int8_linear(None) == _C.HDIT_ERR_BAD_ARG


def test_an_8_bit_layer_takes_its_tail_where_nothing_waits_for_its_call(monkeypatch):
    from hetu_dit_b200.model_executor.layers.int8_linear import Int8Linear, read_rows
    layer = Int8Linear(rows8(24, 40), torch.zeros(24).bfloat16())
    assert layer.rows.shape == (24, 40) and layer.rows.q.stride(0) == 48
    seen = []

    def linear_int8(x, weight, bias=None, epilogue="bias", residual=None, gate=None, out=None):
        seen.append(epilogue)
        return gpu_like(2, 40, 24)

    monkeypatch.setattr(kernels, "linear_int8", linear_int8)
    monkeypatch.setattr(kernels, "gelu_tanh", lambda y, out=None: seen.append("gelu kernel"))
    monkeypatch.setattr(kernels, "gate_residual", lambda r, g, y, out=None: seen.append("gate kernel"))
    x, res, gate = gpu_like(2, 40, 40), gpu_like(2, 40, 24), gpu_like(2, 24)
    with torch.no_grad():
        for held in (x, rows8(2, 40, 40)):
            kernels.linear_tail(layer, held, "gelu_tanh")
            kernels.linear_tails([(layer, held, "gate_residual", res, gate), (layer, held, "gelu_tanh")])
        assert seen == ["gelu_tanh", "gate_residual", "gelu_tanh"] * 2 and read_rows((layer, layer))
        seen.clear()
        handle = layer.register_forward_hook(lambda m, i, o: seen.append("hook"))
        kernels.linear_tail(layer, x, "gate_residual", residual=res, gate=gate)
        assert seen == ["bias", "hook", "gate kernel"] and not read_rows((layer,))
        handle.remove()
        seen.clear()
        monkeypatch.setattr(kernels, "FUSED_LINEAR", False)
        kernels.linear_tail(layer, x, "gelu_tanh")
        assert seen == ["bias", "gelu kernel"]


@pytest.mark.parametrize("batch", [1, 2])
def test_an_8_bit_projection_writes_its_rows_of_a_shared_buffer(monkeypatch, batch):
    from hetu_dit_b200.model_executor.layers.attention_processor import _project_into
    from hetu_dit_b200.model_executor.layers.int8_linear import Int8Linear
    layer = Int8Linear(rows8(24, 40), torch.zeros(24).bfloat16())
    outs = []

    def linear_int8(x, weight, bias=None, epilogue="bias", residual=None, gate=None, out=None):
        outs.append(out)
        return torch.full((batch, x.shape[1], 24), 3.0, dtype=torch.bfloat16) if out is None else out.fill_(3.0)

    monkeypatch.setattr(kernels, "linear_int8", linear_int8)
    x, want = torch.zeros(batch, 5, 40).bfloat16(), torch.zeros(batch, 9, 24).bfloat16()
    want[:, 2:7] = 3.0
    with torch.no_grad():
        for hooks in (0, 1):  # what waits for the layer's call gets it
            buf = torch.zeros(batch, 9, 24).bfloat16()
            calls = []
            if hooks:
                layer.register_forward_hook(lambda m, i, o: calls.append(1))
            _project_into(buf, 2, x, layer)
            assert torch.equal(buf, want) and len(calls) == hooks and (outs.pop() is None) == bool(hooks)


def test_scales_of_an_8_bit_layer_keep_their_type():
    from hetu_dit_b200.model_executor.layers.int8_linear import Int8Linear
    scale = torch.rand(24)
    layer = Int8Linear(kernels.Int8Rows(torch.zeros(24, 32, dtype=torch.int8), scale), torch.zeros(24).bfloat16())
    layer.to(torch.float16)
    assert layer.weight_scale.dtype == torch.float32 and torch.equal(layer.weight_scale, scale) and layer.bias.dtype == torch.float16
    other = Int8Linear(kernels.Int8Rows(torch.zeros(24, 32, dtype=torch.int8), torch.zeros(24)), torch.zeros(24).bfloat16())
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other.weight_scale, scale)


def test_quantize_linears_replaces_plain_layers_only(monkeypatch):
    from hetu_dit_b200.model_executor.layers import int8_linear

    class Adapter(torch.nn.Linear):
        pass

    monkeypatch.setattr(kernels, "quantize_rows", lambda w: rows8(*w.shape))
    net = torch.nn.ModuleDict({"a": torch.nn.Linear(8, 16), "b": torch.nn.ModuleList([torch.nn.Linear(16, 8, bias=False), Adapter(8, 8)])})
    assert int8_linear.quantize_linears_(net) is net
    assert type(net["a"]) is int8_linear.Int8Linear and type(net["b"][0]) is int8_linear.Int8Linear and type(net["b"][1]) is Adapter
    assert net["b"][0].bias is None and (net["a"].out_features, net["a"].in_features) == (16, 8)


def test_an_attention_of_its_own_needs_no_projections():
    from hetu_dit_b200.model_executor.layers.attention_processor import JointAttnProcessor
    from hetu_dit_b200.model_executor.models import shaped_dit
    assert not shaped_dit._sees_rows(torch.nn.Identity(), JointAttnProcessor, ("to_q",))
    assert not shaped_dit._sees_rows(shaped_dit._Wrapped(torch.nn.Identity()), JointAttnProcessor, ("to_q",))


def test_steps_seen_before_layers_were_replaced_are_not_captured_or_replayed(monkeypatch):
    """A step cache that lives anywhere (a model's, a pipeline's) forgets what it holds. Its first run of a key is eager, the
    second one captures, for which it asks the step's inputs for their device: there are none here."""
    from hetu_dit_b200.model_executor.layers.int8_linear import quantize_linears_
    from hetu_dit_b200.model_executor.step_graph import StepGraphCache
    monkeypatch.setattr(kernels, "quantize_rows", lambda w: rows8(*w.shape))
    cache, runs = StepGraphCache(), []
    step = lambda: runs.append(1)  # noqa: E731
    cache.run("step", step)
    with pytest.raises(StopIteration):
        cache.run("step", step)
    net = torch.nn.ModuleList([torch.nn.ModuleList([torch.nn.Linear(8, 16)])])
    quantize_linears_(net)
    cache.run("step", step)
    assert len(runs) == 2
    quantize_linears_(net)  # nothing is left to replace: what was captured since stays
    with pytest.raises(StopIteration):
        cache.run("step", step)


def _wide_rows(B, S, k, width, unsqueezed=False):
    """Rows of k in a buffer of `width` bytes to a row; unsqueezed: the rows of a matrix, each an entry of its own."""
    q = torch.randint(-127, 128, (B, S, width), dtype=torch.int8)[..., :k]
    if unsqueezed:
        q = q[:, 0][:, None]
    return kernels.Int8Rows(q.as_subclass(OnGpu), torch.rand(B, S).as_subclass(OnGpu))


@pytest.mark.parametrize("B, S, unsqueezed", [(4, 1, False), (4, 1, True), (1, 4, False), (2, 3, False)])
def test_rows_wider_than_they_have_to_be_are_addressed_by_their_stride(lib, monkeypatch, B, S, unsqueezed):  # noqa: F811
    monkeypatch.setattr(kernels, "_cuda_index", lambda device: 0)
    x = _wide_rows(B, S, 40, 64, unsqueezed)
    kernels.linear_int8(x, rows8(24, 40), out=gpu_like(B, S, 24))
    (name, args), = lib.calls
    a = args[0]._obj
    assert (name, a.m, a.lda, a.a) == ("hdit_int8_linear", B * S, 64, x.q.data_ptr())


def _tiny_attention(joint, monkeypatch):
    from hetu_dit_b200.core.distributed import parallel_state as ps
    from hetu_dit_b200.model_executor.layers import int8_linear
    from hetu_dit_b200.model_executor.models import shaped_dit
    from tests.test_gpu_model import tiny_shape
    shape, _ = tiny_shape("flux")
    attn = shaped_dit.Attention(shape, joint=joint, out_proj=joint)
    made, products = [], []

    def quantize_rows(x):
        made.append(x)
        return rows8(*x.shape)

    def linear_int8(x, weight, bias=None, epilogue="bias", residual=None, gate=None, out=None):
        products.append(x)
        return torch.zeros(*x.shape[:-1], weight.shape[0], dtype=x.dtype) if out is None else out

    monkeypatch.setattr(kernels, "quantize_rows", quantize_rows)
    monkeypatch.setattr(kernels, "linear_int8", linear_int8)
    monkeypatch.setattr(ps, "get_sequence_parallel_world_size", lambda: 2)
    monkeypatch.setattr(attn.processor._ops, "get", lambda cls: lambda key, q, k, v, **kw: q)
    int8_linear.quantize_linears_(attn)
    made.clear()
    return shape, attn, made, products


@pytest.mark.parametrize("rows_given", [False, True])
def test_sharded_streams_are_quantised_once_for_their_projections(monkeypatch, rows_given):
    """Under sequence parallelism the projections write into the shards' buffers one by one: all of a stream read one set of rows."""
    shape, attn, made, products = _tiny_attention(True, monkeypatch)
    make = rows8 if rows_given else lambda *s: torch.zeros(*s).bfloat16()
    img, txt = make(1, 12, shape.hidden), make(1, 4, shape.hidden)
    with torch.no_grad():
        attn(img, txt, text_len=8, token_offset=12, text_offset=4)
    assert made[:2] == [] if rows_given else made[0] is img and made[1] is txt
    assert len(made) == (0 if rows_given else 2) and len(products) == 8
    assert [type(x) for x in products] == [kernels.Int8Rows] * 6 + [torch.Tensor] * 2  # the projections, then the outputs' 16-bit input
    assert len({id(x) for x in products[:6]}) == 2


@pytest.mark.parametrize("rows_given", [False, True])
def test_a_sharded_single_stream_is_quantised_once_for_its_projections(monkeypatch, rows_given):
    shape, attn, made, products = _tiny_attention(False, monkeypatch)
    x = (rows8 if rows_given else lambda *s: torch.zeros(*s).bfloat16())(1, 16, shape.hidden)
    with torch.no_grad():
        attn(x, text_len=4, token_offset=12, text_offset=4, text_total=8)
    assert len(made) == (0 if rows_given else 1) and len(products) == 3 and len({id(p) for p in products}) == 1
    assert type(products[0]) is kernels.Int8Rows


def test_norms_write_rows_under_sequence_parallelism_too(monkeypatch):
    from hetu_dit_b200.core.distributed import parallel_state as ps
    from hetu_dit_b200.model_executor.layers.attention_processor import SingleAttnProcessor
    from hetu_dit_b200.model_executor.models import shaped_dit
    shape, attn, _, _ = _tiny_attention(False, monkeypatch)
    assert ps.get_sequence_parallel_world_size() == 2
    assert shaped_dit._sees_rows(shaped_dit._Wrapped(attn), SingleAttnProcessor, ("to_q", "to_k", "to_v"))
    assert not shaped_dit._sees_rows(shaped_dit._Wrapped(attn), SingleAttnProcessor, ("to_q", "to_k", "to_v"), torch.nn.Linear(2, 2))


def test_an_8_bit_layer_refuses_a_gradient(monkeypatch):
    from hetu_dit_b200.model_executor.layers.attention_processor import _project_into
    from hetu_dit_b200.model_executor.layers.int8_linear import Int8Linear
    layer = Int8Linear(rows8(24, 40), torch.zeros(24).bfloat16())
    monkeypatch.setattr(kernels, "linear_int8", lambda x, w, b=None, epilogue="bias", residual=None, gate=None, out=None: gpu_like(*x.shape[:-1], 24))
    x, res, gate = gpu_like(1, 5, 40), gpu_like(1, 5, 24), gpu_like(1, 24)
    grad = [t.detach().clone().requires_grad_() for t in (x, res, gate)]
    calls = (lambda: layer(grad[0]), lambda: kernels.linear_tail(layer, grad[0], "gelu_tanh"),
             lambda: kernels.linear_tail(layer, x, "gate_residual", residual=grad[1], gate=gate),
             lambda: kernels.linear_tail(layer, x, "gate_residual", residual=res, gate=grad[2]),
             lambda: _project_into(torch.zeros(1, 9, 24).bfloat16(), 0, grad[0], layer))
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradients"):
            call()
    with torch.no_grad():
        for call in calls:
            call()
    layer(x), layer(rows8(1, 5, 40)), kernels.linear_tail(layer, x, "gate_residual", residual=res, gate=gate)


def test_rows_of_an_input_that_asks_for_a_gradient_are_refused(monkeypatch):
    shape, attn, made, _ = _tiny_attention(False, monkeypatch)
    x = torch.zeros(1, 16, shape.hidden).bfloat16().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        attn(x, text_len=4, token_offset=12, text_offset=4, text_total=8)


def test_a_model_in_8_bits_asks_for_no_gradients(monkeypatch):
    from hetu_dit_b200.model_executor.models.shaped_dit import ShapedDiT
    from tests.test_gpu_model import tiny_shape
    monkeypatch.setattr(kernels, "quantize_rows", lambda w: rows8(*w.shape))
    model = ShapedDiT(tiny_shape("sd3")[0])
    assert any(p.requires_grad for p in model.parameters())
    assert model.quantize_linears_() is model and not any(p.requires_grad for p in model.parameters())


def test_a_layer_that_cannot_be_in_8_bits_leaves_the_module_as_it_was(lib, monkeypatch):  # noqa: F811
    """The first layers could be converted; the last one has another type, or lies on the host."""
    from hetu_dit_b200.model_executor.layers.int8_linear import quantize_linears_
    monkeypatch.setattr(kernels, "_cuda_index", lambda device: 0)
    on_host = torch.nn.Linear(24, 8, dtype=torch.bfloat16)

    def require_cuda(*tensors):
        if any(t.shape == on_host.weight.shape or t.shape == (0, 24) for t in tensors):
            raise RuntimeError("no CPU path")

    monkeypatch.setattr(kernels, "_require_cuda", require_cuda)
    for last in (torch.nn.Linear(16, 8), on_host):
        net = torch.nn.ModuleList([torch.nn.Linear(16, 8, dtype=torch.bfloat16),
                                   torch.nn.ModuleList([torch.nn.Linear(16, 8, dtype=torch.bfloat16)]), last])
        with pytest.raises((TypeError, RuntimeError)):
            quantize_linears_(net)
        assert sum(type(m) is torch.nn.Linear for m in net.modules()) == 3
    assert lib.calls == []


def test_a_layer_that_something_was_put_on_stays(monkeypatch):
    from hetu_dit_b200.model_executor.layers import int8_linear
    from tests.test_host_dispatch import _hook, _other_weight, _own_forward, _pre_hook
    monkeypatch.setattr(kernels, "quantize_rows", lambda w: rows8(*w.shape))
    changes = [_hook, _pre_hook, _own_forward, _other_weight, lambda layer: layer.register_full_backward_hook(lambda m, a, b: None),
               lambda layer: torch.nn.utils.parametrizations.weight_norm(layer)]
    net = torch.nn.ModuleList([torch.nn.Linear(8, 8) for _ in changes] + [torch.nn.Linear(8, 8), None])
    for change, layer in zip(changes, net):
        change(layer)
    kept = list(net)[:len(changes)]
    int8_linear.quantize_linears_(net)
    assert all(a is b for a, b in zip(net, kept)) and type(net[len(changes)]) is int8_linear.Int8Linear
    # what waits for the calls of all modules waits for the 8-bit layer's, too
    net = torch.nn.ModuleList([torch.nn.Linear(8, 8)])
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, a, y: None)
    try:
        int8_linear.quantize_linears_(net)
    finally:
        handle.remove()
    assert type(net[0]) is int8_linear.Int8Linear


@pytest.mark.parametrize("n,k,width,first", [(5, 40, 96, 48), (5, 40, 96, 0), (5, 40, 48, 0), (1, 40, 40, 0), (1, 40, 64, 16), (5, 32, 96, 64), (5, 40, 88, 48),
                                             (5, 40, 88, 0), (5, 32, 40, 8)])
def test_an_8_bit_layer_of_rows_that_a_program_has_laid_out(n, k, width, first):
    """Columns of wider rows; the last ones end where the memory ends."""
    from hetu_dit_b200.model_executor.layers.int8_linear import Int8Linear
    buf = torch.randint(-127, 128, (n, width), dtype=torch.int8)
    q = buf[:, first:first + k]
    layer = Int8Linear(kernels.Int8Rows(q, torch.rand(n)))
    assert layer.weight_q.stride(0) % 16 == 0 and layer.weight_q.data_ptr() % 16 == 0
    for copied in (layer, Int8Linear(kernels.Int8Rows(torch.zeros(n, k, dtype=torch.int8), torch.zeros(n)))):
        copied.load_state_dict(layer.state_dict())
        rows = copied.rows
        assert torch.equal(rows.q, q) and rows.shape == (n, k) and torch.equal(rows.scale, layer.weight_scale)
    moved = layer.weight_q.clone()  # as a copy to another device lays it out
    assert moved.stride(0) % 16 == 0 and torch.equal(moved[:, :k], q)


def test_a_result_whose_rows_overlap_is_refused(lib, monkeypatch):  # noqa: F811
    monkeypatch.setattr(kernels, "_cuda_index", lambda device: 0)
    kw = dict(x=gpu_like(3, 40, 32), residual=gpu_like(3, 40, 24), gate=gpu_like(3, 24))
    for out in (gpu_like(1, 40, 24).expand(3, 40, 24), gpu_like(80, 24).as_strided((3, 40, 24), (20 * 24, 24, 1))):
        with pytest.raises(ValueError, match="overlap"):
            _linear(out=out, **kw)
    assert lib.calls == []
    _linear(out=gpu_like(40, 3, 24).transpose(0, 1), **kw)  # the entries' rows in turn
    assert [c[0] for c in lib.calls] == ["hdit_int8_linear"] * 3


def test_the_library_refuses_an_image_whose_rows_overlap():
    a = _C.GroupNormArgs()
    for name, v in dict(dtype=0, act=0, x=4096, out=4096, batch=3, rows=4, channels=64, groups=8, x_row_stride=64, out_batch_stride=256,
                        out_row_stride=64, eps=1e-6).items():
        setattr(a, name, v)
    for row, image in ((0, 256), (63, 256), (64, 0), (64, 255), (128, 64), (-64, 256), (64, -256)):
        a.out_row_stride, a.out_batch_stride = row, image
        assert _C.lib().hdit_group_norm(ctypes.byref(a)) == _C.HDIT_ERR_SHAPE, (row, image)


def test_a_layer_that_cannot_be_in_8_bits_leaves_all_blocks_as_they_were(monkeypatch):
    from hetu_dit_b200.model_executor.models.shaped_dit import ShapedDiT
    from tests.test_gpu_model import tiny_shape

    def quantize_rows(w):
        if w.dtype == torch.float64:
            raise TypeError("unsupported dtype")
        return rows8(*w.shape)

    monkeypatch.setattr(kernels, "quantize_rows", quantize_rows)
    model = ShapedDiT(tiny_shape("flux")[0])
    layers = sum(type(m) is torch.nn.Linear for m in model.modules())
    model.single_transformer_blocks[-1].proj_out.double()
    with pytest.raises(TypeError):
        model.quantize_linears_()
    assert sum(type(m) is torch.nn.Linear for m in model.modules()) == layers and any(p.requires_grad for p in model.parameters())
