"""Linear layers that hold their weight in 8-bit integers, for the blocks of the -shaped DiT models.

A layer's weight has one scale per output channel, made once; the rows of its input are brought into 8 bits with a scale each
when it is called (kernels.quantize_rows, kernels.ln_modulate_int8), so that no calibration is needed. The products run on
the tensor cores in 8-bit integers at twice the rate of 16-bit values and read half the weight bytes. Each step is off by at
most half a step, 1/254 of the row's or channel's largest value. Inference only. (The reference has no 8-bit path; the layers
are the torch.nn.Linear of the blocks it wraps, hetu_dit/model_executor/diffusion_executor/layers/attention_processor.py:207-449
and layers/feedforward.py:73-78.)
"""
import torch
import torch.nn as nn

from ... import kernels
from ...core.distributed import parallel_state as ps


def refuse_gradients(*tensors):
    """Raises where a gradient is recorded for one of the tensors (None and Int8Rows among them): the result would have none."""
    if torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in tensors):
        raise RuntimeError("8-bit linear layers have no gradients: run them under torch.no_grad() or on tensors that require none")


def _whole_rows(q):
    """The rows (n, k) with what lies behind each up to the next 16-byte boundary, so that a copy of them keeps the rows on such
    boundaries: the same memory, or a copy where the rows are not on such boundaries or the memory ends before the last one's."""
    n, k = q.shape
    width = (k + 15) & ~15
    pitch = q.stride(0) if n > 1 else width
    if pitch % 16 == 0 and pitch >= width and q.data_ptr() % 16 == 0 and \
            q.storage_offset() + (n - 1) * pitch + width <= q.untyped_storage().nbytes():
        return q.as_strided((n, width), (pitch, 1))
    whole = q.new_zeros(n, width)
    whole[:, :k] = q
    return whole


class Int8Linear(nn.Module):
    """x @ weight.T + bias with the weight in 8 bits, in place of a torch.nn.Linear. x: a 16-bit tensor that no gradient is
    recorded for, or kernels.Int8Rows."""

    def __init__(self, weight: kernels.Int8Rows, bias=None):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        self.register_buffer("weight_q", _whole_rows(weight.q))
        self.register_buffer("weight_scale", weight.scale)
        self.register_buffer("bias", None if bias is None else bias.detach().clone())
        self.dtype = weight.dtype

    @classmethod
    def from_linear(cls, linear: nn.Linear):
        """The layer of a 16-bit torch.nn.Linear on the GPU."""
        return cls(kernels.quantize_rows(linear.weight.detach()), linear.bias)

    @property
    def rows(self):
        """The weight as kernels.linear_int8() takes it."""
        q = self.weight_q
        return kernels.Int8Rows(q if q.shape[1] == self.in_features else q[:, :self.in_features], self.weight_scale, self.dtype)

    def _apply(self, fn, recurse=True):
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != scale.dtype:  # a change of the 16-bit type is not one of the scales' type
            self.weight_scale = scale.to(self.weight_scale.device)
        return self

    def forward(self, x):
        refuse_gradients(x)
        return kernels.linear_int8(x, self.rows, self.bias)

    def with_tail(self, x, epilogue, residual=None, gate=None, out=None):
        """kernels.linear_tail() of this layer, or the layer alone ("bias"), in one launch (two with 16-bit x)."""
        refuse_gradients(x, residual, gate)
        return kernels.linear_int8(x, self.rows, self.bias, epilogue, residual=residual, gate=gate, out=out)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


def read_rows(linears):
    """Whether all that reads an input are 8-bit layers that nothing waits for the call of: they may be given Int8Rows, made
    once, in its place."""
    for layer in linears:
        if not kernels.is_plain(layer, Int8Linear):
            return False
    return True


def _replaceable(layer):
    """Whether a layer is a torch.nn.Linear that nothing was put on: a hook, a forward() or a weight of a class of its own would go
    with the layer."""
    own = layer.__dict__
    return type(layer) is nn.Linear and type(layer.weight) is nn.Parameter and "forward" not in own and \
        not (own["_forward_hooks"] or own["_forward_pre_hooks"] or own["_backward_hooks"] or own["_backward_pre_hooks"])


def _places(module):
    """(parent, name) of every layer below `module` that is to be replaced."""
    return [(parent, name) for parent in module.modules() for name, child in parent._modules.items() if child is not None and _replaceable(child)]


@torch.no_grad()
def quantize_linears_(module: nn.Module):
    """Puts an Int8Linear in the place of every torch.nn.Linear below `module` (16-bit, on the GPU); returns module. What has
    another class (an adapter), and a layer with a hook, a forward() or a weight of a class of its own, stays. A layer that
    cannot be brought into 8 bits (another type, another device) raises before any is replaced. Steps captured in CUDA graphs
    before hold the addresses of the 16-bit weights: those of every StepGraphCache are dropped. Block caches address
    torch.nn.Linear weights by name: a module whose slices migrate between plans keeps them."""
    places = _places(module)
    for parent, name in places:
        kernels.quantize_rows(parent._modules[name].weight.detach()[:0])  # all that it asks of a weight, and nothing launched
    try:
        for parent, name in places:  # one by one: its 16-bit weight goes before the next one's 8-bit copy comes
            setattr(parent, name, Int8Linear.from_linear(parent._modules[name]))
    finally:
        if places and ps.model_parallel_is_initialized():
            ps.get_parallel_groups().void_captured_graphs()
    return module
