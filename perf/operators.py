"""Operators of an 8-bit inference path, as cases to be timed: linear layers over rows and weights held in 8-bit integers,
and the norms that feed them.

Kinds (x: 16-bit rows, q: 8-bit integers, s: fp32 scales):

linear      x -> rows in 8 bits, each with a scale of its own (s = max|x| / 127, q = x / s to the nearest integer, ties to
            even); then tail((q_x . q_w) s_x s_w + bias) against weights held in 8 bits with a scale for each output channel.
            tail: "bias" (nothing more), "gelu_tanh", "gate_residual" (residual + gate of the batch entry * value)
norm_linear LayerNorm(x) (1 + scale) + shift of the batch entry, its rows in 8 bits, then the product as above
group_norm  GroupNorm over a channels-last image with an activation
group_linear GroupNorm (no activation), its rows (all channels of a pixel) in 8 bits, then the product as above

Activations are N(0, 1) with a few channels eight times as large, weights N(0, 0.02), all made from the seed.
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # adaLN vectors of one image: one row against a whole weight matrix, the smallest linear layer of a step
        {"name": "linear_one_row", "kind": "linear", "batch": 1, "rows": 1, "k": 1536, "n": 9216, "tail": "bias",
         "bias": True, "dtype": "bf16"},
        # prompt features of one image into the model's width, an odd number of tokens
        {"name": "linear_text", "kind": "linear", "batch": 1, "rows": 333, "k": 4096, "n": 1536, "tail": "bias",
         "bias": True, "dtype": "fp16"},
        # MLP, second layer, of a 1024 x 1024 image with both guidance halves in the batch
        {"name": "linear_gate_4096", "kind": "linear", "batch": 2, "rows": 4096, "k": 6144, "n": 1536,
         "tail": "gate_residual", "bias": True, "dtype": "fp16"},
        # output projection of a single-stream block, a small image of an odd aspect ratio
        {"name": "linear_gate_ragged", "kind": "linear", "batch": 1, "rows": 2192, "k": 15360, "n": 3072,
         "tail": "gate_residual", "bias": True, "dtype": "bf16"},
        # MLP, first layer, of a 1024 x 1024 image with its prompt: the largest linear layer of a step
        {"name": "linear_gelu_4608", "kind": "linear", "batch": 1, "rows": 4608, "k": 3072, "n": 12288,
         "tail": "gelu_tanh", "bias": True, "dtype": "bf16"},
        # text stream of a short prompt, both guidance halves: norm, modulation, MLP's first layer
        {"name": "norm_linear_text", "kind": "norm_linear", "batch": 2, "rows": 77, "k": 1536, "n": 6144,
         "tail": "gelu_tanh", "bias": True, "dtype": "bf16"},
        # image stream of both halves: norm, modulation, Q, K and V as one layer
        {"name": "norm_linear_4096", "kind": "norm_linear", "batch": 2, "rows": 4096, "k": 1536, "n": 4608,
         "tail": "bias", "bias": True, "dtype": "bf16"},
        # first residual block of an image decoder (512 x 512 image, 8 x smaller latents)
        {"name": "group_norm_64", "kind": "group_norm", "batch": 1, "height": 64, "width": 64, "channels": 512,
         "groups": 32, "act": "silu", "dtype": "bf16"},
        # an odd image in the middle of the decoder, two images, channels that do not fill a vector per group
        {"name": "group_norm_odd", "kind": "group_norm", "batch": 2, "height": 117, "width": 203, "channels": 320,
         "groups": 32, "act": "silu", "dtype": "fp16"},
        # last residual block of the decoder at full resolution: larger than the caches
        {"name": "group_norm_1024", "kind": "group_norm", "batch": 1, "height": 1024, "width": 1024, "channels": 128,
         "groups": 32, "act": "silu", "dtype": "bf16"},
        # norm and projection around the attention of a small feature map
        {"name": "group_linear_32", "kind": "group_linear", "batch": 2, "height": 32, "width": 32, "channels": 640,
         "groups": 32, "n": 640, "tail": "bias", "bias": True, "dtype": "fp16"},
        # the same in the middle of a decoder: a 1024 x 1024 image, Q, K and V as one layer
        {"name": "group_linear_128", "kind": "group_linear", "batch": 1, "height": 128, "width": 128, "channels": 512,
         "groups": 32, "n": 1536, "tail": "bias", "bias": True, "dtype": "bf16"},
    ]


_LARGEST = 4608 * 3072 * 12288  # multiply-adds of the largest listed layer


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    kind = rng.choice(["linear", "linear", "linear", "norm_linear", "group_norm", "group_norm", "group_linear"])
    case = {"kind": kind, "batch": rng.randint(1, 3), "dtype": rng.choice(["bf16", "fp16"])}
    if kind in ("linear", "norm_linear"):
        case["k"] = log_int(64, 15360) if kind == "linear" else 8 * log_int(8, 768)
        case["n"] = log_int(64, 12288)
        most = min(8192 // case["batch"], _LARGEST // (case["k"] * case["n"] * case["batch"]))
        case["rows"] = log_int(1, most)
        case["tail"] = rng.choice(["bias", "gelu_tanh", "gate_residual"])
        case["bias"] = rng.random() < 0.75
        return case
    case["groups"] = rng.choice([8, 16, 32, 32])
    case["channels"] = case["groups"] * rng.randint(1, 32)
    case["channels"] += -case["channels"] % 8
    most = 1024 * 1024 * 128 // (case["channels"] * case["batch"])
    case["height"] = log_int(1, min(1024, most))
    case["width"] = log_int(1, min(1024, most // case["height"]))
    if kind == "group_norm":
        case["act"] = rng.choice(["silu", "silu", "none"])
        return case
    case["height"], case["width"] = min(case["height"], 160), min(case["width"], 160)
    case["n"] = log_int(64, 2048)
    case["tail"], case["bias"] = rng.choice(["bias", "gelu_tanh"]), rng.random() < 0.75
    return case


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _activations(gen, *shape):
    """N(0, 1), a few of the channels (the last dimension) eight times as large."""
    large = torch.rand(shape[-1], generator=gen, device=DEV) < 0.01
    return _randn(gen, *shape) * torch.where(large, 8.0, 1.0)


def _weight(gen, n, k):
    """A weight matrix as a program holds it in 8 bits: integers, each row on a 16-byte boundary, and a scale for each
    output channel."""
    w = _randn(gen, n, k) * 0.02
    scale = w.abs().amax(dim=1) / 127
    q = torch.zeros(n, k + -k % 16, dtype=torch.int8, device=DEV)[:, :k]
    q.copy_(torch.round(w / scale[:, None]))
    return q, scale


def prepare(case, seed):
    gen, dtype, kind, batch = _gen(seed), DTYPES[case["dtype"]], case["kind"], case["batch"]
    state = {"case": case}
    if kind in ("group_norm", "group_linear"):
        c, k = case["channels"], case["channels"]
        # what a convolution leaves: channels with means and deviations of their own; channels last in memory
        x = _randn(gen, batch, case["height"], case["width"], c)
        x.mul_(torch.rand(c, generator=gen, device=DEV) * 1.5 + 0.5).add_(_randn(gen, c))
        state["x"] = x.to(dtype).permute(0, 3, 1, 2)
        state["norm_weight"], state["norm_bias"] = (1 + 0.2 * _randn(gen, c)).to(dtype), (0.2 * _randn(gen, c)).to(dtype)
        rows = case["height"] * case["width"]
    else:
        k, rows = case["k"], case["rows"]
        state["x"] = _activations(gen, batch, rows, k).to(dtype)
        if kind == "norm_linear":
            state["shift"], state["scale"] = (0.3 * _randn(gen, 2, batch, k)).to(dtype).unbind(0)
    if kind != "group_norm":
        n = case["n"]
        state["w"], state["w_scale"] = _weight(gen, n, k)
        state["bias"] = (0.1 * _randn(gen, n)).to(dtype) if case["bias"] else None
        if case["tail"] == "gate_residual":
            state["residual"] = _randn(gen, batch, rows, n).to(dtype)
            state["gate"] = (0.5 * _randn(gen, batch, n)).to(dtype)
    return state


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


def _run_own(state):
    from hetu_dit_b200 import kernels
    case, x = state["case"], state["x"]
    kind = case["kind"]
    if kind == "group_norm":
        return kernels.group_norm(x, case["groups"], state["norm_weight"], state["norm_bias"], eps=1e-6,
                                  act=None if case["act"] == "none" else case["act"])
    if kind == "norm_linear":
        x = kernels.ln_modulate_int8(x, state["shift"], state["scale"], eps=1e-6)
    elif kind == "group_linear":
        x = kernels.group_norm_int8(x, case["groups"], state["norm_weight"], state["norm_bias"], eps=1e-6)
    return kernels.linear_int8(x, kernels.Int8Rows(state["w"], state["w_scale"]), state["bias"], case["tail"],
                               residual=state.get("residual"), gate=state.get("gate"))


# ---- plain form -----------------------------------------------------------------------------------------------------

def _rows_in_8_bits(y):
    """(integers as fp32, scale) of the rows of y; the quotient in 64 bits, where it may lie next to a border."""
    y = y.double()
    top = y.abs().amax(dim=-1, keepdim=True)
    q = torch.round(127 * y / torch.where(top == 0, 1.0, top))
    return q.float(), (top / 127).float()


def _plain_norm(state):
    """GroupNorm of the (B, C, H, W) image as rows (B, H W, C), fp32 with statistics in 64 bits."""
    case, x = state["case"], state["x"]
    b, c, h, w = x.shape
    y = x.permute(0, 2, 3, 1).reshape(b, h * w, case["groups"], c // case["groups"])
    mean = y.mean(dim=(1, 3), keepdim=True, dtype=torch.float64)
    var = torch.square(y.double() - mean).mean(dim=(1, 3), keepdim=True)
    a = (var + 1e-6).rsqrt()
    y = ((y.double() - mean) * a).float().reshape(b, h * w, c)
    return y * state["norm_weight"].float() + state["norm_bias"].float()


def _run_plain(state):
    case, x = state["case"], state["x"]
    kind, dtype = case["kind"], state["x"].dtype
    if kind == "group_norm":
        y = _plain_norm(state)
        if case["act"] == "silu":
            y = y / (1 + torch.exp(-y))
        return y.to(dtype).reshape(x.shape[0], x.shape[2], x.shape[3], x.shape[1]).permute(0, 3, 1, 2)
    if kind == "norm_linear":
        y = x.double()
        y = y - y.mean(dim=-1, keepdim=True)
        y = y * (torch.square(y).mean(dim=-1, keepdim=True) + 1e-6).rsqrt()
        y = y * (1 + state["scale"].double()[:, None]) + state["shift"].double()[:, None]
    elif kind == "group_linear":
        y = _plain_norm(state)
    else:
        y = x
    q, s = _rows_in_8_bits(y)
    y = torch.matmul(q, state["w"].float().t()) * (s * state["w_scale"])
    if state["bias"] is not None:
        y = y + state["bias"].float()
    if case["tail"] == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    elif case["tail"] == "gate_residual":
        y = state["residual"].float() + state["gate"].float()[:, None] * y
    return y.to(dtype)


# ---- work and definition --------------------------------------------------------------------------------------------

def work(case):
    kind, b = case["kind"], case["batch"]
    if kind in ("group_norm", "group_linear"):
        rows, k = case["height"] * case["width"], case["channels"]
        elems = b * rows * k
        if kind == "group_norm":
            return {"bytes": 4 * elems + 4 * k, "flops": 10 * elems}
    else:
        rows, k = case["rows"], case["k"]
    m, n = b * rows, case["n"]
    elems = m * n * (2 if case["tail"] == "gate_residual" else 1)
    read = 2 * m * k + n * k + 4 * n + (2 * n if case["bias"] else 0) + (2 * b * n if case["tail"] == "gate_residual" else 0)
    read += 4 * b * k if kind == "norm_linear" else 4 * k if kind == "group_linear" else 0
    return {"bytes": read + 2 * elems, "flops": 2 * m * n * k + 4 * m * k}


def exact(case, seed):
    s = prepare(case, seed)
    f = {name: t.to(torch.float64) for name, t in s.items() if isinstance(t, torch.Tensor)}
    x = f["x"]
    if "norm_weight" in f:
        b, c, h, w = x.shape
        g = case["groups"]
        x = x.reshape(b, g, c // g, h, w)
        var, mean = torch.var_mean(x, dim=(2, 3, 4), correction=0, keepdim=True)
        x = ((x - mean) / torch.sqrt(var + 1e-6)).reshape(b, c, h, w)
        x = x * f["norm_weight"].view(1, c, 1, 1) + f["norm_bias"].view(1, c, 1, 1)
        if case["kind"] == "group_norm":
            return x * torch.sigmoid(x) if case["act"] == "silu" else x
        x = x.flatten(2).transpose(1, 2)
    elif "shift" in f:
        var, mean = torch.var_mean(x, dim=2, correction=0, keepdim=True)
        x = (x - mean) / torch.sqrt(var + 1e-6) * (1 + f["scale"].unsqueeze(1)) + f["shift"].unsqueeze(1)
    step = x.abs().max(dim=2, keepdim=True).values / 127
    held = torch.where(step > 0, torch.round(x / step), 0.0) * step
    y = torch.einsum("bmk,nk->bmn", held, f["w"] * f["w_scale"].unsqueeze(1))
    if "bias" in f:
        y = y + f["bias"]
    if case["tail"] == "gelu_tanh":
        y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    if case["tail"] == "gate_residual":
        y = f["residual"] + f["gate"].unsqueeze(1) * y
    return y
