"""GPU parity of the 8-bit rows, the linear layer over them and the group norm against their definitions in 64 bits.

Every tolerance is the sum of the roundings on the way: half a unit of the 16-bit result, and for each fp32 operation 2^-24 of
its result, carried through what follows."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16]
ids = {torch.bfloat16: "bf16", torch.float16: "fp16"}.get


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    from hetu_dit_b200 import _C
    torch.cuda.synchronize()
    assert _C.device_status(0, clear=True)[0] == 0


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device=DEV).to(dtype)


def _half_step(want, dtype):
    """Half a unit in the last place of a rounding to `dtype`, subnormal numbers included."""
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return torch.finfo(dtype).eps / 2 * want.abs() + tiny


def _within(got, want, tol):
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float((got.double() - want).abs().max()), float(tol.min()))


# ---------------------------------------------------------------------------------------------------------- rows

def _rows64(x):
    top = x.double().abs().amax(-1, keepdim=True)
    q = torch.round(127 * x.double() / torch.where(top > 0, top, 1.0))
    return q.to(torch.int8), (top / 127).float()[..., 0]  # fp32 / 127 would be fp32 * fp32(1 / 127) here


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows", [1, 7, 9, 333])
@pytest.mark.parametrize("k", [1, 7, 8, 17, 255, 256, 264, 777, 1024, 1536, 2000, 3001, 4096, 6144, 8192, 12000, 16384, 16385, 20000])
def test_quantize_rows_is_exact(k, rows, dtype):
    from hetu_dit_b200 import kernels
    x = _randn(_gen(k + rows), rows, k, dtype=dtype)
    got = kernels.quantize_rows(x)
    q, s = _rows64(x)
    assert torch.equal(got.q, q) and torch.equal(got.scale, s) and got.dtype == dtype
    assert got.q.data_ptr() % 16 == 0 and got.q.stride(0) % 16 == 0


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_quantize_rows_at_every_border(dtype):
    """Every 16-bit magnitude up to the row's largest one, for several largest ones: quotients that are n + 1/2 exactly and
    the nearest ones to it are all among them."""
    from hetu_dit_b200 import kernels
    every = torch.arange(0x8000, device=DEV, dtype=torch.int32).to(torch.int16).view(dtype)
    every = every[torch.isfinite(every)]
    for top in (1.0, 127.0, 254.0, 1.9921875, 3.0, 0.15625, 101.0, 2.0 ** -14):
        row = every[every <= top]
        x = torch.stack([torch.cat([row, row.new_tensor([top])]), -torch.cat([row, row.new_tensor([top])])])
        got = kernels.quantize_rows(x)
        q, s = _rows64(x)
        assert torch.equal(got.q, q) and torch.equal(got.scale, s), top


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_quantize_rows_strides_batches_and_what_lies_behind(dtype):
    from hetu_dit_b200 import kernels
    gen = _gen(3)
    wide = _randn(gen, 3, 50, 400, dtype=dtype)
    for view in (wide[:, 5:29, 8:208], wide[:, 5:29, 3:204], wide[1:2, :, 1:], wide.transpose(0, 1)[:, :, :64], wide[0, ::3, 16:]):
        got = kernels.quantize_rows(view)
        q, s = _rows64(view)
        assert got.q.shape == view.shape and torch.equal(got.q, q) and torch.equal(got.scale, s)
    assert kernels.quantize_rows(wide[:, :0]).q.shape == (3, 0, 400)
    # one value repeated along a row of stride 0
    same = wide[:1, :1, :40].expand(2, 6, 40)
    assert torch.equal(kernels.quantize_rows(same).q, _rows64(same)[0])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("k", [1, 2, 5, 7, 8, 9, 13, 16, 31, 250, 1001, 2050, 5003, 9001])
def test_rows_that_start_anywhere(k, dtype):
    """What stands before, between and behind the rows is larger than they are and must not be seen."""
    from hetu_dit_b200 import kernels
    rows = 5
    want = _randn(_gen(k), rows, k, dtype=dtype)
    q, s = _rows64(want)
    for off in range(9):
        for pitch in (k, k + 1, k + 6):
            flat = torch.full((off + rows * pitch + 3,), float("inf"), dtype=dtype, device=DEV)
            x = flat[off:off + rows * pitch].view(rows, pitch)[:, :k]
            x.copy_(want)
            got = kernels.quantize_rows(x)
            assert torch.equal(got.q, q) and torch.equal(got.scale, s)
    exact = torch.empty(rows * k, dtype=dtype, device=DEV).view(rows, k).copy_(want)  # nothing before or behind it
    assert torch.equal(kernels.quantize_rows(exact).q, q)


def test_bytes_behind_a_row_stay():
    from hetu_dit_b200 import _C
    x = _randn(_gen(5), 9, 77, dtype=torch.bfloat16)
    q = torch.full((11, 96), 55, dtype=torch.int8, device=DEV)
    s = torch.full((11,), 7.0, device=DEV)
    _C.check(_C.lib().hdit_quantize_rows(0, x.data_ptr(), q.data_ptr(), s.data_ptr(), 9, 77, 9, 0, 77, 96,
                                         torch.cuda.current_stream().cuda_stream))
    assert torch.equal(q[:9, :77], _rows64(x)[0])
    assert (q[:9, 77:] == 55).all() and (q[9:] == 55).all() and (s[9:] == 7).all()


@pytest.mark.parametrize("k", [40, 1000, 20000])
def test_rows_of_nothing_and_of_no_number(k):
    from hetu_dit_b200 import kernels
    x = _randn(_gen(k), 8, k, dtype=torch.bfloat16)
    x[1] = 0
    x[2, k // 2], x[3, 0], x[4, k - 1] = float("nan"), float("inf"), -float("inf")
    x[5] = 2.0 ** -101
    x[6] *= 2.0 ** 119
    x[7] *= 2.0 ** -95
    got = kernels.quantize_rows(x)
    for r in (0, 6, 7):
        q, s = _rows64(x[r:r + 1])
        assert torch.equal(got.q[r:r + 1], q) and torch.equal(got.scale[r:r + 1], s)
    assert (got.q[1:6] == 0).all()
    assert got.scale[1] == 0 and got.scale[5] == 0 and torch.isnan(got.scale[2:5]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("B,S,dim", [(1, 1, 8), (2, 3, 64), (2, 77, 1536), (1, 40, 264), (3, 9, 2048), (1, 130, 3000), (2, 5, 4096), (1, 33, 8192)])
def test_ln_modulate_int8(B, S, dim, dtype):
    from hetu_dit_b200 import kernels
    gen = _gen(B * S + dim)
    x = (torch.randn(B, S, dim, generator=gen, device=DEV) * 3 + 1.5).to(dtype)
    mod = _randn(gen, B, 6 * dim, dtype=dtype)
    shift, scale = mod[:, dim:2 * dim], mod[:, 4 * dim:5 * dim]
    got = kernels.ln_modulate_int8(x, shift, scale, eps=1e-6)
    X = x.double()
    mean, var = X.mean(-1, keepdim=True), X.var(-1, correction=0, keepdim=True)
    z = (X - mean) / torch.sqrt(var + 1e-6)
    g, h = 1 + scale.double()[:, None], shift.double()[:, None]
    want = z * g + h
    # sums: at most 64 terms one after the other in a thread and 8 levels above: 72 * 2^-24 of the sum of magnitudes
    u = 2.0 ** -24
    d_mean = 72 * u * X.abs().mean(-1, keepdim=True) / torch.sqrt(var + 1e-6)
    off = g.abs() * (d_mean + z.abs() * (72 * u + d_mean ** 2 + 6 * u)) + 3 * u * (want.abs() + h.abs() + (z * g).abs())
    top = want.abs().amax(-1)
    assert ((got.scale.double() - top / 127).abs() <= off.amax(-1) / 127 + 2 * u * top / 127).all()
    _within(got.q.double() * got.scale.double()[..., None], want, off + got.scale.double()[..., None] * (0.5 + 127 * 4 * u))
    assert (got.q.abs().amax(-1) == 127).all()


def test_ln_modulate_int8_strides_and_no_numbers():
    from hetu_dit_b200 import kernels
    gen = _gen(8)
    wide = _randn(gen, 2, 40, 600, dtype=torch.bfloat16)
    sh, sc = _randn(gen, 2, 512, dtype=torch.bfloat16), _randn(gen, 2, 512, dtype=torch.bfloat16)
    for view in (wide[:, 3:20, 8:520], wide[:, 3:20, 5:517], wide[:, ::2, :512]):
        a, b = kernels.ln_modulate_int8(view, sh, sc), kernels.ln_modulate_int8(view.contiguous(), sh, sc)
        assert torch.equal(a.q, b.q) and torch.equal(a.scale, b.scale)
    x = wide[:, :4, :512].contiguous()
    x[0, 1, 3], x[1, 2, 500] = float("inf"), float("nan")
    got = kernels.ln_modulate_int8(x, sh, sc)
    assert torch.isnan(got.scale[0, 1]) and torch.isnan(got.scale[1, 2]) and int(torch.isnan(got.scale).sum()) == 2
    assert (got.q[0, 1] == 0).all()
    assert kernels.ln_modulate_int8(x[:, :0], sh, sc).q.shape == (2, 0, 512)


# -------------------------------------------------------------------------------------------------------- product

def _tail64(x8, w8, bias, epilogue, residual, gate, dtype):
    """(result, tolerance) of the layer over these 8-bit rows: (B, S, K) and (N, K)."""
    u = 2.0 ** -24
    p = torch.matmul(x8.q.double(), w8.q.double().t()) * x8.scale.double()[..., None] * w8.scale.double()
    v = p if bias is None else p + bias.double()
    off = 4 * u * p.abs() + u * v.abs()  # to fp32, two scales; then the sum
    if epilogue == "gelu_tanh":
        inner = math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
        want = 0.5 * v * (1 + torch.tanh(inner))
        # tanh.approx is within 2^-11 of its result; the argument is off by a few roundings, the slope of GELU below 1.13
        off = 1.13 * off + 0.5 * v.abs() * (2.0 ** -11 * torch.tanh(inner).abs() + 8 * u) + 4 * u * want.abs()
    elif epilogue == "gate_residual":
        g = gate.double()[:, None]
        want = residual.double() + g * v
        off = g.abs() * off + u * want.abs()
    else:
        want = v
    return want, off * (1 + torch.finfo(dtype).eps) + _half_step(want, dtype)


def _layer(B, S, K, N, dtype, seed):
    from hetu_dit_b200 import kernels
    gen = _gen(seed)
    x = _randn(gen, B, S, K, dtype=dtype)
    w = kernels.quantize_rows((torch.randn(N, K, generator=gen, device=DEV) / K ** 0.5).to(dtype))
    return (x, w, _randn(gen, N, dtype=dtype), _randn(gen, B, S, N, dtype=dtype), _randn(gen, B, N, dtype=dtype))


EPILOGUES = ["bias", "gelu_tanh", "gate_residual"]
SHAPES = [(1, 1, 1, 1), (1, 1, 64, 64), (1, 2, 1536, 9216), (2, 1, 512, 96), (3, 5, 33, 17), (1, 16, 640, 1000), (4, 9, 300, 200),
          (1, 127, 128, 128), (2, 129, 129, 200), (1, 300, 1000, 264), (1, 257, 4160, 1001), (7, 31, 256, 520), (1, 1300, 192, 776)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("epilogue", EPILOGUES)
@pytest.mark.parametrize("B,S,K,N", SHAPES)
def test_linear_int8(B, S, K, N, epilogue, dtype):
    from hetu_dit_b200 import kernels
    x, w, b, res, gate = _layer(B, S, K, N, dtype, B + S + K + N)
    x8 = kernels.quantize_rows(x)
    want, tol = _tail64(x8, w, b, epilogue, res, gate, dtype)
    a = kernels.linear_int8(x8, w, b, epilogue, residual=res, gate=gate)
    assert a.dtype == dtype and a.shape == (B, S, N)
    _within(a, want, tol)
    assert torch.equal(a, kernels.linear_int8(x, w, b, epilogue, residual=res, gate=gate))  # 16-bit rows: the same
    want, tol = _tail64(x8, w, None, epilogue, res, gate, dtype)
    _within(kernels.linear_int8(x8, w, None, epilogue, residual=res, gate=gate), want, tol)


@pytest.mark.parametrize("tile", [1, 2, 3, 4])
@pytest.mark.parametrize("epilogue", EPILOGUES)
@pytest.mark.parametrize("B,S,K,N", [(1, 40, 96, 72), (2, 333, 1160, 1032), (5, 70, 256, 520), (1, 600, 2500, 333)])
def test_every_tile_gives_the_same_bits(B, S, K, N, epilogue, tile):
    """The sums are exact and the tail runs in one order: every tile shape and number of CTAs gives the same result."""
    from hetu_dit_b200 import kernels
    x, w, b, res, gate = _layer(B, S, K, N, torch.bfloat16, S + N)
    x8 = kernels.quantize_rows(x)
    want, tol = _tail64(x8, w, b, epilogue, res, gate, torch.bfloat16)
    first = kernels.linear_int8(x8, w, b, epilogue, residual=res, gate=gate)
    _within(first, want, tol)
    for ctas in (0, 2, 3, 5):
        assert torch.equal(first, kernels.linear_int8(x8, w, b, epilogue, residual=res, gate=gate, tile=tile, max_ctas=ctas))


@pytest.mark.parametrize("epilogue", EPILOGUES)
@pytest.mark.parametrize("B,S,K,N", [(1, 1, 1536, 4608), (2, 1, 72, 40), (1, 3, 1000, 17), (2, 2, 4096, 160), (1, 5, 63, 100), (1, 8, 65, 33),
                                     (7, 1, 700, 264), (2, 4, 2048, 96), (1, 8, 520, 1001), (1, 4, 20000, 50), (1, 2, 70000, 20)])
def test_few_rows_give_the_bits_of_a_tile(B, S, K, N, epilogue):
    from hetu_dit_b200 import kernels
    x, w, b, res, gate = _layer(B, S, K, N, torch.float16, S + N)
    x8 = kernels.quantize_rows(x)
    tile = kernels.linear_int8(x8, w, b, epilogue, residual=res, gate=gate, tile=1)
    want, tol = _tail64(x8, w, b, epilogue, res, gate, torch.float16)
    _within(tile, want, tol)
    for rows in (x, x8):
        assert torch.equal(tile, kernels.linear_int8(rows, w, b, epilogue, residual=res, gate=gate, tile=5))


@pytest.mark.parametrize("B,S,K", [(1, 3, 8), (3, 1, 2048), (1, 4, 2048), (2, 3, 1365), (5, 1, 1637), (1, 7, 999), (2, 4, 1024), (4, 2, 1025), (1, 8, 1)])
def test_a_few_16_bit_rows_are_the_rows_in_8_bits(B, S, K):
    """Up to 8192 elements the kernel brings them into 8 bits by itself, a row to some of its warps; one row without a number."""
    from hetu_dit_b200 import kernels
    x, w, b, res, gate = _layer(B, S, K, 75, torch.bfloat16, K)
    wide = torch.full((B, S + 1, K + 3), float("inf"), dtype=torch.bfloat16, device=DEV)
    wide[:, :S, 3:] = x
    for rows in (x, wide[:, :S, 3:]):
        want = kernels.linear_int8(kernels.quantize_rows(x), w, b, "gate_residual", residual=res, gate=gate, tile=1)
        assert torch.equal(want, kernels.linear_int8(rows, w, b, "gate_residual", residual=res, gate=gate))
    x[-1, 1 if S > 1 else 0, K // 2] = float("nan")
    got = kernels.linear_int8(x, w, b)
    want = kernels.linear_int8(kernels.quantize_rows(x), w, b, tile=1)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num()) and torch.isnan(got).sum() == 75


@pytest.mark.parametrize("B,S", [(1, 1), (2, 1), (1, 2), (1, 5), (1, 40)])
def test_result_in_the_place_of_x(B, S):
    """x = residual = out: a block's residual written over its input."""
    from hetu_dit_b200 import kernels
    x, w, b, _, gate = _layer(B, S, 4096, 4096, torch.bfloat16, 50 + S)
    want = kernels.linear_int8(x, w, b, "gate_residual", residual=x, gate=gate)
    for _ in range(20):
        y = x.clone()
        assert kernels.linear_int8(y, w, b, "gate_residual", residual=y, gate=gate, out=y) is y
        assert torch.equal(y, want)
    wide = torch.zeros(B, S, 5000, dtype=torch.bfloat16, device=DEV)
    wide[..., 8:4104] = x
    out = wide[..., 904:]
    kernels.linear_int8(wide[..., 8:4104], w, b, out=out)  # the result over a part of x
    assert torch.equal(out, kernels.linear_int8(x, w, b))


def test_linear_int8_sums_are_exact_at_the_largest_k():
    """Rows of the largest and smallest integers only: a sum of 127 * 127 * 131072 fits 32 bits."""
    from hetu_dit_b200 import kernels
    K = 131072
    for S in (3, 200):
        q = torch.full((1, S, K), 127, dtype=torch.int8, device=DEV)
        q[0, 1] = -127
        wq = torch.full((72, K), 127, dtype=torch.int8, device=DEV)
        wq[5] = -127
        x8 = kernels.Int8Rows(q, torch.full((1, S), 2.0 ** -20, device=DEV))
        w8 = kernels.Int8Rows(wq, torch.full((72,), 2.0 ** -11, device=DEV))
        want, tol = _tail64(x8, w8, None, "bias", None, None, torch.bfloat16)
        _within(kernels.linear_int8(x8, w8), want, tol)


@pytest.mark.parametrize("tile", [1, 4])
@pytest.mark.parametrize("epilogue", ["bias", "gate_residual"])
@pytest.mark.parametrize("N", [1, 2, 3, 30, 31, 32, 33, 34, 63, 65, 97, 130, 259])
def test_results_and_residuals_that_start_anywhere(N, epilogue, tile):
    """Columns at any offset of rows of any pitch: the bits of the aligned form, and everything around stays."""
    from hetu_dit_b200 import kernels
    B, S, K = 2, 70, 96
    x, w, b, res, gate = _layer(B, S, K, N, torch.bfloat16, N)
    x8 = kernels.quantize_rows(x)
    want, tol = _tail64(x8, w, b, epilogue, res, gate, torch.bfloat16)
    pad = torch.zeros(B, S, (N + 7) // 8 * 8, dtype=torch.bfloat16, device=DEV)
    pad[..., :N] = res
    first = torch.empty_like(pad)
    kernels.linear_int8(x8, w, b, epilogue, residual=pad[..., :N], gate=gate, out=first[..., :N], tile=tile)
    _within(first[..., :N], want, tol)
    for pitch in (N + 7, N + 8, N + 10):
        for off, res_off in ((0, 1), (1, 0), (3, 3), (4, 6), (6, 7)):
            wide = torch.full((B, S, pitch), 7.0, dtype=torch.bfloat16, device=DEV)
            wide_res = torch.full((B, S, pitch), float("nan"), dtype=torch.bfloat16, device=DEV)
            wide_res[..., res_off:res_off + N] = res
            kernels.linear_int8(x8, w, b, epilogue, residual=wide_res[..., res_off:res_off + N], gate=gate, out=wide[..., off:off + N], tile=tile)
            assert torch.equal(wide[..., off:off + N], first[..., :N])
            assert (wide[..., :off] == 7).all() and (wide[..., off + N:] == 7).all()


@pytest.mark.parametrize("tile", [0, 1, 2, 3, 4, 5])
@pytest.mark.parametrize("K", [1, 7, 15, 17, 33, 100, 127, 129, 250, 1001])
def test_bytes_behind_8_bit_rows_are_not_summed(K, tile):
    from hetu_dit_b200 import kernels
    S, N = (6, 70) if tile in (0, 5) else (140, 300)
    gen, rows = _gen(K), []
    for n in (S, N):
        q = torch.full((n, (K + 15) // 16 * 16 + 16), 101, dtype=torch.int8, device=DEV)
        q[:, :K] = torch.randint(-127, 128, (n, K), generator=gen, device=DEV, dtype=torch.int8)
        rows.append(kernels.Int8Rows(q[:, :K], torch.rand(n, generator=gen, device=DEV)))
    want, tol = _tail64(kernels.Int8Rows(rows[0].q[None], rows[0].scale[None]), rows[1], None, "bias", None, None, torch.bfloat16)
    _within(kernels.linear_int8(rows[0], rows[1], tile=tile), want[0], tol[0])


@pytest.mark.parametrize("S", [5, 70])
@pytest.mark.parametrize("epilogue", EPILOGUES)
@pytest.mark.parametrize("N", [1, 9, 31, 60, 67, 129, 258, 300])
def test_columns_behind_a_result_of_odd_width_stay(N, epilogue, S):
    from hetu_dit_b200 import kernels
    x, w, b, res, gate = _layer(2, S, 96, N, torch.bfloat16, N)
    pitch = (N + 15) // 8 * 8
    x8 = kernels.quantize_rows(x)
    want, tol = _tail64(x8, w, b, epilogue, res, gate, torch.bfloat16)
    wide_res = torch.zeros(2, S, pitch, dtype=torch.bfloat16, device=DEV)
    wide_res[..., :N] = res
    for residual in (res, wide_res[..., :N]):
        for tile in (0, 1, 2, 3, 4):
            wide = torch.full((2, S, pitch), 7.0, dtype=torch.bfloat16, device=DEV)
            kernels.linear_int8(x8, w, b, epilogue, residual=residual, gate=gate, out=wide[..., :N], tile=tile)
            _within(wide[..., :N], want, tol)
            assert (wide[..., N:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("S", [3, 100])
def test_linear_int8_layouts(S, dtype):
    from hetu_dit_b200 import kernels
    B, K, N = 2, 200, 136
    x, w, b, res, gate = _layer(B, S, K, N, dtype, 21)
    want, tol = _tail64(kernels.quantize_rows(x), w, b, "gate_residual", res, gate, dtype)
    # x a column block, out a column block of a wider buffer whose other columns stay; aligned and not
    for off in (64, 3):
        wide_x = torch.zeros(B, S, K + 80, dtype=dtype, device=DEV)
        wide_x[..., off:off + K] = x
        wide = torch.full((B, S, 300), 7.0, dtype=dtype, device=DEV)
        out = wide[..., off:off + N]
        got = kernels.linear_int8(wide_x[..., off:off + K], w, b, "gate_residual", residual=res, gate=gate, out=out)
        assert got is out
        _within(out, want, tol)
        assert (wide[..., :off] == 7).all() and (wide[..., off + N:] == 7).all()
        wide_res = torch.zeros(B, S, 300, dtype=dtype, device=DEV)
        wide_res[..., off:off + N] = res
        _within(kernels.linear_int8(x, w, b, "gate_residual", residual=wide_res[..., off:off + N], gate=gate), want, tol)
    # in place over the residual; gate a column block of the modulation; rows that are a slice of every entry's
    r2 = res.clone()
    mods = torch.zeros(B, 6 * N, dtype=dtype, device=DEV)
    mods[:, 2 * N:3 * N] = gate
    kernels.linear_int8(x, w, b, "gate_residual", residual=r2, gate=mods[:, 2 * N:3 * N], out=r2)
    _within(r2, want, tol)
    tall_x, tall_r = torch.zeros(B, S + 9, K, dtype=dtype, device=DEV), torch.zeros(B, S + 9, N, dtype=dtype, device=DEV)
    tall_x[:, 4:4 + S], tall_r[:, 4:4 + S] = x, res
    tall_o = torch.full((B, S + 9, N), 7.0, dtype=dtype, device=DEV)
    kernels.linear_int8(tall_x[:, 4:4 + S], w, b, "gate_residual", residual=tall_r[:, 4:4 + S], gate=gate, out=tall_o[:, 4:4 + S])
    _within(tall_o[:, 4:4 + S], want, tol)
    assert (tall_o[:, :4] == 7).all() and (tall_o[:, 4 + S:] == 7).all()
    held = kernels.quantize_rows(tall_x)
    part = kernels.Int8Rows(held.q[:, 4:4 + S], held.scale[:, 4:4 + S], dtype)
    _within(kernels.linear_int8(part, w, b, "gate_residual", residual=res, gate=gate), want, tol)
    # (rows, K); nothing
    want2, tol2 = _tail64(kernels.quantize_rows(x), w, b, "bias", None, None, dtype)
    two = kernels.linear_int8(x.reshape(B * S, K), w, b)
    _within(two, want2.reshape(B * S, N), tol2.reshape(B * S, N))
    assert kernels.linear_int8(x[:, :0], w, b).shape == (B, 0, N)


@pytest.mark.parametrize("S", [2, 140])
def test_a_row_without_a_number_stays_alone(S):
    from hetu_dit_b200 import kernels
    x, w, b, res, gate = _layer(1, S, 256, 96, torch.bfloat16, 4)
    want = kernels.linear_int8(x, w, b)
    x[0, 1, 7] = float("nan")
    got = kernels.linear_int8(x, w, b)
    assert torch.isnan(got[0, 1]).all()
    keep = [r for r in range(S) if r != 1]
    assert torch.equal(got[0, keep], want[0, keep])


@pytest.mark.parametrize("S", [1, 9, 200])
def test_linear_int8_on_streams_and_in_graphs(S):
    from hetu_dit_b200 import kernels
    x, w, b, res, gate = _layer(1, S, 1536, 512, torch.bfloat16, 31)
    x2 = torch.randn_like(x)
    want, want2 = kernels.linear_int8(x, w, b), kernels.linear_int8(x2, w, b)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for i in range(6):  # two calls at once, again and again
        with torch.cuda.stream(side[i % 2]):
            outs.append(kernels.linear_int8(x if i % 2 else x2, w, b))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want if i % 2 else want2) for i, o in enumerate(outs))
    static = x.clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = kernels.linear_int8(static, w, b)
        graphs.append((g, out))
    static.copy_(x2)
    for _ in range(2):
        for g, out in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want2) for _, out in graphs)


def test_linear_int8_beyond_2_to_31_elements():
    from hetu_dit_b200 import kernels
    S, K, N = 180000, 48, 12000
    gen = _gen(77)
    x = _randn(gen, 1, S, K, dtype=torch.bfloat16)
    w = kernels.quantize_rows(_randn(gen, N, K, dtype=torch.bfloat16))
    b = _randn(gen, N, dtype=torch.bfloat16)
    got = kernels.linear_int8(x, w, b)
    for rows in (slice(0, 40), slice(S // 2, S // 2 + 40), slice(S - 40, S)):
        want, tol = _tail64(kernels.quantize_rows(x[:, rows].contiguous()), w, b, "bias", None, None, torch.bfloat16)
        _within(got[:, rows], want, tol)
    q = kernels.quantize_rows(got)
    assert torch.equal(q.q[0, -5:], _rows64(got[0, -5:])[0])


def test_norm_rows_product_and_group_norm_in_a_run():
    """What a block does: norm and modulation into 8-bit rows, first layer with GELU, second layer with the gated residual;
    then a feature map's norm into the projection."""
    from hetu_dit_b200 import kernels
    dtype = torch.bfloat16
    gen = _gen(12)
    B, S, d = 2, 210, 320
    x = _randn(gen, B, S, d, dtype=dtype)
    shift, scale, gate = (0.3 * torch.randn(3, B, d, generator=gen, device=DEV)).to(dtype).unbind(0)
    up, down = (kernels.quantize_rows((0.05 * torch.randn(n, k, generator=gen, device=DEV)).to(dtype)) for n, k in ((4 * d, d), (d, 4 * d)))
    b1, b2 = _randn(gen, 4 * d, dtype=dtype), _randn(gen, d, dtype=dtype)
    h8 = kernels.ln_modulate_int8(x, shift, scale)
    h = kernels.linear_int8(h8, up, b1, "gelu_tanh")
    want, tol = _tail64(h8, up, b1, "gelu_tanh", None, None, dtype)
    _within(h, want, tol)
    y = kernels.linear_int8(h, down, b2, "gate_residual", residual=x, gate=gate)
    want, tol = _tail64(kernels.quantize_rows(h), down, b2, "gate_residual", x, gate, dtype)
    _within(y, want, tol)
    image = y.view(B, 14, 15, d).permute(0, 3, 1, 2)
    n8 = kernels.group_norm_int8(image, 32)
    proj = kernels.quantize_rows((0.05 * torch.randn(d, d, generator=gen, device=DEV)).to(dtype))
    z = kernels.linear_int8(n8, proj, b2)
    want, tol = _tail64(n8, proj, b2, "bias", None, None, dtype)
    _within(z, want, tol)
    # against the run of 16-bit values: each 8-bit step is within 1/254 of its row's largest value
    ref = torch.nn.functional.group_norm(y.double().view(B, 14, 15, d).permute(0, 3, 1, 2), 32, eps=1e-6).flatten(2).transpose(1, 2)
    assert ((n8.q.double() * n8.scale.double()[..., None] - ref).abs() <= ref.abs().amax(-1, keepdim=True) / 253).all()


# ----------------------------------------------------------------------------------------------------- group norm

def _gn64(rows, groups, weight, bias, eps, act):
    """(y, largest error of an fp32 computation) for (B, S, C) rows."""
    B, S, C = rows.shape
    X = rows.double().view(B, S, groups, C // groups)
    mean = X.mean((1, 3), keepdim=True)
    var = X.var((1, 3), correction=0, keepdim=True)
    sd = torch.sqrt(var + eps)
    z = (X - mean) / sd
    w = (torch.ones(C, device=DEV) if weight is None else weight).double().view(groups, -1)
    b = (torch.zeros(C, device=DEV) if bias is None else bias).double().view(groups, -1)
    y = z * w + b
    # Sums in a thread, over its rows and then over the lanes, channels and strips: at most 256 + 64 terms one after the
    # other, of distances from a row's values, which are at most D deviations from the mean
    u = 2.0 ** -24
    D = z.abs().amax((1, 3), keepdim=True) + 1
    off = w.abs() * 320 * u * (D + z.abs() * D ** 2) + 3 * u * ((mean / sd * w).abs() + (X / sd * w).abs() + y.abs() + b.abs())
    y, off = y.reshape(B, S, C), off.reshape(B, S, C)
    if act == "silu":
        # slope below 1.1; exp(-y) is off by 2^-22 + 2^-23 |y| of its value, the quotient by 2^-22
        off = 1.1 * off + 2.0 ** -21 * y.abs() * (1 + y.abs())
        y = y * torch.sigmoid(y)
    return y, off


def _image(B, H, W, C, dtype, seed):
    gen = _gen(seed)
    x = torch.randn(B, H, W, C, generator=gen, device=DEV)
    x = x * (0.5 + torch.rand(C, generator=gen, device=DEV)) + torch.randn(C, generator=gen, device=DEV)
    return x.to(dtype).permute(0, 3, 1, 2), _randn(gen, C, dtype=dtype), _randn(gen, C, dtype=dtype)


IMAGES = [(1, 1, 1, 8, 1), (1, 1, 1, 64, 8), (1, 1, 7, 64, 32), (2, 3, 5, 96, 32), (3, 16, 16, 320, 32), (1, 33, 47, 512, 32),
          (1, 64, 64, 128, 32), (2, 9, 31, 640, 16), (1, 5, 9, 1280, 32), (1, 20, 13, 2048, 32), (1, 6, 7, 2560, 32), (2, 4, 5, 4096, 8),
          (1, 3, 5, 4096, 4096), (1, 200, 180, 8, 1), (1, 150, 160, 24, 8)]


def _rows_of(t):
    return t.flatten(2).transpose(1, 2) if t.dim() > 3 else t


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("B,H,W,C,groups", IMAGES)
def test_group_norm(B, H, W, C, groups, act, dtype):
    from hetu_dit_b200 import kernels
    x, w, b = _image(B, H, W, C, dtype, H + W + C)
    want, off = _gn64(_rows_of(x), groups, w, b, 1e-5, act)
    got = kernels.group_norm(x, groups, w, b, eps=1e-5, act=act)
    assert got.shape == x.shape and got.dtype == dtype and got.is_contiguous(memory_format=torch.channels_last)
    _within(_rows_of(got), want, off * (1 + torch.finfo(dtype).eps) + _half_step(want, dtype))
    want, off = _gn64(_rows_of(x), groups, None, None, 1e-5, act)
    _within(_rows_of(kernels.group_norm(x, groups, eps=1e-5, act=act)), want, off * (1 + torch.finfo(dtype).eps) + _half_step(want, dtype))
    got8 = kernels.group_norm_int8(x, groups, w, b, eps=1e-5, act=act)
    want, off = _gn64(_rows_of(x), groups, w, b, 1e-5, act)
    top = want.abs().amax(-1)
    s = got8.scale.double()
    assert got8.q.shape == want.shape
    assert ((s - top / 127).abs() <= off.amax(-1) / 127 + 2.0 ** -23 * top / 127).all()
    _within(got8.q.double() * s[..., None], want, off + s[..., None] * (0.5 + 127 * 2.0 ** -22))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_group_norm_of_a_far_mean(dtype):
    """Channels 200 deviations away from zero (fp16; 40 for bf16, which resolves no more)."""
    from hetu_dit_b200 import kernels
    gen = _gen(9)
    far = 200.0 if dtype == torch.float16 else 40.0
    x = (torch.randn(1, 4000, 64, generator=gen, device=DEV) + far).to(dtype)
    want, off = _gn64(x, 8, None, None, 1e-6, None)
    _within(kernels.group_norm(x, 8), want, off * (1 + torch.finfo(dtype).eps) + _half_step(want, dtype))


def test_group_norm_layouts():
    from hetu_dit_b200 import kernels
    dtype = torch.bfloat16
    x, w, b = _image(2, 6, 10, 64, dtype, 2)
    want = kernels.group_norm(x, 8, w, b, act="silu")
    rows = _rows_of(x)
    assert torch.equal(kernels.group_norm(rows, 8, w, b, act="silu"), _rows_of(want))
    video = x.reshape(2, 64, 3, 2, 10).contiguous(memory_format=torch.channels_last_3d)
    got = kernels.group_norm(video, 8, w, b, act="silu")
    assert got.shape == video.shape and torch.equal(got.reshape(2, 64, 6, 10), want)
    # rows of a wider buffer, aligned and not; the other columns stay
    for off in (16, 5):
        wide = torch.full((2, 60, 100), 3.0, dtype=dtype, device=DEV)
        wide[..., off:off + 64] = rows
        assert torch.equal(kernels.group_norm(wide[..., off:off + 64], 8, w, b, act="silu"), _rows_of(want))
        held, plain = kernels.group_norm_int8(wide[..., off:off + 64], 8, w, b), kernels.group_norm_int8(rows, 8, w, b)
        assert torch.equal(held.q, plain.q) and torch.equal(held.scale, plain.scale)
        out = torch.full((2, 60, 100), 3.0, dtype=dtype, device=DEV)
        kernels.group_norm(rows, 8, w, b, act="silu", out=out[..., off:off + 64])
        assert torch.equal(out[..., off:off + 64], _rows_of(want))
        assert (out[..., :off] == 3).all() and (out[..., off + 64:] == 3).all()
    inplace = x.clone(memory_format=torch.preserve_format)
    assert kernels.group_norm(inplace, 8, w, b, act="silu", out=inplace) is inplace and torch.equal(inplace, want)
    assert kernels.group_norm(x[:0], 8, w, b).shape == (0, 64, 6, 10)
    assert kernels.group_norm(rows[:, :0], 8, w, b).shape == (2, 0, 64)
    assert kernels.group_norm_int8(rows[:, :0], 8, w, b).q.shape == (2, 0, 64)


def test_group_norm_without_numbers_and_of_constants():
    from hetu_dit_b200 import kernels
    x, w, b = _image(2, 40, 40, 64, torch.bfloat16, 6)
    want = kernels.group_norm(x, 8, w, b)
    x[0, 17, 3, 4] = float("nan")
    x[1, 40, 39, 39] = float("inf")
    got = kernels.group_norm(x, 8, w, b)
    assert torch.isnan(got[0, 16:24]).all() and torch.isnan(got[1, 40:48]).all()
    for i, lo in ((0, 16), (1, 40)):
        keep = [c for c in range(64) if not lo <= c < lo + 8]
        assert torch.equal(got[i, keep], want[i, keep])
    q = kernels.group_norm_int8(x, 8, w, b)
    assert torch.isnan(q.scale).all() and (q.q == 0).all()
    same = torch.full((1, 50, 64), 3.0, dtype=torch.bfloat16, device=DEV)
    assert torch.equal(kernels.group_norm(same, 8, w, b)[0], b.expand(50, 64))


def test_group_norm_on_streams_and_in_graphs():
    from hetu_dit_b200 import kernels
    for H in (16, 300):
        x, w, b = _image(1, H, H, 128, torch.bfloat16, H)
        x2 = torch.randn_like(x)
        want, want2 = kernels.group_norm(x, 32, w, b, act="silu"), kernels.group_norm(x2, 32, w, b, act="silu")
        torch.cuda.synchronize()
        side = [torch.cuda.Stream(), torch.cuda.Stream()]
        outs = []
        for i in range(6):
            with torch.cuda.stream(side[i % 2]):
                outs.append(kernels.group_norm(x if i % 2 else x2, 32, w, b, act="silu"))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want if i % 2 else want2) for i, o in enumerate(outs))
        static = x.clone(memory_format=torch.preserve_format)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = kernels.group_norm(static, 32, w, b, act="silu")
            graphs.append((g, out))
        static.copy_(x2)
        for g, out in graphs + graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want2) for _, out in graphs)


def test_group_norm_beyond_2_to_31_elements():
    from hetu_dit_b200 import kernels
    x = torch.randn(1, 1, 128, device=DEV, dtype=torch.bfloat16).expand(1, 64, 128).repeat(1, 270000, 1)  # 2.2e9 elements
    x[0, :, 3] += (torch.arange(x.shape[1], device=DEV) % 2).to(torch.bfloat16)
    got = kernels.group_norm(x, 32)
    want, off = _gn64(x[:, :2], 32, None, None, 1e-6, None)  # two rows that repeat: the same statistics
    tol = off * (1 + 2.0 ** -8) + 2.0 ** -12 + _half_step(want, torch.bfloat16)  # thousands of terms in a thread
    for at in (0, 1 << 23, x.shape[1] - 2):
        _within(got[:, at:at + 2], want, tol)


@pytest.mark.parametrize("B,S", [(4, 1), (9, 1), (140, 1), (1, 9), (3, 50)])
def test_rows_wider_than_they_have_to_be(B, S):
    """Rows that a program has laid out itself: the columns of wider ones, one to an entry or several."""
    from hetu_dit_b200 import kernels
    gen = _gen(B + S)
    w = kernels.quantize_rows(_randn(gen, 33, 40, dtype=torch.bfloat16))
    held = kernels.quantize_rows(_randn(gen, B, S, 40, dtype=torch.bfloat16))
    want = kernels.linear_int8(held, w)
    wide = torch.full((B, S, 64), 77, dtype=torch.int8, device=DEV)
    wide[..., :40] = held.q
    views = [wide[..., :40]]
    if S == 1:
        views.append(wide[:, 0, :40][:, None])  # the same place, another stride of the one row
    for q in views:
        assert torch.equal(kernels.linear_int8(kernels.Int8Rows(q, held.scale), w), want)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("k", [200, 1032, 1033, 2504, 5000, 20000])
def test_more_entries_than_a_grid_has_rows_of_ctas(k, dtype):
    """A CTA goes from one entry to another, with one row of each: windows that move on by eight elements."""
    from hetu_dit_b200 import kernels
    B = 65535 + 300
    long = _randn(_gen(k), 8 * B + k, dtype=dtype)
    x = long.as_strided((B, 1, k), (8, k, 1))
    got = kernels.quantize_rows(x)
    for at in (slice(0, 400), slice(B - 400, B)):
        q, s = _rows64(x[at])
        assert torch.equal(got.q[at], q) and torch.equal(got.scale[at], s)
    again = kernels.quantize_rows(x)
    assert torch.equal(again.q, got.q) and torch.equal(again.scale, got.scale)


def _room_calls():
    """Calls of one kernel that take more and less shared memory than each other, beyond what a launch may have unasked."""
    from hetu_dit_b200 import kernels
    gen = _gen(5)
    dtype = torch.bfloat16
    calls = {}
    for name, sizes in (("few rows", (40000, 20000)), ("norm", (8192, 6152)), ("group norm", (4096, 2048)), ("group norm, 8-bit rows", (4096, 2048))):
        for size in sizes:
            if name == "few rows":
                x, w = _randn(gen, 1, 2, size, dtype=dtype), kernels.quantize_rows(_randn(gen, 16, size, dtype=dtype))
                call = lambda x=x, w=w: kernels.linear_int8(x, w)  # noqa: E731
            elif name == "norm":
                x, m = _randn(gen, 1, 3, size, dtype=dtype), _randn(gen, 2, 1, size, dtype=dtype)
                call = lambda x=x, m=m: kernels.ln_modulate_int8(x, m[0], m[1]).q  # noqa: E731
            else:
                x = _randn(gen, 40, 9, 4096, dtype=dtype)  # too many images for a cluster each
                if name == "group norm":
                    call = lambda x=x, g=size: kernels.group_norm(x, g)  # noqa: E731
                else:
                    call = lambda x=x, g=size: kernels.group_norm_int8(x, g).q  # noqa: E731
            calls.setdefault(name, []).append(call)
    return calls


@pytest.mark.parametrize("name", ["few rows", "norm", "group norm", "group norm, 8-bit rows"])
def test_calls_of_two_threads_leave_each_other_their_shared_memory(name):
    """What a kernel may take belongs to the device, not to the call: the smaller call of one thread must not take the larger
    one's room between its set-up and its launch."""
    import threading
    calls = _room_calls()[name]
    want = [call() for call in calls]
    failed, done = [], []

    def work(call, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(400):
                    got = call()
                torch.cuda.current_stream().synchronize()
                done.append(torch.equal(got, want))
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=a) for a in list(zip(calls, want)) * 2]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and done == [True] * 4, failed[:1]


@pytest.mark.parametrize("name", ["few rows", "norm", "group norm", "group norm, 8-bit rows"])
def test_a_larger_call_and_a_smaller_one_in_one_graph(name):
    calls = _room_calls()[name]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [call() for call in calls]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", ["few rows", "norm", "group norm", "group norm, 8-bit rows"])
def test_a_smaller_call_leaves_a_kernel_what_a_larger_one_takes(name):
    from tests.captured_kernels import MOST_DYNAMIC_SHARED, captured_kernels
    large, small = _room_calls()[name]
    kernels = captured_kernels(large)
    assert max(k.shared_bytes for k in kernels) > 48 * 1024
    small()
    for k in kernels:
        assert k.attribute(MOST_DYNAMIC_SHARED) >= k.shared_bytes


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("value", [3.0, 50.0, -500.0, 5000.0])
@pytest.mark.parametrize("shape", [(2, 50, 64), (1, 3000, 64), (40, 700, 64), (1, 40000, 16)])
def test_group_norm_of_flat_groups(shape, value, dtype):
    """Groups whose variance is nothing, or little beside eps: a step of x counts 1 / sqrt(eps), and so does an error of the
    mean. All but one group are constant; that one differs in one place by the type's step.

    The bound is _gn64()'s without a term of the mean's size: x - pivot is rounded (u of it, below |z| + D deviations), a has three
    roundings and multiplies x - pivot and mean - pivot alike, b is rounded (u of D w and |b|), the result as well."""
    from hetu_dit_b200 import kernels
    B, S, C = shape
    gen, u = _gen(S), 2.0 ** -24
    x = torch.full(shape, value, device=DEV, dtype=dtype)
    x[B - 1, S // 2, C - 3] += torch.finfo(dtype).eps * 2 ** math.floor(math.log2(abs(value)))
    w, b = _randn(gen, C, dtype=dtype), _randn(gen, C, dtype=dtype)
    X = x.double().view(B, S, 8, C // 8)
    z = (X - X.mean((1, 3), keepdim=True)) / torch.sqrt(X.var((1, 3), correction=0, keepdim=True) + 1e-6)
    D = (z.abs().amax((1, 3), keepdim=True) + 1).expand(X.shape).reshape(shape)
    z, w64, b64 = z.reshape(shape), w.double(), b.double()
    want = z * w64 + b64
    off = w64.abs() * 320 * u * (D + z.abs() * D ** 2) + 3 * u * (2 * w64.abs() * (z.abs() + D) + want.abs() + b64.abs())
    got = kernels.group_norm(x, 8, w, b)
    _within(got, want, off * (1 + torch.finfo(dtype).eps) + _half_step(want, dtype))
    inplace = x.clone()
    assert torch.equal(kernels.group_norm(inplace, 8, w, b, out=inplace), got)
    got8 = kernels.group_norm_int8(x, 8, w, b)
    s = got8.scale.double()
    _within(s, want.abs().amax(-1) / 127, off.amax(-1) / 127 + 2.0 ** -23 * s)
    _within(got8.q.double() * s[..., None], want, off + s[..., None] * (0.5 + 127 * 2.0 ** -22))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("epilogue", ["bias", "gelu_tanh", "gate_residual"])
@pytest.mark.parametrize("tile", [1, 2, 3, 4])
def test_aligned_products_keep_their_values_in_registers(tile, epilogue, dtype):
    """A few bytes of local memory for what a failed wait reports, no spilled values beside them."""
    from hetu_dit_b200 import kernels
    from tests.captured_kernels import LOCAL_BYTES, captured_kernels
    x, w, b, res, gate = _layer(1, 300, 512, 264, dtype, 4)
    x8 = kernels.quantize_rows(x)
    rest = (res, gate) if epilogue == "gate_residual" else (None, None)
    (kernel,) = captured_kernels(lambda: kernels.linear_int8(x8, w, b, epilogue, *rest, tile=tile))
    assert kernel.attribute(LOCAL_BYTES) <= 16


@pytest.mark.parametrize("m,k,n,held,placed,count", [
    (1, 1536, 9216, False, False, 1), (2, 1536, 9216, False, True, 1), (2, 70000, 32, False, False, 1), (4, 2048, 2048, False, False, 1),
    (8, 1024, 2368, False, True, 1), (4, 1536, 9216, False, False, 2), (8, 768, 9216, False, False, 2), (5, 1536, 512, False, False, 2),
    (8, 256, 2369, False, False, 2), (9, 64, 64, False, False, 2), (1, 131072, 16, False, False, 1), (2, 81856, 16, False, False, 1), (2, 81857, 16, False, False, 2), (8, 512, 512, True, False, 1), (300, 512, 512, False, True, 2)])
def test_launches_of_a_few_rows(m, k, n, held, placed, count):
    """In a graph a launch more costs less than rows brought into 8 bits by several CTAs of an SM, or in several turns. What is
    counted is what is launched."""
    from hetu_dit_b200 import kernels
    from tests.captured_kernels import captured_kernels
    gen = _gen(m)
    x, w = _randn(gen, 1, m, k, dtype=torch.bfloat16), kernels.quantize_rows(_randn(gen, n, k, dtype=torch.bfloat16))
    x = kernels.quantize_rows(x) if held else x
    out = torch.empty(1, m, n, dtype=torch.bfloat16, device=DEV) if placed else None
    call = lambda: kernels.linear_int8(x, w, out=out)  # noqa: E731
    assert len(captured_kernels(call)) == count
    before = kernels.launch_count()
    call()
    assert kernels.launch_count() - before == count
