"""Every form of the fp8 products (linear_sizes): element by element in whole numbers, which are exact, against
float64 for other values, and where infinities and NaN stand. References are float64 products on the GPU.

Whole numbers: x = -7 .. 7 times 1 or 2 a block, with a 7 in each, is held as 64 x and a scale of 2^-6 or 2^-5; weights are
-2 .. 2 with scales of 1/2 and 1. Products of a group of 8 are within 2^4 of each other (none is cut off), and all
sums multiples of 32 below 2^24 times that, so they are exact in fp32 and the result is rounded once.
Other values: the bound of test_gpu_linear_fp8, and its 2-norm.
"""
import pytest
import torch

import ada_mla
from ada_mla import capi
from linear_sizes import OWN, TILES, all_sizes
from operators_reference import half_step

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
DTYPES = [torch.float16, torch.bfloat16]


def _name(size):
    return "x".join(map(str, size))


def _gen(size):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(size[0] * 31 + size[1] * 7 + size[2])
    return gen


def _wide(scale, like, rows=1):
    """Scales a block as one a value."""
    if rows > 1:
        scale = scale.repeat_interleave(rows, 0)[:like.shape[0]]
    return scale.repeat_interleave(128, 1)[:, :like.shape[1]]


def _whole_numbers(size):
    """x [m, k], its values and scales as they are held, w and its scales, and x W^T in float64, exactly."""
    (m, k, n), gen = size, _gen(size)
    blocks = -(-k // 128)
    x = torch.randint(-7, 8, (m, k), generator=gen, device="cuda").float()
    x[:, ::128] = 7.0
    up = 2.0 ** torch.randint(0, 2, (m, blocks), generator=gen, device="cuda").float()
    w = torch.randint(-2, 3, (n, k), generator=gen, device="cuda").float()
    ws = 2.0 ** -torch.randint(0, 2, (-(-n // 128), blocks), generator=gen, device="cuda").float()
    xq = (64 * x).to(F8)
    x = x * _wide(up, x)
    ref = x.double() @ (w * _wide(ws, w, 128)).double().t().contiguous()
    return x, xq, up / 64, w.to(F8), ws, ref


def _forms():
    return [(s, f) for f, sizes in TILES.items() for s in sizes]


def test_sizes_reach_their_form_here():
    for size, form in _forms():
        got = capi.linear_fp8_plan(*size, quantized=True)
        assert (got[0], got[1], got[2] > 1) == form, size
    for outputs, sizes in OWN.items():
        for size in sizes:
            assert capi.linear_fp8_plan(*size) == (outputs, 16, 1, 1), size


@pytest.mark.parametrize("size", all_sizes(), ids=_name)
def test_whole_numbers(size):
    x, xq, xs, w, ws, ref = _whole_numbers(size)
    for dtype in DTYPES:
        want = ref.to(dtype)
        assert torch.equal(ada_mla.mla_linear_fp8(x.to(dtype), w, ws), want)
        q, s = ada_mla.mla_quantize_fp8(x.to(dtype))
        assert torch.equal(q.view(torch.uint8) & 0x7F, xq.view(torch.uint8) & 0x7F) and torch.equal(s, xs)
        assert torch.equal(ada_mla.mla_linear_fp8(q, w, ws, x_scale=s, dtype=dtype), want)


@pytest.mark.parametrize("size", all_sizes(), ids=_name)
def test_strides(size):
    # NaN beside the rows of x and w, and between the scales, whose order in memory is any
    (m, k, n), f8nan = size, 0x7F
    x, xq, xs, w, ws, ref = _whole_numbers(size)
    want = ref.to(torch.bfloat16)
    raw_w = torch.full((n, k + 48), f8nan, dtype=torch.uint8, device="cuda")
    raw_w[:, 16:16 + k] = w.view(torch.uint8)
    raw_x = torch.full((m, k + 32), f8nan, dtype=torch.uint8, device="cuda")
    raw_x[:, 16:16 + k] = xq.view(torch.uint8)
    wide_x = torch.full((m, k + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide_x[:, 8:8 + k] = x.bfloat16()
    w, xq = raw_w.view(F8)[:, 16:16 + k], raw_x.view(F8)[:, 16:16 + k]
    assert torch.equal(ada_mla.mla_linear_fp8(wide_x[:, 8:8 + k], w, ws), want)
    apart = torch.full((m, 2, xs.shape[1], 3), float("nan"), device="cuda")
    apart[:, 1, :, 1] = xs
    for scale in (xs.contiguous(), xs.t().contiguous().t(), apart[:, 1, :, 1]):
        assert torch.equal(ada_mla.mla_linear_fp8(xq, w, ws, x_scale=scale), want), scale.stride()


@pytest.mark.parametrize("size", all_sizes(), ids=_name)
def test_infinities_and_nans(size):
    (m, k, n) = size
    x, xq, xs, w, ws, ref = _whole_numbers(size)
    clean = ref.to(torch.bfloat16)
    nan_rows, w_rows = sorted({m - 1, m // 2}) if m > 1 else [], sorted({0, n // 2, n - 1})
    x16, raw_w = x.bfloat16(), w.view(torch.uint8).clone()
    places = [k - 1, 0]  # the end of the last block, the beginning of the first
    for r, at in zip(nan_rows, places):
        x16[r, at] = float("nan") if at else float("inf")
    for i, r in enumerate(w_rows):
        raw_w[r, places[i % 2]] = 0xFF
    q, s = ada_mla.mla_quantize_fp8(x16)
    want = clean.clone()
    want[nan_rows] = float("nan")
    want[:, w_rows] = float("nan")
    for y in (ada_mla.mla_linear_fp8(x16, raw_w.view(F8), ws),
              ada_mla.mla_linear_fp8(q, raw_w.view(F8), ws, x_scale=s)):
        assert torch.equal(y.isnan(), want.isnan())
        assert torch.equal(y.nan_to_num(0.0), want.nan_to_num(0.0))


def _bound(xv, wv, ref, blocks, dtype):
    """Element by element, from the values with their scales (xv [m, k], wv [n, k], fp32): the terms of test_gpu_linear_fp8."""
    u = half_step(dtype)
    ax, aw = xv.abs(), wv.abs()
    size = ax.double() @ aw.double().t().contiguous()
    largest, top = torch.zeros_like(ref, dtype=torch.float32), torch.empty_like(ref, dtype=torch.float32)
    axt, awt = ax.t().contiguous(), aw.t().contiguous()
    for at in range(0, xv.shape[1], 8):
        torch.mul(axt[at][:, None], awt[at][None, :], out=top)
        for i in range(at + 1, at + 8):
            torch.maximum(top, axt[i][:, None] * awt[i][None, :], out=top)
        largest += top
    bound = 7 * 2.0 ** -13 * largest.double() * (1 + 2.0 ** -10) + (130 + blocks) * 2.0 ** -23 * size + u * ref.abs() * (1 + u)
    return bound + (2.0 ** -25 if dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", all_sizes(), ids=_name)
def test_other_values(size, dtype):
    (m, k, n), gen = size, _gen(size)
    x = torch.randn(m, k, generator=gen, device="cuda").to(dtype)
    w = (torch.randn(n, k, generator=gen, device="cuda") * 100).clamp(-448, 448).to(F8)
    ws = torch.rand(-(-n // 128), -(-k // 128), generator=gen, device="cuda") * 0.01 / k ** 0.5
    q, s = ada_mla.mla_quantize_fp8(x)
    xv, wv = q.float() * _wide(s, x), w.float() * _wide(ws, w, 128)
    ref = (q.double() * _wide(s, x).double()) @ (w.double() * _wide(ws, w, 128).double()).t().contiguous()
    bound = _bound(xv, wv, ref, s.shape[1], dtype)
    for y in (ada_mla.mla_linear_fp8(x, w, ws), ada_mla.mla_linear_fp8(q, w, ws, x_scale=s, dtype=dtype)):
        err = (y.double() - ref).abs()
        worst = (err / bound).max().item()
        assert worst <= 1.0, worst
        if dtype == torch.bfloat16:
            rel = (err.norm() / ref.norm()).item()
            assert rel <= 0.66 * half_step(dtype), rel


@pytest.mark.parametrize("size", [(13, 2048, 1001), (36, 768, 4411), (65, 800, 4191), (33, 9216, 69), (65, 3536, 4213), (6966, 784, 531),
                                  (1666, 784, 4647), (5477, 8752, 270)], ids=_name)
def test_replays_of_a_captured_call(size):
    x, _, _, w, ws, ref = _whole_numbers(size)
    given = torch.zeros_like(x, dtype=torch.bfloat16)

    def call():
        q, s = ada_mla.mla_quantize_fp8(given)
        return ada_mla.mla_linear_fp8(given, w, ws), ada_mla.mla_linear_fp8(q, w, ws, x_scale=s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        given.copy_(x * (1.0 if i % 2 else -1.0))
        graph.replay()
        torch.cuda.synchronize()
        want = (ref if i % 2 else -ref).to(torch.bfloat16)
        assert torch.equal(out[0], want) and torch.equal(out[1], want), i
        call()  # eager work between the replays
