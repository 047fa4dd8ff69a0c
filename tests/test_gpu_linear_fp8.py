"""Products in e4m3 with a scale for each block of 128, and the quantisation of their rows, against float64.

Quantised values and scales have to be the formula's exactly (the scale is one fp32 division; 448 x / top is
within fp32's rounding of a tie of e4m3's only where it is one, so no rounding changes a value). A product,
with S = sum |xs ws xq wq| and u half a step of the result's type:
  the fp8 matrix instructions add products in groups of 8 neighbours, aligned to the group's largest: of each of
  the other 7 what lies below 2^-13 of that one is cut off (test_groups_of_eight shows it)   7 2^-13 sum of the groups' largest
  the groups' sums, 128 products a block, in fp32, whichever way it rounds; the blocks' sums; the scales'
  product                                                                             (130 + blocks) 2^-23 S
  the result's rounding (+ fp16: 2^-25 below its normal range)                                       u |y|
In the 2-norm the last rounding alone counts: u / sqrt(3), 0.6 u, is asked for with
10% for the rest (what is cut off is 1.5e-5 of N(0, 1) products' sum, 2^-16).
"""
import math

import pytest
import torch

import ada_mla
from ada_mla import capi
from operators_reference import half_step

pytestmark = pytest.mark.gpu

MOST, LEAST = 448.0, 2.0 ** -100


def _nearest(v):
    """The nearest e4m3 value of float64 values within +-448, even at a tie."""
    _, e = torch.frexp(v)
    step = torch.pow(2.0, (e - 4).clamp(min=-9).double())
    return torch.round(v / step) * step


def _quantised(x):
    """(values in float64, scales in float32) of 16-bit rows on the CPU."""
    m, k = x.shape
    blocks = -(-k // 128)
    wide = torch.zeros(m, blocks * 128, dtype=torch.float64)
    wide[:, :k] = x.double()
    wide = wide.view(m, blocks, 128)
    top = wide.abs().amax(2).clamp(min=LEAST)
    return _nearest(wide * MOST / top[..., None]).view(m, -1)[:, :k], top.float() / MOST


def _weight(gen, n, k, spread=False):
    nb, kb = -(-n // 128), -(-k // 128)
    if spread:  # every finite byte there is
        raw = torch.randint(0, 256, (n, k), generator=gen, dtype=torch.uint8)
        raw[(raw & 0x7F) == 0x7F] = 0x3A
        w = raw.view(torch.float8_e4m3fn)
        scale = torch.exp2(torch.randint(-12, 4, (nb, kb), generator=gen).float()) * (1 + torch.rand(nb, kb, generator=gen))
    else:
        w = (torch.randn(n, k, generator=gen) * 100).clamp(-MOST, MOST).to(torch.float8_e4m3fn)
        scale = torch.rand(nb, kb, generator=gen) * 0.01 / math.sqrt(k)
    return w, scale


def _check(got, xq, xs, w, ws, dtype, what="", ends=0.0):
    """xq [m, k] float64 values, xs [m, blocks]; w, ws as given to the call (all on the CPU)."""
    m, k = xq.shape
    n, u = w.shape[0], half_step(dtype)
    wide_x = xq * xs.double().repeat_interleave(128, 1)[:, :k]
    wide_w = w.double() * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    ref, size = wide_x @ wide_w.T, wide_x.abs() @ wide_w.abs().T
    largest = torch.zeros_like(ref)  # of each group of 8 products, added up
    for at in range(0, k, 8):
        top = torch.zeros_like(ref)
        for i in range(at, at + 8):
            torch.maximum(top, wide_x[:, i, None].abs() * wide_w[None, :, i].abs(), out=top)
        largest += top
    bound = 7 * 2.0 ** -13 * largest + (130 + ws.shape[1]) * 2.0 ** -23 * size + u * ref.abs() * (1 + u) + (2.0 ** -25 if dtype == torch.float16 else 0) + ends
    got = got.double().cpu()
    err = (got - ref).abs()
    assert torch.isfinite(got).all(), what
    worst = (err / bound).nan_to_num(0.0, posinf=float("inf")).max().item()
    assert worst <= 1.0, (what, worst)
    if ref.norm() > 0 and not ends and dtype == torch.bfloat16:
        assert err.norm() <= 0.66 * u * ref.norm(), (what, (err.norm() / ref.norm()).item())


def _x(gen, m, k, dtype):
    return torch.randn(m, k, generator=gen).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k", [(1, 16), (1, 128), (3, 144), (17, 1000 // 16 * 16), (130, 640), (5, 7168)])
def test_quantised_rows(dtype, m, k):
    gen = torch.Generator()
    gen.manual_seed(m + k)
    x = _x(gen, m, k, dtype)
    x[0, :8] = torch.tensor([0.0, -0.0, 1.0, -1.0, 0.5, 2.0 ** -14, 3.0, -7.0]).to(dtype)
    if m > 2:
        x[1] = 0  # nothing but zeros
        x[2] = torch.randint(-64, 65, (k,), generator=gen).to(dtype)  # many ties
    for call in (ada_mla.mla_quantize_fp8, capi.quantize_fp8):
        q, s = call(x.cuda())
        want, scales = _quantised(x)
        assert torch.equal(q.double().cpu(), want) and torch.equal(s.cpu(), scales)


@pytest.mark.parametrize("dtype,values", [(torch.bfloat16, [3.38e38, 1e38, -2.5e38]), (torch.bfloat16, [1e-38, 9e-41, -3e-39]),
                                          (torch.bfloat16, [2.0 ** -99, 2.0 ** -101, 2.0 ** -105]),
                                          (torch.float16, [65504.0, 6e-8, -1e-5]), (torch.float16, [6e-8, 6e-8, -1.2e-7])])
def test_quantised_ends_of_the_range(dtype, values):
    x = torch.tensor(values * 48).to(dtype).view(3, 48)
    q, s = ada_mla.mla_quantize_fp8(x.cuda())
    want, scales = _quantised(x)
    assert torch.equal(q.double().cpu(), want) and torch.equal(s.cpu(), scales)


def test_quantised_infinities_and_nans():
    gen = torch.Generator()
    gen.manual_seed(1)
    x = _x(gen, 4, 300, torch.bfloat16)[:, :288]
    x[1, 200], x[2, 5] = float("nan"), float("-inf")
    q, s = ada_mla.mla_quantize_fp8(x.cuda())
    want, scales = _quantised(torch.where(torch.isfinite(x), x, 0.0))
    q, s = q.double().cpu(), s.cpu()
    assert q[1, 200].isnan() and q[2, :128].isnan().all() and s[2, 0] == float("inf")
    q[1, 200], q[2, :128], s[2, 0] = 0.0, want[2, :128], scales[2, 0]
    assert torch.equal(q, want) and torch.equal(s, scales)


SIZES = [(1, 16, 1), (1, 128, 128), (2, 144, 3), (7, 1040, 129), (16, 512, 576), (17, 256, 64), (33, 2000, 255), (64, 640, 300),
         (65, 384, 127), (127, 128, 257), (128, 1152, 128), (129, 272, 640), (200, 1536, 513), (300, 2048, 1024), (513, 400, 385),
         (1000, 528, 4999), (66, 6976, 6698)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_sizes(dtype, m, k, n):
    gen = torch.Generator()
    gen.manual_seed(m * 7 + k + n)
    x = _x(gen, m, k, dtype)
    w, ws = _weight(gen, n, k)
    xq, xs = _quantised(x)
    y = ada_mla.mla_linear_fp8(x.cuda(), w.cuda(), ws.cuda())
    assert y.dtype == dtype and y.shape == (m, n)
    _check(y, xq, xs, w, ws, dtype, "16-bit rows")
    assert torch.equal(y, capi.linear_fp8(x.cuda(), w.cuda(), ws.cuda()))
    q, s = ada_mla.mla_quantize_fp8(x.cuda())
    z = ada_mla.mla_linear_fp8(q, w.cuda(), ws.cuda(), x_scale=s, dtype=dtype)
    _check(z, xq, xs, w, ws, dtype, "quantised rows")
    assert torch.equal(z, capi.linear_fp8(q, w.cuda(), ws.cuda(), x_scale=s, dtype=dtype))
    # scales in any order of memory
    assert torch.equal(z, ada_mla.mla_linear_fp8(q, w.cuda(), ws.cuda(), x_scale=s.contiguous(), dtype=dtype))
    apart = torch.full((m, 2, -(-k // 128), 3), float("nan"), device="cuda")
    apart[:, 1, :, 1] = s
    assert torch.equal(z, ada_mla.mla_linear_fp8(q, w.cuda(), ws.cuda(), x_scale=apart[:, 1, :, 1], dtype=dtype))


@pytest.mark.parametrize("m,k,n", [(3, 272, 200), (40, 640, 130), (150, 1000 // 16 * 16, 300)])
def test_every_byte_and_scale(m, k, n):
    gen = torch.Generator()
    gen.manual_seed(m)
    w, ws = _weight(gen, n, k, spread=True)
    xb, xs = _weight(gen, m, k, spread=True)
    xs = torch.exp2(torch.randint(-10, 3, (m, -(-k // 128)), generator=gen).float()) * (1 + torch.rand(m, -(-k // 128), generator=gen))
    y = ada_mla.mla_linear_fp8(xb.cuda(), w.cuda(), ws.cuda(), x_scale=xs.cuda())
    assert y.dtype == torch.bfloat16
    _check(y, xb.double(), xs, w, ws, torch.bfloat16, "bytes")


def test_groups_of_eight():
    # 2^16 + v - 2^16: v loses all below 2^3 beside 2^16 in its group of 8; in another group what fp32 has no
    # bits for behind 2^16 (2^-9 needs 26 of them)
    x, w = torch.zeros(20, 128), torch.zeros(1, 128)
    w[0, :] = 1.0
    w[0, 0] = w[0, 64] = 256.0
    x[:, 0], x[:, 64] = 256.0, -256.0
    values = [15.0, 8.0, 7.0, 0.5, 2.0 ** -9, -15.0, -8.0, -7.0, -0.5, -13.0]
    for i, v in enumerate(values):
        x[i, 7] = v
        x[10 + i, 8] = v
    one = torch.ones(1, 1, device="cuda")
    y = ada_mla.mla_linear_fp8(x.to(torch.float8_e4m3fn).cuda(), w.to(torch.float8_e4m3fn).cuda(), one,
                               x_scale=one.expand(20, 1), dtype=torch.float16)
    assert y[10:, 0].tolist() == [v if abs(v) > 2.0 ** -9 else 0.0 for v in values]
    assert y[:10, 0].tolist() == [math.copysign(abs(v) // 8 * 8, v) for v in values]


@pytest.mark.parametrize("m", [1, 20, 70, 260])
def test_strides_shapes_and_alignment(m):
    gen = torch.Generator()
    gen.manual_seed(m)
    k, n = 400, 200
    x, (w, ws) = _x(gen, m, k, torch.bfloat16), _weight(gen, n, k)
    xc, wc, sc = x.cuda(), w.cuda(), ws.cuda()
    y = ada_mla.mla_linear_fp8(xc, wc, sc)
    raw = torch.full((n, 1008), 0x7F, dtype=torch.uint8, device="cuda")  # NaN beside the rows
    raw[:, 16:16 + k] = wc.view(torch.uint8)
    strided_w = raw.view(torch.float8_e4m3fn)[:, 16:16 + k]
    wide = torch.full((m, 1016), float("nan"), dtype=torch.bfloat16, device="cuda")
    for at in (8, 13):  # readable in place, and not
        wide[:] = float("nan")
        wide[:, at:at + k] = xc
        assert torch.equal(ada_mla.mla_linear_fp8(wide[:, at:at + k], strided_w, sc), y)
        q, s = ada_mla.mla_quantize_fp8(wide[:, at:at + k])
        want = ada_mla.mla_quantize_fp8(xc)
        assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s, want[1])
    assert torch.equal(ada_mla.mla_linear_fp8(xc.t().contiguous().t(), wc, sc.t().contiguous().t()), y)
    off = torch.empty(n * k + 3, dtype=torch.uint8, device="cuda")[3:].view(n, k)
    off.copy_(wc.view(torch.uint8))
    assert torch.equal(ada_mla.mla_linear_fp8(xc, off.view(torch.float8_e4m3fn), sc), y)
    if m % 2 == 0:
        assert torch.equal(ada_mla.mla_linear_fp8(xc.view(2, m // 2, k), wc, sc), y.view(2, m // 2, n))
    assert torch.equal(ada_mla.mla_linear_fp8(xc[0], wc, sc), ada_mla.mla_linear_fp8(xc[:1], wc, sc)[0])
    assert ada_mla.mla_linear_fp8(xc[:0], wc, sc).shape == (0, n) and ada_mla.mla_quantize_fp8(xc[:0])[1].shape == (0, 4)


@pytest.mark.parametrize("m", [3, 40, 300])
def test_infinities_and_nans(m):
    gen = torch.Generator()
    gen.manual_seed(m)
    k, n = 1040, 300
    x, (w, ws) = _x(gen, m, k, torch.float16), _weight(gen, n, k)
    clean = ada_mla.mla_linear_fp8(x.cuda(), w.cuda(), ws.cuda())
    x[1, 1035], x[2, 3] = float("nan"), float("inf")
    w.view(torch.uint8)[257, 1039] = 0xFF
    y = ada_mla.mla_linear_fp8(x.cuda(), w.cuda(), ws.cuda())
    assert y[1].isnan().all() and y[2].isnan().all() and y[:, 257].isnan().all()
    y[1], y[2], y[:, 257] = clean[1], clean[2], clean[:, 257]
    assert torch.equal(y, clean)


def test_large_and_small_rows():
    # bf16 rows near the ends of its range, weights scaled the other way
    gen = torch.Generator()
    gen.manual_seed(11)
    for size, scale in ((2.0 ** 110, 2.0 ** -100), (2.0 ** -60, 2.0 ** 40)):
        x = (_x(gen, 30, 256, torch.float32) * size).to(torch.bfloat16)
        w, ws = _weight(gen, 70, 256)
        ws = ws * scale
        xq, xs = _quantised(x)
        _check(ada_mla.mla_linear_fp8(x.cuda(), w.cuda(), ws.cuda()), xq, xs, w, ws, torch.bfloat16, str(size))


def test_offsets_past_2_31():
    # 2.2 GB of weights: the last outputs' rows lie past 2^31 bytes
    n, k, gen = 140000, 16384, torch.Generator()
    gen.manual_seed(5)
    w = torch.zeros(n, k, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    tail, _ = _weight(gen, 200, k)
    w.view(torch.uint8)[-200:] = tail.view(torch.uint8).cuda()
    ws = torch.full((-(-n // 128), k // 128), 2.0 ** -10, device="cuda")
    for m in (1, 20, 200):
        x = _x(gen, m, k, torch.bfloat16)
        xq, xs = _quantised(x)
        y = ada_mla.mla_linear_fp8(x.cuda(), w, ws)
        assert not y[:, :-200].any()
        _check(y[:, -200:], xq, xs, tail, torch.full((2, k // 128), 2.0 ** -10), torch.bfloat16, f"{m} rows")


@pytest.mark.parametrize("m", [1, 40, 300])
def test_replays_of_a_captured_call(m):
    gen = torch.Generator()
    gen.manual_seed(m)
    k, n = 1040, 700
    w, ws = _weight(gen, n, k)
    wc, sc, x = w.cuda(), ws.cuda(), torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")

    def call():
        q, s = ada_mla.mla_quantize_fp8(x)
        return ada_mla.mla_linear_fp8(x, wc, sc), ada_mla.mla_linear_fp8(q, wc, sc, x_scale=s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(3):
        new = _x(gen, m, k, torch.bfloat16)
        x.copy_(new)
        graph.replay()
        eager = call()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1]), i
        xq, xs = _quantised(new)
        _check(out[0], xq, xs, w, ws, torch.bfloat16, f"replay {i}")


def test_two_streams_at_once():
    gen = torch.Generator()
    gen.manual_seed(3)
    w, ws = _weight(gen, 1000, 2048)
    wc, sc = w.cuda(), ws.cuda()
    xs = [_x(gen, 100, 2048, torch.bfloat16).cuda() for _ in range(2)]
    want = [ada_mla.mla_linear_fp8(x, wc, sc) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ada_mla.mla_linear_fp8(xs[i], wc, sc))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w_) for i, w_ in enumerate(want) for g in got[i])
