"""Edges of the routed products on the GPU: the quantiser's zeros of either sign, gates over their
whole range, and far rows."""
import pytest
import torch

from test_experts_gpu import (BF16, DEV, E4M3, F16, F32, F64, blocked, eight_bits, ex, gen,
                              pair_parts, quantized, rand, routing, s, same_bits, stream, u)

pytestmark = pytest.mark.gpu


def with_zeros(g, rows, cols, dtype):
    """Values of which a third are zeros of either sign; one row of zeros of both signs alone."""
    x = rand(g, rows, cols, dtype=dtype)
    kind = torch.randint(0, 6, x.shape, generator=g, device=DEV)
    x[kind == 0] = 0.0
    x[kind == 1] = -0.0
    x[rows // 2] = torch.where(kind[rows // 2] > 2, -0.0, 0.0).to(dtype)
    return x


def negative(q):
    return q.contiguous().view(torch.uint8) >> 7 != 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,width,qmore", [(9, 256, 0), (5, 301, None), (7, 200, 3)])
def test_quantize_keeps_the_sign_of_zero(rows, width, qmore, dtype):
    """A quotient of a zero is a zero of its sign, whatever the block's scale is."""
    x = with_zeros(gen(80), rows, width, dtype)
    x[0] *= 2.0 ** -13      # scales of different sizes, in fp32 also one that no short way serves
    if dtype == F32:
        x[1] *= 2.0 ** -70
    q, scale = eight_bits(rows, width, qmore), torch.empty(-(-width // 128), rows, device=DEV)
    ex.Quantize(x, q, scale).run(stream())
    want_q, want_scale = quantized(x)
    assert torch.equal(scale, want_scale)
    zero = x == 0
    assert torch.equal(negative(q)[zero], torch.signbit(x)[zero])
    assert same_bits(q, want_q)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", [256, 75])
def test_dispatch_quantize_keeps_the_sign_of_zero(width, dtype):
    tokens, top_k = 40, 3
    r, _ = routing(tokens, top_k, 8)
    x = with_zeros(gen(81), tokens, width, dtype)
    q = eight_bits(tokens * top_k, width)
    scale = torch.empty(-(-width // 128), tokens * top_k, device=DEV)
    ex.DispatchQuantize(r, x, q, scale).run(stream())
    _, row, token = pair_parts(r)
    assert same_bits(q[row], quantized(x)[0][token])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", [128, 33])
def test_gated_zeros_keep_their_sign(width, dtype):
    """silu(0) = 0 and silu(-0) = -0, and a product's sign is its factors'."""
    g = gen(82)
    x = torch.cat([with_zeros(g, 12, width, dtype), with_zeros(g, 12, width, dtype)], 1)
    q, scale = eight_bits(12, width), torch.empty(1, 12, device=DEV)
    ex.Quantize(x, q, scale, gate="silu").run(stream())
    gate, up = x[:, :width], x[:, width:]
    zero = (gate == 0) | (up == 0)
    assert torch.equal(negative(q)[zero], (torch.signbit(gate) ^ torch.signbit(up))[zero])
    assert (q.float()[zero] == 0).all()


def gated(x, width):
    gate, up = x[:, :width].double(), x[:, width:].double()
    return gate / (1 + torch.exp(-gate)) * up


def gated_in_fp32_range(x, width):
    """The same where silu, and the product, are held in fp32: zero or infinite outside its range."""
    gate, up = x[:, :width].double(), x[:, width:].double()
    return ((gate / (1 + torch.exp(-gate))).float().double() * up).float().double()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", [16, 7])
def test_gates_of_every_size(width, dtype):
    """Gates from -104 to 104, a row of one size each, so that the row's scale shows silu itself.

    Of the value in fp32: 2^x to 2 ulp, its argument's rest, the sum, the quotient to an ulp and two
    products: below 10 half steps. bf16 takes exp(m) as 1 + m with |m| < 4.9e-6 |g|: m^2 / 2 more.
    Below -87 silu may be 0, and where the value is subnormal it is held to half the smallest step."""
    steps = torch.arange(-104 * 8, 104 * 8 + 1, device=DEV, dtype=F64) / 8
    rows = steps.numel()
    g = gen(83)
    x = torch.empty(rows, 2 * width, device=DEV, dtype=F64)
    x[:, :width] = steps[:, None] * rand(g, rows, width, dtype=F64, lo=0.97, hi=1.0)
    # the factors bring the values of negative gates back to ordinary sizes
    big = torch.exp2((-steps).clamp(0, 80).round()) if dtype != F16 else \
        torch.exp2((-steps).clamp(0, 15).round())
    x[:, width:] = big[:, None] * rand(g, rows, width, dtype=F64, lo=1.0, hi=1.9)
    x = x.to(dtype)
    q, scale = eight_bits(rows, width), torch.empty(1, rows, device=DEV)
    ex.Quantize(x, q, scale, gate="silu").run(stream())
    v = gated(x, width)
    gate = x[:, :width].double()
    part = 10 * u(F32) + ((4.9e-6 * gate) ** 2 / 2 if dtype == BF16 else 0.0)
    off = torch.where(gate < -87, 1.0, part) * v.abs() + 1.01 * s(F32)
    top, at = v.abs().max(1)
    want = (top / 448).clamp(min=torch.finfo(F32).tiny)
    worst = (scale[0].double() - want).abs() / (off.gather(1, at[:, None])[:, 0] / 448
                                                + u(F32) * want)
    assert worst.max() <= 1, (float(worst.max()), float(steps[worst.argmax()]))
    step = scale[0].double()[:, None]
    back = q.double() * step
    bad = (back - v).abs() > 1.0001 * (v.abs() * 2 ** -4 + step * 2 ** -10) + off
    assert not bad.any(), steps[bad.any(1)][:8]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", [256, 131])
def test_gates_that_are_extreme_or_no_numbers(width, dtype):
    """The largest and the lowest gates, infinities, NaN, and a product that overflows; each block's
    scale and bytes as the definition has them, and no other block changed."""
    top = torch.finfo(dtype).max
    cases = [(top, 1.0), (-top, 1.0), (-top, -top), (float("inf"), 1.0), (float("-inf"), 1.0),
             (float("nan"), 1.0), (1.0, float("inf")), (-200.0, float("inf")), (-200.0, top),
             (0.0, float("inf")), (top, top), (float("-inf"), 0.0)]
    g = gen(84)
    x = rand(g, len(cases), 2 * width, dtype=dtype)
    for i, (gate, up) in enumerate(cases):
        x[i, 130], x[i, width + 130] = gate, up
    q, scale = eight_bits(len(cases), width), torch.empty(2, len(cases), device=DEV)
    ex.Quantize(x, q, scale, gate="silu").run(stream())
    v = gated_in_fp32_range(x, width)
    b = blocked(v)
    amax = b.abs().amax(-1).t()          # keeps a NaN
    want = (amax / 448).clamp(min=torch.finfo(F32).tiny)
    assert torch.equal(torch.isnan(scale), torch.isnan(want))
    assert torch.equal(torch.isinf(scale), torch.isinf(want))
    fine = torch.isfinite(want)
    assert ((scale - want).abs()[fine] <= 11 * u(F32) * want[fine]).all()
    byte = q.float()[:, 130]
    ratio = v[:, 130] / want[1]
    assert torch.equal(torch.isnan(byte), torch.isnan(ratio))
    assert torch.equal(negative(q)[:, 130][ratio == 0], torch.signbit(v[:, 130])[ratio == 0])
    assert torch.isfinite(q.float()[:, :128]).all()


def test_far_rows():
    """Rows past 2^32 bytes in the gradients and in both quantisers, plain and gated."""
    k, rows = 1 << 16, (1 << 16) + 40
    g = gen(85)
    at = torch.tensor([rows - 1, 0, rows - 2], device=DEV)
    r = ex.Routes(3, 1, at.to(torch.int32))
    w = rand(g, 3, 1)
    dy, some = rand(g, 3, k, dtype=BF16), rand(g, 3, k, dtype=BF16)
    h = torch.zeros(rows, k, dtype=BF16, device=DEV)
    h[at] = some
    dh = torch.zeros(rows, k, dtype=BF16, device=DEV)
    dw = torch.empty(3, 1, device=DEV)
    ex.CombineGrad(r, dy, h, weights=w, dh=dh, dweights=dw).run(stream())
    want = dy.double() * w.double()
    assert ((dh[at].double() - want).abs() <= (u(BF16) + u(F32)) * 1.01 * want.abs()).all()
    term = dy.double() * some.double()
    assert ((dw[:, 0].double() - term.sum(1)).abs() <= k * u(F32) * term.abs().sum(1)).all()
    assert not dh[1:rows - 2].any()
    del dh
    # plain, and as a gate of half the columns
    q = torch.zeros(rows, k, dtype=torch.uint8, device=DEV).view(E4M3)
    scale = torch.empty(k // 128, rows, device=DEV)
    ex.Quantize(h, q, scale).run(stream())
    want_q, want_scale = quantized(some)
    assert same_bits(q[at], want_q) and torch.equal(scale[:, at], want_scale)
    half = k // 2
    ex.Quantize(h, q[:, :half], scale[:half // 128], gate="silu").run(stream())
    v = gated(some, half)
    step = scale[:half // 128, at].t().double().repeat_interleave(128, 1)
    back = q[at, :half].double() * step
    assert ((back - v).abs() <= 1.0001 * (v.abs() * 2 ** -4 + step * 2 ** -10)).all()
    q.view(torch.uint8).zero_()
    ex.DispatchQuantize(r, some, q, scale).run(stream())
    assert same_bits(q[at], want_q) and torch.equal(scale[:, at], want_scale)
    assert not q[1:rows - 2].view(torch.uint8).any()
