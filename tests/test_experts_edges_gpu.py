"""Edges of the routed products' quantiser on the GPU: zeros of either sign."""
import pytest
import torch

from test_experts_gpu import (BF16, DEV, F16, F32, eight_bits, ex, gen, pair_parts, quantized, rand,
                              routing, same_bits, stream)

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
