"""Routed products on the GPU against plain forms in 64 bits.

Tolerances count roundings: u(t) = finfo(t).eps / 2 is the half step of a type, s(t) half its
smallest subnormal step; a sum of n terms in a type of half step u is off by at most n u times the
sum of the terms' magnitudes, in whatever order it is taken.
"""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import appt_spgemm as ap
from appt_spgemm import experts as ex

pytestmark = pytest.mark.gpu

F64, F32, F16, BF16 = torch.float64, torch.float32, torch.float16, torch.bfloat16
E4M3 = torch.float8_e4m3fn
DEV = "cuda:0"


def u(t):
    return torch.finfo(t).eps / 2


def s(t):
    f = torch.finfo(t)
    return f.tiny * f.eps / 2


def acc_of(t):
    return F64 if t == F64 else F32


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rand(g, *shape, dtype=F32, lo=-1.0, hi=1.0):
    x = torch.rand(*shape, generator=g, device=DEV, dtype=F64) * (hi - lo) + lo
    return x.to(dtype)


def close(got, want, tol):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{float((got - want).abs()[bad].max()):.3e} where "
                           f"{float((tol * torch.ones_like(want))[bad].min()):.3e} is allowed")


# ----------------------------------------------------------------------------------------- route
def ids_for(g, tokens, top_k, experts, kind):
    if kind == "same":
        return torch.full((tokens, top_k), experts - 1, device=DEV)
    if kind == "none":
        return torch.full((tokens, top_k), -1, device=DEV)
    ids = torch.randint(0, experts, (tokens, top_k), generator=g, device=DEV)
    if kind == "skew":
        ids = (ids * ids * ids) // max(1, experts * experts)
    if kind == "wild":   # ids outside the range drop their pair
        wild = torch.tensor([-1, experts, -(2 ** 31), 2 ** 31 - 1], device=DEV)
        pick = torch.randint(0, 4, ids.shape, generator=g, device=DEV)
        ids = torch.where(torch.rand(ids.shape, generator=g, device=DEV) < 0.3, wild[pick], ids)
    return ids


def route(ids, experts, run=True):
    pairs = ids.shape[0] * ids.shape[1]
    ptr = torch.full((experts + 1,), -7, dtype=torch.int32, device=DEV)
    row_pair = torch.full((pairs,), -7, dtype=torch.int32, device=DEV)
    pair_row = torch.full((pairs,), -7, dtype=torch.int32, device=DEV)
    ws = torch.full((ex.route_workspace_bytes(ids.shape[0], ids.shape[1], experts),), 255,
                    dtype=torch.uint8, device=DEV)
    call = ex.Route(ids, experts, ptr, row_pair, pair_row, ws)
    if run:
        call.run(stream())
    return call, ptr, row_pair, pair_row


def route_oracle(ids, experts):
    flat = ids.cpu().numpy().astype(np.int64).ravel()
    kept = (flat >= 0) & (flat < experts)
    key = np.where(kept, flat, experts)
    order = np.argsort(key, kind="stable")
    n = int(kept.sum())
    ptr = np.searchsorted(key[order], np.arange(experts + 1))
    pair_row = np.full(flat.size, -1)
    pair_row[order[:n]] = np.arange(n)
    return ptr, order[:n], pair_row


def check_route(ids, experts, ptr, row_pair, pair_row):
    want_ptr, order, want_rows = route_oracle(ids, experts)
    assert np.array_equal(ptr.cpu().numpy(), want_ptr)
    got = row_pair.cpu().numpy()
    assert np.array_equal(got[:order.size], order)
    assert (got[order.size:] == -7).all()          # rows behind the last kept pair
    assert np.array_equal(pair_row.cpu().numpy(), want_rows)


@pytest.mark.parametrize("tokens,top_k,experts,kind", [
    (0, 2, 5, "any"), (1, 1, 1, "any"), (1, 8, 64, "any"), (2, 3, 7, "none"), (31, 1, 2, "any"),
    (33, 3, 1024, "any"), (32, 8, 64, "any"), (511, 8, 64, "same"), (512, 8, 64, "wild"),
    (513, 8, 64, "skew"), (1000, 40, 100, "wild"), (4097, 1, 1023, "any"), (20000, 3, 1, "wild"),
    (5000, 7, 512, "skew"), (70001, 8, 256, "wild"), (131073, 8, 333, "skew"),
    (66000, 8, 1024, "none"), (66000, 8, 1024, "same"), (3000, 4, 1024, "wild"),
    (4000, 8, 100, "skew"), (4096, 8, 33, "any"), (32769, 1, 64, "any")])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_route(tokens, top_k, experts, kind, dtype):
    ids = ids_for(gen(tokens + top_k), tokens, top_k, experts, kind).to(dtype)
    _, *out = route(ids, experts)
    check_route(ids, experts, *out)


def test_route_of_strided_ids_and_far_ids():
    wide = torch.randint(0, 16, (300, 9), generator=gen(1), device=DEV)
    ids = wide[:, 2:6]
    _, *out = route(ids, 16)
    check_route(ids, 16, *out)
    ids = ids.contiguous()
    ids[::5, 1] += 1 << 32      # equal to a valid id in its low 32 bits
    _, *out = route(ids, 16)
    check_route(ids, 16, *out)


FIRST_CALLS = """
import sys
sys.path[:0] = {paths!r}
import numpy as np
import test_experts_gpu as t
for tokens in (100, 2000, 40000):
    ids = t.ids_for(t.gen(1), tokens, 4, {experts}, "wild")
    _, *out = t.route(ids, {experts})
    t.check_route(ids, {experts}, *out)
print("ok")
"""


@pytest.mark.parametrize("experts", [300, 340, 420])
def test_route_as_a_process_s_first_call(experts):
    """Shared memory between what every kernel may have and the most: the opt-in is a kernel's own
    and must not come from an earlier, larger call."""
    code = FIRST_CALLS.format(paths=[str(Path(__file__).parent), *map(str, sys.path)],
                              experts=experts)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "ok" in r.stdout, r.stderr[-2000:]


# --------------------------------------------------------------------------- rows there and back
def routing(tokens, top_k, experts, kind="wild", seed=3):
    ids = ids_for(gen(seed), tokens, top_k, experts, kind).to(torch.int32)
    _, ptr, row_pair, pair_row = route(ids, experts)
    return ex.Routes(tokens, top_k, pair_row), ptr


def pair_parts(r):
    """(kept pairs, their rows, their tokens)"""
    rows = r.pair_row.long()
    p = torch.nonzero(rows >= 0).flatten()
    return p, rows[p], p // r.top_k


SHAPES = [  # tokens, top_k, width, row stride over the width, first column
    (1, 1, 1, 0, 0), (1, 8, 4096, 0, 0), (3, 2, 0, 0, 0), (7, 3, 1111, 0, 0), (64, 8, 128, 8, 0),
    (33, 40, 200, 8, 8), (100, 5, 513, 3, 1), (17, 2, 5000, 0, 0), (2, 33, 72, 8, 0),
    (0, 4, 32, 0, 0), (300, 4, 2048, 0, 0), (50, 6, 24, 0, 0)]
TYPES = [F64, F32, F16, BF16]


def strided(rows, width, more, first, dtype, fill=None, g=None):
    base = torch.full((rows, width + more), -5.0, device=DEV, dtype=F64).to(dtype)
    part = base[:, first:first + width]
    if g is not None:
        part.copy_(rand(g, rows, width, dtype=dtype))
    elif fill is not None:
        part.fill_(fill)
    return base, part


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_dispatch(shape, weighted, dtype):
    tokens, top_k, width, more, first = shape
    r, _ = routing(tokens, top_k, 16)
    g = gen(5)
    _, x = strided(tokens, width, more, first, dtype, g=g)
    base, y = strided(tokens * top_k, width, more, first, dtype, fill=9.0)
    w = rand(g, tokens, top_k, dtype=acc_of(dtype)) if weighted else None
    before = base.clone()
    ex.Dispatch(r, x, y, weights=w).run(stream())
    pair, row, token = pair_parts(r)
    if weighted:
        want = x.double()[token] * w.double().flatten()[pair][:, None]
        # one product and one rounding to the type
        tol = (u(dtype) + u(acc_of(dtype))) * 1.01 * want.abs() + s(dtype)
        close(y[row], want, tol)
    else:
        assert torch.equal(y[row], x[token])
    assert torch.equal(base[:, :first], before[:, :first])
    assert torch.equal(base[:, first + width:], before[:, first + width:])
    rest = torch.ones(tokens * top_k, dtype=torch.bool, device=DEV)
    rest[row] = False
    assert torch.equal(base[rest], before[rest])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_combine(shape, weighted, dtype):
    tokens, top_k, width, more, first = shape
    r, _ = routing(tokens, top_k, 16)
    g = gen(6)
    _, h = strided(tokens * top_k, width, more, first, dtype, g=g)
    base, y = strided(tokens, width, more, first, dtype, fill=9.0)
    w = rand(g, tokens, top_k, dtype=acc_of(dtype)) if weighted else None
    before = base.clone()
    ex.Combine(r, h, y, weights=w).run(stream())
    pair, row, token = pair_parts(r)
    term = h.double()[row] * (w.double().flatten()[pair][:, None] if weighted else 1.0)
    want = torch.zeros(tokens, width, dtype=F64, device=DEV).index_add_(0, token, term)
    size = torch.zeros(tokens, width, dtype=F64, device=DEV).index_add_(0, token, term.abs())
    tol = top_k * u(acc_of(dtype)) * size * 1.01 + u(dtype) * want.abs() * 1.01 + s(dtype)
    close(y, want, tol)
    assert torch.equal(base[:, :first], before[:, :first])
    assert torch.equal(base[:, first + width:], before[:, first + width:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("wanted", ["both", "dh", "dw", "both unweighted"])
@pytest.mark.parametrize("shape", SHAPES)
def test_combine_grad(shape, wanted, dtype):
    tokens, top_k, width, more, first = shape
    r, _ = routing(tokens, top_k, 16)
    g = gen(7)
    acc = acc_of(dtype)
    _, dy = strided(tokens, width, more, first, dtype, g=g)
    _, h = strided(tokens * top_k, width, more, first, dtype, g=g)
    base, dh = strided(tokens * top_k, width, more, first, dtype, fill=9.0)
    w = rand(g, tokens, top_k, dtype=acc) if "unweighted" not in wanted else None
    dw = torch.full((tokens, top_k), 9.0, dtype=acc, device=DEV)
    before = base.clone()
    ex.CombineGrad(r, dy, h if wanted != "dh" else None, weights=w,
                   dh=dh if wanted != "dw" else None,
                   dweights=dw if wanted != "dh" else None).run(stream())
    pair, row, token = pair_parts(r)
    if wanted != "dw":
        want = dy.double()[token] * (w.double().flatten()[pair][:, None] if w is not None else 1.0)
        close(dh[row], want, (u(dtype) + u(acc)) * 1.01 * want.abs() + s(dtype))
        rest = torch.ones(tokens * top_k, dtype=torch.bool, device=DEV)
        rest[row] = False
        assert torch.equal(base[rest], before[rest])
    if wanted != "dh":
        term = dy.double()[token] * h.double()[row]
        want = torch.zeros(tokens * top_k, dtype=F64, device=DEV)
        size = want.clone()
        want[pair], size[pair] = term.sum(1), term.abs().sum(1)
        close(dw.flatten(), want, max(width, 1) * u(acc) * size * 1.01)


def test_dispatch_and_combine_keep_what_is_no_number():
    """Infinities and NaN are copied bit by bit, and reach only the tokens whose pairs hold them; a
    dropped pair's weight and rows behind the last are not read."""
    tokens, top_k, width = 6, 2, 40
    ids = torch.tensor([[0, 1], [-1, 0], [1, -1], [-1, -1], [0, 1], [1, 0]], device=DEV)
    _, ptr, _, pair_row = route(ids, 2)
    r = ex.Routes(tokens, top_k, pair_row)
    x = rand(gen(8), tokens, width, dtype=BF16)
    x[0, 3], x[1, 5] = float("nan"), float("-inf")
    y = torch.zeros(tokens * top_k, width, dtype=BF16, device=DEV)
    ex.Dispatch(r, x, y).run(stream())
    _, row, token = pair_parts(r)
    assert torch.equal(y[row].view(torch.int16), x[token].view(torch.int16))
    w = torch.ones(tokens, top_k, device=DEV)
    w[ids < 0] = float("nan")
    h = torch.full((tokens * top_k, width), float("nan"), dtype=BF16, device=DEV)
    kept = int(ptr[-1])
    h[:kept] = 1.0
    h[int(pair_row[0]), 7] = float("inf")
    out = torch.full((tokens, width), 9.0, dtype=BF16, device=DEV)
    ex.Combine(r, h, out, weights=w).run(stream())
    want = (ids >= 0).sum(1)[:, None].expand(tokens, width).to(BF16).clone()
    want[0, 7] = float("inf")
    assert torch.equal(out, want)
    dw = torch.full((tokens, top_k), 9.0, device=DEV)
    ex.CombineGrad(r, torch.ones_like(out), h, weights=w, dweights=dw).run(stream())
    assert torch.equal(torch.isinf(dw), torch.zeros_like(dw).index_put(
        (torch.tensor([0], device=DEV), torch.tensor([0], device=DEV)),
        torch.ones(1, device=DEV)).bool())
    assert (dw[ids < 0] == 0).all() and (dw[1:][ids[1:] >= 0] == width).all()


def test_rows_outside_the_buffer_are_dropped():
    """A pair_row of more rows than the buffer has is a dropped pair, never a write behind it."""
    rows = torch.tensor([0, 5, 3, 2 ** 31 - 1, -2 ** 31, 1], dtype=torch.int32, device=DEV)
    r = ex.Routes(3, 2, rows)
    x = rand(gen(9), 3, 24, dtype=F32)
    base = torch.full((6, 24), 9.0, device=DEV)
    ex.Dispatch(r, x, base[:4]).run(stream())
    want = torch.full((6, 24), 9.0, device=DEV)
    want[0], want[3], want[1] = x[0], x[1], x[2]
    assert torch.equal(base, want)
    out = torch.full((3, 24), 7.0, device=DEV)
    ex.Combine(r, base[:4], out).run(stream())
    assert torch.equal(out, x)
    dw = torch.full((3, 2), 7.0, device=DEV)
    dh = torch.full((6, 24), 9.0, device=DEV)
    ex.CombineGrad(r, x, base[:4], dh=dh[:4], dweights=dw).run(stream())
    assert torch.equal(dh, want)
    assert (dw[rows.view(3, 2) == 5] == 0).all() and dw[1, 1] == 0 and dw[2, 0] == 0
    q = torch.zeros(4, 32, dtype=torch.uint8, device=DEV).view(E4M3)
    scale = torch.full((1, 6), 9.0, device=DEV)
    ex.DispatchQuantize(r, x, q[:, :24], scale[:, :4]).run(stream())
    assert (scale[0, 4:] == 9.0).all() and scale[0, 2] == 9.0
    assert (scale[0, [0, 1, 3]] < 1).all()


# ------------------------------------------------------------------------------------ gradients
@pytest.mark.parametrize("weighted", [False, True])
def test_gradients_against_differences(weighted):
    """combine and dispatch are linear in the rows and in the weights, so a central difference in
    fp64 is the derivative up to rounding: with values and directions of about 1 and a step of 1 the
    sums of some 200 terms are exact to about 1e-13."""
    tokens, top_k, width = 13, 3, 37
    r, _ = routing(tokens, top_k, 5)
    g = gen(11)
    x, c = rand(g, tokens, width, dtype=F64), rand(g, tokens, width, dtype=F64)
    h = rand(g, tokens * top_k, width, dtype=F64)
    w = rand(g, tokens, top_k, dtype=F64) if weighted else None
    pair, row, token = pair_parts(r)

    def combine(h, w):
        y = torch.empty(tokens, width, dtype=F64, device=DEV)
        ex.Combine(r, h, y, weights=w).run(stream())
        return y

    def dispatch(x, w):
        y = torch.zeros(tokens * top_k, width, dtype=F64, device=DEV)
        ex.Dispatch(r, x, y, weights=w).run(stream())
        return y

    # combine: L = <combine(h, w), c>
    dh = torch.zeros_like(h)
    dw = torch.empty(tokens, top_k, dtype=F64, device=DEV)
    ex.CombineGrad(r, c, h, weights=w, dh=dh, dweights=dw).run(stream())
    v = rand(g, *h.shape, dtype=F64)
    got = float((dh[row] * v[row]).sum())
    diff = float(((combine(h + v, w) - combine(h - v, w)) / 2 * c).sum())
    assert abs(got - diff) < 1e-12 * tokens * top_k * width
    if weighted:
        v = rand(g, *w.shape, dtype=F64)
        diff = float(((combine(h, w + v) - combine(h, w - v)) / 2 * c).sum())
        assert abs(float((dw * v).sum()) - diff) < 1e-12 * tokens * top_k * width
    # dispatch: L = <dispatch(x, w), h>
    dx = combine(h, w)
    v = rand(g, *x.shape, dtype=F64)
    diff = float(((dispatch(x + v, w) - dispatch(x - v, w)) / 2 * h).sum())
    assert abs(float((dx * v).sum()) - diff) < 1e-12 * tokens * top_k * width
    if weighted:
        dw = torch.empty(tokens, top_k, dtype=F64, device=DEV)
        ex.CombineGrad(r, x, h, dweights=dw).run(stream())
        v = rand(g, *w.shape, dtype=F64)
        diff = float(((dispatch(x, w + v) - dispatch(x, w - v)) / 2 * h).sum())
        assert abs(float((dw * v).sum()) - diff) < 1e-12 * tokens * top_k * width


# ----------------------------------------------------------------------------------------- 8 bits
def blocked(x):
    nb = -(-x.shape[-1] // 128)
    return torch.nn.functional.pad(x, (0, nb * 128 - x.shape[-1])).unflatten(-1, (nb, 128))


def quantized(x):
    """The definition in fp32 operations: (q, scale [blocks, rows])."""
    b = blocked(x.float())
    # a true quotient: torch divides by a Python number as a product with its reciprocal
    scale = (b.abs().amax(-1) / torch.full((), 448.0, device=DEV)).clamp(min=torch.finfo(F32).tiny)
    q = (b / scale[..., None]).flatten(1)[:, :x.shape[1]].to(E4M3)
    return q, scale.t().contiguous()


def eight_bits(rows, cols, more=None):
    ld = -(-cols // 16) * 16 if more is None else cols + more
    return torch.full((rows, ld), 0x55, dtype=torch.uint8, device=DEV).view(E4M3)[:, :cols]


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


QSHAPES = [  # rows, rows used, width, columns more in x, in q
    (1, 1, 1, 0, None), (5, 5, 128, 0, None), (9, 4, 129, 3, 2), (64, 64, 1000, 0, None),
    (33, 0, 256, 0, None), (7, 7, 2048, 8, None), (16, 20, 200, 0, 3), (300, 299, 72, 0, None),
    (2, -3, 64, 0, None), (0, 0, 64, 0, None), (3, 3, 0, 0, None), (40, 33, 5000, 0, 0)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", QSHAPES)
def test_quantize(shape, dtype):
    rows, used, width, more, qmore = shape
    x = strided(rows, width, more, 0, dtype, g=gen(13))[1] if width else \
        torch.empty(rows, 0, dtype=dtype, device=DEV)
    x *= torch.exp2(torch.arange(rows, device=DEV, dtype=F32) % 13 - 6)[:, None].to(dtype)
    q = eight_bits(rows, width, qmore)
    scale = torch.full((-(-width // 128), rows), 9.0, device=DEV)
    count = torch.tensor([used], dtype=torch.int32, device=DEV)
    ex.Quantize(x, q, scale, rows_ptr=count).run(stream())
    n = max(0, min(used, rows))
    want_q, want_scale = quantized(x[:n])
    assert same_bits(q[:n], want_q)
    assert torch.equal(scale[:, :n], want_scale)
    assert (scale[:, n:] == 9.0).all()
    assert (q[n:].contiguous().view(torch.uint8) == 0x55).all()
    # against the value itself: half a step of e4m3 (or of its subnormals, 2^-9 scales)
    back = q[:n].double() * scale[:, :n].t().double().repeat_interleave(128, 1)[:, :width]
    step = scale[:, :n].t().double().repeat_interleave(128, 1)[:, :width]
    close(back, x[:n].double(), 1.0001 * (x[:n].double().abs() * 2 ** -4 + step * 2 ** -10))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [s for s in QSHAPES if s[2]])
def test_quantize_gated(shape, dtype):
    rows, used, width, more, qmore = shape
    g = gen(14)
    x = strided(rows, 2 * width, more, 0, dtype, g=g)[1]
    x[:, :width] *= 8
    q = eight_bits(rows, width, qmore)
    scale = torch.full((-(-width // 128), rows), 9.0, device=DEV)
    count = torch.tensor([used], dtype=torch.int32, device=DEV)
    ex.Quantize(x, q, scale, rows_ptr=count, gate="silu").run(stream())
    n = max(0, min(used, rows))
    gate, up = x[:n, :width].double(), x[:n, width:].double()
    v = gate * torch.sigmoid(gate) * up
    # 2^x to 2 ulp and its argument's rounding (|g| half steps, of which the 1 in 1 + exp(-g) leaves
    # less than 1.3 where |silu| is largest), a reciprocal to 1 ulp, a sum and two products of half a
    # step each: below 10 half steps
    amax = blocked(v).abs().amax(-1)
    close(scale[:, :n].t(), (amax / 448).clamp(min=torch.finfo(F32).tiny), 10 * u(F32) * amax / 448)
    step = scale[:, :n].t().double().repeat_interleave(128, 1)[:, :width]
    back = q[:n].double() * step
    close(back, v, 1.0001 * (v.abs() * 2 ** -4 + step * 2 ** -10))
    assert (scale[:, n:] == 9.0).all()
    assert (q[n:].contiguous().view(torch.uint8) == 0x55).all()


def test_quantize_of_zeros_extremes_and_what_is_no_number():
    x = torch.zeros(8, 300, device=DEV)
    x[1] = 1e-45                       # below the smallest scale
    x[2, 5] = 3e38
    x[3, 5] = float("inf")
    x[4, 200] = float("nan")
    x[5] = torch.finfo(F32).tiny * 448
    x[6] = -448.0
    q, scale = eight_bits(8, 300), torch.empty(3, 8, device=DEV)
    ex.Quantize(x, q, scale).run(stream())
    want_q, want_scale = quantized(x)
    assert torch.equal(torch.isnan(scale), torch.isnan(want_scale))
    assert torch.equal(scale.nan_to_num(7.0), want_scale.nan_to_num(7.0))
    fine = torch.isfinite(x).all(1)
    assert same_bits(q[fine], want_q[fine])
    assert scale[0, 3] == float("inf") and torch.isnan(scale[1, 4])
    assert torch.isnan(q[3, 5].float()) and torch.isnan(q[4, 200].float())
    assert (scale[1:, 3] == torch.finfo(F32).tiny).all() and (q[4, :128].float() == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 8, 4096), (7, 3, 1111), (64, 8, 128),
                                   (33, 40, 200), (300, 4, 2048), (0, 2, 64), (4, 2, 0)])
def test_dispatch_quantize(shape, dtype):
    tokens, top_k, width = shape
    r, _ = routing(tokens, top_k, 16)
    x = rand(gen(15), tokens, width, dtype=dtype)
    q = eight_bits(tokens * top_k, width)
    scale = torch.full((-(-width // 128), tokens * top_k), 9.0, device=DEV)
    ex.DispatchQuantize(r, x, q, scale).run(stream())
    _, row, token = pair_parts(r)
    want_q, want_scale = quantized(x)
    assert same_bits(q[row], want_q[token])
    assert torch.equal(scale[:, row], want_scale[:, token])
    rest = torch.ones(tokens * top_k, dtype=torch.bool, device=DEV)
    rest[row] = False
    assert (scale[:, rest] == 9.0).all()
    assert (q[rest].contiguous().view(torch.uint8) == 0x55).all()


# --------------------------------------------------------------------------------------- products
def weights(g, groups, n, k, more=0):
    w = rand(g, groups, n, -(-k // 16) * 16 + more).to(E4M3)[:, :, :k]
    return w, rand(g, groups, -(-n // 128), -(-k // 128), lo=0.5, hi=2.0)


def activations(g, rows, k, more=0):
    base = torch.empty(rows, -(-k // 16) * 16 + more, dtype=E4M3, device=DEV)
    base.copy_((rand(g, *base.shape) * 4).to(E4M3))
    return base[:, :k], rand(g, -(-k // 128), rows, lo=0.5, hi=2.0)


def product_oracle(a, sa, w, sw, ptr):
    """(values, size of the terms) in 64 bits, rows of no group zero."""
    n, k = w.shape[1:]
    ad = a.double() * sa.t().double().repeat_interleave(128, 1)[:, :k]
    want = torch.zeros(a.shape[0], n, dtype=F64, device=DEV)
    size = torch.zeros_like(want)
    for g in range(w.shape[0]):
        lo, hi = ptr[g], ptr[g + 1]
        if hi > lo:
            wd = sw[g].double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
            wd = w[g].double() * wd
            want[lo:hi] = ad[lo:hi] @ wd.t()
            size[lo:hi] = ad[lo:hi].abs() @ wd.abs().t()
    return want, size


def product_tol(want, size, k, dtype):
    """A block's 128 products are exact in fp32; their sum, and the scaled sums of the blocks, are
    off by at most a whole step (2 u, were a sum cut instead of rounded) per addition, the scales'
    product and the scaling by two more."""
    terms = 128 + 2 * (-(-k // 128)) + 4
    return terms * 2 * u(F32) * size + u(dtype) * want.abs() * 1.01 + s(dtype)


PRODUCTS = [  # rows of each group (first and last: rows of no group), n, k
    ([0, 1, 0], 1, 1), ([0, 1, 0], 128, 128), ([0, 5, 0], 130, 200), ([0, 128, 0], 256, 512),
    ([3, 7, 0, 1, 129, 0, 2, 5], 257, 1000), ([0, 0, 0, 0], 64, 64), ([4, 64, 65, 63, 0], 500, 333),
    ([0, 300, 0], 1000, 640), ([0, 1, 1, 1, 1, 0, 2, 0], 512, 2048), ([0, 33, 0], 96, 4100),
    ([0, 1000, 1, 500, 7], 384, 256), ([0, 16, 17, 31, 32, 3], 200, 144), ([0, 9, 1], 40, 17),
    ([0, 260, 515, 0], 640, 1152), ([0, 8, 0], 4096, 2048), ([0, 1, 0], 7000, 4096),
    ([2, 0, 0, 0, 1500, 2], 300, 384)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", PRODUCTS, ids=[f"{sum(c[0])}x{c[1]}x{c[2]}" for c in PRODUCTS])
def test_scaled_product(case, dtype):
    counts, n, k = case
    groups, rows = len(counts) - 2, sum(counts)
    g = gen(17)
    a, sa = activations(g, rows, k)
    w, sw = weights(g, groups, n, k)
    ptr = np.cumsum(counts[:-1]).tolist()
    dptr = torch.tensor(ptr, dtype=torch.int32, device=DEV)
    base = torch.full((rows, n + 3), 9.0, device=DEV, dtype=dtype)
    y = base[:, :n]
    ex.ScaledProduct(a, sa, w, sw, y, expert_ptr=dptr).run(stream())
    want, size = product_oracle(a, sa, w, sw, ptr)
    ex.check_products()
    close(y[ptr[0]:ptr[-1]], want[ptr[0]:ptr[-1]],
          product_tol(want, size, k, dtype)[ptr[0]:ptr[-1]])
    assert (base[:, n:] == 9.0).all()
    assert (base[:ptr[0]] == 9.0).all() and (base[ptr[-1]:] == 9.0).all()


@pytest.mark.parametrize("rows,n,k,more", [(1, 100, 100, 0), (37, 257, 384, 16), (200, 1, 129, 48),
                                           (513, 640, 1024, 0), (0, 64, 64, 0), (1, 1, 16, 16)])
def test_scaled_product_of_one_matrix(rows, n, k, more):
    g = gen(18)
    a, sa = activations(g, rows, k, more)
    w, sw = weights(g, 1, n, k, more)
    y = torch.empty(rows, n, device=DEV)
    ex.ScaledProduct(a, sa, w[0], sw[0], y).run(stream())
    want, size = product_oracle(a, sa, w, sw, [0, rows])
    close(y, want, product_tol(want, size, k, F32))


def test_scaled_product_where_nothing_is_a_number():
    """A NaN in a row of a, or in its scale, reaches that row alone; one in w its column alone."""
    rows, n, k = 70, 260, 300
    g = gen(19)
    a, sa = activations(g, rows, k)
    w, sw = weights(g, 1, n, k)
    nan = torch.tensor([0x7f], dtype=torch.uint8, device=DEV).view(E4M3)
    a[11, 290], w[0, 200, 5] = nan[0], nan[0]
    sa[1, 40] = float("inf")
    y = torch.empty(rows, n, device=DEV)
    ex.ScaledProduct(a, sa, w[0], sw[0], y).run(stream())
    fine = torch.isfinite(y)
    want = torch.ones(rows, n, dtype=torch.bool, device=DEV)
    want[11], want[:, 200] = False, False
    assert not fine[40].any()
    want[40] = False
    assert torch.equal(fine, want)


def test_scaled_product_of_offsets_that_are_none():
    """Offsets outside the rows, or falling ones, are cut to the rows: nothing is read or written
    outside the operands."""
    rows, n, k = 50, 64, 128
    g = gen(20)
    a, sa = activations(g, rows, k)
    w, sw = weights(g, 4, n, k)
    base = torch.full((rows + 20, n), 9.0, device=DEV)
    for offsets in ([-5, 10, 7, 2 ** 31 - 1, 60], [60, 70, 80, 90, 100], [-9, -8, -7, -6, -5],
                    [0, 0, 50, 0, 50]):
        ptr = torch.tensor(offsets, dtype=torch.int32, device=DEV)
        ex.ScaledProduct(a, sa, w, sw, base[:rows], expert_ptr=ptr).run(stream())
        assert (base[rows:] == 9.0).all()
        assert torch.isfinite(base).all()


def test_scaled_product_far_offsets():
    """Rows and matrices whose offsets pass 2^31 and 2^32 bytes."""
    g = gen(21)
    k, n = 1 << 16, 128
    rows = (1 << 16) + 40           # a: over 4 GiB
    a = torch.zeros(rows, k, dtype=torch.uint8, device=DEV).view(E4M3)
    a[-3:] = rand(g, 3, k).to(E4M3)
    sa = torch.ones(k // 128, rows, device=DEV)
    w = rand(g, 1, n, k).to(E4M3)
    sw = torch.ones(1, 1, k // 128, device=DEV)
    y = torch.full((rows, n), 9.0, device=DEV)
    ptr = torch.tensor([rows - 3, rows], dtype=torch.int32, device=DEV)
    ex.ScaledProduct(a, sa, w, sw, y, expert_ptr=ptr).run(stream())
    want = a[-3:].double() @ w[0].double().t()
    size = a[-3:].double().abs() @ w[0].double().abs().t()
    close(y[-3:], want, product_tol(want, size, k, F32))
    assert (y[:-3] == 9.0).all()
    # the same rows through dispatch and combine
    r = ex.Routes(3, 1, torch.tensor([rows - 1, 0, rows - 2], dtype=torch.int32, device=DEV))
    h = torch.zeros(rows, k, dtype=BF16, device=DEV)
    x = rand(g, 3, k, dtype=BF16)
    ex.Dispatch(r, x, h).run(stream())
    assert torch.equal(h[[rows - 1, 0, rows - 2]], x)
    back = torch.empty_like(x)
    ex.Combine(r, h, back).run(stream())
    assert torch.equal(back, x)


# ------------------------------------------------------------------------------- as they are used
def layer(tokens, top_k, experts, width, inner, seed=0):
    """A layer of experts in 8 bits: the calls in order, and what they read and write."""
    g = gen(seed)
    t = {"ids": torch.zeros(tokens, top_k, dtype=torch.int64, device=DEV),
         "x": torch.zeros(tokens, width, dtype=BF16, device=DEV),
         "gates": torch.zeros(tokens, top_k, device=DEV)}
    pairs = tokens * top_k
    i32 = dict(dtype=torch.int32, device=DEV)
    t["ptr"], t["row_pair"], t["pair_row"] = (torch.zeros(m, **i32)
                                              for m in (experts + 1, pairs, pairs))
    ws = torch.empty(ex.route_workspace_bytes(tokens, top_k, experts), dtype=torch.uint8,
                     device=DEV)
    t["q1"], t["s1"] = eight_bits(pairs, width), torch.ones(-(-width // 128), pairs, device=DEV)
    t["w1"], t["sw1"] = weights(g, experts, 2 * inner, width)
    t["mid"] = torch.zeros(pairs, 2 * inner, dtype=BF16, device=DEV)
    t["q2"], t["s2"] = eight_bits(pairs, inner), torch.ones(-(-inner // 128), pairs, device=DEV)
    t["w2"], t["sw2"] = weights(g, experts, width, inner)
    t["h"] = torch.zeros(pairs, width, dtype=BF16, device=DEV)
    t["y"] = torch.zeros(tokens, width, dtype=BF16, device=DEV)
    r = ex.Routes(tokens, top_k, t["pair_row"])
    calls = [ex.Route(t["ids"], experts, t["ptr"], t["row_pair"], t["pair_row"], ws),
             ex.DispatchQuantize(r, t["x"], t["q1"], t["s1"]),
             ex.ScaledProduct(t["q1"], t["s1"], t["w1"], t["sw1"], t["mid"], expert_ptr=t["ptr"]),
             ex.Quantize(t["mid"], t["q2"], t["s2"], rows_ptr=t["ptr"][-1:], gate="silu"),
             ex.ScaledProduct(t["q2"], t["s2"], t["w2"], t["sw2"], t["h"], expert_ptr=t["ptr"]),
             ex.Combine(r, t["h"], t["y"], weights=t["gates"])]
    return t, calls


def new_inputs(t, experts, seed):
    g = gen(seed)
    tokens, top_k = t["ids"].shape
    t["ids"].copy_(ids_for(g, tokens, top_k, experts, "wild"))
    t["x"].copy_(rand(g, *t["x"].shape, dtype=BF16))
    t["gates"].copy_(rand(g, tokens, top_k, lo=0.0))


def check_layer(t, experts):
    """Each step against its definition on the step's own inputs (the bounds of the single tests)."""
    ids = t["ids"]
    want_ptr, order, want_rows = route_oracle(ids, experts)
    assert np.array_equal(t["ptr"].cpu().numpy(), want_ptr)
    assert np.array_equal(t["pair_row"].cpu().numpy(), want_rows)
    kept, top_k = order.size, ids.shape[1]
    token = torch.from_numpy(order // top_k).to(DEV)
    q, scale = quantized(t["x"])
    assert same_bits(t["q1"][:kept], q[token]) and torch.equal(t["s1"][:, :kept], scale[:, token])
    for a, sa, w, sw, y in (("q1", "s1", "w1", "sw1", "mid"), ("q2", "s2", "w2", "sw2", "h")):
        want, size = product_oracle(t[a], t[sa], t[w], t[sw], want_ptr.tolist())
        close(t[y][:kept], want[:kept], product_tol(want, size, t[w].shape[2], BF16)[:kept])
    inner = t["mid"].shape[1] // 2
    gate, up = t["mid"][:kept, :inner].double(), t["mid"][:kept, inner:].double()
    v = gate * torch.sigmoid(gate) * up
    step = t["s2"][:, :kept].t().double().repeat_interleave(128, 1)[:, :inner]
    close(t["q2"][:kept].double() * step, v, 1.0001 * (v.abs() * 2 ** -4 + step * 2 ** -10) + 1e-30)
    term = torch.zeros(ids.numel(), t["h"].shape[1], dtype=F64, device=DEV)
    term[torch.from_numpy(order).to(DEV)] = t["h"][:kept].double()
    term = term.view(*ids.shape, -1) * t["gates"].double()[..., None]
    want = term.sum(1)
    close(t["y"], want, top_k * u(F32) * term.abs().sum(1) * 1.01 + u(BF16) * want.abs() * 1.01
          + s(BF16))


@pytest.mark.parametrize("tokens,top_k,experts,width,inner", [
    (1, 2, 8, 256, 128), (16, 8, 64, 512, 200), (333, 4, 12, 400, 144)])
def test_layer_of_experts(tokens, top_k, experts, width, inner):
    t, calls = layer(tokens, top_k, experts, width, inner)
    new_inputs(t, experts, 31)
    for c in calls:
        c.run(stream())
    check_layer(t, experts)


def test_layer_of_experts_captured_and_replayed():
    """Two graphs of two layers, each with its own buffers, replayed in turn on new inputs."""
    cases = [(24, 4, 16, 256, 128), (700, 2, 8, 384, 256)]
    made = []
    for case in cases:
        t, calls = layer(*case)
        new_inputs(t, case[2], 40)
        for c in calls:
            c.run(stream())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for c in calls:
                c.run(stream())
        made.append((t, case[2], graph))
    for seed in (41, 42):
        for t, experts, graph in made:
            new_inputs(t, experts, seed)
            graph.replay()
        torch.cuda.synchronize()
        for t, experts, _ in made:
            check_layer(t, experts)


FIRST_IN_A_CAPTURE = """
import sys
sys.path[:0] = {paths!r}
import torch
import test_experts_gpu as t
for case in ((24, 4, 16, 256, 128), (3000, 8, 8, 384, 256)):
    made, calls = t.layer(*case)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c in calls:
            c.run(t.stream())
    t.new_inputs(made, case[2], 40)
    graph.replay()
    t.check_layer(made, case[2])
print("ok")
"""


def test_a_process_s_first_calls_are_captured():
    """Nothing is set up by a first call outside of a capture."""
    code = FIRST_IN_A_CAPTURE.format(paths=[str(Path(__file__).parent), *map(str, sys.path)])
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "ok" in r.stdout, r.stderr[-2000:]


def test_route_captured_and_replayed():
    """A route of two kernels, the second of which starts before the first has ended, replayed on new
    ids, back to back and each time after a kernel that writes them."""
    tokens, top_k, experts = 9000, 4, 200
    ids = torch.zeros(tokens, top_k, dtype=torch.int32, device=DEV)
    call, *out = route(ids, experts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call.run(stream())
        call.run(stream())
    for seed in range(4):
        ids.copy_(ids_for(gen(seed), tokens, top_k, experts, "wild"))
        out[1].fill_(-7)
        graph.replay()
        check_route(ids, experts, *out)


def test_a_call_in_another_thread_and_on_the_default_stream():
    """Calls are made from the thread that has the data; errors are a thread's own."""
    import threading
    t, calls = layer(40, 2, 8, 256, 128)
    new_inputs(t, 8, 70)
    torch.cuda.synchronize()
    failed = []

    def work():
        try:
            for c in calls:
                c.run()
            with pytest.raises(ap.ApptError):
                ex.Dispatch(ex.Routes(1, 1, ex.Dense(0, (1,), "i32")), t["x"][:1], t["y"][:1]).run()
        except BaseException as e:   # for the test's own thread
            failed.append(e)

    th = threading.Thread(target=work)
    th.start()
    th.join()
    torch.cuda.synchronize()
    assert not failed, failed
    check_layer(t, 8)


def test_layers_on_two_streams_and_equal_bits():
    """Two layers at once on streams of their own, a side stream's work ordered by the stream
    alone; the same inputs again give the same bits."""
    made = [layer(500, 4, 16, 384, 128, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in made]
    for t, _ in made:
        new_inputs(t, 16, 50)
    torch.cuda.synchronize()
    first = None
    for _ in range(3):
        for (t, calls), st in zip(made, streams):
            with torch.cuda.stream(st):
                t["y"].zero_()
                for c in calls:
                    c.run(st.cuda_stream)
        torch.cuda.synchronize()
        now = [t["y"].clone() for t, _ in made]
        if first is None:
            first = now
            for t, _ in made:
                check_layer(t, 16)
        for a, b in zip(first, now):
            assert torch.equal(a, b)


def test_training_step_through_dispatch_and_combine():
    """Rows to experts, each expert's own factor, and back: gradients of the inputs, the factors
    and the weights against the plain form's by autograd in fp64."""
    tokens, top_k, experts, width = 60, 3, 7, 130
    r, ptr = routing(tokens, top_k, experts)
    pair, row, token = pair_parts(r)
    g = gen(60)
    x, c = rand(g, tokens, width, dtype=F64), rand(g, tokens, width, dtype=F64)
    f, w = rand(g, experts, width, dtype=F64), rand(g, tokens, top_k, dtype=F64)
    kept = int(ptr[-1])
    owner = torch.searchsorted(ptr[1:].long(), torch.arange(kept, device=DEV), right=True)

    leaves = [v.clone().requires_grad_() for v in (x, f, w)]
    rows_of = torch.empty(kept, dtype=torch.long, device=DEV)
    rows_of[row] = token
    pair_of = torch.empty(kept, dtype=torch.long, device=DEV)
    pair_of[row] = pair
    h = leaves[0][rows_of] * leaves[1][owner]
    y = torch.zeros(tokens, width, dtype=F64, device=DEV).index_add(
        0, rows_of, h * leaves[2].flatten()[pair_of][:, None])
    (y * c).sum().backward()

    rows = torch.zeros(tokens * top_k, width, dtype=F64, device=DEV)
    ex.Dispatch(r, x, rows).run(stream())
    hidden = rows.clone()
    hidden[:kept] *= f[owner]
    out = torch.empty(tokens, width, dtype=F64, device=DEV)
    ex.Combine(r, hidden, out, weights=w).run(stream())
    close(out, y.detach(), 1e-13)
    dhidden, dw = torch.zeros_like(hidden), torch.empty_like(w)
    ex.CombineGrad(r, c, hidden, weights=w, dh=dhidden, dweights=dw).run(stream())
    df = torch.zeros_like(f).index_add_(0, owner, dhidden[:kept] * rows[:kept])
    drows = torch.zeros_like(rows)
    drows[:kept] = dhidden[:kept] * f[owner]
    dx = torch.empty_like(x)
    ex.Combine(r, drows, dx).run(stream())
    # up to 180 rows of 130 terms, each below 1, in sums of 2^-53 a term
    for got, leaf in zip((dx, df, dw), leaves):
        close(got, leaf.grad, 1e-11)


def test_refusals_that_need_a_device():
    x = torch.zeros(4, 8, device=DEV)
    y = torch.zeros(8, 8, device=DEV)
    r = ex.Routes(4, 2, torch.zeros(8, dtype=torch.int32, device=DEV))
    host = torch.zeros(4, 8)
    d = ex.Dense(host.data_ptr(), (4, 8), "f32")
    with pytest.raises(ap.ApptError, match="not memory of device"):
        ex.Dispatch(r, d, y).run(stream())
    pinned = torch.zeros(4, 8).pin_memory()
    with pytest.raises(ap.ApptError, match="not memory of device"):
        ex.Dispatch(r, ex.Dense(pinned.data_ptr(), (4, 8), "f32"), y).run(stream())
    for device in (63, -1):
        far = [ex.Dense(t.data_ptr(), tuple(t.shape), "f32", device=device) for t in (x, y)]
        rows = ex.Dense(r.pair_row.data_ptr(), (8,), "i32", device=device)
        with pytest.raises(ap.ApptError, match="device ordinal"):
            ex.Dispatch(ex.Routes(4, 2, rows), *far).run(stream())
    before = ap.kernel_launches()
    ex.Dispatch(r, x, y).run(stream())
    assert ap.kernel_launches() == before + 1
    torch.cuda.synchronize()
