"""Routed products without a GPU: what the entry points and the binding refuse, and that a call
whose arguments hold gets as far as looking for a device. The addresses are never touched: every
check of sizes, pointers, alignment and overlap comes before the first CUDA call."""
import ctypes as ct

import pytest

import appt_spgemm as ap
from appt_spgemm import experts as ex

D = ex.Dense
MB = 1 << 20
NO_DEVICE = "status -6"


def at(i):
    """The i-th of a row of addresses far from each other."""
    return 1 << 32 | i << 28


def dense(i, rows, cols, type, ld=None, off=0):
    return D(at(i) + off, (rows, cols), type, (cols if ld is None else ld, 1))


def flat(i, n, type="i32", off=0):
    return D(at(i) + off, (n,), type)


def routes(tokens=4, top_k=2, i=15):
    return ex.Routes(tokens, top_k, flat(i, tokens * top_k))


def outcome(make):
    with pytest.raises(ap.ApptError) as e:
        make().run()
    return str(e.value)


no_gpu = pytest.mark.skipif(ap.device_count() > 0, reason="made-up addresses")

GOOD = {
    "route": lambda **k: ex.Route(**{**dict(
        ids=dense(0, 4, 2, "i64"), experts=8, expert_ptr=flat(1, 9), row_pair=flat(2, 8),
        pair_row=flat(3, 8), workspace=flat(4, 8)), **k}),
    "dispatch": lambda **k: ex.Dispatch(**{**dict(
        routes=routes(), x=dense(0, 4, 5, "bf16"), y=dense(1, 8, 5, "bf16"),
        weights=D(at(2), (4, 2), "f32")), **k}),
    "combine": lambda **k: ex.Combine(**{**dict(
        routes=routes(), h=dense(0, 8, 5, "f64"), y=dense(1, 4, 5, "f64"),
        weights=D(at(2), (4, 2), "f64")), **k}),
    "combine_grad": lambda **k: ex.CombineGrad(**{**dict(
        routes=routes(), dy=dense(0, 4, 5, "f16"), h=dense(1, 8, 5, "f16"),
        weights=D(at(2), (4, 2), "f32"), dh=dense(3, 8, 5, "f16"),
        dweights=D(at(4), (4, 2), "f32")), **k}),
    "quantize": lambda **k: ex.Quantize(**{**dict(
        x=dense(0, 8, 400, "f16"), q=dense(1, 8, 200, "e4m3"), scale=dense(2, 2, 8, "f32"),
        rows_ptr=flat(3, 1), gate="silu"), **k}),
    "dispatch_quantize": lambda **k: ex.DispatchQuantize(**{**dict(
        routes=routes(), x=dense(0, 4, 200, "bf16"), q=dense(1, 8, 200, "e4m3"),
        scale=dense(2, 2, 8, "f32")), **k}),
    "product": lambda **k: ex.ScaledProduct(**{**dict(
        a=dense(0, 8, 200, "e4m3", ld=208), a_scale=dense(1, 2, 8, "f32"),
        w=D(at(2), (3, 130, 200), "e4m3", (130 * 208, 208, 1)),
        w_scale=D(at(3), (3, 2, 2), "f32"), y=dense(4, 8, 130, "bf16"),
        expert_ptr=flat(5, 4)), **k}),
}


@no_gpu
@pytest.mark.parametrize("op", GOOD)
def test_a_call_that_holds_looks_for_a_device(op):
    assert NO_DEVICE in outcome(GOOD[op])


BAD = [
    # routes
    ("route", dict(experts=0, expert_ptr=flat(1, 1)), "experts"),
    ("route", dict(experts=1025, expert_ptr=flat(1, 1026)), "experts"),
    ("route", dict(ids=dense(0, 4, 2, "f32")), "ids"),
    ("route", dict(ids=dense(0, 4, 2, "i64", ld=1)), "ld"),
    ("route", dict(ids=dense(0, 4, 2, "i64", off=4)), "aligned"),
    ("route", dict(ids=dense(0, 4, 0, "i64"), row_pair=flat(2, 0), pair_row=flat(3, 0)), "column"),
    ("route", dict(expert_ptr=flat(1, 8)), "expert_ptr"),
    ("route", dict(row_pair=flat(2, 7)), "row_pair"),
    ("route", dict(row_pair=flat(2, 8, off=2)), "aligned"),
    ("route", dict(pair_row=flat(2, 8)), "overlaps"),
    ("route", dict(pair_row=flat(0, 8)), "overlaps"),
    ("route", dict(workspace=flat(4, 7)), "workspace"),
    ("route", dict(workspace=flat(4, 8, off=4)), "workspace"),
    ("route", dict(workspace=D(0, (8,), "i32")), "workspace"),
    # rows there and back
    ("dispatch", dict(x=dense(0, 5, 5, "bf16")), "token"),
    ("dispatch", dict(y=dense(1, 8, 6, "bf16")), "columns"),
    ("dispatch", dict(y=dense(1, 8, 5, "f16")), "type"),
    ("dispatch", dict(x=dense(0, 4, 5, "i32"), y=dense(1, 8, 5, "i32")), "type"),
    ("dispatch", dict(y=dense(0, 8, 5, "bf16")), "overlaps"),
    ("dispatch", dict(y=dense(1, 8, 5, "bf16", off=1)), "aligned"),
    ("dispatch", dict(y=dense(1, 8, 5, "bf16", ld=4)), "ld"),
    ("dispatch", dict(weights=D(at(2), (4, 3), "f32")), "weights"),
    ("dispatch", dict(weights=D(at(2), (4, 2), "f64")), "weights"),
    ("dispatch", dict(weights=D(at(2), (4, 2), "f32", (3, 1))), "contiguous"),
    ("dispatch", dict(x=D(0, (4, 5), "bf16")), "null"),
    ("dispatch", dict(routes=ex.Routes(4, 2, D(0, (8,), "i32"))), "pair_row"),
    ("dispatch", dict(routes=ex.Routes(4, 2, flat(15, 7))), "pair_row"),
    ("dispatch", dict(routes=(4, 2, flat(15, 8))), "Routes"),
    ("combine", dict(y=dense(1, 5, 5, "f64")), "token"),
    ("combine", dict(h=dense(0, 8, 4, "f64")), "columns"),
    ("combine", dict(weights=D(at(2), (4, 2), "f32")), "weights"),
    ("combine", dict(y=dense(2, 4, 5, "f64")), "overlaps"),
    ("combine_grad", dict(dh=None, dweights=None), "wanted"),
    ("combine_grad", dict(h=None), "needs H"),
    ("combine_grad", dict(dh=dense(3, 7, 5, "f16")), "rows"),
    ("combine_grad", dict(dh=dense(1, 8, 5, "f16")), "overlaps"),
    ("combine_grad", dict(dweights=D(at(2), (4, 2), "f32")), "overlaps"),
    # 8 bits
    ("quantize", dict(gate=None), "columns"),
    ("quantize", dict(gate="relu"), "gate"),
    ("quantize", dict(x=dense(0, 8, 400, "f64")), "type"),
    ("quantize", dict(q=dense(1, 8, 200, "f16")), "type"),
    ("quantize", dict(scale=dense(2, 1, 8, "f32")), "shape"),
    ("quantize", dict(scale=dense(2, 2, 8, "f32", ld=7)), "scale_ld"),
    ("quantize", dict(q=dense(0, 8, 200, "e4m3")), "overlaps"),
    ("quantize", dict(scale=dense(1, 2, 8, "f32")), "overlaps"),
    ("quantize", dict(rows_ptr=flat(3, 2)), "rows_ptr"),
    ("quantize", dict(rows_ptr=flat(1, 1)), "overlaps"),
    ("dispatch_quantize", dict(x=dense(0, 4, 100, "bf16")), "columns"),
    ("dispatch_quantize", dict(x=dense(0, 3, 200, "bf16")), "token"),
    ("product", dict(a=dense(0, 8, 200, "e4m3")), "multiple of 16"),
    ("product", dict(a=dense(0, 8, 200, "e4m3", ld=208, off=8)), "aligned"),
    ("product", dict(a=dense(0, 8, 100, "e4m3", ld=112), a_scale=dense(1, 1, 8, "f32")), "columns"),
    ("product", dict(w=D(at(2), (3, 130, 200), "e4m3")), "multiple of 16"),
    ("product", dict(w=D(at(2), (3, 130, 200), "e4m3", (100 * 208, 208, 1))), "group_stride"),
    ("product", dict(w=D(at(2) + 4, (3, 130, 200), "e4m3", (130 * 208, 208, 1))), "aligned"),
    ("product", dict(w_scale=D(at(3), (3, 2, 1), "f32")), "w_scale"),
    ("product", dict(expert_ptr=None), "one group"),
    ("product", dict(expert_ptr=flat(5, 3)), "expert_ptr"),
    ("product", dict(y=dense(4, 8, 131, "bf16")), "rows"),
    ("product", dict(y=dense(4, 7, 130, "bf16")), "rows"),
    ("product", dict(y=dense(4, 8, 130, "f64")), "type"),
    ("product", dict(y=dense(2, 8, 130, "bf16")), "overlaps"),
    ("product", dict(y=D(at(4), (8, 130), "bf16", device=1)), "device"),
    ("product", dict(w=D(at(2), (1025, 130, 200), "e4m3", (130 * 208, 208, 1)),
                     w_scale=D(at(3), (1025, 2, 2), "f32"), expert_ptr=flat(5, 1026)), "groups"),
    ("product", dict(a=D(at(0), (8, 0), "e4m3", (16, 1)), a_scale=D(at(1), (0, 8), "f32"),
                     w=D(at(2), (3, 130, 0), "e4m3", (2080, 16, 1)),
                     w_scale=D(at(3), (3, 2, 0), "f32")), "cols"),
]


@pytest.mark.parametrize("op,change,word", BAD, ids=[f"{o}-{i}" for i, (o, _, _) in enumerate(BAD)])
def test_refused(op, change, word):
    message = outcome(lambda: GOOD[op](**change))
    assert word in message and NO_DEVICE not in message, message


@no_gpu
def test_columns_of_one_buffer_do_not_overlap():
    # left and right half of the same rows; one column further they meet
    x, y = dense(0, 4, 8, "f32", ld=16), dense(0, 4, 8, "f32", ld=16, off=32)
    one = ex.Routes(4, 1, flat(15, 4))
    assert NO_DEVICE in outcome(lambda: ex.Dispatch(one, x, y))
    y = dense(0, 4, 8, "f32", ld=16, off=28)
    assert "overlaps" in outcome(lambda: ex.Dispatch(one, x, y))


def test_null_structures_and_reserved_fields():
    lib = ex._lib()
    m = ex.DenseArg(4, 4, 4, at(0), ex.TYPES["f32"], 0)
    r = ex.RoutesArg(4, 1, 0, at(1))
    b = ct.byref
    assert lib.appt_dispatch(None, b(m), None, b(m), 0, None) == -1
    assert lib.appt_dispatch(b(r), None, None, b(m), 0, None) == -1
    assert lib.appt_quantize(b(m), 0, None, None, 0, None) == -1
    assert lib.appt_scaled_product(None, None, None, b(m), 0, None) == -1
    assert lib.appt_route(None, 4, at(2), at(3), at(4), at(5), 1 << 20, 0, None) == -1
    y = ex.DenseArg(4, 4, 4, at(6), ex.TYPES["f32"], 7)
    assert lib.appt_dispatch(b(r), b(m), None, b(y), 0, None) == -1
    assert "reserved" in ap.last_error()
    for t in (-1, 7, 1 << 30):
        y = ex.DenseArg(4, 4, 4, at(6), t, 0)
        assert lib.appt_dispatch(b(r), b(m), None, b(y), 0, None) == -1
    big = ex.RoutesArg(1 << 30, 2, 0, at(1))
    assert lib.appt_dispatch(b(big), b(m), None, b(m), 0, None) == -1


def test_route_workspace():
    assert ex.route_workspace_bytes(0, 1, 1) > 0
    assert ex.route_workspace_bytes(1 << 20, 8, 1024) >= 1024 * 4
    for bad in ((-1, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 1025), (1 << 30, 2, 8)):
        with pytest.raises(ap.ApptError):
            ex.route_workspace_bytes(*bad)


def test_operands_that_are_no_tensors():
    with pytest.raises(ap.ApptError, match="needs a tensor"):
        ex.Dispatch(routes(), [1, 2], dense(1, 8, 5, "f32"))
    torch = pytest.importorskip("torch")
    with pytest.raises(ap.ApptError, match="not on a CUDA device"):
        ex.Dispatch(routes(), torch.zeros(4, 5), dense(1, 8, 5, "f32"))
    with pytest.raises(ap.ApptError, match="neighbours"):
        ex.Dispatch(routes(), D(at(0), (4, 5), "f32", (1, 4)), dense(1, 8, 5, "f32"))
    with pytest.raises(ap.ApptError, match="unknown type"):
        D(at(0), (4, 5), "e5m2")


@pytest.mark.parametrize("op,change", [
    ("dispatch", dict(x=dense(0, 4, 5, "bf16", ld=(1 << 31) - 2),
                      y=D(at(1), ((1 << 31) - 2, 5), "bf16", ((1 << 31) - 2, 1)))),
    ("combine", dict(h=D(at(1), ((1 << 31) - 2, 5), "f64", ((1 << 31) - 2, 1)))),
    ("quantize", dict(x=D(at(1), ((1 << 31) - 2, 400), "f32", ((1 << 31) - 2, 1)),
                      q=D(at(2), ((1 << 31) - 2, 200), "e4m3"),
                      scale=D(at(3), (2, (1 << 31) - 2), "f32"))),
    ("product", dict(w=D(at(2), ((1 << 30), 200), "e4m3", (1 << 36, 1)), expert_ptr=None,
                     w_scale=D(at(3), (1 << 23, 2), "f32"),
                     y=D(at(4), (8, 1 << 30), "bf16", (1 << 30, 1)))),
])
def test_operands_beyond_any_memory(op, change):
    # the spans of these would wrap 64-bit addresses
    message = outcome(lambda: GOOD[op](**change))
    assert "any memory" in message, message


@pytest.mark.parametrize("shape", [(3, 4, 2), (2, 3, 4), (24, 1, 1), (1, 6, 4), (3, 2, 3)])
def test_weights_scales_of_another_shape(shape):
    """As many scales as there are blocks, or nearly, but not one for each where it belongs."""
    long = dict(a=dense(0, 8, 400, "e4m3"), a_scale=dense(1, 4, 8, "f32"),
                w=D(at(2), (3, 130, 400), "e4m3"))
    message = outcome(lambda: GOOD["product"](**long, w_scale=D(at(3), shape, "f32")))
    assert "w_scale" in message and "(3, 2, 4)" in message, message
    one = {**long, "w": D(at(2), (130, 400), "e4m3"), "expert_ptr": None}
    message = outcome(lambda: GOOD["product"](**one, w_scale=D(at(3), (4, 2), "f32")))
    assert "w_scale" in message and "(2, 4)" in message, message


@no_gpu
def test_weights_scales_of_the_right_shape():
    long = dict(a=dense(0, 8, 400, "e4m3"), a_scale=dense(1, 4, 8, "f32"))
    assert NO_DEVICE in outcome(lambda: GOOD["product"](
        **long, w=D(at(2), (3, 130, 400), "e4m3"), w_scale=D(at(3), (3, 2, 4), "f32")))
    assert NO_DEVICE in outcome(lambda: GOOD["product"](
        **long, w=D(at(2), (130, 400), "e4m3"), w_scale=D(at(3), (2, 4), "f32"), expert_ptr=None))


def test_sizes_wider_than_the_arguments():
    """Numbers that a 32- or 64-bit argument would cut to small ones are refused as they are."""
    for bad in ((10, 2 ** 32 + 2, 8), (2 ** 64 + 10, 2, 8), (10, 2, 2 ** 64 + 8),
                (-2 ** 64 + 10, 2, 8), (10, -2 ** 32 + 2, 8), (10, 2, -2 ** 64 + 8)):
        with pytest.raises(ap.ApptError, match="experts"):
            ex.route_workspace_bytes(*bad)
    # four tokens with 2^32 + 2 choices each, of which two would be left
    wide = ex.Routes(4, 2 ** 32 + 2, flat(15, 4 * (2 ** 32 + 2)))
    message = outcome(lambda: GOOD["dispatch"](routes=wide, weights=None))
    assert "top_k" in message and NO_DEVICE not in message, message
    message = outcome(lambda: GOOD["route"](experts=2 ** 64 + 8, expert_ptr=flat(1, 2 ** 64 + 9)))
    assert "experts" in message and NO_DEVICE not in message, message


@pytest.mark.parametrize("rows,n,groups,tile", [
    (1, 4096, 1, (16, 128)), (16, 4096, 1, (16, 128)), (17, 4096, 1, (32, 128)),
    (128, 4096, 64, (16, 128)), (64, 8192, 1, (64, 128)), (513, 640, 1, (64, 128)),
    (1300, 1000, 1, (128, 128)), (2500, 1000, 1, (128, 256)), (32768, 2048, 64, (128, 256)),
    (8192, 8192, 1, (128, 256)), (0, 64, 1, (16, 128)), (1 << 30, 1 << 30, 1024, (128, 256))])
def test_tile_of_a_product(rows, n, groups, tile):
    assert ex.product_tile(rows, n, groups) == tile


def test_tile_of_no_product():
    for bad in ((-1, 64, 1), (4, 0, 1), (4, 64, 0), (4, 64, 1025), (2 ** 32 + 4, 64, 1),
                (4, 64, 1, 0), (4, 2 ** 64 + 64, 1)):
        with pytest.raises(ap.ApptError, match="sizes"):
            ex.product_tile(*bad)
