"""The 8-bit product on the GPU: tiles of many rows, far and unordered offsets, and what is left
where a product gives up a wait."""
import numpy as np
import pytest
import torch

from test_experts_gpu import (BF16, DEV, E4M3, F16, F32, activations, ap, close, ex, gen,
                              product_oracle, product_tol, rand, stream, weights)

pytestmark = pytest.mark.gpu


# rows, n, k, groups of equal sizes: K split over a cluster (with shares of one and of many blocks),
# rows as columns without a split, and rows as lanes with 128 and 256 columns, tiles in turn
GIVING_UP = [(50, 130, 128, 1), (1, 4096, 4096, 1), (40, 128, 1200, 1), (512, 4096, 640, 64),
             (2500, 1000, 1700, 1), (6000, 2048, 900, 2)]


@pytest.fixture
def giving_up():
    ex.check_products()
    ex.make_products_give_up(True)
    yield
    ex.make_products_give_up(False)


@pytest.mark.parametrize("rows,n,k,groups", GIVING_UP)
def test_a_product_that_gives_up(rows, n, k, groups, giving_up):
    """It ends, leaves NaN where it has not computed, which here is everywhere, and nothing outside
    its rows and columns, and is reported once; the next one on the same buffers is right."""
    g = gen(90)
    a, sa = activations(g, rows, k)
    w, sw = weights(g, groups, n, k)
    ptr = [rows * i // groups for i in range(groups + 1)]
    base = torch.full((rows + 3, n + 8), 9.0, device=DEV)
    call = ex.ScaledProduct(a, sa, w, sw, base[1:rows + 1, :n],
                            torch.tensor(ptr, dtype=torch.int32, device=DEV))
    call.run(stream())
    with pytest.raises(ap.ApptError, match="gave up"):
        ex.check_products()
    ex.check_products()
    assert torch.isnan(base[1:rows + 1, :n]).all()
    for outside in (base[0], base[rows + 1:], base[:, n:]):
        assert (outside == 9.0).all()
    ex.make_products_give_up(False)
    call.run(stream())
    ex.check_products()
    want, size = product_oracle(a, sa, w, sw, ptr)
    close(base[1:rows + 1, :n], want, product_tol(want, size, k, F32))
    for outside in (base[0], base[rows + 1:], base[:, n:]):
        assert (outside == 9.0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", [(3, 260), (60, 260), (1300, 1037), (2500, 1037)])
def test_what_reads_a_product_that_gave_up(rows, n, dtype, giving_up):
    """The next steps of a layer get NaN, not the buffer's old values: rows of no group keep theirs."""
    g = gen(98)
    k = 700
    a, sa = activations(g, rows, k)
    w, sw = weights(g, 2, n, k)
    y = torch.full((rows, n + n % 2), 9.0, device=DEV, dtype=dtype)
    ptr = [1, rows // 2, rows - 1]
    dptr = torch.tensor(ptr, dtype=torch.int32, device=DEV)
    q = torch.zeros(rows, n // 2, dtype=torch.uint8, device=DEV).view(E4M3)
    scale = torch.zeros(-(-(n // 2) // 128), rows, device=DEV)
    ex.ScaledProduct(a, sa, w, sw, y[:, :n], expert_ptr=dptr).run(stream())
    ex.Quantize(y[:, :n // 2 * 2], q, scale, gate="silu").run(stream())
    with pytest.raises(ap.ApptError, match="gave up"):
        ex.check_products()
    assert torch.isnan(y[1:rows - 1, :n]).all() and torch.isnan(scale[:, 1:rows - 1]).all()
    assert (y[0] == 9.0).all() and (y[rows - 1] == 9.0).all() and (y[:, n:] == 9.0).all()
    assert torch.isfinite(scale[:, 0]).all()


def test_a_captured_product_that_gives_up(giving_up):
    """A graph keeps what it was captured with; its replays are reported like calls."""
    g = gen(91)
    a, sa = activations(g, 300, 512)
    w, sw = weights(g, 1, 256, 512)
    y = torch.zeros(300, 256, device=DEV)
    call = ex.ScaledProduct(a, sa, w[0], sw[0], y)
    graphs = []
    for on in (True, False):
        ex.make_products_give_up(on)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call.run(stream())
    for _ in range(2):
        graphs[0].replay()
        graphs[1].replay()
        with pytest.raises(ap.ApptError, match="gave up"):
            ex.check_products()
    graphs[1].replay()
    ex.check_products()
    want, size = product_oracle(a, sa, w, sw, [0, 300])
    close(y, want, product_tol(want, size, 512, F32))


# ------------------------------------------------------------------------------ many rows per group
def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


# rows of each group (first and last: rows of no group), columns of y, their tile on 148 SMs
MANY = [([0, 2500, 0], 1000, (128, 256)), ([0, 1300, 0], 1000, (128, 128)),
        ([5, 1000, 0, 1, 31, 32, 33, 2000, 129, 2900, 3], 1037, (128, 256)),
        ([3, 700, 0, 63, 700, 2], 1037, (128, 128))]
MANY_IDS = [f"{sum(c)}x{n}-tile{t[1]}" for c, n, t in MANY]


def check_product(y, base, first, a, sa, w, sw, ptr, k, dtype):
    """y (base's columns up to its own) holds the product in the groups' rows and 9 elsewhere."""
    n = y.shape[1]
    want, size = product_oracle(a, sa, w, sw, ptr)
    tol = product_tol(want, size, k, dtype)
    inside = torch.zeros(y.shape[0], dtype=torch.bool, device=DEV)
    for lo, hi in zip(ptr, ptr[1:]):
        inside[lo:hi] = True
    close(y[inside], want[inside], tol[inside])
    assert (y[~inside] == 9.0).all()
    assert (base[:, :first] == 9.0).all() and (base[:, first + n:] == 9.0).all()


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("k", [17, 128, 300, 4100])
@pytest.mark.parametrize("case", MANY, ids=MANY_IDS)
def test_products_of_many_rows(case, k, dtype, aligned):
    """aligned: rows of y start on 16 bytes and leave by TMA, but for a group's last rows; else one
    element further, from shared memory."""
    counts, n, tile = case
    groups, rows = len(counts) - 2, sum(counts)
    if sms() == 148:
        assert ex.product_tile(rows, n, groups, sms()) == tile
    g = gen(93)
    a, sa = activations(g, rows, k)
    w, sw = weights(g, groups, n, k)
    ptr = np.cumsum(counts[:-1]).tolist()
    first = 0 if aligned else 1
    base = torch.full((rows, -(-n // 8) * 8 + (8 if aligned else 11)), 9.0, device=DEV, dtype=dtype)
    y = base[:, first:first + n]
    dptr = torch.tensor(ptr, dtype=torch.int32, device=DEV)
    ex.ScaledProduct(a, sa, w, sw, y, expert_ptr=dptr).run(stream())
    ex.check_products()
    check_product(y, base, first, a, sa, w, sw, ptr, k, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", [(2500, 1000), (1300, 1000)])
def test_many_rows_where_nothing_is_a_number(rows, n, dtype):
    """A NaN in a row of a, or an infinity in its scale, reaches that row alone, one in w its column
    alone, and one in w's scale its 128 columns."""
    k = 400
    g = gen(94)
    a, sa = activations(g, rows, k)
    w, sw = weights(g, 1, n, k)
    nan = torch.tensor([0x7f], dtype=torch.uint8, device=DEV).view(E4M3)
    a[130, 390], a[rows - 1, 0], w[0, 200, 5] = nan[0], nan[0], nan[0]
    sa[1, 40], sa[3, 1000] = float("inf"), float("nan")
    sw[0, 4, 2] = float("nan")
    y = torch.empty(rows, n, device=DEV, dtype=dtype)
    ex.ScaledProduct(a, sa, w[0], sw[0], y).run(stream())
    want = torch.ones(rows, n, dtype=torch.bool, device=DEV)
    want[[130, rows - 1, 40, 1000]], want[:, 200], want[:, 512:640] = False, False, False
    assert torch.equal(torch.isfinite(y), want)


# ------------------------------------------------------------------------------------------ offsets
@pytest.mark.parametrize("rows,n", [(50, 64), (300, 64), (1468, 1037), (6000, 1037)])
def test_offsets_that_are_none(rows, n):
    """Offsets are cut to the rows and each to the largest before it: what they then are is what is
    computed, rows of no group stay as they were."""
    k, groups = 128, 4
    g = gen(95)
    a, sa = activations(g, rows, k)
    w, sw = weights(g, groups, n, k)
    for offsets in ([-5, rows // 5, rows // 7, 2 ** 31 - 1, 60], [rows + 10, rows + 20, 0, 1, 100],
                    [-9, -8, -7, -6, -5], [0, 0, rows, 0, rows], [7, rows // 2, 3, rows - 2, -2 ** 31],
                    [rows // 3, rows // 3, rows // 2, rows // 2, rows // 2 + 1]):
        base = torch.full((rows + 20, n), 9.0, device=DEV)
        ptr = torch.tensor(offsets, dtype=torch.int32, device=DEV)
        ex.ScaledProduct(a, sa, w, sw, base[:rows], expert_ptr=ptr).run(stream())
        held = np.maximum.accumulate(np.clip(offsets, 0, rows)).tolist()
        check_product(base[:rows], base, 0, a, sa, w, sw, held, k, F32)
        assert (base[rows:] == 9.0).all()


def test_matrices_past_4_gib():
    """The last of five groups begins 4.5 GB behind the first."""
    rows, n, k, step = 200, 256, 512, (9 << 27) + 16
    store = torch.empty(4 * step + n * k, dtype=torch.uint8, device=DEV).view(E4M3)
    w = store.as_strided((5, n, k), (step, k, 1))
    g = gen(96)
    a, sa = activations(g, rows, k)
    some, sw = weights(g, 5, n, k)
    w.copy_(some)
    for per in (rows // 5, rows):      # all groups, or the last alone
        ptr = [max(0, rows - per * (5 - i)) for i in range(5)] + [rows]
        y = torch.full((rows, n), 9.0, device=DEV)
        dptr = torch.tensor(ptr, dtype=torch.int32, device=DEV)
        ex.ScaledProduct(a, sa, w, sw, y, expert_ptr=dptr).run(stream())
        check_product(y, y, 0, a, sa, some, sw, ptr, k, F32)


@pytest.mark.parametrize("rows,n,ld", [(2500, 1000, 1 << 19), (1300, 1000, 1 << 20),
                                       (2500, 1000, (1 << 19) + 1), (40, 200, 1 << 25),
                                       (2, 9000, (1 << 31) - 16)])
def test_rows_of_y_past_4_gib(rows, n, ld):
    """Rows of y whose addresses pass 2^31 elements or 2^32 bytes: by TMA, from shared memory, and
    straight from registers."""
    k = 256
    g = gen(97)
    a, sa = activations(g, rows, k)
    w, sw = weights(g, 1, n, k)
    store = torch.empty((rows - 1) * ld + n, device=DEV)
    y = store.as_strided((rows, n), (ld, 1))
    ex.ScaledProduct(a, sa, w[0], sw[0], y).run(stream())
    want, size = product_oracle(a, sa, w, sw, [0, rows])
    close(y, want, product_tol(want, size, k, F32))
