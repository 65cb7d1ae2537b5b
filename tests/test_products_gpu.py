"""The 8-bit product on the GPU: what is left where a product gives up a wait."""
import pytest
import torch

from test_experts_gpu import (DEV, F32, activations, ap, close, ex, gen, product_oracle, product_tol,
                              stream, weights)

pytestmark = pytest.mark.gpu


# rows, n, k, groups of equal sizes: K split over a cluster (with shares of one and of many blocks),
# rows as columns without a split, and rows as lanes with 128 and 256 columns, tiles in turn
GIVING_UP = [(50, 130, 128, 1), (1, 4096, 4096, 1), (40, 128, 1200, 1), (512, 4096, 640, 64), (2500, 1000, 1700, 1),
             (6000, 2048, 900, 2)]


@pytest.fixture
def giving_up():
    ex.check_products()
    ex.make_products_give_up(True)
    yield
    ex.make_products_give_up(False)


@pytest.mark.parametrize("rows,n,k,groups", GIVING_UP)
def test_a_product_that_gives_up(rows, n, k, groups, giving_up):
    """It ends, writes nothing outside its rows and columns, and is reported once; the next one on
    the same buffers is right."""
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
    for outside in (base[0], base[rows + 1:], base[:, n:]):
        assert (outside == 9.0).all()
    ex.make_products_give_up(False)
    call.run(stream())
    ex.check_products()
    want, size = product_oracle(a, sa, w, sw, ptr)
    close(base[1:rows + 1, :n], want, product_tol(want, size, k, F32))
    for outside in (base[0], base[rows + 1:], base[:, n:]):
        assert (outside == 9.0).all()


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
