"""GPU: the Linear product with an activation (rnn_linear_act_*) where rows,
features and channels are of very different size: each row and each column of a
result against its own statement in 64 bits.

Tolerance: an element a of a sum's operand is within 2^-23 |a| + 2^-35 max |a| of
itself, the maximum over the elements of that sum: its two fp16 parts are of 11
bits each while the second is above 2^-14, and steps of 2^-24 below, at a power of
two that takes the maximum to 2^10 at least (2^-25 / 2^10 = 2^-35).  A result's error
is then a few times 2^-23 of the root of the sum of its terms' squares, for which
TOL (1e-5) stands, and 2^-35 max |a| |b| + 2^-35 |a| max |b| over the terms, which
shows where the elements of one sum lie 2^12 apart and more."""
import pytest
import torch

from conftest import TOL
from diffref import D
from test_gpu_linear_act import inputs

pytestmark = pytest.mark.gpu

# one for each tile of y and dX, and of dW with and without splits of its rows
SIZES = [(8192, 256, 160), (2048, 256, 160), (1813, 387, 251), (130, 70, 90), (4100, 129, 384),
         (200, 130, 140), (4099, 129, 40), (65, 33, 129)]


def close(got, a, b, what):
    """got = a b (64 bits) by row and by column."""
    amax, bmax = a.abs().amax(1, keepdim=True), b.abs().amax(0, keepdim=True)
    err = (got.cpu().to(D) - a @ b) ** 2
    size = TOL ** 2 * ((a * a) @ (b * b)) + 2.0 ** -70 * (
        amax ** 2 * (b * b).sum(0) + (a * a).sum(1, keepdim=True) * bmax ** 2)
    for d in (0, 1):
        e, s = err.sum(d), size.sum(d)
        assert (e <= s).all(), (what, d, float((e / s.clamp(min=1e-300)).max()) ** 0.5)


def spread(n, seed):
    """Powers of two from 2^-36 to 2^24, in no order."""
    g = torch.Generator().manual_seed(seed)
    return 2.0 ** torch.randint(-36, 25, (n,), generator=g).float()


def run(rnn, size, x, w, b, dy, slope):
    X, W, B, DY = (t.cuda() for t in (x, w, b, dy))
    y, _ = rnn.linear_act_forward(*size, X, W, None, "none")
    dw, db = torch.zeros_like(W), torch.zeros_like(B)
    name = "none" if slope is None else "gelu"  # (slope: as a forward would have kept it)
    dx = rnn.linear_act_backward(*size, DY, X, W, None if slope is None else slope.cuda(), name, dw, db)
    return y, dx, dw, db


@pytest.mark.parametrize("sloped", [False, True])
@pytest.mark.parametrize("which", ["features", "channels", "rows"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes_apart(rnn, size, which, sloped):
    """Features (columns of x; with them W's, the other way, so that y sums terms
    of one size), channels (rows of W, columns of dy) and rows of 2^-36 to 2^24."""
    rows, fin, fout = size
    x, w, b, _, dy = inputs(*size, seed=1)
    slope = torch.rand(rows, fout, generator=torch.Generator().manual_seed(2)) if sloped else None
    if which == "features":
        f = spread(fin, 3)
        x, w = x * f, w / f
    elif which == "channels":
        f = spread(fout, 4)
        w, dy = w * f[:, None], dy / f
        if sloped:
            slope = slope * spread(fout, 5)
    else:
        f = spread(rows, 6)[:, None]
        x, dy = x * f, dy / f
    y, dx, dw, db = run(rnn, size, x, w, b, dy, slope)
    X, W = x.to(D), w.to(D)
    dz = dy.to(D) if slope is None else (dy * slope).to(D)  # (one rounding of the product)
    close(y, X, W.T, "y")
    close(dx, dz, W, "dx")
    close(dw, dz.T, X, "dw")
    err = (db.cpu().to(D) - dz.sum(0)).abs()
    assert (err <= 1e-6 * dz.norm(dim=0)).all()


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes_that_grow_along_the_sum(rnn, size):
    """Rows from 2^-30 to 2^30 in order: dW's powers of two follow from stage to
    stage, each column's at its own pace."""
    rows, fin, fout = size
    x, w, b, _, dy = inputs(*size, seed=7)
    up = 2.0 ** torch.linspace(-30, 30, rows).round()[:, None]
    late = (torch.arange(rows)[:, None] >= torch.arange(fin) * rows // fin)
    x = torch.where(late, x * up, x * 2.0 ** -30)
    _, dx, dw, _ = run(rnn, size, x, w, b, dy, None)
    close(dw, dy.to(D).T, x.to(D), "dw")
    x2 = torch.where(late, torch.ones(()), up.flip(0) * torch.ones(fin))
    _, _, dw, _ = run(rnn, size, x2, w, b, dy, None)
    close(dw, dy.to(D).T, x2.to(D), "dw back")
    cols = 2.0 ** torch.linspace(-30, 30, fout).round()  # and dX's
    _, dx, _, _ = run(rnn, size, x, w * cols[:, None], b, dy, None)
    close(dx, dy.to(D), (w * cols[:, None]).to(D), "dx")


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_what_is_not_finite_stays_in_its_sums(rnn, size, bad):
    """A NaN or an infinity in x, W or dy: NaN in the sums that take it, and every
    other sum as before, bit for bit."""
    rows, fin, fout = size
    x, w, b, _, dy = inputs(*size, seed=8)
    r, i, o = rows // 2, fin // 3, fout // 2
    y0, dx0, dw0, db0 = run(rnn, size, x, w, b, dy, None)

    def same(got, ref, hit):
        assert torch.isnan(got[hit]).all()
        got[hit] = ref[hit]
        assert torch.equal(got, ref)

    x1 = x.clone()
    x1[r, i] = bad
    y, dx, dw, db = run(rnn, size, x1, w, b, dy, None)
    same(y, y0, (r, slice(None)))
    same(dw, dw0, (slice(None), i))
    assert torch.equal(dx, dx0) and torch.equal(db, db0)
    w1 = w.clone()
    w1[o, i] = bad
    y, dx, dw, db = run(rnn, size, x, w1, b, dy, None)
    same(y, y0, (slice(None), o))
    same(dx, dx0, (slice(None), i))
    dy1 = dy.clone()
    dy1[r, o] = bad
    y, dx, dw, db = run(rnn, size, x, w, b, dy1, None)
    same(dx, dx0, (r, slice(None)))
    same(dw, dw0, (o, slice(None)))
    assert not torch.isfinite(db[o])
