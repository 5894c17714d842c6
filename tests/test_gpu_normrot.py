"""GPU: head norms with rotary positions (rnn_norm_rotary_*, NormRotary) against
their plain statement in 64 bits.

Tolerances, element by element, U = 2^-24.  Forward: x^ and its product with the
gain are rounded once each (2 U), then the turn: 3 U and 1e-8 for the angle of
|a| + |b| (as rotary positions alone): (5 U + 1e-8) (|a| + |b|) of the normed
pair, second orders below 1e-9.  Backward: the gradient turned back, du, is off by
e = (3 U + 1e-8) (|da| + |db|); x^ by 2 U (1 / norm and the product), t = gain du by
U besides.  mean(t x^): a product and up to eight additions in 32 bits (the lanes'
sums are in 64), so 2 + 1 + 1 + 8 = 12 U of mean |t x^| with its operands' errors.  dx =
(t - x^ mean) / norm: U |t|, x^'s 2 U, the mean's 12 U and its rounding, the
difference's rounding U (|t| + |x^| mean |t x^|), 2 U |dx| for the last product:
U (2 |t| + 17 |x^| mean |t x^|) / norm + 2 U |dx|, and e as it goes through.  dgain: the
sum of (e + 2 U |du|) |x^|, and U |dgain|."""
import pytest
import torch

from decayref import D, U, head_norm, norm_rotary, pair_size, turn
from test_gpu_rotary import grid_pos

pytestmark = pytest.mark.gpu

# name, n, grid, hq, hk, dh, pairs, interleaved, xoff, xextra, yoff, yextra
CASES = [
    ("one", 1, (1,), 1, 0, 2, None, False, 0, 0, 0, 0),
    ("keys_only", 2, (5,), 0, 3, 16, None, False, 0, 0, 0, 0),
    ("line", 2, (37,), 3, 1, 16, None, False, 0, 0, 0, 0),
    ("image", 3, (8, 8), 4, 4, 64, None, False, 0, 512, 0, 0),
    ("image_inter", 3, (8, 8), 4, 4, 64, None, True, 0, 512, 0, 0),
    ("video", 2, (4, 5, 6), 5, 5, 64, None, False, 0, 0, 64, 4),
    ("video_inter", 2, (4, 5, 6), 4, 1, 32, (8, 4, 4), True, 4, 4, 0, 0),
    ("odd", 2, (3, 7), 5, 2, 13, (3, 2), False, 1, 2, 3, 1),
    ("odd_inter", 2, (3, 7), 5, 2, 13, (3, 2), True, 1, 2, 3, 1),
    ("part", 2, (5, 5), 4, 2, 52, (8, 8), False, 0, 0, 0, 0),
    ("part_inter", 2, (5, 5), 4, 2, 52, (12, 8), True, 0, 0, 0, 0),
    ("unaligned", 2, (5, 5), 4, 2, 64, None, False, 1, 4, 0, 0),
    ("idle_axis", 1, (4, 4, 4), 2, 2, 24, (0, 6, 6), False, 0, 0, 0, 0),
    ("no_pairs", 2, (4,), 2, 1, 8, (0,), False, 0, 0, 0, 0),
    ("wide", 1, (300,), 70, 10, 128, None, False, 0, 0, 0, 0),
    ("widest_head", 1, (9,), 2, 1, 256, None, False, 0, 0, 0, 0),
    ("widest_plain", 1, (9,), 2, 1, 255, (1,), False, 0, 0, 0, 0),
    ("many_rows", 24, (40, 40), 2, 1, 20, None, False, 0, 0, 0, 0),
]


def inputs(c, rows, seed=1):
    _, n, grid, hq, hk, dh, pairs, inter, xoff, xex, yoff, yex = c
    g, w = torch.Generator().manual_seed(seed), (hq + hk) * dh
    x = torch.full((rows, xoff + w + xex), float("nan"))
    x[:, xoff:xoff + w] = torch.randn(rows, w, generator=g) * 3
    return x, torch.randn(2, dh, generator=g), torch.randn(rows, w, generator=g)


def tolerances(x, gain, dy, hq, hk, dh, pairs, inter, eps, want):
    """What y, dx and dgain may be off by; x, gain, dy in 64 bits."""
    heads = hq + hk
    hat = head_norm(x.view(-1, heads, dh), eps)
    gh = (torch.ones(heads, dh, dtype=D) if gain is None else gain[[0] * hq + [1] * hk]).abs()
    ty = (5 * U + 1.1e-8) * pair_size((hat * gh).reshape(x.shape), heads, dh, pairs, inter)
    e = (3 * U + 1.1e-8) * pair_size(dy, heads, dh, pairs, inter).view(hat.shape)
    rn = 1 / torch.sqrt((x.view(hat.shape) ** 2).mean(-1, keepdim=True) + eps)
    du = want["du"].abs().view(hat.shape)
    tx = rn * (gh * e + hat.abs() * (gh * e * hat.abs()).mean(-1, keepdim=True))
    tx += U * rn * (2 * gh * du + 17 * hat.abs() * (gh * du * hat.abs()).mean(-1, keepdim=True))
    tx = 1.01 * (tx.reshape(x.shape) + 2 * U * want["dx"].abs())
    s = 1.01 * ((e + 2 * U * du) * hat.abs()).sum(0)
    tg = torch.stack([s[:hq].sum(0), s[hq:].sum(0)]) + 1.01 * U * want["dgain"].abs()
    return ty + 1e-37, tx + 1e-37, tg + 1e-37


def statement(x, gain, dy, hq, hk, dh, pos, pairs, base, inter, eps):
    x, gain = x.requires_grad_(True), gain.requires_grad_(True)
    y = norm_rotary(x, gain, hq, hk, dh, pos, pairs, base, inter, eps)
    dx, dgain = torch.autograd.grad(y, (x, gain), dy)
    x.requires_grad_(False), gain.requires_grad_(False)
    du = turn(dy, hq + hk, dh, pos, pairs, base, inter, inverse=True)
    return dict(y=y.detach(), dx=dx, dgain=dgain, du=du)


@pytest.mark.parametrize("c", CASES, ids=[c[0] for c in CASES])
def test_grid(rnn, c):
    _, n, grid, hq, hk, dh, pairs, inter, xoff, xex, yoff, yex = c
    op = rnn.NormRotary(hq, hk, dh, grid, 100.0, pairs, inter, eps=1e-3)
    w, rows, pairs = (hq + hk) * dh, n * op.t, op.rot.pairs
    x, gain, dy = inputs(c, rows)
    src, pos = x[:, xoff:xoff + w].to(D), grid_pos(grid, n)
    want = statement(src, gain.to(D), dy.to(D), hq, hk, dh, pos, pairs, 100.0, inter, 1e-3)
    ty, tx, tg = tolerances(src, gain.to(D), dy.to(D), hq, hk, dh, pairs, inter, 1e-3, want)
    X, G, DY = x.cuda(), gain.cuda(), dy.cuda()
    y = torch.full((rows, yoff + w + yex), 7.0).cuda()
    op.forward(n, X, X.shape[1], xoff, G, y=y, ystride=y.shape[1], yoff=yoff)
    got = y.cpu()
    assert ((got[:, yoff:yoff + w] - want["y"]).abs() <= ty).all()
    assert (got[:, :yoff] == 7.0).all() and (got[:, yoff + w:] == 7.0).all()
    xi = X.clone()
    op.forward(n, xi, X.shape[1], xoff, G, y=xi)  # in place
    assert torch.equal(xi.cpu()[:, xoff:xoff + w], got[:, yoff:yoff + w])
    assert torch.isnan(xi.cpu()[:, :xoff]).all() and torch.isnan(xi.cpu()[:, xoff + w:]).all()
    new = op.forward(n, X, X.shape[1], xoff, G)
    assert torch.equal(new.cpu().reshape(rows, w), got[:, yoff:yoff + w])
    # backward: into a wider buffer, in place of dy, into a new tensor
    dx = torch.full((rows, yoff + w + yex), 7.0).cuda()
    dgain = torch.zeros(2, dh).cuda()
    op.backward(n, X, X.shape[1], xoff, G, DY, w, 0, dgain, dx=dx, dxstride=dx.shape[1], dxoff=yoff)
    dxc = dx.cpu()
    assert ((dxc[:, yoff:yoff + w] - want["dx"]).abs() <= tx).all()
    assert ((dgain.cpu() - want["dgain"]).abs() <= tg).all()
    assert (dxc[:, :yoff] == 7.0).all() and (dxc[:, yoff + w:] == 7.0).all()
    assert torch.equal(op.backward(n, X, X.shape[1], xoff, G, DY, w).cpu().reshape(rows, w),
                       dxc[:, yoff:yoff + w])
    keep, dg = DY.clone(), dgain.clone()
    op.backward(n, X, X.shape[1], xoff, G, keep, w, 0, dg, dx=keep)
    assert torch.equal(keep.cpu(), dxc[:, yoff:yoff + w])
    assert torch.equal(dg, dgain + dgain)  # accumulates: the same sum once more


def test_no_gain_is_a_gain_of_one(rnn):
    op = rnn.NormRotary(3, 2, 32, (6, 5), 100.0)
    x, dy = torch.randn(2, 30, 160).cuda(), torch.randn(2, 30, 160).cuda()
    one = torch.ones(2, 32).cuda()
    assert torch.equal(op.forward(2, x, 160), op.forward(2, x, 160, 0, one))
    assert torch.equal(op.backward(2, x, 160, 0, None, dy, 160),
                       op.backward(2, x, 160, 0, one, dy, 160))


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("far", [0.0, 1.5e7])
def test_explicit_positions(rnn, far, inter):
    n, t, hq, hk, dh, pairs = 3, 19, 2, 2, 48, (10, 7, 7)
    g = torch.Generator().manual_seed(2)
    pos = (torch.randn(n * t, 3, generator=g) * 50 + far).float()
    x, dy = (torch.randn(n * t, 4 * dh, generator=g) for _ in range(2))
    gain = torch.randn(2, dh, generator=g)
    op = rnn.NormRotary(hq, hk, dh, (2, 2, 2), 10000.0, pairs, inter)
    want = statement(x.to(D), gain.to(D), dy.to(D), hq, hk, dh, pos, pairs, 10000.0, inter, 1e-6)
    ty, tx, tg = tolerances(x.to(D), gain.to(D), dy.to(D), hq, hk, dh, pairs, inter, 1e-6, want)
    dgain = torch.zeros(2, dh).cuda()
    y = op.forward(n, x.cuda(), 4 * dh, 0, gain.cuda(), pos=pos.cuda(), t=t)
    dx = op.backward(n, x.cuda(), 4 * dh, 0, gain.cuda(), dy.cuda(), 4 * dh, 0, dgain,
                     pos=pos.cuda(), t=t)
    assert ((y.cpu().reshape(n * t, -1) - want["y"]).abs() <= ty).all()
    assert ((dx.cpu().reshape(n * t, -1) - want["dx"]).abs() <= tx).all()
    assert ((dgain.cpu() - want["dgain"]).abs() <= tg).all()


@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e19, 1e38])
def test_heads_of_any_size_keep_their_norm(rnn, size):
    """Squares past a float's range, and below it."""
    op = rnn.NormRotary(2, 1, 16, (4,), 100.0, eps=1e-38)
    g = torch.Generator().manual_seed(5)
    x = (torch.rand(4, 48, generator=g) + 0.5).float() * size
    dy = torch.randn(4, 48, generator=g)
    one = torch.ones(2, 16, dtype=D)
    pos = grid_pos((4,), 1)
    eps = float(torch.tensor(1e-38))
    want = statement(x.to(D), one, dy.to(D), 2, 1, 16, pos, op.rot.pairs, 100.0, False, eps)
    ty, tx, _ = tolerances(x.to(D), one, dy.to(D), 2, 1, 16, op.rot.pairs, False, eps, want)
    assert ((op.forward(1, x.cuda(), 48).cpu()[0] - want["y"]).abs() <= ty).all()
    dx = op.backward(1, x.cuda(), 48, 0, None, dy.cuda(), 48).cpu()[0]
    # results below a float's normal range are whole multiples of 2^-149
    assert ((dx - want["dx"]).abs() <= tx + 2.0 ** -149).all()


def test_zero_heads(rnn):
    """A head of zeros has no direction: y = 0, dx = gain dy / sqrt(eps), dgain = 0."""
    op = rnn.NormRotary(1, 1, 8, (1,), 100.0, (0,), eps=0.25)
    x, dy = torch.zeros(1, 1, 16).cuda(), torch.randn(1, 1, 16).cuda()
    dgain = torch.zeros(2, 8).cuda()
    assert (op.forward(1, x, 16) == 0).all()
    dx = op.backward(1, x, 16, 0, torch.ones(2, 8).cuda(), dy, 16, 0, dgain)
    assert torch.equal(dx, 2 * dy) and (dgain == 0).all()


def test_not_a_number_stays_in_its_head(rnn):
    op = rnn.NormRotary(3, 3, 32, (8,), 100.0)
    x = torch.randn(1, 8, 192).cuda()
    clean = op.forward(1, x, 192)
    bad = x.clone()
    bad[0, 3, 70] = float("nan")
    bad[0, 5, 130] = float("inf")
    y = op.forward(1, bad, 192).view(8, 6, 32)
    assert torch.isnan(y[3, 2]).all() and torch.isnan(y[5, 4]).any()
    keep = torch.ones(8, 6, dtype=torch.bool)
    keep[3, 2] = keep[5, 4] = False
    assert torch.equal(y[keep.cuda()], clean.view(8, 6, 32)[keep.cuda()])


def test_an_infinity_leaves_zeros_in_its_head(rnn):
    """As the formula has it: NaN in its own pair, x / infinity in the others."""
    op = rnn.NormRotary(1, 1, 32, (8,), 100.0, (12,))
    x = torch.randn(1, 8, 64).cuda()
    for ch, pair in ((5, (5, 17)), (17, (5, 17)), (30, (30,))):
        bad = x.clone()
        bad[0, 3, 32 + ch] = -float("inf")
        y = op.forward(1, bad, 64).view(8, 2, 32)[3, 1].cpu()
        shows = torch.zeros(32, dtype=torch.bool)
        shows[list(pair)] = True
        assert torch.isnan(y[shows]).all() and (y[~shows] == 0).all()


def test_offsets_past_32_bits(rnn):
    """2200 rows of 2^21 floats."""
    op, wide = rnn.NormRotary(2, 1, 16, (2200,), 100.0), 1 << 21
    x, dy, gain = torch.randn(2200, 48).cuda(), torch.randn(2200, 48).cuda(), torch.randn(2, 16).cuda()
    X = torch.empty(2200, wide, device="cuda")
    X[:, -48:] = x
    y = op.forward(1, x, 48, 0, gain)
    dg = [torch.zeros_like(gain) for _ in range(2)]
    dx = op.backward(1, x, 48, 0, gain, dy, 48, 0, dg[0])
    DX = torch.empty_like(X)
    op.backward(1, X, wide, wide - 48, gain, dy, 48, 0, dg[1], dx=DX, dxstride=wide,
                dxoff=wide - 48)
    assert torch.equal(DX[:, -48:], dx[0]) and torch.equal(dg[0], dg[1])
    op.forward(1, X, wide, wide - 48, gain, y=X)
    assert torch.equal(X[:, -48:], y[0])


def test_gradient_against_differences(rnn):
    """A step along the gradient, central: the outputs' rounding over the step
    (8 U sqrt of the elements over 2^-9) and the third order, 2^-18 of it, stay
    below 1e-3 of the change."""
    op = rnn.NormRotary(3, 2, 32, (6, 5), 100.0)
    g = torch.Generator().manual_seed(6)
    x, dy = (torch.randn(2, 30, 160, generator=g).cuda() for _ in range(2))
    gain = torch.randn(2, 32, generator=g).cuda()
    dgain = torch.zeros_like(gain)
    dx = op.backward(2, x, 160, 0, gain, dy, 160, 0, dgain)
    f = lambda a, b: (op.forward(2, a, 160, 0, b).double() * dy.double()).sum()
    for v, d in ((0, dx), (1, dgain)):
        s = 2.0 ** -9 / float(d.abs().max()) * d
        up, dn = ((f(x + s, gain), f(x - s, gain)) if v == 0 else (f(x, gain + s), f(x, gain - s)))
        want = 2 * (s.double() * d.double()).sum()
        assert abs(float(up - dn - want)) <= 1e-3 * float(want)


def test_refusals(rnn):
    op = rnn.NormRotary(3, 1, 32, (8, 8))
    x = torch.zeros(2, 64, 128, device="cuda")
    gain = torch.ones(2, 32, device="cuda")
    with pytest.raises(ValueError):
        op.forward(3, x, 128)  # too few rows
    with pytest.raises(TypeError):
        op.forward(2, x.half(), 128)
    with pytest.raises(TypeError):
        op.forward(2, x, 128, 0, gain.cpu())
    with pytest.raises(ValueError):
        op.forward(2, x, 128, 0, gain[0].contiguous())  # the queries' gain alone
    with pytest.raises(ValueError):
        op.forward(2, x, 128, t=63)  # not the grid's tokens
    with pytest.raises(ValueError):
        op.forward(2, x, 100)  # heads do not fit a row
    with pytest.raises(rnn.RnnError):
        op.forward(1, x, 128, 0, y=x, ystride=160)  # in place with two layouts
    with pytest.raises(rnn.RnnError):
        op.backward(2, x, 128, 0, gain, x, 128, dx=x)  # dx over the input
    with pytest.raises(rnn.RnnError):
        op.backward(2, x, 128, 0, None, x.clone(), 128, 0, gain)  # dgain without gain
    with pytest.raises(rnn.RnnError):
        op.backward(2, x, 128, 0, gain, torch.zeros(2, 64, 128, device="cuda"), 127)
    assert op.forward(0, x, 128).shape == (0, 64, 128)
    dgain = torch.ones_like(gain)
    assert op.backward(0, x, 128, 0, gain, x, 128, 0, dgain).shape == (0, 64, 128)
    assert (dgain == 1).all()
