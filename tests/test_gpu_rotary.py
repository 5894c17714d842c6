"""GPU: rotary positions (rnn_rotary, Rotary) against their plain statement in
64 bits.

Tolerance, element by element: sine and cosine are rounded once (2^-24 each),
then one product and one fused multiply-add: at most 2^-24 (2 |u| + 2 |v| +
|u| + |v|), so 3 2^-24 (|u| + |v|); the angle's own error, 2^-52 of at most
2^24 quarter turns and the power's last bit, adds 1e-8 of |u| + |v|."""
import pytest
import torch

from diffref import rotary

pytestmark = pytest.mark.gpu


def bound(x, heads, dh, pairs, inter):
    v = x.abs().double().reshape(-1, heads, dh)
    R = sum(pairs)
    tol = torch.zeros_like(v)
    if R:
        ia = torch.arange(R) * 2 if inter else torch.arange(R)
        ib = ia + (1 if inter else R)
        s = (v[..., ia] + v[..., ib]) * (3 * 2.0 ** -24 + 1e-8)
        tol[..., ia] = s
        tol[..., ib] = s
    return tol.reshape(x.shape)


def grid_pos(grid, n):
    axes = [torch.arange(s) for s in grid]
    p = torch.stack([m.reshape(-1) for m in torch.meshgrid(*axes, indexing="ij")], -1)
    return p.repeat(n, 1)


# name, n, grid, heads, dh, pairs, interleaved, xoff, xextra, yoff, yextra
CASES = [
    ("one", 1, (1,), 1, 2, None, False, 0, 0, 0, 0),
    ("line", 2, (37,), 3, 16, None, False, 0, 0, 0, 0),
    ("image", 3, (8, 8), 16, 32, None, False, 0, 256, 0, 0),
    ("image_inter", 3, (8, 8), 16, 32, None, True, 0, 256, 0, 0),
    ("video", 2, (4, 5, 6), 5, 64, None, False, 0, 0, 64, 4),
    ("video_inter", 2, (4, 5, 6), 5, 64, (16, 8, 8), True, 4, 4, 0, 0),
    ("odd", 2, (3, 7), 5, 13, (3, 2), False, 1, 2, 3, 1),
    ("odd_inter", 2, (3, 7), 5, 13, (3, 2), True, 1, 2, 3, 1),
    ("rest_copied", 2, (5, 5), 4, 32, (4, 4), False, 0, 0, 0, 0),
    ("rest_inter", 2, (5, 5), 4, 32, (8, 4), True, 0, 0, 0, 0),
    ("idle_axis", 1, (4, 4, 4), 2, 24, (0, 6, 6), False, 0, 0, 0, 0),
    ("no_pairs", 2, (4,), 2, 8, (0,), False, 0, 0, 0, 0),
    ("wide", 1, (300,), 70, 128, None, False, 0, 0, 0, 0),
    ("widest_head", 1, (9,), 2, 512, None, False, 0, 0, 0, 0),
]


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("c", CASES, ids=[c[0] for c in CASES])
def test_grid(rnn, c, inverse):
    _, n, grid, heads, dh, pairs, inter, xoff, xex, yoff, yex = c
    rot = rnn.Rotary(heads, dh, grid, 100.0, pairs, inter)
    w, g = heads * dh, torch.Generator().manual_seed(1)
    rows = n * rot.t
    x = torch.full((rows, xoff + w + xex), float("nan"))
    x[:, xoff:xoff + w] = torch.randn(rows, w, generator=g)
    y = torch.full((rows, yoff + w + yex), 7.0).cuda()
    fn = rot.backward if inverse else rot.forward
    got = fn(n, x.cuda(), x.shape[1], xoff, y=y, ystride=y.shape[1], yoff=yoff).cpu()
    src = x[:, xoff:xoff + w]
    want = rotary(src, heads, dh, grid_pos(grid, n), rot.pairs, 100.0, inter, inverse)
    assert ((got[:, yoff:yoff + w] - want).abs() <= bound(src, heads, dh, rot.pairs, inter)).all()
    assert (got[:, :yoff] == 7.0).all() and (got[:, yoff + w:] == 7.0).all()
    # in place, and into a new tensor
    xi = x.cuda()
    fn(n, xi, x.shape[1], xoff, y=xi)
    assert torch.equal(xi.cpu()[:, xoff:xoff + w], got[:, yoff:yoff + w])
    assert torch.isnan(xi.cpu()[:, :xoff]).all() and torch.isnan(xi.cpu()[:, xoff + w:]).all()
    new = fn(n, x.cuda(), x.shape[1], xoff)
    assert torch.equal(new.cpu().reshape(rows, w), got[:, yoff:yoff + w])


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("far", [0.0, 1e3, 1.5e7])
def test_explicit_positions(rnn, far, inter):
    """Given positions: fractional, negative and far ones, no grid needed."""
    n, t, heads, dh = 3, 19, 4, 48
    g = torch.Generator().manual_seed(2)
    pos = (torch.randn(n * t, 3, generator=g) * 50 + far).float()
    x = torch.randn(n * t, heads * dh, generator=g)
    rot = rnn.Rotary(heads, dh, (2, 2, 2), 10000.0, (10, 7, 7), inter)
    got = rot.forward(n, x.cuda(), heads * dh, pos=pos.cuda(), t=t).cpu().reshape(n * t, -1)
    want = rotary(x, heads, dh, pos, rot.pairs, 10000.0, inter)
    assert ((got - want).abs() <= bound(x, heads, dh, rot.pairs, inter)).all()


def test_backward_is_the_transpose(rnn):
    """<turn(x), dy> = <x, back(dy)>, and differences: the turn is linear, so
    a difference of any step is the derivative up to the outputs' rounding."""
    rot = rnn.Rotary(6, 32, (7, 9), 100.0)
    g = torch.Generator().manual_seed(3)
    x, dy, d = (torch.randn(2, 63, 192, generator=g).cuda() for _ in range(3))
    y, dx = rot.forward(2, x, 192), rot.backward(2, dy, 192)
    a, b = (y.double() * dy.double()).sum(), (x.double() * dx.double()).sum()
    size = float(x.double().norm() * dy.double().norm())
    assert abs(float(a - b)) <= 6 * 2.0 ** -24 * size
    up, down = rot.forward(2, x + d, 192), rot.forward(2, x - d, 192)
    num = ((up.double() - down.double()) * dy.double()).sum() / 2
    want = (d.double() * dx.double()).sum()
    size = float((x.double().norm() + d.double().norm()) * dy.double().norm())
    assert abs(float(num - want)) <= 8 * 2.0 ** -24 * size


def test_captured_and_replayed(rnn):
    st = torch.cuda.Stream()
    ctx = rnn.Context(0, stream=st)
    rot = rnn.Rotary(8, 32, (8, 8), 100.0, ctx=ctx)
    x = torch.randn(2, 64, 256, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        want = rot.forward(2, x, 256)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        y = rot.forward(2, x, 256)
    for _ in range(3):
        with torch.cuda.stream(st):
            y.zero_()
            graph.replay()
        st.synchronize()
        assert torch.equal(y, want)
    ctx.close()


def test_refusals(rnn):
    rot = rnn.Rotary(4, 32, (8, 8))
    x = torch.zeros(2, 64, 128, device="cuda")
    with pytest.raises(ValueError):
        rot.forward(3, x, 128)  # too few rows
    with pytest.raises(TypeError):
        rot.forward(2, x.half(), 128)
    with pytest.raises(TypeError):
        rot.forward(2, x.cpu(), 128, y=x)
    with pytest.raises(rnn.RnnError):
        rot.forward(2, x, 128, t=63)  # not the grid's tokens
    with pytest.raises(rnn.RnnError):
        rot.forward(2, x, 100)  # heads do not fit a row
    with pytest.raises(rnn.RnnError):
        rot.forward(1, x, 128, 0, y=x, ystride=160)  # in place with two layouts
    with pytest.raises(ValueError):
        rot.forward(2, x, 128, pos=torch.zeros(5, 2, device="cuda"))
    assert rot.forward(0, x, 128).shape == (0, 64, 128)
