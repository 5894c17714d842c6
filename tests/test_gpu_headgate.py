"""GPU: normed and gated heads (rnn_head_gate_*, HeadGate) against their plain
statement in 64 bits.

Tolerances, element by element, U = 2^-24.  sigma(z): the power of two is within 2 U
(an ulp), two products and the sum round by U each, the reciprocal after a Newton
step is within 1.5 U: 6.5 U.  y: x^, the gain's, z's and the last product: 6.5 + 4,
11 U with second orders.  z (1 - sigma) is within (6.5 + 2) U |z|, f = 1 + z (1 - sigma) by
U |f| more, silu'(z) = sigma f within sigma (8.5 |z| + 8.5 |f|) U, dz besides by 5
roundings (x^'s two among them): |dy x^ gain| sigma (8.5 |z| + 14 |f|) U.  du = dy
silu(z) is within e = 8.5 U |du|; what follows is as for head norms with rotary
positions.  sigma below exp(-88) counts as 0."""
import pytest
import torch

from decayref import D, U, gate, head_norm

pytestmark = pytest.mark.gpu

# name, rows, h, d, zoff, zextra
CASES = [("one", 1, 1, 1, 0, 0), ("image", 64, 4, 64, 768, 0), ("tail", 37, 3, 20, 0, 4),
         ("odd", 53, 5, 77, 1, 2), ("unaligned", 9, 2, 64, 3, 0), ("few", 2, 16, 128, 0, 0),
         ("widest", 5, 2, 512, 0, 0), ("widest_odd", 5, 2, 511, 0, 1), ("many", 30000, 2, 24, 0, 0),
         ("many_heads", 3, 1100, 8, 0, 0)]


@pytest.mark.parametrize("c", CASES, ids=[c[0] for c in CASES])
def test_forward_backward(rnn, c):
    _, rows, h, d, zoff, zex = c
    g, w = torch.Generator().manual_seed(1), h * d
    x, dy = torch.randn(rows, w, generator=g) * 3, torch.randn(rows, w, generator=g)
    z = torch.full((rows, zoff + w + zex), float("nan"))
    z[:, zoff:zoff + w] = torch.randn(rows, w, generator=g) * 2
    gain, eps = torch.randn(w, generator=g), 1e-3
    leaves = [v.to(D).requires_grad_(True) for v in (x, z[:, zoff:zoff + w], gain)]
    y64 = gate(*leaves, h, d, eps)
    dx64, dz64, dg64 = torch.autograd.grad(y64, leaves, dy.to(D))
    x64, z64, g64 = (v.detach() for v in leaves)
    hat = head_norm(x64.view(-1, h, d), eps)
    sig = torch.sigmoid(z64)
    f = 1 + z64 * (1 - sig)
    u = (hat.reshape(rows, w) * g64).abs()
    e = 8.51 * U * (dy * z64 * sig).abs().view(hat.shape)
    gh = g64.abs().view(h, d)
    rn = 1 / torch.sqrt((x64.view(hat.shape) ** 2).mean(-1, keepdim=True) + eps)
    tx = rn * (gh * e + hat.abs() * (gh * e * hat.abs()).mean(-1, keepdim=True))
    t = gh * (dy * z64 * sig).abs().view(hat.shape)
    tx += U * rn * (2 * t + 17 * hat.abs() * (t * hat.abs()).mean(-1, keepdim=True))
    X, Z, G, DY = x.cuda(), z.cuda(), gain.cuda(), dy.cuda()
    op = rnn.HeadGate(h, d, eps)
    zs = z.shape[1]
    y = op.forward(rows, X, Z, zs, zoff, G)
    assert ((y.cpu() - y64.detach()).abs() <= 11 * U * y64.detach().abs() + 1e-37).all()
    xi = X.clone()
    assert torch.equal(op.forward(rows, xi, Z, zs, zoff, G, y=xi), y)  # in place
    dz, dgain = torch.full((rows, zoff + w + zex), 7.0).cuda(), torch.zeros(w).cuda()
    dx = op.backward(rows, X, Z, zs, zoff, G, DY, dz, zs, zoff, dgain)
    assert ((dx.cpu() - dx64).abs() <= 1.01 * (tx.reshape(rows, w) + 2 * U * dx64.abs()) + 1e-37).all()
    tz = (dy.abs() * u) * sig * (8.5 * z64.abs() + 14 * f.abs()) * U
    dzc = dz.cpu()
    assert ((dzc[:, zoff:zoff + w] - dz64).abs() <= 1.01 * tz + 1e-37).all()
    assert (dzc[:, :zoff] == 7.0).all() and (dzc[:, zoff + w:] == 7.0).all()
    du = (dy * z64 * sig).abs().view(hat.shape)
    tg = 1.01 * ((e + 2 * U * du) * hat.abs()).sum(0).reshape(-1) + 1.01 * U * dg64.abs() + 1e-37
    assert ((dgain.cpu() - dg64).abs() <= tg).all()
    # without dgain, over dy, and dz over z
    zz, dd = Z.clone(), DY.clone()
    op.backward(rows, X, zz, zs, zoff, G, dd, zz, zs, zoff, dx=dd)
    assert torch.equal(dd, dx) and torch.equal(zz.cpu()[:, zoff:zoff + w], dzc[:, zoff:zoff + w])
    again = dgain.clone()
    op.backward(rows, X, Z, zs, zoff, G, DY, dz, zs, zoff, again)
    assert torch.equal(again, dgain + dgain)


def test_no_gain_is_a_gain_of_one(rnn):
    op, one = rnn.HeadGate(3, 20), torch.ones(60).cuda()
    x, z, dy = (torch.randn(17, 60).cuda() for _ in range(3))
    assert torch.equal(op.forward(17, x, z, 60), op.forward(17, x, z, 60, 0, one))
    a, b = torch.empty_like(x), torch.empty_like(x)
    assert torch.equal(op.backward(17, x, z, 60, 0, None, dy, a, 60),
                       op.backward(17, x, z, 60, 0, one, dy, b, 60)) and torch.equal(a, b)


def test_far_gates_and_large_heads(rnn):
    """Gates beyond exp's range close or open; squares past a float's range."""
    op = rnn.HeadGate(1, 8, eps=1e-6)
    x = torch.full((1, 8), 1e30).cuda()
    z = torch.tensor([[-200.0, -89.0, -1e30, 0.0, 90.0, 200.0, 1e30, -0.0]]).cuda()
    y = op.forward(1, x, z, 8).cpu()[0]
    assert (y[:4].abs() <= 1e-36).all() and y[7] == 0
    assert torch.equal(y[4:7], torch.tensor([90.0, 200.0, 1e30]))
    dz = torch.empty_like(z)
    dx = op.backward(1, x, z, 8, 0, None, torch.ones_like(x), dz, 8).cpu()
    assert torch.isfinite(dx).all()
    assert (dz.cpu()[0, :3].abs() <= 1e-36).all() and (dz.cpu()[0, 4:7] == 1).all()


def test_numbers_that_are_none(rnn):
    op, g = rnn.HeadGate(2, 12), torch.Generator().manual_seed(7)
    x, z = (torch.randn(3, 24, generator=g).cuda() for _ in range(2))
    clean = op.forward(3, x, z, 24).view(3, 2, 12)
    nan, inf = float("nan"), float("inf")
    for v in (nan, inf):
        bad = x.clone()
        bad[1, 15] = v
        y = op.forward(3, bad, z, 24).view(3, 2, 12)
        assert torch.equal(y[::2], clean[::2]) and torch.equal(y[1, 0], clean[1, 0])
        rest = torch.cat([y[1, 1, :3], y[1, 1, 4:]])
        assert torch.isnan(y[1, 1, 3]) and (torch.isnan(rest).all() if v != v else (rest == 0).all())
        bad = z.clone()
        bad[1, 15] = v
        y = op.forward(3, x, bad, 24).view(3, 2, 12)
        assert not torch.isfinite(y[1, 1, 3])
        y[1, 1, 3] = clean[1, 1, 3]
        assert torch.equal(y, clean)


def test_offsets_past_32_bits(rnn):
    """Gates in 2200 rows of 2^21 floats."""
    op, wide, g = rnn.HeadGate(2, 12), 1 << 21, torch.Generator().manual_seed(8)
    x, z, dy = (torch.randn(2200, 24, generator=g).cuda() for _ in range(3))
    Z = torch.empty(2200, wide, device="cuda")
    Z[:, -24:] = z
    dz = torch.empty_like(z)
    dx = op.backward(2200, x, z, 24, 0, None, dy, dz, 24)
    assert torch.equal(op.forward(2200, x, Z, wide, wide - 24), op.forward(2200, x, z, 24))
    assert torch.equal(op.backward(2200, x, Z, wide, wide - 24, None, dy, Z, wide, wide - 24), dx)
    assert torch.equal(Z[:, -24:], dz)


def test_gradient_against_differences(rnn):
    """As for head norms with rotary positions: within 1e-3 of the change."""
    op = rnn.HeadGate(3, 40)
    g = torch.Generator().manual_seed(6)
    x, z, dy = (torch.randn(50, 120, generator=g).cuda() for _ in range(3))
    gain = torch.randn(120, generator=g).cuda()
    dz, dgain = torch.empty_like(z), torch.zeros_like(gain)
    dx = op.backward(50, x, z, 120, 0, gain, dy, dz, 120, 0, dgain)
    f = lambda *v: (op.forward(50, v[0], v[1], 120, 0, v[2]).double() * dy.double()).sum()
    for i, d in enumerate((dx, dz, dgain)):
        s = 2.0 ** -9 / float(d.abs().max()) * d
        up, dn = [x, z, gain], [x, z, gain]
        up[i], dn[i] = up[i] + s, dn[i] - s
        want = 2 * (s.double() * d.double()).sum()
        assert abs(float(f(*up) - f(*dn) - want)) <= 1e-3 * float(want)


def test_refusals(rnn):
    op = rnn.HeadGate(4, 16)
    x, z = torch.zeros(10, 64, device="cuda"), torch.zeros(10, 128, device="cuda")
    with pytest.raises(ValueError):
        op.forward(11, x, z, 128)
    with pytest.raises(ValueError):
        op.forward(10, x, z, 128, 65)  # the last row's gate is past the buffer's end
    with pytest.raises(rnn.RnnError):
        op.forward(9, x, z, 128, 65)  # the gate does not fit a row
    with pytest.raises(rnn.RnnError):
        op.forward(10, x, z, 63)
    with pytest.raises(TypeError):
        op.forward(10, x.double(), z, 128)
    with pytest.raises(ValueError):
        op.forward(10, x, z, 128, 0, torch.ones(63, device="cuda"))
    with pytest.raises(rnn.RnnError):
        op.backward(10, x, z, 128, 0, None, x, z.clone(), 128, 0, torch.zeros(64, device="cuda"))
    with pytest.raises(rnn.RnnError):
        op.backward(10, x, z, 128, 0, None, x, z.clone(), 60)
    with pytest.raises(rnn.RnnError):
        op.forward(10, x, z, 128, y=z)
    with pytest.raises(rnn.RnnError):  # in place with two layouts
        op.backward(10, x, z, 128, 0, None, x.clone(), z, 128, 64)
    for dx in (z, x):
        with pytest.raises(rnn.RnnError):
            op.backward(10, x, z, 128, 0, None, x.clone(), x if dx is x else dx, 64, dx=dx)
    assert op.forward(0, x, z, 128).shape == (0, 64)
