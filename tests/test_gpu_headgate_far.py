"""GPU: gates over the whole range in which z sigma(z) is a number of 32 bits.

Tolerances as for gates near zero: y within 11 U, dz within |dy x^ gain|
sigma (8.5 |z| + 14 |f|) U, f = 1 + z (1 - sigma), and half of the least number,
2^-150, where a result is below the normal range.  dgain sums, in 64 bits, terms
of one sign: du within 8.5 U and 2^-150, x^ within 2 U, and the result's rounding."""
import pytest
import torch

from decayref import D, U, gate, head_norm

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -150


@pytest.mark.parametrize("lo,hi", [(-119.9, -80.0), (-88.5, -86.5), (-80.0, -20.0), (-20.0, 20.0),
                                   (20.0, 120.0)])
def test_far_gates_keep_their_bits(rnn, lo, hi):
    rows, h, d = 3, 32, 64
    g, w = torch.Generator().manual_seed(9), h * d
    x, dy, gain = (torch.rand(*s, generator=g) + 0.5 for s in ((rows, w), (rows, w), (w,)))
    z = torch.linspace(lo, hi, w).expand(rows, w).contiguous()
    op, eps = rnn.HeadGate(h, d, 1e-3), float(torch.tensor(1e-3))
    x64, z64, g64, dy64 = (v.to(D) for v in (x, z, gain, dy))
    want = gate(x64, z64, g64, h, d, eps)
    y = op.forward(rows, x.cuda(), z.cuda(), w, 0, gain.cuda()).cpu().to(D)
    assert ((y - want).abs() <= 11 * U * want.abs() + LEAST).all()
    hat = head_norm(x64.view(rows, h, d), eps).reshape(rows, w)
    sig = torch.sigmoid(z64)
    f = 1 + z64 * (1 - sig)
    dz, dgain = torch.empty_like(z).cuda(), torch.zeros(w).cuda()
    op.backward(rows, x.cuda(), z.cuda(), w, 0, gain.cuda(), dy.cuda(), dz, w, 0, dgain)
    size = (dy64 * hat * g64).abs() * sig
    tz = 1.01 * size * (8.5 * z64.abs() + 14 * f.abs()) * U
    assert ((dz.cpu().to(D) - size * f).abs() <= tz + LEAST).all()
    dg = (dy64 * z64 * sig * hat).sum(0)
    tg = 1.01 * (10.5 + 1) * U * dg.abs() + LEAST * (hat.sum(0) + 1)
    assert ((dgain.cpu().to(D) - dg).abs() <= tg).all()


def test_closed_gates(rnn):
    """Below -120, z sigma(z) comes to 0 in 32 bits, whatever stands beside it."""
    op = rnn.HeadGate(1, 8, 1e-6)
    z = torch.tensor([[-120.5, -121.0, -500.0, -1e10, -1e30, -3e38, 0.5, -2.0]]).cuda()
    x = torch.full((1, 8), 1e30).cuda()
    y = op.forward(1, x, z, 8)
    assert (y[0, :6] == 0).all() and (y[0, 6:] != 0).all()
    dz = torch.empty_like(z)
    dx = op.backward(1, x, z, 8, 0, None, torch.ones_like(x), dz, 8)
    assert (dz[0, :6] == 0).all() and (dz[0, 6:] != 0).all() and torch.isfinite(dx).all()


def test_large_factors_beside_small_gates(rnn):
    """Products with factors near a float's range: nothing overflows on the way."""
    op = rnn.HeadGate(1, 8, 1e-3)
    z = torch.tensor([[-45.0, -60.0, -68.0, -70.0, -75.0, -90.0, -100.0, -110.0]])
    x, gain = torch.ones(1, 8), torch.full((8,), 1e37)
    eps = float(torch.tensor(1e-3))
    want = gate(x.to(D), z.to(D), gain.to(D), 1, 8, eps)
    y = op.forward(1, x.cuda(), z.cuda(), 8, 0, gain.cuda()).cpu().to(D)
    assert ((y - want).abs() <= 11 * U * want.abs()).all()
    dz = torch.empty(1, 8).cuda()
    op.backward(1, x.cuda(), z.cuda(), 8, 0, gain.cuda(), torch.ones(1, 8).cuda(), dz, 8)
    sig = torch.sigmoid(z.to(D))
    f, u = 1 + z.to(D) * (1 - sig), head_norm(x.to(D), eps) * gain.to(D)
    tz = 1.01 * u * sig * (8.5 * z.to(D).abs() + 14 * f.abs()) * U
    assert ((dz.cpu().to(D) - u * sig * f).abs() <= tz).all()
