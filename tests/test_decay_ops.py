"""CPU: what the operators of the linear-attention block refuse on the host,
before anything reaches a device, and the plain statements that their GPU tests
compare with (decayref.py), against each other and against differences."""
import ctypes as C
import math

import pytest
import torch

import decayref
import rustnn_amd as R
from decayref import D


def test_null_context_is_refused():
    L = R.lib()
    d, e = R.RotaryDesc(), R.DecayAttnDesc()
    assert L.rnn_norm_rotary_forward(None, C.byref(d), 1, 1e-6, 1, 1, *[None] * 4) == R.RNN_E_NULL
    assert L.rnn_norm_rotary_backward(None, C.byref(d), 1, 1e-6, 1, 1, *[None] * 4, 8, 0, None, 0,
                                      None, None) == R.RNN_E_NULL
    assert L.rnn_decay_attn_forward(None, C.byref(e), 1, 1, *[None] * 7, 0, None, None) == \
        R.RNN_E_NULL
    assert L.rnn_decay_attn_backward(None, C.byref(e), 1, 1, *[None] * 9, 0, *[None] * 5, 0) == \
        R.RNN_E_NULL
    assert L.rnn_head_gate_forward(None, 1, 1, 1, 1e-6, None, None, 1, 0, None, None) == R.RNN_E_NULL
    assert L.rnn_head_gate_backward(None, 1, 1, 1, 1e-6, None, None, 1, 0, None, None, None, 0, None,
                                    None, 1, 0, None) == R.RNN_E_NULL


@pytest.mark.parametrize("kw", [
    dict(hq=0, hk=0), dict(hq=-1), dict(hk=-1), dict(dh=0), dict(pairs=(16, 17)), dict(pairs=(8,)),
    dict(grid=(8, 0)), dict(base=0.0), dict(base=math.nan), dict(eps=0.0), dict(eps=-1.0),
    dict(eps=math.nan), dict(eps=math.inf), dict(dh=257), dict(dh=320), dict(hq=1 << 20)])
def test_norm_rotary_refuses(kw):
    with pytest.raises(ValueError):
        R.NormRotary(**dict(dict(hq=4, hk=2, dh=32, grid=(8, 8)), **kw))


def test_norm_rotary_is_checked():
    op = R.NormRotary(4, 2, 32, (8, 8))
    d, nb = op.rot._desc(192, 0, 192, 0), C.c_size_t()
    ws = lambda hq, eps, n, t, pos, out=nb: R.lib().rnn_norm_rotary_workspace(
        C.byref(d), hq, eps, n, t, pos, None if out is None else C.byref(out))
    assert ws(4, 1e-6, 2, 64, 0) == R.RNN_OK and nb.value >= 2 * 32 * 8
    assert ws(0, 1e-6, 2, 64, 0) == R.RNN_OK and ws(6, 1e-6, 0, 64, 0) == R.RNN_OK
    assert nb.value == 0
    assert ws(7, 1e-6, 2, 64, 0) == R.RNN_E_INVALID  # more queries than heads
    assert ws(4, 1e-6, 2, 63, 0) == R.RNN_E_INVALID and ws(4, 1e-6, 2, 63, 1) == R.RNN_OK
    assert ws(4, 0.0, 2, 64, 0) == R.RNN_E_INVALID
    assert ws(4, 1e-6, 1 << 40, 64, 0) == R.RNN_E_UNSUPPORTED
    assert ws(4, 1e-6, 2, 64, 0, None) == R.RNN_E_NULL
    assert R.lib().rnn_norm_rotary_workspace(None, 4, 1e-6, 2, 64, 0, C.byref(nb)) == R.RNN_E_NULL


@pytest.mark.parametrize("kw", [
    dict(h=0), dict(dk=0), dict(dv=0), dict(hkv=0), dict(hkv=3), dict(hkv=8), dict(reverse=5),
    dict(reverse=-1), dict(h=-4), dict(scale=math.nan), dict(scale=math.inf), dict(dk=129),
    dict(dv=129), dict(h=1 << 18, hkv=1 << 18)])
def test_decay_core_refuses(kw):
    with pytest.raises(ValueError):
        R.DecayCore(**dict(dict(h=4, dk=32), **kw))


def test_decay_description_is_checked():
    core, nb = R.DecayCore(4, 32, 48, 2), C.c_size_t()
    ok = dict(qstride=288, qoff=0, kstride=288, koff=128, vstride=288, voff=192)

    def code(n=2, t=8, back=1, out=nb, **kw):
        d = core.desc(**dict(ok, **kw))
        return R.lib().rnn_decay_attn_workspace(C.byref(d), n, t, back,
                                                None if out is None else C.byref(out))

    assert code() == R.RNN_OK and code(back=0) == R.RNN_OK and code(n=0) == R.RNN_OK
    assert code(out=None) == R.RNN_E_NULL
    for kw in (dict(qstride=127), dict(qoff=200), dict(voff=193), dict(koff=225), dict(vstride=287),
               dict(koff=1 << 40)):
        assert code(**kw) == R.RNN_E_INVALID, kw
    assert code(kstride=(1 << 22) + 1) == R.RNN_E_UNSUPPORTED
    assert code(vstride=(1 << 22) + 1) == R.RNN_E_UNSUPPORTED
    for koff, voff in ((128, 191), (230, 160), (160, 100)):  # in one buffer keys and values overlap
        with pytest.raises(ValueError):
            core._plan(2, 8, 0, (288, 0, 288, koff, None, voff))
    assert code(n=1 << 40) == R.RNN_E_UNSUPPORTED and code(t=1 << 40) == R.RNN_E_UNSUPPORTED
    assert code(n=1, t=1 << 29) == R.RNN_E_UNSUPPORTED
    assert code(n=2, t=1 << 28) == R.RNN_E_UNSUPPORTED  # n h t = 2^31
    assert code(n=2, t=(1 << 28) - 1) == R.RNN_OK
    assert code(n=1 << 19, t=1) == R.RNN_E_UNSUPPORTED  # n h dk dv > 2^31
    one = R.DecayCore(1, 1).desc(1, 0, 2, 0, 2, 1)
    ws = lambda n: R.lib().rnn_decay_attn_workspace(C.byref(one), n, 1, 1, C.byref(nb))
    assert ws((1 << 22) - 1) == R.RNN_OK and ws(1 << 22) == R.RNN_E_UNSUPPORTED
    assert R.lib().rnn_decay_attn_workspace(None, 1, 1, 0, C.byref(nb)) == R.RNN_E_NULL


def test_decay_values_apart_need_their_stride():
    core, x = R.DecayCore(1, 4), torch.zeros(1, 1, 12)
    geo = (x, 12, 0, x, 12, 4, 8)
    for kw in (dict(v=x), dict(vstride=12)):
        with pytest.raises(ValueError):
            core.forward(1, 1, *geo, x, **kw)
    for kw in (dict(v=x), dict(vstride=12), dict(dv=x), dict(v=x, dv=x), dict(v=x, vstride=12)):
        with pytest.raises(ValueError):
            core.backward(1, 1, *geo, x, x, x, x, **kw)


@pytest.mark.parametrize("kw", [dict(h=0), dict(d=0), dict(h=-1), dict(d=513), dict(h=65537),
                                dict(eps=0.0), dict(eps=math.nan), dict(eps=math.inf)])
def test_head_gate_refuses(kw):
    with pytest.raises(ValueError):
        R.HeadGate(**dict(dict(h=4, d=32), **kw))


def test_head_gate_is_checked():
    nb = C.c_size_t()
    ws = R.lib().rnn_head_gate_workspace
    assert ws(100, 4, 32, C.byref(nb)) == R.RNN_OK and nb.value >= 4 * 32 * 8
    assert ws(0, 4, 32, C.byref(nb)) == R.RNN_OK and nb.value == 0
    assert ws(100, 4, 32, None) == R.RNN_E_NULL
    assert ws(1 << 40, 4, 32, C.byref(nb)) == R.RNN_E_UNSUPPORTED


def close(a, b):
    return float((a - b).abs().max()) <= 1e-11 * (1 + float(b.abs().max()))


@pytest.mark.parametrize("kw", [dict(), dict(reverse=2, lens=[7, 4]), dict(lens=[0, 1]),
                                dict(reverse=4, state=False)])
def test_decay_statements_agree(kw):
    """The recurrence and the whole map, outputs and gradients."""
    cs = decayref.DecayCase(2, 7, 4, 2, 5, 6, seed=1, **kw)
    a, b = cs.want(decayref.decay_attn), cs.want(decayref.decay_map)
    for k in a:
        assert close(a[k], b[k]), k


def test_decay_statement_against_differences():
    """Central differences in 64 bits (step 1e-5: 1e-10 and rounding 1e-11)."""
    cs = decayref.DecayCase(2, 6, 4, 2, 3, 5, reverse=1, lens=[6, 3], seed=2)
    q, k, v, s0, dy = cs._leaves()
    x, want = [q, k, v, cs.rate.to(D), s0], cs.want(decayref.decay_attn)

    def f(xs):
        y, st = decayref.decay_attn(*xs, cs.scale, cs.reverse, cs.lens)
        return (y * dy).sum() + (st * cs.dstate.to(D)).sum()

    g = torch.Generator().manual_seed(0)
    for i, nm in enumerate(("dq", "dk", "dv", "drate", "dstate")):
        d = torch.randn(x[i].shape, generator=g, dtype=D)
        up, dn = list(x), list(x)
        up[i], dn[i] = x[i] + 1e-5 * d, x[i] - 1e-5 * d
        num = (f(up) - f(dn)) / 2e-5
        ref = (want[nm].reshape(-1) * d.reshape(-1)).sum()
        assert abs(num - ref) < 1e-6 * (1 + abs(ref)), nm


def test_norm_rotary_statement():
    """The turn keeps a head's length, and gradients agree with differences."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, 3 * 10, generator=g, dtype=D, requires_grad=True)
    gain = torch.randn(2, 10, generator=g, dtype=D, requires_grad=True)
    pos, dy = torch.randn(6, 2, generator=g) * 9, torch.randn(6, 30, generator=g, dtype=D)
    for inter in (False, True):
        f = lambda x, gain: (decayref.norm_rotary(x, gain, 2, 1, 10, pos, (3, 1), 50.0, inter, 1e-3)
                             * dy).sum()
        y = decayref.norm_rotary(x, None, 2, 1, 10, pos, (3, 1), 50.0, inter, 1e-12)
        assert close(y.detach().view(6, 3, 10).norm(dim=-1), torch.full((6, 3), math.sqrt(10.0), dtype=D))
        for i, got in enumerate(torch.autograd.grad(f(x, gain), (x, gain))):
            args = [x.detach(), gain.detach()]
            d = torch.randn(args[i].shape, generator=g, dtype=D)
            up, dn = list(args), list(args)
            up[i], dn[i] = args[i] + 1e-5 * d, args[i] - 1e-5 * d
            assert abs((f(*up) - f(*dn)) / 2e-5 - (got * d).sum()) < 1e-6 * (1 + got.norm() * d.norm())


def test_gate_statement():
    g = torch.Generator().manual_seed(4)
    x, z, gain, dy = (torch.randn(*s, generator=g, dtype=D) for s in ((5, 12), (5, 12), (12,), (5, 12)))
    leaves = [v.requires_grad_(True) for v in (x, z, gain)]
    f = lambda *v: (decayref.gate(*v, 3, 4, 1e-3) * dy).sum()
    for i, got in enumerate(torch.autograd.grad(f(*leaves), leaves)):
        d = torch.randn(got.shape, generator=g, dtype=D)
        up, dn = [v.detach() for v in leaves], [v.detach() for v in leaves]
        up[i], dn[i] = up[i] + 1e-5 * d, dn[i] - 1e-5 * d
        assert abs((f(*up) - f(*dn)) / 2e-5 - (got * d).sum()) < 1e-6 * (1 + got.norm() * d.norm())
