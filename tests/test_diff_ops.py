"""CPU: what the operators of the differential block refuse on the host, before
anything reaches a device, and the plain statements that their GPU tests
compare with (diffref.py), against differences."""
import ctypes as C
import math

import pytest
import torch

import diffref
import rustnn_amd as R


def test_null_context_is_refused():
    L = R.lib()
    d, e = R.RotaryDesc(), R.DiffAttnDesc()
    assert L.rnn_rotary(None, C.byref(d), 1, 1, None, None, None, 0) == R.RNN_E_NULL
    assert L.rnn_diff_attn_forward(None, C.byref(e), 1, *[None] * 7, 0, None, None, None) == \
        R.RNN_E_NULL
    assert L.rnn_diff_attn_backward(None, C.byref(e), 1, *[None] * 10, 0, *[None] * 4, 0) == \
        R.RNN_E_NULL
    assert L.rnn_linear_act_forward(None, 1, 1, 1, None, None, None, 0, None, None, None) == \
        R.RNN_E_NULL
    assert L.rnn_linear_act_backward(None, 1, 1, 1, *[None] * 5, 0, None, None, None, 0) == \
        R.RNN_E_NULL
    nb = C.c_size_t()
    assert L.rnn_linear_act_workspace(8, 8, 8, None) == R.RNN_E_NULL
    assert L.rnn_linear_act_workspace(8, 1 << 21, 8, C.byref(nb)) == R.RNN_E_UNSUPPORTED
    assert L.rnn_linear_act_workspace(0, 0, 0, C.byref(nb)) == R.RNN_OK and nb.value == 0


@pytest.mark.parametrize("kw", [
    dict(heads=0), dict(dh=0), dict(pairs=(8, 9)), dict(pairs=(8,)), dict(grid=(8, 0)),
    dict(grid=(2, 2, 2, 2), pairs=(4, 4, 4, 4)), dict(base=0.0), dict(base=-1.0),
    dict(base=math.inf), dict(base=math.nan), dict(heads=-1), dict(pairs=(-1, 2)),
    dict(dh=1024, pairs=(256, 1)), dict(grid=(65536, 65536)), dict(heads=1 << 20, dh=32)])
def test_rotary_refuses(kw):
    with pytest.raises(ValueError):
        R.Rotary(**dict(dict(heads=4, dh=32, grid=(8, 8)), **kw))


def test_rotary_description_is_checked():
    L = R.lib()
    d = R.Rotary(4, 32, (8, 8))._desc(128, 0, 128, 0)
    check = lambda n, t, pos: L.rnn_rotary_check(C.byref(d), n, t, pos)
    assert check(2, 64, 0) == R.RNN_OK and check(0, 64, 0) == R.RNN_OK
    assert check(2, 63, 0) == R.RNN_E_INVALID and check(2, 63, 1) == R.RNN_OK
    assert check(1 << 30, 64, 0) == R.RNN_E_UNSUPPORTED
    assert check(1 << 62, 1 << 40, 1) == R.RNN_E_UNSUPPORTED
    for field, bad in (("axes", 0), ("axes", 4), ("axes", 1), ("xstride", 127), ("xoff", 1),
                       ("ystride", 127), ("yoff", 1 << 40), ("g2", 2)):
        old = getattr(d, field)
        setattr(d, field, bad)
        assert check(2, 64, 0) == R.RNN_E_INVALID, field
        setattr(d, field, old)
    assert L.rnn_rotary_check(None, 1, 1, 0) == R.RNN_E_NULL


@pytest.mark.parametrize("kw,code", [
    (dict(h=0), -1), (dict(dh=0), -1), (dict(hkv=3), -1), (dict(hkv=0), -1),
    (dict(lam_heads=2), -1), (dict(lam_heads=0), -1), (dict(scale=0.0), -1),
    (dict(scale=-1.0), -1), (dict(scale=math.nan), -1), (dict(scale=math.inf), -1),
    (dict(lam_init=1.0), -1), (dict(lam_init=-0.1), -1), (dict(lam_init=math.nan), -1),
    (dict(eps=0.0), -1), (dict(eps=math.nan), -1), (dict(dh=65), -5), (dict(tk=1 << 28), -5),
    (dict(tq=1 << 28), -5), (dict(h=4096, lam_heads=1, dh=1), -5), (dict(tq=-1), -1)])
def test_diff_core_refuses(kw, code):
    with pytest.raises(ValueError):
        R.DiffCore(**dict(dict(h=4, dh=32, tq=8, tk=8), **kw))


def test_diff_description_is_checked():
    core = R.DiffCore(4, 32, 8, 8)
    nb = C.c_size_t()
    ok = dict(qstride=768, qoff=0, kvstride=768, koff=256, voff=512)

    def code(n=2, out=nb, **kw):
        d = core.desc(**dict(ok, **kw))
        return R.lib().rnn_diff_attn_workspace(C.byref(d), n, 1, None if out is None else C.byref(out))

    assert code() == R.RNN_OK and nb.value > 0
    assert code(out=None) == R.RNN_E_NULL
    for kw in (dict(qstride=255), dict(qoff=600), dict(voff=513), dict(koff=257), dict(voff=300),
               dict(koff=1 << 40)):
        assert code(**kw) == R.RNN_E_INVALID, kw
    assert code(kvstride=1 << 40) == R.RNN_E_UNSUPPORTED
    assert code(n=1 << 40) == R.RNN_E_UNSUPPORTED
    assert code(n=1 << 29) == R.RNN_E_UNSUPPORTED
    assert code(n=1 << 25) == R.RNN_E_UNSUPPORTED  # n tq h = 2^30
    assert code(n=(1 << 25) - 1) == R.RNN_OK
    assert R.lib().rnn_diff_attn_workspace(None, 1, 0, C.byref(nb)) == R.RNN_E_NULL


def test_unknown_activation():
    with pytest.raises(ValueError):
        R.linear_act_forward(1, 1, 1, None, None, act="tanh")


def test_statement_against_differences():
    """The oracle of differential attention: automatic derivatives against
    central differences in 64 bits (step 1e-5: 1e-10 and rounding 1e-11)."""
    cs = diffref.DiffCase(2, 4, 2, 6, 5, 7, True, causal=True, klen=[7, 2], per_head=True, seed=3)
    want = cs.want()
    see = diffref.seen(cs.n, cs.tq, cs.tk, cs.causal, cs.diag, cs.qlen, cs.klen)
    x = [t.double() for t in (cs.qv, cs.kvv, cs.vv, cs.lam, cs.gain)]
    f = lambda v: (diffref.diff_attn(*v, see, cs.scale, cs.lam_init, cs.eps) * cs.dyv).sum()
    g = torch.Generator().manual_seed(0)
    for i, nm in enumerate(("dq", "dk", "dv", "dlam", "dgain")):
        d = torch.randn(x[i].shape, generator=g, dtype=torch.float64)
        up, dn = list(x), list(x)
        up[i], dn[i] = x[i] + 1e-5 * d, x[i] - 1e-5 * d
        num = (f(up) - f(dn)) / 2e-5
        ref = (want[nm].reshape(-1) * d.reshape(-1)).sum()
        assert abs(num - ref) < 1e-6 * (1 + abs(ref)), nm
    # a query that sees no key, and an image without keys, give zeros
    assert (want["y"][1, :3] == 0).all()


def test_rotary_statement_keeps_lengths_and_composes():
    """A turn keeps each pair's length; two turns add their angles."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(10, 2 * 12, generator=g, dtype=torch.float64)
    p, q = torch.randn(10, 2, generator=g) * 9, torch.randn(10, 2, generator=g) * 9
    for inter in (False, True):
        a = diffref.rotary(x, 2, 12, p, (3, 2), 50.0, inter)
        assert abs(a.norm() - x.norm()) < 1e-12 * x.norm()
        ab = diffref.rotary(a, 2, 12, q, (3, 2), 50.0, inter)
        both = diffref.rotary(x, 2, 12, p.double() + q.double(), (3, 2), 50.0, inter)
        assert (ab - both).abs().max() < 1e-12
        assert (diffref.rotary(a, 2, 12, p, (3, 2), 50.0, inter, True) - x).abs().max() < 1e-12
