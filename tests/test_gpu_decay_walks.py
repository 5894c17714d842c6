"""GPU: the launches of linear attention with a decay that need many sequences,
long ones or absent results: walks of many chunks without segments, a backward
without the rates' gradient, forwards in twice as many segments.  Tolerances are
DecayCase.tol()'s."""
import pytest
import torch

from decayref import D, DecayCase
from test_gpu_decay import check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(n=70, t=200, h=8, hkv=8, dk=16, dv=16, reverse=3),
                                dict(n=65, t=193, h=8, hkv=4, dk=24, dv=8,
                                     lens=[193, 96, 1, 160, 0] * 13)])
def test_many_sequences_walk_whole(rnn, kw):
    """More walks than the device has places for: no segments, seven chunks each."""
    cs = DecayCase(seed=21, **kw)
    core = rnn.DecayCore(cs.h, cs.dk, cs.dv, cs.hkv)
    layout = (cs.qstride, 0, cs.kvstride, cs.koff, None, cs.voff)
    assert core._plan(cs.n, cs.t, 0, layout)[1] == 0  # a segment's state is workspace
    got, want = run(rnn, cs), cs.want()
    check(cs, got, want, cs.sizes())
    if cs.lens is not None:
        for b, m in enumerate(cs.lens.tolist()):
            assert all((got[nm][b, m:] == 0).all() for nm in ("y", "dq", "dk", "dv"))


@pytest.mark.parametrize("kw", [dict(n=2, t=80, h=4, hkv=2, dk=64, dv=64, reverse=1),
                                dict(n=2, t=80, h=4, hkv=4, dk=24, dv=24, reverse=2),
                                dict(n=1, t=70, h=2, hkv=2, dk=40, dv=64, reverse=1),
                                dict(n=3, t=500, h=4, hkv=2, dk=64, dv=64, reverse=2,
                                     lens=[500, 33, 0]),
                                dict(n=3, t=500, h=4, hkv=4, dk=24, dv=24, reverse=1,
                                     lens=[411, 500, 1]),
                                dict(n=2, t=500, h=2, hkv=2, dk=44, dv=24, reverse=1)])
def test_backward_without_the_rates(rnn, kw):
    """dq without the rates' gradient is another kernel's, in one launch with dk
    and dv where keys and values have as many 32-channel tiles; segments give it
    their states."""
    cs = DecayCase(seed=22, **kw)
    full, want, size = run(rnn, cs), cs.want(), cs.sizes()
    dev = lambda x: None if x is None else x.cuda()
    core = rnn.DecayCore(cs.h, cs.dk, cs.dv, cs.hkv, reverse=cs.reverse)
    kv, lens, state = cs.kv.cuda(), dev(cs.lens), cs.state.cuda()
    dx, ds = torch.full_like(kv, float("nan")), torch.full_like(state, float("nan"))
    core.backward(cs.n, cs.t, *cs.geo(kv, kv), cs.rate.cuda(), cs.dy.cuda(), dx, dx, lens=lens,
                  state=state, dstate_out=cs.dstate.cuda(), dstate=ds, set_dq=True, set_dkv=True)
    got = dict(dq=dx[..., :cs.qw], dk=dx[..., cs.koff:cs.koff + cs.kw],
               dv=dx[..., cs.voff:cs.voff + cs.vw], dstate=ds)
    check(cs, got, want, size, tuple(got))
    for nm in ("dk", "dv", "dstate"):  # the same kernel's, in other launches
        assert torch.equal(got[nm], full[nm]), nm
    if cs.lens is not None:
        for b, m in enumerate(cs.lens.tolist()):
            assert all((got[nm][b, m:] == 0).all() for nm in ("dq", "dk", "dv"))


def recurrence(q, k, v, rate, s0, scale, lens):
    """decayref.decay_attn's outputs for all heads at once (key heads as many as
    query heads, none reversed)."""
    gam = torch.exp(-torch.exp(rate)).view(1, -1, 1, 1)
    s, y = s0, torch.zeros(*q.shape[:3], v.shape[3], dtype=D)
    for i in range(q.shape[1]):
        ok = (lens > i).view(-1, 1, 1, 1)
        s = torch.where(ok, gam * s + k[:, i, :, :, None] * v[:, i, :, None, :], s)
        y[:, i] = scale * (q[:, i, :, None] @ s)[:, :, 0] * ok[..., 0]
    return y, s


@pytest.mark.parametrize("n,t,h,dk,dv,nseg", [(64, 509, 4, 24, 40, 4), (25, 1300, 8, 16, 8, 10)])
def test_two_waves_a_place(rnn, n, t, h, dk, dv, nseg):
    """Forwards long enough for twice as many segments as fill the device once."""
    lens = [t, t - 1, 31, t // 2, 0] * (n // 5 + 1)
    cs = DecayCase(n, t, h, h, dk, dv, lens=lens[:n], seed=23)
    core = rnn.DecayCore(h, dk, dv)
    layout = (cs.qstride, 0, cs.kvstride, cs.koff, None, cs.voff)
    assert core._plan(n, t, 0, layout)[1] == nseg * n * h * dk * dv * 4
    got = run(rnn, cs, train=False)
    q, k, v, s0, _ = cs._leaves()
    y, st = recurrence(q, k, v, cs.rate.to(D), s0, cs.scale, cs.lens)
    ya, sa = recurrence(q.abs(), k.abs(), v.abs(), cs.rate.to(D), s0.abs(), cs.scale, cs.lens)
    flat = lambda x: x.reshape(n, t, h * dv)
    check(cs, got, dict(y=flat(y), state=st), dict(y=flat(ya), state=sa), ("y", "state"))


@pytest.mark.parametrize("t", [1, 9])
def test_states_past_32_bits(rnn, t):
    """Offsets of states above 2^32 bytes: the last sequences of 17000 with 256 KB
    each as on their own, forward in place and backward."""
    n, h, dk, dv = 17000, 8, 64, 128
    cs = DecayCase(3, t, h, h, dk, dv, reverse=3, seed=24)
    one = run(rnn, cs)
    core, rate = rnn.DecayCore(h, dk, dv, reverse=3), cs.rate.cuda()
    kv = torch.zeros(n, t, cs.kvstride, device="cuda")
    kv[-3:] = cs.kv.cuda()
    st = torch.zeros(n, h, dk, dv, device="cuda")
    st[-3:] = cs.state.cuda()
    dy, ds1 = torch.zeros(n, t, h * dv, device="cuda"), torch.zeros_like(st)
    dy[-3:], ds1[-3:] = cs.dy.cuda(), cs.dstate.cuda()
    dx, ds0 = torch.empty_like(kv), torch.empty_like(st)
    drate = torch.zeros_like(rate)
    core.backward(n, t, *cs.geo(kv, kv), rate, dy, dx, dx, drate, state=st, dstate_out=ds1,
                  dstate=ds0, set_dq=True, set_dkv=True)
    assert torch.equal(dx[-3:], one["rest"][0]) and torch.equal(ds0[-3:], one["dstate"])
    assert (ds0[:-3] == 0).all() and (dx[:-3] == 0).all()
    y, _ = core.forward(n, t, *cs.geo(kv, kv), rate, state=st, state_out=st)
    assert torch.equal(y[-3:], one["y"]) and torch.equal(st[-3:], one["state"])
    assert (st[:-3] == 0).all() and (y[:-3] == 0).all()
