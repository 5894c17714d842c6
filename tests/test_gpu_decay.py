"""GPU: linear attention with a decay for each head (rnn_decay_attn_*, DecayCore)
against its plain statement in 64 bits.  Tolerances, element by element: those of
DecayCase.tol(), of the size that the element's terms come to without signs."""
import pytest
import torch

from decayref import D, U, DecayCase

pytestmark = pytest.mark.gpu

NAMES = ("y", "state", "dq", "dk", "dv", "drate", "dstate")

# name, arguments of DecayCase
CASES = [
    ("one_token", dict(n=1, t=1, h=1, hkv=1, dk=1, dv=1)),
    ("one_token_heads", dict(n=3, t=1, h=4, hkv=2, dk=64, dv=64, reverse=1)),
    ("two", dict(n=2, t=2, h=2, hkv=2, dk=8, dv=8)),
    ("few", dict(n=2, t=7, h=4, hkv=4, dk=32, dv=64, reverse=2)),
    ("few_ragged", dict(n=4, t=5, h=4, hkv=2, dk=24, dv=40, reverse=2, lens=[5, 0, 1, 3])),
    ("eight", dict(n=2, t=8, h=4, hkv=2, dk=40, dv=36, reverse=2)),
    ("nine", dict(n=2, t=9, h=2, hkv=1, dk=33, dv=31, state=False)),
    ("a_tile", dict(n=2, t=32, h=2, hkv=2, dk=32, dv=32, reverse=1)),
    ("past_a_tile", dict(n=1, t=33, h=2, hkv=2, dk=64, dv=32, reverse=1)),
    ("image", dict(n=3, t=64, h=4, hkv=4, dk=64, dv=64, reverse=2, state=False)),
    ("odd", dict(n=2, t=101, h=3, hkv=3, dk=13, dv=27, reverse=1, gap=1)),
    ("shared", dict(n=2, t=70, h=6, hkv=2, dk=44, dv=72, reverse=3)),
    ("shared_one", dict(n=1, t=50, h=4, hkv=1, dk=16, dv=16, reverse=4, fused=False)),
    ("apart", dict(n=2, t=65, h=2, hkv=2, dk=32, dv=48, fused=False, gap=4)),
    ("widest", dict(n=1, t=130, h=2, hkv=2, dk=128, dv=128, reverse=1)),
    ("wide_odd", dict(n=1, t=45, h=2, hkv=1, dk=127, dv=97, reverse=1, gap=3)),
    ("narrow_values", dict(n=1, t=70, h=2, hkv=2, dk=96, dv=1)),
    ("narrow_keys", dict(n=1, t=70, h=2, hkv=2, dk=1, dv=96)),
    ("ragged", dict(n=5, t=97, h=2, hkv=2, dk=64, dv=64, reverse=1, lens=[97, 0, 1, 32, 64])),
    ("ragged_shared", dict(n=4, t=75, h=4, hkv=2, dk=24, dv=40, reverse=2, lens=[75, 33, 2, 65],
                           state=False)),
    ("long", dict(n=1, t=1100, h=2, hkv=2, dk=32, dv=32, reverse=1)),
    ("long_ragged", dict(n=2, t=1500, h=2, hkv=1, dk=20, dv=64, reverse=1, lens=[1500, 700])),
    ("segments_of_many_lengths", dict(n=9, t=1000, h=4, hkv=2, dk=40, dv=24, reverse=2,
                                      lens=[1000, 999, 33, 500, 0, 31, 64, 97, 1200])),
    ("uneven_segments", dict(n=1, t=2245, h=2, hkv=2, dk=8, dv=12, reverse=1)),
    ("few_wide_segments", dict(n=16, t=420, h=8, hkv=4, dk=36, dv=128, reverse=4,
                               lens=[420, 7, 300, 1] * 4)),
    ("slow_decay", dict(n=1, t=700, h=2, hkv=2, dk=32, dv=32, rates=(-30.0, -12.0))),
    ("fast_decay", dict(n=1, t=200, h=2, hkv=2, dk=32, dv=32, rates=(1.0, 6.0), reverse=1)),
]


def run(rnn, cs, train=True, set_=True, ctx=None, over=None):
    dev = lambda x: None if x is None else x.cuda()
    kv = cs.kv.cuda()
    q = kv if cs.fused else cs.q.cuda()
    core = rnn.DecayCore(cs.h, cs.dk, cs.dv, cs.hkv, reverse=cs.reverse, ctx=ctx)
    geo, lens, state, rate = cs.geo(q, kv), dev(cs.lens), dev(cs.state), dev(cs.rate)
    y, st = core.forward(cs.n, cs.t, *geo, rate, lens=lens, state=state, keep_state=True)
    out = dict(y=y, state=st)
    if not train:
        return out
    fill = float("nan") if set_ else 2.0
    dkv = torch.full_like(kv, fill)
    dq = dkv if cs.fused else torch.full_like(q, fill)
    drate = torch.zeros_like(rate)
    ds = torch.full_like(st, float("nan"))
    core.backward(cs.n, cs.t, *geo, rate, cs.dy.cuda(), dq, dkv, drate, lens=lens, state=state,
                  dstate_out=dev(cs.dstate), dstate=ds, set_dq=set_, set_dkv=set_)
    out.update(dq=dq[..., :cs.qw], dk=dkv[..., cs.koff:cs.koff + cs.kw],
               dv=dkv[..., cs.voff:cs.voff + cs.vw], drate=drate, dstate=ds)
    out["rest"] = (dq, dkv)
    return out


def check(cs, got, want, size, names=NAMES, extra=0.0):
    for nm in names:
        a, w = got[nm].cpu().to(D).reshape(want[nm].shape), want[nm]
        tol = (cs.tol() + extra) * size[nm].reshape(w.shape) + 1e-37
        assert torch.isfinite(a).all(), nm
        worst = ((a - w).abs() / tol).max() if a.numel() else 0
        assert worst <= 1, (nm, float(worst))


@pytest.mark.parametrize("c", CASES, ids=[c[0] for c in CASES])
def test_forward_backward(rnn, c):
    cs = DecayCase(seed=3, **c[1])
    want, size = cs.want(), cs.sizes()
    got = run(rnn, cs)
    check(cs, got, want, size)
    if cs.lens is not None:  # padding: zeros, whatever the inputs hold there
        for b, m in enumerate(cs.lens.tolist()):
            for nm in ("y", "dq", "dk", "dv"):
                assert (got[nm][b, m:] == 0).all(), nm
    # accumulated: 2 + the gradient; what is not a head's column stays
    acc = run(rnn, cs, set_=False)
    for nm in ("dq", "dk", "dv"):
        one = (2.0 + want[nm]).abs() * U
        tol = cs.tol() * size[nm] + (2 * (cs.h // cs.hkv) + 1) * (2.0 + size[nm]) * U + one
        assert ((acc[nm].cpu().to(D) - 2.0 - want[nm]).abs() <= tol).all(), nm
        if cs.lens is not None:
            for b, m in enumerate(cs.lens.tolist()):
                assert (acc[nm][b, m:] == 2.0).all()
    for buf in acc["rest"]:
        seen = torch.zeros(buf.shape[-1], dtype=torch.bool)
        if buf is acc["rest"][0]:
            seen[:cs.qw] = True
        if buf is acc["rest"][1]:
            seen[cs.koff:cs.voff + cs.vw] = True
        assert (buf.cpu()[..., ~seen] == 2.0).all()
    again = run(rnn, cs)  # the same bits: sums in a fixed order
    for nm in NAMES:
        assert torch.equal(got[nm], again[nm]), nm


def test_without_states_and_rates(rnn):
    """What is not wanted is not needed: the same outputs without it."""
    cs = DecayCase(2, 80, 4, 2, 40, 24, reverse=1, seed=5, state=False)
    full = run(rnn, cs)
    core = rnn.DecayCore(4, 40, 24, 2, reverse=1)
    kv, rate = cs.kv.cuda(), cs.rate.cuda()
    y, st = core.forward(2, 80, *cs.geo(kv, kv), rate)
    assert st is None and torch.equal(y, full["y"])
    dx = torch.empty_like(kv)
    core.backward(2, 80, *cs.geo(kv, kv), rate, cs.dy.cuda(), dx, dx, set_dq=True, set_dkv=True)
    for nm, col in (("dq", slice(0, cs.qw)), ("dk", slice(cs.koff, cs.koff + cs.kw)),
                    ("dv", slice(cs.voff, cs.voff + cs.vw))):
        assert torch.equal(dx[..., col], full[nm]), nm


@pytest.mark.parametrize("pieces", [[1] * 12, [5, 1, 1, 30, 3], [33, 64, 1, 2], [1, 200, 1]])
def test_pieces_are_the_whole(rnn, pieces):
    """A prompt, then single tokens or further pieces, the state handed on in
    place: as one call over all of it."""
    t = sum(pieces)
    cs = DecayCase(2, t, 4, 2, 48, 64, seed=6)
    want, size = cs.want(), cs.sizes()
    core = rnn.DecayCore(4, 48, 64, 2)
    kv, rate, st = cs.kv.cuda(), cs.rate.cuda(), cs.state.cuda()
    at, ys = 0, []
    for m in pieces:
        part = kv[:, at:at + m].contiguous()
        y, out = core.forward(2, m, *cs.geo(part, part), rate, state=st, state_out=st)
        assert out is st
        ys.append(y)
        at += m
    got = dict(y=torch.cat(ys, 1), state=st)
    # each piece rounds the state once more
    check(cs, got, want, size, ("y", "state"), extra=4 * U * len(pieces) ** 0.5)


def test_a_thousand_single_tokens_keep_the_decay(rnn):
    """gamma rounded to 32 bits would be off by up to 1000 U after them."""
    n, h, dk, dv, t = 2, 2, 8, 16, 1000
    core = rnn.DecayCore(h, dk, dv)
    rate = torch.tensor([-9.3, -7.7]).cuda()
    zero = torch.zeros(n, 1, h * (2 * dk + dv)).cuda()
    geo = (zero, zero.shape[-1], 0, zero, zero.shape[-1], h * dk, 2 * h * dk)
    s0 = torch.randn(n, h, dk, dv).cuda()
    st = s0.clone()
    for _ in range(t):
        core.forward(n, 1, *geo, rate, state=st, state_out=st)
    gam = torch.exp(-t * torch.exp(rate.cpu().to(D))).view(1, h, 1, 1)
    want = gam * s0.cpu().to(D)
    # a rounding a token, of no common sign: within 4 sqrt(1000) U, and gamma in
    # two parts within 2^-47 a token
    assert ((st.cpu().to(D) - want).abs() <= 4 * t ** 0.5 * U * want.abs()).all()


@pytest.mark.parametrize("t", [1, 5, 40, 300])
def test_extreme_rates(rnn, t):
    """-infinity: no decay; +infinity and far rates: a token sees itself alone."""
    cs = DecayCase(1, t, 3, 3, 16, 16, seed=7)
    cs.rate = torch.tensor([-float("inf"), float("inf"), 80.0])
    got = run(rnn, cs)
    ref = DecayCase(1, t, 3, 3, 16, 16, seed=7)
    ref.rate = torch.tensor([-100.0, 60.0, 60.0])
    want, size = ref.want(), ref.sizes()
    check(ref, got, want, size, ("y", "state", "dq", "dk", "dv", "dstate"))
    assert (got["drate"] == 0).all()


@pytest.mark.parametrize("t", [1, 5, 40, 300])
def test_a_rate_that_is_no_number_shows_in_its_head(rnn, t):
    cs = DecayCase(2, t, 3, 3, 16, 16, seed=7)
    clean = run(rnn, cs)
    cs.rate[1] = float("nan")
    got = run(rnn, cs)
    for nm in ("y", "dq", "dk", "dv"):
        a, b = (v[nm].view(2, t, 3, 16) for v in (got, clean))
        assert torch.isnan(a[:, :, 1]).all(), nm
        assert torch.equal(a[:, :, ::2], b[:, :, ::2]), nm
    for nm in ("state", "dstate"):
        assert torch.isnan(got[nm][:, 1]).all() and torch.equal(got[nm][:, ::2], clean[nm][:, ::2])
    assert torch.isnan(got["drate"][1]) and torch.equal(got["drate"][::2], clean["drate"][::2])


@pytest.mark.parametrize("t", [3, 70])
def test_values_in_a_buffer_of_their_own(rnn, t):
    """The same bits as from one buffer, and gradients in two."""
    cs = DecayCase(2, t, 4, 2, 24, 40, reverse=1, seed=11, lens=[t, t // 2])
    full, kv, rate, st = run(rnn, cs), cs.kv.cuda(), cs.rate.cuda(), cs.state.cuda()
    core, lens = rnn.DecayCore(4, 24, 40, 2, reverse=1), cs.lens.cuda()
    v = torch.full((2, t, 100), 7.0).cuda()
    v[..., 3:83] = kv[..., cs.voff:cs.voff + 80]
    qk = kv[..., :cs.voff].contiguous()
    geo = (qk, cs.voff, 0, qk, cs.voff, cs.koff, 3)
    y, out = core.forward(2, t, *geo, rate, lens=lens, state=st, keep_state=True, v=v, vstride=100)
    assert torch.equal(y, full["y"]) and torch.equal(out, full["state"])
    dqk, dv, drate = torch.empty_like(qk), torch.full_like(v, 7.0), torch.zeros_like(rate)
    core.backward(2, t, *geo, rate, cs.dy.cuda(), dqk, dqk, drate, lens=lens, state=st,
                  dstate_out=cs.dstate.cuda(), set_dq=True, set_dkv=True, v=v, vstride=100, dv=dv)
    assert torch.equal(dqk[..., :cs.qw], full["dq"])
    assert torch.equal(dqk[..., cs.koff:cs.koff + cs.kw], full["dk"])
    assert torch.equal(dv[..., 3:83], full["dv"]) and torch.equal(drate, full["drate"])
    assert (dv[..., :3] == 7).all() and (dv[..., 83:] == 7).all()


@pytest.mark.parametrize("n,t", [(1, 300), (75, 4)])
def test_offsets_past_32_bits(rnn, n, t):
    """Rows of 2^22 floats, the most that there may be: 300 of them take 5 GB."""
    cs = DecayCase(n, t, 2, 1, 24, 40, reverse=1, seed=12, rates=(-5.0, -3.0))
    full, wide = run(rnn, cs), 1 << 22
    x = torch.empty(n, t, wide, device="cuda")
    off = wide - cs.kvstride
    x[..., off:] = cs.kv.cuda()
    geo = (x, wide, off, x, wide, off + cs.koff, off + cs.voff)
    core, rate, st = rnn.DecayCore(2, 24, 40, 1, reverse=1), cs.rate.cuda(), cs.state.cuda()
    y, out = core.forward(n, t, *geo, rate, state=st, keep_state=True)
    assert torch.equal(y, full["y"]) and torch.equal(out, full["state"])
    dx, drate = torch.empty_like(x), torch.zeros_like(rate)
    core.backward(n, t, *geo, rate, cs.dy.cuda(), dx, dx, drate, state=st,
                  dstate_out=cs.dstate.cuda(), set_dq=True, set_dkv=True)
    assert torch.equal(dx[..., off:], full["rest"][0]) and torch.equal(drate, full["drate"])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("reverse", [0, 1])
@pytest.mark.parametrize("t,at", [(6, 3), (100, 37), (100, 64), (700, 600)])
def test_bad_tokens_show_where_they_are_seen(rnn, t, at, reverse, bad):
    """A token's query, key or value that is no number leaves the tokens that do
    not see it as they were, in the outputs and, through dy, in the gradients."""
    n, dk, dv = 1, 24, 40
    cs = DecayCase(n, t, 1, 1, dk, dv, reverse=reverse, seed=8, state=False, rates=(-5.0, -4.0))
    clean = run(rnn, cs)
    sees = torch.arange(t) <= at if reverse else torch.arange(t) >= at
    alone = torch.arange(t) == at
    for col, shows, where in ((3, alone, slice(None)), (cs.koff + 3, sees, slice(None)),
                              (cs.voff + 3, sees, slice(3, 4))):
        old = cs.kv[0, at, col].clone()
        cs.kv[0, at, col] = bad
        y = run(rnn, cs, train=False)["y"]
        cs.kv[0, at, col] = old
        assert torch.equal(y[0, ~shows], clean["y"][0, ~shows])
        assert not torch.isfinite(y[0, shows][..., where]).any()
        rest = torch.ones(dv, dtype=torch.bool)
        rest[where] = False
        assert torch.equal(y[0][:, rest.cuda()], clean["y"][0][:, rest.cuda()])
    cs.dy[0, at, 5] = bad
    got = run(rnn, cs)
    before = torch.arange(t) >= at if reverse else torch.arange(t) <= at
    assert torch.equal(got["dq"][0, ~alone], clean["dq"][0, ~alone])
    assert not torch.isfinite(got["dq"][0, at]).any()
    for nm in ("dk", "dv"):
        assert torch.equal(got[nm][0, ~before], clean[nm][0, ~before]), nm
    assert not torch.isfinite(got["dk"][0, before]).any()
    assert not torch.isfinite(got["dv"][0, before][:, 5]).any()


@pytest.mark.parametrize("size", [1e-18, 1e9])
def test_sizes_far_from_one(rnn, size):
    """Products of 1e-36, and of 1e18 with sums of 1e27."""
    cs = DecayCase(1, 90, 2, 2, 32, 32, reverse=1, seed=9, std=size)
    cs.state = None
    cs.dy /= size
    cs.dstate = None
    got = run(rnn, cs)
    check(cs, got, cs.want(), cs.sizes(), NAMES[:6], extra=0)


def test_gradient_against_differences(rnn):
    """A step along each gradient, central.  The outputs are linear in q, v and
    the state and quadratic in k's and the rates' step of 2^-7, whose third order
    is below 2^-14 of the change; the outputs' rounding over the step is 1e-4 of
    it: within 1e-3."""
    cs = DecayCase(2, 90, 4, 2, 24, 40, reverse=2, seed=10)
    core = rnn.DecayCore(4, 24, 40, 2, reverse=2)
    got = run(rnn, cs)
    x, rate, st = cs.kv.cuda(), cs.rate.cuda(), cs.state.cuda()

    def f(x, rate, st):
        y, s = core.forward(2, 90, *cs.geo(x, x), rate, state=st, keep_state=True)
        return ((y.double() * cs.dy.cuda().double()).sum() +
                (s.double() * cs.dstate.cuda().double()).sum())

    dx = got["rest"][0].clone()
    for i, d in enumerate((dx, got["drate"], got["dstate"])):
        s = 2.0 ** -7 / float(d.abs().max()) * d
        up, dn = [x, rate, st], [x, rate, st]
        up[i], dn[i] = up[i] + s, dn[i] - s
        want = 2 * (s.double() * d.double()).sum()
        assert abs(float(f(*up) - f(*dn) - want)) <= 1e-3 * float(want), i


def test_refusals(rnn):
    core = rnn.DecayCore(4, 16, 24, 2)
    x = torch.zeros(2, 10, 64 + 32 + 48, device="cuda")
    geo, rate = (x, 144, 0, x, 144, 64, 96), torch.zeros(4, device="cuda")
    y = torch.zeros(2, 10, 96, device="cuda")
    with pytest.raises(ValueError):
        core.forward(3, 10, *geo, rate)
    with pytest.raises(ValueError):
        core.forward(2, 11, *geo, rate)
    with pytest.raises(ValueError):
        core.forward(2, 10, x, 144, 0, x, 144, 64, 97, rate)
    with pytest.raises(ValueError):
        core.forward(2, 10, *geo, rate[:3])
    with pytest.raises(TypeError):
        core.forward(2, 10, *geo, rate.double())
    with pytest.raises(TypeError):
        core.forward(2, 10, *geo, rate, lens=torch.tensor([1, 2], device="cuda"))
    with pytest.raises(ValueError):
        core.forward(2, 10, *geo, rate, state=torch.zeros(2, 4, 16, 23, device="cuda"))
    with pytest.raises(rnn.RnnError):
        core.backward(2, 10, *geo, rate, y, None, torch.empty_like(x))
    st = torch.zeros(2, 4, 16, 24, device="cuda")
    with pytest.raises(rnn.RnnError):
        core.backward(2, 10, *geo, rate, y, torch.empty_like(x), torch.empty_like(x), state=st,
                      dstate_out=st, dstate=st)
    with pytest.raises(rnn.RnnError):  # y over the queries, a gradient over its operand
        core.forward(2, 10, *geo, rate, y=x)
    for dq, dkv, dy in ((x, x.clone(), y), (x.clone(), x, y), (x.clone(), x.clone(), None)):
        with pytest.raises(rnn.RnnError):
            core.backward(2, 10, *geo, rate, dq if dy is None else dy, dq, dkv)
    assert core.forward(0, 10, *geo, rate)[0].shape == (0, 10, 96)
    # no tokens: the state passes through
    st = torch.randn(2, 4, 16, 24, device="cuda")
    y0, s0 = core.forward(2, 0, *geo, rate, state=st, keep_state=True)
    assert y0.shape == (2, 0, 96) and torch.equal(s0, st)
    ds = torch.empty_like(st)
    core.backward(2, 0, *geo, rate, y0, torch.empty_like(x), torch.empty_like(x),
                  torch.zeros_like(rate), state=st, dstate_out=st.clone(), dstate=ds)
    assert torch.equal(ds, st)
