"""GPU: differential attention (rnn_diff_attn_*, DiffCore) against its plain
statement in 64 bits (diffref.py).

Tolerances.  Results are compared by relative Frobenius error with the parity
tolerance of the other fp32 products, 1e-5.  It is the size of: a score's
error, at most 2^-22 |q| |k| scale (two roundings of half a step, 2^-24 each,
to an element of q and k, and the sums' own), about 2^-22 * 8 = 1.9e-6 at
|q| |k| scale = 8, which is a relative error of its P; the norm and the
differences P_1 - lambda P_2 and dA - D enlarge it by the ratio of the terms'
size to their difference's, below 5 for these inputs.  dlambda sums one term
dO . (P_2 V) a (row, head); the norm makes dO perpendicular to O, so that a
term can vanish (it does with one key).  A term's error is at most |dO| |P_2 V|
times the relative errors of the two, each within the tolerance; over the rows
they add like a random walk's steps (and if they all had one sign, 1000 rows of
the error expected above, 3e-7, would still come to 30 * 3e-7 of that).
"""
import math

import pytest
import torch

from conftest import TOL, rel_frob
from diffref import DiffCase

pytestmark = pytest.mark.gpu


def run(rnn, cs, ctx=None, train=True, set_q=True, set_kv=True, init=None):
    dev = lambda t: None if t is None else t.cuda()
    core = rnn.DiffCore(cs.h, cs.dh, cs.tq, cs.tk, cs.hkv, cs.diag, cs.causal,
                        cs.h if cs.per_head else 1, cs.scale, cs.lam_init, cs.eps, ctx=ctx)
    q = dev(cs.q)
    kv = dev(cs.kv) if cs.cross else q
    geo = (q, cs.qstride, cs.qoff, kv, cs.kvstride, cs.koff, cs.voff)
    lam, gain, qlen, klen = dev(cs.lam), dev(cs.gain), dev(cs.qlen), dev(cs.klen)
    y, saved = core.forward(cs.n, *geo, lam, gain, qlen, klen, train=train)
    out = dict(y=y.cpu())
    if not train:
        return out
    fill = float("nan") if init is None else init
    dq = torch.full_like(q, fill)
    dkv = torch.full_like(kv, fill) if cs.cross else dq
    dlam = torch.zeros_like(lam)
    dgain = None if gain is None else torch.zeros_like(gain)
    core.backward(cs.n, *geo, lam, gain, saved, dev(cs.dy), dq, dkv, dlam, dgain, qlen, klen,
                  set_dq=set_q, set_dkv=set_kv)
    torch.cuda.synchronize()
    dq, dkv = dq.cpu(), dkv.cpu()
    out.update(dq=dq[..., cs.qoff:cs.qoff + cs.qw], dk=dkv[..., cs.koff:cs.koff + cs.kw],
               dv=dkv[..., cs.voff:cs.voff + cs.kw], dlam=dlam.cpu(), full_dq=dq, full_dkv=dkv)
    if gain is not None:
        out["dgain"] = dgain.cpu()
    return out


def compare(cs, got, what=("y", "dq", "dk", "dv", "dgain")):
    want = cs.want()
    for nm in what:
        if nm in want and nm in got:
            assert torch.isfinite(got[nm]).all(), nm
            assert rel_frob(got[nm], want[nm]) < TOL, (nm, rel_frob(got[nm], want[nm]))
    if "dlam" in got:
        err = float((got["dlam"].to(torch.float64) - want["dlam"]).norm())
        assert err <= TOL * want["lam_size"], ("dlam", err, want["lam_size"])


# name, n, h, hkv, dh, tq, tk, cross, options
CASES = [
    ("one_token", 2, 2, 2, 32, 1, 1, False, {}),
    ("one_query", 3, 4, 4, 32, 1, 200, True, {}),
    ("one_key", 2, 2, 2, 16, 40, 1, True, {}),
    ("grid_8x8", 3, 4, 4, 32, 64, 64, False, dict(diag=True)),
    ("grid_4x4_dh64", 2, 3, 3, 64, 16, 16, False, {}),
    ("memory_256", 2, 4, 4, 32, 64, 256, True, {}),
    ("tile_minus", 2, 2, 2, 32, 31, 63, True, {}),
    ("tile_plus", 2, 2, 2, 32, 33, 65, True, {}),
    ("two_tiles", 1, 2, 2, 64, 129, 127, True, {}),
    ("odd_dh", 2, 2, 1, 5, 37, 50, True, dict(gap=1)),
    ("dh_20", 2, 4, 2, 20, 70, 70, False, dict(gap=4)),
    ("dh_48_aligned", 2, 2, 2, 48, 100, 100, False, dict(gap=0)),
    ("dh_64_aligned", 1, 4, 1, 64, 130, 130, False, dict(gap=0)),
    ("dh_16_shared", 2, 6, 2, 16, 90, 150, True, dict(per_head=True, gap=0)),
    ("causal", 2, 2, 2, 32, 150, 150, False, dict(causal=True, gap=0)),
    ("causal_diag", 2, 2, 2, 32, 70, 70, False, dict(causal=True, diag=True)),
    ("causal_longer_keys", 2, 2, 1, 32, 40, 170, True, dict(causal=True)),
    ("causal_shorter_keys", 2, 2, 2, 32, 170, 40, True, dict(causal=True)),
    ("ragged_self", 4, 2, 2, 32, 100, 100, False, dict(qlen=[100, 1, 0, 67], klen=[100, 1, 0, 67])),
    ("ragged_cross", 4, 2, 2, 64, 33, 130, True, dict(klen=[130, 1, 0, 64], per_head=True)),
    ("ragged_causal", 4, 4, 2, 32, 90, 90, False,
     dict(qlen=[90, 64, 3, 89], klen=[90, 64, 3, 89], causal=True)),
    ("ragged_causal_uneven", 4, 2, 2, 32, 90, 90, True,
     dict(qlen=[90, 20, 70, 33], klen=[10, 90, 65, 1], causal=True)),
    ("length_past_end", 2, 2, 2, 32, 50, 60, True, dict(qlen=[99, 4], klen=[77, 5])),
    ("no_gain", 2, 2, 2, 32, 65, 80, True, dict(gain=False)),
    ("few_queries_shared", 3, 8, 2, 64, 3, 700, True, dict(klen=[700, 333, 1], gap=0)),
    ("few_queries_long", 1, 4, 4, 32, 1, 3001, True, dict(gap=0)),
    ("few_queries_causal", 2, 4, 1, 48, 4, 900, True, dict(causal=True, klen=[900, 2], gap=2)),
    ("peaked", 2, 2, 2, 32, 64, 200, True, dict(amp=8.0, gap=0)),
    # one for every way that rows and keys are shared out
    ("one_token_aligned", 3, 4, 2, 64, 1, 1, True, dict(gap=0, causal=True)),
    ("small_shared_48", 3, 6, 2, 48, 21, 60, True, dict(gap=0, causal=True, klen=[60, 7, 0])),
    ("small_shared_16", 2, 4, 1, 16, 16, 64, True, dict(gap=0, per_head=True)),
    ("small_64_ragged", 4, 2, 2, 64, 64, 64, False,
     dict(gap=0, causal=True, diag=True, qlen=[64, 33, 0, 1], klen=[64, 33, 0, 1])),
    ("small_32_shared", 3, 6, 2, 32, 20, 33, True, dict(gap=0, qlen=[20, 3, 11], gain=False)),
    ("few_keys_32", 2, 4, 1, 32, 150, 20, True, dict(gap=0, diag=True)),
    ("few_keys_64", 2, 2, 2, 64, 70, 31, True, dict(gap=0, causal=True)),
    ("few_rows_16", 2, 2, 2, 16, 9, 333, True, dict(gap=0, klen=[333, 70])),
    ("splits_past_32", 1, 2, 2, 16, 1, 8300, True, dict(gap=0, gain=False)),
    ("splits_past_32_odd", 1, 2, 1, 5, 2, 9001, True, dict(gap=1)),
    ("rows_64_split", 1, 2, 2, 32, 50, 600, True, dict(gap=0)),
    ("rows_128_split", 1, 2, 1, 64, 65, 700, True, dict(gap=0, causal=True)),
    ("group_of_three", 2, 6, 2, 32, 47, 140, True, dict(gap=0, causal=True, per_head=True)),
    ("many_few_rows_32", 64, 4, 4, 32, 20, 150, True, dict(gap=0, causal=True, diag=True)),
    ("many_few_rows_64", 128, 4, 2, 64, 9, 201, True,
     dict(gap=0, klen=[37 * i % 202 for i in range(128)])),
    ("many_few_rows_48", 128, 4, 2, 48, 32, 66, True, dict(gap=0, per_head=True)),
    ("many_problems_16", 64, 4, 4, 16, 130, 70, True, dict(gap=0)),
    ("many_problems_64", 64, 8, 8, 64, 66, 65, True, dict(gap=0, causal=True)),
    ("halves_48", 2, 4, 2, 48, 100, 140, True, dict(gap=0, qlen=[100, 7], klen=[140, 65])),
    ("halves_64", 1, 3, 3, 64, 200, 200, False, dict(gap=0, causal=True, diag=True)),
]
IDS = [c[0] for c in CASES]


def case(c, **kw):
    return DiffCase(*c[1:8], **dict(c[8], **kw))


@pytest.mark.parametrize("c", CASES, ids=IDS)
def test_forward_and_gradients(rnn, c):
    cs = case(c)
    got = run(rnn, cs)
    pq = cs.padq.expand_as(got["y"])
    assert (got["y"][pq] == 0).all() and (got["dq"][pq] == 0).all(), "padding queries"
    pk = cs.padk.expand_as(got["dk"])
    assert (got["dk"][pk] == 0).all() and (got["dv"][pk] == 0).all(), "padding keys"
    compare(cs, got)
    # what lies between the heads' columns stays as it was (NaN)
    cols = torch.ones(cs.qstride, dtype=torch.bool)
    cols[cs.qoff:cs.qoff + cs.qw] = False
    if not cs.cross:
        cols[cs.koff:cs.koff + cs.kw] = cols[cs.voff:cs.voff + cs.kw] = False
    assert torch.isnan(got["full_dq"][..., cols]).all()


@pytest.mark.parametrize("c", CASES, ids=IDS)
def test_eval_gives_the_same_output(rnn, c):
    cs = case(c, seed=1)
    a, b = run(rnn, cs, train=False), run(rnn, cs)
    assert torch.equal(a["y"], b["y"])


@pytest.mark.parametrize("name", ["grid_8x8", "memory_256", "ragged_cross", "ragged_self",
                                  "dh_64_aligned", "one_query", "small_shared_48", "few_keys_32"])
def test_gradients_accumulate(rnn, name):
    """Unflagged operands receive old + gradient: one rounding of the sum."""
    cs = case(CASES[IDS.index(name)], seed=2)
    base, acc = run(rnn, cs), run(rnn, cs, set_q=False, set_kv=False, init=0.5)
    for nm in ("dq", "dk", "dv"):
        want = base[nm] + 0.5
        assert (acc[nm] - want).abs().max() <= 2.0 ** -22 * max(1.0, float(want.abs().max())), nm
    part = run(rnn, cs, set_q=True, set_kv=False, init=0.5)
    assert torch.equal(part["dq"], base["dq"]) and torch.equal(part["dv"], acc["dv"])


@pytest.mark.parametrize("name", ["memory_256", "ragged_causal", "few_queries_long"])
def test_same_bits_every_time(rnn, name):
    cs = case(CASES[IDS.index(name)], seed=3)
    a, b = run(rnn, cs), run(rnn, cs)
    for nm in ("y", "dq", "dk", "dv", "dlam", "dgain"):
        assert torch.equal(a[nm], b[nm]), nm


@pytest.mark.parametrize("amp", [1e-18, 1e-6, 1e6, 1e15])
def test_any_magnitude(rnn, amp):
    """Powers of two far from 1 in q, k and v that cancel in the scores leave
    the result but for v's own: q amp, k / amp, v amp.  Without the norm: its
    eps, 1e-5 beside mean(O^2) of 0.02, shows as 2.5e-4 where v is scaled."""
    cs = DiffCase(2, 2, 2, 32, 70, 90, True, gap=0, gain=False, seed=4)
    two = 2.0 ** round(math.log2(amp))
    ref = run(rnn, cs, train=False)["y"]
    cs.q = cs.q * two
    cs.kv = torch.cat([cs.kv[..., :cs.kw] / two, cs.kv[..., cs.kw:] * max(two, 1.0)], -1)
    assert rel_frob(run(rnn, cs, train=False)["y"], ref.double() * max(two, 1.0)) < TOL


def test_gradients_against_differences(rnn):
    """Central differences of <y, dy> along random directions.  Step 2^-6: the
    third-order term is of size step^2 (2.4e-4) relative to the directional
    derivative, the rounding of <y, dy> (2^-24 of sum |y dy|, random) over two
    steps below it."""
    cs = DiffCase(2, 4, 2, 32, 40, 50, True, gap=0, causal=True, seed=5)
    got = run(rnn, cs)
    h = 2.0 ** -6
    g = torch.Generator().manual_seed(9)

    def value():
        return float((run(rnn, cs, train=False)["y"].double() * cs.dy.double()).sum())

    for nm, attr, grad in (("q", "q", got["full_dq"]), ("kv", "kv", got["full_dkv"]),
                           ("lam", "lam", got["dlam"]), ("gain", "gain", got["dgain"])):
        x0 = getattr(cs, attr)
        d = torch.randn(x0.shape, generator=g)
        d = d / d.norm()
        # along the gradient as well, where the derivative is largest
        d = d + grad / grad.norm()
        d = d / d.norm()
        setattr(cs, attr, x0 + h * d)
        up = value()
        setattr(cs, attr, x0 - h * d)
        down = value()
        setattr(cs, attr, x0)
        want = float((grad.double() * d.double()).sum())
        assert abs((up - down) / (2 * h) - want) <= 2e-3 * abs(want), nm


def test_other_stream_and_context(rnn):
    cs = case(CASES[IDS.index("memory_256")], seed=6)
    ref = run(rnn, cs)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx = rnn.Context(0, stream=st)
    got = run(rnn, cs, ctx=ctx)  # called on the current stream, run on st
    st.synchronize()
    ctx.close()
    with torch.cuda.stream(torch.cuda.Stream()):
        ctx = rnn.Context(0)
        again = run(rnn, cs, ctx=ctx)
        ctx.close()
    for nm in ("dlam", "dgain"):
        assert torch.equal(ref[nm], again[nm])
    assert torch.equal(ref["y"], again["y"]) and torch.equal(ref["dq"], again["dq"])
    del got


@pytest.mark.parametrize("name", ["grid_8x8", "ragged_cross", "few_queries_shared",
                                  "few_keys_32"])
def test_captured_and_replayed(rnn, name):
    """Two graphs of two calls share nothing but their context: replayed in
    turn, with eager calls between, each gives its eager result."""
    import numpy as np
    del np
    cs = case(CASES[IDS.index(name)], seed=7)
    core = rnn.DiffCore(cs.h, cs.dh, cs.tq, cs.tk, cs.hkv, cs.diag, cs.causal,
                        cs.h if cs.per_head else 1, cs.scale, cs.lam_init, cs.eps)
    st = torch.cuda.Stream()
    core.ctx = rnn.Context(0, stream=st)
    dev = lambda t: None if t is None else t.cuda()
    lam, gain, qlen, klen, dy = (dev(t) for t in (cs.lam, cs.gain, cs.qlen, cs.klen, cs.dy))
    runs = []
    for s in range(2):
        q = dev(cs.q) * (1.0 + s)
        kv = dev(cs.kv) if cs.cross else q
        geo = (q, cs.qstride, cs.qoff, kv, cs.kvstride, cs.koff, cs.voff)
        out = dict(dq=torch.zeros_like(q), dkv=torch.zeros_like(kv), dlam=torch.zeros_like(lam),
                   dgain=torch.zeros_like(gain))
        if not cs.cross:
            out["dkv"] = out["dq"]

        def call(geo=geo, out=out):
            out["dlam"].zero_()
            out["dgain"].zero_()
            y, saved = core.forward(cs.n, *geo, lam, gain, qlen, klen)
            core.backward(cs.n, *geo, lam, gain, saved, dy, out["dq"], out["dkv"], out["dlam"],
                          out["dgain"], qlen, klen, set_dq=True, set_dkv=True)
            return y

        with torch.cuda.stream(st):
            y = call()
        st.synchronize()
        want = dict(y=y.clone(), **{k: v.clone() for k, v in out.items()})
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            y = call()
        runs.append((graph, y, out, want, call))
    for rep in range(3):
        for graph, y, out, want, call in runs:
            with torch.cuda.stream(st):
                for v in out.values():
                    v.fill_(0.25)
                graph.replay()
            st.synchronize()
            assert torch.equal(y, want["y"]), rep
            for k in ("dlam", "dgain"):
                assert torch.equal(out[k], want[k]), (rep, k)
            for k, off, w in (("dq", cs.qoff, cs.qw), ("dkv", cs.koff, cs.kw),
                              ("dkv", cs.voff, cs.kw)):
                assert torch.equal(out[k][..., off:off + w], want[k][..., off:off + w]), (rep, k)
            with torch.cuda.stream(st):
                call()
            st.synchronize()
    core.ctx.close()


def test_rows_past_32_bit_offsets(rnn):
    """A key and value buffer of more than 2^31 floats, rows 16 MiB apart."""
    n, h, dh, tq, tk = 1, 2, 32, 5, 530
    kw = 2 * h * dh
    stride = 2 ** 22
    cs = DiffCase(n, h, h, dh, tq, tk, True, gap=0, seed=8)
    buf = torch.empty((tk - 1) * stride + 2 * kw, device="cuda")
    view = buf.as_strided((tk, 2 * kw), (stride, 1))
    view.copy_(cs.kv[0])
    core = rnn.DiffCore(h, dh, tq, tk)
    q, lam, gain = cs.q.cuda(), cs.lam.cuda(), cs.gain.cuda()
    geo = (q, cs.qstride, 0, buf, stride, 0, kw)
    y, saved = core.forward(n, *geo, lam, gain)
    ref = run(rnn, cs)
    assert torch.equal(y.cpu(), ref["y"])
    dbuf = torch.empty_like(buf)
    dq = torch.empty_like(q)
    dlam, dgain = torch.zeros_like(lam), torch.zeros_like(gain)
    core.backward(n, *geo, lam, gain, saved, cs.dy.cuda(), dq, dbuf, dlam, dgain, set_dq=True,
                  set_dkv=True)
    got = dbuf.as_strided((tk, 2 * kw), (stride, 1)).cpu()
    assert torch.equal(got[None], ref["full_dkv"]) and torch.equal(dq.cpu(), ref["full_dq"])


def test_empty_sizes(rnn):
    for n, tq, tk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        cs = DiffCase(n, 2, 2, 32, tq, tk, True, gap=0)
        got = run(rnn, cs)
        for nm in ("y", "dq", "dk", "dv", "dlam", "dgain"):
            assert (got[nm] == 0).all(), (n, tq, tk, nm)


def test_refusals(rnn):
    cs = DiffCase(2, 2, 2, 32, 8, 8, True, gap=0)
    core = rnn.DiffCore(2, 32, 8, 8)
    q, kv, lam, gain = cs.q.cuda(), cs.kv.cuda(), cs.lam.cuda(), cs.gain.cuda()
    geo = (q, cs.qstride, 0, kv, cs.kvstride, 0, cs.kw)
    with pytest.raises(TypeError):
        core.forward(2, q.double(), *geo[1:], lam, gain)
    with pytest.raises(TypeError):
        core.forward(2, *geo, lam, gain, klen=torch.zeros(2, device="cuda"))
    with pytest.raises(TypeError):
        core.forward(2, *geo, lam.cpu(), gain)
    with pytest.raises(ValueError):
        core.forward(3, *geo, lam, gain)  # too few rows
    with pytest.raises(ValueError):
        core.forward(2, q, cs.qw - 1, 0, *geo[3:], lam, gain)  # heads do not fit
    with pytest.raises(ValueError):
        core.forward(2, *geo[:5], 0, cs.kw - 1, lam, gain)  # keys over values
    with pytest.raises(ValueError):
        core.forward(2, q, cs.qstride, 0, kv, 2 ** 22 + 1, 0, cs.kw, lam, gain)  # rows too far apart
    y, saved = core.forward(2, *geo, lam, gain, train=False)
    assert saved is None
    with pytest.raises(ValueError):
        core.backward(2, *geo, lam, gain, None, y, q, kv, lam, gain)
    import ctypes as C
    L, ctx, d = rnn.lib(), rnn.default_ctx(), core.desc(cs.qstride, 0, cs.kvstride, 0, cs.kw)
    p = lambda t: t.data_ptr()
    o12, stats = torch.zeros(2 * 8 * 2 * cs.qw, device="cuda"), torch.zeros(2 * 8 * 2 * 4, device="cuda")
    nb = C.c_size_t()
    assert L.rnn_diff_attn_workspace(C.byref(d), 2, 1, C.byref(nb)) == 0 and nb.value > 256
    ws = torch.empty(nb.value + 256, dtype=torch.uint8, device="cuda")
    args = lambda w, nbytes, dgain, flags: (
        ctx.h, C.byref(d), 2, p(q), p(kv), p(lam), p(gain), None, None, p(o12), p(stats), p(y), w,
        nbytes, p(q.clone()), p(kv.clone()), p(lam.clone()), dgain, flags)
    bwd = L.rnn_diff_attn_backward
    assert bwd(*args(p(ws), nb.value - 1, p(gain), 0)) == rnn.RNN_E_INVALID
    assert bwd(*args(None, nb.value, p(gain), 0)) == rnn.RNN_E_NULL
    assert bwd(*args(p(ws) + 16, nb.value, p(gain), 0)) == rnn.RNN_E_INVALID
    assert bwd(*args(p(ws), nb.value, None, 0)) == rnn.RNN_E_NULL
    assert bwd(*args(p(ws), nb.value, p(gain), 8)) == rnn.RNN_E_INVALID
