"""GPU: differential attention away from magnitude 1: blocks of values that are
zero or small, gradients of any size, tiny queries and keys, long keys,
outliers, and what is not finite, against the operator's formulas in 64 bits.

Tolerances.  A gradient is compared row by row or block by block, each against
TOL (1e-5) of its own terms' size before they cancel: dS_ij = P_ij (dA_ij - D_i)
has the terms P_ij |dA_ij| and P_ij |dO_i| |O_i|, and a sum's size is the root of
the sum of its terms' squares (the terms' errors have no common sign).  A term's
error is a few times 2^-22 (two operands of two fp16 parts, 2^-23 each; the
score's error, 2^-22 |q| |k| scale = 2e-6 at a score of 8, in P; O from the forward,
2^-24 of itself and P's again), so TOL leaves a factor of three at least."""
import pytest
import torch

from conftest import TOL
from diffref import D, DiffCase, seen
from test_gpu_diffattn import run

pytestmark = pytest.mark.gpu


def refill(cs):
    """The buffers of a case again, after its values were changed."""
    nan = float("nan")
    kl = cs.kvv.reshape(cs.n, cs.tk, cs.kw).masked_fill(cs.padk, nan)
    vl = cs.vv.reshape(cs.n, cs.tk, cs.kw).masked_fill(cs.padk, nan)
    cs.q[..., cs.qoff:cs.qoff + cs.qw] = cs.qv.reshape(cs.n, cs.tq, cs.qw).masked_fill(cs.padq, nan)
    cs.kv[..., cs.koff:cs.koff + cs.kw] = kl
    cs.kv[..., cs.voff:cs.voff + cs.kw] = vl
    cs.dy = cs.dyv.masked_fill(cs.padq, nan)
    return cs


def formulas(cs):
    """y, dq, dk, dv and the sizes of their terms, image by image in 64 bits."""
    h, g, dh = cs.h, cs.h // cs.hkv, cs.dh
    lam = cs.lam.to(D)
    e1 = torch.exp((lam[:, 0] * lam[:, 1]).sum(-1))
    e2 = torch.exp((lam[:, 2] * lam[:, 3]).sum(-1))
    lam = (e1 - e2 + cs.lam_init).expand(h).view(h, 1, 1)
    gain = None if cs.gain is None else (1.0 - cs.lam_init) * cs.gain.to(D)
    see = seen(cs.n, cs.tq, cs.tk, cs.causal, cs.diag, cs.qlen, cs.klen)
    out = {k: [] for k in ("y", "dq", "dk", "dv", "sq", "sk", "sv")}
    rep = lambda t: t.repeat_interleave(g, 0)
    fold = lambda t: t.view(cs.hkv, g, *t.shape[1:]).sum(1)
    for b in range(cs.n):
        q = cs.qv[b].to(D).permute(1, 2, 0, 3)                       # [h, 2, tq, dh]
        k = rep(cs.kvv[b].to(D).permute(1, 2, 0, 3))
        v = rep(cs.vv[b].to(D).permute(1, 0, 2))                     # [h, tk, 2 dh]
        dy = cs.dyv[b].to(D).masked_fill(cs.padq[b], 0.0).view(cs.tq, h, 2 * dh).permute(1, 0, 2)
        p, o = [], []
        for m in range(2):
            s = q[:, m] @ k[:, m].transpose(1, 2) * cs.scale
            s = torch.softmax(s.masked_fill(~see[b], -1e300), -1) * see[b].any(-1, keepdim=True)
            p.append(s)
            o.append(s @ v)
        O = o[0] - lam * o[1]
        if gain is None:
            y, do = O, dy
        else:
            r = 1.0 / torch.sqrt((O * O).mean(-1, keepdim=True) + cs.eps)
            y = O * r * gain
            t = dy * gain
            do = r * (t - O * r * (t * O * r).mean(-1, keepdim=True))
        da, a = do @ v.transpose(1, 2), p[0] - lam * p[1]
        big = do.norm(dim=-1, keepdim=True)
        out["y"].append(y.permute(1, 0, 2).reshape(cs.tq, -1))
        out["dv"].append(fold(a.transpose(1, 2) @ do))
        out["sv"].append(fold(((p[0] + lam * p[1]) ** 2).transpose(1, 2) @ big ** 2).sqrt())
        grads = {n: [] for n in ("dq", "dk", "sq", "sk")}
        for m in range(2):
            c = 1.0 if m == 0 else -lam
            ds = c * p[m] * (da - (do * o[m]).sum(-1, keepdim=True)) * cs.scale
            t = (c * p[m] * (da.abs() + big * o[m].norm(dim=-1, keepdim=True)) * cs.scale) ** 2
            grads["dq"].append(ds @ k[:, m])
            grads["dk"].append(fold(ds.transpose(1, 2) @ q[:, m]))
            grads["sq"].append((t @ k[:, m].norm(dim=-1, keepdim=True) ** 2).sqrt())
            grads["sk"].append(fold(t.transpose(1, 2) @ q[:, m].norm(dim=-1, keepdim=True) ** 2).sqrt())
        for n, x in grads.items():
            out[n].append(torch.stack(x, 1))
    t = {n: torch.stack(x) for n, x in out.items()}
    t["dq"] = t["dq"].permute(0, 3, 1, 2, 4)                         # [n, tq, h, 2, dh]
    t["sq"] = t["sq"].permute(0, 3, 1, 2, 4)
    t["dk"] = t["dk"].permute(0, 3, 1, 2, 4)
    t["sk"] = t["sk"].permute(0, 3, 1, 2, 4)
    t["dv"] = t["dv"].permute(0, 2, 1, 3)                            # [n, tk, hkv, 2 dh]
    t["sv"] = t["sv"].permute(0, 2, 1, 3)
    return t


def shaped(cs, got):
    return dict(y=got["y"].to(D), dq=got["dq"].to(D).reshape(cs.n, cs.tq, cs.h, 2, cs.dh),
                dk=got["dk"].to(D).reshape(cs.n, cs.tk, cs.hkv, 2, cs.dh),
                dv=got["dv"].to(D).reshape(cs.n, cs.tk, cs.hkv, 2 * cs.dh))


def check(cs, got, per_row=False, tol=TOL, what=("dq", "dk", "dv")):
    """Gradients per block of 64 queries or keys of an image, or per query row
    and per key, each against tol of its terms' size; y by its norm."""
    want, got = formulas(cs), shaped(cs, got)
    assert torch.isfinite(got["y"]).all() and (got["y"] - want["y"]).norm() <= TOL * want["y"].norm()
    for nm in what:
        assert torch.isfinite(got[nm]).all(), nm
        err, size = (got[nm] - want[nm]) ** 2, want["s" + nm[1]] ** 2
        if per_row:  # each head's, each map's own row
            bad = (err.sum(-1) > tol ** 2 * size[..., 0]).nonzero()
            assert not len(bad), (nm, bad[:4].tolist(), float((err.sum(-1) / size[..., 0]).max()) ** 0.5)
            continue
        err, size = err.flatten(2).sum(-1), size.flatten(2).sum(-1)
        for r0 in range(0, err.shape[1], 64):
            e, s = err[:, r0:r0 + 64].sum(1), size[:, r0:r0 + 64].sum(1)
            assert (e <= tol ** 2 * s).all(), (nm, r0, float((e / s).max()) ** 0.5)


# one for each kernel and sharing of rows and keys of the backward
PATHS = [
    ("rows_by_key_64", 1, 2, 2, 64, 100, 300, {}),
    ("rows_by_key_32", 1, 4, 2, 32, 90, 330, {}),
    ("rows_by_key_shared_48", 2, 4, 1, 48, 70, 200, dict(causal=True)),
    ("few_rows", 1, 2, 2, 32, 9, 333, {}),
    ("four_groups_16", 64, 4, 4, 16, 130, 140, {}),
    ("four_groups_64", 32, 8, 8, 64, 66, 150, {}),
    ("joint_one_tile", 3, 2, 2, 32, 50, 64, {}),
    ("joint_tiles_32", 64, 4, 4, 32, 20, 200, {}),
    ("joint_tiles_64", 128, 4, 2, 64, 9, 201, dict(causal=True)),
    ("unaligned", 2, 2, 1, 5, 70, 200, dict(gap=1)),
]
NAMES = [p[0] for p in PATHS]


def path(p, **kw):
    return DiffCase(*p[1:7], True, **dict(dict(gap=0), **p[7], **kw))


# one for each sharing of the forward: one group of rows, two, four, two waves on
# a row's keys, split keys, unaligned
FORWARD = [
    ("one_group", 3, 4, 2, 32, 10, 150, {}),
    ("two_groups", 3, 4, 2, 32, 50, 150, {}),
    ("four_groups", 3, 4, 2, 32, 150, 150, {}),
    ("halves", 1, 2, 2, 64, 200, 190, {}),
    ("split", 2, 2, 2, 64, 3, 900, {}),
    ("split_of_many", 1, 2, 2, 32, 2, 5000, {}),
    ("unaligned", 2, 2, 2, 5, 40, 90, dict(gap=1)),
]


@pytest.mark.parametrize("factor", [0.0, 2.0 ** -20, 2.0 ** -60])
@pytest.mark.parametrize("p", PATHS, ids=NAMES)
def test_a_block_of_small_values(rnn, p, factor):
    """The first, a middle and the last 64 keys' values times factor, in turn:
    D_i, a mean over all of a row's keys, is then far above that block's dA."""
    tk = p[6]
    for k0 in sorted({0, 64 * (tk // 128), (tk - 1) // 64 * 64}):
        cs = path(p, seed=k0 + 1)
        cs.vv[:, k0:k0 + 64] *= factor
        check(cs, run(rnn, refill(cs)))


@pytest.mark.parametrize("p", PATHS, ids=NAMES)
def test_values_all_zero(rnn, p):
    cs = path(p, seed=5)
    cs.vv.zero_()
    got = run(rnn, refill(cs))
    for nm in ("y", "dq", "dk"):
        assert (got[nm] == 0).all(), nm
    assert torch.isfinite(got["dv"]).all()


@pytest.mark.parametrize("two", [-100, -84, -60, 40])
@pytest.mark.parametrize("p", PATHS, ids=NAMES)
def test_gradients_of_any_magnitude(rnn, p, two):
    """All of dy times a power of two: the gradients' too."""
    cs = path(p, seed=6)
    cs.dyv *= 2.0 ** two
    check(cs, run(rnn, refill(cs)))


@pytest.mark.parametrize("two", [-110, -84, -40, -12, 12])
@pytest.mark.parametrize("p", PATHS, ids=NAMES)
def test_rows_of_another_magnitude(rnn, p, two):
    """Every third query's dy, and then all but one query's, times a power of
    two: each row of dQ stays within its own size."""
    for part in (slice(0, None, 3), slice(1, None)):
        cs = path(p, seed=7)
        cs.dyv[:, part] *= 2.0 ** two
        got = run(rnn, refill(cs))
        check(cs, got, per_row=True, what=("dq",))
        check(cs, got)


@pytest.mark.parametrize("p", PATHS, ids=NAMES)
def test_rows_without_gradient(rnn, p):
    """dy of zeros, in some rows and in all, with values far from 1."""
    for part in (slice(0, None, 2), slice(None)):
        cs = path(p, seed=8, gain=False)
        cs.vv *= 2.0 ** 60
        cs.dyv[:, part] = 0.0
        got = run(rnn, refill(cs))
        assert (got["dq"][:, part] == 0).all()
        check(cs, got)
        if part == slice(None):
            assert (got["dk"] == 0).all() and (got["dv"] == 0).all()


@pytest.mark.parametrize("p", PATHS, ids=NAMES)
def test_tiny_queries_and_keys(rnn, p):
    """Scores below the smallest float: every key that is seen weighs the same,
    also where a mask or the last tile's end hides some."""
    for opt in (dict(), dict(causal=True), dict(klen=[max(1, p[6] - 3)] * p[1])):
        cs = path(p, seed=9, **opt) if not p[7].get("causal") else path(p, seed=9)
        cs.qv *= 2.0 ** -70
        cs.kvv *= 2.0 ** -70
        check(cs, run(rnn, refill(cs)))


@pytest.mark.parametrize("tq,tk,dh", [(70, 65536, 64), (33, 262144, 16), (3, 200000, 32)])
def test_gradients_over_long_keys(rnn, tq, tk, dh):
    """P falls with the number of keys; dS keeps its bits: 4 times 2^-22 (1e-6) of
    the terms' size, by row and by block.  dQ is besides a sum of 3 tk / 16 matrix
    instructions, each cut off by at most 2^-23, 2^-24 in the mean, of a partial sum
    that is at most as large; half-way signs turn, so that these add like a random
    walk: 2^-24 sqrt(3 tk / 16), 6.6e-6 at 65536 keys.  So is the O that D in dK
    comes from; dV has neither."""
    cs = DiffCase(1, 1, 1, dh, tq, tk, True, gap=0, seed=10)
    got = run(rnn, cs)
    tol = 1e-6 + 2.0 ** -24 * (3 * tk / 16) ** 0.5
    check(cs, got, per_row=True, tol=tol, what=("dq",))
    check(cs, got, tol=tol, what=("dk",))
    check(cs, got, tol=1e-6, what=("dv",))


@pytest.mark.parametrize("p", PATHS, ids=NAMES)
def test_an_outlier_among_the_values(rnn, p):
    """One value 2^14 times larger than the others', at a key that hardly counts
    (a score 14 below the others'): dS of the other keys keeps its bits.  That key
    itself has |q| |k| scale up to 12 * 14 = 170, so its scores, and P, are within
    2^-22 170 = 4e-5."""
    cs = path(p, seed=11)
    key = p[6] // 2
    cs.qv[..., 0] = 1.0
    cs.kvv[..., 0] = 0.0
    cs.kvv[:, key, :, :, 0] = -14.0 * p[4] ** 0.5
    cs.vv[:, key] *= 2.0 ** 14
    got = run(rnn, refill(cs))
    check(cs, got, per_row=True, what=("dq",))
    check(cs, got, per_row=True, tol=TOL + 4e-5, what=("dk",))
    rest = [j for j in range(p[6]) if j != key]
    want, have = formulas(cs), shaped(cs, got)
    err = ((have["dk"] - want["dk"])[:, rest] ** 2).sum(-1)
    assert (err <= TOL ** 2 * want["sk"][:, rest, ..., 0] ** 2).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("f", FORWARD, ids=[f[0] for f in FORWARD])
def test_what_is_not_finite_shows(rnn, f, bad):
    """A NaN or an infinity in a query, or in a key, of either map: NaN in every
    row that takes it, of that key head's query heads alone."""
    g = f[2] // f[3]
    clean = run(rnn, path(f, seed=12), train=False)["y"]
    view = lambda y: y.view(f[1], f[5], f[2], 2 * f[4])
    for m in range(2):
        cs = path(f, seed=12)
        cs.qv[0, 1, 1, m, 2] = bad
        y = view(run(rnn, refill(cs), train=False)["y"])
        assert torch.isnan(y[0, 1, 1]).all(), ("query", m)
        y[0, 1, 1] = view(clean)[0, 1, 1]
        assert torch.equal(y, view(clean)), ("query", m)
        for key in (0, f[6] // 2, f[6] - 1):
            cs = path(f, seed=12)
            cs.kvv[0, key, 1, m, 2] = bad
            got = run(rnn, refill(cs))
            y = view(got["y"])
            assert torch.isnan(y[0, :, g:2 * g]).all(), ("key", m, key)
            dq = got["dq"].view(f[1], f[5], f[2], -1)
            assert not torch.isfinite(dq[0, :, g:2 * g]).any(), ("dq", m, key)
            y[0, :, g:2 * g] = view(clean)[0, :, g:2 * g]
            assert torch.equal(y, view(clean)), ("key", m, key)


@pytest.mark.parametrize("f", [f for f in FORWARD if f[5] >= 40],
                         ids=[f[0] for f in FORWARD if f[5] >= 40])
def test_hidden_keys_that_are_not_finite(rnn, f):
    """Keys (not values) that a mask hides from a row may hold anything, finite or
    not: causal rows before such a key stay as they were, to the rounding of
    another power of two.  (With fewer rows, every row sees the key.)"""
    for bad in (float("nan"), float("inf")):
        cs = path(f, seed=13, causal=True)
        want = formulas(cs)["y"]
        key = f[6] - 8
        cs.kvv[0, key] = bad
        y = run(rnn, refill(cs), train=False)["y"].to(D)
        # query i sees keys up to i + tk - tq
        blind = key - (f[6] - f[5])
        err = (y[0, :blind] - want[0, :blind]).norm()
        assert err <= TOL * want[0, :blind].norm()
        assert torch.isnan(y[0, blind:]).all()


@pytest.mark.parametrize("f", FORWARD, ids=[f[0] for f in FORWARD])
def test_scores_far_below_zero(rnn, f):
    """Every score about -2^112: the largest still takes all.  Key j's is
    -(tk - j + 2) 2^100 or so, exact in its leading bits: the last key wins by
    2^100 over a score's error of 2^-22 2^112."""
    cs = path(f, seed=14, gain=False)
    tk = f[6]
    cs.qv.zero_()
    cs.kvv.zero_()
    cs.qv[..., 1] = 2.0 ** 50
    cs.kvv[..., 1] = -(2.0 ** 50) * (tk + 2.0 - torch.arange(tk).view(1, -1, 1, 1))
    cs.scale = 1.0
    y = run(rnn, refill(cs), train=False)["y"].to(D)
    want = formulas(cs)["y"]
    assert (y - want).norm() <= TOL * want.norm()


@pytest.mark.parametrize("two", [-80, 40, 80])
@pytest.mark.parametrize("f", FORWARD, ids=[f[0] for f in FORWARD])
def test_norm_of_any_magnitude(rnn, f, two):
    """Values far from 1 under the norm: mean O^2 passes a float's range (2^160)."""
    cs = path(f, seed=15)
    cs.vv *= 2.0 ** two
    check(cs, run(rnn, refill(cs)))


@pytest.mark.parametrize("two", [12, 20, 26, 60, 110])
@pytest.mark.parametrize("f", FORWARD, ids=[f[0] for f in FORWARD])
def test_large_scores(rnn, f, two):
    """Scores far apart and of any size: the largest takes all (the two largest of
    these are some 2^two / 16 apart, a score's error 2^-22 of it), and gradients
    stay numbers."""
    cs = path(f, seed=16, gain=False)
    cs.qv *= 2.0 ** (two // 2)
    cs.kvv *= 2.0 ** (two - two // 2)
    got = run(rnn, refill(cs))
    want = formulas(cs)["y"]
    assert (got["y"].to(D) - want).norm() <= TOL * want.norm()
    for nm in ("dq", "dk", "dv", "dlam"):
        assert torch.isfinite(got[nm]).all(), nm


@pytest.mark.parametrize("p", PATHS, ids=NAMES)
def test_gradients_near_the_largest_float(rnn, p):
    """dA of some 2^118: within a float's range, |dO| sqrt(W) max |V| past it."""
    cs = path(p, seed=17, gain=False)
    cs.vv *= 2.0 ** 60
    cs.vv[:, p[6] // 2, :, 1] *= 2.0 ** 6
    cs.dyv *= 2.0 ** 56
    cs.qv[..., 0] = 0.0
    check(cs, run(rnn, refill(cs)))
