"""Plain statements in 64 bits of head norms with rotary positions, linear
attention with decay, and gated heads: what their GPU tests compare with.  The
inputs are CPU tensors; a statement's gradients come from automatic
differentiation, its sizes from the same statement on magnitudes."""
import math

import torch

from diffref import D, rotary

U = 2.0 ** -24  # a rounding to 32 bits, relative


# ------------------------------------------------------------ norm and rotary
def head_norm(x, eps):
    return x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + eps)


def norm_rotary(x, gain, hq, hk, dh, pos, pairs, base, inter, eps):
    """x [rows, (hq + hk) dh]; gain [2, dh] or None."""
    u = head_norm(x.view(-1, hq + hk, dh), eps)
    if gain is not None:
        u = u * gain[[0] * hq + [1] * hk]
    return turn(u.reshape(x.shape), hq + hk, dh, pos, pairs, base, inter)


def turn(x, heads, dh, pos, pairs, base, inter, inverse=False):
    """diffref's rotary as a product with its coefficients, through which
    gradients flow."""
    R = sum(pairs)
    one = torch.zeros(x.shape[0], dh, dtype=D)
    ia = torch.arange(R) * 2 if inter else torch.arange(R)
    ib = ia + 1 if inter else ia + R
    one[:, ia] = 1.0
    r = rotary(one, 1, dh, pos, pairs, base, inter, inverse)  # (cos, sin) of each pair
    cos, sin = r[:, None, ia], r[:, None, ib]
    v = x.view(-1, heads, dh)
    y = v.clone()
    a, b = v[..., ia], v[..., ib]
    y[..., ia] = a * cos - b * sin
    y[..., ib] = a * sin + b * cos
    return y.view(x.shape)


def pair_size(x, heads, dh, pairs, inter):
    """|a| + |b| of each channel's pair, |x| of a channel that does not turn."""
    v = x.abs().view(-1, heads, dh)
    s, R = v.clone(), sum(pairs)
    ia = torch.arange(R) * 2 if inter else torch.arange(R)
    ib = ia + 1 if inter else ia + R
    s[..., ia] = s[..., ib] = v[..., ia] + v[..., ib]
    return s.view(x.shape)


# ------------------------------------------------------------ decay
def order(n, t, h, reverse, lens):
    """Rows of a head's tokens in its order: [n][h] lists."""
    out = []
    for b in range(n):
        m = t if lens is None else min(int(lens[b]), t)
        fwd = list(range(m))
        out.append([fwd if j < h - reverse else fwd[::-1] for j in range(h)])
    return out


def decay_attn(q, k, v, rate, s0, scale, reverse=0, lens=None):
    """q [n, t, h, dk], k [n, t, hkv, dk], v [n, t, hkv, dv], s0 [n, h, dk, dv]:
    (y [n, t, h, dv], the last states), by the recurrence, token by token."""
    n, t, h, dk = q.shape
    grp, dv = h // k.shape[2], v.shape[3]
    gam = torch.exp(-torch.exp(rate))
    rows = order(n, t, h, reverse, lens)
    ys, st = {}, []
    zero = torch.zeros(dv, dtype=D)
    for b in range(n):
        for j in range(h):
            s = s0[b, j]
            for i in rows[b][j]:
                s = gam[j] * s + k[b, i, j // grp][:, None] * v[b, i, j // grp][None, :]
                ys[b, i, j] = scale * (q[b, i, j] @ s)
            st.append(s)
    y = torch.stack([ys.get((b, i, j), zero) for b in range(n) for i in range(t) for j in range(h)]
                    ) if n * t else torch.zeros(0, dv, dtype=D)
    return y.view(n, t, h, dv), torch.stack(st).view(n, h, dk, dv)


def decay_map(q, k, v, rate, s0, scale, reverse=0, lens=None, power=0):
    """The same by the whole map gamma^(i - l) (q_i . k_l), each term times its
    distance to the given power: for sizes at which the recurrence is slow."""
    n, t, h, dk = q.shape
    grp = h // k.shape[2]
    g = -torch.exp(rate)
    end = torch.full((n,), t) if lens is None else torch.as_tensor(lens).long().clamp(max=t)
    row = torch.arange(t)
    y, st = [], []
    for j in range(h):
        place = (end[:, None] - 1 - row if j >= h - reverse else row.expand(n, t)).to(D)
        ok = row[None] < end[:, None]
        dist = place[:, :, None] - place[:, None, :]
        see = (dist >= 0) & ok[:, :, None] & ok[:, None, :]
        dist = dist.clamp(min=0)
        w = torch.exp(g[j] * dist) * dist ** power * see
        p = (q[:, :, j] @ k[:, :, j // grp].transpose(1, 2)) * w
        first = (place + 1).clamp(min=0)
        last = (end[:, None] - 1 - place).clamp(min=0)
        f = (torch.exp(g[j] * first) * first ** power * ok)[..., None]
        z = (torch.exp(g[j] * last) * last ** power * ok)[..., None]
        a = torch.exp(g[j] * end) * end.to(D) ** power
        y.append(scale * (p @ v[:, :, j // grp] + (q[:, :, j] @ s0[:, j]) * f))
        st.append(a.view(n, 1, 1) * s0[:, j] +
                  (k[:, :, j // grp] * z).transpose(1, 2) @ v[:, :, j // grp])
    return torch.stack(y, 2), torch.stack(st, 1)


class DecayCase:
    """Inputs of one size in a fused buffer (q | k | v, or q apart from k | v),
    padding rows NaN; want(): outputs and gradients; sizes(): what each could
    come to with all terms of one sign, which bounds its rounding."""

    def __init__(self, n, t, h, hkv, dk, dv, reverse=0, lens=None, state=True, gap=0, seed=0,
                 fused=True, rates=(-6.0, 0.5), std=1.0, stated=True):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g) * std
        self.n, self.t, self.h, self.hkv, self.dk, self.dv = n, t, h, hkv, dk, dv
        self.reverse, self.scale = reverse, 1 / math.sqrt(dk)
        self.lens = None if lens is None else torch.tensor(lens, dtype=torch.int32)
        self.qw, self.kw, self.vw = h * dk, hkv * dk, hkv * dv
        off = 0 if not fused else self.qw
        self.kvstride = off + self.kw + self.vw + 2 * gap
        self.qstride = self.kvstride if fused else self.qw + gap
        self.koff, self.voff = off + gap, off + gap + self.kw
        self.kv = rnd(n, t, self.kvstride)
        self.q = self.kv if fused else rnd(n, t, self.qstride)
        self.fused = fused
        self.rate = rates[0] + torch.rand(h, generator=g) * (rates[1] - rates[0])
        self.state = rnd(n, h, dk, dv) if state else None
        self.dy, self.dstate = rnd(n, t, h * dv), rnd(n, h, dk, dv) if state else None
        if self.lens is not None:  # padding may hold anything
            for b, m in enumerate(lens):
                self.kv[b, m:] = self.q[b, m:] = self.dy[b, m:] = float("nan")

    def geo(self, q, kv):
        return q, self.qstride, 0, kv, self.kvstride, self.koff, self.voff

    def _leaves(self):
        n, t = self.n, self.t
        z = lambda x: torch.nan_to_num(x).to(D) if self.lens is not None else x.to(D)
        q = z(self.q[..., :self.qw]).reshape(n, t, self.h, self.dk)
        k = z(self.kv[..., self.koff:self.koff + self.kw]).reshape(n, t, self.hkv, self.dk)
        v = z(self.kv[..., self.voff:self.voff + self.vw]).reshape(n, t, self.hkv, self.dv)
        s0 = (torch.zeros(n, self.h, self.dk, self.dv, dtype=D) if self.state is None
              else self.state.to(D))
        return q, k, v, s0, z(self.dy).reshape(n, t, self.h, self.dv)

    def want(self, f=decay_map):
        q, k, v, s0, dy = self._leaves()
        xs = [x.requires_grad_(True) for x in (q, k, v, self.rate.to(D), s0)]
        y, st = f(*xs, self.scale, self.reverse, self.lens)
        outs, grads = [y], [dy]
        if self.dstate is not None:
            outs, grads = [y, st], [dy, self.dstate.to(D)]
        got = torch.autograd.grad(outs, xs, grads)
        names = ("dq", "dk", "dv", "drate", "dstate")
        flat = lambda x: x.detach().reshape(self.n, self.t, -1)
        out = dict(y=flat(y), state=st.detach(), drate=got[3], dstate=got[4])
        out.update({m: flat(x) for m, x in zip(names[:3], got[:3])})
        return out

    def sizes(self):
        """want() of magnitudes: no term cancels another, none is negative."""
        q, k, v, s0, dy = (x.detach().abs() for x in self._leaves())
        scale, rev, lens = abs(self.scale), self.reverse, self.lens
        ds = torch.zeros_like(s0) if self.dstate is None else self.dstate.to(D).abs()
        r = self.rate.to(D)
        xs = [x.requires_grad_(True) for x in (q, k, v, s0)]
        y, st = decay_map(*xs[:3], r, xs[3], scale, rev, lens)
        got = torch.autograd.grad([y, st], xs, [dy, ds])
        y1, st1 = decay_map(*xs[:3], r, xs[3], scale, rev, lens, power=1)
        dr = torch.exp(r) * ((y1 * dy).sum((0, 1, 3)) + (st1 * ds).sum((0, 2, 3)))
        flat = lambda x: x.detach().reshape(self.n, self.t, -1)
        return dict(y=flat(y), state=st.detach(), dq=flat(got[0]), dk=flat(got[1]), dv=flat(got[2]),
                    drate=dr.detach(), dstate=got[3])

    def tol(self):
        """Of a sum's terms' size: a product or a factor formed in 32 bits is off
        by a few half steps (8 U: the operands' parts, the power of gamma, the
        product, scale, the last rounding).  The sums take N additions one after
        the other, dk or dv of a dot and a token each; a partial sum is at most
        the terms' size, a rounding at most U of that and of no common sign, so
        that N of them come to sqrt(N) U / 3 of it (their mean square is U^2 / 3,
        partial sums are a half on the average) and three times that is not passed."""
        return U * (8 + math.sqrt(self.t * (self.h // self.hkv) + self.dk + self.dv))


# ------------------------------------------------------------ gate
def gate(x, z, gain, h, d, eps):
    """x, z [rows, h d]; gain [h d] or None."""
    y = head_norm(x.view(-1, h, d), eps) * torch.nn.functional.silu(z).view(-1, h, d)
    return (y if gain is None else y * gain.view(h, d)).reshape(x.shape)
