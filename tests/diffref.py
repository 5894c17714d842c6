"""Plain statements in 64 bits (CPU) of the operators of the differential
block: rotary positions, differential attention and the Linear product with
activation and residual; gradients by automatic differentiation."""
import math

import torch

D = torch.float64


def rotary(x, heads, dh, pos, pairs, base, interleaved, inverse=False):
    """x [rows, heads * dh], pos [rows, axes]."""
    rows, R = x.shape[0], sum(pairs)
    ang = []
    for a, k in enumerate(pairs):
        for p in range(k):
            ang.append(pos[:, a].to(D) * float(base) ** (-p / k))
    v = x.to(D).reshape(rows, heads, dh).clone()
    if R:
        ang = torch.stack(ang, -1)[:, None]
        c, s = torch.cos(ang), torch.sin(ang) * (-1.0 if inverse else 1.0)
        ia = torch.arange(R) * 2 if interleaved else torch.arange(R)
        ib = ia + (1 if interleaved else R)
        a, b = v[..., ia].clone(), v[..., ib].clone()
        v[..., ia], v[..., ib] = a * c - b * s, a * s + b * c
    return v.reshape(rows, -1)


def seen(n, tq, tk, causal, diag, qlen, klen):
    """[n, tq, tk]: whether a query sees a key."""
    nq = torch.full((n,), tq) if qlen is None else qlen.long().clamp(max=tq)
    nk = torch.full((n,), tk) if klen is None else klen.long().clamp(max=tk)
    i, j = torch.arange(tq).view(1, -1, 1), torch.arange(tk).view(1, 1, -1)
    nq, nk = nq.view(-1, 1, 1), nk.view(-1, 1, 1)
    s = (i < nq) & (j < nk)
    if causal:
        s = s & (j <= i + nk - nq)
    if diag:
        s = s & (i != j)
    return s


def diff_attn(q, k, v, lam, gain, see, scale, lam_init, eps, parts=None):
    """q [n, tq, h, 2, dh], k [n, tk, hkv, 2, dh], v [n, tk, hkv, 2 dh], lam
    [1 or h, 4, dh] in 64 bits -> y [n, tq, h * 2 dh]; parts (a dict) receives
    O and P_2 V, [n, h, tq, 2 dh]."""
    n, tq, h, _, dh = q.shape
    tk, hkv = k.shape[1], k.shape[2]
    k = k.repeat_interleave(h // hkv, 2)
    v = v.repeat_interleave(h // hkv, 2).permute(0, 2, 1, 3)
    some = see.any(-1)[:, None, :, None]
    p = []
    for m in range(2):
        s = q[:, :, :, m].permute(0, 2, 1, 3) @ k[:, :, :, m].permute(0, 2, 3, 1) * scale
        s = s.masked_fill(~see[:, None], -1e300)
        p.append(torch.softmax(s, -1) * some if tk else s)
    l = (torch.exp((lam[:, 0] * lam[:, 1]).sum(-1)) - torch.exp((lam[:, 2] * lam[:, 3]).sum(-1))
         + lam_init).expand(h).view(1, h, 1, 1)
    o = (p[0] - l * p[1]) @ v
    if parts is not None:
        parts.update(o=o, o2=p[1] @ v)
    if gain is not None:
        o = (1.0 - lam_init) * gain * o / torch.sqrt((o * o).mean(-1, keepdim=True) + eps)
    return o.permute(0, 2, 1, 3).reshape(n, tq, -1)


def act(name, z):
    F = torch.nn.functional
    return {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu,
            "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[name](z)


class DiffCase:
    """Inputs of one differential-attention call in a fused buffer (self) or
    queries and a memory (cross), with extra columns around the heads; what
    the call must not read -- the columns between, padding rows -- is NaN."""

    def __init__(self, n, h, hkv, dh, tq, tk, cross, causal=False, diag=False, qlen=None,
                 klen=None, per_head=False, gain=True, gap=3, scale=None, amp=1.0, seed=0):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float32)
        self.__dict__.update(n=n, h=h, hkv=hkv, dh=dh, tq=tq, tk=tk, cross=cross, causal=causal,
                             diag=diag, per_head=per_head)
        self.qw, self.kw = 2 * h * dh, 2 * hkv * dh
        self.scale = 1.0 / math.sqrt(dh) if scale is None else scale
        self.lam_init, self.eps = 0.8, 1e-5
        self.qlen = None if qlen is None else torch.tensor(qlen, dtype=torch.int32)
        self.klen = None if klen is None else torch.tensor(klen, dtype=torch.int32)
        self.qv = rnd(n, tq, h, 2, dh) * amp
        self.kvv = rnd(n, tk, hkv, 2, dh)
        self.vv = rnd(n, tk, hkv, 2 * dh)
        self.lam = rnd(h if per_head else 1, 4, dh) * 0.2
        self.gain = 1.0 + 0.1 * rnd(2 * dh) if gain else None
        self.dyv = rnd(n, tq, self.qw)
        nan = float("nan")
        self.padq = self._pad(self.qlen, tq)
        self.padk = self._pad(self.klen, tk)
        ql = self.qv.reshape(n, tq, self.qw).masked_fill(self.padq, nan)
        kl = self.kvv.reshape(n, tk, self.kw).masked_fill(self.padk, nan)
        vl = self.vv.reshape(n, tk, self.kw).masked_fill(self.padk, nan)
        self.dy = self.dyv.masked_fill(self.padq, nan)
        if cross:
            self.qoff, self.qstride = gap, self.qw + 2 * gap
            self.koff, self.voff, self.kvstride = gap, self.kw + 2 * gap, 2 * self.kw + 3 * gap
            self.q = torch.full((n, tq, self.qstride), nan)
            self.kv = torch.full((n, tk, self.kvstride), nan)
        else:
            self.qoff, self.koff = gap, self.qw + 2 * gap
            self.voff = self.koff + self.kw + gap
            self.qstride = self.kvstride = self.voff + self.kw + gap
            self.q = self.kv = torch.full((n, tq, self.qstride), nan)
        self.q[..., self.qoff:self.qoff + self.qw] = ql
        self.kv[..., self.koff:self.koff + self.kw] = kl
        self.kv[..., self.voff:self.voff + self.kw] = vl

    def _pad(self, lens, t):
        if lens is None:
            return torch.zeros(self.n, t, 1, dtype=torch.bool)
        return (torch.arange(t).view(1, -1) >= lens.long().clamp(max=t).view(-1, 1))[..., None]

    def want(self):
        """y, dq, dk, dv (columns of the heads), dlam, dgain in 64 bits, and
        lam_size: each head's |dO| |P_2 V| over its rows, root of the sum of
        squares, times what turns lambda's gradient into dlam."""
        see = seen(self.n, self.tq, self.tk, self.causal, self.diag, self.qlen, self.klen)
        leaf = lambda t: None if t is None else t.to(D).requires_grad_(True)
        q, k, v, lam, gain = (leaf(t) for t in (self.qv, self.kvv, self.vv, self.lam, self.gain))
        parts = {}
        y = diff_attn(q, k, v, lam, gain, see, self.scale, self.lam_init, self.eps, parts)
        dy = self.dyv.to(D).masked_fill(self.padq, 0.0)
        leaves = [t for t in (q, k, v, lam, gain) if t is not None]
        do, *got = torch.autograd.grad(y, [parts["o"]] + leaves, dy, allow_unused=True)
        got = [torch.zeros_like(l) if t is None else t for t, l in zip(got, leaves)]
        keys = ["dq", "dk", "dv", "dlam"] + (["dgain"] if gain is not None else [])
        out = dict(zip(keys, got), y=y.detach().masked_fill(self.padq, 0.0))
        e = torch.exp((lam[:, ::2] * lam[:, 1::2]).sum(-1)).max()
        rows = do.norm(dim=-1) * parts["o2"].norm(dim=-1)
        out["lam_size"] = float((rows.norm() * e * lam.norm()).detach())
        for nm, t in (("dq", self.tq), ("dk", self.tk), ("dv", self.tk)):
            out[nm] = out[nm].reshape(self.n, t, -1)
        return out
