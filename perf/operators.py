"""The operators of a differential-attention block, as cases that can be timed.

Three operators, each in its plain form (elementary torch operations in 32
bits) and, with ``own`` set, through the package's public entry points:

* ``rotary``: rotary positions with up to three axes (time, height, width) on
  the heads of a fused QKV buffer, forward and its backward (``R.Rotary``);
* ``diff``: differential attention, the difference of two softmax maps with
  learned weights and a norm per head, forward and backward (``R.DiffCore``);
* ``linear``: the product x W^T with bias, activation and residual, forward
  and backward (``R.linear_act_forward`` / ``R.linear_act_backward``).

All data is float32, which is the only type that the framework computes in.
"""
import math

import torch

own = False

DEV = "cuda"
D = torch.float64
BASE = {1: 10000.0, 2: 100.0, 3: 10000.0}  # frequencies' base by the number of axes
LAM0, EPS = 0.8, 1e-5


def listed():
    return [
        # One image's queries and keys, 8 x 8 tokens: the least a serving program asks for.
        _rot("rotary_eval_one", 1, (8, 8), 16, 32),
        # Clips of 8 x 14 x 14 tokens whose frames lie at given, fractional positions.
        _rot("rotary_video_train", 16, (8, 14, 14), 24, 64, explicit=True, interleaved=True,
             train=True),
        # One image of 8 x 8 tokens through a stage-3 block's heads.
        _diff("diff_eval_one", 1, 64, 64, 4, 4, 32),
        # The stage-3 self-attention at the training batch, diagonal masked.
        _diff("diff_self_train", 128, 64, 64, 4, 4, 32, diag=True, train=True),
        # A reader block's cross-attention over the 16 x 16 memory.
        _diff("diff_cross_train", 128, 64, 256, 4, 4, 32, cross=True, train=True),
        # A padded batch of images of up to 24 x 24 patches and a class token.
        _diff("diff_ragged_train", 8, 577, 577, 6, 6, 32, ragged=True, per_head=True, train=True),
        # Clips of 8 x 14 x 14 tokens in time order, each seeing what came before it.
        _diff("diff_video_train", 2, 1568, 1568, 8, 8, 64, causal=True, train=True),
        # A large image of 64 x 64 patches, key heads shared by four query heads.
        _diff("diff_large_eval", 1, 4096, 4096, 8, 2, 64),
        # One pooling query over the tokens of long clips.
        _diff("diff_pool_long", 4, 1, 16384, 8, 2, 64, cross=True, ragged=True),
        # The MLP's first product for one image.
        _lin("linear_eval_one", 64, 256, 1024, "gelu"),
        # The same at the training batch, forward and backward.
        _lin("linear_train", 8192, 256, 1024, "gelu", train=True),
        # A partial batch, sizes that no tile or 16-byte load divides, with a residual.
        _lin("linear_ragged_train", 1813, 387, 1003, "silu", residual=True, train=True),
    ]


def _rot(name, n, grid, heads, dh, explicit=False, interleaved=False, train=False):
    g = (1,) * (3 - len(grid)) + tuple(grid)
    return dict(name=name, kind="rotary", n=n, axes=len(grid), g0=g[0], g1=g[1], g2=g[2],
                heads=heads, dh=dh, explicit=explicit, interleaved=interleaved, train=train)


def _diff(name, n, tq, tk, h, hkv, dh, cross=False, causal=False, diag=False, ragged=False,
          per_head=False, train=False):
    return dict(name=name, kind="diff", n=n, tq=tq, tk=tk, h=h, hkv=hkv, dh=dh, cross=cross,
                causal=causal, diag=diag, ragged=ragged, per_head=per_head, train=train)


def _lin(name, rows, fin, fout, act, residual=False, train=False):
    return dict(name=name, kind="linear", rows=rows, fin=fin, fout=fout, act=act,
                residual=residual, train=train)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case, its batch or length halved until it is no larger than a listed one."""
    c = _draw(rng)
    c.pop("name")
    if c["kind"] == "diff":
        while work(c)["flops"] > (3e10 if c["train"] else 6e10) or \
                c["n"] * c["h"] * c["tq"] * c["tk"] > 1.3e8:
            if c["n"] > 1:
                c["n"] = (c["n"] + 1) // 2
            else:
                c["tq"] = (c["tq"] + 1) // 2
                c["tk"] = c["tk"] if c["cross"] else c["tq"]
    return c


def _draw(rng):
    kind = rng.choice(["rotary", "diff", "diff", "diff", "diff", "linear", "linear"])
    if kind == "rotary":
        axes = rng.randint(1, 3)
        side = rng.randint(4, 24)
        grid = [(_log(rng, 16, 2048),), (side, rng.randint(4, 24)),
                (rng.randint(2, 8), rng.randint(4, 14), rng.randint(4, 14))][axes - 1]
        return _rot("", _log(rng, 1, 24), grid, rng.randint(1, 24), 2 * rng.randint(8, 32),
                    explicit=rng.random() < 0.4, interleaved=rng.random() < 0.5,
                    train=rng.random() < 0.7)
    if kind == "linear":
        mult = rng.choice([1, 1, 4, 32])
        size = lambda lo, hi: max(mult, _log(rng, lo, hi) // mult * mult)
        return _lin("", size(8, 8192), size(64, 1152), size(64, 1152),
                    rng.choice(["relu", "gelu", "gelu_tanh", "silu"]),
                    residual=rng.random() < 0.4, train=rng.random() < 0.6)
    hkv = rng.choice([1, 2, 2, 4])
    h = hkv * rng.choice([1, 1, 2, 3])
    dh = rng.choice([16, 32, 32, 48, 64, 64])
    shape = rng.choice(["self", "self", "cross", "few"])
    flags = dict(ragged=rng.random() < 0.4, per_head=rng.random() < 0.4)
    if shape == "few":
        return _diff("", _log(rng, 1, 32), rng.randint(1, 4), _log(rng, 256, 16384), h, hkv, dh,
                     cross=True, **flags)
    flags["train"] = rng.random() < 0.7
    if shape == "cross":
        return _diff("", _log(rng, 1, 128), _log(rng, 16, 1024), _log(rng, 16, 2048), h, hkv, dh,
                     cross=True, **flags)
    t = _log(rng, 1, 2048)
    return _diff("", _log(rng, 1, 128), t, t, h, hkv, dh, causal=rng.random() < 0.4,
                 diag=rng.random() < 0.3, **flags)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEV) * std


def _grid(c):
    return (c["g0"], c["g1"], c["g2"])[3 - c["axes"]:]


def _pairs(c):
    """Pairs of each axis: an even share, what is left over to the first ones."""
    r, a = c["dh"] // 2, c["axes"]
    return [r // a + (i < r % a) for i in range(a)]


def _rotary_inputs(c, seed):
    """The fused QKV buffer (queries and keys, then as much again for the
    values), a gradient, and explicit positions where the case has them."""
    g = _gen(seed)
    n, t, w = c["n"], c["g0"] * c["g1"] * c["g2"], c["heads"] * c["dh"]
    x, dy = _normal(g, (n, t, w + w // 2)), _normal(g, (n, t, w), 1e-3)
    pos = None
    if c["explicit"]:
        # each clip starts at a frame of its own and is sampled at its own rate
        axes = [torch.arange(s, device=DEV, dtype=torch.float32) for s in _grid(c)]
        co = torch.stack([m.reshape(-1) for m in torch.meshgrid(*axes, indexing="ij")], -1)
        rate = torch.rand((n, 1, c["axes"]), generator=g, device=DEV) + 0.5
        start = torch.randint(0, 20000, (n, 1, 1), generator=g, device=DEV).float()
        first = torch.tensor([1.0] + [0.0] * (c["axes"] - 1), device=DEV)
        pos = (co * rate + start * first).reshape(n * t, c["axes"]).contiguous()
    return x, dy, pos


def _diff_width(c):
    """Floats of a query row, and of a key and value row."""
    return 2 * c["h"] * c["dh"], 4 * c["hkv"] * c["dh"]


def _diff_inputs(c, seed):
    """Self-attention's fused buffer, or queries and a memory; the four
    vectors of each lambda, the norm's gain, lengths of a padded batch and
    the output's gradient."""
    g = _gen(seed)
    n, dh = c["n"], c["dh"]
    qw, kw = _diff_width(c)
    if c["cross"]:
        q, kv = _normal(g, (n, c["tq"], qw)), _normal(g, (n, c["tk"], kw))
    else:
        q = kv = _normal(g, (n, c["tq"], qw + kw))
    lam = _normal(g, (c["h"] if c["per_head"] else 1, 4, dh), 0.1)
    gain = 1.0 + _normal(g, 2 * dh, 0.1)
    dy = _normal(g, (n, c["tq"], qw), 1e-3)
    qlen = klen = None
    if c["ragged"]:
        klen = torch.randint((c["tk"] + 1) // 2, c["tk"] + 1, (n,), generator=g, device=DEV,
                             dtype=torch.int32)
        qlen = klen if not c["cross"] else None
    return q, kv, lam, gain, qlen, klen, dy


def _linear_inputs(c, seed):
    g = _gen(seed)
    r, i, o = c["rows"], c["fin"], c["fout"]
    return (_normal(g, (r, i)), _normal(g, (o, i), 1.0 / math.sqrt(i)), _normal(g, o, 0.1),
            _normal(g, (r, o)) if c["residual"] else None, _normal(g, (r, o), 1e-3))


def prepare(case, seed):
    c = case
    s = {"c": c}
    if c["kind"] == "rotary":
        s["x"], s["dy"], s["pos"] = _rotary_inputs(c, seed)
    elif c["kind"] == "diff":
        s["q"], s["kv"], s["lam"], s["gain"], s["qlen"], s["klen"], s["dy"] = _diff_inputs(c, seed)
    else:
        s["x"], s["w"], s["b"], s["res"], s["dy"] = _linear_inputs(c, seed)
    if own:
        import rustnn_amd as R
        s["R"] = R
        if c["kind"] == "rotary":
            s["rot"] = R.Rotary(c["heads"], c["dh"], _grid(c), BASE[c["axes"]], _pairs(c),
                                c["interleaved"])
        elif c["kind"] == "diff":
            s["core"] = R.DiffCore(c["h"], c["dh"], c["tq"], c["tk"], c["hkv"],
                                   mask_diag=c["diag"], causal=c["causal"],
                                   lam_heads=s["lam"].shape[0], lam_init=LAM0, eps=EPS)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["c"]
    return (_OWN if own else _PLAIN)[c["kind"]](c, s)


def _own_rotary(c, s):
    n, w = c["n"], c["heads"] * c["dh"]
    out = dict(y=s["rot"].forward(n, s["x"], w + w // 2, 0, pos=s["pos"]))
    if c["train"]:
        out["dx"] = s["rot"].backward(n, s["dy"], w, 0, pos=s["pos"])
    return out


def _own_diff(c, s):
    qw, kw = _diff_width(c)
    if c["cross"]:
        geo = (s["q"], qw, 0, s["kv"], kw, 0, kw // 2)
    else:
        geo = (s["q"], qw + kw, 0, s["kv"], qw + kw, qw, qw + kw // 2)
    core, n = s["core"], c["n"]
    y, saved = core.forward(n, *geo, s["lam"], s["gain"], qlen=s["qlen"], klen=s["klen"],
                            train=c["train"])
    out = dict(y=y)
    if c["train"]:
        dq = torch.empty_like(s["q"])
        dkv = torch.empty_like(s["kv"]) if c["cross"] else dq
        dlam, dgain = torch.zeros_like(s["lam"]), torch.zeros_like(s["gain"])
        core.backward(n, *geo, s["lam"], s["gain"], saved, s["dy"], dq, dkv, dlam, dgain,
                      qlen=s["qlen"], klen=s["klen"], set_dq=True, set_dkv=True)
        out.update(dq=dq, dlam=dlam, dgain=dgain)
        if c["cross"]:
            out["dkv"] = dkv
    return out


def _own_linear(c, s):
    R, size = s["R"], (c["rows"], c["fin"], c["fout"])
    y, z = R.linear_act_forward(*size, s["x"], s["w"], s["b"], c["act"], res=s["res"],
                                train=c["train"])
    out = dict(y=y)
    if c["train"]:
        dw, db = torch.zeros_like(s["w"]), torch.zeros_like(s["b"])
        dx = R.linear_act_backward(*size, s["dy"], s["x"], s["w"], z, c["act"], dw, db)
        out.update(dx=dx, dw=dw, db=db)
    return out


# ------------------------------------------------------------------ plain forms
def _angles(c, pos):
    """[n or 1, t, pairs] in 64 bits: far positions lose the angle in 32."""
    if pos is None:
        axes = [torch.arange(s, device=DEV, dtype=D) for s in _grid(c)]
        p = torch.stack([m.reshape(-1) for m in torch.meshgrid(*axes, indexing="ij")], -1)[None]
    else:
        p = pos.to(D).view(c["n"], -1, c["axes"])
    base = BASE[c["axes"]]
    parts = []
    for a, k in enumerate(_pairs(c)):
        w = torch.pow(base, -torch.arange(k, device=DEV, dtype=D) / k)
        parts.append(p[..., a:a + 1] * w)
    return torch.cat(parts, -1)


def _rotate(c, x, ang):
    """x [n, t, heads * dh] turned by ang."""
    n, t, _ = x.shape
    h, r = c["heads"], c["dh"] // 2
    cos, sin = torch.cos(ang).float()[:, :, None], torch.sin(ang).float()[:, :, None]
    if c["interleaved"]:
        v = x.reshape(n, t, h, r, 2)
        a, b = v[..., 0], v[..., 1]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).reshape(n, t, -1)
    v = x.reshape(n, t, h, 2, r)
    a, b = v[..., 0, :], v[..., 1, :]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -2).reshape(n, t, -1)


def _plain_rotary(c, s):
    ang = _angles(c, s["pos"])
    out = dict(y=_rotate(c, s["x"][..., :c["heads"] * c["dh"]], ang))
    if c["train"]:
        out["dx"] = _rotate(c, s["dy"], -ang)
    return out


def _hidden(c, qlen, klen):
    """Which keys a query does not see, [n or 1, 1, tq, tk], and which
    queries are padding, [n or 1, 1, tq, 1] (None: none)."""
    i = torch.arange(c["tq"], device=DEV)[:, None]
    j = torch.arange(c["tk"], device=DEV)[None, :]
    lens = lambda v, t: t if v is None else v.long().view(-1, 1, 1, 1)
    nq, nk = lens(qlen, c["tq"]), lens(klen, c["tk"])
    hide, pad = None, None
    if klen is not None:
        hide = j >= nk
    if c["causal"]:
        late = j > i + (nk - nq)
        hide = late if hide is None else hide | late
    if c["diag"]:
        hide = (j == i) if hide is None else hide | (j == i)
    if qlen is not None:
        pad = i >= nq
        hide = hide | pad
    if hide is not None:
        hide = hide.expand(-1, 1, -1, -1) if hide.dim() == 4 else hide[None, None]
    return hide, pad


def _split(c, q, kv):
    """Queries [n, h, 2, tq, dh], keys [n, h, 2, tk, dh], values
    [n, h, tk, 2 dh], the key heads repeated for their query heads."""
    n, h, hkv, dh = c["n"], c["h"], c["hkv"], c["dh"]
    qw, kw = _diff_width(c)
    rows = kv if c["cross"] else kv[..., qw:]
    qq = q[..., :qw].reshape(n, c["tq"], h, 2, dh).permute(0, 2, 3, 1, 4)
    kk = rows[..., :kw // 2].reshape(n, c["tk"], hkv, 2, dh).permute(0, 2, 3, 1, 4)
    vv = rows[..., kw // 2:].reshape(n, c["tk"], hkv, 2 * dh).permute(0, 2, 1, 3)
    if h != hkv:
        kk = kk.repeat_interleave(h // hkv, 1)
        vv = vv.repeat_interleave(h // hkv, 1)
    return qq.contiguous(), kk.contiguous(), vv.contiguous()


def _plain_diff(c, s):
    n, h, hkv, dh, tq, tk = (c[k] for k in ("n", "h", "hkv", "dh", "tq", "tk"))
    scale = 1.0 / math.sqrt(dh)
    q, k, v = _split(c, s["q"], s["kv"])
    hide, pad = _hidden(c, s["qlen"], s["klen"])
    lam4 = s["lam"].expand(h, 4, dh)
    e1 = torch.exp((lam4[:, 0] * lam4[:, 1]).sum(-1))
    e2 = torch.exp((lam4[:, 2] * lam4[:, 3]).sum(-1))
    lam = (e1 - e2 + LAM0).view(1, h, 1, 1)
    p, o = [], []
    for m in range(2):
        x = (q[:, :, m] @ k[:, :, m].transpose(-1, -2)) * scale
        if hide is not None:
            x = x.masked_fill(hide, -math.inf)
        top = x.amax(-1, keepdim=True)
        x = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = x.sum(-1, keepdim=True)
        p.append(x / torch.where(total == 0, torch.ones_like(total), total))
        o.append(p[m] @ v)
    out = o[0] - lam * o[1]
    r = torch.rsqrt((out * out).mean(-1, keepdim=True) + EPS)
    hat = out * r
    back = lambda t: t.permute(0, 2, 1, 3).reshape(n, t.shape[2], -1)
    gain = (1.0 - LAM0) * s["gain"]
    res = dict(y=back(hat * gain))
    if not c["train"]:
        return res
    dy = s["dy"].view(n, tq, h, 2 * dh).permute(0, 2, 1, 3)
    if pad is not None:
        dy = dy.masked_fill(pad, 0.0)
    res["dgain"] = (dy * hat).sum((0, 1, 2)) * (1.0 - LAM0)
    t = dy * gain
    do = r * (t - hat * (t * hat).mean(-1, keepdim=True))
    da = do @ v.transpose(-1, -2)
    dv = (p[0] - lam * p[1]).transpose(-1, -2) @ do
    d2 = (do * o[1]).sum(-1, keepdim=True)
    ds = [p[0] * (da - (do * o[0]).sum(-1, keepdim=True)), p[1] * (d2 - da) * lam]
    dq = [ds[m] @ k[:, :, m] * scale for m in range(2)]
    dk = [ds[m].transpose(-1, -2) @ q[:, :, m] * scale for m in range(2)]
    dl = -d2.sum((0, 2, 3))
    dlam = torch.stack([(dl * e1)[:, None] * lam4[:, 1], (dl * e1)[:, None] * lam4[:, 0],
                        -(dl * e2)[:, None] * lam4[:, 3], -(dl * e2)[:, None] * lam4[:, 2]], 1)
    res["dlam"] = dlam if s["lam"].shape[0] == h else dlam.sum(0, keepdim=True)
    dq = torch.stack(dq, 2).permute(0, 3, 1, 2, 4).reshape(n, tq, -1)
    dk = torch.stack(dk, 2).view(n, hkv, h // hkv, 2, tk, dh).sum(2)
    dv = dv.view(n, hkv, h // hkv, tk, 2 * dh).sum(2)
    dkv = torch.cat([dk.permute(0, 3, 1, 2, 4).reshape(n, tk, -1),
                     dv.permute(0, 2, 1, 3).reshape(n, tk, -1)], -1)
    if c["cross"]:
        res["dq"], res["dkv"] = dq, dkv
    else:
        res["dq"] = torch.cat([dq, dkv], -1)
    return res


def _act(kind, z):
    """act(z) and act'(z)."""
    if kind == "relu":
        on = (z > 0).float()
        return z * on, on
    if kind == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return z * sig, sig * (1.0 + z * (1.0 - sig))
    if kind == "gelu":
        phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    k = math.sqrt(2.0 / math.pi)
    th = torch.tanh(k * (z + 0.044715 * z * z * z))
    return (0.5 * z * (1.0 + th),
            0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * k * (1.0 + 3 * 0.044715 * z * z))


def _plain_linear(c, s):
    z = s["x"] @ s["w"].T + s["b"]
    a, slope = _act(c["act"], z)
    out = dict(y=a if s["res"] is None else a + s["res"])
    if c["train"]:
        dz = s["dy"] * slope
        out.update(dx=dz @ s["w"], dw=dz.T @ s["x"], db=dz.sum(0))
    return out


_OWN = dict(rotary=_own_rotary, diff=_own_diff, linear=_own_linear)
_PLAIN = dict(rotary=_plain_rotary, diff=_plain_diff, linear=_plain_linear)


# ------------------------------------------------------------------ work
def work(case):
    c = case
    if c["kind"] == "rotary":
        rows = c["n"] * c["g0"] * c["g1"] * c["g2"]
        el = rows * c["heads"] * c["dh"] * (2 if c["train"] else 1)
        return dict(bytes=8 * el + (4 * rows * c["axes"] if c["explicit"] else 0), flops=3 * el)
    if c["kind"] == "diff":
        qw, kw = _diff_width(c)
        tk, tq = c["tk"], c["tq"]
        if c["ragged"]:  # lengths lie between a half and the whole
            tk = 0.75 * tk
            tq = tq if c["cross"] else 0.75 * tq
        seen = tq * tk * (0.5 if c["causal"] else 1.0) * c["n"] * c["h"]
        q, kv = c["n"] * tq * qw, c["n"] * tk * kw
        # queries, keys and values read, the output written; for the backward
        # the output's gradient read and three gradients written besides
        el = 2 * q + kv + (2 * q + kv if c["train"] else 0)
        return dict(bytes=4 * el, flops=(28 if c["train"] else 8) * c["dh"] * seen)
    r, i, o = c["rows"], c["fin"], c["fout"]
    el = r * i + o * i + r * o * (2 if c["residual"] else 1)
    if c["train"]:
        el += r * o + r * i + o * i
    return dict(bytes=4 * el, flops=2 * r * i * o * (3 if c["train"] else 1))


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    return _EXACT[case["kind"]](case, seed)


def _exact_rotary(c, seed):
    """A rotation as the product of complex numbers, its backward as the
    product with the conjugate."""
    x, dy, pos = _rotary_inputs(c, seed)
    n, t, h, r = c["n"], x.shape[1], c["heads"], c["dh"] // 2
    idx = torch.arange(t, device=DEV)
    coords = []
    for size in reversed(_grid(c)):
        coords.append((idx % size).to(D).expand(n, t))
        idx = idx // size
    coords = coords[::-1]
    if pos is not None:
        coords = [pos[:, a].to(D).view(n, t) for a in range(c["axes"])]
    ang = []
    for a, k in enumerate(_pairs(c)):
        for p in range(k):
            ang.append(coords[a] * BASE[c["axes"]] ** (-p / k))
    turn = torch.exp(1j * torch.stack(ang, -1))[:, :, None]

    def apply(v, turn):
        v = v.to(D).reshape(n, t, h, *((r, 2) if c["interleaved"] else (2, r)))
        if not c["interleaved"]:
            v = v.transpose(-1, -2)
        w = torch.view_as_real(torch.view_as_complex(v.contiguous()) * turn)
        return (w if c["interleaved"] else w.transpose(-1, -2)).reshape(n, t, -1)

    out = dict(y=apply(x[..., :h * c["dh"]], turn))
    if c["train"]:
        out["dx"] = apply(dy, turn.conj())
    return out


def _exact_diff(c, seed):
    """One query head at a time, its gradients by automatic differentiation."""
    q, kv, lam, gain, qlen, klen, dy = _diff_inputs(c, seed)
    n, h, hkv, dh, tq, tk = (c[k] for k in ("n", "h", "hkv", "dh", "tq", "tk"))
    qw, kw = _diff_width(c)
    see = torch.ones(n, tq, tk, dtype=torch.bool, device=DEV)
    nq = torch.full((n,), tq, device=DEV) if qlen is None else qlen.long()
    nk = torch.full((n,), tk, device=DEV) if klen is None else klen.long()
    qi = torch.arange(tq, device=DEV).view(1, tq, 1)
    kj = torch.arange(tk, device=DEV).view(1, 1, tk)
    see &= (kj < nk.view(n, 1, 1)) & (qi < nq.view(n, 1, 1))
    if c["causal"]:
        see &= kj - nk.view(n, 1, 1) <= qi - nq.view(n, 1, 1)
    if c["diag"]:
        see &= kj != qi
    some = see.any(-1, keepdim=True)
    train = c["train"]
    q64, kv64 = q.to(D).requires_grad_(train), kv.to(D).requires_grad_(train)
    lam64, gain64 = lam.to(D).requires_grad_(train), gain.to(D).requires_grad_(train)
    leaves = [q64] + ([kv64] if c["cross"] else []) + [lam64, gain64]
    off = 0 if c["cross"] else qw
    src = kv64 if c["cross"] else q64
    y = torch.empty(n, tq, qw, dtype=D, device=DEV)
    grads = [torch.zeros_like(t) for t in leaves]
    with torch.set_grad_enabled(train):
        for j in range(h):
            g = j // (h // hkv)
            l4 = lam64[j if lam.shape[0] == h else 0]
            lj = torch.exp(l4[0] @ l4[1]) - torch.exp(l4[2] @ l4[3]) + LAM0
            maps = []
            for m in range(2):
                qa, ka = (2 * j + m) * dh, off + (2 * g + m) * dh
                sc = torch.bmm(q64[..., qa:qa + dh].contiguous(),
                               src[..., ka:ka + dh].transpose(1, 2).contiguous()) / dh ** 0.5
                maps.append(torch.softmax(sc.masked_fill(~see, -1e300), -1) * some)
            va = off + kw // 2 + g * 2 * dh
            o = torch.bmm(maps[0] - lj * maps[1], src[..., va:va + 2 * dh].contiguous())
            yj = (1.0 - LAM0) * gain64 * o / torch.sqrt((o ** 2).mean(-1, keepdim=True) + EPS)
            cols = slice(j * 2 * dh, (j + 1) * 2 * dh)
            y[..., cols] = yj.detach()
            if train:
                got = torch.autograd.grad(yj, leaves, dy[..., cols].to(D))
                grads = [a + b for a, b in zip(grads, got)]
    out = dict(y=y)
    if train:
        out.update(dq=grads[0], dlam=grads[-2], dgain=grads[-1])
        if c["cross"]:
            out["dkv"] = grads[1]
    return out


def _exact_linear(c, seed):
    x, w, b, res, dy = _linear_inputs(c, seed)
    x, w, b = (t.to(D).requires_grad_(c["train"]) for t in (x, w, b))
    F = torch.nn.functional
    z = F.linear(x, w, b)
    y = {"relu": F.relu, "silu": F.silu, "gelu": F.gelu,
         "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}[c["act"]](z)
    out = dict(y=(y if res is None else y + res.to(D)).detach())
    if c["train"]:
        out["dx"], out["dw"], out["db"] = torch.autograd.grad(y, (x, w, b), dy.to(D))
    return out


_EXACT = dict(rotary=_exact_rotary, diff=_exact_diff, linear=_exact_linear)
