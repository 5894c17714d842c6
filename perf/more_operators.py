"""The operators of a linear-attention block, as cases that can be timed.

Three operators, each in its plain form (elementary torch operations in 32
bits) and, with ``own`` set, through the package's public entry points:

* ``normrot``: the norm of each query and key head and its rotary position in
  one pass, forward and backward (``R.NormRotary``);
* ``decay``: linear attention with a decay for each head, over whole sequences
  with or without a state carried in and out, forward and backward, and over
  single tokens (``R.DecayCore``);
* ``gate``: the norm of each output head times SiLU of a gate, forward and
  backward (``R.HeadGate``).

All data is float32, which is the only type that the framework computes in.
"""
import math

import torch

own = False

DEV = "cuda"
D = torch.float64
BASE = {1: 10000.0, 2: 100.0, 3: 10000.0}  # frequencies' base by the number of axes
EPS = 1e-6
CHUNK = 64  # tokens of a chunk of the plain form


def listed():
    return [
        # One image's queries and keys, 8 x 8 tokens: the least a serving program asks for.
        _rot("normrot_eval_one", 1, (8, 8), 4, 4, 64),
        # Clips of 8 x 14 x 14 tokens whose frames lie at given, fractional positions.
        _rot("normrot_video_train", 16, (8, 14, 14), 12, 12, 64, explicit=True, train=True),
        # An odd grid, key heads shared by query heads, channels of a head that do not turn.
        _rot("normrot_partial_train", 37, (13, 17), 6, 2, 52, pairs=20, interleaved=True,
             train=True),
        # One more frame's token for one stream: four heads' states read and written.
        _dec("decay_step_one", 1, 1, 4, 4, 64, 64, state=True),
        # The same for the streams of a full server.
        _dec("decay_step_batch", 64, 1, 8, 8, 64, 128, state=True),
        # The stage-3 heads at the training batch, 8 x 8 tokens read from both ends.
        _dec("decay_image_train", 128, 64, 4, 4, 64, 64, reverse=2, train=True),
        # Padded clips of up to 8 x 14 x 14 tokens in time order.
        _dec("decay_video_train", 8, 1568, 8, 8, 64, 64, ragged=True, train=True),
        # Sizes that no tile divides, key heads shared by three query heads, states passed on.
        _dec("decay_odd_train", 5, 577, 6, 2, 44, 72, ragged=True, state=True, reverse=2,
             train=True),
        # One long clip, its state kept for the tokens that follow.
        _dec("decay_prompt_long", 1, 16384, 8, 8, 64, 128, state=True),
        # The outputs of one image.
        _gate("gate_eval_one", 64, 4, 64),
        # The outputs of the clips, forward and backward.
        _gate("gate_video_train", 25088, 8, 64, train=True),
        # A partial batch of heads that no 16-byte load divides.
        _gate("gate_odd_train", 1813, 5, 77, train=True),
    ]


def _rot(name, n, grid, hq, hk, dh, pairs=None, explicit=False, interleaved=False, train=False):
    g = (1,) * (3 - len(grid)) + tuple(grid)
    return dict(name=name, kind="normrot", n=n, axes=len(grid), g0=g[0], g1=g[1], g2=g[2], hq=hq,
                hk=hk, dh=dh, pairs=dh // 2 if pairs is None else pairs, explicit=explicit,
                interleaved=interleaved, train=train)


def _dec(name, n, t, h, hkv, dk, dv, reverse=0, ragged=False, state=False, train=False):
    return dict(name=name, kind="decay", n=n, t=t, h=h, hkv=hkv, dk=dk, dv=dv, reverse=reverse,
                ragged=ragged, state=state, train=train)


def _gate(name, rows, h, d, train=False):
    return dict(name=name, kind="gate", rows=rows, h=h, d=d, train=train)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case, its batch or length halved until it is no larger than a listed one."""
    c = _draw(rng)
    c.pop("name")
    if c["kind"] == "decay":
        while work(c)["flops"] > 4e9 or work(c)["bytes"] > 1.2e8 or \
                (c["train"] and c["n"] * c["t"] ** 2 > 2e7):
            if c["n"] > 1:
                c["n"] = (c["n"] + 1) // 2
            else:
                c["t"] = (c["t"] + 1) // 2
    return c


def _draw(rng):
    kind = rng.choice(["normrot", "normrot", "decay", "decay", "decay", "decay", "gate"])
    if kind == "normrot":
        axes = rng.randint(1, 3)
        grid = [(_log(rng, 16, 2048),), (rng.randint(4, 24), rng.randint(4, 24)),
                (rng.randint(2, 8), rng.randint(4, 14), rng.randint(4, 14))][axes - 1]
        hk = rng.randint(1, 8)
        dh = rng.choice([2 * rng.randint(8, 64), 32, 64, 128])
        return _rot("", _log(rng, 1, 12), grid, hk * rng.randint(1, 2), hk, dh,
                    pairs=rng.choice([dh // 2, dh // 2, rng.randint(axes, dh // 2)]),
                    explicit=rng.random() < 0.4, interleaved=rng.random() < 0.5,
                    train=rng.random() < 0.7)
    if kind == "gate":
        return _gate("", _log(rng, 16, 16384), rng.randint(1, 12), rng.choice(
            [rng.randint(16, 128), 32, 64, 128]), train=rng.random() < 0.7)
    hkv = rng.choice([1, 2, 4, 4])
    h = hkv * rng.choice([1, 1, 1, 2, 3])
    size = lambda: rng.choice([rng.randint(16, 128), 32, 64, 64, 128])
    dk = size()
    dv = rng.choice([dk, size()])
    flags = dict(reverse=rng.choice([0, 0, h // 2, h]), ragged=rng.random() < 0.4,
                 state=rng.random() < 0.4)
    if rng.random() < 0.25:  # single tokens, or a few at once
        return _dec("", _log(rng, 1, 128), rng.choice([1, 1, rng.randint(2, 8)]), h, hkv, dk, dv,
                    state=True)
    train = rng.random() < 0.6
    return _dec("", _log(rng, 1, 128), _log(rng, 9, 4096 if train else 16384), h, hkv, dk, dv,
                train=train, **flags)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEV) * std


def _grid(c):
    return (c["g0"], c["g1"], c["g2"])[3 - c["axes"]:]


def _shares(c):
    """Pairs of each axis: an even share, what is left over to the first ones."""
    r, a = c["pairs"], c["axes"]
    return [r // a + (i < r % a) for i in range(a)]


def _rot_inputs(c, seed):
    """A fused buffer whose rows begin with the queries' and keys' heads, the
    gains of both, a gradient, and explicit positions where the case has them."""
    g = _gen(seed)
    n, t, w = c["n"], c["g0"] * c["g1"] * c["g2"], (c["hq"] + c["hk"]) * c["dh"]
    x, dy = _normal(g, (n, t, w + w // 2)), _normal(g, (n, t, w), 1e-3)
    gain = 1.0 + _normal(g, (2, c["dh"]), 0.1)
    pos = None
    if c["explicit"]:
        # each clip starts at a frame of its own and is sampled at its own rate
        axes = [torch.arange(s, device=DEV, dtype=torch.float32) for s in _grid(c)]
        co = torch.stack([m.reshape(-1) for m in torch.meshgrid(*axes, indexing="ij")], -1)
        rate = torch.rand((n, 1, c["axes"]), generator=g, device=DEV) + 0.5
        start = torch.randint(0, 20000, (n, 1, 1), generator=g, device=DEV).float()
        first = torch.tensor([1.0] + [0.0] * (c["axes"] - 1), device=DEV)
        pos = (co * rate + start * first).reshape(n * t, c["axes"]).contiguous()
    return x, dy, gain, pos


def _widths(c):
    """Floats of the queries, of the keys and of the values in a row."""
    return c["h"] * c["dk"], c["hkv"] * c["dk"], c["hkv"] * c["dv"]


def _dec_inputs(c, seed):
    """The fused buffer of normed queries and keys and of values, each head's
    rate of decay (memories of two tokens to some thousands), lengths of a
    padded batch, the state carried in, and the gradients of what comes out."""
    g = _gen(seed)
    n, t, h = c["n"], c["t"], c["h"]
    x = _normal(g, (n, t, sum(_widths(c))))
    rate = math.log(2.0 ** -12) + torch.rand(h, generator=g, device=DEV) * math.log(2.0 ** 11)
    lens = None
    if c["ragged"]:
        lens = torch.randint((t + 1) // 2, t + 1, (n,), generator=g, device=DEV,
                             dtype=torch.int32)
    shape = (n, h, c["dk"], c["dv"])
    state = _normal(g, shape) if c["state"] else None
    dy = _normal(g, (n, t, h * c["dv"]), 1e-3) if c["train"] else None
    dstate = _normal(g, shape, 1e-3) if c["train"] and c["state"] else None
    return x, rate, lens, state, dy, dstate


def _gate_inputs(c, seed):
    """The heads' outputs, the fused buffer with the gate in its last part,
    the gain of each channel and a gradient."""
    g = _gen(seed)
    r, w = c["rows"], c["h"] * c["d"]
    return (_normal(g, (r, w), 3.0), _normal(g, (r, 4 * w)), 1.0 + _normal(g, w, 0.1),
            _normal(g, (r, w), 1e-3))


def prepare(case, seed):
    c = case
    s = {"c": c}
    if c["kind"] == "normrot":
        s["x"], s["dy"], s["gain"], s["pos"] = _rot_inputs(c, seed)
    elif c["kind"] == "decay":
        s["x"], s["rate"], s["lens"], s["state"], s["dy"], s["dstate"] = _dec_inputs(c, seed)
    else:
        s["x"], s["z"], s["gain"], s["dy"] = _gate_inputs(c, seed)
    if own:
        import rustnn_amd as R
        if c["kind"] == "normrot":
            s["op"] = R.NormRotary(c["hq"], c["hk"], c["dh"], _grid(c), BASE[c["axes"]], _shares(c),
                                   c["interleaved"], eps=EPS)
        elif c["kind"] == "decay":
            s["op"] = R.DecayCore(c["h"], c["dk"], c["dv"], c["hkv"], reverse=c["reverse"])
        else:
            s["op"] = R.HeadGate(c["h"], c["d"], eps=EPS)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["c"]
    return (_OWN if own else _PLAIN)[c["kind"]](c, s)


def _own_rot(c, s):
    n, w = c["n"], (c["hq"] + c["hk"]) * c["dh"]
    x, xw, op = s["x"], w + w // 2, s["op"]
    out = dict(y=op.forward(n, x, xw, 0, s["gain"], pos=s["pos"]))
    if c["train"]:
        dgain = torch.zeros_like(s["gain"])
        out["dx"] = op.backward(n, x, xw, 0, s["gain"], s["dy"], w, 0, dgain, pos=s["pos"])
        out["dgain"] = dgain
    return out


def _own_dec(c, s):
    qw, kw, vw = _widths(c)
    x, w, n, t, core = s["x"], qw + kw + vw, c["n"], c["t"], s["op"]
    geo = (x, w, 0, x, w, qw, qw + kw)
    y, state = core.forward(n, t, *geo, s["rate"], lens=s["lens"], state=s["state"],
                            keep_state=c["state"])
    out = dict(y=y)
    if c["state"]:
        out["state"] = state
    if c["train"]:
        dx, drate = torch.empty_like(x), torch.zeros_like(s["rate"])
        ds = torch.empty_like(s["state"]) if c["state"] else None
        core.backward(n, t, *geo, s["rate"], s["dy"], dx, dx, drate, lens=s["lens"],
                      state=s["state"], dstate_out=s["dstate"], dstate=ds, set_dq=True,
                      set_dkv=True)
        out.update(dx=dx, drate=drate)
        if c["state"]:
            out["dstate"] = ds
    return out


def _own_gate(c, s):
    w, op = c["h"] * c["d"], s["op"]
    out = dict(y=op.forward(c["rows"], s["x"], s["z"], 4 * w, 3 * w, s["gain"]))
    if c["train"]:
        dz, dgain = torch.empty_like(s["x"]), torch.zeros_like(s["gain"])
        out["dx"] = op.backward(c["rows"], s["x"], s["z"], 4 * w, 3 * w, s["gain"], s["dy"], dz, w,
                                0, dgain)
        out.update(dz=dz, dgain=dgain)
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
    parts = [p[..., a:a + 1] * torch.pow(base, -torch.arange(k, device=DEV, dtype=D) / max(k, 1))
             for a, k in enumerate(_shares(c))]
    return torch.cat(parts, -1)


def _turn(c, x, cos, sin):
    """x [n, t, heads, dh], its first 2 pairs channels turned."""
    r = c["pairs"]
    rest = x[..., 2 * r:]
    if c["interleaved"]:
        a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :r], x[..., r:2 * r]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, rest], -1) if rest.shape[-1] else y


def _plain_rot(c, s):
    n, h, dh = c["n"], c["hq"] + c["hk"], c["dh"]
    ang = _angles(c, s["pos"])
    cos, sin = torch.cos(ang).float()[:, :, None], torch.sin(ang).float()[:, :, None]
    x = s["x"][..., :h * dh].reshape(n, -1, h, dh)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    hat = x * r
    gain = torch.cat([s["gain"][0].expand(c["hq"], dh), s["gain"][1].expand(c["hk"], dh)])
    out = dict(y=_turn(c, hat * gain, cos, sin).flatten(-2))
    if c["train"]:
        du = _turn(c, s["dy"].view(n, -1, h, dh), cos, -sin)
        dg = (du * hat).sum((0, 1))
        out["dgain"] = torch.stack([dg[:c["hq"]].sum(0), dg[c["hq"]:].sum(0)])
        du = du * gain
        out["dx"] = (r * (du - hat * (du * hat).mean(-1, keepdim=True))).flatten(-2)
    return out


def _order(c, lens):
    """The row at each place of a head's scan, [n, h, t, 1], and which places
    lie behind the sequence's end (None: none).  The last ``reverse`` heads go
    from the last token to the first.  The map is its own inverse."""
    n, h, t = c["n"], c["h"], c["t"]
    place = torch.arange(t, device=DEV)
    end = torch.full((n, 1, 1), t, device=DEV) if lens is None else lens.long().view(n, 1, 1)
    back = (torch.arange(h, device=DEV) >= h - c["reverse"]).view(1, h, 1)
    rows = torch.where(back, (end - 1 - place).clamp(min=0), place).expand(n, h, t)
    pad = None if lens is None else (place >= end).expand(n, h, t)[..., None]
    return rows[..., None], pad


def _scan(c, x, d, order, whole):
    """x [n, t, heads * d] as [n, h, whole, d] in the scan's order, zeros behind the end."""
    rows, pad = order
    x = x.reshape(c["n"], c["t"], -1, d).permute(0, 2, 1, 3)
    if x.shape[1] != c["h"]:
        x = x.repeat_interleave(c["h"] // x.shape[1], 1)
    x = torch.gather(x, 2, rows.expand(-1, -1, -1, d))
    if pad is not None:
        x = x.masked_fill(pad, 0.0)
    return torch.nn.functional.pad(x, (0, 0, 0, whole - c["t"]))


def _rows(c, y, order, heads):
    """The way back, [n, t, heads * d], shared heads' parts summed."""
    rows, pad = order
    y = torch.gather(y[:, :, :c["t"]], 2, rows.expand(-1, -1, -1, y.shape[-1]))
    if pad is not None:
        y = y.masked_fill(pad, 0.0)
    if heads != c["h"]:
        y = y.view(c["n"], heads, -1, c["t"], y.shape[-1]).sum(2)
    return y.permute(0, 2, 1, 3).flatten(-2)


def _tables(g, size, nc):
    """Powers of the decays exp(g) [h], in 64 bits and rounded once: between a
    chunk's places, of its rows and keys, between chunks; and the distances."""
    i = torch.arange(size, device=DEV, dtype=D)
    k = torch.arange(nc, device=DEV, dtype=D)
    gg = g.view(-1, 1, 1)
    near = (i[:, None] - i[None, :]).expand(len(g), -1, -1)
    far = ((k[:, None] - k[None, :] - 1) * size).expand(len(g), -1, -1)
    power = lambda m: torch.where(m >= 0, torch.exp(gg * m.clamp(min=0)), torch.zeros_like(m))
    within, between = power(near), power(far)
    first, last = torch.exp(gg * (i + 1).view(1, -1, 1)), torch.exp(gg * (size - 1 - i).view(1, -1, 1))
    f = lambda v: v.float()
    return dict(within=f(within), between=f(between), first=f(first)[:, None], last=f(last)[:, None],
                within1=f(within * near), between1=f(between * far),
                first1=f(first * (i + 1).view(1, -1, 1))[:, None],
                last1=f(last * (size - 1 - i).view(1, -1, 1))[:, None])


def _lin(a, b, v, tab, size, slope=False):
    """sum_{j <= i} gamma^(i - j) (a_i . b_j) v_j over [n, h, whole, *], by chunks;
    slope: each term times i - j."""
    n, h, whole, _ = a.shape
    nc = whole // size
    a, b, v = (x.view(n, h, nc, size, -1) for x in (a, b, v))
    one = "1" if slope else ""
    y = ((a @ b.transpose(-1, -2)) * tab["within" + one][:, None]) @ v
    if nc > 1:
        loc = ((b * tab["last"]).transpose(-1, -2) @ v).view(n, h, nc, -1)
        st = (tab["between"] @ loc).view(n, h, nc, a.shape[-1], -1)
        if slope:
            loc1 = ((b * tab["last1"]).transpose(-1, -2) @ v).view(n, h, nc, -1)
            st1 = (tab["between1"] @ loc + tab["between"] @ loc1).view(st.shape)
            y = y + (a * tab["first"]) @ st1 + (a * tab["first1"]) @ st
        else:
            y = y + (a * tab["first"]) @ st
    return y.view(n, h, whole, -1)


def _plain_token(c, s):
    """One token a sequence, no gradients: the recurrence itself."""
    n, h, hkv, dk, dv = (c[k] for k in ("n", "h", "hkv", "dk", "dv"))
    qw, kw, _ = _widths(c)
    x = s["x"].view(n, -1)
    q, k = x[:, :qw].reshape(n, h, 1, dk), x[:, qw:qw + kw].reshape(n, hkv, dk, 1)
    kv = k * x[:, qw + kw:].reshape(n, hkv, 1, dv)
    if h != hkv:
        kv = kv.repeat_interleave(h // hkv, 1)
    st = torch.exp(-torch.exp(s["rate"])).view(1, h, 1, 1) * s["state"] + kv
    return dict(state=st, y=((q / math.sqrt(dk)) @ st).view(n, 1, -1))


def _plain_dec(c, s):
    n, t, h, hkv, dk, dv = (c[k] for k in ("n", "t", "h", "hkv", "dk", "dv"))
    if t == 1 and c["state"] and not c["train"] and s["lens"] is None:
        return _plain_token(c, s)
    scale = 1.0 / math.sqrt(dk)
    size = min(CHUNK, t)
    nc = -(-t // size)
    order = _order(c, s["lens"])
    qw, kw, _ = _widths(c)
    x = s["x"]
    q = _scan(c, x[..., :qw], dk, order, nc * size) * scale
    k = _scan(c, x[..., qw:qw + kw], dk, order, nc * size)
    v = _scan(c, x[..., qw + kw:], dv, order, nc * size)
    g = -torch.exp(s["rate"].to(D))
    tab = _tables(g, size, nc)
    y = _lin(q, k, v, tab, size)
    place = torch.arange(nc * size, device=DEV, dtype=D)
    end = (torch.full((n,), t, device=DEV) if s["lens"] is None else s["lens"]).to(D)
    left = end.view(n, 1, 1) - 1 - place
    gg = g.view(1, h, 1)
    first = torch.exp(gg * (place + 1)).float()[..., None]
    last = torch.where(left >= 0, torch.exp(gg * left.clamp(min=0)),
                       torch.zeros_like(left)).float()[..., None]
    all_ = torch.exp(gg * end.view(n, 1, 1)).float()[..., None]
    out = {}
    if c["state"]:
        y = y + (q * first) @ s["state"]
        out["state"] = all_ * s["state"] + (k * last).transpose(-1, -2) @ v
    out["y"] = _rows(c, y, order, h)
    if not c["train"]:
        return out
    do = _scan(c, s["dy"], dv, order, nc * size)
    fq, fk, fv, fo = (m.flip(2) for m in (q, k, v, do))
    dq = _lin(do, v, k, tab, size)
    dk_ = _lin(fv, fo, fq, tab, size).flip(2)
    dv_ = _lin(fk, fq, fo, tab, size).flip(2)
    dg = (do * _lin(q, k, v, tab, size, slope=True)).sum((0, 2, 3))
    if c["state"]:
        s0, ds = s["state"], s["dstate"]
        dq = dq + (do * first) @ s0.transpose(-1, -2)
        dk_ = dk_ + (v * last) @ ds.transpose(-1, -2)
        dv_ = dv_ + (k * last) @ ds
        out["dstate"] = (q * first).transpose(-1, -2) @ do + all_ * ds
        steps = (place + 1).float().view(1, 1, -1, 1)
        dg = dg + (do * ((q * (first * steps)) @ s0)).sum((0, 2, 3))
        dg = dg + (ds * (k * (last * left.float()[..., None])).transpose(-1, -2).matmul(v)
                   ).sum((0, 2, 3))
        dg = dg + (ds * s0 * (all_ * end.float().view(n, 1, 1, 1))).sum((0, 2, 3))
    out["dx"] = torch.cat([_rows(c, dq * scale, order, h), _rows(c, dk_, order, hkv),
                           _rows(c, dv_, order, hkv)], -1)
    out["drate"] = dg * g.float()
    return out


def _plain_gate(c, s):
    h, d = c["h"], c["d"]
    x = s["x"].view(-1, h, d)
    z = s["z"][:, 3 * h * d:].reshape(-1, h, d)
    gain = s["gain"].view(h, d)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    hat = x * r
    sig = 1.0 / (1.0 + torch.exp(-z))
    act = z * sig
    out = dict(y=(hat * gain * act).flatten(1))
    if c["train"]:
        dy = s["dy"].view(-1, h, d)
        out["dz"] = (dy * hat * gain * (sig * (1.0 + z * (1.0 - sig)))).flatten(1)
        du = dy * act
        out["dgain"] = (du * hat).sum(0).flatten()
        du = du * gain
        out["dx"] = (r * (du - hat * (du * hat).mean(-1, keepdim=True))).flatten(1)
    return out


_OWN = dict(normrot=_own_rot, decay=_own_dec, gate=_own_gate)
_PLAIN = dict(normrot=_plain_rot, decay=_plain_dec, gate=_plain_gate)


# ------------------------------------------------------------------ work
def work(case):
    c = case
    if c["kind"] == "normrot":
        rows = c["n"] * c["g0"] * c["g1"] * c["g2"]
        el = rows * (c["hq"] + c["hk"]) * c["dh"]
        # x read and y written; for the backward dy read and dx written besides
        return dict(bytes=4 * el * (4 if c["train"] else 2) +
                    (4 * rows * c["axes"] if c["explicit"] else 0),
                    flops=el * (19 if c["train"] else 7))
    if c["kind"] == "gate":
        el = c["rows"] * c["h"] * c["d"]
        return dict(bytes=4 * el * (6 if c["train"] else 3), flops=el * (25 if c["train"] else 9))
    n, h, dk, dv = c["n"], c["h"], c["dk"], c["dv"]
    rows = n * c["t"] * (0.75 if c["ragged"] else 1.0)  # lengths lie between a half and the whole
    ins, y, st = rows * sum(_widths(c)), rows * h * dv, n * h * dk * dv
    # inputs read and outputs written; for the backward dy read and dx written
    # besides.  A state is updated and read with two operations an element each;
    # the backward does so for the state and its gradient, which has two readers,
    # and once more with the tokens' distances for the rates
    el = ins + y + (2 * st if c["state"] else 0)
    if c["train"]:
        el += ins + y + (2 * st if c["state"] else 0)
    return dict(bytes=4 * el, flops=(18 if c["train"] else 4) * rows * h * dk * dv)


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    return _EXACT[case["kind"]](case, seed)


def _norm64(x, gain):
    return x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + EPS) * gain


def _exact_rot(c, seed):
    """A rotation as the product of complex numbers; gradients by automatic
    differentiation."""
    x, dy, gain, pos = _rot_inputs(c, seed)
    n, t, h, dh, r = c["n"], x.shape[1], c["hq"] + c["hk"], c["dh"], c["pairs"]
    idx = torch.arange(t, device=DEV)
    coords = []
    for size in reversed(_grid(c)):
        coords.append((idx % size).to(D).expand(n, t))
        idx = idx // size
    coords = coords[::-1]
    if pos is not None:
        coords = [pos[:, a].to(D).view(n, t) for a in range(c["axes"])]
    ang = [coords[a] * BASE[c["axes"]] ** (-p / k) for a, k in enumerate(_shares(c))
           for p in range(k)]
    turn = torch.exp(1j * torch.stack(ang, -1))[:, :, None]
    u = x[..., :h * dh].reshape(n, t, h, dh).to(D).requires_grad_(c["train"])
    g64 = gain.to(D).requires_grad_(c["train"])
    which = torch.tensor([0] * c["hq"] + [1] * c["hk"], device=DEV)
    w = _norm64(u, g64[which])
    head = w[..., :2 * r].reshape(n, t, h, *((r, 2) if c["interleaved"] else (2, r)))
    if not c["interleaved"]:
        head = head.transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn)
    z = z if c["interleaved"] else z.transpose(-1, -2)
    y = torch.cat([z.reshape(n, t, h, 2 * r), w[..., 2 * r:]], -1)
    out = dict(y=y.detach().reshape(n, t, -1))
    if c["train"]:
        dx, out["dgain"] = torch.autograd.grad(y, (u, g64), dy.to(D).view(y.shape))
        out["dx"] = dx.reshape(n, t, -1)
    return out


def _exact_dec(c, seed):
    """The whole map of a head, gamma^(i - j) (q_i . k_j), its gradients by
    automatic differentiation; a few images at a time where sequences are long."""
    x, rate, lens, state, dy, dstate = _dec_inputs(c, seed)
    n, t, h = c["n"], c["t"], c["h"]
    if n * h * t * t > 2e10:
        return None
    step = max(1, int(2e8) // (t * t))
    cut = lambda v, b: None if v is None else v[b:b + step]
    parts = [_exact_images(c, rate, *(cut(v, b) for v in (x, lens, state, dy, dstate)))
             for b in range(0, n, step)]
    return {k: sum(p[k] for p in parts) if k == "drate" else torch.cat([p[k] for p in parts])
            for k in parts[0]}


def _exact_images(c, rate, x, lens, state, dy, dstate):
    t, h, dk, dv = (c[k] for k in ("t", "h", "dk", "dv"))
    n, train, grp = x.shape[0], c["train"], h // c["hkv"]
    qw, kw, vw = _widths(c)
    need = lambda v: None if v is None else v.to(D).requires_grad_(train)
    x64, r64, s64 = need(x), need(rate), need(state)
    leaves = [x64, r64] + ([s64] if c["state"] else [])
    grads = [torch.zeros_like(v) for v in leaves]
    end = torch.full((n,), t, device=DEV) if lens is None else lens.long()
    row = torch.arange(t, device=DEV)
    ok = row[None] < end[:, None]
    y = torch.zeros(n, t, h, dv, dtype=D, device=DEV)
    last = torch.zeros(n, h, dk, dv, dtype=D, device=DEV) if c["state"] else None
    with torch.set_grad_enabled(train):
        for j in range(h):
            m = j // grp
            qj = x64[..., j * dk:(j + 1) * dk] / dk ** 0.5
            kj = x64[..., qw + m * dk:qw + (m + 1) * dk]
            vj = x64[..., qw + kw + m * dv:qw + kw + (m + 1) * dv]
            g = -torch.exp(r64[j])
            back = j >= h - c["reverse"]
            # a row's place in the scan; the distance that a key lies before a query
            place = (end[:, None] - 1 - row[None] if back else row[None].expand(n, t)).to(D)
            dist = place[:, :, None] - place[:, None, :]
            see = (dist >= 0) & ok[:, :, None] & ok[:, None, :]
            p = torch.bmm(qj, kj.transpose(1, 2).contiguous())
            p = p * torch.exp(g * dist.clamp(min=0)) * see
            yj = torch.bmm(p, vj.contiguous())
            res, dres = [yj], [] if dy is None else [dy[..., j * dv:(j + 1) * dv].to(D)]
            if c["state"]:
                res[0] = yj = yj + torch.bmm(qj, s64[:, j]) * (
                    torch.exp(g * (place + 1).clamp(min=0)) * ok)[..., None]
                left = end[:, None].to(D) - 1 - place
                w = (torch.exp(g * left.clamp(min=0)) * ok)[..., None]
                sj = s64[:, j] * torch.exp(g * end.to(D)).view(n, 1, 1) + torch.bmm(
                    (kj * w).transpose(1, 2).contiguous(), vj.contiguous())
                last[:, j] = sj.detach()
                res.append(sj)
                dres += [] if dy is None else [dstate[:, j].to(D)]
            y[:, :, j] = yj.detach()
            if train:
                got = torch.autograd.grad(res, leaves, dres)
                grads = [a + b for a, b in zip(grads, got)]
    out = dict(y=y.view(n, t, h * dv))
    if c["state"]:
        out["state"] = last
    if train:
        out.update(dx=grads[0], drate=grads[1])
        if c["state"]:
            out["dstate"] = grads[2]
    return out


def _exact_gate(c, seed):
    x, z, gain, dy = _gate_inputs(c, seed)
    w, shape = c["h"] * c["d"], (-1, c["h"], c["d"])
    x, z, gain = (v.to(D).requires_grad_(c["train"]) for v in (x, z[:, 3 * w:], gain))
    y = _norm64(x.view(shape), gain.view(shape[1:])) * torch.nn.functional.silu(z).view(shape)
    y = y.reshape(-1, w)
    out = dict(y=y.detach())
    if c["train"]:
        out["dx"], out["dz"], out["dgain"] = torch.autograd.grad(y, (x, z, gain), dy.to(D))
    return out


_EXACT = dict(normrot=_exact_rot, decay=_exact_dec, gate=_exact_gate)
