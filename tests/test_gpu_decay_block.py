"""GPU: the operators of the linear-attention block as they are used together --
Block(attn="decay"): LayerNorm, fused q / k / v / gate Linear, head norms with
rotary positions, linear attention with decay in both directions, gated heads,
projection, depthwise branch, MLP -- against a statement of the block in 64 bits,
in a RustViT train step, and on other streams than the current one.

Tolerance of the block: 1e-5 relative Frobenius, as the other blocks'
(test_gpu_vit.py): each operator's own, of which none enlarges what comes in."""
import math

import pytest
import torch

from conftest import TOL, rel_frob
from decayref import D, DecayCase, decay_map, gate, norm_rotary
from diffref import act
from test_gpu_diff_streams import busy, rnn_context

pytestmark = pytest.mark.gpu


def block64(c, heads, th, x, ps, kind, sizes):
    """Block with DecaySelfAttn and Mlp from the parameters in their order; sizes
    receives what the rates' gradients are sums of."""
    n, t, _ = x.shape
    F, it, dh = torch.nn.functional, iter(ps), c // heads
    lin = lambda v, fout: v @ next(it).view(fout, -1).T + next(it)
    norm = lambda v: F.layer_norm(v, (c,), next(it), next(it), 1e-5)
    h = norm(x)
    ab = lin(h, 4 * c)
    wp, bp, rate, gain, ogain = (next(it) for _ in range(5))
    idx = torch.arange(t)
    pos = torch.stack([idx // th, idx % th], -1).repeat(n, 1)
    r = dh // 2
    qk = norm_rotary(ab[..., :2 * c].reshape(n * t, 2 * c), gain.view(2, dh), heads, heads, dh, pos,
                     (r // 2 + r % 2, r // 2), 100.0, False, 1e-6)
    q, k = (v.reshape(n, t, heads, dh) for v in qk.split(c, -1))
    v = ab[..., 2 * c:3 * c].reshape(n, t, heads, dh)
    s0 = torch.zeros(n, heads, dh, dh, dtype=D)
    o, _ = decay_map(q, k, v, rate, s0, 1 / math.sqrt(dh), heads // 2)
    sizes["o"] = o
    sizes["rate"] = lambda do: torch.exp(rate) * (decay_map(
        q.abs(), k.abs(), v.abs(), rate, s0, 1 / math.sqrt(dh), heads // 2, power=1)[0] *
        do.abs()).sum((0, 1, 3))
    u = gate(o.reshape(n * t, c), ab[..., 3 * c:].reshape(n * t, c), ogain, heads, dh, 1e-6)
    a = u.view(n, t, c) @ wp.view(c, c).T + bp
    w9, b9 = next(it).view(9, c), next(it)
    img = F.pad(h.view(n, th, th, c), (0, 0, 1, 1, 1, 1))
    dw = b9 + sum(w9[3 * i + j] * img[:, i:i + th, j:j + th] for i in range(3) for j in range(3))
    gamma, ls1 = next(it), next(it)
    y = x + ls1 * (a + gamma * dw.reshape(n, t, c))
    m = lin(act(kind, lin(norm(y), 4 * c)), c)
    return y + next(it) * m


@pytest.mark.parametrize("n,c,heads,th,kind", [(2, 32, 2, 4, "gelu"), (3, 48, 4, 5, "silu"),
                                               (2, 64, 1, 6, "gelu")])
def test_block(rnn, n, c, heads, th, kind):
    from rustnn_amd import vit
    blk = vit.Block(c, heads, th, th, None, 4, 0.0, 2, 0.5, 7, attn="decay", mlp=kind)
    ps = []
    blk.for_each_param(ps.append)
    g = torch.Generator().manual_seed(1)
    for p in ps:  # away from 0 and 1, as training leaves them
        p.v += (torch.randn(p.v.shape, generator=g) * 0.1).cuda()
    x, dz = (torch.randn(n, th * th, c, generator=g) for _ in range(2))
    xl = x.to(D).requires_grad_(True)
    leaves = [p.v.cpu().to(D).requires_grad_(True) for p in ps]
    sizes = {}
    want = block64(c, heads, th, xl, leaves, kind, sizes)
    do, *grads = torch.autograd.grad(want, [sizes["o"], xl] + leaves, dz.to(D))
    y = blk.forward(x.cuda(), None, True, 0)
    assert rel_frob(y.cpu(), want.detach()) < TOL
    assert torch.equal(blk.forward(x.cuda(), None, False, 0), y)
    dx = blk.backward(dz.cuda())
    assert rel_frob(dx.cpu(), grads[0]) < TOL
    for i, (p, ref) in enumerate(zip(ps, grads[1:])):
        err = (p.g.cpu().to(D) - ref).norm()
        # the rates': sums of terms of both signs, which their error goes by
        size = ref.norm() if p is not blk.attn.rate else sizes["rate"](do).detach().norm()
        assert float(err) < TOL * float(size), (i, float(err), float(size))


CFG = dict(width=4, cmid=6, dim=16, heads=2, depth3=2, dim4=24, heads4=2, depth4=1, mem_at=(1,),
           droppath=0.0, img=16, attn="decay", mlp="gelu")


def make_step(seed=3):
    from rustnn_amd import vit
    parent = torch.tensor([0, 0, 1, 1, 2, 2], dtype=torch.int32).cuda()
    net = vit.RustViT(CFG, parent, 3, seed)
    return vit.ViTStep(net, parent, 3, dict(batch=8))


def batch():
    g = torch.Generator().manual_seed(5)
    x = torch.randn(8, 3, 16, 16, generator=g).cuda()
    labels = torch.randint(0, 6, (8,), generator=g, dtype=torch.int32)
    return x, labels.cuda(), (labels // 2).cuda()


def test_train_steps(rnn):
    """Three train steps of a network of such blocks: twice the same bits."""
    out = []
    for _ in range(2):
        step = make_step()
        losses = [float(step(*batch())[0]) for _ in range(3)]
        assert all(math.isfinite(v) for v in losses)
        out.append((losses, torch.cat([p.v for p in step.params])))
        assert {type(b.attn).__name__ for b in step.net.blocks3 + step.net.blocks4} == \
            {"DecaySelfAttn"}
    assert out[0][0] == out[1][0] and torch.equal(out[0][1], out[1][1])


def test_step_gradient_against_differences(rnn):
    """The loss along its own gradient: step 2^-7 of a unit vector over all
    parameters (third-order terms vanish); the loss' rounding, 1e-6 over twice
    the step, is below 1e-4 of a gradient of this size (above 1)."""
    step = make_step()
    x, labels, coarse = batch()
    step.forward_backward(x, labels, coarse)
    gs = [p.g.clone() for p in step.params]
    norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in gs))
    v0 = [p.v.clone() for p in step.params]
    h, vals = 2.0 ** -7, []
    for s in (1, -1):
        for p, v, g in zip(step.params, v0, gs):
            p.v.copy_(v + s * h * g / norm)
        vals.append(float(step.forward_backward(x, labels, coarse)[0]))
    assert norm > 1
    assert abs((vals[0] - vals[1]) / (2 * h) - norm) < 2e-2 * norm


def test_refusals_and_checkpoint(rnn, tmp_path):
    from rustnn_amd import ckpt, vit
    with pytest.raises(ValueError):
        vit.DecaySelfAttn(20, 4, (4, 4), 1)
    with pytest.raises(ValueError):
        vit.DecaySelfAttn(32, 2, (4, 4), 1, reverse=3)
    base = {k: v for k, v in CFG.items() if k not in ("attn", "mlp")}
    h = lambda cfg: ckpt.rustvit_config_hash(cfg, 6, 3, True, [0, 0, 1, 1, 2, 2])
    assert len({h(base), h(CFG), h(dict(CFG, attn="diff"))}) == 3
    a, b = make_step(3).net, make_step(4).net
    path = str(tmp_path / "net.ckpt")
    ckpt.save_rustvit(a, path)
    ckpt.load_rustvit(b, path)
    va, vb = [], []
    a.for_each_param(lambda p: va.append(p.v))
    b.for_each_param(lambda p: vb.append(p.v))
    assert all(torch.equal(x, y) for x, y in zip(va, vb))


# ------------------------------------------------------------------ streams
def norms(rnn):
    g = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g)
    data = dict(x=rnd(50 * 96, 128), dy=rnd(50 * 96, 128), gain=rnd(2, 32),
                pos=torch.rand(50 * 96, 2, generator=g) * 99)

    def calls(ctx, t):
        op = rnn.NormRotary(3, 1, 32, (8, 12), ctx=ctx)
        y = op.forward(50, t["x"], 128, 0, t["gain"], pos=t["pos"])
        dgain = torch.zeros_like(t["gain"])
        dx = op.backward(50, t["x"], 128, 0, t["gain"], t["dy"], 128, 0, dgain, pos=t["pos"])
        return dict(y=y, dx=dx, dgain=dgain)
    return data, calls


def attention(rnn, **kw):
    cs = DecayCase(**dict(dict(n=3, t=500, h=4, hkv=2, dk=40, dv=64, reverse=2, lens=[500, 7, 64],
                               seed=1), **kw))
    data = dict(kv=cs.kv, rate=cs.rate, lens=cs.lens, dy=cs.dy, state=cs.state, ds=cs.dstate)

    def calls(ctx, t):
        core = rnn.DecayCore(cs.h, cs.dk, cs.dv, cs.hkv, reverse=cs.reverse, ctx=ctx)
        geo = cs.geo(t["kv"], t["kv"])
        y, st = core.forward(cs.n, cs.t, *geo, t["rate"], lens=t["lens"], state=t["state"],
                             keep_state=True)
        out = dict(y=y, state=st, dx=torch.zeros_like(t["kv"]), drate=torch.zeros_like(t["rate"]),
                   dstate=torch.zeros_like(st))
        core.backward(cs.n, cs.t, *geo, t["rate"], t["dy"], out["dx"], out["dx"], out["drate"],
                      lens=t["lens"], state=t["state"], dstate_out=t["ds"], dstate=out["dstate"],
                      set_dq=True, set_dkv=True)
        return out
    return data, calls


def tokens(rnn):
    cs = DecayCase(64, 1, 8, 8, 64, 128, seed=2)
    data = dict(kv=cs.kv, rate=cs.rate, state=cs.state)

    def calls(ctx, t):
        core = rnn.DecayCore(8, 64, 128, ctx=ctx)
        st = t["state"].clone()
        for _ in range(3):
            y, _ = core.forward(64, 1, *cs.geo(t["kv"], t["kv"]), t["rate"], state=st, state_out=st)
        return dict(y=y, state=st)
    return data, calls


def gates(rnn):
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g)
    data = dict(x=rnd(4099, 190), z=rnd(4099, 190), gain=rnd(190), dy=rnd(4099, 190))

    def calls(ctx, t):
        op = rnn.HeadGate(5, 38, ctx=ctx)
        y = op.forward(4099, t["x"], t["z"], 190, 0, t["gain"])
        dz, dgain = torch.zeros_like(t["z"]), torch.zeros_like(t["gain"])
        dx = op.backward(4099, t["x"], t["z"], 190, 0, t["gain"], t["dy"], dz, 190, 0, dgain)
        return dict(y=y, dx=dx, dz=dz, dgain=dgain)
    return data, calls


def short(rnn):
    return attention(rnn, n=64, t=64, h=4, hkv=4, dk=64, lens=None)


ALL = [norms, attention, short, tokens, gates]


@pytest.mark.parametrize("make", ALL, ids=lambda f: f.__name__)
def test_inputs_and_results_in_order(rnn, make):
    """Inputs that the current stream is still to write, memory that it still
    uses, and inputs and results that it overwrites at once after the calls."""
    data, calls = make(rnn)
    data = {k: v for k, v in data.items() if v is not None}
    full = lambda t: {**{k: None for k in ("lens",)}, **t}
    dev = {k: v.cuda() for k, v in data.items()}
    with rnn_context(rnn, torch.cuda.current_stream()) as ctx:
        want = {k: v.clone() for k, v in calls(ctx, full(dev)).items()}
    torch.cuda.synchronize()
    for side in (torch.cuda.Stream(), torch.cuda.default_stream()):
        cur = torch.cuda.Stream()
        with rnn_context(rnn, side) as ctx:
            with torch.cuda.stream(cur):
                late = {k: torch.zeros_like(v) for k, v in dev.items()}
                torch.cuda.synchronize()
                held = torch.empty(1 << 26, device="cuda")
                busy()
                for k, v in dev.items():
                    late[k].copy_(v)
                held.fill_(7.0)  # memory that the calls' results may be given next
                del held
                out = calls(ctx, full(late))
                got = {k: v.clone() for k, v in out.items()}
                for v in [*late.values(), *out.values()]:
                    v.zero_()
            torch.cuda.synchronize()
        for k, v in want.items():
            assert torch.equal(got[k], v), k


@pytest.mark.parametrize("make", ALL, ids=lambda f: f.__name__)
def test_two_graphs_captured_and_replayed(rnn, make):
    """Two graphs of the same calls, captured one after the other from a context
    on another stream and replayed in turn with eager calls between them."""
    data, calls = make(rnn)
    data = {k: v for k, v in data.items() if v is not None}
    full = lambda t: {**{k: None for k in ("lens",)}, **t}
    dev = [{k: v.cuda() for k, v in data.items()} for _ in range(2)]
    for k in ("kv", "x"):
        if k in dev[1]:
            dev[1][k] *= 0.5
    with rnn_context(rnn, torch.cuda.Stream()) as ctx:
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            want = [{k: v.clone() for k, v in calls(ctx, full(t)).items()} for t in dev]
        torch.cuda.synchronize()
        graphs, outs = [], []
        for t in dev:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                outs.append(calls(ctx, full(t)))
            graphs.append(graph)
        for _ in range(3):
            for graph, out, ref in zip(graphs, outs, want):
                with torch.cuda.stream(st):
                    for v in out.values():
                        v.fill_(0.5)
                    graph.replay()
                    got = {k: v.clone() for k, v in out.items()}
                torch.cuda.synchronize()
                for k, v in ref.items():
                    assert torch.equal(got[k], v), k
                with torch.cuda.stream(st):
                    calls(ctx, full(dev[0]))
                torch.cuda.synchronize()
