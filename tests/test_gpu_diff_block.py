"""GPU: the operators of the differential block as they are used together --
Block(attn="diff", mlp=...): LayerNorm, fused QKV Linear, rotary positions in
place, differential attention, projection, depthwise branch, cross-attention,
MLP with its activation and residual -- against a statement of the block in 64
bits, and in a RustViT train step.

Tolerance: 1e-5 relative Frobenius, as the other blocks' (test_gpu_vit.py): each
operator's own, of which none enlarges what comes in."""
import math

import pytest
import torch

from conftest import TOL, rel_frob
from diffref import D, act, diff_attn, rotary

pytestmark = pytest.mark.gpu


def block64(c, heads, th, x, mem, ps, lam0, kind, parts):
    """Block with DiffSelfAttn and Mlp from the parameters in their order; parts
    receives the attention's O and P_2 V."""
    n, t, _ = x.shape
    F, it = torch.nn.functional, iter(ps)
    lin = lambda v, fout: v @ next(it).view(fout, -1).T + next(it)
    norm = lambda v: F.layer_norm(v, (c,), next(it), next(it), 1e-5)
    h = norm(x)
    qkv = lin(h, 3 * c)
    wp, bp, lam, gain = next(it), next(it), next(it), next(it)
    dh = c // (2 * heads)
    idx = torch.arange(t)
    pos = torch.stack([idx // th, idx % th], -1).repeat(n, 1)
    r = dh // 2
    pairs = (r // 2 + r % 2, r // 2)
    # the rotation's coefficients by the statement, applied so that gradients flow
    eye = torch.eye(4 * heads * dh, dtype=D)
    basis = torch.stack([rotary(eye, 4 * heads, dh, pos[i:i + 1].expand(4 * heads * dh, 2), pairs,
                                100.0, False) for i in range(t)])
    qk = torch.einsum("ntc,tcd->ntd", qkv[..., :2 * c], basis)
    q, k = (v.reshape(n, t, heads, 2, dh) for v in qk.split(c, -1))
    see = torch.ones(n, t, t, dtype=torch.bool)
    a = diff_attn(q, k, qkv[..., 2 * c:].reshape(n, t, heads, 2 * dh), lam.view(1, 4, dh), gain,
                  see, 1 / math.sqrt(dh), lam0, 1e-5, parts)
    a = a @ wp.view(c, c).T + bp
    w9, b9 = next(it).view(9, c), next(it)
    img = F.pad(h.view(n, th, th, c), (0, 0, 1, 1, 1, 1))
    dw = b9 + sum(w9[3 * i + j] * img[:, i:i + th, j:j + th] for i in range(3) for j in range(3))
    gamma, ls1 = next(it), next(it)
    y = x + ls1 * (a + gamma * dw.reshape(n, t, c))
    h2 = norm(y)
    u = act(kind, lin(h2, 4 * c))
    m = lin(u, c)
    return y + next(it) * m


@pytest.mark.parametrize("kind", ["gelu", "silu"])
@pytest.mark.parametrize("n,c,heads,th", [(2, 32, 2, 4), (3, 48, 2, 5), (2, 64, 1, 6)])
def test_block(rnn, n, c, heads, th, kind):
    from rustnn_amd import vit
    blk = vit.Block(c, heads, th, th, None, 4, 0.0, 2, 0.5, 7, attn="diff", mlp=kind)
    ps = []
    blk.for_each_param(ps.append)
    g = torch.Generator().manual_seed(1)
    for p in ps:  # away from 0 and 1, as training leaves them
        p.v += (torch.randn(p.v.shape, generator=g) * 0.1).cuda()
    x = torch.randn(n, th * th, c, generator=g)
    dz = torch.randn(n, th * th, c, generator=g)
    xl = x.to(D).requires_grad_(True)
    leaves = [p.v.cpu().to(D).requires_grad_(True) for p in ps]
    parts = {}
    want = block64(c, heads, th, xl, None, leaves, blk.attn.core.lam_init, kind, parts)
    do, *grads = torch.autograd.grad(want, [parts["o"], xl] + leaves, dz.to(D))
    lam = blk.attn.lam.v.cpu().to(D).view(4, -1)
    lam_size = float((do.norm(dim=-1) * parts["o2"].norm(dim=-1)).norm().detach() * lam.norm()
                     * torch.exp((lam[::2] * lam[1::2]).sum(-1)).max())
    y = blk.forward(x.cuda(), None, True, 0)
    assert rel_frob(y.cpu(), want.detach()) < TOL
    assert torch.equal(blk.forward(x.cuda(), None, False, 0), y)
    dx = blk.backward(dz.cuda())
    assert rel_frob(dx.cpu(), grads[0]) < TOL
    for i, (p, ref) in enumerate(zip(ps, grads[1:])):
        err = float((p.g.cpu().to(D) - ref).norm())
        # lambda's vectors: a sum of terms dO . (P_2 V) that the norm makes small
        # beside |dO| |P_2 V|, which its error goes by (test_gpu_diffattn.py)
        size = float(ref.norm()) if p is not blk.attn.lam else lam_size
        assert err < TOL * size, (i, err, size)


CFG = dict(width=4, cmid=6, dim=16, heads=2, depth3=2, dim4=24, heads4=2, depth4=1, mem_at=(1,),
           droppath=0.0, img=16, attn="diff", mlp="gelu")


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
        kinds = {type(b.attn).__name__ + type(b.mlp).__name__
                 for b in step.net.blocks3 + step.net.blocks4}
        assert kinds == {"DiffSelfAttnMlp"}
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


def test_refusals_and_checkpoint_hash(rnn):
    from rustnn_amd import ckpt, vit
    with pytest.raises(ValueError):
        vit.DiffSelfAttn(20, 2, (4, 4), 1)
    with pytest.raises(ValueError):
        vit.Block(32, 2, 4, 4, None, 1, 0.0, 1, 0.5, attn="softmax")
    with pytest.raises(ValueError):
        vit.Block(32, 2, 4, 4, None, 1, 0.0, 1, 0.5, mlp="tanh")
    base = {k: v for k, v in CFG.items() if k not in ("attn", "mlp")}
    h = lambda cfg: ckpt.rustvit_config_hash(cfg, 6, 3, True, [0, 0, 1, 1, 2, 2])
    assert h(base) == h(dict(base, attn="lsa", mlp="swiglu")) != h(CFG)
    assert h(CFG) != h(dict(CFG, mlp="silu"))
