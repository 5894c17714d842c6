"""GPU: batches whose grids pass 2^32 threads, which run in several launches: what
a batch gives an image is what the image gives alone, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu

N = 2 ** 24 + 3


@pytest.mark.parametrize("dh", [1, 4])  # four groups of rows a workgroup; joint backward
def test_attention(rnn, dh):
    w = 2 * dh
    core = rnn.DiffCore(1, dh, 1, 2)
    g = torch.Generator(device="cuda").manual_seed(dh)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    q, kv, dy = rnd(N, w), rnd(N, 2, 2 * w), rnd(N, w)
    lam, gain = rnd(1, 4, dh) * 0.1, 1 + 0.1 * rnd(w)

    def call(n, q, kv, dy):
        geo = (q, w, 0, kv, 2 * w, 0, w)
        y, saved = core.forward(n, *geo, lam, gain)
        dq, dkv = torch.full_like(q, float("nan")), torch.full_like(kv, float("nan"))
        dlam, dgain = torch.zeros_like(lam), torch.zeros_like(gain)
        core.backward(n, *geo, lam, gain, saved, dy, dq, dkv, dlam, dgain, set_dq=True, set_dkv=True)
        return y.view(n, w), dq, dkv, dlam, dgain

    got = call(N, q, kv, dy)
    assert all(bool(torch.isfinite(t).all()) for t in got)
    # the first images, both sides of every launch's end, the last ones
    ends = [i * 2 ** k for k in (22, 23) for i in range(1, 5) if i * 2 ** k < N]
    for i in [0] + [e - 2 for e in ends] + [N - 4]:
        s = slice(i, i + 4)
        one = call(4, q[s].contiguous(), kv[s].contiguous(), dy[s].contiguous())
        for nm, a, b in zip(("y", "dq", "dkv"), got, one):
            assert torch.equal(a[s], b), (nm, i)
    # the parameters' gradients: those of the batch in parts (the sums of 2^24 terms
    # are in 64 bits, each part is rounded once and added in 32)
    parts = torch.zeros_like(got[4])
    for s in torch.arange(N).split(2 ** 21):
        i, n = int(s[0]), len(s)
        parts += call(n, q[i:i + n], kv[i:i + n], dy[i:i + n])[4]
    assert (got[4] - parts).abs().max() <= 16 * 2.0 ** -24 * float(parts.abs().max() + N ** 0.5)


def test_rotary(rnn):
    """131 channels in place, so that a workgroup has one row."""
    n, c = N, 131
    rot = rnn.Rotary(1, c, n, pairs=(2,))
    x = torch.zeros(n, c, device="cuda")
    rows = [0, 1, 2 ** 23 - 1, 2 ** 23, 2 ** 23 + 1, 2 ** 24 - 1, 2 ** 24, n - 1]
    g = torch.Generator(device="cuda").manual_seed(1)
    vals = torch.randn(len(rows), c, generator=g, device="cuda")
    x[rows] = vals
    rot.forward(1, x, c, y=x)
    pos = torch.tensor(rows, dtype=torch.float32, device="cuda")[:, None]
    want = rot.forward(1, vals, c, pos=pos, t=len(rows))[0]
    assert torch.equal(x[rows], want)
    rest = x.clone()
    rest[rows] = 0
    assert not rest.any()
