"""GPU: linear attention with decay refuses results over what it still reads,
before anything is launched, and takes columns of one buffer that are apart."""
import pytest
import torch

pytestmark = pytest.mark.gpu

N, T, H, DK, DV = 2, 10, 4, 16, 16  # queries, keys, values and y are of one size
SIZE = dict(q=N * T * H * DK, k=N * T * H * DK, v=N * T * H * DV, dy=N * T * H * DV, rate=H, lens=N,
            state=N * H * DK * DV, dstate_out=N * H * DK * DV, dq=N * T * H * DK, dk=N * T * H * DK,
            dv=N * T * H * DV, drate=H, dstate=N * H * DK * DV)


def buffers(**at):
    """Every operand in a piece of its own of one buffer, or, where `at` names
    another one, from the given float of that on."""
    off, end = {}, 4096
    for k, m in SIZE.items():
        off[k], end = end, end + m + 8
    for k, (other, shift) in at.items():
        off[k] = off[other] + shift
    buf = torch.zeros(end + 4096, device="cuda")
    return buf, {k: buf[off[k]:off[k] + m] for k, m in SIZE.items()}


def backward(rnn, b):
    core, w = rnn.DecayCore(H, DK, DV), H * DK
    core.backward(N, T, b["q"], w, 0, b["k"], w, 0, 0, b["rate"], b["dy"], b["dq"], b["dk"],
                  b["drate"], lens=b["lens"].view(torch.int32), state=b["state"],
                  dstate_out=b["dstate_out"], dstate=b["dstate"], set_dq=True, set_dkv=True,
                  v=b["v"], vstride=w, dv=b["dv"])


READ = ("q", "k", "v", "dy", "rate", "lens", "state", "dstate_out")
WRITTEN = ("dq", "dk", "dv", "drate", "dstate")


@pytest.mark.parametrize("out,other", [(o, i) for o in WRITTEN for i in READ + WRITTEN if i != o])
def test_gradients_over_operands(rnn, out, other):
    last = SIZE[other] - 1
    for shift in {0, last, -(SIZE[out] - 1)}:  # all of it, its last float, its first
        buf, b = buffers(**{out: (other, shift)})
        with pytest.raises(rnn.RnnError):
            backward(rnn, b)
        torch.cuda.synchronize()
        assert (buf == 0).all()


@pytest.mark.parametrize("out,other", [(o, i) for o in ("y", "state_out") for i in
                                       ("q", "k", "v", "rate", "lens", "state")] + [("y", "state_out")])
def test_results_over_operands(rnn, out, other):
    names = dict(y="dy", state_out="dstate")
    buf, b = buffers(**{names[out]: (names.get(other, other), 1)})
    core, w = rnn.DecayCore(H, DK, DV), H * DK
    with pytest.raises(rnn.RnnError):
        core.forward(N, T, b["q"], w, 0, b["k"], w, 0, 0, b["rate"], lens=b["lens"].view(torch.int32),
                     state=b["state"], state_out=b["dstate"], y=b["dy"], v=b["v"], vstride=w)
    torch.cuda.synchronize()
    assert (buf == 0).all()


def test_columns_of_one_buffer(rnn):
    """Queries, keys and values and their gradients side by side in one buffer, as
    from buffers of their own; a column less apart is refused."""
    g, w = torch.Generator().manual_seed(2), H * DK
    x = torch.randn(N, T, 6 * w + 2, generator=g).cuda()
    rate, dy = torch.randn(H, generator=g).cuda(), torch.randn(N, T, w, generator=g).cuda()
    core = rnn.DecayCore(H, DK, DV)
    s = 6 * w + 2
    parts = [x[..., k * w:(k + 1) * w].contiguous() for k in range(3)]
    want = [torch.empty_like(p) for p in parts]
    core.backward(N, T, parts[0], w, 0, parts[1], w, 0, 0, rate, dy, want[0], want[1], set_dq=True,
                  set_dkv=True, v=parts[2], vstride=w, dv=want[2])

    def call(buf, at):
        q, k, v, dq, dk, dv = (buf.view(-1)[m:] for m in at)
        core.backward(N, T, q, s, 0, k, s, 0, 0, rate, dy, dq, dk, set_dq=True, set_dkv=True, v=v,
                      vstride=s, dv=dv)

    at = [0, w, 2 * w, 3 * w, 4 * w + 1, 5 * w + 2]
    call(x, at)
    for k, ref in zip(at[3:], want):
        assert torch.equal(x[..., k:k + w], ref)
    for i, shift in ((3, -1), (4, 2), (4, -2), (5, -2)):
        bad, before = list(at), x.clone()
        bad[i] += shift
        with pytest.raises(rnn.RnnError):
            call(x, bad)
        torch.cuda.synchronize()
        assert torch.equal(x, before)
