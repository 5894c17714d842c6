"""GPU: head norms with rotary positions and gated heads refuse results over
what they still read, before anything is launched, and take columns of one
buffer that are apart."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS, W = 24, 64  # two heads of 32 channels


def pieces(sizes, **at):
    """Every operand in a piece of its own of one buffer, or from the given float
    of another one on."""
    off, end = {}, 4096
    for k, m in sizes.items():
        off[k], end = end, end + m + 8
    for k, (other, shift) in at.items():
        off[k] = off[other] + shift
    buf = torch.zeros(end + 4096, device="cuda")
    return buf, {k: buf[off[k]:off[k] + m] for k, m in sizes.items()}


def refused(rnn, buf, call):
    with pytest.raises(rnn.RnnError):
        call()
    torch.cuda.synchronize()
    assert (buf == 0).all()


NORM = dict(x=ROWS * W, gain=64, pos=ROWS, y=ROWS * W, dy=ROWS * W, dgain=64)


@pytest.mark.parametrize("other", ["x", "gain", "pos"])
def test_norm_rotary_forward(rnn, other):
    op = rnn.NormRotary(1, 1, 32, (ROWS,))
    for shift in {1, NORM[other] - 1, -(ROWS * W - 1)}:
        buf, b = pieces(NORM, y=(other, shift))
        refused(rnn, buf, lambda: op.forward(1, b["x"], W, 0, b["gain"], pos=b["pos"], y=b["y"],
                                             ystride=W))


@pytest.mark.parametrize("other", ["x", "gain", "pos", "dy", "dgain"])
def test_norm_rotary_backward(rnn, other):
    op = rnn.NormRotary(1, 1, 32, (ROWS,))
    for shift in {1, NORM[other] - 1, -(ROWS * W - 1)} | ({0} if other != "dy" else set()):
        buf, b = pieces(NORM, y=(other, shift))
        refused(rnn, buf, lambda: op.backward(1, b["x"], W, 0, b["gain"], b["dy"], W, 0, b["dgain"],
                                              pos=b["pos"], dx=b["y"], dxstride=W))


def test_norm_rotary_beside_its_input(rnn):
    """Other columns of x's buffer: the bits of a buffer of its own; one column less
    apart is refused."""
    op, g = rnn.NormRotary(1, 1, 32, (ROWS,)), torch.Generator().manual_seed(1)
    buf = torch.randn(ROWS, 2 * W + 1, generator=g).cuda()
    dy = torch.randn(ROWS, W, generator=g).cuda()
    x = buf[:, :W].contiguous()
    s = 2 * W + 1
    op.forward(1, buf, s, 0, y=buf, ystride=s, yoff=W + 1)
    assert torch.equal(buf[:, W + 1:], op.forward(1, x, W)[0])
    op.backward(1, buf, s, 0, None, dy, W, dx=buf, dxstride=s, dxoff=W)
    assert torch.equal(buf[:, W:2 * W], op.backward(1, x, W, 0, None, dy, W)[0])
    assert torch.equal(buf[:, :W], x)
    with pytest.raises(rnn.RnnError):
        op.forward(1, buf, s, 0, y=buf, ystride=s, yoff=W - 1)
    with pytest.raises(rnn.RnnError):
        op.backward(1, buf, s, 0, None, dy, W, dx=buf, dxstride=s, dxoff=W - 1)


GATE = dict(x=ROWS * W, z=ROWS * W, gain=W, y=ROWS * W, dy=ROWS * W, dz=ROWS * W, dgain=W)


@pytest.mark.parametrize("other", ["x", "z", "gain"])
def test_head_gate_forward(rnn, other):
    op = rnn.HeadGate(2, 32)
    for shift in {1, GATE[other] - 1, -(ROWS * W - 1)} | ({0} if other != "x" else set()):
        buf, b = pieces(GATE, y=(other, shift))
        refused(rnn, buf, lambda: op.forward(ROWS, b["x"], b["z"], W, 0, b["gain"], b["y"]))


@pytest.mark.parametrize("out", ["y", "dz"])  # dx, dz
@pytest.mark.parametrize("other", ["x", "z", "gain", "dy", "dgain", "the other"])
def test_head_gate_backward(rnn, out, other):
    op = rnn.HeadGate(2, 32)
    name = dict(y="dz", dz="y")[out] if other == "the other" else other
    may = name in (("x", "dy") if out == "y" else ("z",))
    for shift in {1, GATE[name] - 1, -(ROWS * W - 1)} | (set() if may else {0}):
        buf, b = pieces(GATE, **{out: (name, shift)})
        refused(rnn, buf, lambda: op.backward(ROWS, b["x"], b["z"], W, 0, b["gain"], b["dy"], b["dz"],
                                              W, 0, b["dgain"], dx=b["y"]))


@pytest.mark.parametrize("dx", ["x", "dy"])
def test_head_gate_both_in_place(rnn, dx):
    op, g = rnn.HeadGate(2, 32), torch.Generator().manual_seed(2)
    x, z, dy = (torch.randn(ROWS, W, generator=g).cuda() for _ in range(3))
    dz = torch.empty_like(z)
    want = op.backward(ROWS, x, z, W, 0, None, dy, dz, W)
    into = dict(x=x, dy=dy)[dx]
    op.backward(ROWS, x, z, W, 0, None, dy, z, W, dx=into)
    assert torch.equal(into, want) and torch.equal(z, dz)
    buf = torch.randn(ROWS, 2 * W, generator=g).cuda()
    z, x = buf[:, W:].contiguous(), torch.randn(ROWS, W, generator=g).cuda()
    want = op.backward(ROWS, x, z, W, 0, None, dy, dz, W)
    # over the gate by another view of its buffer
    assert torch.equal(op.backward(ROWS, x, buf, 2 * W, W, None, dy, buf.view(-1)[W:], 2 * W), want)
    assert torch.equal(buf[:, W:], dz)
    with pytest.raises(rnn.RnnError):  # dz over the operand that dx takes the place of
        op.backward(ROWS, x, z, W, 0, None, dy, into, W, dx=into)
