"""GPU: rotary positions, differential attention and the Linear product with an
activation on a context whose stream is not the current one: every output
equals, bit for bit, that of the same calls on one stream."""
import pytest
import torch

from diffref import DiffCase

pytestmark = pytest.mark.gpu


def busy(n=12):
    """Some ten milliseconds of work for the current stream."""
    a = torch.ones(4096, 4096, device="cuda")
    for _ in range(n):
        a = a @ a
    return a


def attention(rnn):
    cs = DiffCase(3, 4, 2, 32, 70, 150, True, gap=0, causal=True, klen=[150, 7, 64], seed=1)
    data = dict(q=cs.q, kv=cs.kv, lam=cs.lam, gain=cs.gain, klen=cs.klen, dy=cs.dy)

    def calls(ctx, t):
        core = rnn.DiffCore(cs.h, cs.dh, cs.tq, cs.tk, cs.hkv, causal=True, ctx=ctx)
        geo = (t["q"], cs.qstride, 0, t["kv"], cs.kvstride, 0, cs.kw)
        y, saved = core.forward(cs.n, *geo, t["lam"], t["gain"], klen=t["klen"])
        out = dict(y=y, dq=torch.zeros_like(t["q"]), dkv=torch.zeros_like(t["kv"]),
                   dlam=torch.zeros_like(t["lam"]), dgain=torch.zeros_like(t["gain"]))
        core.backward(cs.n, *geo, t["lam"], t["gain"], saved, t["dy"], out["dq"], out["dkv"],
                      out["dlam"], out["dgain"], klen=t["klen"], set_dq=True, set_dkv=True)
        return out
    return data, calls


def split_attention(rnn):
    cs = DiffCase(1, 2, 2, 64, 2, 4000, True, gap=0, seed=2)
    data = dict(q=cs.q, kv=cs.kv, lam=cs.lam, gain=cs.gain)

    def calls(ctx, t):
        core = rnn.DiffCore(2, 64, 2, 4000, ctx=ctx)
        return dict(y=core.forward(1, t["q"], cs.qstride, 0, t["kv"], cs.kvstride, 0, cs.kw,
                                   t["lam"], t["gain"], train=False)[0])
    return data, calls


def linear(rnn):
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g)
    size = (4099, 130, 190)
    data = dict(x=rnd(4099, 130), w=rnd(190, 130), b=rnd(190), res=rnd(4099, 190), dy=rnd(4099, 190))

    def calls(ctx, t):
        y, slope = rnn.linear_act_forward(*size, t["x"], t["w"], t["b"], "gelu", res=t["res"], ctx=ctx)
        dw, db = torch.zeros_like(t["w"]), torch.zeros_like(t["b"])
        dx = rnn.linear_act_backward(*size, t["dy"], t["x"], t["w"], slope, "gelu", dw, db, ctx=ctx)
        return dict(y=y, dx=dx, dw=dw, db=db)
    return data, calls


def rotary(rnn):
    g = torch.Generator().manual_seed(4)
    data = dict(x=torch.randn(50 * 96, 128, generator=g), pos=torch.rand(50 * 96, 2, generator=g) * 99)

    def calls(ctx, t):
        rot = rnn.Rotary(4, 32, (8, 12), ctx=ctx)
        y = rot.forward(50, t["x"], 128, pos=t["pos"])
        return dict(y=y, dx=rot.backward(50, y, 128, pos=t["pos"]))
    return data, calls


ALL = [attention, split_attention, linear, rotary]


@pytest.mark.parametrize("make", ALL, ids=lambda f: f.__name__)
def test_inputs_and_results_in_order(rnn, make):
    """Inputs that the current stream is still to write, memory that it still
    uses, and inputs and results that it overwrites at once after the calls."""
    data, calls = make(rnn)
    dev = {k: v.cuda() for k, v in data.items()}
    with rnn_context(rnn, torch.cuda.current_stream()) as ctx:
        want = {k: v.clone() for k, v in calls(ctx, dev).items()}
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
                out = calls(ctx, late)
                got = {k: v.clone() for k, v in out.items()}
                for v in [*late.values(), *out.values()]:
                    v.zero_()
            torch.cuda.synchronize()
        for k, v in want.items():
            assert torch.equal(got[k], v), k


@pytest.mark.parametrize("make", ALL, ids=lambda f: f.__name__)
def test_captured_from_another_stream(rnn, make):
    """A graph captured on one stream from a context on another holds the calls,
    and replays them to the eager result."""
    data, calls = make(rnn)
    dev = {k: v.cuda() for k, v in data.items()}
    with rnn_context(rnn, torch.cuda.Stream()) as ctx:
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            want = {k: v.clone() for k, v in calls(ctx, dev).items()}
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = calls(ctx, dev)
        for _ in range(3):
            with torch.cuda.stream(st):
                for v in out.values():
                    v.fill_(0.5)
                graph.replay()
                got = {k: v.clone() for k, v in out.items()}
            torch.cuda.synchronize()
            for k, v in want.items():
                assert torch.equal(got[k], v), k
            with torch.cuda.stream(st):
                calls(ctx, dev)
            torch.cuda.synchronize()


class rnn_context:
    def __init__(self, rnn, stream):
        self.ctx = rnn.Context(0, stream=stream)

    def __enter__(self):
        return self.ctx

    def __exit__(self, *_):
        torch.cuda.synchronize()
        self.ctx.close()
