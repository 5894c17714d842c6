"""GPU: the Linear product with activation and residual (rnn_linear_act_*)
against its plain statement in 64 bits.

Tolerance: 1e-5 relative Frobenius, as the products of the GEMM core that it
runs on; the activation adds a few steps of 2^-24.  RELU's slope jumps at 0, so
its inputs are small whole numbers, whose z is exact."""
import pytest
import torch

from conftest import TOL, rel_frob
from diffref import D, act

pytestmark = pytest.mark.gpu

# small and odd ones, then one for every tile and split of each product
SIZES = [(1, 1, 1), (1, 256, 1024), (3, 7, 5), (64, 256, 1024), (65, 33, 129), (200, 96, 352),
         (1813, 387, 251), (513, 64, 64), (8192, 32, 48), (37, 0, 9), (4096, 40, 36),
         (2048, 256, 160), (130, 1030, 70), (4099, 129, 131), (8192, 33, 511), (4099, 129, 384),
         (2100, 70, 330), (8200, 513, 40), (4099, 384, 33), (2100, 330, 70)]


def inputs(rows, fin, fout, seed=0, whole=False):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    x, w, b = rnd(rows, fin), rnd(fout, fin) / max(fin, 1) ** 0.5, rnd(fout)
    if whole:
        x, w, b = ((t * 2).round() for t in (rnd(rows, fin), rnd(fout, fin), rnd(fout)))
    return x, w, b, rnd(rows, fout), rnd(rows, fout)


def want(x, w, b, res, dy, name):
    x, w, b = (t.to(D).requires_grad_(True) for t in (x, w, b))
    y = act(name, x @ w.T + b) + res.to(D)
    g = torch.autograd.grad(y, (x, w, b), dy.to(D))
    return y.detach(), *g


@pytest.mark.parametrize("name", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward_and_gradients(rnn, size, name):
    rows, fin, fout = size
    x, w, b, res, dy = inputs(*size, whole=name == "relu")
    yw, dxw, dww, dbw = want(x, w, b, res, dy, name)
    X, W, B, RES, DY = (t.cuda() for t in (x, w, b, res, dy))
    y, z = rnn.linear_act_forward(*size, X, W, B, name, res=RES)
    assert (z is None) == (name == "none")
    assert rel_frob(y.cpu(), yw) < TOL
    ev, none = rnn.linear_act_forward(*size, X, W, B, name, res=RES, train=False)
    assert none is None and torch.equal(ev, y)
    inpl = RES.clone()
    rnn.linear_act_forward(*size, X, W, B, name, res=inpl, y=inpl)
    assert torch.equal(inpl, y)
    dw, db = torch.full_like(W, 0.5), torch.full_like(B, 0.25)
    z0 = None if z is None else z.clone()
    if fin == 0:
        return
    dx = rnn.linear_act_backward(*size, DY, X, W, z, name, dw, db)
    assert z is None or torch.equal(z, z0)
    assert rel_frob(dx.cpu(), dxw) < TOL
    # accumulated onto 0.5 and 0.25: the sum's own rounding besides
    for got, ref, old in ((dw, dww, 0.5), (db, dbw, 0.25)):
        err = (got.cpu().double() - old - ref).norm()
        assert err <= TOL * ref.norm() + 2.0 ** -23 * (ref.norm() + old * ref.numel() ** 0.5)
    acc = torch.full_like(X, 0.75)
    rnn.linear_act_backward(*size, DY, X, W, z, name, dw, None, dx=acc, acc_dx=True)
    assert (acc - (dx + 0.75)).abs().max() <= 2.0 ** -22 * (1 + float(dx.abs().max()))


@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
def test_wide_range(rnn, name):
    """z from -1e30 to 1e30 through a 1 x 1 product: outputs and slopes stay
    finite and keep their limits.  Relative 2^-20 of |y|, or 2^-20 where the
    value itself cancels towards 0."""
    z = torch.cat([torch.linspace(-12, 12, 4001), torch.tensor(
        [-1e30, -1e10, -200.0, -88.0, -30.0, 0.0, 30.0, 88.0, 200.0, 1e10, 1e30])])
    if name == "relu":
        z = z[z != 0]
    n = z.numel()
    one, dy = torch.ones(1, 1), torch.ones(n, 1)
    zd = z.to(D).requires_grad_(True)
    yw = act(name, zd)
    sw, = torch.autograd.grad(yw.sum(), zd)
    y, zz = rnn.linear_act_forward(n, 1, 1, z.cuda()[:, None], one.cuda(), None, name)
    dw = torch.zeros(1, 1, device="cuda")
    dx = rnn.linear_act_backward(n, 1, 1, dy.cuda(), z.cuda()[:, None], one.cuda(), zz, name, dw)
    tol = 2.0 ** -20
    assert ((y.cpu()[:, 0] - yw.detach()).abs() <= tol * (1 + yw.detach().abs())).all()
    sw = torch.nan_to_num(sw, nan=0.0)  # the statement's own 0 * inf
    fin = z.abs() <= 200
    assert ((dx.cpu()[:, 0] - sw).abs()[fin] <= tol * 2).all()
    lim = (z > 0).float()
    assert (dx.cpu()[:, 0][~fin] == lim[~fin]).all()


def test_gradients_against_differences(rnn):
    """Central differences of <y, dy> in x and w; step 2^-5: the third-order
    term is below 1e-3 of the derivative."""
    size = (33, 40, 50)
    x, w, b, res, dy = (t.cuda() for t in inputs(*size, seed=4))
    _, z = rnn.linear_act_forward(*size, x, w, b, "gelu", res=res)
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    dx = rnn.linear_act_backward(*size, dy, x, w, z, "gelu", dw, db)

    def value(x, w, b):
        y, _ = rnn.linear_act_forward(*size, x, w, b, "gelu", res=res, train=False)
        return float((y.double() * dy.double()).sum())

    h = 2.0 ** -5
    for k, g in ((0, dx), (1, dw), (2, db)):
        d = g / g.norm()
        up = [t + h * d if i == k else t for i, t in enumerate((x, w, b))]
        dn = [t - h * d if i == k else t for i, t in enumerate((x, w, b))]
        num = (value(*up) - value(*dn)) / (2 * h)
        assert abs(num - float(g.double().norm())) <= 2e-3 * float(g.norm()), k


def test_refusals(rnn):
    size = (8, 16, 4)
    x, w, b, res, dy = (t.cuda() for t in inputs(*size))
    with pytest.raises(ValueError):
        rnn.linear_act_forward(*size, x, w, b, "tanh")
    with pytest.raises(TypeError):
        rnn.linear_act_forward(*size, x.double(), w, b, "gelu")
    with pytest.raises(ValueError):
        rnn.linear_act_forward(9, 16, 4, x, w, b, "gelu")
    with pytest.raises(ValueError):
        rnn.linear_act_forward(*size, x, w, b[:3], "gelu")
    with pytest.raises(rnn.RnnError):
        rnn.linear_act_forward(4, 4, 4, x, w, b, "gelu", y=x)
    with pytest.raises(ValueError):
        rnn.linear_act_backward(*size, dy, x, w, None, "gelu", w.clone())
    with pytest.raises(ValueError):
        rnn.linear_act_backward(*size, dy, x, w, dy, "gelu", w.clone(), acc_dx=True)
    L, ctx = rnn.lib(), rnn.default_ctx()
    p = lambda t: t.data_ptr()
    y = torch.zeros(8, 4, device="cuda")
    assert L.rnn_linear_act_forward(ctx.h, *size, p(x), p(w), None, 5, None, None, p(y)) == \
        rnn.RNN_E_INVALID
    assert L.rnn_linear_act_forward(ctx.h, *size, p(x), None, None, 1, None, None, p(y)) == \
        rnn.RNN_E_NULL
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    bwd = lambda sz, ws, nb, dx, db=None, flags=0: L.rnn_linear_act_backward(
        ctx.h, *sz, p(dy), p(x), p(w), p(y), ws, nb, p(dw), db, dx, flags)
    assert bwd(size, None, 0, p(dy)) == rnn.RNN_E_INVALID  # dx over dy
    assert bwd(size, None, 0, p(dx), None, 2) == rnn.RNN_E_INVALID
    assert bwd(size, None, 0, None) == rnn.RNN_E_NULL
    assert bwd((8, 0, 4), None, 0, p(dx), p(db)) == rnn.RNN_E_UNSUPPORTED  # db without inputs
    assert bwd((1 << 31, 16, 4), None, 0, p(dx)) == rnn.RNN_E_UNSUPPORTED
    import ctypes as C
    nb = C.c_size_t()
    big = (4096, 64, 64)
    assert L.rnn_linear_act_workspace(*big, C.byref(nb)) == 0 and nb.value > 0
    ws = torch.zeros(nb.value + 256, dtype=torch.uint8, device="cuda")
    assert bwd(big, None, nb.value, p(dx)) == rnn.RNN_E_NULL
    assert bwd(big, p(ws), nb.value - 1, p(dx)) == rnn.RNN_E_INVALID
    assert bwd(big, p(ws) + 16, nb.value, p(dx)) == rnn.RNN_E_INVALID


def test_same_bits_captured_and_replayed(rnn):
    """Two graphs of forward and backward on one context, replayed in turn with
    eager calls between, each to its eager result, bit for bit."""
    size = (700, 130, 190)
    st = torch.cuda.Stream()
    ctx = rnn.Context(0, stream=st)
    runs = []
    for s in range(2):
        x, w, b, res, dy = (t.cuda() for t in inputs(*size, seed=10 + s))
        dw, db = torch.zeros_like(w), torch.zeros_like(b)

        def call(x=x, w=w, b=b, res=res, dy=dy, dw=dw, db=db):
            dw.zero_()
            db.zero_()
            y, sl = rnn.linear_act_forward(*size, x, w, b, "gelu", res=res, ctx=ctx)
            return y, rnn.linear_act_backward(*size, dy, x, w, sl, "gelu", dw, db, ctx=ctx)

        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            y, dx = call()
        st.synchronize()
        want = [t.clone() for t in (y, dx, dw, db)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            y, dx = call()
        runs.append((graph, (y, dx, dw, db), want, call))
    for _ in range(3):
        for graph, out, want, call in runs:
            with torch.cuda.stream(st):
                for t in out:
                    t.fill_(0.5)
                graph.replay()
            st.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            with torch.cuda.stream(st):
                call()
            st.synchronize()
    ctx.close()
