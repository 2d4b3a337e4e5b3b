"""ops.layer_norm against its definition in 64 bits: types, widths of every kernel shape and the edges between them,
strides, missing parameters, rows that are constant or not finite, graph replay, other streams."""
import pytest
import torch

from blocks_util import DEV, TYPES, bits, check, rnd

pytestmark = pytest.mark.gpu


def reference(x, w, b, eps, dy):
    """-> y, dx, dw, db and the scales of their fp32 errors, in 64 bits"""
    x, dy = x.double(), dy.double()
    D = x.size(-1)
    w = torch.ones(D, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(D, dtype=torch.float64) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = c * rstd
    # the mean is off by a few roundings of mean|x|, xh by that times rstd
    off = rstd * x.abs().mean(-1, keepdim=True)
    gw = dy * w
    s1, s2 = gw.mean(-1, keepdim=True), (gw * xh).mean(-1, keepdim=True)
    dx = rstd * (gw - s1 - xh * s2)
    sdx = rstd * (1 + off) * (gw.abs() + gw.abs().mean(-1, keepdim=True) * (1 + xh.abs()) +
                              (1 + xh.abs()) * (gw * xh).abs().mean(-1, keepdim=True))
    return (xh * w + b, dx, (dy * xh).sum(0), dy.sum(0),
            w.abs() * (xh.abs() + off) + b.abs(), sdx, (dy.abs() * (xh.abs() + off)).sum(0), dy.abs().sum(0))


def run(x, w, b, eps, dy):
    from dss_vae_amd import ops
    leaves = [t.detach().clone().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = ops.layer_norm(leaves[0], leaves[1], leaves[2], eps)
    y.backward(dy)
    return [y] + [None if t is None else t.grad for t in leaves]


# slack: a sum of D terms is a chain of at most 32 in a thread (40 in the wide form here) plus ten shuffle / LDS steps,
# twice (mean, then variance or the two gradient means), plus the closing products: 2 * 50 + 8 < 128
SLACK = 128


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 2), (5, 7), (9, 64), (50, 150), (31, 300), (17, 301), (4, 512), (6, 513),
                                    (50, 1024), (3, 1025), (2, 2047), (33, 2048), (2, 4100), (3, 8192), (2, 8193),
                                    (2, 40000), (700, 36), (2100, 300)])
def test_forward_and_gradients(dtype, rows, D):
    for params in (dtype, torch.float32):
        x = rnd(rows, D, seed=D, scale=1.5, shift=0.4, dtype=dtype)
        w, b = rnd(D, seed=1, scale=0.3, shift=1.0, dtype=params), rnd(D, seed=2, scale=0.3, dtype=params)
        dy = rnd(rows, D, seed=3, dtype=dtype)
        eps = 1e-5
        ref = reference(x, w, b, eps, dy)
        got = run(x.to(DEV), w.to(DEV), b.to(DEV), eps, dy.to(DEV))
        if D == 1:  # xh is 0 / sqrt(eps): exact
            assert (got[0].cpu() == b.to(dtype)).all() and (got[1].cpu() == 0).all()
        for name, g, r, s in zip(("y", "dx", "dw", "db"), got, ref[:4], ref[4:]):
            check(g, r, s, SLACK, (name, rows, D, dtype, params))
        if params == torch.float32 and dtype == params:
            break


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [300, 256, 77])
def test_strides_and_alignment(dtype, D):
    """rows cut out of a wider buffer at every offset, a transposed input, an expanded gradient: as their copies"""
    from dss_vae_amd import ops
    wide = rnd(11, D + 40, seed=4, dtype=dtype).to(DEV)
    w, b = rnd(D + 3, seed=5, dtype=dtype).to(DEV), rnd(D + 3, seed=6, dtype=dtype).to(DEV)
    for off in (0, 1, 2, 3, 8):
        x, wo, bo = wide[:, off:off + D], w[off % 4:][:D], b[off % 4:][:D]
        if wo.numel() < D:
            wo, bo = w[:D], b[:D]
        # against the definition, not against the copy's result: two roundings of nearly the same value may end a step apart
        ref = reference(x.cpu(), wo.cpu(), bo.cpu(), 1e-5, x.cpu())
        check(ops.layer_norm(x, wo, bo), ref[0], ref[4], SLACK, ("offset", off))
    xt = rnd(D, 9, seed=7, dtype=dtype).to(DEV).t()
    assert torch.equal(bits(ops.layer_norm(xt)), bits(ops.layer_norm(xt.contiguous())))
    xe = wide[:1, :D].expand(6, D)
    assert torch.equal(bits(ops.layer_norm(xe)), bits(ops.layer_norm(xe.contiguous())))
    x3 = wide[:10, :D].unflatten(0, (5, 2)).detach().requires_grad_()
    ops.layer_norm(x3).sum().backward()  # dy is an expanded scalar
    assert x3.grad.shape == x3.shape
    ref = reference(x3.detach().cpu().reshape(10, D), None, None, 1e-5, torch.ones(10, D))
    check(x3.grad.reshape(10, D), ref[1], ref[5], SLACK)


@pytest.mark.parametrize("params", [(False, False), (True, False), (False, True)])
def test_missing_parameters(params):
    x, dy = rnd(21, 300, seed=8), rnd(21, 300, seed=9)
    w = rnd(300, seed=10) if params[0] else None
    b = rnd(300, seed=11) if params[1] else None
    ref = reference(x, w, b, 1e-3, dy)
    got = run(x.to(DEV), None if w is None else w.to(DEV), None if b is None else b.to(DEV), 1e-3, dy.to(DEV))
    for name, g, r, s in zip(("y", "dx", "dw", "db"), got, ref[:4], ref[4:]):
        if g is not None:
            check(g, r, s, SLACK, name)


def test_rows_do_not_touch_each_other():
    """a row of NaN, one with an infinity, a constant one: their neighbours keep the bits they have without them"""
    from dss_vae_amd import ops
    for D in (64, 300, 3000, 9000):
        x = rnd(12, D, seed=12).to(DEV)
        clean = ops.layer_norm(x)
        y = x.clone()
        y[3], y[5, D // 2], y[7] = float("nan"), float("inf"), 2.5
        got = ops.layer_norm(y)
        keep = [0, 1, 2, 4, 6, 8, 9, 10, 11]
        assert torch.equal(got[keep], clean[keep])
        assert got[3].isnan().all() and got[5].isnan().all() and (got[7] == 0).all()


def test_no_rows_and_frozen_inputs():
    from dss_vae_amd import ops
    w = torch.ones(40, device=DEV, requires_grad=True)
    y = ops.layer_norm(torch.zeros(0, 40, device=DEV), w)
    assert y.shape == (0, 40)
    y.sum().backward()
    assert torch.equal(w.grad, torch.zeros(40, device=DEV))
    x = rnd(5, 40, seed=13).to(DEV).requires_grad_()
    ops.layer_norm(x, w.detach()).sum().backward()
    only_x = x.grad.clone()
    x.grad = None
    ops.layer_norm(x, w).sum().backward()
    assert torch.equal(bits(only_x), bits(x.grad))


def test_gradient_against_differences():
    x, w, b, dy = rnd(3, 10, seed=14), rnd(10, seed=15), rnd(10, seed=16), rnd(3, 10, seed=17)
    got = run(x.to(DEV), w.to(DEV), b.to(DEV), 1e-5, dy.to(DEV))[1].cpu().double()
    h = 1e-5
    for i in range(3):
        for j in range(10):
            up, down = x.double().clone(), x.double().clone()
            up[i, j] += h
            down[i, j] -= h
            f = lambda t: (torch.nn.functional.layer_norm(t, (10,), w.double(), b.double(), 1e-5) * dy.double()).sum()  # noqa: E731
            assert abs(float((f(up) - f(down)) / (2 * h)) - float(got[i, j])) < 1e-4


def test_same_bits_twice_and_in_a_replayed_graph():
    from dss_vae_amd import ops
    x = rnd(700, 300, seed=18).to(DEV)
    w, b, dy = rnd(300, seed=19).to(DEV), rnd(300, seed=20).to(DEV), rnd(700, 300, seed=21).to(DEV)
    eager = run(x, w, b, 1e-5, dy)
    for a, c in zip(eager, run(x, w, b, 1e-5, dy)):
        assert torch.equal(bits(a), bits(c))
    xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))

    def step():
        y = ops.layer_norm(xs, ws, bs, 1e-5)
        return (y,) + torch.autograd.grad(y, (xs, ws, bs), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        xs.data.copy_(x * (k + 1))
        want = run(xs.detach(), w, b, 1e-5, dy)
        for o in out:
            o.detach().fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(bits(a.detach()), bits(c.detach())), k


def test_refusals():
    from dss_vae_amd import ops
    x = torch.zeros(4, 8, device=DEV)
    for bad in (lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x.long()),
                lambda: ops.layer_norm(torch.zeros((), device=DEV)), lambda: ops.layer_norm(x[:, :0]),
                lambda: ops.layer_norm(x, torch.zeros(7, device=DEV)), lambda: ops.layer_norm(x, torch.zeros(8)),
                lambda: ops.layer_norm(x, torch.zeros(8, device=DEV).bfloat16()),
                lambda: ops.layer_norm(x, torch.zeros(8, device=DEV).half(), torch.zeros(8, device=DEV)),
                lambda: ops.layer_norm(x, eps=-1.0), lambda: ops.layer_norm(x, eps=float("nan")),
                lambda: ops.layer_norm(x.cpu())):
        with pytest.raises(RuntimeError):
            bad()
    z = x.clone().requires_grad_()
    g, = torch.autograd.grad(ops.layer_norm(z).sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative
        g.sum().backward()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,D", [(40, 4), (33, 9), (70, 127), (70, 128), (70, 129), (33, 511), (20, 1023), (9, 2049), (9, 4095),
                                    (5, 4097), (3, 8191), (600, 1001)])
def test_ragged_widths(dtype, rows, D):
    """rows that end inside a granule, at every border of the kernels' shapes; many rows to a block and fewer than a block"""
    x, w, b = rnd(rows, D, seed=D, shift=0.2, dtype=dtype), rnd(D, seed=1, shift=1.0, dtype=dtype), rnd(D, seed=2, dtype=dtype)
    dy = rnd(rows, D, seed=3, dtype=dtype)
    ref = reference(x, w, b, 1e-5, dy)
    got = run(x.to(DEV), w.to(DEV), b.to(DEV), 1e-5, dy.to(DEV))
    for name, g, r, s in zip(("y", "dx", "dw", "db"), got, ref[:4], ref[4:]):
        check(g, r, s, SLACK, (name, rows, D, dtype))


def test_ragged_rows_beside_values_that_are_not_finite():
    """what stands right behind a ragged row (the next row, or the buffer around it) does not reach it"""
    from dss_vae_amd import ops
    for dtype in TYPES:
        for D in (5, 77, 333, 1100):
            clean = rnd(6, D, seed=D, dtype=dtype).to(DEV)
            dy = rnd(6, D, seed=1, dtype=dtype).to(DEV)
            wide = torch.full((6, D + 9), float("inf"), dtype=dtype, device=DEV)
            gwide = torch.full((6, D + 9), float("nan"), dtype=dtype, device=DEV)
            wide[:, 4:4 + D], gwide[:, 4:4 + D] = clean, dy
            a, b = clean.clone().requires_grad_(), wide[:, 4:4 + D].detach().requires_grad_()
            ya, yb = ops.layer_norm(a), ops.layer_norm(b)
            ga, = torch.autograd.grad(ya, a, dy)
            gb, = torch.autograd.grad(yb, b, gwide[:, 4:4 + D])
            assert torch.equal(bits(ya.detach()), bits(yb.detach())) and torch.equal(bits(ga), bits(gb))
