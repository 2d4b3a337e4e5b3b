"""ops.linear_act's backward pass in 16-bit types: dz = dy act'(z) goes into the products unrounded, so that dx and dw carry one rounding,
that of the result, whatever the size of dy; `round_dz` rounds it for half the matrix work."""
import math

import pytest
import torch

from blocks_util import DEV, bits, half_step, rnd
from test_blocks_linear_gpu import act

pytestmark = pytest.mark.gpu
TYPES16 = [torch.bfloat16, torch.float16]


def operands(M, N, K, dtype, dy_scale=1.0, w_scale=1.0):
    return (rnd(M, K, seed=70, dtype=dtype), rnd(N, K, seed=71, scale=w_scale * K ** -0.5, dtype=dtype), rnd(N, seed=72, scale=0.3, dtype=dtype),
            rnd(M, N, seed=73, scale=dy_scale, dtype=dtype))


def gradients(x, w, b, name, dy, **more):
    from dss_vae_amd import ops
    xs, ws, bs = (t.to(DEV).requires_grad_() for t in (x, w, b))
    return [g.cpu() for g in torch.autograd.grad(ops.linear_act(xs, ws, bs, name, **more), (xs, ws, bs), dy.to(DEV))]


def off(x, w, b, name, dy, got):
    """per gradient: (error of `got`, error of the exact values rounded once, what the 16-bit codes of act'(z) add), each as a
    norm.  A code is the fourth root in steps of 1 / 31744, off by 1 / sqrt(12) of one in the mean square, which moves the slope s by
    4 |s|^(3/4) times that, independently from element to element."""
    x, w, b, d = x.double(), w.double(), b.double(), dy.double()
    z = x @ w.t() + b
    slope = act(z, name)[1]
    dz = d * slope
    c = (d * 4 * slope.abs() ** 0.75 / 31744 / math.sqrt(12)) ** 2
    out = []
    for g, want, code in zip(got, (dz @ w, dz.t() @ x, dz.sum(0)), (c @ (w * w), c.t() @ (x * x), c.sum(0))):
        out.append((float((g.double() - want).norm()), float((want.to(g.dtype).double() - want).norm()), float(code.sum().sqrt())))
    return out


# Errors of many elements add up by their squares; 5 % over that for the spread of some ten thousand elements.  A dz rounded to
# the type adds as much again as the rounding of the result: 1.41 times.
@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("name", ["gelu", "silu", "tanh"])
@pytest.mark.parametrize("M,N,K", [(300, 260, 200), (513, 129, 67), (40, 600, 300), (2000, 72, 520), (1100, 1030, 264)])
def test_one_rounding(dtype, name, M, N, K):
    ops_ = operands(M, N, K, dtype)
    for key, (err, once, code) in zip(("dx", "dw"), off(*ops_[:3], name, ops_[3], gradients(*ops_[:3], name, ops_[3]))):
        assert err <= 1.05 * math.hypot(once, code), (key, err / once, code / once)


def test_upstream_gradients_at_the_ends_of_fp16():
    """dz beyond the type's largest number (gelu's slope reaches 1.13) and among its smallest ones: the results are ordinary numbers"""
    x, w, b, dy = operands(200, 160, 96, torch.float16, w_scale=1e-3)
    x, dy = (x.abs() + 1.0) * 0, torch.full_like(dy, 60000.0)
    b = torch.full_like(b, 1.4)
    for key, (err, once, code) in zip(("dx", "dw"), off(x, w, b, "gelu", dy, gradients(x, w, b, "gelu", dy))):
        assert err <= 1.05 * math.hypot(once, code) + 1e-30, (key, err, once, code)
    for name in ("gelu", "tanh"):
        x, w, b, dy = operands(300, 128, 96, torch.float16, dy_scale=2.0 ** -18)
        x, w = x * 2.0 ** -7, w * 2.0 ** 7
        for key, (err, once, code) in zip(("dx",), off(x, w, b, name, dy, gradients(x, w, b, name, dy))):
            assert err <= 1.05 * math.hypot(once, code), (key, err / once, code / once)


@pytest.mark.parametrize("dtype", TYPES16)
def test_values_that_are_not_finite(dtype):
    """infinite upstream gradients, inputs and weights give what the formula gives: infinities of the sign, NaN from 0 x inf and inf - inf"""
    x, w, b, dy = operands(150, 140, 100, dtype)
    w = w.abs() + 0.01
    clean = gradients(x, w, b, "gelu", dy)
    d = dy.clone()
    d[3, 5], d[4, 5], d[9, 7] = float("inf"), float("-inf"), float("nan")
    dx, dw, _ = gradients(x, w, b, "gelu", d)
    z = x.double() @ w.double().t() + b.double()
    s = act(z, "gelu")[1]
    for r, v in ((3, 1.0), (4, -1.0)):
        assert (dx[r] == math.copysign(math.inf, v * float(s[r, 5]))).all()
    assert dx[9].isnan().all() and dw[5].isnan().sum() + dw[5].isinf().sum() == 100 and dw[7].isnan().all()
    rows = [i for i in range(150) if i not in (3, 4, 9)]
    assert torch.equal(bits(dx[rows]), bits(clean[0][rows]))
    assert torch.equal(bits(dw[[0, 1, 2, 8]]), bits(clean[1][[0, 1, 2, 8]]))
    # an infinite input column whose dz are exact in the type (slope 1): inf of their sign, not NaN
    x2, d2 = x.abs() + 2.0, dy.abs() + 0.5
    w2 = torch.zeros_like(w)
    w2[:, 0] = 20.0
    for name in ("gelu", "tanh", "silu"):
        xs, ws = x2.to(DEV).requires_grad_(), w2.to(DEV).requires_grad_()
        from dss_vae_amd import ops
        y = ops.linear_act(xs, ws, None, name)
        xs.data[7, 3] = float("inf")  # (in backward only)
        dw = torch.autograd.grad(y, ws, d2.to(DEV))[0].cpu()
        if name != "tanh":
            assert (dw[:, 3] == math.inf).all(), name
        keep = [i for i in range(100) if i != 3]
        assert dw[:, keep].isfinite().all()


def test_rounded_dz_on_demand():
    """round_dz: dz rounded to the type, sqrt(2) times the error; the bias gradient and types or activations that need no second part
    stay as they are"""
    from dss_vae_amd import ops
    for dtype in TYPES16:
        x, w, b, dy = operands(300, 260, 200, dtype)
        wide, slim = gradients(x, w, b, "gelu", dy), gradients(x, w, b, "gelu", dy, round_dz=True)
        for (err, once, code), (err2, _, _) in zip(off(x, w, b, "gelu", dy, wide)[:2], off(x, w, b, "gelu", dy, slim)[:2]):
            assert 1.2 * once < err2 <= 1.05 * math.sqrt(2 * once ** 2 + code ** 2) and err < err2
        assert torch.equal(bits(wide[2]), bits(slim[2]))
        for name in ("none", "relu"):
            for p, q in zip(gradients(x, w, b, name, dy), gradients(x, w, b, name, dy, round_dz=True)):
                assert torch.equal(bits(p), bits(q)), name
    x, w, b, dy = operands(60, 50, 40, torch.float32)
    for p, q in zip(gradients(x, w, b, "gelu", dy), gradients(x, w, b, "gelu", dy, round_dz=True)):
        assert torch.equal(bits(p), bits(q))
    with torch.no_grad():
        xd, wd = x.to(DEV), w.to(DEV)
        assert torch.equal(ops.linear_act(xd, wd, None, "gelu", None, True), ops.linear_act(xd, wd, None, "gelu"))


@pytest.mark.parametrize("dtype", TYPES16)
def test_same_bits_whichever_gradient_is_wanted(dtype):
    x, w, b, dy = operands(520, 1030, 264, dtype)
    from dss_vae_amd import ops
    full = gradients(x, w, b, "silu", dy)
    for which in range(3):
        leaves = [t.to(DEV).requires_grad_(i == which) for i, t in enumerate((x, w, b))]
        g, = torch.autograd.grad(ops.linear_act(*leaves, "silu"), leaves[which], dy.to(DEV))
        assert torch.equal(bits(g.cpu()), bits(full[which])), which
    again = gradients(x, w, b, "silu", dy)
    assert all(torch.equal(bits(p), bits(q)) for p, q in zip(full, again))


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("name", ["gelu", "silu", "tanh"])
def test_slopes_that_are_kept(dtype, name):
    """every z of the type: the slope backward sees is off by half a step h = 1 / 63488 of its code (c = |s|^(1/4), 1 % on h for the root's
    roundings: t^4 is convex, so the slope by at most (c + h)^4 - c^4) and the roundings of its formula (20 units of 2^-24 of the terms it
    adds, at most 1.2; tanh's slope 2 |z| + 16 of itself), then rounded to the type; 0 and 1 are exact, infinite z have the slope they tend to, NaN stays"""
    from dss_vae_amd import ops
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    x = every.to(DEV).view(-1, 1).requires_grad_()
    y = ops.linear_act(x, torch.ones(1, 1, device=DEV, dtype=dtype), None, name)
    g = torch.autograd.grad(y, x, torch.ones_like(y))[0].cpu().double().view(-1)
    z = every.double()
    ok = z.isfinite()
    slope = torch.cosh(z[ok].clamp(-300, 300)) ** -2 if name == "tanh" else act(z[ok].clamp(-700, 700), name)[1]  # (1 - tanh^2 cancels in 64 bits)
    units = (2 * z[ok].abs() + 16) * slope if name == "tanh" else torch.full_like(slope, 24.0)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    code = (slope.abs() ** 0.25 + 1.01 / 63488) ** 4 - slope.abs()
    bound = torch.finfo(dtype).eps / 2 * 1.01 * slope.abs() + code + units * 2.0 ** -24 + tiny
    err = (g[ok] - slope).abs()
    assert (err <= bound).all(), (float((err / bound).max()), z[ok][(err / bound).argmax()])
    assert (g[z == math.inf] == (0 if name == "tanh" else 1)).all() and (g[z == -math.inf] == 0).all() and g[z.isnan()].isnan().all()
    if name != "tanh":
        assert (g[(z > 20) & ok] == 1).all()
