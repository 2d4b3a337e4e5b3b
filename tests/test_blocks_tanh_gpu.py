"""tanh and its slope keep their relative accuracy in fp32, near 0 and where tanh saturates: ops.linear_act and ops.gated_scan / gated_step."""
import pytest
import torch

from blocks_util import DEV, U32

pytestmark = pytest.mark.gpu


def points():
    z = torch.cat((torch.logspace(-30, -2, 400), torch.linspace(0.01, 2.0, 2000), torch.linspace(2.0, 12.0, 1000)))
    return torch.cat((z, -z))


# u = exp(-2 |z|) is off by 2 |z| units of 2^-24 (its argument's rounding) and 2 of the instruction; tanh = (1 - u) / (1 + u) is only
# formed where u < 2 / 3, which at most doubles that, and 4 for the sums, the quotient and the product: 16 units hold everywhere.
# The slope 4 u / (1 + u)^2: 2 |z| + 2, twice 4, and 3 products.
TANH = 16


def slope_units(z):
    return 2 * z.abs() + 16


def test_linear_act():
    from dss_vae_amd import ops
    z = points()
    for rows in (1, 50, 100):  # the few-row kernel and the tiles
        x = z.to(DEV).view(-1, 1).expand(z.numel(), 1).contiguous() if rows == 100 else None
        if x is not None:
            xs, w = x.requires_grad_(), torch.ones(1, 1, device=DEV)
        else:  # z along the columns
            xs, w = torch.ones(rows, 1, device=DEV).requires_grad_(), z.to(DEV).view(-1, 1)
        ws = w.clone().requires_grad_()
        y = ops.linear_act(xs, ws, None, "tanh")
        got = (y.reshape(-1) if rows == 100 else y[-1]).detach().cpu().double()
        want = torch.tanh(z.double())
        assert ((got - want).abs() <= TANH * U32 * want.abs()).all(), float(((got - want) / want).abs().max() / U32)
        dy = torch.zeros_like(y)
        (dy.view(-1) if rows == 100 else dy[-1]).fill_(1.0)
        gx, gw = torch.autograd.grad(y, (xs, ws), dy)
        slope = (1.0 / torch.cosh(z.double())) ** 2
        s = gx.reshape(-1).cpu().double() if rows == 100 else gw.reshape(-1).cpu().double()
        err = (s - slope).abs() / slope
        assert (err <= slope_units(z.double()) * U32).all(), float((err / U32).max())


def test_gated_scan():
    from dss_vae_amd import ops
    v = points()
    H = v.numel()
    for T in (1, 2, 200):
        x = torch.zeros(1, T, 2 * H)
        x[0, 0, H:] = v
        x[0, 1:, :H] = float("inf")  # the steps behind keep the state
        xs = x.to(DEV).requires_grad_()
        out, last = ops.gated_scan(xs, None, None, False, "tanh")
        want = 0.5 * torch.tanh(v.double())
        got = last[0].detach().cpu().double()
        assert ((got - want).abs() <= (TANH + 4) * U32 * want.abs()).all(), float(((got - want) / want).abs().max() / U32)
        last.sum().backward()
        d = xs.grad[0, 0].cpu().double()
        slope = 0.5 / torch.cosh(v.double()) ** 2
        err = (d[H:] - slope).abs() / slope
        assert (err <= (slope_units(v.double()) + 4) * U32).all(), float((err / U32).max())
        dz = 0.25 * (0.0 - torch.tanh(v.double()))  # a (1 - a) (h_0 - n)
        assert ((d[:H] - dz).abs() <= (TANH + 8) * U32 * dz.abs()).all()
    out, h = ops.gated_step(x[:, 0].to(DEV), None, "tanh")
    assert ((h[0].cpu().double() - want).abs() <= (TANH + 4) * U32 * want.abs()).all()
