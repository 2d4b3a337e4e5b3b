"""ops.layer_norm over rows whose values share a large offset: the mean is that of the values to half a step, not that of rounded partial sums."""
import pytest
import torch

from blocks_util import DEV, TYPES, U32, half_step, rnd

pytestmark = pytest.mark.gpu
WIDTHS = [7, 150, 300, 512, 1024, 1581, 4096, 8192, 8200, 20000]


@pytest.mark.parametrize("D", WIDTHS)
def test_equal_values(D):
    """the mean of equal values is that value: the bias comes out, exactly, and the gradient is that of a row of zeros"""
    from dss_vae_amd import ops
    c = torch.cat((torch.tensor([0.1, 178.86284, 99999.9, -3.3e7, 1.1e-20, 3.3e30, 2.5, 0.0]), rnd(200, seed=90, scale=100.0)))
    x = c.view(-1, 1).expand(-1, D).contiguous().to(DEV)
    w, b = rnd(D, seed=91, shift=1.0).to(DEV), rnd(D, seed=92).to(DEV)
    y = ops.layer_norm(x, w, b)
    assert torch.equal(y, b.expand_as(y))
    xs, zs = x.requires_grad_(), torch.zeros_like(x).requires_grad_()
    dy = rnd(c.numel(), D, seed=93).to(DEV)
    g, = torch.autograd.grad(ops.layer_norm(xs, w, b), xs, dy)
    z, = torch.autograd.grad(ops.layer_norm(zs, w, b), zs, dy)
    assert torch.equal(g, z)


@pytest.mark.parametrize("D", WIDTHS)
def test_large_offsets(D):
    """values around 1e4 and 1e6: the mean is rounded once (half a step of it), and a hundredth of that again for its sums; the deviations
    are exact, their squares, the root and the products stay below D / 16 + 40 units"""
    from dss_vae_amd import ops
    for offset in (1e4, 1e6):
        x = rnd(40, D, seed=94, scale=offset / 100, shift=offset)
        y = ops.layer_norm(x.to(DEV)).cpu().double()
        xd = x.double()
        m = xd.mean(1, keepdim=True)
        rstd = ((xd - m).square().mean(1, keepdim=True) + 1e-5).rsqrt()
        want = (xd - m) * rstd
        _, e = torch.frexp(m.float().abs())
        half = torch.ldexp(torch.ones_like(m), e - 25)  # half the spacing of fp32 numbers at the mean
        bound = rstd * half * 1.01 + (40 + D / 16) * U32 * (want.abs() + rstd * half)
        assert ((y - want).abs() <= bound).all(), (offset, float(((y - want).abs() / bound).max()))


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_values_in_every_type(dtype):
    from dss_vae_amd import ops
    c = rnd(60, seed=95, scale=50.0).to(dtype)
    for D in (33, 301, 2050):
        x = c.view(-1, 1).expand(-1, D).contiguous().to(DEV)
        assert (ops.layer_norm(x) == 0).all()
