"""ops.linear_act's exact gelu and its slope in fp32 have the accuracy of the error function, near 0 and in the tail."""
import math

import pytest
import torch

from blocks_util import DEV, U32

pytestmark = pytest.mark.gpu


def test_relative_accuracy():
    """z / sqrt 2 is off by one rounding and 0.3 of the constant, which the tail of Phi multiplies by z^2 + 1: 1.3 (z^2 + 1) units; the error
    function adds 8 and the products 3.  The slope Phi + z phi: the same of the first term, and of the second the exponential's argument
    z^2 / 2, off by 2.3 roundings of it, 1.15 z^2, and 6 for the instruction and the products."""
    from dss_vae_amd import ops
    z = torch.cat((torch.logspace(-20, -1, 300), torch.linspace(0.1, 10.0, 3000)))
    z = torch.cat((z, -z))
    x = z.to(DEV).view(-1, 1).requires_grad_()
    y = ops.linear_act(x, torch.ones(1, 1, device=DEV), None, "gelu")
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    d = z.double()
    cdf = 0.5 * torch.special.erfc(-d / math.sqrt(2))
    pdf = torch.exp(-d * d / 2) / math.sqrt(2 * math.pi)
    units = 16 + 1.3 * d * d
    got, want = y.detach().cpu().double().view(-1), d * cdf
    err = (got - want).abs() / want.abs()
    assert (err <= units * U32).all(), float((err / units / U32).max())
    got, want = g.cpu().double().view(-1), cdf + d * pdf
    err = (got - want).abs() / (cdf + (d * pdf).abs())
    assert (err <= units * U32).all(), float((err / units / U32).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_value_of_the_16_bit_types(dtype):
    """one rounding: half a step of the type, and a twentieth of it for what comes before (1e-6 of the rational form; exp2's argument z^2 / 2 log2 e,
    off by 2.3 roundings: 1.2 z^2 units of 2^-24, 1.4e-5 at z = -14).  The slope goes through a 16-bit code, its fourth
    root in steps of 1 / 31744: off by 2 / 31744 |s|^(3/4), and the product over one column is rounded to the type."""
    from dss_vae_amd import ops
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    z = every[every.isfinite() & (every.abs() < 13) & ((every.abs() > 1e-30) | (every == 0))]
    for rows in (z.numel(), 1):  # z along the rows: the tiles; along the columns of one row: the few-row kernel
        x = z.to(DEV).view(-1, 1) if rows > 1 else torch.ones(1, 1, device=DEV, dtype=dtype)
        w = torch.ones(1, 1, device=DEV, dtype=dtype) if rows > 1 else z.to(DEV).view(-1, 1)
        x.requires_grad_(rows > 1)
        y = ops.linear_act(x, w, None, "gelu")
        d = z.double()
        cdf = 0.5 * torch.special.erfc(-d / math.sqrt(2))
        want = d * cdf
        smallest = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        bound = torch.finfo(dtype).eps / 2 * 1.05 * want.abs() + smallest
        err = (y.detach().cpu().double().view(-1) - want).abs()
        assert (err <= bound).all(), float((err / bound).max())
        if rows > 1:
            g, = torch.autograd.grad(y, x, torch.ones_like(y))
            slope = cdf + d * torch.exp(-d * d / 2) / math.sqrt(2 * math.pi)
            err = (g.cpu().double().view(-1) - slope).abs()
            assert (err <= torch.finfo(dtype).eps / 2 * 1.05 * slope.abs() + 2.02 / 31744 * slope.abs() ** 0.75 + 1.2e-7).all()
