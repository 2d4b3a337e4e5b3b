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
