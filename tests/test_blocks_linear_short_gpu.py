"""ops.linear_act in fp32 over short sums: no fewer bits than fp32 products and sums have."""
import math

import pytest
import torch

from blocks_util import DEV, U32, bits, rnd

pytestmark = pytest.mark.gpu


def test_one_product_is_rounded_once():
    from dss_vae_amd import ops
    for M, N in ((300, 200), (70, 500), (20, 100)):
        x, w, dy = rnd(M, 1, seed=100).to(DEV), rnd(N, 1, seed=101).to(DEV), rnd(M, N, seed=102).to(DEV)
        assert torch.equal(bits(ops.linear_act(x, w)), bits(x * w.t()))
        # the sums of the gradients: over one column, over one row
        xs, ws = x.clone().requires_grad_(), w[:1].clone().requires_grad_()
        gx, = torch.autograd.grad(ops.linear_act(xs, ws), xs, dy[:, :1].contiguous())
        assert torch.equal(bits(gx), bits(dy[:, :1] * w[:1]))
        xs, ws = x[:1].clone(), w.clone().requires_grad_()
        gw, = torch.autograd.grad(ops.linear_act(xs, ws), ws, dy[:1].contiguous())
        assert torch.equal(bits(gw), bits(dy[:1].t() * x[:1]))


@pytest.mark.parametrize("K", [2, 3, 4, 8, 16, 17, 31, 64, 65, 100])
def test_short_sums(K):
    """a sum of K products by fused multiply-adds in any order: K roundings, each to nearest and so off by at most 2^-24 of a partial sum, which
    is at most sum |x w|: K units of 2^-24 of it (fp32's eps is 2^-23, half a step of it 2^-24; and one unit for the bound's second
    order).  Sums of more than 32, from three-part operands, leave out 2^-22 of each product beside that: 4 units"""
    from dss_vae_amd import ops
    for M, N in ((300, 200), (129, 70)):
        x, w = rnd(M, K, seed=103), rnd(N, K, seed=104)
        want, mag = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
        got = ops.linear_act(x.to(DEV), w.to(DEV)).cpu().double()
        bound = (K + 1 + (4 if K > 32 else 0)) * U32 * mag
        assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())
        # and in the mean square no more than sequential fp32 sums have (the order differs: 1.3 times)
        seq = torch.zeros(M, N)
        for k in range(K):
            seq = (seq.double() + x[:, k:k + 1].double() * w[:, k].double()).float()
        assert float((got - want).norm()) <= 1.3 * float((seq.double() - want).norm()) + 1e-30


def test_gradients_do_not_depend_on_which_is_wanted():
    """fp32: dx and dw have the same bits alone and together"""
    from dss_vae_amd import ops
    for M, N, K in ((40, 24, 32), (520, 300, 200), (2000, 600, 300)):
        x, w, dy = rnd(M, K, seed=105).to(DEV), rnd(N, K, seed=106).to(DEV), rnd(M, N, seed=107).to(DEV)
        leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
        both = torch.autograd.grad(ops.linear_act(*leaves, None, "gelu"), leaves, dy)
        for i in range(2):
            one = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w))]
            g, = torch.autograd.grad(ops.linear_act(*one, None, "gelu"), one[i], dy)
            assert torch.equal(bits(g), bits(both[i])), (M, i)
