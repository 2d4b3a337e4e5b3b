"""ops.linear_act: a gradient that backward could not sum is refused before the forward pass runs; without that gradient the rows are free."""
import pytest
import torch

from blocks_util import DEV

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_weight_gradient_sums():
    from dss_vae_amd import ops
    M = (1 << 21) + 3
    x = torch.ones(M, 2, device=DEV, dtype=torch.bfloat16)
    w = torch.full((2, 2), 0.5, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="gradient of w sums over rows"):
        ops.linear_act(x, w.clone().requires_grad_())
    xs = x.clone().requires_grad_()
    y = ops.linear_act(xs, w)
    assert (y == 1).all()
    g, = torch.autograd.grad(y, xs, torch.ones_like(y))
    assert (g == 1).all()
    b = torch.zeros(2, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(ops.linear_act(x, w, b), b, torch.ones_like(y))
    assert (g == M).all()
    with torch.no_grad():
        assert (ops.linear_act(x, w.clone().requires_grad_()) == 1).all()
    wide = torch.zeros(M, 1, device=DEV, dtype=torch.bfloat16)
    one = torch.ones(3, 1, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="gradient of x sums over N"):
        ops.linear_act(one.clone().requires_grad_(), wide)
    ws = wide.clone().requires_grad_()
    g, = torch.autograd.grad(ops.linear_act(one, ws), ws, torch.ones(3, M, device=DEV, dtype=torch.bfloat16))
    assert (g == 3).all()
