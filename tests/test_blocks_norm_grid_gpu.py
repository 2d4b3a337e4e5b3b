"""ops.layer_norm over a row of 2^26 columns: the sums of the parameters' gradients take 64 threads a column, 2^32 in all, more than a launch holds."""
import pytest
import torch

from blocks_util import DEV

pytestmark = pytest.mark.gpu


def test_one_row_of_64_mi_columns():
    from dss_vae_amd import ops
    D = (1 << 26) + 40
    g = torch.Generator(device=DEV).manual_seed(7)
    x = torch.randn(1, D, device=DEV, generator=g).bfloat16()
    w = torch.ones(D, device=DEV, dtype=torch.bfloat16).requires_grad_()
    b = torch.zeros(D, device=DEV, dtype=torch.bfloat16).requires_grad_()
    dy = torch.randn(1, D, device=DEV, generator=g).bfloat16()
    y = ops.layer_norm(x, w, b)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    assert torch.equal(db, dy[0])
    # one row: dw = dy xh in fp32, rounded; y = xh rounded.  Half a step of bf16 each, and the statistics' 2^-12 of long fp32 chains
    want = dy[0].float() * y[0].detach().float()
    assert ((dw.float() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -8 + 2.0 ** -11)).all()
    assert float(dw.float().abs().sum()) > 0
