"""ops.gated_step's h_out is a write in place: graphs that saved the buffer notice it, leaves are refused."""
import pytest
import torch

from blocks_util import DEV, rnd

pytestmark = pytest.mark.gpu


def test_a_saved_state_that_is_overwritten():
    from dss_vae_amd import ops
    x, h, w = rnd(4, 16, seed=1).to(DEV), rnd(4, 8, seed=2).to(DEV), rnd(4, 8, seed=3).to(DEV).requires_grad_()
    loss = (h * w).sum()  # saves h
    with torch.no_grad():
        ops.gated_step(x, h, "tanh", h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    loss = (h * w).sum()
    with torch.no_grad():
        ops.gated_step(x, h, "tanh", torch.empty_like(h))
        ops.gated_step(x, h)
    loss.backward()
    assert torch.equal(w.grad, h)


def test_leaves_are_refused():
    from dss_vae_amd import ops
    x, h = rnd(4, 16, seed=1).to(DEV), rnd(4, 8, seed=2).to(DEV)
    leaf = torch.zeros(4, 8, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="h_out requires grad"):
        ops.gated_step(x, h, "tanh", leaf)
    want = ops.gated_step(x, h)[1]
    with torch.no_grad():
        ops.gated_step(x, h, "tanh", leaf)
    assert torch.equal(leaf.detach(), want)
    with torch.inference_mode():
        s = h.clone()
        ops.gated_step(x, s, "tanh", s)
        assert torch.equal(s, want)
