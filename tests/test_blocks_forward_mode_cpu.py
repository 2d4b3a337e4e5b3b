"""What the sequence-block operators ask of their arguments before they record a graph or launch anything: no dual tensors."""
import pytest
import torch
from torch.autograd import forward_ad as fwad

from dss_vae_amd import ops


def test_dual_tensors_are_seen():
    x, g = torch.ones(3), torch.ones(3, requires_grad=True)
    assert not ops._wants_grad("op", x, None) and ops._wants_grad("op", x, g)
    with fwad.dual_level():
        assert not ops._wants_grad("op", x, None) and ops._wants_grad("op", None, g)
        d = fwad.make_dual(x, torch.zeros(3))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(RuntimeError, match="op: no forward-mode"):
                ops._wants_grad("op", None, d)
    assert not ops._wants_grad("op", x)
    with torch.no_grad():
        assert not ops._wants_grad("op", g)
