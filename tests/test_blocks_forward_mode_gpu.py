"""Forward-mode derivatives are refused: a dual tensor does not require grad, and an output without a tangent would be a derivative of zero."""
import pytest
import torch
from torch.autograd import forward_ad as fwad

from blocks_util import DEV, rnd

pytestmark = pytest.mark.gpu


def test_dual_tensors_are_refused():
    from dss_vae_amd import ops
    x, w, b = rnd(2, 3, 8, seed=1).to(DEV), rnd(4, 8, seed=2).to(DEV), rnd(8, seed=3).to(DEV)
    h, ids, t = rnd(2, 4, seed=4).to(DEV), torch.zeros(2, 3, 2, dtype=torch.long, device=DEV), rnd(2, 3, 2, seed=5).to(DEV)
    rows = torch.ones(2, 3, device=DEV)
    calls = [(lambda a: ops.layer_norm(a), x), (lambda a: ops.layer_norm(x, a), b), (lambda a: ops.layer_norm(x, None, a), b),
             (lambda a: ops.gated_scan(a), x), (lambda a: ops.gated_scan(x, a), h), (lambda a: ops.gated_step(a), x[:, 0]),
             (lambda a: ops.gated_step(x[:, 0], a), h), (lambda a: ops.gated_step(a, h, "tanh", torch.empty_like(h)), x[:, 0]),
             (lambda a: ops.linear_act(a, w), x), (lambda a: ops.linear_act(x, a), w), (lambda a: ops.linear_act(x, w, a), b[:4].clone()),
             (lambda a: ops.linear_act(x, w, None, "relu", a), rnd(2, 3, 4, seed=6).to(DEV)),
             (lambda a: ops.distill_loss(a, ids, t), x), (lambda a: ops.distill_loss(x, ids, a), t),
             (lambda a: ops.distill_loss(x, ids, t, 1.0, a), rows)]
    for i, (call, v) in enumerate(calls):
        call(v)
        with fwad.dual_level():
            call(v)  # nothing dual among the arguments
            dual = fwad.make_dual(v, torch.ones_like(v))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises((RuntimeError, NotImplementedError)):
                    call(dual)
        call(v)
