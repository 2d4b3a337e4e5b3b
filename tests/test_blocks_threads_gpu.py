"""The operators' graphs hold autograd's threads off for the thread that recorded them, and for no longer than they live."""
import threading

import pytest
import torch

from blocks_util import DEV, rnd

pytestmark = pytest.mark.gpu


def enabled():
    return torch._C._is_multithreading_enabled()


def test_graphs_and_the_setting(monkeypatch):
    from dss_vae_amd import ops
    monkeypatch.setattr(ops, "_AUTOGRAD_THREADS", "")
    x, w = rnd(2, 5, 8, seed=1).to(DEV).requires_grad_(), rnd(8, 8, seed=2).to(DEV).requires_grad_()
    ids, t = torch.zeros(2, 5, 1, dtype=torch.long, device=DEV), torch.zeros(2, 5, 1, device=DEV)
    calls = [lambda: ops.layer_norm(x).sum(), lambda: ops.gated_scan(x)[0].sum(), lambda: ops.gated_step(x[:, 0])[1].sum(),
             lambda: ops.linear_act(x, w, None, "gelu").sum(), lambda: ops.distill_loss(x, ids, t)[0]]
    with torch.autograd.set_multithreading_enabled(True):
        for i, call in enumerate(calls):
            with torch.no_grad():
                call()
                assert enabled(), i
            y = call()
            assert not enabled(), i
            seen = []
            first, = torch.autograd.grad(y, x)
            other = threading.Thread(target=lambda: seen.append(enabled()))
            other.start()
            other.join()
            assert seen == [True] and not enabled(), i
            del y
            assert enabled(), i
            y = call()
            with torch.autograd.set_multithreading_enabled(True):  # backward on autograd's own thread
                again, = torch.autograd.grad(y, x)
            assert torch.equal(first, again), i
            del y
            call()
            assert enabled(), i


def test_an_operator_that_fails_keeps_nothing(monkeypatch):
    from dss_vae_amd import ops
    monkeypatch.setattr(ops, "_AUTOGRAD_THREADS", "")
    x = rnd(2, 8, seed=1).to(DEV).requires_grad_()
    with torch.autograd.set_multithreading_enabled(True):
        with pytest.raises(RuntimeError):
            ops.linear_act(x, torch.zeros(3, (1 << 21) + 8, device=DEV)[:, :8], torch.zeros(2, device=DEV))
        monkeypatch.setattr(ops, "_layer_norm_fwd", lambda *a: (_ for _ in ()).throw(RuntimeError("stop")))
        with pytest.raises(RuntimeError, match="stop"):
            ops.layer_norm(x)
        assert enabled()
