"""Importing the operators leaves autograd's threads as they are; backward passes on the calling thread are a scope."""
import os
import subprocess
import sys
import threading

import pytest
import torch

from dss_vae_amd import ops


def test_the_import_changes_nothing():
    src = "import torch; a = torch._C._is_multithreading_enabled(); import dss_vae_amd.ops, dss_vae_amd.train; print(a, torch._C._is_multithreading_enabled())"
    env = {k: v for k, v in os.environ.items() if k != "DSSVAE_AUTOGRAD_THREADS"}
    out = subprocess.run([sys.executable, "-c", src], env=env, capture_output=True, text=True)
    assert out.stdout.strip() == "True True", out.stderr


def test_the_scope_ends():
    with torch.autograd.set_multithreading_enabled(True):
        seen = []
        with pytest.raises(KeyError):
            with ops.backward_on_caller():
                assert not torch._C._is_multithreading_enabled()
                t = threading.Thread(target=lambda: seen.append(torch._C._is_multithreading_enabled()))
                t.start()
                t.join()
                raise KeyError
        assert torch._C._is_multithreading_enabled() and seen == [True]
        ops.backward_on_caller()  # (entered by `with` alone)
        assert torch._C._is_multithreading_enabled()
    with torch.autograd.set_multithreading_enabled(False):
        with ops.backward_on_caller():
            pass
        assert not torch._C._is_multithreading_enabled()
