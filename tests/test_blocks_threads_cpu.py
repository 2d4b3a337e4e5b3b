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


def enabled():
    return torch._C._is_multithreading_enabled()


@pytest.fixture
def threads_on(monkeypatch):
    """torch's default on this thread, whatever ran before"""
    monkeypatch.setattr(ops, "_AUTOGRAD_THREADS", "")
    with torch.autograd.set_multithreading_enabled(True):
        yield


def test_a_lease_lasts_as_long_as_its_graphs(threads_on):
    a = ops._lease()
    b = ops._lease()
    assert not enabled()
    with torch.autograd.set_multithreading_enabled(True):  # an explicit scope inside
        assert enabled()
    assert not enabled()
    del a
    assert not enabled()
    del b
    assert enabled()
    a = ops._lease()
    assert not enabled()
    del a
    assert enabled()


def test_a_setting_of_the_program_stays(threads_on, monkeypatch):
    with ops.backward_on_caller():
        assert ops._lease() is None and not enabled()
    assert enabled()
    monkeypatch.setattr(ops, "_AUTOGRAD_THREADS", "1")
    assert ops._lease() is None and enabled()
    monkeypatch.setattr(ops, "_AUTOGRAD_THREADS", "")
    monkeypatch.setattr(ops, "_gpus", lambda: 2)
    assert ops._lease() is None and enabled()


def test_threads_are_apart(threads_on):
    """a lease is its thread's: others keep their setting, and one that ends elsewhere gives its thread nothing to wait for"""
    a = ops._lease()
    seen, box = [], []

    def other():
        seen.append(enabled())
        box.append(ops._lease())
        seen.append(enabled())

    t = threading.Thread(target=other)
    t.start()
    t.join()
    assert seen == [True, False] and not enabled()
    del a
    assert enabled()
    box.clear()  # (the other thread's, dropped here)
    assert enabled()
    box.append(ops._lease())
    t = threading.Thread(target=box.clear)
    t.start()
    t.join()
    assert not enabled()  # its thread has not come by since
    b = ops._lease()
    del b
    assert enabled()
