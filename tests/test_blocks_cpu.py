"""Sequence-block operators without a GPU: what the C-ABI and the Python entry points refuse before anything is launched, and the
host arithmetic of workspace sizes and plans."""
import ctypes as C

import pytest
import torch

from dss_vae_amd import lib as L
from dss_vae_amd import ops

P = 1 << 20  # an aligned address that is never read
EINVAL, ETOOBIG = -1, -2


def call(name, args, **change):
    """the entry point with `args` (an ordered dict of a valid call), some replaced"""
    a = dict(args)
    for k, v in change.items():
        assert k in a, k
        a[k] = v
    return getattr(L.load(), name)(*a.values())


NORM_FWD = dict(x=P, ldx=8, dtype=0, w=P, b=P, f32=1, rows=4, D=8, eps=1e-5, y=P, ldy=8, stats=P, stream=None)
NORM_BWD = dict(x=P, ldx=8, dtype=1, dy=P, lddy=8, w=P, f32=0, stats=P, rows=4, D=8, dx=P, lddx=8, dw=P, db=P, ws=P, n=1 << 20, stream=None)
SCAN_FWD = dict(x=P, xb=48, xt=16, dtype=0, h0=P, lengths=None, rev=0, tanh=1, B=2, T=3, H=8, out=P, ob=24, ot=8, last=P, ckpt=P, ws=None, n=0,
                stream=None)
SCAN_BWD = dict(x=P, xb=48, xt=16, dtype=0, lengths=None, rev=0, tanh=1, ckpt=P, dout=P, ob=24, ot=8, dlast=P, B=2, T=3, H=8, dx=P, gb=48,
                gt=16, dh0=P, ws=None, n=0, stream=None)
STEP = dict(x=P, xb=16, dtype=0, h=P, tanh=1, B=2, H=8, out=P, ob=8, hout=P, stream=None)
DISTILL = dict(z=P, ldz=9, dtype=1, N=4, V=9, ids=P, teacher=P, k=3, tau=1.0, weight=P, all=0.25, dz=P, lddz=9, rows=P, total=P, stream=None)
SCALE = dict(x=P, ld=9, dtype=0, rows=4, V=9, f=P, stream=None)
LIN_FWD = dict(x=P, ldx=8, w=P, ldw=8, b=P, f32=0, res=P, ldr=16, dtype=1, act=2, M=4, N=16, K=8, y=P + 4096, ldy=16, z=P + 8192, ldz=16,
               ws=P, n=1 << 24, stream=None)
LIN_BWD = dict(dy=P, lddy=16, z=P, ldz=16, x=P, ldx=8, w=P, ldw=8, dtype=1, act=2, M=4, N=16, K=8, dx=P, lddx=8, dw=P, lddw=8, db=P, f32=0,
               ws=P, n=1 << 24, stream=None)


@pytest.mark.parametrize("name,args,bad", [
    ("dssvae_layer_norm_fwd", NORM_FWD, [dict(x=None), dict(y=None), dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(D=0), dict(ldx=7),
                                         dict(ldy=7), dict(eps=-1.0), dict(eps=float("nan"))]),
    ("dssvae_layer_norm_bwd", NORM_BWD, [dict(x=None), dict(dy=None), dict(stats=None), dict(ws=None), dict(n=10), dict(lddx=7), dict(lddy=7),
                                         dict(dtype=9), dict(D=0)]),
    ("dssvae_gated_scan_fwd", SCAN_FWD, [dict(x=None), dict(out=None), dict(dtype=3), dict(H=0), dict(T=-1), dict(B=-1), dict(xt=15),
                                         dict(xb=15), dict(ot=7), dict(ob=7), dict(T=(1 << 30) + 1)]),
    ("dssvae_gated_scan_fwd", dict(SCAN_FWD, T=3000, xb=48000, ob=24000), [dict(), dict(ws=P), dict(ws=P, n=8)]),  # needs a workspace
    ("dssvae_gated_scan_bwd", SCAN_BWD, [dict(x=None), dict(dx=None), dict(ckpt=None), dict(gt=15), dict(gb=15), dict(ot=7), dict(ob=7),
                                         dict(dtype=3)]),
    ("dssvae_gated_step", STEP, [dict(x=None), dict(out=None), dict(hout=None), dict(xb=15), dict(ob=7), dict(H=0), dict(dtype=4)]),
    ("dssvae_distill", DISTILL, [dict(z=None), dict(ids=None), dict(teacher=None), dict(rows=None), dict(total=None), dict(k=0),
                                 dict(k=1025), dict(V=0), dict(ldz=8), dict(lddz=8), dict(tau=0.0), dict(tau=float("inf")),
                                 dict(tau=float("nan")), dict(dtype=3), dict(N=-1), dict(z=P + 1), dict(dz=P + 2), dict(lddz=10)]),
    ("dssvae_scale_rows", SCALE, [dict(x=None), dict(f=None), dict(ld=8), dict(V=0), dict(rows=-1), dict(dtype=5)]),
    ("dssvae_linear_act_fwd", LIN_FWD, [dict(x=None), dict(w=None), dict(y=None), dict(act=5), dict(act=-1), dict(dtype=3), dict(N=0),
                                        dict(K=0), dict(M=-1), dict(ldx=7), dict(ldw=7), dict(ldy=15), dict(ldr=15), dict(ldz=15),
                                        dict(z=P + 4096), dict(M=100, K=9, ldx=9, ldw=9, n=0), dict(M=100, K=9, ldx=9, ldw=9, ws=None),
                                        dict(M=100, K=9, ldx=9, ldw=9, ws=P + 1)]),
    ("dssvae_linear_act_bwd", LIN_BWD, [dict(dy=None), dict(x=None), dict(w=None), dict(z=None), dict(lddy=15), dict(ldz=15), dict(ldx=7),
                                        dict(ldw=7), dict(lddx=7), dict(lddw=7), dict(ws=None), dict(n=100), dict(act=9), dict(dtype=3)]),
])
def test_c_abi_refuses(name, args, bad):
    for change in bad:
        assert call(name, args, **change) == EINVAL, change


def test_summed_axes_have_a_limit():
    big = (1 << 21) + 8
    assert call("dssvae_linear_act_fwd", LIN_FWD, K=big, ldx=big, ldw=big) == ETOOBIG
    assert call("dssvae_linear_act_bwd", LIN_BWD, M=big) == ETOOBIG
    assert call("dssvae_linear_act_bwd", LIN_BWD, N=big, lddy=big, ldz=big) == ETOOBIG


def test_nothing_to_do_is_no_error():
    assert call("dssvae_layer_norm_fwd", NORM_FWD, rows=0, x=None, y=None) == 0
    assert call("dssvae_layer_norm_bwd", NORM_BWD, dx=None, dw=None, db=None, ws=None, n=0) == 0
    assert call("dssvae_gated_scan_fwd", SCAN_FWD, T=0, x=None, out=None) == 0
    assert call("dssvae_gated_scan_bwd", SCAN_BWD, B=0, x=None, dx=None, ckpt=None) == 0
    assert call("dssvae_gated_step", STEP, B=0, x=None, out=None, hout=None) == 0
    assert call("dssvae_scale_rows", SCALE, rows=0, x=None) == 0
    assert call("dssvae_linear_act_fwd", LIN_FWD, M=0, x=None, w=None, y=None) == 0


def test_workspaces():
    lib = L.load()
    assert lib.dssvae_layer_norm_bwd_workspace_bytes(1, 300) == 2 * 300 * 4
    assert lib.dssvae_layer_norm_bwd_workspace_bytes(0, 300) == 2 * 300 * 4
    most = lib.dssvae_layer_norm_bwd_workspace_bytes(1 << 40, 300)
    assert most == lib.dssvae_layer_norm_bwd_workspace_bytes(1 << 20, 300) == 512 * 2 * 300 * 4  # (256 CUs without a GPU)
    assert lib.dssvae_layer_norm_bwd_workspace_bytes(-1, 300) == EINVAL and lib.dssvae_layer_norm_bwd_workspace_bytes(1, 0) == EINVAL
    assert [lib.dssvae_gated_scan_chunks(t) for t in (-1, 0, 1, 128, 129)] == [EINVAL, 0, 1, 1, 2]
    scan = lib.dssvae_gated_scan_workspace_bytes
    assert scan(256, 90, 300, 0) == 0 and scan(2, 256, 64, 1) == 0  # enough blocks; few chunks
    segs = scan(2, 16384, 2048, 1) // (2 * 2 * 2048 * 4)
    assert segs == 8 and scan(1, 300, 8, 0) == 3 * 2 * 8 * 4
    assert scan(0, 300, 8, 0) == 0 and scan(1, 300, 0, 0) == EINVAL and scan(1, 300, 8, 7) == EINVAL
    fwd = lib.dssvae_linear_act_fwd_workspace_bytes
    assert fwd(P, 8192, P, 8192, 1, 8192, 8192, 8192) == 0  # usable as they are, one split
    assert fwd(P, 300, P, 300, 0, 7936, 300, 300) == 0
    packed = fwd(P, 301, P, 301, 1, 7936, 300, 301)
    assert packed == -(-7936 * 304 * 2 // 256) * 256 + -(-300 * 304 * 2 // 256) * 256
    assert fwd(P + 2, 8192, P, 8192, 1, 8192, 8192, 8192) == 8192 * 8192 * 2  # x starts off a granule
    assert fwd(P, 8, P, 8, 1, -1, 8, 8) == EINVAL
    bwd = lib.dssvae_linear_act_bwd_workspace_bytes
    assert bwd(P, 16, 0, 1, 4, 16, 8, 0, 0, 0) == 0
    assert 0 < bwd(P, 16, 1, 1, 4, 16, 8, 1, 0, 0) < bwd(P, 16, 1, 1, 4, 16, 8, 1, 1, 1)
    assert bwd(P, 16, 1, 1, 4, 0, 8, 1, 1, 1) == EINVAL


def test_python_refuses_host_tensors():
    x, w = torch.zeros(4, 8), torch.zeros(3, 8)
    ids = torch.zeros(4, 2, dtype=torch.long)
    for bad in (lambda: ops.layer_norm(x), lambda: ops.gated_scan(x.view(1, 4, 8)), lambda: ops.gated_step(x), lambda: ops.linear_act(x, w),
                lambda: ops.distill_loss(x, ids, torch.zeros(4, 2))):
        with pytest.raises(RuntimeError):
            bad()


def test_backward_runs_on_the_calling_thread():
    """the import's setting, and the way back to torch's default"""
    import os
    import subprocess
    import sys
    src = "import torch; import dss_vae_amd.ops; print(torch._C._is_multithreading_enabled())"
    for value, want in (("0", "False"), ("1", "True")):
        out = subprocess.run([sys.executable, "-c", src], env=dict(os.environ, DSSVAE_AUTOGRAD_THREADS=value), capture_output=True, text=True)
        assert out.stdout.strip() == want, out.stderr
    assert isinstance(L.load().dssvae_distill, C._CFuncPtr)


def test_leaves_of_older_graphs_are_noticed():
    """the stream a leaf was first used on is noted while a graph holds it, and forgotten with the graph"""
    from dss_vae_amd import ops
    a, b = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)
    y = a * b
    assert not ops._leaves_on_null(y.grad_fn, 0)
    z = a * 2
    assert not ops._leaves_on_null(z.grad_fn, 0) and ops._leaves_on_null(z.grad_fn, 8)
    c = b * 3
    del y, z
    fresh = a * 2
    assert not ops._leaves_on_null(fresh.grad_fn, 8)
    assert ops._leaves_on_null(c.grad_fn, 8)
    assert not ops._leaves_on_null(fresh.grad_fn, 9)  # (noted for 8: an ordinary stream may join a capture)
    inner = fresh * 2  # (no leaf right behind it)
    assert not ops._leaves_on_null(inner.grad_fn, 9)


def test_launches_beyond_the_grid_are_refused():
    """2^32 threads or more in a launch: refused before anything is enqueued"""
    big = (1 << 31) - 1
    assert call("dssvae_gated_step", STEP, B=big, H=64, xb=128, ob=64) == ETOOBIG
    assert call("dssvae_gated_scan_fwd", SCAN_FWD, B=big) == ETOOBIG
    assert call("dssvae_linear_act_fwd", LIN_FWD, M=big, N=1 << 20, ldy=1 << 20, res=None, z=None, n=1 << 62) == ETOOBIG


def test_import_in_any_grad_mode():
    import subprocess
    import sys
    for mode in ("torch.inference_mode()", "torch.no_grad()", "torch.device('meta')"):
        src = "import torch\nwith %s:\n    import dss_vae_amd.ops as o\nprint(o._ACCUMULATE.__name__)" % mode
        out = subprocess.run([sys.executable, "-c", src], capture_output=True, text=True)
        assert out.stdout.strip() == "AccumulateGrad", out.stderr
