"""ops.distill_loss under an upstream gradient that is not 1 (a loss scale, a mixing weight, a quotient of accumulation): the factor is
applied before the gradient's one rounding."""
import pytest
import torch

from blocks_util import DEV, TYPES, bits, check, rnd
from test_blocks_distill_gpu import SLACK, case, reference

pytestmark = pytest.mark.gpu
# factor and the products behind it: three roundings more
MORE = SLACK + 3


def gradient(z, ids, t, tau, w, factor):
    from dss_vae_amd import ops
    zd = z.to(DEV).requires_grad_()
    total, _ = ops.distill_loss(zd, ids.to(DEV), t.to(DEV), tau, None if w is None else w.to(DEV))
    return torch.autograd.grad(total * factor, zd)[0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factor", [65536.0, 3.0, 0.3, -1.7, 1.0, 0.0])
def test_rounded_once(dtype, factor):
    """default weights 1 / rows over a whole vocabulary: the unit gradient of a word is of the order of 1e-7, below fp16's smallest number"""
    for N, V, k in ((300, 30000, 16), (5, 777, 6), (4, 70003, 9), (3, 140001, 5), (7, 33, 3)):
        z, ids, t, _ = case(N, V, k, dtype, seed=V)
        want = reference(z, ids, t, 2.0, torch.full((N,), 1.0 / N))
        got = gradient(z, ids, t, 2.0, None, factor)
        check(got, want[2] * factor, want[5] * abs(factor), MORE, (factor, N, V))
        if dtype == torch.float16 and factor == 65536.0 and N == 300:
            assert float((got == 0).float().mean()) < 0.01  # (unscaled, nearly all of them are)


def test_a_unit_gradient_beyond_the_type():
    """fp16: weights whose unit gradient overflows, under a factor that brings it back"""
    z, ids, t, w = case(6, 500, 4, torch.float16, seed=3, holes=False)
    w = (w + 0.1) * 1e6
    want = reference(z, ids, t, 1.0, w)
    got = gradient(z, ids, t, 1.0, w, 2.0 ** -10)
    assert got.isfinite().all()
    check(got, want[2] * 2.0 ** -10, want[5] * 2.0 ** -10, MORE, "small factor")


@pytest.mark.parametrize("dtype", TYPES)
def test_alignment_shapes_and_rows_that_are_not_read(dtype):
    from dss_vae_amd import ops
    z, ids, t, w = case(6, 333, 9, dtype, seed=5)
    w[1], ids[2] = 0.0, -1
    want = reference(z, ids, t, 2.0, w)
    for off, pad in ((0, 0), (1, 0), (3, 7), (8, 1)):
        wide = torch.full((6, off + 333 + pad), float("nan"), dtype=dtype)
        wide[:, off:off + 333] = z
        leaf = wide.to(DEV).requires_grad_()
        total, _ = ops.distill_loss(leaf[:, off:off + 333], ids.to(DEV), t.to(DEV), 2.0, w.to(DEV))
        g, = torch.autograd.grad(total / 3, leaf)
        assert (g[:, :off] == 0).all() and (g[:, off + 333:] == 0).all()
        check(g[:, off:off + 333], want[2] / 3, want[5] / 3, MORE, (off, pad))
    zn = z.clone()
    zn[1], zn[2] = float("nan"), float("inf")
    g = gradient(zn, ids, t, 2.0, w, float("inf"))
    assert (g[1:3] == 0).all()
    z3 = z.to(DEV).view(2, 3, 333).requires_grad_()
    total, _ = ops.distill_loss(z3, ids.to(DEV).view(2, 3, 9), t.to(DEV).view(2, 3, 9), 2.0, w.to(DEV).view(2, 3))
    (0.3 * total).backward()
    check(z3.grad.reshape(6, 333), want[2] * 0.3, want[5] * 0.3, MORE, "three axes")


def test_logits_that_changed_in_between_are_noticed():
    """what backward reads again is guarded as any saved tensor is"""
    from dss_vae_amd import ops
    z, ids, t, w = (v.to(DEV) for v in case(5, 100, 4, torch.float32, seed=6))
    for which in range(3):
        leaf = z.clone().requires_grad_()
        logits, i2, w2 = leaf * 1, ids.clone(), w.clone()
        total, _ = ops.distill_loss(logits, i2, t, 1.0, w2)
        with torch.no_grad():
            (logits, i2, w2)[which].zero_()
        with pytest.raises(RuntimeError):
            (total * 2).backward()


def test_replayed_with_factors_that_change():
    """a captured step whose loss scale lives on the device: 1 takes the gradient of the forward pass, others form it anew, replay by replay"""
    from dss_vae_amd import ops
    z, ids, t, w = (v.to(DEV) for v in case(40, 5003, 8, torch.float16, seed=7))
    zs, f = z.clone().requires_grad_(), torch.ones((), device=DEV)

    def step(a):
        total, _ = ops.distill_loss(a, ids, t, 2.0, w)
        return torch.autograd.grad(total, a, f)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(zs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(zs)
    seen = []
    for n, factor in enumerate((1.0, 1024.0, 0.3, 1.0)):
        f.fill_(factor)
        zs.data.copy_(z * (1 + n % 2))
        want = step(zs.detach().requires_grad_())
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(out), bits(want)), factor
        seen.append(out.clone())
    assert not torch.equal(seen[0], seen[1])


def test_saved_logits_that_come_back_at_another_place():
    """hooks on saved tensors may hand back a copy whose rows start elsewhere"""
    from dss_vae_amd import ops
    z, ids, t, w = case(6, 333, 9, torch.bfloat16, seed=8)
    leaf = torch.cat((torch.zeros(6, 3, dtype=torch.bfloat16), z), 1).to(DEV).requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s.cpu(), lambda s: s.to(DEV)):
        total, _ = ops.distill_loss(leaf[:, 3:], ids.to(DEV), t.to(DEV), 2.0, w.to(DEV))
        same, _ = ops.distill_loss(leaf[:, 3:], ids.to(DEV), t.to(DEV), 2.0, w.to(DEV))
    want = reference(z, ids, t, 2.0, w)
    g, = torch.autograd.grad(total * 3, leaf)
    check(g[:, 3:], want[2] * 3, want[5] * 3, MORE, "three times")
    g, = torch.autograd.grad(same, leaf)
    check(g[:, 3:], want[2], want[5], MORE, "once")


def test_refusals_of_the_second_pass():
    import dss_vae_amd.lib as L
    P = 1 << 20
    good = [P, 9, 1, 4, 9, P, P, 3, 1.0, P, 0.25, P, P, 9, None]
    for i, v in ((0, None), (1, 8), (2, 3), (3, -1), (4, 0), (5, None), (6, None), (7, 0), (8, 0.0), (11, None), (12, None), (12, P + 2), (13, 8), (13, 10)):
        bad = list(good)
        bad[i] = v
        assert L.load().dssvae_distill_again(*bad) == -1, (i, v)


def test_a_teacher_in_inference_mode():
    from dss_vae_amd import ops
    z, ids, t, w = case(6, 333, 9, torch.float32, seed=9)
    want = reference(z, ids, t, 2.0, w)
    with torch.inference_mode():
        ids, t, w = ids.to(DEV), t.to(DEV), w.to(DEV)
    leaf = z.to(DEV).requires_grad_()
    total, _ = ops.distill_loss(leaf, ids, t, 2.0, w)
    g, = torch.autograd.grad(total * 3, leaf)
    check(g, want[2] * 3, want[5] * 3, MORE, "inference mode")
