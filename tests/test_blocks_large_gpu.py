"""The sequence-block operators on tensors of more than 2^31 elements: what lies behind that border gets the same bits as on its
own (or, where the split of a sum depends on the size, the same values within the operator's bound)."""
import math

import pytest
import torch

from blocks_util import DEV, bits, check

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def release():
    yield
    torch.cuda.empty_cache()


def fill(*shape, seed=0):
    t = torch.empty(*shape, device=DEV, dtype=BF)
    return t.normal_(generator=torch.Generator(DEV).manual_seed(seed))


def test_layer_norm():
    from dss_vae_amd import ops
    R, D, n = 1_100_000, 2048, 300
    x, w, dy = fill(R, D).requires_grad_(), fill(D, seed=1).requires_grad_(), fill(R, D, seed=2)
    y = ops.layer_norm(x, w)
    dx, _ = torch.autograd.grad(y, (x, w), dy)
    part = x[-n:].detach().clone().requires_grad_()
    yp = ops.layer_norm(part, w)
    dp, = torch.autograd.grad(yp, part, dy[-n:].contiguous())
    assert torch.equal(bits(y[-n:]), bits(yp)) and torch.equal(bits(dx[-n:]), bits(dp))


def test_gated_scan():
    from dss_vae_amd import ops
    B, T, H, n = 40, 32768, 1024, 16  # (16 sequences fill the chip as 40 do: the time axis is not cut in either)
    x, do = fill(B, T, 2 * H).requires_grad_(), fill(B, T, H, seed=1)
    out, last = ops.gated_scan(x, candidate="tanh")
    dx, = torch.autograd.grad(out, x, do)
    part = x[-n:].detach().requires_grad_()
    op, lp = ops.gated_scan(part, candidate="tanh")
    dp, = torch.autograd.grad(op, part, do[-n:])
    assert torch.equal(bits(out[-n:]), bits(op)) and torch.equal(bits(last[-n:]), bits(lp)) and torch.equal(bits(dx[-n:]), bits(dp))


def test_gated_scan_with_far_strides():
    from dss_vae_amd import ops
    T, H, far = 5, 40, (1 << 30) + 64
    base = torch.empty(4 * far, device=DEV, dtype=BF)
    for shape, stride in (((3, T, 2 * H), (far, 2 * H, 1)), ((2, 3, 2 * H), (96, far, 1))):
        x = base.as_strided(shape, stride)
        near = fill(*shape)
        x.copy_(near)
        for reverse in (False, True):
            a, b = (ops.gated_scan(v.detach().requires_grad_(), reverse=reverse)[0] for v in (x, near))
            assert torch.equal(bits(a.detach()), bits(b.detach()))


def test_distill_loss():
    from dss_vae_amd import ops
    N, V, k, n = 20_000, 131_000, 8, 50
    z = fill(N, V).requires_grad_()
    g = torch.Generator(DEV).manual_seed(3)
    ids, t = torch.randint(0, V, (N, k), device=DEV, generator=g), torch.randn(N, k, device=DEV, generator=g)
    w = torch.full((N,), 0.5, device=DEV)
    total, rows = ops.distill_loss(z, ids, t, 2.0, w)
    dz, = torch.autograd.grad(total, z)
    part = z[-n:].detach().requires_grad_()
    tp, rp = ops.distill_loss(part, ids[-n:], t[-n:], 2.0, w[-n:])
    dp, = torch.autograd.grad(tp, part)
    assert torch.equal(bits(rows[-n:]), bits(rp)) and torch.equal(bits(dz[-n:].contiguous()), bits(dp.contiguous()))
    total = float(total.detach())
    assert abs(total - float((rows.double() * 0.5).sum())) <= 2.0 ** -23 * total


def test_linear_act():
    """dx and y of the last rows, dw over all of them; bounds as in the small cases: 3 sqrt(n) + 8 units of the magnitudes"""
    from dss_vae_amd import ops
    M, K, N, n = 1_100_000, 2048, 64, 200
    x, w, dy = fill(M, K).requires_grad_(), fill(N, K, seed=1).mul_(K ** -0.5).requires_grad_(), fill(M, N, seed=2)
    y = ops.linear_act(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    xd, wd, gd = x[-n:].detach().double(), w.detach().double(), dy[-n:].double()
    check(y[-n:], xd @ wd.t(), xd.abs() @ wd.abs().t(), 3 * math.sqrt(K) + 8, "y")
    check(dx[-n:], gd @ wd, gd.abs() @ wd.abs(), 3 * math.sqrt(N) + 8, "dx")
    want, mag = torch.zeros(N, K, device=DEV, dtype=torch.float64), torch.zeros(N, K, device=DEV, dtype=torch.float64)
    for i in range(0, M, 100_000):
        a, b = dy[i:i + 100_000].double().t().contiguous(), x[i:i + 100_000].detach().double()
        want += a @ b
        mag += a.abs() @ b.abs()
    check(dw, want, mag, 3 * math.sqrt(M) + 8, "dw")
    far = (1 << 30) + 8
    base = torch.empty(3 * far, device=DEV, dtype=BF)
    v = base.as_strided((3, 64), (far, 1))
    v.copy_(fill(3, 64, seed=5))
    w2 = fill(16, 64, seed=6)
    assert torch.equal(bits(ops.linear_act(v, w2)), bits(ops.linear_act(v.contiguous(), w2)))


def test_distill_loss_of_many_rows():
    """more rows than one launch takes"""
    from dss_vae_amd import ops
    N, V, n = (1 << 21) + 700, 24, 1000
    z, ids = fill(N, V).requires_grad_(), torch.randint(0, V, (N, 3), device=DEV)
    t = torch.randn(N, 3, device=DEV)
    w = torch.rand(N, device=DEV) / N
    total, rows = ops.distill_loss(z, ids, t, 2.0, w)
    dz, = torch.autograd.grad(total, z)
    part = z[-n:].detach().requires_grad_()
    tp, rp = ops.distill_loss(part, ids[-n:], t[-n:], 2.0, w[-n:])
    dp, = torch.autograd.grad(tp, part)
    assert torch.equal(bits(rows[-n:]), bits(rp)) and torch.equal(bits(dz[-n:]), bits(dp))
    total, want = float(total.detach()), float((rows.double() * w.double()).sum())
    assert abs(total - want) <= 2.0 ** -23 * want
