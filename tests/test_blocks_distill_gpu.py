"""ops.distill_loss against its definition in 64 bits: vocabularies of every kernel shape and rows at every alignment, empty and
repeated slots, padded rows, infinities, weights, the upstream factor, graph replay."""
import math

import pytest
import torch

from blocks_util import DEV, TYPES, bits, check, rnd

pytestmark = pytest.mark.gpu


def reference(z, ids, t, tau, w):
    """-> total, rows, dlogits and their fp32 error scales, in 64 bits.  A row without a valid slot (all -inf among it) or of
    weight 0 is 0."""
    z, t, w = z.double() / tau, t.double() / tau, w.double()
    valid = (ids >= 0) & (t > -math.inf)
    t = t.masked_fill(~valid, -math.inf)
    live = valid.any(1) & (w != 0)
    top = torch.where(live, t.amax(1), torch.zeros_like(w)).unsqueeze(1)
    p = torch.exp(t - top)
    p = torch.where(live.unsqueeze(1), p / p.sum(1, keepdim=True).clamp(min=1e-300), torch.zeros_like(p))
    lse = torch.logsumexp(z, 1, keepdim=True)
    zi = z.gather(1, ids.clamp(min=0))
    term = torch.where(p > 0, p * (torch.log(p.clamp(min=1e-300)) - zi + lse), torch.zeros_like(p))
    rows = tau * tau * term.sum(1)
    q = torch.exp(z - lse)
    g = torch.where(live.unsqueeze(1), q.clone(), torch.zeros_like(q)).scatter_add(1, ids.clamp(min=0), -p)
    far = (z - z.amax(1, keepdim=True)).abs().clamp(max=1e4)
    big = torch.where(live.unsqueeze(1), q * (1 + far), torch.zeros_like(q)).scatter_add(1, ids.clamp(min=0), p)
    wt = (w.abs() * tau).unsqueeze(1)
    farp = torch.where(p > 0, (zi - z.amax(1, keepdim=True)).abs(), torch.zeros_like(p))
    rs = tau * tau * ((p * (torch.log(p.clamp(min=1e-300)).abs() + farp)).sum(1) + (lse - z.amax(1, keepdim=True)).squeeze(1) + 1)
    return (w * rows).sum(), rows, g * (w * tau).unsqueeze(1), (w.abs() * rs).sum(), rs, wt * big


# slack: exp2's argument is off by two roundings of |z - max| / tau (in the scale), the hardware's exp2 by 1 ulp, the sum over
# the vocabulary by a chain of at most 128 + 22 (the wide form: 131080 / 1024) of its own magnitude, the quotient and products by 4
SLACK = 160


def case(N, V, k, dtype, seed=0, holes=True):
    g = torch.Generator().manual_seed(seed)
    z = rnd(N, V, seed=seed, scale=2.0, dtype=dtype)
    ids = torch.randint(0, V, (N, k), generator=g)
    if holes:
        ids = ids.masked_fill(torch.rand(N, k, generator=g) < 0.15, -1)
    t = rnd(N, k, seed=seed + 1, scale=2.0, shift=3.0)
    w = torch.rand(N, generator=g) + 0.1
    w[torch.rand(N, generator=g) < 0.2] = 0.0
    return z, ids, t, w


def run(z, ids, t, tau, w, factor=None):
    from dss_vae_amd import ops
    zd = z.to(DEV).requires_grad_()
    total, rows = ops.distill_loss(zd, ids.to(DEV), t.to(DEV), tau, None if w is None else w.to(DEV))
    (total if factor is None else total * factor).backward()
    return total, rows, zd.grad


def compare(z, ids, t, tau, w, got, factor=1.0):
    want = reference(z, ids, t, tau, torch.full((z.size(0),), 1.0 / z.size(0)) if w is None else w)
    check(got[0], want[0], want[3], SLACK, "total")
    check(got[1], want[1], want[4], SLACK, "rows")
    # the gradient is rounded to its type before the factor (a power of two here) is applied: in units of the factor it is
    # within half a step of the unit gradient, also among fp16's subnormal numbers, where the factor spreads the steps
    check(got[2].double() / factor, want[2], want[5], SLACK, "dlogits", dtype=z.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (3, 2, 4), (5, 7, 3), (4, 8, 2), (9, 100, 5), (7, 1001, 8), (4, 2049, 64),
                                   (3, 4097, 33), (3, 16390, 16), (5, 30000, 32), (3, 33001, 8), (2, 65541, 100), (2, 70003, 7),
                                   (2, 131083, 1024)])
def test_forward_and_gradient(dtype, N, V, k):
    for tau in (1.0, 2.5):
        z, ids, t, w = case(N, V, k, dtype, seed=V)
        compare(z, ids, t, tau, w, run(z, ids, t, tau, w))
    z, ids, t, _ = case(N, V, k, dtype, seed=V + 1, holes=False)
    compare(z, ids, t, 1.0, None, run(z, ids, t, 1.0, None))


@pytest.mark.parametrize("dtype", TYPES)
def test_every_alignment_and_leading_shape(dtype):
    from dss_vae_amd import ops
    z, ids, t, w = case(6, 333, 9, dtype, seed=3)
    for off, pad in ((0, 0), (1, 0), (3, 7), (5, 12), (8, 1)):
        wide = torch.full((6, off + 333 + pad), float("nan"), dtype=dtype)
        wide[:, off:off + 333] = z
        leaf = wide.to(DEV).requires_grad_()
        total, rows = ops.distill_loss(leaf[:, off:off + 333], ids.to(DEV), t.to(DEV), 2.0, w.to(DEV))
        g, = torch.autograd.grad(total, leaf)
        assert (g[:, :off] == 0).all() and (g[:, off + 333:] == 0).all()
        compare(z, ids, t, 2.0, w, (total, rows, g[:, off:off + 333]))
    z3 = z.to(DEV).view(2, 3, 333).requires_grad_()
    total, rows = ops.distill_loss(z3, ids.to(DEV).view(2, 3, 9), t.to(DEV).view(2, 3, 9), 2.0, w.to(DEV).view(2, 3))
    total.backward()
    assert rows.shape == (2, 3) and not rows.requires_grad
    compare(z, ids, t, 2.0, w, (total, rows.reshape(6), z3.grad.reshape(6, 333)))
    zt = z.t().contiguous().to(DEV).t()
    assert torch.equal(ops.distill_loss(zt, ids.to(DEV), t.to(DEV))[1], ops.distill_loss(z.to(DEV), ids.to(DEV), t.to(DEV))[1])


def test_rows_that_are_not_read():
    """weight 0, no valid slot, a teacher of -inf: zeros, whatever the logits hold; their neighbours as without them"""
    from dss_vae_amd import ops
    for V in (50, 5000, 70001):
        z, ids, t, w = case(6, V, 4, torch.float32, seed=4, holes=False)
        w = w + 0.5
        clean = run(z, ids, t, 1.0, w)
        zn, idn, tn, wn = z.clone(), ids.clone(), t.clone(), w.clone()
        zn[1], zn[2], zn[4] = float("nan"), float("inf"), float("nan")
        wn[1], idn[2], tn[4] = 0.0, -1, float("-inf")
        got = [o.detach() for o in run(zn, idn, tn, 1.0, wn)]
        for r in (1, 2, 4):
            assert got[1][r] == 0 and (got[2][r] == 0).all()
        for r in (0, 3, 5):
            assert torch.equal(got[1][r], clean[1][r]) and torch.equal(got[2][r], clean[2][r])
        want = sum(float(w[r]) * float(clean[1][r]) for r in (0, 3, 5))
        assert abs(float(got[0]) - want) <= 1e-6 * abs(want)
    total, rows = ops.distill_loss(torch.zeros(0, 9, device=DEV), torch.zeros(0, 2, device=DEV, dtype=torch.long),
                                   torch.zeros(0, 2, device=DEV))
    assert total == 0 and rows.shape == (0,)


def test_repeated_ids_add_up():
    z, _, t, w = case(2, 40, 6, torch.float32, seed=5)
    ids = torch.tensor([[3, 3, 3, 39, 0, 39], [7, 7, 7, 7, 7, 7]])
    w[:] = 1.0
    compare(z, ids, t, 1.5, w, run(z, ids, t, 1.5, w))


def test_infinities_and_errors_show():
    """-inf logits (masked words) are probability 0; a word outside the vocabulary, a NaN or +inf teacher logit and a NaN
    logit make their row NaN, and only theirs"""
    z, ids, t, w = case(7, 600, 4, torch.float32, seed=6, holes=False)
    w[:] = 1.0
    z[:, 100:200] = float("-inf")
    ids = ids % 100
    t[0, 2] = float("-inf")  # probability 0
    compare(z, ids, t, 1.0, w, run(z, ids, t, 1.0, w))
    ids[1, 3] = 600
    t[2, 0] = float("nan")
    z[3, 300] = float("nan")
    t[4, 1] = float("inf")
    ids[5, 0] = 150  # the teacher's mass on a word the student excludes: an infinite loss, a finite gradient
    got = [o.detach() for o in run(z, ids, t, 1.0, w)]
    assert got[1][1:5].isnan().all() and got[2][1:5, :100].isnan().all() and got[1][5] == float("inf")
    assert got[2][5].isfinite().all() and got[2][5, 150] < 0
    assert got[1][[0, 6]].isfinite().all() and got[2][[0, 6]].isfinite().all() and bool(got[0].isnan())


@pytest.mark.parametrize("dtype", TYPES)
def test_upstream_factor(dtype):
    z, ids, t, w = case(5, 777, 6, dtype, seed=7)
    got = run(z, ids, t, 1.0, w, factor=4.0)
    compare(z, ids, t, 1.0, w, got, factor=4.0)
    assert torch.equal(bits(run(z, ids, t, 1.0, w)[2] * 4.0), bits(got[2]))


def test_forward_only_and_one_backward():
    from dss_vae_amd import ops
    z, ids, t, w = (x.to(DEV) for x in case(5, 777, 6, torch.float32, seed=8))
    a = ops.distill_loss(z, ids, t, 1.0, w)
    zg = z.clone().requires_grad_()
    b = ops.distill_loss(zg, ids, t, 1.0, w)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not a[0].requires_grad
    b[0].backward(retain_graph=True)
    with pytest.raises(RuntimeError):
        b[0].backward()
    h = ops.distill_loss(z, ids, t.double().float(), 1.0, w)
    assert torch.equal(a[0], h[0])
    zb = z.bfloat16()
    x, y = ops.distill_loss(zb, ids, t.bfloat16()), ops.distill_loss(zb, ids, t.bfloat16().float())
    assert torch.equal(x[0], y[0])


def test_gradient_against_differences():
    z, ids, t, w = case(2, 12, 3, torch.float32, seed=9)
    w[:] = torch.tensor([0.7, 1.3])
    got = run(z, ids, t, 2.0, w)[2].cpu().double()
    h = 1e-6
    for i in range(2):
        for j in range(12):
            up, down = z.double().clone(), z.double().clone()
            up[i, j] += h
            down[i, j] -= h
            d = (reference(up, ids, t, 2.0, w)[0] - reference(down, ids, t, 2.0, w)[0]) / (2 * h)
            assert abs(float(d) - float(got[i, j])) < 1e-5


def test_same_bits_twice_and_in_a_replayed_graph():
    from dss_vae_amd import ops
    z, ids, t, w = (x.to(DEV) for x in case(40, 5003, 8, torch.bfloat16, seed=10))
    zs = z.clone().requires_grad_()

    def step(a):
        total, rows = ops.distill_loss(a, ids, t, 2.0, w)
        return total, rows, torch.autograd.grad(total, a)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(zs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(zs)
    for n in range(3):
        zs.data.copy_(z * (1 + n))
        want = step(zs.detach().requires_grad_())
        for o in out:
            o.detach().fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(bits(a.detach()), bits(c.detach())), n


def test_refusals():
    from dss_vae_amd import ops
    z, ids, t = torch.zeros(4, 9, device=DEV), torch.zeros(4, 2, device=DEV, dtype=torch.long), torch.zeros(4, 2, device=DEV)
    for bad in (lambda: ops.distill_loss(z.cpu(), ids, t), lambda: ops.distill_loss(z.double(), ids, t),
                lambda: ops.distill_loss(z[0], ids[0], t[0]), lambda: ops.distill_loss(z[:, :0], ids, t),
                lambda: ops.distill_loss(z, ids.int(), t), lambda: ops.distill_loss(z, ids[:3], t[:3]),
                lambda: ops.distill_loss(z, ids, t[:, :1]), lambda: ops.distill_loss(z, ids, t.half()),
                lambda: ops.distill_loss(z, ids[:, :0], t[:, :0]),
                lambda: ops.distill_loss(z, ids.repeat(1, 600), t.repeat(1, 600)), lambda: ops.distill_loss(z, ids.cpu(), t),
                lambda: ops.distill_loss(z, ids, t, 0.0), lambda: ops.distill_loss(z, ids, t, float("inf")),
                lambda: ops.distill_loss(z, ids, t, float("nan")), lambda: ops.distill_loss(z, ids, t, 1.0, torch.ones(3, device=DEV)),
                lambda: ops.distill_loss(z, ids, t, 1.0, torch.ones(4, device=DEV).half()),
                lambda: ops.distill_loss(z, ids, t.clone().requires_grad_()),
                lambda: ops.distill_loss(z, ids, t, 1.0, torch.ones(4, device=DEV, requires_grad=True))):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("granules", [64, 256, 512, 1024, 2048, 4096, 8192, 16384, 24576])
def test_borders_of_the_row_kernels(dtype, granules):
    """rows that just fit the registers (or registers and LDS) of each kernel, and one element more"""
    from dss_vae_amd import ops
    per = 4 if dtype == torch.float32 else 8
    for V in (granules * per, granules * per + 1):
        z, ids, t, w = case(3, V, 9, dtype, seed=V)
        w = w + 0.1
        got = run(z, ids, t, 1.5, w)
        compare(z, ids, t, 1.5, w, got)
        with torch.no_grad():
            total, rows = ops.distill_loss(z.to(DEV), ids.to(DEV), t.to(DEV), 1.5, w.to(DEV))
        want = reference(z, ids, t, 1.5, w)
        check(total, want[0], want[3], SLACK, "total without a gradient")
        check(rows, want[1], want[4], SLACK, "rows without a gradient")
