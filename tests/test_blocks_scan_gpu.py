"""ops.gated_scan / gated_step against a step-by-step recurrence in 64 bits: both directions, padded batches (empty and full
rows), both candidates, lengths around the chunk and segment borders, strides, graph replay."""
import pytest
import torch

from blocks_util import DEV, TYPES, bits, check, rnd

pytestmark = pytest.mark.gpu


def reference(x, h0, lengths, reverse, candidate, dout=None, dh=None):
    """-> out, h_last, dx, dh0 in 64 bits (gradients by automatic differentiation of the recurrence)"""
    B, T, H2 = x.shape
    H = H2 // 2
    x = x.double().requires_grad_()
    h0 = (torch.zeros(B, H) if h0 is None else h0).double().requires_grad_()
    lengths = torch.full((B,), T) if lengths is None else lengths
    h, outs = h0, [None] * T
    for t in (range(T - 1, -1, -1) if reverse else range(T)):
        a = torch.sigmoid(x[:, t, :H])
        n = torch.tanh(x[:, t, H:]) if candidate == "tanh" else x[:, t, H:]
        live = (t < lengths).unsqueeze(1)
        h = torch.where(live, a * h + (1 - a) * n, h)
        outs[t] = torch.where(live, h, torch.zeros_like(h))
    out = torch.stack(outs, 1) if T else torch.zeros(B, 0, H, dtype=torch.float64)
    if dout is None and dh is None:
        return out.detach(), h.detach(), None, None
    s = (out * dout.double()).sum() if dout is not None else 0.0
    s = s + ((h * dh.double()).sum() if dh is not None else 0.0)
    dx, dh0 = torch.autograd.grad(s, (x, h0), allow_unused=True)
    return out.detach(), h.detach(), dx, dh0


def inputs(B, T, H, dtype, seed=0):
    x = rnd(B, T, 2 * H, seed=seed, scale=1.5)
    x[..., :H] += 1.0
    return x.to(dtype), rnd(B, H, seed=seed + 1), rnd(B, T, H, seed=seed + 2, dtype=dtype), rnd(B, H, seed=seed + 3)


# Slack.  The gates have hardware exp2 / rcp (1 ulp each) behind an argument rounding: |da| <= a (1 - a) |z| 2^-24 + 3 ulp,
# below 8 units of 2^-24 for the |z| < 12 here; n likewise below 8 (max(1, |v|)).  A step adds a' error of at most
# (8 + 2) units times the magnitude (1 - a)(|h| + |n|) that the gate blends and the next steps damp it by a: the sum stays
# within a constant times the largest |h| and |n| of the row: 10 / (1 - a) * (1 - a) * 2 = 20 units of max(|h|, |n|), and the
# composition of the maps (a product per step, at most log2(128) + 8 levels deep) adds no more than 16.  Gradients multiply
# two such errors' operands: twice that, times the magnitude of D, which is at most sum |dout| damped: its own scale.
SLACK = 64


def scales(x, h0, dout, dh, lengths, reverse, candidate):
    """magnitudes the recurrence blends: per (sequence, channel) the largest |h| and |n|, and the damped sum of |dout|"""
    H = x.size(2) // 2
    n = x[..., H:].double()
    n = torch.tanh(n).abs() if candidate == "tanh" else n.abs()
    top = n.amax(1) if x.size(1) else torch.zeros(x.size(0), H, dtype=torch.float64)
    top = torch.maximum(top, h0.double().abs() if h0 is not None else torch.zeros_like(top)).clamp(min=1e-3)
    if dout is None and dh is None:
        return top, None
    d = torch.zeros_like(top) if dh is None else dh.double().abs()
    B, T = x.shape[:2]
    a = torch.sigmoid(x[..., :H].double())
    g, worst = d, d.clone()
    for t in (range(T) if reverse else range(T - 1, -1, -1)):
        live = (t < lengths).unsqueeze(1) if lengths is not None else True
        D = g + (0 if dout is None else dout[:, t].double().abs())
        worst = torch.where(torch.as_tensor(live), torch.maximum(worst, D), worst)
        g = torch.where(torch.as_tensor(live), a[:, t] * D, g)
    return top, worst


def compare(x, h0, lengths, reverse, candidate, dout, dh, got):
    want = reference(x, h0, lengths, reverse, candidate, dout, dh)
    top, D = scales(x, h0, dout, dh, lengths, reverse, candidate)
    check(got[0], want[0], top.unsqueeze(1), SLACK, "out")
    check(got[1], want[1], top, SLACK, "h_last")
    if len(got) > 2 and want[2] is not None:
        check(got[2], want[2], torch.cat((D * top, D), 1).unsqueeze(1) * 2, SLACK, "dx")
        if got[3] is not None:
            check(got[3], want[3], D, 2 * SLACK, "dh0")


def run(x, h0, lengths, reverse, candidate, dout, dh):
    from dss_vae_amd import ops
    xd = x.to(DEV).requires_grad_()
    hd = None if h0 is None else h0.to(DEV).requires_grad_()
    out, h = ops.gated_scan(xd, hd, None if lengths is None else lengths.to(DEV), reverse, candidate)
    outs = [o for o, g in ((out, dout), (h, dh)) if g is not None]
    grads = [g.to(DEV) for g in (dout, dh) if g is not None]
    got = torch.autograd.grad(outs, [xd] + ([] if hd is None else [hd]), grads)
    return [out, h, got[0], got[1] if hd is not None else None]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,H", [(1, 1, 1), (3, 2, 5), (2, 7, 16), (1, 127, 20), (2, 128, 9), (1, 129, 64), (2, 300, 33),
                                   (40, 90, 150), (1, 1030, 300), (2, 520, 34), (600, 3, 300)])
@pytest.mark.parametrize("reverse", [False, True])
def test_forward_and_gradients(dtype, B, T, H, reverse):
    candidate = "tanh" if H % 2 else "linear"
    x, h0, dout, dh = inputs(B, T, H, dtype, seed=B + T + H)
    compare(x, h0, None, reverse, candidate, dout, dh, run(x, h0, None, reverse, candidate, dout, dh))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("candidate", ["tanh", "linear"])
@pytest.mark.parametrize("T,H", [(37, 24), (390, 40), (260, 7)])
def test_padded_batch(dtype, reverse, candidate, T, H):
    """lengths from none to all, values outside the range clamped, NaN in the padding of x and dout"""
    x, h0, dout, dh = inputs(9, T, H, dtype, seed=T)
    lengths = torch.tensor([0, 1, T, T - 1, T // 2, T + 5, -3, min(T, 128), min(T, 129)], dtype=torch.int32)
    clean = lengths.clamp(0, T)
    xn, dn = x.clone(), dout.clone()
    for b in range(9):
        xn[b, clean[b]:] = float("nan")
        dn[b, clean[b]:] = float("nan")
        x[b, clean[b]:] = 0
        dout[b, clean[b]:] = 0
    got = run(xn, h0, lengths, reverse, candidate, dn, dh)
    compare(x, h0, clean, reverse, candidate, dout, dh, got)
    for b in range(9):
        assert (got[0][b, clean[b]:] == 0).all() and (got[2][b, clean[b]:] == 0).all()
    assert torch.equal(got[1][0].cpu(), h0[0]) and torch.equal(got[3][0].cpu(), dh[0])


def test_long_sequences_are_cut_in_segments():
    """few channels, many steps: the form with segment maps"""
    from dss_vae_amd import lib
    for T, H, dtype, lengths in ((5000, 8, torch.float32, None), (3001, 100, torch.bfloat16, [3001, 1500]),
                                 (2049, 3, torch.float16, [0, 2000])):
        assert lib.load().dssvae_gated_scan_workspace_bytes(2, T, H, lib.DTYPES[dtype]) > 0
        x, h0, dout, dh = inputs(2, T, H, dtype, seed=T)
        lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
        for reverse in (False, True):
            compare(x, h0, lengths, reverse, "tanh", dout, dh, run(x, h0, lengths, reverse, "tanh", dout, dh))


def test_saturated_gates():
    """gates at 0 and 1 exactly (infinite logits), huge candidates"""
    x, h0, dout, dh = inputs(2, 140, 8, torch.float32, seed=5)
    x[:, 3, :8], x[:, 50, :8], x[:, 100, 8:], x[:, 130, 8:] = float("inf"), float("-inf"), 60.0, -90.0
    compare(x, h0, None, False, "tanh", dout, dh, run(x, h0, None, False, "tanh", dout, dh))


@pytest.mark.parametrize("which", ["out", "h_last"])
def test_one_gradient_missing_and_no_state(which):
    x, _, dout, dh = inputs(3, 150, 20, torch.float32, seed=6)
    dout, dh = (dout, None) if which == "out" else (None, dh)
    compare(x, None, None, False, "tanh", dout, dh, run(x, None, None, False, "tanh", dout, dh))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    """time-major storage, a slice of a wider projection at odd offsets, an expanded batch: the same bits as the copies or,
    where another granule is taken, the reference"""
    from dss_vae_amd import ops
    x, h0, dout, dh = inputs(4, 70, 24, dtype, seed=7)
    tm = x.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    assert tm.stride(0) < tm.stride(1)
    a, b = ops.gated_scan(tm, h0.to(DEV)), ops.gated_scan(x.to(DEV), h0.to(DEV))
    assert torch.equal(bits(a[0]), bits(b[0])) and torch.equal(a[1], b[1])
    for off in (1, 4, 8):
        wide = torch.zeros(4, 70, 64, dtype=dtype)
        wide[:, :, off:off + 48] = x
        compare(x, h0, None, False, "tanh", None, None, ops.gated_scan(wide.to(DEV)[:, :, off:off + 48], h0.to(DEV)))
    e = x[:1].to(DEV).expand(4, 70, 48)
    a, b = ops.gated_scan(e), ops.gated_scan(e.contiguous())
    assert torch.equal(bits(a[0]), bits(b[0]))
    xe = x.to(DEV).requires_grad_()
    ops.gated_scan(xe, h0.to(DEV))[0].sum().backward()  # an expanded scalar as the upstream gradient
    ones = torch.ones(4, 70, 24, dtype=dtype)
    want = reference(x, h0, None, False, "tanh", ones, None)
    top, D = scales(x, h0, ones, None, None, False, "tanh")
    check(xe.grad, want[2], torch.cat((D * top, D), 1).unsqueeze(1) * 2, SLACK)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,H", [(1, 1), (3, 7), (50, 300), (50, 1024), (2000, 36)])
@pytest.mark.parametrize("candidate", ["tanh", "linear"])
def test_step(dtype, B, H, candidate):
    """a token at a time gives what the whole scan gives; the state buffer may be updated in place"""
    from dss_vae_amd import ops
    x, h0, _, _ = inputs(B, 4, H, dtype, seed=B)
    want = reference(x, h0, None, False, candidate)
    top, _ = scales(x, h0, None, None, None, False, candidate)
    xd, h = x.to(DEV), h0.to(DEV)
    state = h.clone()
    for t in range(4):
        out, h = ops.gated_step(xd[:, t], h, candidate)
        out2, state2 = ops.gated_step(xd[:, t], state, candidate, h_out=state)
        assert state2 is state and torch.equal(state, h) and torch.equal(bits(out), bits(out2))
        check(out, want[0][:, t], top, SLACK, t)
    check(h, want[1], top, SLACK)
    first, _ = ops.gated_step(xd[:, 0], None, candidate)
    check(first, reference(x[:, :1], None, None, False, candidate)[0][:, 0], top, SLACK)
    xg = xd[:, 0].detach().requires_grad_()
    out, hn = ops.gated_step(xg, h0.to(DEV), candidate)
    (out.float().sum() + hn.sum()).backward()
    assert xg.grad.shape == xg.shape and bool(xg.grad.isfinite().all())


def test_empty():
    from dss_vae_amd import ops
    h0 = rnd(3, 8).to(DEV).requires_grad_()
    out, h = ops.gated_scan(torch.zeros(3, 0, 16, device=DEV), h0)
    assert out.shape == (3, 0, 8) and torch.equal(h, h0)
    h.sum().backward()
    assert torch.equal(h0.grad, torch.ones_like(h0))
    out, h = ops.gated_scan(torch.zeros(0, 5, 16, device=DEV))
    assert out.shape == (0, 5, 8) and h.shape == (0, 8)
    assert ops.gated_step(torch.zeros(0, 16, device=DEV))[0].shape == (0, 8)


def test_gradient_against_differences():
    x, h0, dout, dh = inputs(1, 6, 3, torch.float32, seed=8)
    got = run(x, h0, None, False, "tanh", dout, dh)
    f = lambda t: sum((a * b.double()).sum() for a, b in zip(reference(t, h0.double(), None, False, "tanh")[:2], (dout, dh)))  # noqa: E731
    h = 1e-6
    for i in range(x.numel()):
        up, down = x.double().clone(), x.double().clone()
        up.view(-1)[i] += h
        down.view(-1)[i] -= h
        assert abs(float((f(up) - f(down)) / (2 * h)) - float(got[2].reshape(-1)[i])) < 1e-4


def test_same_bits_twice_and_in_a_replayed_graph():
    from dss_vae_amd import ops
    x, h0, dout, dh = (t.to(DEV) for t in inputs(2, 3000, 40, torch.bfloat16, seed=9))
    xs, hs = x.clone().requires_grad_(), h0.clone().requires_grad_()

    def step(a, b):
        o = ops.gated_scan(a, b)
        return o + torch.autograd.grad(o, (a, b), (dout, dh))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = step(xs, hs)
        del warm
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xs, hs)
    for k in range(3):
        xs.data.copy_(x * (1 + 0.25 * k))
        want = step(xs.detach().requires_grad_(), h0.clone().requires_grad_())
        for o in out:
            o.detach().fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(bits(a.detach()), bits(c.detach())), k


def test_refusals():
    from dss_vae_amd import ops
    x, h = torch.zeros(2, 3, 8, device=DEV), torch.zeros(2, 4, device=DEV)
    for bad in (lambda: ops.gated_scan(x.cpu()), lambda: ops.gated_scan(x.double()), lambda: ops.gated_scan(x[0]),
                lambda: ops.gated_scan(x[..., :7]), lambda: ops.gated_scan(x[..., :0]), lambda: ops.gated_scan(x, h[:1]),
                lambda: ops.gated_scan(x, h.half()), lambda: ops.gated_scan(x, h.cpu()), lambda: ops.gated_scan(x, candidate="relu"),
                lambda: ops.gated_scan(x, h, torch.zeros(2, device=DEV)),
                lambda: ops.gated_scan(x, h, torch.zeros(3, device=DEV, dtype=torch.int32)),
                lambda: ops.gated_scan(x, h, torch.zeros(2, dtype=torch.int32)), lambda: ops.gated_step(x),
                lambda: ops.gated_step(x[:, 0], h[:1]), lambda: ops.gated_step(x[:, 0], h, h_out=h.half()),
                lambda: ops.gated_step(x[:, 0], h, h_out=torch.zeros(4, 2, device=DEV).t()),
                lambda: ops.gated_step(x[:, 0].clone().requires_grad_(), h, h_out=h)):
        with pytest.raises(RuntimeError):
            bad()


def test_step_refuses_overlapping_buffers():
    from dss_vae_amd import ops
    buf = torch.zeros(100, device=DEV)
    h = buf[:8].view(2, 4)
    x = torch.ones(2, 8, device=DEV)
    for h_out in (buf[4:12].view(2, 4), buf[7:15].view(2, 4)):
        with pytest.raises(RuntimeError, match="h_out overlaps h"):
            ops.gated_step(x, h, h_out=h_out)
    with pytest.raises(RuntimeError, match="h_out overlaps xproj"):
        ops.gated_step(buf[16:32].view(2, 8), h, h_out=buf[30:38].view(2, 4))
    with pytest.raises(RuntimeError, match="h_out overlaps h"):  # (a transposed view of the same memory)
        ops.gated_step(x, buf[:8].view(4, 2).t(), h_out=buf[1:9].view(2, 4))
    want = ops.gated_step(x, h)[1].clone()
    assert torch.equal(ops.gated_step(x, h, h_out=buf[8:16].view(2, 4))[1], want)
    ops.gated_step(x, h, h_out=h)
    assert torch.equal(h, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [31, 32, 33, 63, 64, 65])
def test_sequences_of_part_of_a_chunk(dtype, T):
    """blocks of a quarter, half and the whole of a chunk's threads, on both sides of their borders"""
    for H, reverse, candidate in ((35, False, "tanh"), (64, True, "linear")):
        x, h0, dout, dh = inputs(5, T, H, dtype, seed=T + H)
        lengths = torch.tensor([T, 0, 1, T - 1, T // 2], dtype=torch.int32)
        compare(x, h0, lengths, reverse, candidate, dout, dh, run(x, h0, lengths, reverse, candidate, dout, dh))
