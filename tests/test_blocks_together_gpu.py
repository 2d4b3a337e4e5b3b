"""The sequence-block operators as they are used together: a pre-normalised residual block around a gated scan, its vocabulary
projection and the distillation loss that trains it, in fp32 with the framework's optimiser and in bf16; the same weights token by
token; profiling spans; use from another stream."""
import math

import pytest
import torch
import torch.nn as nn

from blocks_util import DEV, rnd

pytestmark = pytest.mark.gpu
B, T, D, H, V, K = 6, 37, 40, 56, 203, 5


class Student(nn.Module):
    """logits of a one-block student; the weight w is used by two layers"""

    def __init__(self, dtype=torch.float32):
        super().__init__()
        shapes = {"g": (D,), "c": (D,), "wi": (2 * H, D), "bi": (2 * H,), "wo": (D, H), "bo": (D,), "w": (D, D), "b": (D,), "wv": (V, D),
                  "bv": (V,)}
        for i, (n, s) in enumerate(shapes.items()):
            t = rnd(*s, seed=40 + i, scale=0.2 if len(s) == 1 else s[1] ** -0.5) + (1.0 if n == "g" else 0.0)
            self.register_parameter(n, nn.Parameter(t.to(dtype)))

    def block(self, ops, x, lengths):
        n = ops.layer_norm(x, self.g, self.c)
        s, _ = ops.gated_scan(ops.linear_act(n, self.wi, self.bi), None, lengths)
        return ops.linear_act(s, self.wo, self.bo, "none", x)

    def logits(self, ops, x, lengths):
        y = self.block(ops, x, lengths)
        y = ops.linear_act(y, self.w, self.b, "gelu", y)
        y = ops.linear_act(y, self.w, self.b, "silu", y)  # the same weight again: its gradients add up
        return ops.linear_act(y, self.wv, self.bv)


class Plain(object):
    """the operators' definitions, for autograd in any float type on the CPU"""

    @staticmethod
    def layer_norm(x, g, c):
        m = x.mean(-1, keepdim=True)
        return (x - m) / torch.sqrt((x - m).square().mean(-1, keepdim=True) + 1e-5) * g + c

    @staticmethod
    def linear_act(x, w, b, act="none", residual=None):
        z = x @ w.t() + b
        y = {"none": lambda: z, "gelu": lambda: 0.5 * z * torch.erfc(-z / math.sqrt(2.0)), "silu": lambda: z * torch.sigmoid(z)}[act]()
        return y if residual is None else y + residual

    @staticmethod
    def gated_scan(x, h0, lengths):
        h, outs = torch.zeros(x.size(0), x.size(2) // 2, dtype=x.dtype), []
        for t in range(x.size(1)):
            a, n = torch.sigmoid(x[:, t, :h.size(1)]), torch.tanh(x[:, t, h.size(1):])
            live = (t < lengths).unsqueeze(1)
            h = torch.where(live, a * h + (1 - a) * n, h)
            outs.append(torch.where(live, h, torch.zeros_like(h)))
        return torch.stack(outs, 1), h

    @staticmethod
    def distill_loss(z, ids, t, tau, w):
        t = (t.to(z.dtype) / tau).masked_fill(ids < 0, -math.inf)
        p = torch.softmax(t, -1)
        logq = torch.log_softmax(z / tau, -1).gather(-1, ids.clamp(min=0))
        rows = tau * tau * torch.where(p > 0, p * (torch.log(p.clamp(min=1e-30)) - logq), torch.zeros_like(p)).sum(-1)
        return (rows * w.to(z.dtype)).sum(), rows


def data():
    x = rnd(B, T, D, seed=60)
    lengths = torch.tensor([T, 1, 17, 30, 0, T], dtype=torch.int32)
    g = torch.Generator().manual_seed(61)
    ids = torch.randint(0, V, (B, T, K), generator=g)
    ids[:, :, 3:] = ids[:, :, 3:].masked_fill(torch.rand(B, T, K - 3, generator=g) < 0.3, -1)
    w = (torch.arange(T).unsqueeze(0) < lengths.unsqueeze(1)).float()
    return x, lengths, ids, rnd(B, T, K, seed=62, scale=2.0), w / w.sum()


def wanted(dtype):
    """loss, logits and gradients of the same (rounded) weights and inputs in 64 bits"""
    m = Student(dtype).double()
    x, lengths, ids, t, w = data()
    x = x.to(dtype).double().requires_grad_()
    z = m.logits(Plain, x, lengths)
    loss, _ = Plain.distill_loss(z, ids, t, 2.0, w)
    loss.backward()
    return loss.detach(), z.detach(), dict([(n, p.grad) for n, p in m.named_parameters()] + [("x", x.grad)])


def near(a, b, tol, what):
    """each operator is held to its own bound elsewhere; here a mistake in how they are joined would show as a difference of the
    size of the values"""
    a, b = a.detach().cpu().double(), b.double()
    assert a.shape == b.shape and float((a - b).norm()) <= tol * float(b.norm()), (what, float((a - b).norm() / b.norm()))


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 4e-2), (torch.float16, 5e-3)])
def test_a_students_loss_and_gradients(dtype, tol):
    from dss_vae_amd import ops
    loss, z, grads = wanted(dtype)
    m = Student(dtype).to(DEV)
    x, lengths, ids, t, w = (v.to(DEV) for v in data())
    x = x.to(dtype).requires_grad_()
    got_z = m.logits(ops, x, lengths)
    # (fp16 needs a loss scale, as in training: a power of two, taken out again)
    scale = 4096.0 if dtype == torch.float16 else 1.0
    total, rows = ops.distill_loss(got_z, ids, t, 2.0, w * scale)
    total.backward()
    live = (torch.arange(T).unsqueeze(0) < data()[1].unsqueeze(1)).to(DEV)
    assert (rows[~live] == 0).all()
    near(got_z, z, tol, "logits")
    near(total.reshape(1) / scale, loss.reshape(1), tol, "loss")
    for n, g in grads.items():
        near((x.grad if n == "x" else getattr(m, n).grad) / scale, g, tol, n)


def test_with_the_flat_optimiser():
    """gradients land in the optimiser's flat buffer (the twice-used weight's are summed there) and a step moves every weight"""
    from dss_vae_amd import ops
    from dss_vae_amd.train import FlatAdam
    _, _, grads = wanted(torch.float32)
    m = Student().to(DEV)
    opt = FlatAdam(m, lr=1e-3, clip_grad=5.0)
    x, lengths, ids, t, w = (v.to(DEV) for v in data())
    for _ in range(2):
        opt.zero_grad()
        before = {n: p.detach().clone() for n, p in m.named_parameters()}
        ops.distill_loss(m.logits(ops, x, lengths), ids, t, 2.0, w)[0].backward()
        if not opt.t:
            for n, p in m.named_parameters():
                near(p.grad, grads[n], 1e-5, n)
                assert p.grad.data_ptr() in {v.data_ptr() for v in opt.views}
            assert opt.adopted >= 8  # all but the weight and bias that two layers share
        opt.step()
        assert all(not torch.equal(before[n], p) for n, p in m.named_parameters())
    ops.GRAD_SINK = None


def test_token_by_token():
    """serving: one position at a time through the same operators gives the whole sequence's outputs"""
    from dss_vae_amd import ops
    m = Student().to(DEV)
    x, lengths, _, _, _ = data()
    with torch.no_grad():
        whole = m.block(ops, x.to(DEV), torch.full((B,), T, dtype=torch.int32, device=DEV))
        h = torch.zeros(B, H, device=DEV)
        for t in range(T):
            xt = x[:, t].to(DEV)
            out, _ = ops.gated_step(ops.linear_act(ops.layer_norm(xt, m.g, m.c), m.wi, m.bi), h, h_out=h)
            near(ops.linear_act(out, m.wo, m.bo, "none", xt), whole[:, t].cpu(), 1e-5, t)


def test_spans_and_another_stream():
    """a KernelTimer sees every operator; on a side stream, and with autograd's own thread, the results are the same bits"""
    from dss_vae_amd import ops
    m = Student().to(DEV)
    x, lengths, ids, t, w = (v.to(DEV) for v in data())

    def step():
        m.zero_grad(set_to_none=True)
        total, rows = ops.distill_loss(m.logits(ops, x, lengths), ids, t, 2.0, w)
        total.backward()
        return [total.detach(), rows] + [p.grad for p in m.parameters()]

    want = step()
    torch.cuda.synchronize()
    ops.PROFILE = ops.KernelTimer()
    try:
        got = step()
        torch.cuda.synchronize()
        names = set(ops.PROFILE.summary())
    finally:
        ops.PROFILE = None
    assert {"layer_norm_fwd_kernel", "layer_norm_bwd_kernel", "gated_scan_fwd_kernel", "gated_scan_bwd_kernel", "linear_tile_kernel",
            "linear_act_bwd", "distill_kernel"} <= names
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.autograd.set_multithreading_enabled(True)
    try:
        threaded = step()
    finally:
        torch.autograd.set_multithreading_enabled(False)
    for a, b, c, d in zip(want, got, other, threaded):
        assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)


def test_two_graphs_side_by_side():
    """two captured training steps of the same weights, replayed in turn with eager work between: each has its own workspaces"""
    from dss_vae_amd import ops
    m = Student().to(DEV)
    x, lengths, ids, t, w = (v.to(DEV) for v in data())
    xs = [x.clone(), x.flip(0).contiguous()]
    params = list(m.parameters())

    def step(v):
        total, rows = ops.distill_loss(m.logits(ops, v, lengths), ids, t, 2.0, w)
        return [total, rows] + list(torch.autograd.grad(total, params))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for v in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(v))
        graphs.append(g)
    for k in range(3):
        for v in xs:
            v.mul_(1.25)
        want = [[o.detach().clone() for o in step(v)] for v in xs]
        for i in (0, 1, 1, 0):
            graphs[i].replay()
            step(xs[1 - i])
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(p.detach(), q) for p, q in zip(a, b)), k


def test_capture_refuses_leaves_of_a_graph_on_the_default_stream():
    """an eager graph of the same leaves lives on the default stream: every operator refuses the capture before it records anything, the capture ends
    in order, and once that graph is gone the same step is captured and replays"""
    from dss_vae_amd import ops
    x = torch.randn(6, 8, 32, device=DEV).requires_grad_()
    w = torch.randn(32, 32, device=DEV).requires_grad_()
    ids, t = torch.zeros(6, 8, 1, dtype=torch.int64, device=DEV), torch.zeros(6, 8, 1, device=DEV)
    calls = {"layer_norm": lambda: ops.layer_norm(x).sum(), "gated_scan": lambda: ops.gated_scan(x)[0].sum(),
             "linear_act": lambda: ops.linear_act(x, w, None, "tanh").sum(), "distill_loss": lambda: ops.distill_loss(x, ids, t)[0]}
    for name, call in calls.items():
        want = torch.autograd.grad(call(), x)[0]
        held = call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = torch.ones(4, device=DEV) * 2
            with pytest.raises(RuntimeError, match="%s: this stream is being captured" % name):
                call()
        del held, g, y
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = torch.autograd.grad(call(), x)[0]
        for _ in range(3):
            got.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want), name


def test_capture_after_a_warm_up_on_a_side_stream():
    """the usual recipe: eager steps on a side stream, whose last loss is still held, then the capture of such a step"""
    from dss_vae_amd import ops
    m = Student().to(DEV)
    x, lengths, ids, t, w = (v.to(DEV) for v in data())
    params = list(m.parameters())

    def step():
        total, _ = ops.distill_loss(m.logits(ops, x, lengths), ids, t, 2.0, w)
        total.backward()
        return total

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            m.zero_grad(set_to_none=True)
            loss = step()
    torch.cuda.current_stream().wait_stream(side)
    want = [loss.detach().clone()] + [p.grad.clone() for p in params]
    m.zero_grad(set_to_none=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        static = step()
    for _ in range(3):
        for p in params:
            p.grad.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), b) for a, b in zip([static] + [p.grad for p in params], want))
    assert float(loss.detach()) == float(want[0])
