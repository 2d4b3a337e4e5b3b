"""Work cases of the sequence-block operators: layer_norm, gated_scan / gated_step, linear_act and distill_loss.

Each case is one pass of one operator as a program calls it: a forward pass (serving) or a forward and a backward pass
(training).  `run` computes it with elementary torch operations in 32 bits, or, with `own`, through `dss_vae_amd.ops`.
`exact` is the operator's definition in 64 bits, with its gradients from automatic differentiation."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the 50 hypotheses of one greedy decoding step at the stress width: launch latency
        {"name": "norm token bf16", "op": "norm", "dtype": "bf16", "rows": 50, "width": 1024, "train": False, "w32": False},
        # all positions of a batch of 256 sentences (31 steps) at the default width 300, training
        {"name": "norm sentences fp32", "op": "norm", "dtype": "fp32", "rows": 7936, "width": 300, "train": True, "w32": True},
        # a long batch at the stress configuration's decoder width, weights kept in fp32
        {"name": "norm long bf16", "op": "norm", "dtype": "bf16", "rows": 32768, "width": 2048, "train": True, "w32": True},
        # one token of a decoding batch: the state goes forward one step
        {"name": "scan token bf16", "op": "scan", "dtype": "bf16", "batch": 50, "steps": 1, "width": 1024, "train": False,
         "padded": False, "reverse": False, "candidate": "tanh"},
        # a backward-running direction of a tree encoder: 90 symbols at most, padded, the default width
        {"name": "scan trees fp32", "op": "scan", "dtype": "fp32", "batch": 256, "steps": 90, "width": 300, "train": True,
         "padded": True, "reverse": True, "candidate": "tanh"},
        # two long documents: little parallelism beside the time axis
        {"name": "scan long bf16", "op": "scan", "dtype": "bf16", "batch": 2, "steps": 16384, "width": 2048, "train": True,
         "padded": False, "reverse": False, "candidate": "linear"},
        # projection of one decoding step back onto the residual stream: bound by the weight's read
        {"name": "linear token fp16", "op": "linear", "dtype": "fp16", "rows": 50, "inner": 1024, "outer": 2048,
         "act": "none", "residual": True, "train": False},
        # hidden-to-latent sized layer over a batch of sentences, in the framework's fp32
        {"name": "linear sentences fp32", "op": "linear", "dtype": "fp32", "rows": 7936, "inner": 600, "outer": 300,
         "act": "tanh", "residual": True, "train": True},
        # widening projection over a long batch: the matrix pipe's case
        {"name": "linear long bf16", "op": "linear", "dtype": "bf16", "rows": 16384, "inner": 2048, "outer": 8192,
         "act": "gelu", "residual": False, "train": True},
        # one decoding step's worth of rows against the 30k vocabulary
        {"name": "distill few fp32", "op": "distill", "dtype": "fp32", "rows": 50, "vocab": 30000, "top": 8, "train": True},
        # every target position of the headline batch
        {"name": "distill sentences fp32", "op": "distill", "dtype": "fp32", "rows": 7936, "vocab": 30000, "top": 32,
         "train": True},
        # a large subword vocabulary of odd size in 16 bits: rows start at every alignment
        {"name": "distill large bf16", "op": "distill", "dtype": "bf16", "rows": 2048, "vocab": 100003, "top": 64,
         "train": True},
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(("norm", "scan", "linear", "distill"))
    case = {"op": op, "dtype": rng.choice(("fp32", "bf16", "fp16")), "train": rng.random() < 0.7}
    if op == "norm":
        width = size(32, 8192)
        case.update(rows=size(1, min(32768, 32768 * 2048 // width)), width=width, w32=rng.random() < 0.5)
    elif op == "scan":
        width = size(16, 2048)
        batch = size(1, 512)
        steps = 1 if rng.random() < 0.15 else size(2, min(16384, 2 * 16384 * 2048 // (2 * width * batch)))
        case.update(batch=batch, steps=steps, width=width, padded=rng.random() < 0.5, reverse=rng.random() < 0.5,
                    candidate=rng.choice(("tanh", "linear")), train=case["train"] and steps > 1)
    elif op == "linear":
        inner, outer = size(64, 4096), size(64, 8192)
        most = 7936 if case["dtype"] == "fp32" else 16384
        case.update(rows=size(1, max(1, min(most, 16384 * 2048 * 8192 // (2 * inner * outer)))), inner=inner, outer=outer,
                    act=rng.choice(("none", "relu", "gelu", "silu", "tanh")), residual=rng.random() < 0.5)
    else:
        vocab = size(100, 131072)
        case.update(rows=size(1, min(8192, 7936 * 30000 // (2 * vocab))), vocab=vocab, top=min(size(1, 64), vocab // 2))
    return case


def work(case):
    s = 4 if case["dtype"] == "fp32" else 2
    train = case["train"]
    if case["op"] == "norm":
        n, d, ws = case["rows"] * case["width"], case["width"], 4 if case["w32"] else s
        return {"bytes": n * s * (4 if train else 2) + d * ws * (4 if train else 2), "flops": n * (20 if train else 8)}
    if case["op"] == "scan":
        row = case["batch"] * case["width"]
        n = row * case["steps"]
        return {"bytes": n * s * (6 if train else 3) + row * 4 * (4 if train else 2), "flops": n * (30 if train else 12)}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        b = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
        if train:
            b += m * n + m * k + n * k + n
        return {"bytes": b * s, "flops": (6 if train else 2) * m * k * n}
    m, v, k = case["rows"], case["vocab"], case["top"]
    return {"bytes": m * v * s * (2 if train else 1) + m * k * 12 + m * 8, "flops": m * v * (10 if train else 6)}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    dt = DTYPES[case["dtype"]]
    train = case["train"]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt, leaf=False):
        t = torch.randn(*shape, device="cuda", generator=g).mul_(scale).add_(shift).to(dtype)
        return t.requires_grad_() if leaf and train else t

    st = dict(case)
    if case["op"] == "norm":
        r, d = case["rows"], case["width"]
        wd = torch.float32 if case["w32"] else dt
        st.update(x=normal(r, d, scale=1.5, shift=0.3, leaf=True), weight=normal(d, scale=0.2, shift=1.0, dtype=wd, leaf=True),
                  bias=normal(d, scale=0.2, dtype=wd, leaf=True))
        if train:
            st["dy"] = normal(r, d)
    elif case["op"] == "scan":
        b, t, h = case["batch"], case["steps"], case["width"]
        # gates around sigmoid(1) = 0.73 with a wide spread: memories from one step to some hundred
        x = torch.randn(b, t, 2 * h, device="cuda", generator=g)
        x[:, :, :h].mul_(2.0).add_(1.0)
        x = x.to(dt)
        st["xproj"] = x.requires_grad_() if train else x
        st["h0"] = normal(b, h, scale=0.5, dtype=torch.float32, leaf=True)
        st["lengths"] = None
        if case["padded"]:
            st["lengths"] = torch.randint((t + 3) // 4, t + 1, (b,), device="cuda", generator=g, dtype=torch.int32)
        if train:
            st.update(dout=normal(b, t, h), dh=normal(b, h, dtype=torch.float32))
    elif case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        st.update(x=normal(m, k, leaf=True), w=normal(n, k, scale=k ** -0.5, leaf=True), b=normal(n, scale=0.1, leaf=True),
                  res=normal(m, n, leaf=True) if case["residual"] else None)
        if train:
            st["dy"] = normal(m, n)
    else:
        m, v, k = case["rows"], case["vocab"], case["top"]
        st["logits"] = normal(m, v, scale=2.0, leaf=True)
        # distinct ids per row: one from each of k equal stretches of the vocabulary; a tenth of the slots is empty
        stretch = v // k
        ids = torch.randint(0, stretch, (m, k), device="cuda", generator=g) + torch.arange(k, device="cuda") * stretch
        st["ids"] = ids.masked_fill(torch.rand(m, k, device="cuda", generator=g) < 0.1, -1)
        st["teacher"] = torch.randn(m, k, device="cuda", generator=g).mul_(2.0).add_(4.0).sort(dim=1, descending=True)[0]
        # every eighth position or so is padding
        keep = (torch.rand(m, device="cuda", generator=g) > 0.125).float()
        # (fp16 training scales its loss: without it most of the gradient lies below the type's normal numbers)
        st["weight"] = keep / keep.sum().clamp(min=1.0) * (16384.0 if dt == torch.float16 else 1.0)
        st["temperature"] = 2.0
    return st


# ---- plain forms -----------------------------------------------------------------------------------------------------
def _norm_plain(st):
    x, w, b = st["x"].float(), st["weight"].float(), st["bias"].float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = (c.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    xh = c * rstd
    y = (xh * w + b).to(st["x"].dtype)
    if not st["train"]:
        return {"y": y}
    dy = st["dy"].float()
    gw = dy * w
    dx = (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True)) * rstd
    wd = st["weight"].dtype
    return {"y": y, "dx": dx.to(y.dtype), "dw": (dy * xh).sum(0).to(wd), "db": dy.sum(0).to(wd)}


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 by doubling: log2(steps) passes"""
    a, b, step = a.clone(), b.clone(), 1
    while step < a.size(1):
        b[:, step:] = b[:, step:] + a[:, step:] * b[:, :-step]
        a[:, step:] = a[:, step:] * a[:, :-step]
        step *= 2
    return b


def _scan_plain(st):
    x, h0 = st["xproj"], st["h0"]
    dt, h, t = x.dtype, st["width"], st["steps"]
    tanh = st["candidate"] == "tanh"
    turn = (lambda v: v.flip(1)) if st["reverse"] else (lambda v: v)
    f = turn(x.float())
    a, n = torch.sigmoid(f[:, :, :h]), f[:, :, h:]
    n = torch.tanh(n) if tanh else n
    live = torch.ones(x.size(0), t, 1, dtype=torch.bool, device=x.device)
    if st["lengths"] is not None:
        live = turn((torch.arange(t, device=x.device) < st["lengths"].unsqueeze(1)).unsqueeze(2))
    am = torch.where(live, a, torch.ones_like(a))
    bm = torch.where(live, (1.0 - a) * n, torch.zeros_like(a))
    bm[:, 0] += am[:, 0] * h0
    hs = _scan(am, bm)
    zero = torch.zeros_like(hs)
    out = {"out": turn(torch.where(live, hs, zero)).to(dt).contiguous(), "h_last": hs[:, -1].clone()}
    if not st["train"]:
        return out
    g = torch.where(live, turn(st["dout"].float()), zero)
    g[:, -1] += st["dh"]
    nxt = torch.cat((am[:, 1:], torch.ones_like(am[:, :1])), 1)
    d = _scan(nxt.flip(1), g.flip(1)).flip(1)
    prev = torch.cat((h0.unsqueeze(1), hs[:, :-1]), 1)
    dz = d * (prev - n) * a * (1.0 - a)
    dn = d * (1.0 - a) * ((1.0 - n * n) if tanh else 1.0)
    dx = torch.where(live, torch.cat((dz, dn), 2), torch.zeros_like(f))
    out.update(dxproj=turn(dx).to(dt).contiguous(), dh0=am[:, 0] * d[:, 0])
    return out


def _act(z, act):
    """-> act(z), act'(z)"""
    if act == "relu":
        return z.clamp(min=0.0), (z > 0).to(z.dtype)
    if act == "tanh":
        t = torch.tanh(z)
        return t, 1.0 - t * t
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        c = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    return z, torch.ones_like(z)


def _linear_plain(st):
    x, w, dt = st["x"].float(), st["w"].float(), st["x"].dtype
    y, slope = _act(x @ w.t() + st["b"].float(), st["act"])
    if st["res"] is not None:
        y = y + st["res"].float()
    out = {"y": y.to(dt)}
    if st["train"]:
        dz = st["dy"].float() * slope
        out.update(dx=(dz @ w).to(dt), dw=(dz.t() @ x).to(dt), db=dz.sum(0).to(dt))
        if st["res"] is not None:
            out["dres"] = st["dy"]
    return out


def _distill_plain(st):
    tau, ids, w = st["temperature"], st["ids"], st["weight"]
    z = st["logits"].float() / tau
    lse = z.amax(1, keepdim=True)
    e = torch.exp(z - lse)
    total = e.sum(1, keepdim=True)
    valid = ids >= 0
    at = ids.clamp(min=0)
    t = torch.where(valid, st["teacher"] / tau, torch.full_like(st["teacher"], -math.inf))
    top = t.amax(1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    pe = torch.exp(t - top)
    ps = pe.sum(1, keepdim=True)
    p = pe / torch.where(ps > 0, ps, torch.ones_like(ps))
    logp = torch.where(valid, t - top - torch.log(ps), torch.zeros_like(t))
    logq = z.gather(1, at) - lse - torch.log(total)
    rows = (p * (logp - logq)).sum(1) * (tau * tau)
    rows = torch.where(w != 0, rows, torch.zeros_like(rows))
    out = {"total": (w * rows).sum(), "rows": rows}
    if st["train"]:
        q = e / total * p.sum(1, keepdim=True)
        q.scatter_add_(1, at, -p)
        out["dlogits"] = (q * (w * tau).unsqueeze(1)).to(st["logits"].dtype)
    return out


# ---- through the framework -------------------------------------------------------------------------------------------
def _norm_own(st):
    from dss_vae_amd import ops
    y = ops.layer_norm(st["x"], st["weight"], st["bias"], 1e-5)
    if not st["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["dy"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _scan_own(st):
    from dss_vae_amd import ops
    if st["steps"] == 1 and not st["train"] and st["lengths"] is None:
        out, h = ops.gated_step(st["xproj"][:, 0], st["h0"], candidate=st["candidate"])
        return {"out": out.unsqueeze(1), "h_last": h}
    out, h = ops.gated_scan(st["xproj"], st["h0"], st["lengths"], st["reverse"], st["candidate"])
    if not st["train"]:
        return {"out": out, "h_last": h}
    dx, dh0 = torch.autograd.grad((out, h), (st["xproj"], st["h0"]), (st["dout"], st["dh"]))
    return {"out": out, "h_last": h, "dxproj": dx, "dh0": dh0}


def _linear_own(st):
    from dss_vae_amd import ops
    y = ops.linear_act(st["x"], st["w"], st["b"], st["act"], st["res"])
    out = {"y": y}
    if st["train"]:
        leaves = (st["x"], st["w"], st["b"]) + (() if st["res"] is None else (st["res"],))
        out.update(zip(("dx", "dw", "db", "dres"), torch.autograd.grad(y, leaves, st["dy"])))
    return out


def _distill_own(st):
    from dss_vae_amd import ops
    total, rows = ops.distill_loss(st["logits"], st["ids"], st["teacher"], st["temperature"], st["weight"])
    out = {"total": total, "rows": rows}
    if st["train"]:
        out["dlogits"], = torch.autograd.grad(total, (st["logits"],))
    return out


_PLAIN = {"norm": _norm_plain, "scan": _scan_plain, "linear": _linear_plain, "distill": _distill_plain}
_OWN = {"norm": _norm_own, "scan": _scan_own, "linear": _linear_own, "distill": _distill_own}


def run(state):
    if own:
        return _OWN[state["op"]](state)
    with torch.no_grad():
        return _PLAIN[state["op"]](state)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    train = case["train"]

    def wide(t):
        return None if t is None else t.detach().double().requires_grad_(train)

    if case["op"] == "norm":
        x, w, b = wide(st["x"]), wide(st["weight"]), wide(st["bias"])
        std = torch.sqrt(x.var(1, unbiased=False, keepdim=True) + 1e-5)
        y = (x - x.mean(1, keepdim=True)) / std * w + b
        out = {"y": y.detach()}
        if train:
            out.update(zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), st["dy"].double())))
        return out
    if case["op"] == "scan":
        if case["steps"] * (3 if train else 1) > 60000:
            return None
        x, h0, width, steps = wide(st["xproj"]), wide(st["h0"]), case["width"], case["steps"]
        keep = 1.0 / (1.0 + torch.exp(-x[..., :width]))
        new = torch.tanh(x[..., width:]) if case["candidate"] == "tanh" else x[..., width:]
        lengths = st["lengths"] if st["lengths"] is not None else torch.full((case["batch"],), steps, device="cuda")
        live = (torch.arange(steps, device="cuda").unsqueeze(0) < lengths.unsqueeze(1)).unsqueeze(2)
        keep, add = torch.where(live, keep, 1.0), torch.where(live, (1.0 - keep) * new, 0.0)
        keep, add, state, states = keep.unbind(1), add.unbind(1), h0, [None] * steps
        for t in (range(steps - 1, -1, -1) if case["reverse"] else range(steps)):
            state = torch.addcmul(add[t], keep[t], state)
            states[t] = state
        y = torch.where(live, torch.stack(states, 1), 0.0)
        out = {"out": y.detach(), "h_last": state.detach()}
        if train:
            got = torch.autograd.grad((y, state), (x, h0), (st["dout"].double(), st["dh"].double()))
            out.update(zip(("dxproj", "dh0"), got))
        return out
    if case["op"] == "linear":
        x, w, b, r = wide(st["x"]), wide(st["w"]), wide(st["b"]), wide(st["res"])
        z = torch.addmm(b, x, w.t())
        y = {"none": lambda: z, "relu": lambda: torch.relu(z), "tanh": lambda: torch.tanh(z),
             "silu": lambda: z / (1.0 + torch.exp(-z)), "gelu": lambda: 0.5 * z * torch.erfc(-z / math.sqrt(2.0))}[case["act"]]()
        y = y if r is None else y + r
        out = {"y": y.detach()}
        if train:
            leaves = (x, w, b) if r is None else (x, w, b, r)
            out.update(zip(("dx", "dw", "db", "dres"), torch.autograd.grad(y, leaves, st["dy"].double())))
        return out
    z, tau, w = wide(st["logits"]), st["temperature"], st["weight"].double()
    valid = st["ids"] >= 0
    some = valid.any(1)
    t = (st["teacher"].double() / tau).masked_fill(~valid & some.unsqueeze(1), -math.inf)
    logp = torch.log_softmax(t, 1)
    p = torch.exp(logp) * (valid & (w != 0).unsqueeze(1))
    logq = torch.log_softmax(z / tau, 1).gather(1, st["ids"].clamp(min=0))
    rows = tau * tau * (p * (logp.masked_fill(p == 0, 0.0) - logq)).sum(1)
    total = (w * rows).sum()
    out = {"total": total.detach(), "rows": rows.detach()}
    if train:
        out["dlogits"], = torch.autograd.grad(total, (z,))
    return out
