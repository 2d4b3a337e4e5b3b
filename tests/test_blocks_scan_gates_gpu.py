"""ops.gated_scan / gated_step with gates close to 1 and 0: the update, and the gradients of both halves, are proportional to 1 - a, which
keeps its relative accuracy; gates beyond the exponential's range."""
import math

import pytest
import torch

from blocks_util import DEV, TYPES, U32, half_step, rnd
from test_blocks_scan_gpu import reference

pytestmark = pytest.mark.gpu


def run(x, h0, dout, candidate, reverse=False, lengths=None):
    from dss_vae_amd import ops
    xd = x.to(DEV).requires_grad_()
    hd = None if h0 is None else h0.to(DEV).requires_grad_()
    out, last = ops.gated_scan(xd, hd, lengths, reverse, candidate)
    (out.float() * dout.to(DEV).float()).sum().backward()
    return out.detach().cpu(), last.detach().cpu(), xd.grad.cpu()


def magnitudes(x, h0, dout, candidate):
    """64 bits, per element: the sums of magnitudes that make up h, and D"""
    B, T, H = dout.shape
    z, v = x[..., :H].double(), x[..., H:].double()
    a, oma = torch.sigmoid(z), torch.sigmoid(-z)
    n = (torch.tanh(v) if candidate == "tanh" else v).abs()
    h = torch.zeros(B, H, dtype=torch.float64) if h0 is None else h0.double().abs()
    hs, D = [], [None] * T
    for t in range(T):
        h = a[:, t] * h + oma[:, t] * n[:, t]
        hs.append(h)
    g = torch.zeros(B, H, dtype=torch.float64)
    for t in range(T - 1, -1, -1):
        D[t] = dout[:, t].double().abs() + g
        g = a[:, t] * D[t]
    return torch.stack(hs, 1), torch.stack(D, 1), n, a, oma


@pytest.mark.parametrize("candidate", ["linear", "tanh"])
@pytest.mark.parametrize("B,T,H", [(2, 60, 50), (3, 2000, 48), (40, 300, 130)])
def test_long_memory(candidate, B, T, H):
    """fp32, gates at 8, 10, 12, 16, 20.  u = exp(-z) is off by |z| units of 2^-24 (its argument's rounding) and 2 of the instruction, 1 - a = u a by
    4 more: 26 at z = 20, and 8 for the candidate.  a, rounded to nearest, moves what passes T steps by T / 2 units, and sums of T
    terms by as many: 40 + 2 T units of the magnitudes summed up."""
    g = torch.Generator().manual_seed(T)
    pick = torch.tensor([8.0, 10.0, 12.0, 16.0, 20.0])
    z = pick[torch.randint(0, 5, (B, T, H), generator=g)]
    x = torch.cat((z + 0.1 * torch.rand(B, T, H, generator=g), rnd(B, T, H, seed=81)), 2)
    dout = rnd(B, T, H, seed=82)
    want = reference(x, None, None, False, candidate, dout)
    hs, D, n, a, oma = magnitudes(x, None, dout, candidate)
    out, last, dx = run(x, None, dout, candidate)
    few, many = (40 + 0 * T) * U32, (40 + 2 * T) * U32
    assert ((out.double() - want[0]).abs() <= many * hs).all()
    assert ((last.double() - want[1]).abs() <= many * hs[:, -1]).all()
    prev = torch.cat((torch.zeros(B, 1, H, dtype=torch.float64), hs[:, :-1]), 1)
    bound = oma * D * many
    err = (dx.double() - want[2]).abs()
    assert (err[..., :H] <= bound * (prev + n) + 1e-40).all(), float((err[..., :H] / (bound * (prev + n))).max())
    assert (err[..., H:] <= bound + 1e-40).all(), float((err[..., H:] / bound).max())
    # one step's share alone
    from dss_vae_amd import ops
    one, h1 = ops.gated_step(x[:, 0].to(DEV), None, candidate)
    v = torch.tanh(x[:, 0, H:].double()) if candidate == "tanh" else x[:, 0, H:].double()
    exact = torch.sigmoid(-x[:, 0, :H].double()) * v
    assert ((h1.cpu().double() - exact).abs() <= few * exact.abs()).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_gates_beyond_the_exponential(dtype):
    """z = +-inf, +-200, +-90: the state is kept, or replaced by the candidate, exactly; NaN shows in the state and both gradients"""
    from dss_vae_amd import ops
    for z, keep in ((200.0, True), (math.inf, True), (-200.0, False), (-math.inf, False), (-60000.0, False)):
        for T in (1, 3, 700):
            x = torch.cat((torch.full((2, T, 8), z), rnd(2, T, 8, seed=83)), 2).to(dtype)
            h0 = rnd(2, 8, seed=84)
            out, last, dx = run(x, h0, torch.ones(2, T, 8), "linear")
            want = h0.unsqueeze(1).expand(2, T, 8).to(dtype) if keep else x[..., 8:]
            assert torch.equal(out, want), (z, T)
            assert torch.equal(last, h0 if keep else x[:, -1, 8:].float())
            assert (dx[..., :8] == 0).all() and (dx[..., 8:] == (0 if keep else 1)).all(), (z, T)
            one, h1 = ops.gated_step(x[:, 0].to(DEV), h0.to(DEV), "linear")
            assert torch.equal(h1.cpu(), h0 if keep else x[:, 0, 8:].float())
    x = torch.cat((torch.zeros(1, 5, 8), rnd(1, 5, 8, seed=85)), 2).to(dtype)
    x[0, 2, 3] = math.nan
    out, last, dx = run(x, None, torch.ones(1, 5, 8), "tanh")
    assert out[0, 2:, 3].isnan().all() and last[0, 3].isnan() and dx[0, 2, 3].isnan() and dx[0, 2, 11].isnan()
    assert out[0, :, :3].isfinite().all() and out[0, :2, 3].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_small_gates(dtype):
    """z down to -30: what passes a step is a itself, to its own accuracy (|z| + 6 units), and out's rounding"""
    H = 64
    z = torch.linspace(-30, 0, H).to(dtype)
    x = torch.cat((z, torch.zeros(H).to(dtype))).view(1, 1, 2 * H)
    h0 = torch.full((1, H), 3.0)
    out, last, _ = run(x, h0, torch.zeros(1, 1, H), "linear")
    want = 3.0 * torch.sigmoid(z.double()).view(1, H)
    assert ((last.double() - want).abs() <= want * 40 * U32).all()
    assert ((out[:, 0].double() - want).abs() <= want * (half_step(dtype) + 41 * U32) + (torch.finfo(dtype).tiny * torch.finfo(dtype).eps)).all()
