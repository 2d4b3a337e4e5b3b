"""Shared by the sequence-block tests: seeded inputs and the error bound they are held to.

Bound of an output: half a step of its type at the value (one rounding) plus `slack` times the fp32 unit roundoff at a
`scale` that the operator's formula gives (the magnitudes that its fp32 sums add up): derived beside each use."""
import torch

DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rnd(*shape, seed=0, scale=1.0, shift=0.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(1000 + seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def check(got, want, scale, slack, what="", dtype=None):
    """|got - want| <= half a step of got's type at want (+ the type's smallest step) + slack * 2^-24 * scale"""
    dtype = dtype or got.dtype
    got, want = got.detach().cpu().double(), want.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    scale = torch.as_tensor(scale, dtype=torch.float64).cpu().expand_as(want)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    fp = slack * U32 * scale
    bound = half_step(dtype) * (want.abs() + fp) + fp + tiny
    err = (got - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), "of", bad.numel(), "worst ratio", float((err / bound).nan_to_num(1e9).max()))


def bits(t):
    """the exact bits, for equality with NaN"""
    return t.contiguous().view(torch.int32 if t.element_size() == 4 else torch.int16)
