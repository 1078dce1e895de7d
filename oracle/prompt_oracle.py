"""The rotation of queries and keys and the attention of whole prompts in plain arithmetic (torch), on
the device of the inputs: the definitions that the HIP kernels are tested against.  Nothing here is
shared with them."""
from __future__ import annotations

import math

import torch

BF16 = 2.0 ** -8   # half a step of bf16, relative to the value
FP32 = 2.0 ** -24  # of fp32


def turn(x, positions, rotary, base, weight=None, eps=1e-6):
    """x [rows, heads, dim] normed and rotated, in 64 bits, angles from the formula; and the size of the
    terms that each channel is the sum of."""
    x = x.double()
    if weight is not None:
        x = x * (x.square().mean(-1, keepdim=True) + eps) ** -0.5 * weight.double()
    half = rotary // 2
    frequency = float(base) ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    angle = (positions.double()[:, None] * frequency)[:, None]
    a, b, rest = x[..., :half], x[..., half:rotary], x[..., rotary:]
    c, s = angle.cos(), angle.sin()
    return (torch.cat((a * c - b * s, b * c + a * s, rest), -1),
            torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), rest.abs()), -1))


def turn_fp32(x, positions, table, weight=None, eps=1e-6):
    """The same in the arithmetic that the library documents, step by step: the bits it returns."""
    x = x.float()
    if weight is not None:
        mean = (x.double().square().sum(-1, keepdim=True) / x.shape[-1]).float()
        x = x * ((mean + torch.tensor(eps, dtype=torch.float32, device=x.device)).double() ** -0.5).float()
        x = x * weight.float()
    row = table[positions.long()][:, None]
    half = row.shape[-1] // 2
    c, s = row[..., :half], row[..., half:]
    a, b = x[..., :half], x[..., half:2 * half]
    ac, bs, bc, as_ = a * c, b * s, b * c, a * s
    return torch.cat((ac - bs, bc + as_, x[..., 2 * half:]), -1).to(torch.bfloat16)


def turn_tolerance(want, size):
    """Of turn()'s results in bf16: one rounding to bf16, and in front of it at most ten fp32 roundings of
    terms of that size (mean, root, two products, the table's entry, the rotation's product and sum)."""
    return BF16 * want.abs() * (1 + 16 * FP32) + 16 * FP32 * size + 2.0 ** -133


def prompt(q, k, v, offsets, scale=None):
    """(out, spread, reach, power) of causal attention of packed rows in 64 bits: out [rows, heads, dim],
    zeros for rows of no sequence; spread = sum w |v| and power = sum w^2 v^2 with the normalized weights
    w; reach [rows, heads] the largest scale * sum |q k| that a row meets."""
    q, k, v = q.double(), k.double(), v.double()
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out, spread, power = (torch.zeros_like(q) for _ in range(3))
    reach = torch.zeros(rows, heads, dtype=torch.float64, device=q.device)
    for first, end in zip(offsets, offsets[1:]):
        later = torch.ones(end - first, end - first, dtype=torch.bool, device=q.device).triu(1)
        for h in range(heads):
            g = h // group
            a, b, c = q[first:end, h], k[first:end, g], v[first:end, g]
            if not len(a):
                continue
            s = (a @ b.t().contiguous() * scale).masked_fill(later, -math.inf)
            w = torch.exp(s - s.amax(-1, keepdim=True))
            w = w / w.sum(-1, keepdim=True)
            out[first:end, h] = w @ c
            spread[first:end, h] = w @ c.abs()
            power[first:end, h] = w.square() @ c.square()
            reach[first:end, h] = (a.abs() @ b.abs().t().contiguous() * scale).masked_fill(later, 0).amax(-1)
    return out, spread, reach, power


def prompt_tolerance(want, spread, reach, longest):
    """Element by element: the weights' rounding to bf16 (each off by BF16 of itself, so the sum by BF16 of
    the spread) and the output's; in fp32 a score's 128 products and its way into the exponent, off by
    (dim + 4) FP32 of reach in the scores of a row and of its reference, the exponential by 2^-22, and sums
    of `longest` terms, each once in the numerator and once in the sum of weights."""
    e = 2 * (FP32 * (4 * (want.shape[-1] + 4) * reach[..., None] + longest + 16) + 2.0 ** -22)
    return BF16 * (want.abs() + spread) * (1 + BF16) + spread * torch.expm1(e) + 2.0 ** -130


def check_prompt(got, want, spread, reach, power, longest):
    """got within the tolerance everywhere, and the squares of all errors together below what independent
    roundings of weights and outputs give: a rounding's variance is a third of its bound's square at
    most.  (A tenth more for the sample, from some thousand elements on.)"""
    off = (got.double() - want).abs()
    bad = ~(off <= prompt_tolerance(want, spread, reach, longest))
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, worst {float((off - prompt_tolerance(want, spread, reach, longest)).max()):.3g}"
    if want.numel() >= 4096:
        most = (BF16 ** 2 / 3 * (want.square() + power)).sum() * 1.1 + (spread * 2 * FP32 * (want.shape[-1] + longest + 64)).square().sum()
        assert float(off.square().sum()) <= float(most), (float(off.square().sum()), float(most))
