"""Prompt attention where its arithmetic is at its limits: sums over very long prompts."""
import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

attn = importlib.import_module("llm-serve_amd.layers.attention")


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_sums_of_equal_weights_over_a_long_prompt(gpu_lib):
    """350000 rows whose first key weighs 1 and has the value 0, and whose others weigh p = 179/256 each, a
    number of bf16, and have values of 0 or 1: in channel c the first m_c of each 4096 runs of 16 keys have
    ones, so row t is p n / (1 + p t) with n the ones that it sees.

    The numerator's sums (16 p at a time, a multiple of 2^-4, below 2^18) are formed without an error but for a
    run that a prompt or a share of it cuts, and the weights lose nothing in bf16.  What is left: p by 2^-18 (its
    2e-6 and its score's two roundings) and the exponential by 2^-22, the sum of weights (5469 tiles of some 40
    additions before them) by 2^-24 each, ten roundings of cut runs, joins and the quotient, and half a step of
    the output.  The p of the scores lies 2e-6 above 179/256, so that a running sum of single
    weights, whose last place is 2^-7 here, would round each of them up by 2^-8."""
    rows, p = 350000, 179 / 256
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k = (torch.zeros(rows, 1, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q[:, 0, 0] = 1
    k[0, 0, 0] = 1
    at = torch.arange(rows, device="cuda")
    ones = torch.randint(2048, 4096, (128,), generator=gen, device="cuda")
    v = (at[:, None] // 16 % 4096 < ones) & (at[:, None] > 0)
    out = attn.attention_prompt(q, k, v[:, None].to(torch.bfloat16), int32([0, rows]), scale=-math.log(p * (1 + 2e-6)))
    want = p * v.cumsum(0) / (1 + p * at[:, None].double())
    half_step = 2.0 ** (torch.frexp(want.clamp(min=2.0 ** -100)).exponent - 9)
    off = (out[:, 0].double() - want).abs() - half_step
    error = 2.0 ** -18 + 2.0 ** -22 + (5469 + 40 + 10) * 2.0 ** -24
    bad = off > error * want
    assert not bool(bad.any()), (int(bad.sum()), int(bad.any(1).nonzero()[0]), float((off / want.clamp(min=1e-9)).max()))
