"""Norm and rotation of rows whose mean square leaves fp32's range."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

rope = importlib.import_module("llm-serve_amd.layers.rotary_embedding")


def test_rows_whose_mean_square_passes_fp32(gpu_lib):
    """They become zero, as the fp32 arithmetic that is documented gives them (1 / sqrt(inf) is 0); without a weight, and
    in other rows, nothing changes."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k = (torch.randn(40, 3, 128, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    positions, table = torch.arange(40, device="cuda", dtype=torch.int32), rope.rotary_table(128, 64)
    w = torch.rand(128, generator=gen, device="cuda").to(torch.bfloat16)
    want = rope.qk_norm_rope(q, k, positions, table, q_weight=w)
    large = q.clone()
    large[7] *= 2.0 ** 66
    got = rope.qk_norm_rope(large, k, positions, table, q_weight=w)
    assert not bool(got[0][7].any()) and torch.equal(got[1], want[1])
    others = torch.arange(40, device="cuda") != 7
    assert torch.equal(got[0][others], want[0][others])
    assert bool(rope.qk_norm_rope(large, k, positions, table)[0][7].any())
