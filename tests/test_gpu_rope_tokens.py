"""Norm and rotation of as many tokens as a launch takes."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

rope = importlib.import_module("llm-serve_amd.layers.rotary_embedding")


def test_the_most_tokens(gpu_lib):
    """2^26 - 32 tokens of the same row at positions that repeat after 32: outputs of 8.6 GB each repeat too; one
    token more is refused."""
    tokens = (1 << 26) - 32
    gen = torch.Generator(device="cuda").manual_seed(1)
    row = torch.randn(1, 2, 64, generator=gen, device="cuda").to(torch.bfloat16)
    table = rope.rotary_table(64, 32)
    positions = torch.arange(32, device="cuda", dtype=torch.int32).repeat(tokens // 32 + 1)
    w = row[0, 0].contiguous()
    want = rope.qk_norm_rope(row[:, :1].expand(32, 1, 64), row[:, 1:].expand(32, 1, 64), positions[:32], table, q_weight=w)
    q, k = (t.expand(tokens, 1, 64) for t in (row[:, :1], row[:, 1:]))
    got = rope.qk_norm_rope(q, k, positions[:tokens], table, q_weight=w)
    for x, y in zip(got, want):
        assert bool((x.view(-1, 32, 64) == y.view(1, 32, 64)).all())
    q, k = (t.expand(tokens + 1, 1, 64) for t in (row[:, :1], row[:, 1:]))
    with pytest.raises(RuntimeError, match="too many"):
        rope.qk_norm_rope(q, k, positions[:tokens + 1], table)
