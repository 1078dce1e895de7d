"""``kv_step`` behind more than 2^30 cached tokens."""
import pytest
import torch

from test_gpu_kv_cache import attn, int32

pytestmark = pytest.mark.gpu


def test_contexts_beyond_2_30(gpu_lib):
    context = 2 ** 30 + 5 * 256 + 255
    table = torch.zeros(1, context // 256 + 2, dtype=torch.int32, device="cuda")
    table[0, context // 256] = 77
    s = attn.kv_step(int32([3]), int32([context]), table, int32([99]), block_size=256, num_tokens=3)
    assert s.seq_lens.tolist() == [context + 3] and s.positions.tolist() == [context, context + 1, context + 2]
    assert s.slots.tolist() == [77 * 256 + 255, 99 * 256, 99 * 256 + 1]
    assert int(table[0, context // 256 + 1]) == 99 and int(s.blocks_used) == 1
