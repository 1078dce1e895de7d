"""Values of very different size among one row's keys: the large ones make the output, and the small
ones, or rows of zeros, still have their weight in the softmax's sum."""
import pytest
import torch

from kv4_helpers import mark_values
from oracle import kv4_oracle as ora
from test_gpu_attention import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hint", [1, 300])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("marked", [False, True])
@pytest.mark.parametrize("large,small", [(90, -90), (90, None), (50, -50), (100, 0), (0, -100)])
@pytest.mark.parametrize("new,seq", [([90, 70], [200, 150]), ([100], [2500])])
def test_large_values_beside_small_ones(gpu_lib, hint, dim, marked, large, small, new, seq):
    """Every third page's values times 2^large, the others' times 2^small, or zero; large ones come
    first in one sequence and later in the other, and rows that see no large one are as exact as any."""
    b = Batch(new, seq, 8, 2, dim, 16, seed=120 + dim)
    if marked:
        mark_values(b, dim)
    meta = b.cache.view(torch.int32)[..., 16 * dim // 4 + 16:]
    for r, n in enumerate(seq):
        for i in range(0, n, 16):
            page, live = meta[b.tables[r][i // 16]], min(16, n - i)
            if i // 16 % 3 == r:
                page[:, :live] += large << 23
            elif small is None:
                page[:, :live] = 0x00004300
            else:
                page[:, :live] += small << 23
    b.qkv.mul_(0.25)
    print("sizes", hint, dim, marked, large, small, new, flush=True)
    kernel = "split" if hint == 1 else "prompt"
    want = ora.attention_errors(b.q, b.cache, b.tables, b.seq, b.offsets, b.block, kernel)
    assert ora.check_errors(b.run(max_query_len=hint), *want) is None
