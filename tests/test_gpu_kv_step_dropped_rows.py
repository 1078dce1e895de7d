"""``kv_step`` with fewer rows than the lengths count: the tables hold every block that blocks_used
counts, so that a step behind the truncated one names no page of another request."""
import random

import pytest
import torch

from test_gpu_kv_cache import attn, int32, run_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [0, 1, 16, 17, 33, 40, 95])
def test_blocks_of_dropped_rows(gpu_lib, tokens):
    """Three requests of 96 rows in all: rows behind the last one, none of them, all of them opened
    blocks; the free list runs out, and a table is too narrow for its request."""
    query, context = [20, 36, 40], [5, 16, 0]
    for free in ([7, 8, 9, 10, 11, 12, 13], [7, 8, 9]):
        for width in (5, 3):
            print("dropped", tokens, len(free), width, flush=True)
            run_step(query, context, [[1] * width, [2] * width, [3] * width], free, 16, tokens)


def test_one_query_longer_than_the_rows(gpu_lib):
    """Its sequence's length is its context and its whole query, however many rows are missing."""
    run_step([100], [3], [[5] * 8], [20, 21, 22, 23, 24, 25, 26, 27], 16, 7)
    run_step([300, 2], [0, 31], [[5] * 20, [6] * 20], list(range(40, 70)), 16, 0)


def test_many_requests_dropped(gpu_lib):
    rng = random.Random(1)
    query = [rng.randint(0, 60) for _ in range(700)]
    context = [rng.randint(0, 90) for _ in range(700)]
    run_step(query, context, [[9] * 10 for _ in range(700)], list(range(100, 2500)), 16, 300)


def test_step_behind_a_truncated_one(gpu_lib):
    """Both requests continue from seq_lens: the pages of the second step's tokens are the ones that
    the first step took from the free list, not what the tables held before."""
    tables = int32([[0, 50, 50, 50], [1, 50, 50, 50]])
    first = attn.kv_step(int32([30, 30]), int32([10, 10]), tables, int32([60, 61, 62, 63, 64]), block_size=16, num_tokens=8)
    assert int(first.blocks_used) == 4 and first.seq_lens.tolist() == [40, 40]
    assert tables.tolist() == [[0, 60, 61, 50], [1, 62, 63, 50]]
    second = attn.kv_step(int32([1, 1]), first.seq_lens, tables, int32([64]), block_size=16, num_tokens=2)
    assert second.slots.tolist() == [61 * 16 + 8, 63 * 16 + 8] and int(second.blocks_used) == 0
