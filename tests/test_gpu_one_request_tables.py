"""Block tables of one request or of one block: the stride of a dimension of one entry says nothing,
and torch leaves anything there (a column turned into a row, a slice of a wider table)."""
import pytest
import torch

from test_gpu_attention import Batch, attn
from test_gpu_kv_cache import int32

pytestmark = pytest.mark.gpu


def rows_of(values):
    """The same [1, n] table with strides that differ: a row, a turned column, an expanded row."""
    n = len(values)
    row = int32([values])
    column = int32([[v] for v in values]).t()
    wide = torch.zeros(3, n + 4, dtype=torch.int32, device="cuda")[1:2, :n]
    wide.copy_(row)
    narrow = torch.zeros(n + 3, dtype=torch.int32, device="cuda").as_strided((1, n), (2, 1))
    narrow.copy_(row)
    return row, column, wide, narrow


def test_attention_of_one_request(gpu_lib):
    b = Batch([3], [90], 8, 2, 128, 16, seed=81)
    q, cache, _, seq, offsets = b.args()
    want = b.run()
    b.check(want)
    for tables in rows_of(b.tables[0]):
        for lens in (seq, torch.stack((seq, seq), 1)[:, 0]):
            print("one request", tables.stride(), lens.stride(), flush=True)
            assert torch.equal(attn.attention_int4(q, cache, tables, lens, offsets, block_size=16), want)


@pytest.mark.parametrize("strided", [False, True])
def test_step_of_one_request(gpu_lib, strided):
    for tables in rows_of([3, 4, 0, 0]):
        query = torch.tensor([[20, 0]], dtype=torch.int32, device="cuda")[:, 0]
        free = torch.stack((int32([7, 8, 9]),) * 2, 1)[:, 0] if strided else int32([7, 8, 9])
        print("one request's step", tables.stride(), flush=True)
        s = attn.kv_step(query, int32([30]), tables, free, block_size=16, num_tokens=20)
        assert s.block_tables is tables and tables.tolist() == [[3, 4, 7, 8]]
        assert s.slots.tolist() == [4 * 16 + 14, 4 * 16 + 15] + [7 * 16 + i for i in range(16)] + [8 * 16, 8 * 16 + 1]


@pytest.mark.parametrize("strided", [False, True])
def test_tables_of_one_block(gpu_lib, strided):
    """[requests, 1]: the first column of a wider table, the turned row of a taller one."""
    free = torch.stack((int32([7, 8, 9]),) * 2, 1)[:, 0] if strided else int32([7, 8, 9])
    for tables in (int32([[3], [0]]), int32([[3, 1], [0, 1]])[:, :1], int32([[3, 0]]).t(), int32([[3, 0], [5, 5]])[:1].t()):
        print("one block", tables.stride(), flush=True)
        s = attn.kv_step(int32([2, 1]), int32([5, 0]), tables, free, block_size=16, num_tokens=3)
        assert tables.tolist() == [[3], [7]] and s.slots.tolist() == [3 * 16 + 5, 3 * 16 + 6, 7 * 16]
