"""Each attention kernel against the bound of what it rounds itself (oracle/kv4_oracle.py,
attention_errors), element by element and in the squared error of all; and long sequences cut over
many workgroups, whose values name their keys, so that a lost or repeated part shows in some channel."""
import pytest
import torch

from kv4_helpers import mark_values
from oracle import kv4_oracle as ora
from test_gpu_attention import SHAPES, Batch

pytestmark = pytest.mark.gpu


def check(b, kernel, **kw):
    out = b.run(**kw)
    want = ora.attention_errors(b.q, b.cache, b.tables, b.seq, b.offsets, b.block, kernel)
    assert ora.check_errors(out, *want) is None


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("new,seq", [([1] * 6, [1, 17, 128, 300, 777, 1500]), ([8, 3, 5], [8, 200, 900]),
                                     ([100, 70], [100, 400])])
def test_split_kernel(gpu_lib, heads, kv_heads, dim, new, seq):
    """Decode rows, drafts, and whole prompts too where the caller's hint says that none is longer."""
    b = Batch(new, seq, heads, kv_heads, dim, 16, seed=90 + sum(new))
    print("split", heads, kv_heads, dim, new, flush=True)
    check(b, "split", max_query_len=1)


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("new,seq", [([80], [80]), ([70, 130], [600, 130]), ([257], [900])])
def test_prompt_kernel(gpu_lib, heads, kv_heads, dim, new, seq):
    """Prompts and chunks, more than 64 rows a kv head each."""
    b = Batch(new, seq, heads, kv_heads, dim, 16, seed=95 + sum(new))
    print("prompt", heads, kv_heads, dim, new, flush=True)
    check(b, "prompt", max_query_len=max(new))


@pytest.mark.parametrize("zero_queries", [True, False])
@pytest.mark.parametrize("heads,kv_heads,dim,block,new,seq", [
    (4, 1, 128, 256, [1], [20000]), (1, 1, 64, 16, [1], [20000]), (8, 8, 128, 64, [1, 1], [9000, 3]),
    (4, 1, 128, 16, [1] * 9, [6000, 1, 2, 3, 700, 1, 1, 40, 2500]), (8, 2, 128, 32, [9, 1], [5000, 4100])])
def test_split_parts_all_count_once(gpu_lib, heads, kv_heads, dim, block, new, seq, zero_queries):
    """Sequences over up to 768 workgroups: every 16 keys have a channel of their own."""
    b = Batch(new, seq, heads, kv_heads, dim, block, seed=100 + len(new))
    mark_values(b, dim)
    if zero_queries:
        b.qkv.zero_()
    print("split parts", heads, dim, block, seq, zero_queries, flush=True)
    check(b, "split", max_query_len=1)


@pytest.mark.parametrize("zero_queries", [True, False])
@pytest.mark.parametrize("heads,kv_heads,dim,block,new,seq", [
    (8, 1, 128, 64, [300], [3000]), (4, 4, 64, 16, [65, 80], [2500, 700]), (4, 1, 128, 256, [20], [9000]),
    (1, 1, 128, 32, [700], [2000])])
def test_prompt_parts_all_count_once(gpu_lib, heads, kv_heads, dim, block, new, seq, zero_queries):
    """Row tiles whose keys several workgroups share."""
    b = Batch(new, seq, heads, kv_heads, dim, block, seed=110 + len(new))
    mark_values(b, dim)
    if zero_queries:
        b.qkv.zero_()
    print("prompt parts", heads, dim, block, seq, zero_queries, flush=True)
    check(b, "prompt", max_query_len=max(new))
