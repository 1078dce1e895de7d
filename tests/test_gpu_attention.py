"""Attention over the 4-bit cache against its definition in 64 bits (oracle/kv4_oracle.py): one
token to long prompts, ragged and empty sequences, pages that end inside a tile, stale pages,
trees, bad tables, strides, streams and graph replays.  The tolerance is the oracle's bound."""
import importlib
import random

import pytest
import torch

from oracle import kv4_oracle as ora

pytestmark = pytest.mark.gpu

attn = importlib.import_module("llm-serve_amd.layers.attention")


def bf16(shape, gen, spread=1.0):
    return (torch.randn(shape, generator=gen) * spread).to(torch.bfloat16)


class Batch:
    """Sequences of `seq` tokens whose last `new` are queries, on shuffled pages of a cache that
    the oracle filled; everything behind a sequence's end holds NaN scales and zero points."""

    def __init__(self, new, seq, heads, kv_heads, dim, block, seed=0, pad=0, width=None, extra_blocks=3):
        gen = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.new, self.seq, self.block = new, seq, block
        counts = [-(-s // block) for s in seq]
        blocks = sum(counts) + extra_blocks
        order = list(range(blocks))
        rng.shuffle(order)
        self.width = width or max(1, max(counts))
        self.tables, at = [], 0
        for n in counts:
            self.tables.append(order[at:at + n] + [order[-1]] * (self.width - n))
            at += n
        page = block * (dim + 8)
        self.cache = torch.empty(blocks, kv_heads, page, dtype=torch.uint8)
        self.cache.view(torch.int32).fill_(0x7FC07FC0)
        self.cache[..., : block * dim] = torch.randint(0, 256, (blocks, kv_heads, block * dim), generator=gen,
                                                       dtype=torch.uint8)
        words = self.cache.view(torch.int32)
        first = block * dim // 4
        for r, n in enumerate(seq):
            for p in range(0, n, block):
                page_words = words[self.tables[r][p // block]]
                held = min(block, n - p)
                for part in (0, 1):
                    scale = (torch.rand(kv_heads, held, generator=gen) * 0.4 + 0.02).to(torch.bfloat16)
                    zero = torch.randint(0, 16, (kv_heads, held), generator=gen, dtype=torch.int32)
                    bits = scale.view(torch.int16).to(torch.int32) << 16
                    page_words[:, first + part * block:first + part * block + held] = bits | 0x4300 | zero
        self.offsets = [0]
        for n in new:
            self.offsets.append(self.offsets[-1] + n)
        rows = self.offsets[-1] + pad
        self.qkv = bf16((rows, heads + 2 * kv_heads, dim), gen).cuda()
        self.q = self.qkv[:, :heads]

    def int32(self, values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def args(self):
        return (self.q, self.cache.cuda(), self.int32(self.tables), self.int32(self.seq), self.int32(self.offsets))

    def check(self, got, **kw):
        want, spread = ora.attention(self.q, self.cache, self.tables, self.seq, self.offsets, self.block, **kw)
        got = got.cpu().double()
        off = (got - want).abs()
        limit = ora.tolerance(want, spread)
        bad = ~(off <= limit)
        assert not bool(bad.any()), (int(bad.sum()), float((off / limit).nan_to_num(9e9).max()), bad.nonzero()[:3])

    def run(self, **kw):
        return attn.attention_int4(*self.args(), block_size=self.block, **kw)


SHAPES = [(32, 8, 128), (8, 8, 64), (10, 2, 128), (16, 1, 128), (16, 2, 64)]


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("block", [16, 64, 256])
def test_decode(gpu_lib, heads, kv_heads, dim, block):
    """One row a request: sequences of 1 token, around 16- and 32-key tiles, 128-key units, blocks."""
    seq = [1, 15, 16, 17, 31, 33, 127, 128, 129, 255, 257, 300]
    b = Batch([1] * len(seq), seq, heads, kv_heads, dim, block, seed=heads + block)
    print("decode", heads, kv_heads, dim, block, flush=True)
    b.check(b.run(max_query_len=1))


@pytest.mark.parametrize("new,seq", [([1], [1]), ([1], [1000]), ([4, 4, 4], [4, 70, 333]), ([8, 1, 3], [8, 500, 3]),
                                     ([17], [17]), ([100, 1, 2], [100, 64, 200]), ([33, 65], [200, 65])])
@pytest.mark.parametrize("hint", [1, None])
def test_causal_rows(gpu_lib, new, seq, hint):
    """Several rows a request, whole prompts among them; the hint changes no result's validity."""
    b = Batch(new, seq, 8, 2, 128, 32, seed=sum(seq))
    print("causal", new, seq, hint, flush=True)
    b.check(b.run(max_query_len=hint))


@pytest.mark.parametrize("dim", [64, 128])
def test_tree_masks(gpu_lib, dim):
    """Rows see their cached tokens and the new ones their bits name; no bits and no cached
    tokens leave a row empty, which is zero."""
    new, seq = [8, 5, 64, 3], [200, 5, 64, 3]
    b = Batch(new, seq, 8, 2, dim, 16, seed=5)
    gen = random.Random(3)
    masks = [gen.getrandbits(64) for _ in range(sum(new))]
    masks[8] = 0               # the second request's first row: nothing at all
    masks[9] = 1 << 63         # and a bit behind its new tokens
    masks[-1] = (1 << 64) - 1  # every new token, later ones too
    signed = [m - (1 << 64) if m >> 63 else m for m in masks]
    out = b.run(tree_mask=torch.tensor(signed, dtype=torch.int64, device="cuda"))
    assert torch.equal(out[8], torch.zeros_like(out[8])) and torch.equal(out[9], torch.zeros_like(out[9]))
    b.check(out, tree_mask=masks)


def test_empty_sequences_and_padding(gpu_lib):
    """Requests without rows, rows without keys (a sequence length of 0), padded rows."""
    b = Batch([1, 0, 2, 0], [40, 7, 30, 0], 8, 2, 128, 16, seed=9, pad=5)
    q, cache, tables, seq, offsets = b.args()
    out = attn.attention_int4(q, cache, tables, seq, offsets, block_size=16)
    b.check(out)
    assert torch.equal(out[3:], torch.zeros_like(out[3:]))
    mine = torch.full_like(out, 7.0)
    got = attn.attention_int4(q, cache, tables, seq, offsets, block_size=16, out=mine)
    assert got is mine and torch.equal(mine[:3], out[:3]) and bool((mine[3:] == 7.0).all())
    none = attn.attention_int4(q, cache, tables, seq * 0, offsets, block_size=16)
    assert torch.equal(none, torch.zeros_like(none))


def test_bad_pages_are_not_seen(gpu_lib):
    """Table entries outside the cache: their keys are masked, nothing is read there; a length
    beyond the table's width reaches only the table's keys."""
    b = Batch([1, 2], [100, 90], 8, 2, 128, 16, seed=12)
    b.tables[0][1] = -1
    b.tables[0][4] = b.cache.shape[0]
    b.tables[1] = [2 ** 31 - 1] * b.width
    b.check(b.run())
    b.seq = [b.width * 16 + 1000, 90]
    b.new, b.offsets = [1, 2], [0, 1, 3]
    words = b.cache.view(torch.int32)
    for page in b.tables[0]:
        if 0 <= page < b.cache.shape[0]:
            words[page, :, 16 * 128 // 4:] = 0x3E004305
    b.check(b.run())


def test_nan_in_unseen_keys(gpu_lib):
    """A stored row that is NaN reaches the rows that see it and no other: later drafts of a
    causal batch, hidden nodes of a tree."""
    b = Batch([4], [50], 8, 2, 128, 16, seed=2)
    words = b.cache.view(torch.int32)
    token = 48
    page = words[b.tables[0][token // 16]]
    for part in (0, 1):
        page[:, 16 * 128 // 4 + part * 16 + token % 16] = 0x7FC04300
    out = b.run()
    assert bool(torch.isfinite(out[:2].float()).all()) and bool(torch.isnan(out[2:].float()).all())
    masks = [1, 1, 4, 9]
    out = b.run(tree_mask=torch.tensor(masks, dtype=torch.int64, device="cuda"))
    nan = torch.isnan(out.float()).flatten(1)
    assert [bool(x.all()) for x in nan] == [False, False, True, False] and not bool(nan[[0, 1, 3]].any())


def test_extreme_queries(gpu_lib):
    """Scores far beyond exp's range, of either sign, and a query of zeros."""
    b = Batch([1, 1, 1], [300, 300, 40], 8, 2, 128, 64, seed=4)
    b.qkv[0] *= 1000
    b.qkv[1] = 0
    b.check(b.run())
    b.qkv[0, 0, 0] = float("nan")
    out = b.run()
    assert bool(torch.isnan(out[0, 0].float()).all()) and bool(torch.isfinite(out[0, 1:].float()).all())


@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_scale(gpu_lib, scale):
    b = Batch([2, 1], [70, 129], 4, 2, 64, 16, seed=6)
    b.check(b.run(scale=scale), scale=scale)


def test_long_sequence_split(gpu_lib):
    """One sequence over many workgroups, and a batch of very unequal lengths."""
    b = Batch([1], [20000], 4, 1, 128, 256, seed=8)
    b.check(b.run(max_query_len=1))
    b = Batch([1] * 9, [6000, 1, 2, 3, 700, 1, 1, 40, 2500], 4, 1, 128, 16, seed=8)
    b.check(b.run(max_query_len=1))


def test_pages_beyond_4_gib(gpu_lib):
    """Pages whose byte offset passes 32 bits give the same output as pages at the start."""
    b = Batch([1, 3], [300, 100], 8, 8, 128, 64, seed=3)
    want = b.run()
    page = b.cache.shape[1] * b.cache.shape[2]
    blocks = (5 << 30) // page
    big = torch.empty(blocks, *b.cache.shape[1:], dtype=torch.uint8, device="cuda")
    n = b.cache.shape[0]
    big[blocks - n:] = b.cache.cuda()
    tables = b.int32(b.tables) + (blocks - n)
    got = attn.attention_int4(b.q, big, tables, b.int32(b.seq), b.int32(b.offsets), block_size=64)
    assert torch.equal(got, want)


def test_layouts(gpu_lib):
    """Queries at any strides, lists in strided views: the same bits."""
    b = Batch([3, 1], [90, 200], 8, 2, 128, 16, seed=10)
    q, cache, tables, seq, offsets = b.args()
    want = attn.attention_int4(q.contiguous(), cache, tables, seq, offsets, block_size=16)
    assert torch.equal(b.run(), want)
    odd = torch.empty(4, 8, 129, dtype=torch.bfloat16, device="cuda")[..., 1:]
    odd.copy_(q)
    assert torch.equal(attn.attention_int4(odd, cache, tables, seq, offsets, block_size=16), want)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(attn.attention_int4(heads_first, cache, tables, seq, offsets, block_size=16), want)
    wide = torch.zeros(2, b.width + 5, dtype=torch.int32, device="cuda")
    wide[:, :b.width] = tables
    assert torch.equal(attn.attention_int4(q, cache, wide[:, :b.width], seq, offsets, block_size=16), want)
    turned = tables.t().contiguous().t()
    assert torch.equal(attn.attention_int4(q, cache, turned, seq, offsets, block_size=16), want)


def test_repeated_and_concurrent_calls_agree(gpu_lib):
    """Bit for bit, on one stream and on two at once (each call has its own workspace)."""
    b = Batch([1] * 5, [3000, 5, 900, 70, 2000], 8, 2, 128, 16, seed=11)
    args = b.args()
    want = attn.attention_int4(*args, block_size=16)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(attn.attention_int4(*args, block_size=16))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_graph_replays_follow_the_lengths(gpu_lib):
    """Two captured graphs with lengths that change between replays, eager calls in between."""
    b = Batch([1] * 4, [400, 300, 200, 100], 8, 2, 128, 16, seed=13)
    q, cache, tables, seq, offsets = b.args()
    q = q.clone()
    attn.attention_int4(q, cache, tables, seq, offsets, block_size=16, max_query_len=1)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = attn.attention_int4(q, cache, tables, seq, offsets, block_size=16, max_query_len=1)
        graphs.append((graph, out))
    for i, lens in enumerate([[400, 300, 200, 100], [1, 2, 3, 4], [399, 1, 150, 16]]):
        seq.copy_(b.int32(lens))
        want = attn.attention_int4(q, cache, tables, seq, offsets, block_size=16, max_query_len=1)
        torch.cuda.synchronize()
        for graph, out in graphs:
            out.fill_(9)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), i


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (10, 2, 128), (4, 4, 64), (16, 1, 64)])
@pytest.mark.parametrize("new,seq", [([80], [80]), ([65, 129], [65, 700]), ([1, 200, 3, 1], [300, 260, 3, 90]),
                                     ([100, 0, 70], [1100, 5, 70])])
def test_prompts(gpu_lib, heads, kv_heads, dim, new, seq):
    """Whole prompts and chunks behind cached tokens, alone and among decode rows: tiles of 256
    rows and 64 keys that end anywhere."""
    b = Batch(new, seq, heads, kv_heads, dim, 16, seed=heads + sum(seq), pad=2)
    print("prompts", heads, kv_heads, dim, new, seq, flush=True)
    b.check(b.run(max_query_len=max(new)))


def test_prompt_tree_masks(gpu_lib):
    new, seq = [90, 2], [300, 40]
    b = Batch(new, seq, 8, 2, 128, 32, seed=21)
    gen = random.Random(4)
    masks = [gen.getrandbits(64) for _ in range(sum(new))]
    masks[7] = 0
    signed = [m - (1 << 64) if m >> 63 else m for m in masks]
    b.check(b.run(tree_mask=torch.tensor(signed, dtype=torch.int64, device="cuda")), tree_mask=masks)


def test_prompt_bad_pages_and_nan_rows(gpu_lib):
    """As for decode rows: pages outside the cache are not seen, a NaN row (its keys, or its values
    alone) reaches the rows that see it and no other."""
    b = Batch([150], [400], 8, 2, 128, 16, seed=22)
    b.tables[0][3], b.tables[0][17] = -1, b.cache.shape[0] + 5
    b.check(b.run())
    words = b.cache.view(torch.int32)
    token = 330  # new token 80
    words[b.tables[0][token // 16], :, 16 * 128 // 4 + 16 + token % 16] = 0x7FC04300
    out = b.run()
    assert bool(torch.isfinite(out[:80].float()).all()) and bool(torch.isnan(out[80:].float()).all())


def test_long_prompt_split(gpu_lib):
    """A chunk whose row tiles are shared by many workgroups."""
    b = Batch([300], [3000], 8, 1, 128, 64, seed=23)
    b.check(b.run())


def test_extreme_prompt_queries(gpu_lib):
    b = Batch([70], [200], 8, 2, 128, 16, seed=24)
    b.qkv[3] *= 1000
    b.qkv[4] = 0
    b.check(b.run())
    b.qkv[5, 0, 0] = float("inf")
    out = b.run()
    assert bool(torch.isnan(out[5, 0].float()).all()) and bool(torch.isfinite(out[5, 1:].float()).all())


def test_graphs_replayed_beside_each_other(gpu_lib):
    """Two captured graphs of split work replayed on two streams while eager calls run on a third:
    none shares a workspace or counters with another."""
    b = Batch([1, 40], [3000, 900], 8, 2, 128, 16, seed=31)
    args = b.args()
    want = attn.attention_int4(*args, block_size=16, max_query_len=40)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [attn.attention_int4(*args, block_size=16, max_query_len=40) for _ in range(4)]
        graphs.append((graph, outs, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, outs, stream in graphs:
            for o in outs:
                o.fill_(3)
        torch.cuda.synchronize()
        for graph, outs, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [attn.attention_int4(*args, block_size=16, max_query_len=40) for _ in range(4)]
        torch.cuda.synchronize()
        for o in eager + graphs[0][1] + graphs[1][1]:
            assert torch.equal(o, want)


def test_capture_without_reserved_counters(gpu_lib, monkeypatch):
    """A pool that has no set yet (or none left) gives a captured call a tensor that its graph clears."""
    monkeypatch.setattr(attn, "SCRATCH", attn._ScratchPool())
    b = Batch([1, 3], [2500, 700], 8, 2, 128, 16, seed=32)
    args = b.args()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attn.attention_int4(*args, block_size=16)
    want = attn.attention_int4(*args, block_size=16)
    for _ in range(3):
        out.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    pool = attn.SCRATCH
    pool._free[0].clear()
    pool._streams.clear()
    assert torch.equal(attn.attention_int4(*args, block_size=16), want)


def test_counters_are_left_zero(gpu_lib):
    b = Batch([1, 300, 5], [3000, 900, 900], 8, 2, 128, 16, seed=33)
    counters = torch.zeros(1024, dtype=torch.int32, device="cuda")
    size = gpu_lib.kv_attention_workspace(306, 3, 8, 2, 128, 16, b.width, 300)
    workspace = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    q, cache, tables, seq, offsets = b.args()
    out = torch.empty(306, 8, 128, dtype=torch.bfloat16, device="cuda")
    gpu_lib.kv_attention(q, cache, tables, seq, offsets, None, out, 128 ** -0.5, 16, 300, True, workspace, counters)
    torch.cuda.synchronize()
    assert not bool(counters.any())
    b.check(out)


@pytest.mark.parametrize("n", [0, 1, 16, 100])
def test_single_request_of_any_length(gpu_lib, n):
    """A single request goes to the prompt kernel alone when the caller's longest query may be a
    prompt: also where it is shorter than said, or empty, with rows behind it."""
    b = Batch([n], [max(n, 1) + 150], 8, 2, 128, 16, seed=40 + n, pad=101 - n)
    out = b.run(max_query_len=101)
    b.check(out)
    assert torch.equal(out[n:], torch.zeros_like(out[n:]))


@pytest.mark.parametrize("hint", [1, 40])
def test_many_requests(gpu_lib, hint):
    """More requests than a wave has lanes, twice over: empty ones, decode rows, drafts, chunks."""
    rng = random.Random(7)
    new = [rng.choice([0, 1, 1, 1, 2, 5, 16, 17, 40]) for _ in range(150)]
    seq = [n + rng.choice([0, 0, 3, 60, 200, 390]) for n in new]
    b = Batch(new, seq, 4, 1, 64, 16, seed=50, pad=3)
    print("many", hint, sum(new), flush=True)
    b.check(b.run(max_query_len=hint))


@pytest.mark.parametrize("heads,kv_heads,new", [(8, 2, [16, 17]), (4, 4, [64, 65]), (32, 1, [2, 3, 20]), (128, 1, [1, 3]),
                                                (7, 1, [9, 10, 37])])
def test_around_the_kernels_border(gpu_lib, heads, kv_heads, new):
    """Requests of up to 64 rows (tokens x heads of a group) and the next longer ones in one call."""
    b = Batch(new, [n + 70 * i for i, n in enumerate(new)], heads, kv_heads, 64, 16, seed=heads)
    b.check(b.run(max_query_len=max(new)))


@pytest.mark.parametrize("hint", [1, 100])
@pytest.mark.parametrize("requests", [1, 2])
def test_fewer_keys_than_rows(gpu_lib, hint, requests):
    """A sequence shorter than its new rows, or empty: the first rows see nothing and are zero."""
    b = Batch([100] * requests, [37, 0][:requests], 8, 2, 128, 16, seed=51)
    out = b.run(max_query_len=hint)
    b.check(out)
    assert torch.equal(out[:63], torch.zeros_like(out[:63])) and torch.equal(out[100:], torch.zeros_like(out[100:]))
    none = Batch([100], [0], 8, 2, 128, 16, seed=52)
    assert not bool(none.run(max_query_len=hint).any())


@pytest.mark.parametrize("hint", [1, 100])
def test_decreasing_offsets_name_no_rows(gpu_lib, hint):
    """Offsets that decrease somewhere: a zero result, `out` left as it was, and the next call right."""
    b = Batch([100, 90, 1], [150, 90, 300], 8, 2, 128, 16, seed=53)
    q, cache, tables, seq, offsets = b.args()
    for broken in ([0, 100, 50, 191], [0, 191, 0, 191], [5, 0, 0, 191], [0, 100, 190, -1]):
        print("offsets", broken, flush=True)
        args = q, cache, tables, seq, b.int32(broken)
        assert not bool(attn.attention_int4(*args, block_size=16, max_query_len=hint).any())
        mine = torch.full((191, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
        attn.attention_int4(*args, block_size=16, max_query_len=hint, out=mine)
        assert bool((mine == 7.0).all())
    b.check(b.run(max_query_len=hint))


@pytest.mark.parametrize("hint", [1, 100])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_power,k_power,v_power,jumps", [(40, -40, 0, 0), (-40, 40, 0, 0), (0, 0, 100, 0), (0, 0, -50, 0),
                                                           (-100, 0, 0, 0), (0, 0, 0, 30)])
def test_powers_of_two(gpu_lib, hint, dim, q_power, k_power, v_power, jumps):
    """Queries, keys and values far from 1, and values whose size differs by up to 2^16 between neighbours
    and up to 2^60 between pages."""
    b = Batch([90, 70], [200, 70], 8, 2, dim, 16, seed=60 + dim)
    gen = torch.Generator().manual_seed(61)
    meta = b.cache.view(torch.int32)[..., 16 * dim // 4:].view(b.cache.shape[0], 2, 2, 16)
    power = torch.zeros(meta.shape, dtype=torch.int32)
    power[:, :, 0], power[:, :, 1] = k_power, v_power
    if jumps:
        power[:, :, 1] += torch.randint(-8, 9, power[:, :, 1].shape, generator=gen, dtype=torch.int32)
        power[:, :, 1] += torch.randint(-jumps, jumps + 1, (power.shape[0], 2, 1), generator=gen, dtype=torch.int32)
    live = (meta >> 23 & 255) != 255
    meta += torch.where(live, power << 23, 0)
    b.qkv.mul_(2.0 ** q_power)
    print("powers", hint, dim, q_power, k_power, v_power, jumps, flush=True)
    b.check(b.run(max_query_len=hint))


@pytest.mark.parametrize("hint", [1, 300])
def test_in_place(gpu_lib, hint):
    """out = q: tiles whose keys several workgroups share read their rows before any is written."""
    b = Batch([1, 300, 5], [3000, 900, 900], 8, 2, 128, 16, seed=70, pad=2)
    q, cache, tables, seq, offsets = b.args()
    want = attn.attention_int4(q, cache, tables, seq, offsets, block_size=16, max_query_len=hint)
    for _ in range(5):
        mine = q.clone(memory_format=torch.contiguous_format)
        got = attn.attention_int4(mine, cache, tables, seq, offsets, block_size=16, max_query_len=hint, out=mine)
        assert got is mine and torch.equal(mine[:306], want[:306]) and torch.equal(mine[306:], q[306:])


def test_largest_and_smallest_batches(gpu_lib):
    """One row and one key in all; 4096 requests of a row or two."""
    one = Batch([1], [1], 1, 1, 64, 16, seed=71)
    one.check(one.run())
    rng = random.Random(72)
    new = [rng.choice([0, 1, 1, 2]) for _ in range(4096)]
    b = Batch(new, [n + rng.choice([0, 1, 14]) for n in new], 1, 1, 64, 16, seed=72)
    print("4096 requests", flush=True)
    for hint in (2, 65):
        b.check(b.run(max_query_len=hint))
