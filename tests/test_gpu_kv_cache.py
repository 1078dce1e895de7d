"""The 4-bit cache's step bookkeeping, store and read-back against oracle/kv4_oracle.py: integers
and cache bytes are equal, values equal the definition's rounded to bf16."""
import importlib
import random

import pytest
import torch

from oracle import kv4_oracle as ora

pytestmark = pytest.mark.gpu

attn = importlib.import_module("llm-serve_amd.layers.attention")


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def run_step(query, context, tables, free, block, tokens):
    t = int32(tables)
    for _ in range(2):  # the lists are not consumed: again, the same
        s = attn.kv_step(int32(query), int32(context), t, int32(free), block_size=block, num_tokens=tokens)
    assert s.block_tables is t
    want = ora.step(query, context, tables, free, block, tokens)
    got = (s.cu_query_lens.tolist(), s.seq_lens.tolist(), s.positions.tolist(), s.slots.tolist(), t.tolist(),
           int(s.blocks_used))
    for g, w in zip(got, want):
        assert g == w


def random_step(rng, requests, block, most_new, most_context, pad):
    query = [rng.choice([0, 1, 1, rng.randint(0, most_new)]) for _ in range(requests)]
    context = [rng.choice([0, rng.randint(0, most_context), block * rng.randint(0, most_context // block + 1)])
               for _ in range(requests)]
    have = [-(-c // block) for c in context]
    need = [-(-(c + n) // block) for c, n in zip(context, query)]
    width = max(1, max(need)) + rng.randint(0, 2)
    ids = list(range(sum(need) + 4))
    rng.shuffle(ids)
    tables, at = [], 0
    for n in have:
        tables.append(ids[at:at + n] + [rng.randint(0, 9)] * (width - n))
        at += n
    return query, context, tables, ids[at:], sum(query) + pad


@pytest.mark.parametrize("requests,block,most_new,most_context,pad", [
    (1, 16, 1, 40, 0), (3, 16, 20, 100, 2), (8, 256, 600, 700, 1), (64, 32, 9, 300, 7), (255, 16, 3, 64, 0),
    (257, 64, 5, 500, 3), (600, 128, 4, 400, 0)])
def test_step(gpu_lib, requests, block, most_new, most_context, pad):
    rng = random.Random(requests)
    for _ in range(3):
        run_step(*_reorder(random_step(rng, requests, block, most_new, most_context, pad), block))


def _reorder(s, block):
    query, context, tables, free, tokens = s
    return query, context, tables, free, block, tokens


def test_step_edges(gpu_lib):
    run_step([0], [0], [[3, 4]], [7], 16, 0)                     # nothing
    run_step([0, 0], [5, 16], [[1, 2], [3, 4]], [7], 16, 3)      # padded requests and rows only
    run_step([16], [16], [[1, 2]], [7], 16, 16)                  # exactly one new block
    run_step([1], [0], [[9]], [0], 256, 1)                       # the first token
    run_step([40, 40], [0, 0], [[0] * 3, [0] * 3], [5, 6, 7, 8], 16, 80)  # the free list runs out
    run_step([40], [16], [[4, 0]], [5, 6, 7], 16, 40)            # the table is too narrow
    run_step([3], [2], [[-1]], [5], 16, 3)                       # a bad entry names no slot
    run_step([-4, 2, 3], [7, -9, 1], [[1], [2], [3]], [5, 6], 16, 5)  # negative lengths are none
    run_step([5, 5], [0, 0], [[0], [0]], [5, 6], 16, 7)          # more tokens than rows
    run_step([2], [2 ** 20], [[2 ** 27 + 1] * 65540], [5], 16, 2)  # slots beyond 2^31 are none
    run_step([1], [0], [[0]], [], 16, 1)                         # no free list


def test_step_strided_tables(gpu_lib):
    wide = torch.full((3, 8), 77, dtype=torch.int32, device="cuda")
    tables = wide[:, :4]
    tables.copy_(int32([[1, 2, 0, 0], [3, 0, 0, 0], [0, 0, 0, 0]]))
    s = attn.kv_step(int32([20, 1, 2]), int32([20, 16, 0]), tables, int32([10, 11, 12, 13]), block_size=16, num_tokens=23)
    assert tables.tolist() == [[1, 2, 10, 0], [3, 11, 0, 0], [12, 0, 0, 0]] and bool((wide[:, 4:] == 77).all())
    assert s.slots.tolist()[20:] == [11 * 16, 12 * 16, 12 * 16 + 1]


def test_step_largest(gpu_lib):
    """4096 requests, 2^18 rows: offsets and slots against sums on the host."""
    gen = torch.Generator().manual_seed(1)
    query = torch.full((4096,), 64, dtype=torch.int32)
    context = torch.randint(0, 1000, (4096,), generator=gen, dtype=torch.int32)
    have, need = (context + 15) // 16, (context + query + 15) // 16
    tables = torch.arange(4096, dtype=torch.int32)[:, None] * 70 + torch.arange(70, dtype=torch.int32)
    free = torch.arange(4096 * 70, 4096 * 70 + int((need - have).sum()), dtype=torch.int32)
    s = attn.kv_step(query.cuda(), context.cuda(), tables.cuda(), free.cuda(), block_size=16, num_tokens=1 << 18)
    row = torch.arange(1 << 18)
    request = row // 64
    position = context[request] + row % 64
    first = torch.cumsum(need - have, 0) - (need - have)
    index = position // 16
    block = torch.where(index < have[request], request * 70 + index,
                        4096 * 70 + first[request] + index - have[request])
    assert torch.equal(s.positions.cpu().long(), position.long())
    assert torch.equal(s.slots.cpu().long(), (block * 16 + position % 16).long())
    assert int(s.blocks_used) == len(free)


def rows(gen, tokens, kv_heads, dim):
    x = torch.randn(tokens, 3 * kv_heads, dim, generator=gen)
    x[:, :, ::17] *= 8
    return x.to(torch.bfloat16)


def check_store(k, v, slots, blocks, block, seed=0):
    """Bytes equal the oracle's, untouched ones included; read back, values equal too."""
    gen = torch.Generator().manual_seed(seed)
    heads, dim = k.shape[1:]
    cache = torch.randint(0, 256, (blocks, heads, block * (dim + 8)), generator=gen, dtype=torch.uint8)
    mine = cache.cuda()
    attn.store_kv_int4(k, v, mine, int32(slots), block_size=block)
    ora.store(k, v, cache, torch.tensor(slots), block)
    assert torch.equal(mine.cpu(), cache)
    got = attn.load_kv_int4(mine, int32(slots), block_size=block)
    want = ora.load(cache, slots, block)[:2]
    for g, w in zip(got, want):
        w = w.to(torch.bfloat16)
        assert torch.equal(g.cpu().nan_to_num(5.0), w.nan_to_num(5.0))
    return got


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,kv_heads,block", [(1, 1, 16), (1, 8, 256), (3, 2, 16), (5, 8, 32), (17, 3, 64),
                                                   (130, 2, 128)])
def test_store_and_load(gpu_lib, tokens, kv_heads, dim, block):
    gen = torch.Generator().manual_seed(tokens)
    qkv = rows(gen, tokens, kv_heads, dim).cuda()
    blocks = -(-tokens // block) + 2
    slots = torch.randperm(blocks * block, generator=gen)[:tokens].tolist()
    check_store(qkv[:, kv_heads:2 * kv_heads], qkv[:, 2 * kv_heads:], slots, blocks, block)


def test_store_skips_slots_outside(gpu_lib):
    gen = torch.Generator().manual_seed(3)
    qkv = rows(gen, 6, 2, 128).cuda()
    check_store(qkv[:, :2], qkv[:, 2:4], [-1, 3, 32, 2 ** 31 - 1, -2 ** 31, 31], 2, 16)


@pytest.mark.parametrize("dim", [64, 128])
def test_store_special_rows(gpu_lib, dim):
    """Zeros, constants, one sign, one large channel, exact halves, subnormals, the largest finite
    values, NaN and infinities."""
    big = 3.3895313892515355e38
    x = torch.zeros(16, 1, dim)
    x[1] = 1.0
    x[2] = -2.5
    x[3] = torch.linspace(1, 3, dim)
    x[4] = -torch.linspace(0.5, 90, dim)
    x[5, 0, 7] = 1e30
    x[6] = torch.arange(dim).float() % 16 * 0.5 - 3.75  # quotients half way between codes
    x[6, 0, 0], x[6, 0, 1] = -3.75, 3.75
    x[7] = torch.linspace(-9e-41, 9e-41, dim)
    x[8] = torch.linspace(-1e-38, 1e-38, dim)
    x[9, 0, 3], x[9, 0, 4] = big, -big
    x[10] = torch.randn(dim, generator=torch.Generator().manual_seed(1))
    x[10, 0, dim - 1] = float("nan")
    x[11, 0, 0] = float("inf")
    x[12, 0, 5] = -float("inf")
    x[13] = torch.linspace(-7.5, 7.5, dim)
    x[14, 0, 0] = 1e-45
    x[15] = -1e-40
    x = x.to(torch.bfloat16).cuda()
    k, _ = check_store(x, x.flip(0).contiguous(), list(range(5, 21)), 2, 16)
    bad = torch.isnan(k.float()).flatten(1)
    assert [bool(b.all()) for b in bad] == [i in (10, 11, 12) for i in range(16)]


def test_store_halves_are_exact(gpu_lib):
    """Every pair of a bf16 scale's mantissa and a value near a border between two codes."""
    scales = (torch.arange(128, 256).double() / 128).to(torch.bfloat16).double()
    x = torch.zeros(128, 1, 128, dtype=torch.float64)
    for i, s in enumerate(scales.tolist()):
        border = (torch.arange(-7, 7).double() + 0.5) * s
        near = border.to(torch.bfloat16)
        step = near.view(torch.int16)
        row = torch.cat([(step + d).view(torch.bfloat16).double() for d in (-1, 0, 1)])
        x[i, 0, :42] = row
        x[i, 0, 100], x[i, 0, 101] = float(torch.tensor(-7 * s).bfloat16()), float(torch.tensor(8 * s).bfloat16())
    x = x.to(torch.bfloat16).cuda()
    check_store(x, x, list(range(128)), 8, 16)


def test_store_and_load_beyond_4_gib(gpu_lib):
    gen = torch.Generator().manual_seed(4)
    qkv = rows(gen, 9, 8, 128).cuda()
    blocks = (5 << 30) // (8 * 64 * 136)
    cache = torch.empty(blocks, 8, 64 * 136, dtype=torch.uint8, device="cuda")
    slots = [(blocks - 1) * 64 + i for i in range(9)]
    attn.store_kv_int4(qkv[:, 8:16], qkv[:, 16:], cache, int32(slots), block_size=64)
    got = attn.load_kv_int4(cache, int32(slots), block_size=64)
    small = check_store(qkv[:, 8:16], qkv[:, 16:], list(range(9)), 1, 64)
    assert torch.equal(got[0], small[0]) and torch.equal(got[1], small[1])


def test_round_trip_error(gpu_lib):
    """A channel is within half a step of its value, and half a step more where the bf16 scale
    (rounded by up to 2^-8) misses the range's ends: 15 steps of 2^-8 each."""
    gen = torch.Generator().manual_seed(6)
    x = rows(gen, 200, 8, 128).cuda()[:, :8]
    cache = attn.new_kv_cache_int4(2, 128, 8, 128)
    slots = int32(list(range(200)))
    attn.store_kv_int4(x, x, cache, slots, block_size=128)
    k, v = attn.load_kv_int4(cache, slots, block_size=128)
    f = x.double()
    step = (f.amax(-1, True).clamp(min=0) - f.amin(-1, True).clamp(max=0)) / 15
    limit = step * (1 + 2.0 ** -8) * (0.5 + 15 * 2.0 ** -8) + 2.0 ** -8 * f.abs()
    for y in (k, v):
        assert bool(((y.double() - f).abs() <= limit * (1 + 1e-6)).all())
