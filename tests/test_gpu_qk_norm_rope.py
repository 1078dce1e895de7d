"""Per-head norm and position rotation, alone and on the way into the 4-bit cache: the bits of the
documented fp32 arithmetic, within the derived tolerance of the 64-bit formula (oracle/prompt_oracle.py),
for head layouts, sizes, strides and positions where they can go wrong."""
import importlib

import pytest
import torch

from oracle import prompt_oracle as ora

pytestmark = pytest.mark.gpu

attn = importlib.import_module("llm-serve_amd.layers.attention")
rope = importlib.import_module("llm-serve_amd.layers.rotary_embedding")

LAYOUTS = [(32, 8, 128), (5, 1, 128), (16, 16, 64), (7, 7, 64), (40, 8, 128), (1, 1, 64), (6, 3, 128)]


def rows(gen, tokens, heads, kv_heads, dim, factor=1.0):
    """q, k, v as views of one projection's output."""
    x = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=gen, device="cuda") * factor
    return x.to(torch.bfloat16).split((heads, kv_heads, kv_heads), 1)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def weight(gen, dim):
    return (1 + 0.3 * torch.randn(dim, generator=gen, device="cuda")).to(torch.bfloat16)


def check(got, x, positions, table, rotary, w=None, eps=1e-6, base=10000.0):
    assert got.dtype == torch.bfloat16 and got.is_contiguous() and got.shape == x.shape
    assert torch.equal(got, ora.turn_fp32(x, positions, table, w, eps))
    want, size = ora.turn(x, positions, rotary, base, w, eps)
    assert bool(((got.double() - want).abs() <= ora.turn_tolerance(want, size)).all())


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("tokens", [1, 3, 64, 511, 513, 700])
def test_rows(gpu_lib, heads, kv_heads, dim, tokens):
    gen = generator(tokens + heads)
    q, k, _ = rows(gen, tokens, heads, kv_heads, dim)
    positions = torch.randint(0, 3000, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    wq, wk = weight(gen, dim), weight(gen, dim)
    for rotary in (dim, dim // 2, 16, dim - 16):
        table = rope.rotary_table(rotary, 3000)
        for q_weight, k_weight in ((wq, wk), (None, None), (None, wk), (wq, None)):
            a, b = rope.qk_norm_rope(q, k, positions, table, q_weight=q_weight, k_weight=k_weight)
            check(a, q, positions, table, rotary, q_weight)
            check(b, k, positions, table, rotary, k_weight)


@pytest.mark.parametrize("dim", [64, 128])
def test_far_positions_and_the_table(gpu_lib, dim):
    """Positions to the end of a long context, of which 32-bit angles would have lost the digits."""
    gen = generator(1)
    q, k, _ = rows(gen, 40, 4, 2, dim)
    count = 131072
    layer = rope.RotaryEmbedding(dim, dim, count, 1000000.0)
    positions = (count - 1 - torch.arange(40, device="cuda") * 3000).to(torch.int32)
    a, b = layer(positions, q, k, q_weight=weight(gen, dim), eps=1e-5)
    check(b, k, positions, layer.cos_sin_cache, dim, base=1000000.0)
    assert bool(torch.isfinite(a.float()).all())


@pytest.mark.parametrize("factor,eps", [(1e-18, 1e-6), (1e-18, 0.0), (1e18, 1e-6), (3e-3, 1e-2), (0.0, 1e-6)])
def test_row_sizes(gpu_lib, factor, eps):
    """Rows far from 1, whose squares leave fp32's range, and rows of zeros."""
    gen = generator(2)
    q, k, _ = rows(gen, 33, 4, 4, 128, factor)
    positions = torch.arange(33, device="cuda", dtype=torch.int32)
    table = rope.rotary_table(128, 64)
    w = weight(gen, 128)
    a, b = rope.qk_norm_rope(q, k, positions, table, q_weight=w, k_weight=None, eps=eps)
    assert torch.equal(a, ora.turn_fp32(q, positions, table, w, eps))
    check(b, k, positions, table, 128)


@pytest.mark.parametrize("tokens", [5, 600])
def test_rows_that_are_no_numbers_stay_their_own(gpu_lib, tokens):
    """NaN and infinities reach their own row alone, and in a row without a norm their own channels and
    those that turn with them; channels that do not turn keep infinities."""
    gen = generator(3)
    q, k, _ = rows(gen, tokens, 6, 2, 128)
    clean_q, clean_k = q.clone(), k.clone()
    q[2, 3, 5], q[1, 0, 100], k[0, 1, 70] = float("nan"), float("inf"), float("-inf")
    positions = torch.arange(1, tokens + 1, device="cuda", dtype=torch.int32)
    table = rope.rotary_table(64, 4096)
    a, b = rope.qk_norm_rope(q, k, positions, table)
    c, d = rope.qk_norm_rope(clean_q, clean_k, positions, table)
    spoilt = torch.zeros(tokens, 6, 128, dtype=torch.bool, device="cuda")
    spoilt[2, 3, [5, 37]] = True
    spoilt[1, 0, 100] = True
    assert torch.equal(a[~spoilt], c[~spoilt]) and bool(torch.isnan(a[2, 3, [5, 37]]).all()) and float(a[1, 0, 100]) == float("inf")
    assert float(b[0, 1, 70]) == float("-inf") and torch.equal(b[1:], d[1:])
    w = weight(gen, 128)
    a, _ = rope.qk_norm_rope(q, k, positions, table, q_weight=w, k_weight=w)
    c, _ = rope.qk_norm_rope(clean_q, clean_k, positions, table, q_weight=w, k_weight=w)
    row = spoilt.any(-1)
    assert torch.equal(a[~row], c[~row]) and bool(torch.isnan(a[2, 3]).all()) and bool(torch.isnan(a[1, 0, 100]))


@pytest.mark.parametrize("tokens", [7, 520])
def test_positions_outside_the_table(gpu_lib, tokens):
    gen = generator(4)
    q, k, v = rows(gen, tokens, 6, 2, 128)
    positions = torch.arange(tokens, device="cuda", dtype=torch.int32) % 60
    positions[1], positions[4], positions[5] = -1, 60, -(1 << 31)
    table = rope.rotary_table(64, 60)
    bad = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    bad[[1, 4, 5]] = True
    a, b = rope.qk_norm_rope(q, k, positions, table, q_weight=weight(gen, 128))
    for x in (a, b):
        assert bool(torch.isnan(x[bad]).all()) and bool(torch.isfinite(x[~bad]).all())
    cache = attn.new_kv_cache_int4(tokens // 16 + 1, 16, 2, 128)
    slots = torch.arange(tokens, device="cuda", dtype=torch.int32)
    attn.append_kv_int4(q, k, v, cache, slots, positions, table, block_size=16)
    x, y = attn.load_kv_int4(cache, slots, block_size=16)
    assert bool(torch.isnan(x[bad]).all()) and bool(torch.isfinite(x[~bad]).all()) and bool(torch.isfinite(y).all())


def test_strides_and_alignment(gpu_lib):
    """Rows padded, tensors off their alignment, heads apart by any stride, a table and weights that are
    views, positions strided: the values of their contiguous copies."""
    gen = generator(5)
    tokens, dim = 50, 128
    wide = torch.randn(tokens, 9, dim + 8, generator=gen, device="cuda").to(torch.bfloat16)
    q, k, v = wide[:, :5, :dim], wide[:, 5:7, 8:], wide[:, 7:9, 4:dim + 4]  # v: rows off 16 bytes
    flat = torch.randn(tokens * 3 * dim + 1, generator=gen, device="cuda").to(torch.bfloat16)
    odd = flat[1:].view(tokens, 3, dim)
    swapped = torch.randn(5, tokens, dim, generator=gen, device="cuda").to(torch.bfloat16).transpose(0, 1)
    strided = torch.randint(0, 90, (tokens, 2), generator=gen, device="cuda", dtype=torch.int32)[:, 1]
    table = torch.cat((torch.zeros(90, 3, device="cuda"), rope.rotary_table(128, 90)), 1)[:, 3:]
    w = torch.randn(dim * 2, generator=gen, device="cuda").to(torch.bfloat16)[1::2]
    one = odd[:, :1].expand(tokens, 4, dim)  # heads that share their rows
    for a, b in ((q, k), (odd, k), (swapped, odd), (one, q), (q[::2].repeat_interleave(2, 0), v)):
        got = rope.qk_norm_rope(a, b, strided, table, q_weight=w, k_weight=w)
        want = rope.qk_norm_rope(a.contiguous(), b.contiguous(), strided.contiguous(), table.contiguous(),
                                 q_weight=w.contiguous(), k_weight=w.contiguous())
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        check(got[0], a, strided, table, 128, w)
    cache, other = (attn.new_kv_cache_int4(8, 16, 2, dim) for _ in range(2))
    slots = torch.randperm(100, generator=gen, device="cuda").to(torch.int32)[::2]
    attn.append_kv_int4(q, k, v, cache, slots, strided, table, block_size=16, k_weight=w)
    attn.store_kv_int4(rope.qk_norm_rope(q, k, strided, table, k_weight=w)[1], v.contiguous(), other, slots, block_size=16)
    assert torch.equal(cache, other)


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("tokens,block", [(1, 16), (61, 256), (512, 32), (514, 64), (1030, 128)])
def test_append_is_the_two_calls(gpu_lib, heads, kv_heads, dim, tokens, block):
    """One launch gives the bits of the rotation and the store after it: queries, keys, every byte of
    the cache, those of the slots that are not named as they were."""
    gen = generator(tokens + kv_heads)
    q, k, v = rows(gen, tokens, heads, kv_heads, dim)
    blocks = tokens // block + 2
    positions = torch.randint(0, 5000, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    slots = torch.randperm(blocks * block, generator=gen, device="cuda")[:tokens].to(torch.int32)
    slots[1::5] = -1
    slots[2::17] = blocks * block + 3
    for rotary, norm, keys in ((dim, True, True), (dim // 2, False, False)):
        table = rope.rotary_table(rotary, 5000)
        w = weight(gen, dim) if norm else None
        cache = torch.randint(0, 256, (blocks, kv_heads, block * (dim + 8)), generator=gen, device="cuda", dtype=torch.uint8)
        other = cache.clone()
        got = attn.append_kv_int4(q, k, v, cache, slots, positions, table, block_size=block, q_weight=w, k_weight=w,
                                  return_keys=keys)
        a, b = rope.qk_norm_rope(q, k, positions, table, q_weight=w, k_weight=w)
        attn.store_kv_int4(b, v, other, slots, block_size=block)
        assert torch.equal(got[0] if keys else got, a) and (not keys or torch.equal(got[1], b))
        assert torch.equal(cache, other)


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("tokens,block", [(2047, 64), (2049, 256), (2501, 16)])
def test_larger_steps(gpu_lib, heads, kv_heads, dim, tokens, block):
    """Where a wave takes more of a token's rows, and in front of that."""
    gen = generator(tokens + heads)
    q, k, v = rows(gen, tokens, heads, kv_heads, dim)
    positions = torch.randint(0, 3000, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    wq, wk = weight(gen, dim), weight(gen, dim)
    table = rope.rotary_table(dim, 3000)
    a, b = rope.qk_norm_rope(q, k, positions, table, q_weight=wq, k_weight=wk)
    check(a, q, positions, table, dim, wq)
    check(b, k, positions, table, dim, wk)
    blocks = tokens // block + 2
    slots = torch.randperm(blocks * block, generator=gen, device="cuda")[:tokens].to(torch.int32)
    cache, other = (attn.new_kv_cache_int4(blocks, block, kv_heads, dim) for _ in range(2))
    attn.store_kv_int4(b, v, cache, slots, block_size=block)
    c, d = attn.append_kv_int4(q, k, v, other, slots, positions, table, block_size=block, q_weight=wq, k_weight=wk,
                               return_keys=True)
    assert torch.equal(a, c) and torch.equal(b, d) and torch.equal(cache, other)


def test_no_tokens(gpu_lib):
    q = torch.zeros(0, 4, 128, dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    table = rope.rotary_table(128, 4)
    a, b = rope.qk_norm_rope(q, q[:, :2], none, table)
    assert a.shape == (0, 4, 128) and b.shape == (0, 2, 128)
    cache = attn.new_kv_cache_int4(1, 16, 2, 128)
    a, b = attn.append_kv_int4(q, q[:, :2], q[:, :2], cache, none, none, table, block_size=16, return_keys=True)
    assert a.shape == (0, 4, 128) and b.shape == (0, 2, 128) and not bool(cache.any())


def test_captured_and_on_another_stream(gpu_lib):
    """A captured append replayed over new rows, eager work of its own between the replays, and the same
    call on a side stream."""
    gen = generator(8)
    tokens = 24
    q, k, v = (t.contiguous() for t in rows(gen, tokens, 8, 2, 128))
    positions = torch.randint(0, 500, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    slots = torch.randperm(64, generator=gen, device="cuda")[:tokens].to(torch.int32)
    table, w = rope.rotary_table(128, 500), weight(gen, 128)
    cache = attn.new_kv_cache_int4(4, 16, 2, 128)

    def call(into):
        return attn.append_kv_int4(q, k, v, into, slots, positions, table, block_size=16, q_weight=w, k_weight=w,
                                   return_keys=True)

    call(cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(cache)
    side = torch.cuda.Stream()
    for i in range(5):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        positions.copy_(torch.randint(0, 500, (tokens,), generator=gen, device="cuda"))
        other = cache.clone()
        want = call(other)
        third = cache.clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = call(third)
        torch.cuda.current_stream().wait_stream(side)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(got, want, again)), i
        assert torch.equal(cache, other) and torch.equal(cache, third), i


def test_refusals(gpu_lib):
    """Arguments that the kernels cannot take raise in front of any launch."""
    gen = generator(9)
    q, k, v = rows(gen, 6, 4, 2, 128)
    positions = torch.arange(6, device="cuda", dtype=torch.int32)
    table, w = rope.rotary_table(128, 64), weight(gen, 128)
    cache = attn.new_kv_cache_int4(2, 16, 2, 128)
    for change in ({"q": q.float()}, {"q": q[..., :96]}, {"q": q[0]}, {"k": k[:5]}, {"k": k[..., :64]}, {"k": k.cpu()},
                   {"k": k[:, :0]}, {"positions": positions.long()}, {"positions": positions[:5]},
                   {"positions": positions.cpu()}, {"table": table.half()}, {"table": table[:0]}, {"table": table[:, :8]},
                   {"table": table[:, :24]}, {"table": torch.cat((table, table), -1)}, {"table": table.cpu()},
                   {"q_weight": w.float()}, {"k_weight": w[:64]}, {"q_weight": w.cpu()}, {"eps": -1e-6},
                   {"eps": float("nan")}, {"eps": float("inf")}):
        args = {**dict(q=q, k=k, positions=positions, table=table), **change}
        with pytest.raises(ValueError):
            rope.qk_norm_rope(**args)
        with pytest.raises(ValueError):
            attn.append_kv_int4(**{**dict(v=v, cache=cache, slots=positions, block_size=16), **args})
    for change in ({"v": v[:5]}, {"v": v.float()}, {"v": v[:, :1]}, {"v": v.cpu()}, {"slots": positions[:5]},
                   {"slots": positions.long()}, {"slots": positions.cpu()}, {"cache": cache[..., :64]}, {"cache": cache.cpu()},
                   {"cache": attn.new_kv_cache_int4(2, 16, 2, 64)}, {"cache": attn.new_kv_cache_int4(2, 16, 4, 128)},
                   {"block_size": 32}):
        with pytest.raises(ValueError):
            attn.append_kv_int4(**{**dict(q=q, k=k, v=v, cache=cache, slots=positions, positions=positions, table=table,
                                          block_size=16), **change})
    assert not bool(cache.any())
