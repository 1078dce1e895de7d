"""Which sizes prompt attention takes, on the CPU (nothing is launched): every step that ``kv_step`` makes, whatever
its number of requests; and steps that it refuses leave the cache as it was."""
import importlib

import pytest
import torch

from prompt_helpers import form

attn = importlib.import_module("llm-serve_amd.layers.attention")


@pytest.fixture(scope="module")
def dll(pkg):
    return pkg.lib().dll


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (40, 8, 128), (64, 8, 128), (128, 8, 128), (16, 16, 64), (32, 32, 64),
                                                (16, 1, 128)])
@pytest.mark.parametrize("requests", [1, 512, 513, 600, 1000, 4096])
@pytest.mark.parametrize("rows", [attn.MAX_STEP_TOKENS, 240000, 180000, 131073])
def test_steps_of_any_number_of_requests(dll, rows, requests, heads, kv_heads, dim):
    assert requests <= attn.MAX_STEP_REQUESTS
    assert dll.w4a16_prompt_attention_workspace(rows, requests, heads, kv_heads, dim) > 0


def test_a_long_prompt(dll):
    """The documented limit of one call: 350000 rows with 32 heads."""
    assert dll.w4a16_prompt_attention_workspace(350000, 1, 32, 8, 128) > 0
    assert dll.w4a16_prompt_attention_workspace(350000, 680, 32, 8, 128) > 0
    assert dll.w4a16_prompt_attention_workspace(380000, 1, 32, 8, 128) == 0


def units(lengths, group, kv_heads, n, shift):
    """The cost units of sequences' row tiles of n rows (sixteenths of a tile of 64 keys, 2^shift of them)."""
    step = -(-(n // 4 >> shift) // group)
    first = step + (64 >> shift)
    tiles = [-(-x * group // n) for x in lengths]
    return kv_heads * sum(m * first + step * m * (m - 1) // 2 for m in tiles)


def shares(lengths, group, kv_heads, n, shift, workers):
    """The parts that equal shares cut the row tiles of one head into: {(sequence, tile): [(first key tile, end)]}."""
    step = -(-(n // 4 >> shift) // group)
    first = step + (64 >> shift)
    total = units(lengths, group, kv_heads, n, shift)
    borders = [w * (total // workers) + min(w, total % workers) for w in range(workers + 1)]
    parts, at = {}, 0
    cuts = iter(borders)
    cut = next(cuts)
    for r, x in enumerate(lengths):
        for head in range(kv_heads):
            for j in range(-(-x * group // n)):
                cost = first + step * j
                keys = -(-((min((j + 1) * n, x * group) - 1) // group + 1) // 64)
                while cut <= at:
                    cut = next(cuts)
                inside = []
                while cut < at + cost:
                    inside.append(cut - at)
                    cut = next(cuts)
                ends = [int(c * (keys * (1.0 / cost))) for c in inside] + [keys]
                parts[r, head, j] = list(zip([0] + ends[:-1], ends))
                at += cost
    assert at == total
    return parts


@pytest.mark.parametrize("shift", [0, 1, 4])
def test_shares_in_coarser_units_cover_every_key_once(shift):
    """The shares' arithmetic with units of up to a whole tile of keys: each row tile's parts follow each other from its
    first tile of keys to its last."""
    for lengths, group, kv_heads, n in (([9000, 0, 70, 1, 4000], 8, 2, 256), ([20000], 4, 1, 256), ([1] * 300 + [6000], 5, 2, 256)):
        for parts in shares(lengths, group, kv_heads, n, shift, 256).values():
            assert parts[0][0] == 0 and all(a <= b for a, b in parts) and all(x[1] == y[0] for x, y in zip(parts, parts[1:]))


def test_counts_stay_below_32_bits():
    """The longest prompts of a step's rows, in the form and unit that the library takes for them."""
    most = attn.MAX_STEP_TOKENS
    assert units([most], 4, 8, 128, 0) > 2 ** 31 > units([most], 4, 8, 256, 0)  # why 32 + 8 heads take 256 rows
    assert units([most], 8, 8, 256, 0) > 2 ** 31 > units([most - 4095] + [1] * 4095, 8, 8, 256, 1)
    assert units([most - 4095] + [1] * 4095, 1, 32, 256, 2) < 2 ** 31


@pytest.fixture
def layer(monkeypatch, pkg):
    """A layer whose cache must not be written."""
    def written(*args, **kwargs):
        raise AssertionError("the cache was written")

    monkeypatch.setattr(attn, "append_kv_int4", written)
    layer = attn.Attention(32, 128, 0.1, 8, block_size=16)
    layer.kv_cache = torch.zeros(4, 8, 16 * 136, dtype=torch.uint8)
    return layer


def step(rows, requests, width=2):
    lists = torch.zeros(1, dtype=torch.int32)
    tables = torch.zeros(1, width, dtype=torch.int32).expand(requests, width)
    return attn.KVStep(lists.expand(requests + 1), lists.expand(requests), lists.expand(rows), lists.expand(rows), tables, lists)


@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("rows,requests,change", [(400000, 1000, {}), (1 << 27, 1, {}), (8, 0, {}), (8, 2, {"max_query_len": 0}),
                                                  (8, 2, {"scale": 0.0}), (8, 2, {"scale": float("nan")})])
def test_a_step_that_attention_refuses_is_not_stored(layer, rows, requests, change, whole):
    if not whole and rows == 400000:
        rows, requests = 1 << 26, 4096  # chunks behind cached tokens have another bound
    change = dict(change)
    layer.scale = change.pop("scale", layer.scale)
    qkv = torch.zeros(1, 48 * 128, dtype=torch.bfloat16).expand(rows, 48 * 128)
    with pytest.raises(ValueError):
        layer.forward_qkv(qkv, step(rows, requests), None, whole_prompts=whole, **change)


@pytest.mark.parametrize("mask", [torch.zeros(8, dtype=torch.int32), torch.zeros(7, dtype=torch.int64)])
def test_a_step_with_a_wrong_tree_mask_is_not_stored(layer, mask):
    qkv = torch.zeros(8, 48 * 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="tree_mask"):
        layer.forward_qkv(qkv, step(8, 2), None, tree_mask=mask)


@pytest.mark.parametrize("whole", [True, False])
def test_a_step_that_attention_takes_is_stored(layer, whole):
    for rows, requests in ((8, 2), (attn.MAX_STEP_TOKENS, 4096) if whole else (16384, 64), (0, 2)):
        qkv = torch.zeros(1, 48 * 128, dtype=torch.bfloat16).expand(rows, 48 * 128)
        with pytest.raises(AssertionError, match="written"):
            layer.forward_qkv(qkv, step(rows, requests), None, whole_prompts=whole)


def workers_with_parts(lengths, group, kv_heads, dim, n):
    """The workers among whom the kernel deals out these sequences' row tiles, 0 where it cuts none."""
    grid = 256 * (4 if dim == 64 else 2) * 4 // (8 if n == 256 else 4)
    tiles = [-(-x * group // n) for x in lengths]
    step = -(-(n // 4) // group)
    longest = max((64 + step * m for m in tiles if m), default=0)
    if longest <= 128 or (longest <= 256 and kv_heads * sum(tiles) <= grid):
        return 0
    total = units(lengths, group, kv_heads, n, 0)
    return min(grid, (total - 1) // max(48, longest // 12) + 1)


def test_the_workspace_holds_what_a_call_may_hand_over(dll):
    """Room for two row tiles (a row's channels and two numbers, in fp32) of each worker that shares one, whatever the
    requests' lengths; calls that cut none need next to nothing."""
    import random

    rng = random.Random(4)
    for _ in range(400):
        kv_heads, group, dim = rng.choice([1, 2, 8, 16]), rng.choice([1, 4, 5, 8, 40]), rng.choice([64, 128])
        rows, requests = int(2 ** rng.uniform(0, 16)), int(2 ** rng.uniform(0, 8))
        size = dll.w4a16_prompt_attention_workspace(rows, requests, kv_heads * group, kv_heads, dim)
        n = form(rows, requests, kv_heads * group, kv_heads)
        for lengths in ([rows], [rows // requests] * requests, [max(rows - requests + 1, 0)] + [1] * min(requests - 1, rows - 1)):
            assert len(lengths) <= requests and sum(lengths) <= rows
            assert 2 * workers_with_parts(lengths, group, kv_heads, dim, n) * n * (dim + 2) * 4 <= size


@pytest.mark.parametrize("sizes", [(1, 1, 32, 8, 128), (120, 1, 32, 8, 128), (511, 1, 32, 8, 128), (16, 16, 32, 8, 128), (300, 1, 16, 16, 64)])
def test_short_prompts_need_no_workspace_to_speak_of(dll, sizes):
    assert 0 < dll.w4a16_prompt_attention_workspace(*sizes) <= 4096


def test_a_workspace_for_the_largest_step_serves_smaller_ones(dll):
    import random

    rng = random.Random(5)
    for _ in range(3000):
        kv_heads, group, dim = rng.choice([1, 2, 8, 16]), rng.choice([1, 4, 5, 8, 40]), rng.choice([64, 128])
        rows, requests = int(2 ** rng.uniform(0, 17)), int(2 ** rng.uniform(0, 10))
        most = dll.w4a16_prompt_attention_workspace(rows, requests, kv_heads * group, kv_heads, dim)
        if most == 0:  # refused
            continue
        for fewer in ((rng.randint(1, rows), rng.randint(1, requests)), (max(rows - 1, 1), requests), (rows, max(requests - 1, 1)),
                      (rows // 2 + 1, requests), (rows, requests // 2 + 1)):
            assert dll.w4a16_prompt_attention_workspace(*fewer, kv_heads * group, kv_heads, dim) <= most, (rows, requests, fewer)


@pytest.mark.parametrize("group", range(1, 17))
def test_every_step_of_up_to_128_heads_is_taken(dll, group):
    """The documented range: 2^18 rows, any number of requests, up to 128 heads in groups of up to 16."""
    for kv_heads in {1, 2, 3, 8, 128 // group}:
        if kv_heads * group <= 128:
            for rows in (1, 1000, 16385, 60000, 131073, 200001, attn.MAX_STEP_TOKENS):
                for requests in (1, 7, 512, 513, 4096, 1 << 18, 1 << 30):
                    assert dll.w4a16_prompt_attention_workspace(rows, requests, kv_heads * group, kv_heads, 128) > 0
