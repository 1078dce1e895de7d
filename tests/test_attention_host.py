"""Refusals of the 4-bit cache's entry points, on the CPU: Python argument errors, the C ABI's
status codes and messages (nothing is launched), workspace sizes, and the oracle's own arithmetic."""
import ctypes
import importlib

import pytest
import torch

from oracle import kv4_oracle as ora

attn = importlib.import_module("llm-serve_amd.layers.attention")

P = 1 << 20  # a pointer that no refused call follows


@pytest.fixture(scope="module")
def dll(pkg):
    return pkg.lib().dll


def error(pkg):
    return pkg.lib().last_error()


STEP = dict(query=P, context=P, tables=P, stride=8, free=P, cu=P, seq=P, positions=P, slots=P, used=P, R=2, width=8,
            num_free=4, block=16, T=3, stream=None)
STORE = dict(k=P, kt=1024, kh=128, v=P, vt=1024, vh=128, cache=P, slots=P, T=3, KV=8, D=128, blocks=4, block=16,
             stream=None)
LOAD = dict(cache=P, slots=P, k=P, v=P, T=3, KV=8, D=128, blocks=4, block=16, stream=None)
ATTENTION = dict(q=P, qt=4096, qh=128, cache=P, tables=P, stride=8, seq=P, cu=P, mask=None, out=P,
                 scale=ctypes.c_float(0.1), T=3, R=2, H=32, KV=8, D=128, blocks=4, block=16, width=8, longest=1, zero=1,
                 ws=P, ws_bytes=1 << 40, counters=P, stream=None)


@pytest.mark.parametrize("change,status,message", [
    ({"query": None}, 1, "null"), ({"used": None}, 1, "null"), ({"free": None}, 1, "null"), ({"R": -1}, 1, "negative"),
    ({"T": -1}, 1, "negative"), ({"num_free": -1}, 1, "negative"), ({"R": 4097}, 2, "at most"),
    ({"T": (1 << 18) + 1}, 2, "at most"), ({"width": 0}, 1, "width"), ({"stride": 7}, 1, "width"),
    ({"block": 8}, 2, "block_size"), ({"block": 48}, 2, "block_size"), ({"block": 512}, 2, "block_size")])
def test_step_refusals(pkg, dll, change, status, message):
    assert dll.w4a16_kv_step(*{**STEP, **change}.values()) == status and message in error(pkg)


@pytest.mark.parametrize("change,status,message", [
    ({"cache": None}, 1, "null"), ({"slots": None}, 1, "null"), ({"k": None}, 1, "null"), ({"v": None}, 1, "null"),
    ({"T": -1}, 1, "negative"), ({"KV": 0}, 1, "positive"), ({"blocks": 0}, 1, "positive"), ({"D": 96}, 2, "head size"),
    ({"block": 24}, 2, "block_size"), ({"blocks": 1 << 27}, 2, "2^31"), ({"cache": P + 8}, 3, "aligned"),
    ({"k": P + 2}, 3, "aligned"), ({"vt": 1028}, 3, "multiples of 8"), ({"kh": 4}, 3, "multiples of 8"),
    ({"T": 1 << 30}, 2, "too many")])
def test_store_refusals(pkg, dll, change, status, message):
    assert dll.w4a16_kv_store(*{**STORE, **change}.values()) == status and message in error(pkg)


@pytest.mark.parametrize("change,status,message", [
    ({"cache": None}, 1, "null"), ({"slots": None}, 1, "null"), ({"k": None}, 1, "null"), ({"v": P + 4}, 3, "aligned"),
    ({"T": -1}, 1, "negative"), ({"D": 32}, 2, "head size"), ({"block": 0}, 2, "block_size")])
def test_load_refusals(pkg, dll, change, status, message):
    assert dll.w4a16_kv_load(*{**LOAD, **change}.values()) == status and message in error(pkg)


@pytest.mark.parametrize("change,status,message", [
    ({"q": None}, 1, "null"), ({"cache": None}, 1, "null"), ({"tables": None}, 1, "null"), ({"seq": None}, 1, "null"),
    ({"cu": None}, 1, "null"), ({"out": None}, 1, "null"), ({"T": -1}, 1, "negative"), ({"R": 0}, 1, "no request"),
    ({"H": 30}, 2, "multiple"), ({"KV": 0}, 1, "positive"), ({"D": 256}, 2, "head size"), ({"width": 0}, 1, "width"),
    ({"stride": 7}, 1, "apart"), ({"block": 8}, 2, "block_size"), ({"longest": 0}, 1, "max_query_len"),
    ({"scale": ctypes.c_float(0.0)}, 1, "scale"), ({"scale": ctypes.c_float(-1.0)}, 1, "scale"),
    ({"scale": ctypes.c_float(float("nan"))}, 1, "scale"), ({"scale": ctypes.c_float(float("inf"))}, 1, "scale"),
    ({"q": P + 8}, 3, "aligned"), ({"qt": 4097}, 3, "multiples of 8"), ({"out": P + 8}, 3, "aligned"),
    ({"ws": None}, 4, "workspace"), ({"ws_bytes": 64}, 4, "workspace"), ({"ws": P + 4}, 3, "aligned"), ({"counters": None}, 4, "counters"),
    ({"T": 1 << 28}, 2, "too many"), ({"T": 1 << 18, "width": 1 << 20, "stride": 1 << 20}, 2, "too much work")])
def test_attention_refusals(pkg, dll, change, status, message):
    assert dll.w4a16_kv_attention(*{**ATTENTION, **change}.values()) == status and message in error(pkg)


def test_nothing_to_do_is_no_error(dll):
    assert dll.w4a16_kv_store(*{**STORE, "T": 0, "k": None, "v": None, "slots": None}.values()) == 0
    assert dll.w4a16_kv_load(*{**LOAD, "T": 0, "k": None, "v": None, "slots": None}.values()) == 0
    assert dll.w4a16_kv_attention(*{**ATTENTION, "T": 0, "R": 0, "q": None, "out": None, "ws": None}.values()) == 0


def test_workspace_is_bounded(dll):
    """Whatever the batch, the workspace stays far below the memory it reads, and an invalid
    problem needs none."""
    for rows, requests, width, longest in ((1, 1, 1, 1), (512, 512, 512, 1), (16384, 4, 512, 4096), (16384, 1, 64, 16384)):
        size = dll.w4a16_kv_attention_workspace(rows, requests, 32, 8, 128, 256, width, longest)
        assert 0 < size < 1 << 30
    assert dll.w4a16_kv_attention_workspace(4, 1, 30, 8, 128, 256, 1, 1) == 0
    assert dll.w4a16_kv_attention_workspace(4, 1, 32, 8, 128, 100, 1, 1) == 0


def test_python_refusals():
    cache = torch.zeros(4, 2, 16 * 136, dtype=torch.uint8)
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        attn.store_kv_int4(k, k, cache, slots, block_size=16)
    with pytest.raises(ValueError, match="GPU"):
        attn.load_kv_int4(cache, slots, block_size=16)
    with pytest.raises(ValueError, match="GPU"):
        attn.attention_int4(k, cache, slots[None], slots[:1], slots[:2], block_size=16)
    with pytest.raises(ValueError, match="GPU"):
        attn.kv_step(slots, slots, slots[:, None], slots, block_size=16, num_tokens=1)
    with pytest.raises(ValueError, match="block_size"):
        attn.load_kv_int4(cache, slots, block_size=24)
    for bad in (cache.to(torch.int8), cache[0], cache.transpose(0, 1)):
        with pytest.raises(ValueError, match="contiguous uint8"):
            attn.load_kv_int4(bad, slots, block_size=16)
    for args in ((0, 16, 2, 128), (4, 16, 0, 128), (4, 20, 2, 128), (4, 16, 2, 100), (1 << 28, 16, 2, 128)):
        with pytest.raises(ValueError):
            attn.new_kv_cache_int4(*args, device="cpu")
    with pytest.raises(ValueError, match="multiple"):
        attn.Attention(30, 128, 0.1, 8)
    with pytest.raises(ValueError, match="block_size"):
        attn.Attention(32, 128, 0.1, 8, block_size=100)
    with pytest.raises(ValueError, match="head_dim"):
        attn.Attention(32, 96, 0.1, 8)
    with pytest.raises(RuntimeError, match="kv_cache"):
        attn.Attention(32, 128, 0.1, 8)(k, k, k, None)


def test_oracle_rows_survive_packing():
    gen = torch.Generator().manual_seed(0)
    for dim in (64, 128):
        k, v = (torch.randn(20, 2, dim, generator=gen).to(torch.bfloat16) for _ in range(2))
        cache = torch.zeros(3, 2, 16 * (dim + 8), dtype=torch.uint8)
        slots = torch.randperm(48, generator=gen)[:20]
        ora.store(k, v, cache, slots, 16)
        got = ora.load(cache, slots.tolist(), 16)
        for x, y, s in zip((k, v), got[:2], got[2:]):
            assert torch.equal(ora.row_values(*ora.quantize_rows(x)), y)
            assert bool(((x.double() - y).abs() <= s[..., None] * (0.5 + 15 * 2.0 ** -8)).all())


def test_oracle_attention_of_one_key_is_its_value():
    cache = torch.zeros(1, 1, 16 * 72, dtype=torch.uint8)
    x = torch.randn(1, 1, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    ora.store(x, x, cache, torch.tensor([0]), 16)
    out, spread = ora.attention(x, cache, [[0]], [1], [0, 1], 16)
    assert torch.equal(out, ora.load(cache, [0], 16)[1])
    assert bool((spread >= 2 * 2.0 ** -8 * out.abs()).all())  # the weights' and the values' roundings


def test_wrong_ranks_are_refused():
    cache = torch.zeros(4, 2, 16 * 136, dtype=torch.uint8)
    lists = torch.zeros(2, dtype=torch.int32)
    for shape in ((), (128,), (3, 256), (1, 3, 2, 128)):
        with pytest.raises(ValueError):
            attn.attention_int4(torch.zeros(shape, dtype=torch.bfloat16), cache, lists[None], lists[:1], lists,
                                block_size=16)


def test_work_beyond_32_bits_is_refused(dll):
    """Prompt work is counted as 8 heads x 513 tiles x (2^20 + 2^17) / 4 = 1.2e9 units for 2^17 rows over
    2^20 keys, and as 8 x 1025 x (2^20 + 2^18) / 4 = 2.7e9 for 2^18 rows, beyond 2^31."""
    assert dll.w4a16_kv_attention_workspace(1 << 17, 1, 8, 8, 128, 256, 1 << 12, 1 << 17) > 0
    assert dll.w4a16_kv_attention_workspace(1 << 18, 1, 8, 8, 128, 256, 1 << 12, 1 << 18) == 0
    for t, r, h, kv, width, longest in ((1 << 18, 1, 8, 8, 1 << 20, 1 << 18),     # a long prompt over 2^28 keys
                                        (4096, 4096, 64, 64, 1 << 21, 1),         # decode rows over 2^29 keys
                                        (1 << 20, 1, 1024, 1, 1 << 20, 1 << 20),  # many heads of one kv head
                                        (1 << 24, 1, 128, 1, 16, 1)):             # rows x heads
        assert dll.w4a16_kv_attention_workspace(t, r, h, kv, 128, 256, width, longest) == 0
