"""Refusals of the rotating, appending and prompt attention entry points, on the CPU: the C ABI's status
codes and messages (nothing is launched), Python argument errors, and what the oracle's bounds catch."""
import ctypes
import importlib

import pytest
import torch

from oracle import prompt_oracle as ora

attn = importlib.import_module("llm-serve_amd.layers.attention")
rope = importlib.import_module("llm-serve_amd.layers.rotary_embedding")

P = 1 << 20  # a pointer that no refused call follows


@pytest.fixture(scope="module")
def dll(pkg):
    return pkg.lib().dll


def error(pkg):
    return pkg.lib().last_error()


EPS = ctypes.c_float(1e-6)
ROPE = dict(q=P, qt=4096, qh=128, k=P, kt=4096, kh=128, positions=P, table=P, table_rows=64, rotary=128, qw=P, kw=P, eps=EPS,
            q_out=P, k_out=P, T=3, H=32, KV=8, D=128, stream=None)
APPEND = dict(q=P, qt=4096, qh=128, k=P, kt=4096, kh=128, v=P, vt=4096, vh=128, cache=P, slots=P, positions=P, table=P,
              table_rows=64, rotary=128, qw=None, kw=None, eps=EPS, q_out=P, k_out=None, T=3, H=32, KV=8, D=128, blocks=4,
              block=16, stream=None)
PROMPT = dict(q=P, qt=4096, qh=128, k=P, kt=4096, kh=128, v=P, vt=4096, vh=128, cu=P, out=P, scale=ctypes.c_float(0.1), T=3,
              R=2, H=32, KV=8, D=128, zero=1, ws=P, ws_bytes=1 << 40, counters=P, stream=None)

SHARED = [
    ({"T": -1}, 1, "negative"), ({"H": 0}, 1, "positive"), ({"KV": -1}, 1, "positive"), ({"H": 70000}, 2, "too many"),
    ({"D": 96}, 2, "head size"), ({"rotary": 0}, 2, "multiple of 16"), ({"rotary": 24}, 2, "multiple of 16"),
    ({"rotary": 144}, 2, "multiple of 16"), ({"table_rows": 0}, 1, "table"), ({"eps": ctypes.c_float(-1.0)}, 1, "eps"),
    ({"eps": ctypes.c_float(float("nan"))}, 1, "eps"), ({"eps": ctypes.c_float(float("inf"))}, 1, "eps"),
    ({"positions": None}, 1, "null"), ({"table": None}, 1, "null"), ({"q_out": None}, 1, "null"), ({"q": None}, 1, "null"),
    ({"k": None}, 1, "null"), ({"q": P + 8}, 3, "aligned"), ({"kt": 4097}, 3, "multiples of 8"), ({"qh": 4}, 3, "multiples of 8"),
    ({"table": P + 4}, 3, "aligned"), ({"qw": P + 2}, 3, "aligned"), ({"kw": P + 8}, 3, "aligned"), ({"q_out": P + 2}, 3, "aligned"),
    ({"k_out": P + 2}, 3, "aligned")]


@pytest.mark.parametrize("change,status,message", SHARED + [({"k_out": None}, 1, "null"), ({"T": (1 << 30) + 1}, 2, "too many")])
def test_rope_refusals(pkg, dll, change, status, message):
    assert dll.w4a16_qk_norm_rope(*{**ROPE, **change}.values()) == status and message in error(pkg)


@pytest.mark.parametrize("change,status,message", [c for c in SHARED if "KV" not in c[0]] + [
    ({"KV": 0}, 1, "positive"), ({"cache": None}, 1, "null"), ({"slots": None}, 1, "null"), ({"v": None}, 1, "null"),
    ({"vt": 4}, 3, "multiples of 8"), ({"cache": P + 8}, 3, "aligned"), ({"blocks": 0}, 1, "positive"), ({"block": 24}, 2, "block_size"),
    ({"blocks": 1 << 27}, 2, "2^31")])
def test_append_refusals(pkg, dll, change, status, message):
    assert dll.w4a16_kv_append(*{**APPEND, **change}.values()) == status and message in error(pkg)


@pytest.mark.parametrize("change,status,message", [
    ({"q": None}, 1, "null"), ({"k": None}, 1, "null"), ({"v": None}, 1, "null"), ({"cu": None}, 1, "null"), ({"out": None}, 1, "null"),
    ({"T": -1}, 1, "negative"), ({"R": -1}, 1, "negative"), ({"R": 0}, 1, "no request"), ({"H": 30}, 2, "multiple"),
    ({"KV": 0}, 2, "multiple"), ({"D": 256}, 2, "head size"), ({"scale": ctypes.c_float(0.0)}, 1, "scale"),
    ({"scale": ctypes.c_float(float("nan"))}, 1, "scale"), ({"scale": ctypes.c_float(3e38)}, 1, "scale"),
    ({"q": P + 8}, 3, "aligned"), ({"kt": 4}, 3, "multiples of 8"), ({"vh": 12}, 3, "multiples of 8"), ({"out": P + 8}, 3, "aligned"),
    ({"kt": (1 << 22) + 8}, 2, "2^22"), ({"vt": -8}, 2, "2^22"), ({"qt": 1 << 23}, 2, "2^22"), ({"qh": 1 << 27}, 2, "2^28"), ({"H": 32768, "KV": 1}, 2, "too many"), ({"ws": None}, 4, "workspace"), ({"ws_bytes": 64}, 4, "workspace"),
    ({"ws": P + 4}, 3, "aligned"), ({"counters": None}, 4, "counters"), ({"T": 1 << 28}, 2, "too many"),
    ({"T": 1 << 20}, 2, "too much work")])
def test_prompt_refusals(pkg, dll, change, status, message):
    assert dll.w4a16_prompt_attention(*{**PROMPT, **change}.values()) == status and message in error(pkg)


def test_nothing_to_do_is_no_error(dll):
    assert dll.w4a16_qk_norm_rope(*{**ROPE, "T": 0, "q": None, "k": None, "positions": None, "q_out": None, "k_out": None}.values()) == 0
    assert dll.w4a16_kv_append(*{**APPEND, "T": 0, "q": None, "v": None, "slots": None, "q_out": None}.values()) == 0
    assert dll.w4a16_prompt_attention(*{**PROMPT, "T": 0, "R": 0, "q": None, "out": None, "ws": None}.values()) == 0


def test_workspace_is_bounded(dll):
    for rows, requests, heads, kv_heads in ((1, 1, 32, 8), (16384, 4, 32, 8), (16384, 700, 16, 16), (1 << 18, 1, 32, 8)):
        assert 0 < dll.w4a16_prompt_attention_workspace(rows, requests, heads, kv_heads, 128) < 1 << 28
    for bad in ((4, 1, 30, 8, 128), (4, 1, 32, 8, 96), (0, 1, 32, 8, 128), (4, 0, 32, 8, 128), (1 << 28, 1, 32, 8, 128)):
        assert dll.w4a16_prompt_attention_workspace(*bad) == 0


def test_work_beyond_32_bits_is_refused(dll):
    """A prompt of 2^19 rows of 8 heads counts 8 x (2^11 + 1) x (2^16 + 2^10 + 129) = 1.1e9 units at most,
    one of 2^20 rows 8 x (2^12 + 1) x (2^17 + 2^11 + 129) = 4.4e9, beyond 2^31.  Where a kv head has 1024
    heads, a tile is a quarter of a token but costs a unit at least."""
    assert dll.w4a16_prompt_attention_workspace(1 << 19, 1, 8, 8, 128) > 0
    assert dll.w4a16_prompt_attention_workspace(1 << 20, 1, 8, 8, 128) == 0
    assert dll.w4a16_prompt_attention_workspace(1 << 13, 1, 1024, 1, 128) > 0
    assert dll.w4a16_prompt_attention_workspace(1 << 15, 1, 1024, 1, 128) == 0


def test_work_of_smaller_row_tiles_beyond_32_bits_is_refused(dll):
    """With more than a request a 512 rows, row tiles have 128 rows and there are twice as many: one prompt of
    2^19 rows among 1100 requests counts 8 x 2^12 x (64 + 32 (2^12 + 1) / 2) = 2.15e9 units, beyond 2^31."""
    assert 8 * 2 ** 12 * (64 + 16 * (2 ** 12 + 1)) > 2 ** 31
    assert dll.w4a16_prompt_attention_workspace(1 << 19, 1100, 8, 8, 128) == 0
    assert dll.w4a16_prompt_attention_workspace(1 << 18, 1100, 8, 8, 128) > 0


def test_python_refusals():
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    k = q[:, :2]
    lists = torch.zeros(3, dtype=torch.int32)
    table = rope.rotary_table(128, 10, device="cpu")
    cache = torch.zeros(4, 2, 16 * 136, dtype=torch.uint8)
    with pytest.raises(ValueError, match="GPU"):
        rope.qk_norm_rope(q, k, lists, table)
    with pytest.raises(ValueError, match="GPU"):
        attn.append_kv_int4(q, k, k, cache, lists, lists, table, block_size=16)
    with pytest.raises(ValueError, match="GPU"):
        attn.attention_prompt(q, k, k, lists)
    with pytest.raises(ValueError, match="block_size"):
        attn.append_kv_int4(q, k, k, cache, lists, lists, table, block_size=20)
    for args in ((8, 10), (24, 10), (0, 10), (128, 0), (128, 10, 0.0), (128, 10, float("inf"))):
        with pytest.raises(ValueError):
            rope.rotary_table(*args, device="cpu")
    with pytest.raises(ValueError, match="head_size"):
        rope.RotaryEmbedding(96, 96, 10, device="cpu")
    with pytest.raises(ValueError, match="rotary_dim"):
        rope.RotaryEmbedding(64, 128, 10, device="cpu")
    with pytest.raises(RuntimeError, match="kv_cache"):
        attn.Attention(4, 128, 0.1, 2).forward_qkv(q, None, table)
    layer = attn.Attention(4, 128, 0.1, 2)
    layer.kv_cache = cache
    with pytest.raises(ValueError, match="tree_mask"):
        layer.forward_qkv(q, None, table, whole_prompts=True, tree_mask=lists)


def test_table_of_far_positions():
    """Angles are formed in 64 bits: a table's last rows are the functions of the exact angles to half a
    step of fp32 (and 2^-53 of the angle)."""
    from fractions import Fraction
    import math

    table = rope.rotary_table(64, 131072, 1000000.0, device="cpu").double()
    for position in (1, 777, 131071):
        for i in (0, 1, 17, 31):
            angle = position * 1000000.0 ** (-i / 32)
            assert abs(Fraction(angle) - Fraction(position) * Fraction(1000000.0 ** (-i / 32))) < Fraction(1, 1 << 30)
            assert abs(float(table[position, i]) - math.cos(angle)) <= 2.0 ** -25 + 1e-10
            assert abs(float(table[position, 32 + i]) - math.sin(angle)) <= 2.0 ** -25 + 1e-10


def emulate(q, k, v, offsets, weights=torch.bfloat16, lost=None):
    """Prompt attention that rounds its weights and its output, and may lose a key."""
    rows, heads, dim = q.shape
    out = torch.zeros(rows, heads, dim, dtype=torch.float64)
    for first, end in zip(offsets, offsets[1:]):
        for h in range(heads):
            g = h // (heads // k.shape[1])
            s = q[first:end, h].double() @ k[first:end, g].double().t() * dim ** -0.5
            s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), float("-inf"))
            if lost is not None and lost < end - first:
                s[lost + 1:, lost] = float("-inf")
            p = torch.exp(s - s.amax(-1, keepdim=True) - 0.3)
            out[first:end, h] = p.to(weights).double() @ v[first:end, g].double() / p.sum(-1, keepdim=True)
    return out.to(torch.bfloat16)


def test_the_bounds_hold_for_the_kernels_roundings_and_catch_others():
    gen = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(300, h, 64, generator=gen).to(torch.bfloat16) for h in (4, 2, 2))
    offsets = [0, 200, 201, 300]
    want = ora.prompt(q, k, v, offsets)
    ora.check_prompt(emulate(q, k, v, offsets), *want, 200)
    for wrong in (dict(weights=torch.float8_e4m3fn), dict(lost=150), dict(lost=60)):
        with pytest.raises(AssertionError):
            ora.check_prompt(emulate(q, k, v, offsets, **wrong), *want, 200)


def test_the_two_forms_of_the_rotation_agree():
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(50, 3, 128, generator=gen).to(torch.bfloat16)
    positions = torch.randint(0, 4000, (50,), generator=gen)
    w = torch.rand(128, generator=gen).to(torch.bfloat16)
    for rotary in (16, 64, 128):
        table = rope.rotary_table(rotary, 4000, device="cpu")
        for weight in (None, w):
            want, size = ora.turn(x, positions, rotary, 10000.0, weight)
            got = ora.turn_fp32(x, positions, table, weight).double()
            assert bool(((got - want).abs() <= ora.turn_tolerance(want, size)).all())
            wrong = ora.turn_fp32(x, positions + 1, torch.cat((table, table[:1])), weight).double()
            assert not bool(((wrong - want).abs() <= ora.turn_tolerance(want, size)).all())
