"""Prompt attention where its arithmetic is at its limits: sums over very long prompts, scores of any size; its
largest steps, and each of its forms for each size of group."""
import importlib
import math

import pytest
import torch

from oracle import prompt_oracle as ora
from prompt_helpers import form

pytestmark = pytest.mark.gpu

attn = importlib.import_module("llm-serve_amd.layers.attention")


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_sums_of_equal_weights_over_a_long_prompt(gpu_lib):
    """350000 rows whose first key weighs 1 and has the value 0, and whose others weigh p = 179/256 each, a
    number of bf16, and have values of 0 or 1: in channel c the first m_c of each 4096 runs of 16 keys have
    ones, so row t is p n / (1 + p t) with n the ones that it sees.

    The numerator's sums (16 p at a time, a multiple of 2^-4, below 2^18) are formed without an error but for a
    run that a prompt or a share of it cuts, and the weights lose nothing in bf16.  What is left: p by 2^-18 (its
    2e-6 and its score's two roundings) and the exponential by 2^-22, the sum of weights (5469 tiles of some 40
    additions before them) by 2^-24 each, ten roundings of cut runs, joins and the quotient, and half a step of
    the output.  The p of the scores lies 2e-6 above 179/256, so that a running sum of single
    weights, whose last place is 2^-7 here, would round each of them up by 2^-8."""
    rows, p = 350000, 179 / 256
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k = (torch.zeros(rows, 1, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q[:, 0, 0] = 1
    k[0, 0, 0] = 1
    at = torch.arange(rows, device="cuda")
    ones = torch.randint(2048, 4096, (128,), generator=gen, device="cuda")
    v = (at[:, None] // 16 % 4096 < ones) & (at[:, None] > 0)
    out = attn.attention_prompt(q, k, v[:, None].to(torch.bfloat16), int32([0, rows]), scale=-math.log(p * (1 + 2e-6)))
    want = p * v.cumsum(0) / (1 + p * at[:, None].double())
    half_step = 2.0 ** (torch.frexp(want.clamp(min=2.0 ** -100)).exponent - 9)
    off = (out[:, 0].double() - want).abs() - half_step
    error = 2.0 ** -18 + 2.0 ** -22 + (5469 + 40 + 10) * 2.0 ** -24
    bad = off > error * want
    assert not bool(bad.any()), (int(bad.sum()), int(bad.any(1).nonzero()[0]), float((off / want.clamp(min=1e-9)).max()))


@pytest.mark.parametrize("heads,kv_heads,dim,lengths", [(4, 2, 128, [300]), (4, 4, 64, [100, 270]), (16, 4, 64, [1500]), (32, 8, 128, [700, 600]),
                                                        (32, 8, 128, [2039]), (16, 4, 64, [4000])])
@pytest.mark.parametrize("size", [2.0 ** 13, 2.0 ** 17, 2.0 ** 20, 2.0 ** 45])
def test_rows_of_very_large_scores(gpu_lib, heads, kv_heads, dim, lengths, size):
    """Scores of 2^23 to 2^95, where a last place of fp32 is worth far more than 1: a row is the value of its
    largest score.  (The scale is no power of two, so that scores are rounded on their way into the exponent.)

    Key j of a sequence is size (1 + j // dim) in channel j % dim; query t is size in one channel and -size in all
    others.  Of the keys in its channel that it sees the last one wins, by at least size^2 / 16; where it sees none
    in it, all that it sees (fewer than dim) have the same score, and it is their mean.  All weights are 1 or 0, so
    what is left is the sums' and the quotient's roundings, below 2 dim 2^-24 of values below 8, and the output's."""
    rows, group = sum(lengths), heads // kv_heads
    gen = torch.Generator(device="cuda").manual_seed(8)
    v = torch.randn(rows, kv_heads, dim, generator=gen, device="cuda").to(torch.bfloat16)
    q = torch.full((rows, heads, dim), -size, device="cuda")
    k, want = torch.zeros(rows, kv_heads, dim, device="cuda"), torch.zeros(rows, heads, dim, dtype=torch.float64, device="cuda")
    offsets = [0]
    for n in lengths:
        first, t = offsets[-1], torch.arange(n, device="cuda")
        k[first + t, :, t % dim] = (size * (1 + t // dim))[:, None]
        for h in range(heads):
            channel = (7 * t + h) % dim
            q[first + t, h, channel] = size
            last = t - (t - channel) % dim
            seen = v[first:first + n, h // group].double()
            mean = seen.cumsum(0) / (1 + t)[:, None]
            want[first:first + n, h] = torch.where((last >= 0)[:, None], seen[last.clamp(min=0)], mean)
        offsets.append(first + n)
    assert float(v.abs().max()) < 8
    out = attn.attention_prompt(q.to(torch.bfloat16), k.to(torch.bfloat16), v, int32(offsets), scale=0.11)
    off = (out.double() - want).abs()
    bad = ~(off <= 2.0 ** -8 * want.abs() + 8 * 2 * dim * 2.0 ** -24)
    assert not bool(bad.any()), (int(bad.any(-1).sum()), bad.any(-1).nonzero()[0].tolist())


@pytest.mark.parametrize("heads,lengths", [(4, [300]), (16, [700, 400]), (32, [2039])])
def test_rows_of_very_large_scores_are_alone(gpu_lib, heads, lengths):
    """A row beside one of very large scores keeps its bits."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    q, k, v = (torch.randn(sum(lengths), h, 128, generator=gen, device="cuda").to(torch.bfloat16) for h in (heads, 4, 4))
    offsets = int32([0] + [sum(lengths[:i + 1]) for i in range(len(lengths))])
    want = attn.attention_prompt(q, k, v, offsets)
    large = torch.rand(sum(lengths), heads, generator=gen, device="cuda") < 0.05
    q = torch.where(large[..., None], q * 2.0 ** 40, q)
    out = attn.attention_prompt(q, k, v, offsets)
    assert torch.equal(out[~large], want[~large]) and bool(torch.isfinite(out).all())
    assert not torch.equal(out[large], want[large])


def check_rows(out, q, k, v, first, rows, scale):
    """Some rows of a sequence that begins at `first`, against their 64-bit sums."""
    group, dim = q.shape[1] // k.shape[1], q.shape[2]
    for row in rows:
        n = row - first + 1
        for g in range(k.shape[1]):
            keys, values = k[first:row + 1, g].double(), v[first:row + 1, g].double()
            for h in range(g * group, (g + 1) * group):
                s = (keys * q[row, h].double()).sum(-1) * scale
                w = torch.softmax(s, 0)[:, None]
                want, spread = (w * values).sum(0), (w * values.abs()).sum(0)
                reach = (keys.abs() * q[row, h].double().abs()).sum(-1).amax().expand(1) * scale
                off = (out[row, h].double() - want).abs()
                # tiles of keys, and the additions of one of them
                assert bool((off <= ora.prompt_tolerance(want[None], spread[None], reach, n // 64 + 64)[0]).all()), (row, h)


@pytest.mark.parametrize("heads,kv_heads,requests", [(32, 8, 513), (64, 8, 4096)])
def test_largest_steps_of_many_requests(gpu_lib, heads, kv_heads, requests):
    """2^18 rows of more than a request a 512 rows: prompts of the same length, whose sequences are those of a smaller
    call, and one prompt of all rows but one for each other request."""
    rows = 1 << 18
    gen = torch.Generator(device="cuda").manual_seed(10)
    q, k, v = (torch.randn(rows, h, 128, generator=gen, device="cuda", dtype=torch.bfloat16) for h in (heads, kv_heads, kv_heads))
    each = rows // requests
    even = [i * each for i in range(requests)] + [rows]
    out = attn.attention_prompt(q, k, v, int32(even))
    for r in (0, 1, requests // 2, requests - 1):
        a, b = even[r], even[r + 1]
        ora.check_prompt(out[a:b], *ora.prompt(q[a:b], k[a:b], v[a:b], [0, b - a]), b - a)
    long = rows - (requests - 1)
    out = attn.attention_prompt(q, k, v, int32([0] + list(range(long, rows + 1))))
    check_rows(out, q, k, v, 0, (0, 63, 4097, 100000, long - 1), 128 ** -0.5)
    assert torch.equal(out[long:], v[long:].repeat_interleave(heads // kv_heads, 1))


@pytest.mark.parametrize("heads,kv_heads,dim,lengths", [(8, 2, 128, [1, 3]), (32, 8, 128, [511]), (32, 8, 128, [700]), (32, 8, 128, [2039]),
                                                        (40, 8, 128, [300, 1, 0, 1111, 7]), (32, 8, 128, [50] * 40), (4, 2, 128, [3000]),
                                                        (16, 16, 64, [1500, 1, 333]), (2, 1, 64, [2500, 900]), (1, 1, 128, [6000])])
def test_the_workspace_is_as_large_as_a_call_needs(gpu_lib, heads, kv_heads, dim, lengths):
    """With exactly the bytes that are asked for: the same bits, the bytes behind them as they were, counters at zero."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    q, k, v = (torch.randn(sum(lengths), h, dim, generator=gen, device="cuda").to(torch.bfloat16) for h in (heads, kv_heads, kv_heads))
    offsets = int32([0] + [sum(lengths[:i + 1]) for i in range(len(lengths))])
    want = attn.attention_prompt(q, k, v, offsets)
    size = gpu_lib.prompt_attention_workspace(sum(lengths), len(lengths), heads, kv_heads, dim)
    space = torch.full((size + (1 << 20),), 0x5A, dtype=torch.uint8, device="cuda")
    counters = torch.zeros(1024, dtype=torch.int32, device="cuda")
    for _ in range(3):
        out = torch.full_like(want, 9.0)
        gpu_lib.prompt_attention(q, k, v, offsets, out, dim ** -0.5, True, space[:size], counters)
        assert torch.equal(out, want)
        assert bool((space[size:] == 0x5A).all()) and not bool(counters.any())


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (40, 8, 128), (5, 1, 64), (6, 2, 128), (14, 2, 64), (16, 16, 64), (24, 2, 128)])
@pytest.mark.parametrize("tile,least", [(64, 0), (128, 17000), (256, 52000)])
def test_packed_lengths_in_each_form(gpu_lib, heads, kv_heads, dim, tile, least):
    """Groups of 1 to 12 heads in each form, the last prompt as long as the form needs: with groups that do not divide
    a tile's or a wave's rows, tokens are cut between them."""
    lengths = [0, 129, 1, 33]
    if tile != 64:
        lengths.append(max(-(-least // heads) - sum(lengths), 2600 if tile == 256 else 130))
    assert form(sum(lengths), len(lengths), heads, kv_heads) == tile
    gen = torch.Generator(device="cuda").manual_seed(12)
    q, k, v = torch.randn(sum(lengths), heads + 2 * kv_heads, dim, generator=gen,
                          device="cuda").to(torch.bfloat16).split((heads, kv_heads, kv_heads), 1)
    offsets = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    ora.check_prompt(attn.attention_prompt(q, k, v, int32(offsets)), *ora.prompt(q, k, v, offsets), max(lengths))


@pytest.mark.parametrize("heads,lengths", [(4, [90]), (16, [700, 400]), (32, [2039])])
def test_scores_beyond_fp32(gpu_lib, heads, lengths):
    """Finite queries and keys whose product passes fp32's range: above it a row is NaN, and where all of a row's
    scores lie below it the row is zero; other rows keep their bits."""
    gen = torch.Generator(device="cuda").manual_seed(13)
    q, k, v = (torch.randn(sum(lengths), h, 128, generator=gen, device="cuda").abs().add(0.5).to(torch.bfloat16) for h in (heads, 4, 4))
    offsets = int32([0] + [sum(lengths[:i + 1]) for i in range(len(lengths))])
    k = k * 2.0 ** 60
    q = q * 2.0 ** -60
    want = attn.attention_prompt(q, k, v, offsets)
    row = torch.rand(q.shape[:2], generator=gen, device="cuda")
    above, below = row < 0.05, row > 0.95
    large = q * 2.0 ** 65 * 2.0 ** 65  # 2^130 itself is no fp32 number
    q = torch.where(above[..., None], large, torch.where(below[..., None], -large, q))
    assert bool(torch.isfinite(q).all()) and bool(torch.isfinite(k).all())
    out = attn.attention_prompt(q, k, v, offsets)
    assert bool(out[above].isnan().all()) and not bool(out[below].any())
    assert torch.equal(out[~(above | below)], want[~(above | below)])


def test_infinite_values_are_not_finite_anywhere(gpu_lib):
    """An infinite value whose weight underflows leaves infinity or NaN in its channel, and nothing in others."""
    q, k, v = (torch.zeros(500, 1, 64, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    q[:, 0, 0], k[:, 0, 0] = 100, 100
    k[100, 0, 0] = k[420, 0, 0] = -100
    v[:, 0, 1], v[100, 0, 0], v[420, 0, 0] = 1, float("inf"), float("inf")
    out = attn.attention_prompt(q, k, v, int32([0, 500]), scale=1.0)
    assert not bool(out[:100, 0, 0].any()) and not bool(torch.isfinite(out[100:, 0, 0]).any())
    assert bool((out[:, 0, 1] == 1).all()) and not bool(out[:, 0, 2:].any())
