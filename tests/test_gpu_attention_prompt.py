"""Causal attention of whole prompts over their own bf16 keys and values against 64-bit attention
(oracle/prompt_oracle.py), for packed lengths, head layouts, strides and masked places where it can go
wrong."""
import importlib

import pytest
import torch

from oracle import prompt_oracle as ora

pytestmark = pytest.mark.gpu

attn = importlib.import_module("llm-serve_amd.layers.attention")

LAYOUTS = [(8, 2, 128), (4, 4, 64), (5, 1, 128), (16, 2, 64), (3, 3, 128)]
LENGTHS = [[1], [0, 1, 0, 2], [31, 33], [63, 64, 65], [127, 128, 129, 1], [0, 257, 0], [517], [1500], [900, 700, 3, 64]]


def batch(lengths, heads, kv_heads, dim, seed, before=0, behind=0):
    """q, k, v as views of one projection's output, and the offsets."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(before + sum(lengths) + behind, heads + 2 * kv_heads, dim, generator=gen, device="cuda")
    q, k, v = x.to(torch.bfloat16).split((heads, kv_heads, kv_heads), 1)
    offsets = [before]
    for n in lengths:
        offsets.append(offsets[-1] + n)
    return q, k, v, offsets


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def check(out, q, k, v, offsets, scale=None):
    assert out.shape == q.shape and out.dtype == torch.bfloat16 and out.is_contiguous()
    ora.check_prompt(out, *ora.prompt(q, k, v, offsets, scale), max(b - a for a, b in zip(offsets, offsets[1:])))


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_packed_lengths(gpu_lib, heads, kv_heads, dim, lengths):
    q, k, v, offsets = batch(lengths, heads, kv_heads, dim, seed=sum(lengths) + heads, before=2, behind=5)
    out = attn.attention_prompt(q, k, v, int32(offsets))
    check(out, q, k, v, offsets)
    assert not bool(out[:2].any()) and not bool(out[offsets[-1]:].any())


@pytest.mark.parametrize("heads,kv_heads,dim,lengths", [(32, 8, 128, [2039]), (40, 8, 128, [300, 1, 0, 1111, 7, 640]),
                                                        (64, 8, 128, [777, 900]), (16, 16, 64, [1500, 1, 333]), (8, 1, 64, [3500])])
def test_larger_batches(gpu_lib, heads, kv_heads, dim, lengths):
    """Batches whose row tiles are cut and joined."""
    q, k, v, offsets = batch(lengths, heads, kv_heads, dim, seed=len(lengths))
    check(attn.attention_prompt(q, k, v, int32(offsets), max_query_len=max(lengths)), q, k, v, offsets)


def test_many_short_prompts(gpu_lib):
    """More prompts than a wave has lanes and than there are workgroups, empty ones among them."""
    lengths = [(i * 7) % 23 for i in range(700)]
    q, k, v, offsets = batch(lengths, 4, 2, 64, seed=5, behind=1)
    check(attn.attention_prompt(q, k, v, int32(offsets)), q, k, v, offsets)


@pytest.mark.parametrize("scale", [1e-30, 0.01, 1.0, 30.0])
def test_scales(gpu_lib, scale):
    q, k, v, offsets = batch([70, 300], 4, 2, 128, seed=6)
    check(attn.attention_prompt(q, k, v, int32(offsets), scale=scale), q, k, v, offsets, scale)


@pytest.mark.parametrize("dim", [64, 128])
def test_references_that_move(gpu_lib, dim):
    """Scores that rise and fall along the keys by far more than the exponent's range, so that the
    reference of a row moves late, often and by jumps."""
    for seed, trend in enumerate((torch.linspace(0, 40, 900), torch.linspace(40, 0, 900), 20 * torch.sin(torch.arange(900) / 9.0))):
        q, k, v, offsets = batch([900], 2, 1, dim, seed=20 + seed)
        q, k = q.clone(), k.clone()
        q[:, :, 0] = 4.0
        k[:, 0, 0] = trend.cuda().to(torch.bfloat16)
        check(attn.attention_prompt(q, k, v, int32(offsets), scale=1.0), q, k, v, offsets, 1.0)


@pytest.mark.parametrize("factor", [1e-30, 1e30])
def test_values_far_from_one(gpu_lib, factor):
    q, k, v, offsets = batch([400, 30], 4, 1, 128, seed=9)
    v = (v.float() * factor).to(torch.bfloat16)
    v[::3] = (v[::3].float() * 1e-6).to(torch.bfloat16)
    check(attn.attention_prompt(q, k, v, int32(offsets)), q, k, v, offsets)


def test_marked_keys(gpu_lib):
    """Each key's value names it in channels of its own, so that a key lost, doubled or swapped
    changes some row by that key's whole share."""
    for lengths in ([128], [200, 56, 1], [1024]):
        q, k, _, offsets = batch(lengths, 8, 2, 128, seed=30)
        rows = q.shape[0]
        v = torch.zeros(rows, 2, 128, device="cuda")
        at = torch.arange(rows, device="cuda")
        v[at, :, at % 128] = 1.0
        v[at, :, (at // 128 * 37 + at) % 128] += 2.0
        v = v.to(torch.bfloat16)
        check(attn.attention_prompt(q, k, v, int32(offsets)), q, k, v, offsets)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64), (1, 1, 128)])
@pytest.mark.parametrize("what", ["k", "v", "both"])
def test_masked_places_that_are_no_numbers(gpu_lib, heads, kv_heads, dim, what):
    """NaN and infinities in keys and values reach the rows that see them, and only those."""
    lengths = [300, 200, 64]
    q, k, v, offsets = batch(lengths, heads, kv_heads, dim, seed=40)
    k, v = k.clone(), v.clone()
    clean = attn.attention_prompt(q, k, v, int32(offsets))
    first_bad = torch.full((q.shape[0], kv_heads), 1 << 30, device="cuda")
    places = [(130, 0, "nan"), (299, 0, "inf"), (300 + 70, kv_heads - 1, "-inf"), (563, 0, "nan"), (505, 0, "inf")]
    for place, head, value in places:
        if what != "v":
            k[place, head] = float(value)
        if what != "k":
            v[place, head, 3::7] = float(value)
        end = next(b for a, b in zip(offsets, offsets[1:]) if a <= place < b)
        first_bad[place:end, head] = 0
    out = attn.attention_prompt(q, k, v, int32(offsets))
    spoilt = (first_bad == 0).repeat_interleave(heads // kv_heads, 1)
    assert torch.equal(out[~spoilt], clean[~spoilt])
    if what == "v":  # infinities and NaN in their own channels, other channels as they were
        touched = torch.zeros(dim, dtype=torch.bool, device="cuda")
        touched[3::7] = True
        assert torch.equal(out[:, :, ~touched], clean[:, :, ~touched])
        assert not bool(torch.isfinite(out[spoilt][:, touched]).any())
        group = heads // kv_heads
        assert bool((out[299, :group, 3::7].isnan()).all())  # it sees a NaN at 130
        assert bool((out[370:500, (kv_heads - 1) * group:, 3::7] == float("-inf")).all())


def test_rows_that_are_no_numbers(gpu_lib):
    q, k, v, offsets = batch([100], 4, 2, 128, seed=41)
    q = q.clone()
    clean = attn.attention_prompt(q, k, v, int32(offsets))
    q[7, 1, 3], q[50, 2, 0] = float("nan"), float("inf")
    out = attn.attention_prompt(q, k, v, int32(offsets))
    row = torch.zeros(100, 4, dtype=torch.bool, device="cuda")
    row[7, 1] = row[50, 2] = True
    assert torch.equal(out[~row], clean[~row]) and bool(torch.isnan(out[7, 1]).all())


def test_scores_of_minus_infinity_leave_zero(gpu_lib):
    """Rows all of whose scores are minus infinity weigh nothing, as in attention_int4."""
    q, k, v, offsets = batch([90], 2, 1, 64, seed=42)
    q, k = q.abs() + 0.5, k.clone()
    k[:70] = float("-inf")
    out = attn.attention_prompt(q, k, v, int32(offsets))
    assert not bool(out[:70].any())
    want = ora.prompt(q[70:], k[70:], v[70:], [0, 20])
    ora.check_prompt(out[70:], *want, 20)


def test_out(gpu_lib):
    q, k, v, offsets = batch([40, 0, 100], 4, 2, 128, seed=43, before=3, behind=4)
    want = attn.attention_prompt(q, k, v, int32(offsets))
    out = torch.full_like(want, 7.0)
    assert attn.attention_prompt(q, k, v, int32(offsets), out=out) is out
    assert torch.equal(out[3:offsets[-1]], want[3:offsets[-1]])
    assert bool((out[:3] == 7).all()) and bool((out[offsets[-1]:] == 7).all())
    into = q.contiguous()
    attn.attention_prompt(into, k, v, int32(offsets), out=into)
    assert torch.equal(into[3:offsets[-1]], want[3:offsets[-1]]) and torch.equal(into[:3], q[:3])


def test_offsets_are_not_trusted(gpu_lib):
    """Offsets beyond the rows name no rows there, offsets that decrease none at all."""
    q, k, v, _ = batch([64], 4, 2, 128, seed=44)
    assert not bool(attn.attention_prompt(q, k, v, int32([0, 50, 20, 64])).any())
    out = torch.full((64, 4, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    attn.attention_prompt(q, k, v, int32([0, 50, 20, 64]), out=out)
    assert bool((out == 5).all())
    got = attn.attention_prompt(q, k, v, int32([-7, 30, 1 << 30, 2147483647]))
    want = attn.attention_prompt(q, k, v, int32([0, 30, 64]))
    assert torch.equal(got, want)
    assert not bool(attn.attention_prompt(q, k, v, int32([64, 64])).any())
    assert not bool(attn.attention_prompt(q, k, v, int32([100, 200])).any())


def test_strides(gpu_lib):
    q, k, v, offsets = batch([150, 33], 6, 2, 128, seed=45)
    o = int32(offsets)
    want = attn.attention_prompt(q.contiguous(), k.contiguous(), v.contiguous(), o)
    rows = q.shape[0]
    flat = torch.zeros(rows * 2 * 128 + 1, dtype=torch.bfloat16, device="cuda")
    odd = flat[1:].view(rows, 2, 128)
    odd.copy_(v)
    wide = torch.zeros(rows, 2, 136, dtype=torch.bfloat16, device="cuda")
    wide[:, :, :128] = k
    turned = k.transpose(0, 1).contiguous().transpose(0, 1)
    strided = torch.stack((o, o), 1)[:, 0]
    for args in ((q, k, v, o), (q, wide[:, :, :128], odd, o), (q.transpose(0, 1).contiguous().transpose(0, 1), turned, v, strided)):
        assert torch.equal(attn.attention_prompt(*args), want)
    one = k[:, :1].expand(rows, 2, 128)  # heads that share their rows; then one row for all tokens
    assert torch.equal(attn.attention_prompt(q, one, one, o), attn.attention_prompt(q, one.contiguous(), one.contiguous(), o))
    same = k[:1].expand(rows, 2, 128)
    assert torch.equal(attn.attention_prompt(q, same, same, o), attn.attention_prompt(q, same.contiguous(), same.contiguous(), o))


def test_results_do_not_depend_on_the_run(gpu_lib):
    """A batch whose row tiles are cut and joined gives the same bits every time."""
    q, k, v, offsets = batch([1100, 60, 900], 16, 4, 128, seed=46)
    o = int32(offsets)
    want = attn.attention_prompt(q, k, v, o)
    for _ in range(20):
        assert torch.equal(attn.attention_prompt(q, k, v, o), want)


def test_captured(gpu_lib):
    """Two captured graphs and eager calls of the same operator, replayed in turn and beside each other."""
    q, k, v, offsets = batch([500, 20, 130], 8, 2, 128, seed=47)
    q, k, v, o = q.contiguous(), k.contiguous(), v.contiguous(), int32(offsets)
    attn.attention_prompt(q, k, v, o)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(attn.attention_prompt(q, k, v, o))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i, cut in enumerate((500, 1, 650, 300, 64)):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        o.copy_(int32([0, cut, max(cut, 640), 650]))
        want = attn.attention_prompt(q, k, v, o)
        for out in outs:
            out.fill_(9)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        assert torch.equal(attn.attention_prompt(q, k, v, o), want), i
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs), i


def test_streams(gpu_lib):
    """Calls on two streams at once, cut row tiles in both."""
    cases = [batch(lengths, 16, 4, 128, seed=50 + i) for i, lengths in enumerate(([1400], [700, 650]))]
    want = [attn.attention_prompt(q, k, v, int32(o)) for q, k, v, o in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    offsets = [int32(c[3]) for c in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for (q, k, v, _), o, stream in zip(cases, offsets, streams):
            with torch.cuda.stream(stream):
                got.append([attn.attention_prompt(q, k, v, o) for _ in range(3)])
        torch.cuda.synchronize()
        assert all(torch.equal(x, w) for g, w in zip(got, want) for x in g)


def test_far_rows(gpu_lib):
    """A batch whose byte offsets pass 32 bits: rows 32 KiB apart, prompts beyond 4 GiB of them."""
    rows, stride = 140000, 16384
    store = torch.empty(rows, stride, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    small = torch.randn(900, 4 * 128, generator=gen, device="cuda").to(torch.bfloat16)
    store[139000:139900, :512] = small
    x = store[:, :512].view(rows, 4, 128)
    q, k, v = x.split((2, 1, 1), 1)
    out = attn.attention_prompt(q, k, v, int32([139000, 139600, 139900]))
    y = small.view(900, 4, 128)
    want = ora.prompt(y[:, :2], y[:, 2:3], y[:, 3:], [0, 600, 900])
    ora.check_prompt(out[139000:139900], *want, 600)
    assert not bool(out[:139000].any())


def test_keys_beyond_4_gib_of_a_prompt(gpu_lib):
    """One prompt whose keys span more than 4 GiB: the last rows' own keys are beyond it.  All keys but a few
    are the same row, so the 64-bit result is a sum of few terms."""
    rows, stride = 70000, 32768
    store = torch.zeros(rows, stride, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(4)
    special = torch.tensor([5, 33000, 65537, 69999], device="cuda")
    store[special, :192] = torch.randn(4, 192, generator=gen, device="cuda").to(torch.bfloat16)
    x = store[:, :192].view(rows, 3, 64)
    q, k, v = x.split((1, 1, 1), 1)
    out = attn.attention_prompt(q, k, v, int32([0, rows]))
    for row in special.tolist():
        seen = special[special <= row]
        s = (k[seen, 0].double() @ q[row, 0].double()) * 64 ** -0.5
        w, zeros = torch.exp(s - s.amax().clamp(min=0)), torch.exp(-s.amax().clamp(min=0)) * (row + 1 - len(seen))
        total = w.sum() + zeros
        want = (w[:, None] * v[seen, 0].double()).sum(0) / total
        spread = (w[:, None] * v[seen, 0].double().abs()).sum(0) / total
        off = (out[row, 0].double() - want).abs()
        reach = (k[seen, 0].double().abs() @ q[row, 0].double().abs()).amax().expand(1) * 64 ** -0.5
        assert bool((off <= ora.prompt_tolerance(want[None], spread[None], reach, row)[0]).all())


@pytest.mark.parametrize("rows,heads", [(300, 2), (600, 86)])
def test_rows_at_the_widest_steps(gpu_lib, rows, heads):
    """Rows of q, k and v 2^22 elements apart, which the kernel steps through, and further, which are copied;
    a tile of one token a row then spans 2 GiB."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(rows, 3 * heads, 64, generator=gen, device="cuda").to(torch.bfloat16)
    o = int32([0, rows - 40, rows])
    want = attn.attention_prompt(*x.split(heads, 1), o)
    for stride in (1 << 22, (1 << 22) + 8):
        store = torch.empty(rows, stride, dtype=torch.bfloat16, device="cuda")
        wide = store[:, :3 * heads * 64].view(rows, 3 * heads, 64)
        wide.copy_(x)
        assert torch.equal(attn.attention_prompt(*wide.split(heads, 1), o), want)
        del wide, store
    q, k, v = x.split(heads, 1)
    check(want, q, k, v, [0, rows - 40, rows])


def test_heads_far_apart(gpu_lib):
    """Heads of q up to 2^28 elements apart in a group, and beyond (copied)."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(70, 6, 64, generator=gen, device="cuda").to(torch.bfloat16)
    q, k, v = x.split((4, 1, 1), 1)
    want = attn.attention_prompt(q, k, v, int32([0, 70]))
    for apart in (1 << 26, (1 << 26) + 8):
        store = torch.empty(4 * apart, dtype=torch.bfloat16, device="cuda")
        far = store.as_strided((70, 4, 64), (64, apart, 1))
        far.copy_(q)
        assert torch.equal(attn.attention_prompt(far, k, v, int32([0, 70])), want)
        del far, store


def test_refusals(gpu_lib):
    """Arguments that the kernel cannot take raise in front of any launch."""
    q, k, v, offsets = batch([20, 5], 4, 2, 128, seed=51)
    o = int32(offsets)
    out = torch.empty(25, 4, 128, dtype=torch.bfloat16, device="cuda")
    for change in ({"q": q.float()}, {"q": q.cpu()}, {"q": q[..., :96]}, {"q": q[:, :3]}, {"q": q[:24]}, {"q": q[0]},
                   {"k": k[..., :64]}, {"k": k[:, :0], "v": v[:, :0]}, {"k": k.half()}, {"k": k[:24]}, {"v": v[:, :1]}, {"v": v[:24]},
                   {"v": v.cpu()}, {"cu_query_lens": o.long()}, {"cu_query_lens": o[:1]}, {"cu_query_lens": o.cpu()},
                   {"cu_query_lens": o[None]}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")},
                   {"scale": float("inf")}, {"max_query_len": 0}, {"out": out[:24]}, {"out": out.float()},
                   {"out": out.transpose(0, 1).contiguous().transpose(0, 1)}, {"out": out.cpu()}):
        with pytest.raises(ValueError):
            attn.attention_prompt(**{**dict(q=q, k=k, v=v, cu_query_lens=o), **change})


def test_more_requests_than_lanes(gpu_lib):
    """Empty places and prompts of one to some tokens, more than a wave looks at in one turn, and a long one
    behind them."""
    lengths = ([0, 1, 2, 0, 5] * 60) + [400] + [0] * 70 + [3]
    for heads, kv_heads, dim in ((8, 2, 128), (3, 3, 64)):
        q, k, v, offsets = batch(lengths, heads, kv_heads, dim, seed=52, before=3, behind=9)
        out = attn.attention_prompt(q, k, v, int32(offsets))
        check(out, q, k, v, offsets)
        assert not bool(out[:3].any()) and not bool(out[-9:].any())


@pytest.mark.parametrize("heads,kv_heads,dim,lengths", [(32, 8, 128, [2039]), (86, 86, 64, [300, 333]), (32, 8, 128, [40] * 30)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_no_numbers_in_larger_batches(gpu_lib, heads, kv_heads, dim, lengths, value):
    """One channel of some values is no number: every row in front of them, every other channel and every
    other sequence keeps its bits; rows that see one get it."""
    q, k, v, offsets = batch(lengths, heads, kv_heads, dim, seed=53)
    v = v.clone()
    rows, o = q.shape[0], int32(offsets)
    want = attn.attention_prompt(q, k, v, o)
    clean = v.clone()
    spots = [(0, 0, 3), (rows // 3, 1, dim - 1), (rows - 1, kv_heads - 1, 17), (offsets[1] - 1, 0, 40), (rows // 2, 2, 0)]
    hit = torch.zeros(rows, heads, dim, dtype=torch.bool, device="cuda")
    group = heads // kv_heads
    for row, head, channel in spots:
        v[row, head, channel] = value
        clean[row, head, channel] = 0
        end = next(e for e in offsets if e > row)
        hit[row:end, head * group:(head + 1) * group, channel] = True
    got = attn.attention_prompt(q, k, v, o)
    base = attn.attention_prompt(q, k, clean, o)
    touched = torch.zeros_like(hit)
    for row, head, channel in spots:
        touched[:, head * group:(head + 1) * group, channel] = True
    assert torch.equal(got[~hit], base[~hit]) and torch.equal(got[~touched], want[~touched])
    assert torch.equal(got[hit].float().nan_to_num(7.0, 8.0, 9.0), torch.full_like(got[hit].float(), value).nan_to_num(7.0, 8.0, 9.0))


def larger(lengths, heads, rows):
    """The lengths and a prompt behind them that makes it that many rows of all heads together."""
    return lengths + [max(1, -(-rows // heads) - sum(lengths))]


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (16, 2, 64), (40, 8, 128), (12, 12, 64)])
@pytest.mark.parametrize("rows", [16000, 17000, 52000])
def test_packed_lengths_in_batches_of_each_size(gpu_lib, heads, kv_heads, dim, rows):
    """The same lengths where keys are split among waves, and in workgroups of four waves and of eight."""
    lengths = larger([0, 129, 1, 33], heads, rows)
    q, k, v, offsets = batch(lengths, heads, kv_heads, dim, seed=54)
    check(attn.attention_prompt(q, k, v, int32(offsets)), q, k, v, offsets)


@pytest.mark.parametrize("rows", [16000, 17000, 52000])
@pytest.mark.parametrize("dim", [64, 128])
def test_keys_that_are_no_numbers_in_batches_of_each_size(gpu_lib, dim, rows):
    """A key that is no number reaches the rows that see it, and no others; rows whose every score is
    minus infinity stay zero; scores that lead all before them by far take over."""
    lengths = larger([200, 70], 16, rows)
    q, k, v, offsets = batch(lengths, 16, 4, dim, seed=55)
    o = int32(offsets)
    want = attn.attention_prompt(q, k, v, o)
    k = k.clone()
    k[150, 0, 5] = float("nan")
    k[230, 3, 5] = float("inf")
    out = attn.attention_prompt(q, k, v, o)
    spoilt = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    spoilt[150:200, :4] = True
    spoilt[230:270, 12:] = True
    assert torch.equal(out[~spoilt], want[~spoilt])
    assert bool(out[150:200, :4].isnan().all())
    q, k = q.clone(), k.nan_to_num(0.0, 0.0, 0.0)
    q[200:270, 2] = 1.0
    k[200:270, 0] = -float("inf")
    out = attn.attention_prompt(q, k, v, o)
    assert not bool(out[200:270, 2].any())
    q, k, v, offsets = batch(lengths, 16, 4, dim, seed=56)
    k = k.clone()
    k[190] *= 20  # leads by far in about half of the rows
    k[offsets[-1] - 40:] *= 12
    check(attn.attention_prompt(q, k, v, int32(offsets)), q, k, v, offsets)


@pytest.mark.parametrize("heads,lengths", [(8, [700, 900]), (16, [1100, 60, 900]), (32, [2039]), (32, [1500, 0, 1100, 1])])
def test_each_form_captured_repeated_and_in_place(gpu_lib, heads, lengths):
    """The same bits from eager calls, from a captured one on every replay with eager calls between them, and
    with the output in the queries' place."""
    q, k, v, offsets = batch(lengths, heads, 4, 128, seed=57)
    q, o = q.contiguous(), int32(offsets)
    want = attn.attention_prompt(q, k, v, o)
    check(want, q, k, v, offsets)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = attn.attention_prompt(q, k, v, o)
    for _ in range(4):
        got.fill_(5)
        graph.replay()
        assert torch.equal(attn.attention_prompt(q, k, v, o), want)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    for _ in range(4):
        mine = q.clone()
        assert attn.attention_prompt(mine, k, v, o, out=mine) is mine
        assert torch.equal(mine, want)


@pytest.mark.parametrize("heads,kv_heads,lengths", [(16, 16, [290] * 50), (16, 4, [64] * 120 + [3]), (16, 16, [4100])])
def test_grids_of_small_heads(gpu_lib, heads, kv_heads, lengths):
    """Heads of 64 channels in batches that fill four waves a SIMD, cut row tiles and whole ones."""
    q, k, v, offsets = batch(lengths, heads, kv_heads, 64, seed=58)
    o = int32(offsets)
    out = attn.attention_prompt(q, k, v, o)
    check(out, q, k, v, offsets)
    assert all(torch.equal(attn.attention_prompt(q, k, v, o), out) for _ in range(5))


@pytest.mark.parametrize("heads,kv_heads,dim,lengths", [(130, 1, 64, [1, 40, 3]), (300, 2, 128, [150, 1, 60]), (100, 1, 64, [600]),
                                                        (96, 1, 128, [1030]), (77, 1, 128, [333, 9])])
def test_large_groups(gpu_lib, heads, kv_heads, dim, lengths):
    """Groups of more heads than a wave, or a row tile, has rows: a tile is part of a token, or ends inside one."""
    q, k, v, offsets = batch(lengths, heads, kv_heads, dim, seed=59, before=1, behind=2)
    check(attn.attention_prompt(q, k, v, int32(offsets)), q, k, v, offsets)
