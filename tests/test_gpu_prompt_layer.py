"""A decoder layer's attention half with everything between its projections in the library:
``Attention.forward_qkv`` over whole prompts, then over chunks and decode tokens behind them, as a server
runs it -- padded rows, captured steps, two engines at once.

Each step's queries, keys, cache bytes and output are the bits of the calls that it is made of
(``qk_norm_rope``, ``store_kv_int4`` and the attention of its kind) on a copy of the cache, and lie within the
bounds of the 64-bit definitions (oracle/prompt_oracle.py, oracle/kv4_oracle.py)."""
import importlib

import pytest
import torch

from awq_helpers import random_x_gpu
from oracle import kv4_oracle, prompt_oracle
from test_gpu_attention_layer import BLOCK, BLOCKS, HEADS, HIDDEN, KV_HEADS, REQUESTS, WIDTH, Layer, int32

pytestmark = pytest.mark.gpu

attn = importlib.import_module("llm-serve_amd.layers.attention")
rope = importlib.import_module("llm-serve_amd.layers.rotary_embedding")


class FusedLayer(Layer):
    def __init__(self, head_dim, seed=1):
        super().__init__(head_dim)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for norm in (self.q_norm, self.k_norm):
            norm.weight.data.copy_(1 + 0.2 * torch.randn(head_dim, generator=gen, device="cuda"))
        self.rotary = rope.RotaryEmbedding(head_dim, head_dim, 256, 10000.0)

    def parts(self, qkv):
        return qkv.view(-1, HEADS + 2 * KV_HEADS, self.dim).split((HEADS, KV_HEADS, KV_HEADS), 1)

    def run(self, h, residual, step, max_query_len, whole=False, record=None):
        qkv, residual = self.qkv.forward_rmsnorm(self.norm, h, residual)
        out = self.attention.forward_qkv(qkv, step, self.rotary.cos_sin_cache, q_weight=self.q_norm.weight,
                                         k_weight=self.k_norm.weight, eps=self.q_norm.eps, whole_prompts=whole,
                                         max_query_len=max_query_len)
        if record is not None:
            record.update(qkv=qkv, out=out.view(-1, HEADS, self.dim))
        return self.o.forward_residual(out, residual), residual

    def apart(self, qkv, step, cache, whole):
        """(q, k, v, out) of the same step from its single calls, into another cache."""
        q, k, v = self.parts(qkv)
        q, k = self.rotary(step.positions, q, k, q_weight=self.q_norm.weight, k_weight=self.k_norm.weight,
                           eps=self.q_norm.eps)
        attn.store_kv_int4(k, v, cache, step.slots, block_size=BLOCK)
        if whole:
            return q, k, v, attn.attention_prompt(q, k, v, step.cu_query_lens)
        return q, k, v, attn.attention_int4(q, cache, step.block_tables, step.seq_lens, step.cu_query_lens, block_size=BLOCK)


def check_step(layer, record, step, before, whole):
    q, k, v, out = layer.apart(record["qkv"], step, before, whole)
    assert torch.equal(record["out"], out) and torch.equal(layer.attention.kv_cache, before)
    xq, xk, _ = layer.parts(record["qkv"])
    for got, x, norm in ((q, xq, layer.q_norm), (k, xk, layer.k_norm)):
        want, size = prompt_oracle.turn(x, step.positions, layer.dim, 10000.0, norm.weight, norm.eps)
        assert bool(((got.double() - want).abs() <= prompt_oracle.turn_tolerance(want, size)).all())
    offsets = step.cu_query_lens.tolist()
    if whole:
        prompt_oracle.check_prompt(out, *prompt_oracle.prompt(q, k, v, offsets),
                                   max(b - a for a, b in zip(offsets, offsets[1:])))
    else:
        want, spread = kv4_oracle.attention(q, before.cpu(), step.block_tables.tolist(), step.seq_lens.tolist(), offsets, BLOCK)
        assert bool(((out.cpu().double() - want).abs() <= kv4_oracle.tolerance(want, spread)).all())
    assert not bool(out[offsets[-1]:].any())


@pytest.mark.parametrize("head_dim", [64, 128])
@torch.inference_mode()
def test_serving_steps(gpu_lib, head_dim):
    layer = FusedLayer(head_dim)
    cache = layer.attention.kv_cache
    free, tables, context = list(range(BLOCKS)), int32([[-1] * WIDTH for _ in range(REQUESTS)]), [0] * REQUESTS
    plan = [([70, 17, 0, 1], 3, True),     # prompts, an empty place, padded rows
            ([1, 1, 90, 1], 0, False),     # a prompt beside decode tokens: all from the cache
            ([4, 1, 20, 8], 2, False),     # drafts and a chunk behind cached tokens
            ([1, 0, 1, 1], 1, False)]
    for i, (new, pad, whole) in enumerate(plan):
        rows, before = sum(new) + pad, cache.clone()
        print("step", head_dim, i, new, flush=True)
        step = attn.kv_step(int32(new), int32(context), tables, int32(free), block_size=BLOCK, num_tokens=rows)
        record = {}
        h, _ = layer.run(random_x_gpu(rows, HIDDEN, seed=30 + i), random_x_gpu(rows, HIDDEN, seed=40 + i), step, max(new),
                         whole, record)
        assert bool(torch.isfinite(h.float()).all())
        check_step(layer, record, step, before, whole)
        free = free[int(step.blocks_used):]
        context = [c + n for c, n in zip(context, new)]


@pytest.mark.parametrize("whole,rows", [(True, 100), (False, 16)])
@torch.inference_mode()
def test_captured_steps(gpu_lib, whole, rows):
    """One captured graph of a whole step of padded rows, replayed over other lengths and inputs, each
    against the eager step on a copy of the cache, whose own run lies between the replays."""
    layer = FusedLayer(128)
    cache = layer.attention.kv_cache
    context = [0] * REQUESTS
    free, tables = list(range(BLOCKS)), int32([[-1] * WIDTH for _ in range(REQUESTS)])
    if not whole:
        context = [30, 15, 33, 1]
        step = attn.kv_step(int32(context), int32([0] * REQUESTS), tables, int32(free), block_size=BLOCK, num_tokens=79)
        layer.run(random_x_gpu(79, HIDDEN, seed=1), random_x_gpu(79, HIDDEN, seed=2), step, 33, True)
        free = free[int(step.blocks_used):]
    new, lengths, blocks, first = int32([1] * REQUESTS), int32(context), int32(free[:24]), tables.clone()
    h, residual = random_x_gpu(rows, HIDDEN, seed=3), random_x_gpu(rows, HIDDEN, seed=4)

    def run():
        s = attn.kv_step(new, lengths, tables, blocks, block_size=BLOCK, num_tokens=rows)
        return layer.run(h, residual, s, None, whole) + (s.slots,)

    run()
    tables.copy_(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i in range(12):
        h.copy_(random_x_gpu(rows, HIDDEN, seed=100 + i))
        residual.copy_(random_x_gpu(rows, HIDDEN, seed=200 + i))
        new.copy_(int32([[1, 1, 1, 1], [rows - 3, 1, 0, 2], [3, 2, 5, 0]][i % 3]))
        state = cache.clone()
        tables.copy_(first)
        want = [t.clone() for t in run()]
        after = cache.clone(), tables.clone()
        cache.copy_(state)
        tables.copy_(first)
        for t in got:
            t.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i
        assert torch.equal(cache, after[0]) and torch.equal(tables, after[1]), i


@torch.inference_mode()
def test_two_engines_on_two_streams(gpu_lib):
    layers = [FusedLayer(128, seed) for seed in (1, 2)]
    streams = [torch.cuda.Stream() for _ in layers]

    def steps(layer, seed):
        outs, context = [], [0] * REQUESTS
        free, tables = list(range(BLOCKS)), int32([[-1] * WIDTH for _ in range(REQUESTS)])
        for i, n in enumerate(([100, 30, 1, 20], [1] * REQUESTS, [5] * REQUESTS)):
            s = attn.kv_step(int32(n), int32(context), tables, int32(free), block_size=BLOCK, num_tokens=sum(n))
            outs.append(layer.run(random_x_gpu(sum(n), HIDDEN, seed=seed + i), random_x_gpu(sum(n), HIDDEN, seed=seed + 9), s,
                                  max(n), i == 0)[0])
            free = free[sum(-(-(c + x) // BLOCK) - -(-c // BLOCK) for c, x in zip(context, n)):]
            context = [c + x for c, x in zip(context, n)]
        return outs

    want = [steps(layer, 400 + 50 * i) for i, layer in enumerate(layers)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for i, (layer, stream) in enumerate(zip(layers, streams)):
            with torch.cuda.stream(stream):
                got.append(steps(layer, 400 + 50 * i))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for a, b in zip(got, want) for x, y in zip(a, b))


@torch.inference_mode()
def test_a_prompt_in_parts_is_near_the_prompt_at_once(gpu_lib):
    """The same prompt through the bf16 path at once and from the cache in two chunks: both attend to the
    same tokens, the second to 4-bit copies of them.  A code's rounding (half a step of a fifteenth of the
    range of a row of some 2.5 sigma to either side) moves a value by 0.1 sigma: the outputs, averages of
    values, agree to a correlation far above what a key out of place would leave."""
    layer = FusedLayer(128)
    gen = torch.Generator(device="cuda").manual_seed(9)
    qkv = torch.randn(100, (HEADS + 2 * KV_HEADS) * 128, generator=gen, device="cuda").to(torch.bfloat16)
    outs = []
    for cuts, whole in (([100], True), ([60, 40], False)):
        tables, context, free, got = int32([[-1] * WIDTH]), 0, list(range(BLOCKS)), []
        for n in cuts:
            step = attn.kv_step(int32([n]), int32([context]), tables, int32(free), block_size=BLOCK, num_tokens=n)
            got.append(layer.attention.forward_qkv(qkv[context:context + n], step, layer.rotary.cos_sin_cache,
                                                   q_weight=layer.q_norm.weight, k_weight=layer.k_norm.weight,
                                                   whole_prompts=whole))
            free = free[int(step.blocks_used):]
            context += n
        outs.append(torch.cat(got).double().view(100, HEADS, 128))
    for x, y in zip(outs[0].flatten(0, 1), outs[1].flatten(0, 1)):
        assert float((x * y).sum()) > 0.9 * float(x.norm() * y.norm())
