"""A decoder layer's attention half as a server runs it, step after step: ``kv_step``, the fused
input norm and QKV projection, per-head norms, rotary (plain torch, from the step's positions),
``Attention`` over a 4-bit cache, and O with the residual add -- prompts, a chunk, drafts and
decode tokens mixed, padded rows, and decode steps from a captured graph.

Every step's bookkeeping and cache bytes are the oracle's of the rows that the layer stored, and its
attention output lies within the oracle's bound (oracle/kv4_oracle.py); a captured step gives the
eager one's bits on every replay, with the eager program's own work in between."""
import importlib

import pytest
import torch

from awq_helpers import awq_mod, random_awq_gpu, random_x_gpu
from oracle import kv4_oracle as ora

pytestmark = pytest.mark.gpu

attn = importlib.import_module("llm-serve_amd.layers.attention")

HIDDEN, HEADS, KV_HEADS = 1024, 8, 2
BLOCK, BLOCKS, WIDTH, REQUESTS = 16, 40, 8, 4


class Layer:
    def __init__(self, head_dim):
        linear = importlib.import_module("llm-serve_amd.layers.linear")
        layernorm = importlib.import_module("llm-serve_amd.layers.layernorm")
        cfg = awq_mod().AWQRuntimeConfig(bits=4, group_size=128, zero_point=True, version="gemm", backend="autoawq",
                                         activation_dtype=torch.bfloat16)
        self.dim = head_dim
        with torch.device("cuda"):
            self.qkv = linear.QKVParallelLinear(HIDDEN, head_dim, HEADS, KV_HEADS, quant_config=cfg)
            self.o = linear.RowParallelLinear(HEADS * head_dim, HIDDEN, quant_config=cfg)
            self.norm, self.q_norm, self.k_norm = (layernorm.RMSNorm(n) for n in (HIDDEN, head_dim, head_dim))
        for i, part in enumerate((self.qkv, self.o)):
            qw, qz, s = random_awq_gpu(part.qweight.shape[0], part.scales.shape[1], seed=700 + i)
            part.qweight.data.copy_(qw)
            part.qzeros.data.copy_(qz)
            part.scales.data.copy_(s)
            part.quant_method.process_weights_after_loading(part)
        self.attention = attn.Attention(HEADS, head_dim, head_dim ** -0.5, KV_HEADS, block_size=BLOCK)
        self.attention.kv_cache = attn.new_kv_cache_int4(BLOCKS, BLOCK, KV_HEADS, head_dim)
        half = torch.arange(head_dim // 2, device="cuda", dtype=torch.float32)
        self.frequency = 10000.0 ** (-half / (head_dim // 2))

    def rotary(self, x, positions):
        angle = (positions.float()[:, None] * self.frequency)[:, None]
        a, b = x.float().chunk(2, -1)
        return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1).to(torch.bfloat16)

    def run(self, h, residual, step, max_query_len, record=None):
        rows, dim = h.shape[0], self.dim
        qkv, residual = self.qkv.forward_rmsnorm(self.norm, h, residual)
        q, k, v = qkv.split((HEADS * dim, KV_HEADS * dim, KV_HEADS * dim), -1)
        q = self.rotary(self.q_norm(q.view(rows, HEADS, dim)), step.positions)
        k = self.rotary(self.k_norm(k.view(rows, KV_HEADS, dim)), step.positions)
        out = self.attention(q, k, v, step, max_query_len=max_query_len)
        if record is not None:
            record.update(q=q, k=k, v=v.reshape(rows, KV_HEADS, dim), out=out.view(rows, HEADS, dim))
        return self.o.forward_residual(out, residual), residual


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def check_step(layer, record, step, before, new, context, tables, free):
    """The recorded step against the oracle, from the cache and tables before it."""
    rows = record["q"].shape[0]
    offsets, seq, positions, slots, want_tables, used = ora.step(new, context, tables, free, BLOCK, rows)
    assert (step.cu_query_lens.tolist(), step.seq_lens.tolist()) == (offsets, seq)
    assert (step.positions.tolist(), step.slots.tolist()) == (positions, slots)
    assert (step.block_tables.tolist(), step.blocks_used.tolist()) == (want_tables, [used])
    ora.store(record["k"], record["v"], before, torch.tensor(slots), BLOCK)
    assert torch.equal(layer.attention.kv_cache.cpu(), before)
    want, spread = ora.attention(record["q"], before, want_tables, seq, offsets, BLOCK)
    off = (record["out"].cpu().double() - want).abs()
    assert bool((off <= ora.tolerance(want, spread)).all())
    assert not bool(record["out"][offsets[-1]:].any())
    return want_tables, used


@pytest.mark.parametrize("head_dim", [64, 128])
@torch.inference_mode()
def test_serving_steps(gpu_lib, head_dim):
    layer = Layer(head_dim)
    free = list(range(BLOCKS - 1, -1, -1))
    tables = [[-1] * WIDTH for _ in range(REQUESTS)]
    context = [0] * REQUESTS
    plan = [([40, 17, 0, 1], 0),     # prompts, one of a single token, an empty place
            ([1, 1, 70, 1], 3),      # a prompt beside decode tokens, padded rows
            ([4, 1, 20, 8], 0),      # drafts and a chunk behind cached tokens
            ([1, 1, 1, 1], 2),
            ([1, 0, 1, 1], 1)]
    for i, (new, pad) in enumerate(plan):
        rows = sum(new) + pad
        print("step", head_dim, i, new, flush=True)
        before = layer.attention.kv_cache.cpu()
        step = attn.kv_step(int32(new), int32(context), int32(tables), int32(free), block_size=BLOCK, num_tokens=rows)
        record = {}
        h, _ = layer.run(random_x_gpu(rows, HIDDEN, seed=10 + i), random_x_gpu(rows, HIDDEN, seed=20 + i), step, max(new),
                         record)
        assert bool(torch.isfinite(h.float()).all())
        tables, used = check_step(layer, record, step, before, new, context, tables, free)
        free = free[used:]
        context = [c + n for c, n in zip(context, new)]


@torch.inference_mode()
def test_captured_decode_steps(gpu_lib):
    """One captured graph of a whole decode step, ``kv_step`` included, for each sequence's next
    token: replayed over steps that open new blocks, each against the eager step on a copy of the
    cache, whose own run lies between the replays."""
    layer = Layer(128)
    context = [30, 15, 63, 1]
    free = list(range(BLOCKS))
    tables = int32([[-1] * WIDTH for _ in range(REQUESTS)])
    step = attn.kv_step(int32(context), int32([0] * REQUESTS), tables, int32(free), block_size=BLOCK,
                        num_tokens=sum(context))
    layer.run(random_x_gpu(sum(context), HIDDEN, seed=1), random_x_gpu(sum(context), HIDDEN, seed=2), step, max(context))
    free = free[int(step.blocks_used):]

    ones, lengths, blocks = int32([1] * REQUESTS), int32(context), int32(free[:REQUESTS])
    h, residual = random_x_gpu(REQUESTS, HIDDEN, seed=3), random_x_gpu(REQUESTS, HIDDEN, seed=4)

    def decode():
        s = attn.kv_step(ones, lengths, tables, blocks, block_size=BLOCK, num_tokens=REQUESTS)
        return layer.run(h, residual, s, 1) + (s.slots, s.blocks_used)

    cache = layer.attention.kv_cache
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = decode()
    for i in range(20):
        h.copy_(random_x_gpu(REQUESTS, HIDDEN, seed=100 + i))
        residual.copy_(random_x_gpu(REQUESTS, HIDDEN, seed=200 + i))
        lengths.copy_(int32(context))
        blocks.copy_(int32(free[:REQUESTS]))
        state = cache.clone(), tables.clone()
        want = [t.clone() for t in decode()]
        after = cache.clone(), tables.clone()
        cache.copy_(state[0])
        tables.copy_(state[1])
        for t in got:
            t.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i
        assert torch.equal(cache, after[0]) and torch.equal(tables, after[1]), i
        assert bool((got[2] >= 0).all())
        free = free[int(got[3]):]
        context = [c + 1 for c in context]


@torch.inference_mode()
def test_two_servers_on_two_streams(gpu_lib):
    """Two engines' steps on streams of their own at once give what they give alone."""
    layers = [Layer(128) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    new = [90, 30, 1, 20]

    def steps(layer, seed):
        outs, tables = [], int32([[-1] * WIDTH for _ in range(REQUESTS)])
        context, free = [0] * REQUESTS, list(range(BLOCKS))
        for i, n in enumerate((new, [1] * REQUESTS, [5] * REQUESTS)):
            s = attn.kv_step(int32(n), int32(context), tables, int32(free), block_size=BLOCK, num_tokens=sum(n))
            h, _ = layer.run(random_x_gpu(sum(n), HIDDEN, seed=seed + i), random_x_gpu(sum(n), HIDDEN, seed=seed + 9), s,
                             max(n))
            outs.append(h)
            free = free[sum(-(-(c + x) // BLOCK) - -(-c // BLOCK) for c, x in zip(context, n)):]
            context = [c + x for c, x in zip(context, n)]
        return outs

    want = [steps(layer, 300 + 50 * i) for i, layer in enumerate(layers)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for i, (layer, stream) in enumerate(zip(layers, streams)):
            with torch.cuda.stream(stream):
                got.append(steps(layer, 300 + 50 * i))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for a, b in zip(got, want) for x, y in zip(a, b))
