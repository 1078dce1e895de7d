"""Batches for the tests of attention's precision: values that name their keys, and the kernels'
roundings in plain arithmetic."""
import torch

from oracle import kv4_oracle as ora


def mark_values(batch, dim, keys=16):
    """Overwrites the batch's values: those of each `keys` neighbouring keys of a sequence are zero but
    in one channel, 15 times their scale there, so that a group of keys that is lost, or counted
    twice, changes that channel by its whole share.  Neighbouring groups have channels far apart."""
    words = batch.cache.view(torch.int32)
    n, block = dim // 8, batch.block
    bit = torch.tensor([4 * ora.AWQ_ORDER.index(c) for c in range(8)])
    for r, seq in enumerate(batch.seq):
        p = torch.arange(seq)
        page, token = torch.tensor(batch.tables[r])[p // block], p % block
        at = block * n + token // 4 * n * 4 + token % 4
        for w in range(n):
            words[page, :, at + 4 * w] = 0
        channel = marked_channel(p, dim, keys)
        word = 15 << bit[channel % 8]
        words[page, :, at + 4 * (channel // 8)] = torch.where(word >> 31 > 0, word - (1 << 32), word).to(torch.int32)[:, None]
        meta = 2 * block * n + block + token
        words[page, :, meta] = (words[page, :, meta] & -65536) | 0x4300  # its scale, zero point 0


def marked_channel(key, dim, keys=16):
    return key // keys * (dim // 2 + 13) % dim


def emulate(q, cache, tables, seq_lens, offsets, block, kernel):
    """The output of a kernel that rounds what the split ("split") or the prompt kernel ("prompt") rounds,
    or keys, values and weights to bf16 ("bf16"), or weights times scales alone to bf16 ("weights"), and nothing
    else, as bf16."""
    rows, heads, dim = q.shape
    kv_heads = cache.shape[1]
    group = heads // kv_heads
    out = torch.zeros(rows, heads, dim, dtype=torch.float64)
    to = {"split": lambda x: x, "weights": lambda x: x, "prompt": lambda x: x.half().double(), "bf16": lambda x: x.bfloat16().double()}[kernel]
    for r, seq in enumerate(seq_lens):
        first, n = offsets[r], offsets[r + 1] - offsets[r]
        slots = [tables[r][p // block] * block + p % block for p in range(seq)]
        k, v, _, vs = ora.load(cache, slots, block)
        for t in range(n):
            sees = seq - n + t + 1
            for h in range(heads):
                g = h // group
                s = dim ** -0.5 * to(k[:sees, g]) @ q[first + t, h].double()
                p = torch.exp(s - s.max())
                if kernel == "split":
                    x = p * vs[:sees, g]
                    high = x.bfloat16().double()
                    w = (high + (x - high).bfloat16().double()) / vs[:sees, g]
                elif kernel == "weights":
                    w = (p * vs[:sees, g]).bfloat16().double() / vs[:sees, g]
                else:
                    w = to(p)
                out[first + t, h] = w @ to(v[:sees, g]) / p.sum()
    return out.bfloat16()
