"""The 4-bit key/value cache and attention over it in plain 64-bit arithmetic on the CPU (torch):
the definition that the HIP kernels are tested against.  Nothing here is shared with them.

A cache is a uint8 tensor [blocks, kv heads, block_size * (dim + 8)]; a row's channel stands for
scale * (code - zero)."""
from __future__ import annotations

import torch

AWQ_ORDER = (0, 2, 4, 6, 1, 3, 5, 7)  # nibble i of a word holds channel AWQ_ORDER[i]


def bf16_rne(x: torch.Tensor) -> torch.Tensor:
    """x (float64) rounded once to bf16, as float64: exact where x has at most 24 significant
    bits or is not within 2^-24 of a rounding border (torch rounds through float32)."""
    return x.to(torch.bfloat16).double()


def quantize_rows(x: torch.Tensor):
    """(codes, scale, zero) of rows x [..., dim], all float64."""
    x = x.double()
    low = x.amin(-1).clamp(max=0)
    scale = bf16_rne((x.amax(-1).clamp(min=0) - low) / 15)
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    zero = torch.round(-low / safe).clamp(0, 15)
    code = (torch.round(x / safe[..., None]) + zero[..., None]).clamp(0, 15)
    dead = ~(scale > 0)
    zero, code = torch.where(dead, 0, zero), torch.where(dead[..., None], 0, code)
    broken = ~torch.isfinite(x).all(-1)
    scale = torch.where(broken, torch.nan, scale)
    zero, code = torch.where(broken, 0, zero), torch.where(broken[..., None], 0, code)
    return code, scale, zero


def row_values(code, scale, zero):
    return scale[..., None] * (code - zero[..., None])


def _words(code: torch.Tensor) -> torch.Tensor:
    """Codes [..., dim] -> words [..., dim / 8] (int64 below 2^32)."""
    groups = code.to(torch.int64).unflatten(-1, (-1, 8))
    return sum(groups[..., channel] << (4 * nibble) for nibble, channel in enumerate(AWQ_ORDER))


def _put(page: torch.Tensor, index: int, word: int) -> None:
    for b in range(4):
        page[4 * index + b] = (word >> (8 * b)) & 255


def _get(page: torch.Tensor, index: int) -> int:
    return sum(int(page[4 * index + b]) << (8 * b) for b in range(4))


def _where(token: int, word: int, block: int, dim: int):
    """Word indices of a token's K word, V word, K meta and V meta in its page."""
    n = dim // 8
    return (token * n + word, block * n + (token // 4 * n + word) * 4 + token % 4, 2 * block * n + token,
            2 * block * n + block + token)


def store(k, v, cache, slots, block):
    """Rows into `cache` (CPU, in place)."""
    dim = k.shape[2]
    parts = []
    for x in (k, v):
        code, scale, zero = quantize_rows(x.cpu())
        bits = scale.to(torch.bfloat16).view(torch.int16).to(torch.int64) & 0xFFFF
        bits = torch.where(torch.isnan(scale), 0x7FC0, bits)
        parts.append((_words(code), (bits << 16) | 0x4300 | zero.to(torch.int64)))
    for t, slot in enumerate(slots.tolist()):
        if slot < 0 or slot >= cache.shape[0] * block:
            continue
        for h in range(cache.shape[1]):
            page = cache[slot // block, h]
            for w in range(dim // 8):
                at = _where(slot % block, w, block, dim)
                _put(page, at[0], int(parts[0][0][t, h, w]))
                _put(page, at[1], int(parts[1][0][t, h, w]))
            _put(page, at[2], int(parts[0][1][t, h]))
            _put(page, at[3], int(parts[1][1][t, h]))


def load(cache, slots, block):
    """(k, v, k scale, v scale) float64 of the rows at slots; zeros outside the cache."""
    heads, dim = cache.shape[1], cache.shape[2] // block - 8
    out = [torch.zeros(len(slots), heads, dim, dtype=torch.float64) for _ in range(2)]
    scales = [torch.zeros(len(slots), heads, dtype=torch.float64) for _ in range(2)]
    words = cache.cpu().reshape(-1).view(torch.int32).view(cache.shape[0], heads, -1).to(torch.int64) & 0xFFFFFFFF
    at = torch.as_tensor(slots).to(torch.int64).cpu()
    live = (at >= 0) & (at < cache.shape[0] * block)
    page = words[torch.where(live, at // block, 0)]  # [T, heads, words]
    token = torch.where(live, at % block, 0)
    n = dim // 8
    w = torch.arange(n)
    index_k = token[:, None] * n + w
    index_v = block * n + (token[:, None] // 4 * n + w) * 4 + token[:, None] % 4
    meta = [2 * block * n + token, 2 * block * n + block + token]
    for part, index in enumerate((index_k, index_v)):
        row = page.gather(2, index[:, None].expand(-1, heads, -1))
        m = page.gather(2, meta[part][:, None, None].expand(-1, heads, 1))[..., 0]
        code = torch.zeros(len(at), heads, dim, dtype=torch.float64)
        for nibble, channel in enumerate(AWQ_ORDER):
            code[..., channel::8] = ((row >> (4 * nibble)) & 15).double()
        high = (m >> 16).to(torch.int32).to(torch.int16).view(torch.bfloat16).double()
        zero = (m & 0xFFFF).to(torch.int32).to(torch.int16).view(torch.bfloat16).double() - 128
        out[part] = torch.where(live[:, None, None], row_values(code, high, zero), 0)
        scales[part] = torch.where(live[:, None], high, 0)
    return out[0], out[1], scales[0], scales[1]


def step(query_lens, context_lens, tables, free, block, tokens):
    """(offsets, seq_lens, positions, slots, tables, used) as lists; tables is a list of rows."""
    tables = [list(row) for row in tables]
    width = len(tables[0])
    offsets, seq, positions, slots = [0], [], [0] * tokens, [-1] * tokens
    used = 0
    for r, (n, c) in enumerate(zip(query_lens, context_lens)):
        n, c = max(n, 0), max(c, 0)
        have, need = -(-c // block), -(-(c + n) // block)
        for index in range(have, min(need, width)):
            at = used + index - have
            tables[r][index] = free[at] if at < len(free) else -1
        for t in range(n):
            row, position = offsets[-1] + t, c + t
            if row >= tokens:
                break
            positions[row] = position
            index = position // block
            if index < width and tables[r][index] >= 0:
                slots[row] = tables[r][index] * block + position % block
        used += need - have
        offsets.append(offsets[-1] + n)
        seq.append(c + n)
    return offsets, seq, positions, slots, tables, used


def attention(q, cache, tables, seq_lens, offsets, block, scale=None, tree_mask=None):
    """(out, spread) float64 [rows, heads, dim] and a bound [rows, heads, dim] on how far a kernel
    with bf16 weights may be off before its output is rounded (see ``tolerance``)."""
    rows, heads, dim = q.shape
    kv_heads = cache.shape[1]
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(rows, heads, dim, dtype=torch.float64)
    spread = torch.zeros(rows, heads, dim, dtype=torch.float64)
    q = q.cpu().double()
    cache = cache.cpu()
    for r, seq in enumerate(seq_lens):
        first, n = offsets[r], offsets[r + 1] - offsets[r]
        keys = min(seq, len(tables[r]) * block)
        slots = [tables[r][p // block] * block + p % block if 0 <= tables[r][p // block] < cache.shape[0] else -1
                 for p in range(keys)]
        k, v, ks, vs = load(cache, slots, block)
        there = torch.tensor([s >= 0 for s in slots], dtype=torch.bool)
        cached = seq - n
        for t in range(n):
            row = first + t
            if row >= rows:
                break
            sees = there.clone()
            if tree_mask is None:
                sees[max(cached + t + 1, 0):] = False
            else:
                for j in range(max(keys - cached, 0)):
                    if cached + j >= 0 and not (j < 64 and (tree_mask[row] >> j) & 1):
                        sees[cached + j] = False
            if not bool(sees.any()):
                continue
            for h in range(heads):
                g = h // group
                s = scale * (k[sees, g] @ q[row, h])
                p = torch.softmax(s, 0)
                values = v[sees, g]
                out[row, h] = p @ values
                spread[row, h] = _spread(p, s, values, k[sees, g], ks[sees, g], vs[sees, g], q[row, h], scale)
    return out, spread


def _spread(p, s, values, k, k_scale, v_scale, q, scale):
    """Error bound of one row before the output's rounding, u = 2^-8 being bf16's half step:
    * each weight p s_v rounded to bf16: u sum p |v|;
    * keys and values as bf16(s (c - z)), as a kernel for long queries takes them: another
      u sum p |v|, and scores off by u scale sum_x |q_x k_x|, which changes p by that much
      relatively, on both sides of the quotient -- as independent roundings, 4 standard deviations
      of a uniform error in [-u, u]: 4 u / sqrt(3) scale sqrt(sum_x (q_x k_x)^2);
    * fp32: a score's sum has products of up to (128 + 15) |q|, rounded at most D / 16 + 2 times by
      2^-23; sums of weights times (128 + 15) s_v, rounded once for each 32 keys of a wave and a
      few times in joining: (n / 128 + 24) 2^-23 143 sum p s_v."""
    u = 2.0 ** -8
    absolute = p @ values.abs()
    rounding = 4 * u / 3 ** 0.5 * scale * (k * q).square().sum(-1).sqrt()
    exact = scale * k_scale.abs() * 143 * q.abs().sum() * (q.numel() / 16 + 2) * 2.0 ** -23
    moved = 2 * float((rounding + exact + 2.0 ** -20).max())
    sums = (len(p) / 128 + 24) * 2.0 ** -23 * 143 * float(p @ v_scale.abs())
    return (2 * u + moved) * absolute + sums


def tolerance(out, spread):
    """How far a bf16 output may be from `out`: the bound above, and its own rounding."""
    return spread + 2.0 ** -8 * (out.abs() + spread) + 1e-30
