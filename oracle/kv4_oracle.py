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
    """(out, spread) float64 [rows, heads, dim] and a bound [rows, heads, dim] on how far any kernel
    with bf16 operands may be off before its output is rounded (see ``tolerance``).  What the present
    kernels round is less: ``attention_errors`` has a bound for each."""
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
    * keys and values as bf16(s (c - z)), as a kernel might take them (none does now): another
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


def attention_errors(q, cache, tables, seq_lens, offsets, block, kernel, scale=None, values=None):
    """(out, sigma, worst) float64 [rows, heads, dim] of causal attention: the output, and the error
    of one of the two kernels before its output is rounded, as a standard deviation of independent
    roundings and as what all of them together cannot pass.  ``values`` (a function of a request, its
    keys' values and its slots) may replace values, for errors planted by a test.

    With P = p / sum p, u the half step of a rounding and r = u / sqrt(3) the standard deviation of one
    that is uniform in [-u, u]:

    * "split" (requests of up to 64 rows a kv head, all where the caller's longest query is that
      short): codes and zero points are exact and a weight times its value's scale becomes two bf16
      values, the second one the first one's error (u = 2^-16): sigma^2 = r^2 sum P^2 v^2, worst
      u sum P |v|.  A score's sum has products of up
      to (128 + 15) |q|, rounded at most D / 16 + 2 times by 2^-23; sums of weights times
      (128 + 15) s_v are rounded once for each 32 keys of a wave and a few times in joining.
    * "prompt" (longer requests): keys, values and weights are fp16 (u = 2^-11; queries fit it).  Values
      and weights: sigma^2 = 2 r^2 sum P^2 v^2, worst 2 u sum P |v|.  A score is off by
      r scale sqrt(sum_x (q_x k_x)^2), at worst u scale sum_x |q_x k_x|, which changes P by as much
      relatively, on both sides of the quotient: sigma^2 += sum P^2 (score's)^2 (v - out)^2.  A score is rounded
      once for each 16 channels, sums of weights once for each 16 keys, by 2^-23 of their absolute sums;
      weights 2^-21 below the row's largest lose bits, 2^-32 of it each.
    * Both: the exponent's argument and the exponential, 2^-20 of a weight."""
    rows, heads, dim = q.shape
    kv_heads = cache.shape[1]
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    u = 2.0 ** -16 if kernel == "split" else 2.0 ** -11
    r2 = u * u / 3
    out, sigma, worst = (torch.zeros(rows, heads, dim, dtype=torch.float64) for _ in range(3))
    q, cache = q.cpu().double(), cache.cpu()
    for r, seq in enumerate(seq_lens):
        first, n = offsets[r], offsets[r + 1] - offsets[r]
        slots = [tables[r][p // block] * block + p % block for p in range(seq)]
        k, v, ks, vs = load(cache, slots, block)
        if values is not None:
            v = values(r, v, slots)
        sees = torch.arange(seq)[None] < (seq - n + torch.arange(n) + 1)[:, None]
        sees = sees.repeat_interleave(group, 0)
        for g in range(kv_heads):
            own = q[first:first + n, g * group:(g + 1) * group].reshape(n * group, dim)
            s = (scale * own @ k[:, g].t()).masked_fill(~sees, -torch.inf)
            p = torch.softmax(s, 1)
            x, magnitude = v[:, g], p @ v[:, g].abs()
            o = p @ x
            if kernel == "split":
                variance, most = r2 * (p * p) @ (x * x), u * magnitude
                score = scale * ks[:, g].abs() * 143 * own.abs().sum(1, True) * (dim / 16 + 2) * 2.0 ** -23
                sums = (seq / 128 + 24) * 2.0 ** -23 * 143 * (p @ vs[:, g].abs())[:, None]
            else:
                of_score = r2 * scale * scale * (own * own) @ (k[:, g] * k[:, g]).t()
                w = p * p * of_score
                variance = 2 * r2 * (p * p) @ (x * x)
                variance = variance + w @ (x * x) - 2 * o * (w @ x) + o * o * w.sum(1, True)
                score = scale * own.abs() @ k[:, g].abs().t()
                most = 2 * u * magnitude + 2 * u * torch.where(sees, score, 0).amax(1, True) * magnitude
                score = score * (dim / 16 + 4) * 2.0 ** -23
                sums = (seq / 16 + 24) * 2.0 ** -23 * magnitude
                seen = torch.where(sees, vs[:, g].abs(), 0).amax(1)
                sums = sums + seq * 2.0 ** -32 * 15 * (p.amax(1) * seen)[:, None]
            exact = 2 * (torch.where(sees, score, 0).amax(1, True) + 2.0 ** -20) * magnitude + sums

            def put(to, what):
                to[first:first + n, g * group:(g + 1) * group] = what.reshape(n, group, dim)

            put(out, o)
            put(sigma, variance.clamp(min=0).sqrt())
            put(worst, exact)
            worst[first:first + n, g * group:(g + 1) * group] += torch.minimum(
                most, 7 * variance.clamp(min=0).sqrt()).reshape(n, group, dim)
    return out, sigma, worst


def check_errors(got, out, sigma, worst):
    """What is wrong with a bf16 output, as a text, or None.

    * Every element lies within its bound: ``worst`` (of which roundings count 7 standard deviations, or
      all of them at once where that is less) and its own rounding, 2^-8.
    * The squared error of all elements together is what a kernel's must be.  Rounding the exact output
      once gives E0 = sum (bf16(out) - out)^2, and a kernel's own error moves values across rounding
      borders without changing that sum but by chance: N elements' squares, each in [0, 1] of a
      half step's with a variance of 4/45 around 1/3, vary by sqrt(4/45) / (1/3) = 0.9 of 1 / sqrt(N), and unequal
      elements by some more; 8 / sqrt(N) is allowed.  The kernel's own error adds sum sigma^2, of
      which one (row, head) pair's part may be a single rounding's, so that M pairs' sum of squares varies by
      sqrt(2 / M): 1 + 8 / sqrt(M) times it is allowed."""
    got = got.cpu().double()
    off = (got - out).abs()
    limit = worst + 2.0 ** -8 * (out.abs() + worst) + 1e-30
    bad = ~(off <= limit)
    if bool(bad.any()):
        return f"{int(bad.sum())} elements, up to {float((off / limit).nan_to_num(9e9).max()):.2f} of their bound"
    live = out.abs().amax((1, 2)) > 0
    n, m = int(live.sum()) * out.shape[1] * out.shape[2], int(live.sum()) * out.shape[1]
    if n == 0:
        return None
    # heads of one size: an error in a row of small values counts as much as in one of large ones
    size = out[live].square().mean((2,), True).sqrt()
    whole = float((off[live] / size).square().sum())
    once = float(((bf16_rne(out[live]) - out[live]) / size).square().sum())
    own = float((sigma[live] / size).square().sum())
    allowed = once * (1 + 8 / n ** 0.5) + own * (1 + 8 / m ** 0.5) + n * 2.0 ** -40
    return None if whole <= allowed else f"squared error {whole:.4g}, allowed {allowed:.4g} (rounding once: {once:.4g})"
