"""What a decoder layer does between its QKV projection and the attention's output, in a serving engine.

Three operators, in the order a layer uses them:

* ``rope``: each head of the queries and keys is normed by its root mean square and rotated by
  its row's position, in one pass.
* ``append``: the same for a step's rows on their way into a cache held in 4 bits; the queries come
  back, the keys and values are quantized into the cache's slots (and are read back here as the
  values that they stand for).
* ``prompt``: causal attention of whole prompts of different lengths, packed one behind the
  other, over their own keys and values in bfloat16, query heads sharing key heads.

The rotation's table holds the cosines and then the sines of a position's angles,
``[positions, rotated channels]``; channel i turns with channel i + rotated / 2.

The cache: ``[blocks, kv heads, block_size * (head_dim + 8)]`` bytes.  A page holds, in 32-bit
words of eight channels (channel c at bit ``SHIFTS[c]``), its tokens' keys ``[token][word]``,
then their values ``[token / 4][word][token % 4]``, then one word a token for the keys and one
for the values: the scale's bfloat16 bits above those of 128 + zero.  Channel c of a row stands
for ``scale * (code - zero)``.

Head counts are those of the layers in the tests and the benchmark (``q8`` is the benchmark's),
and two generic ones.
"""
import importlib
import math

import torch

own = False

# query heads, kv heads, head size
HEADS = {"q8": (32, 8, 128), "q14": (40, 8, 128), "wide": (64, 8, 128), "mha64": (16, 16, 64)}
SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)
EPS = 1e-6


def listed():
    return [
        # a small decode batch: the smallest call there is
        {"name": "rope_decode_t8", "kind": "rope", "model": "q8", "tokens": 8, "pad": 0, "context": 2000, "new": 1,
         "norm": True, "rotated": 128},
        # the engine's largest packed batch: prompts of up to 4096
        {"name": "rope_prefill_t16384", "kind": "rope", "model": "q8", "tokens": 16384, "pad": 0, "context": 0,
         "new": 4096, "norm": True, "rotated": 128},
        # a decode batch of mixed lengths, padded to a captured size
        {"name": "append_decode_t61", "kind": "append", "model": "q8", "tokens": 61, "pad": 3, "context": 8192, "new": 1,
         "norm": True, "rotated": 128, "keys": False, "block": 256},
        # chunks of prompts behind cached tokens, a model without norms that rotates half the channels
        {"name": "append_chunk_t2039", "kind": "append", "model": "q14", "tokens": 2039, "pad": 9, "context": 3500,
         "new": 480, "norm": False, "rotated": 64, "keys": False, "block": 16},
        # the largest packed batch of prompts, whose keys the prompts' own attention reads
        {"name": "append_prefill_t16384", "kind": "append", "model": "q8", "tokens": 16384, "pad": 0, "context": 0,
         "new": 4096, "norm": True, "rotated": 128, "keys": True, "block": 256},
        # a burst of short questions of different lengths
        {"name": "prompts_r24_q120", "kind": "prompt", "model": "q8", "requests": 24, "longest": 120, "pad": 5},
        # one ordinary question
        {"name": "prompt_q511", "kind": "prompt", "model": "q8", "requests": 1, "longest": 511, "pad": 0},
        # a whole prompt of an odd length
        {"name": "prompt_q2039", "kind": "prompt", "model": "q8", "requests": 1, "longest": 2039, "pad": 0},
        # documents of different lengths in one batch
        {"name": "prompts_r9_q2500", "kind": "prompt", "model": "q14", "requests": 9, "longest": 2500, "pad": 0},
        # small heads that share nothing
        {"name": "prompts_mha64_r3_q1500", "kind": "prompt", "model": "mha64", "requests": 3, "longest": 1500, "pad": 0},
        # a few long prompts of different lengths
        {"name": "prompts_r4_q4096", "kind": "prompt", "model": "q8", "requests": 4, "longest": 4096, "pad": 0},
        # one prompt that fills the engine's largest batch
        {"name": "prompt_q16384", "kind": "prompt", "model": "q8", "requests": 1, "longest": 16384, "pad": 0},
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["rope", "append", "prompt", "prompt", "prompt"])
    model = rng.choice(["q8", "q8", "q14", "wide", "mha64"])
    heads, _, dim = HEADS[model]
    pad = rng.choice([0, 0, 1, 7])
    if kind == "prompt":
        requests = rng.choice([1, 1, 2, size(3, 32)])
        # no more pairs of rows and keys than the largest listed prompt has
        most = int((32 * 16384 ** 2 / (heads * requests)) ** 0.5)
        return {"kind": kind, "model": model, "requests": requests, "longest": size(1, min(12000, most)), "pad": pad}
    case = {"kind": kind, "model": model, "tokens": size(1, 16384 * 32 // max(heads, 32)), "pad": pad,
            "context": rng.choice([0, size(1, 32000)]), "new": rng.choice([1, 8, size(2, 4096)]), "norm": rng.random() < 0.7,
            "rotated": rng.choice([dim, dim, dim // 2])}
    if kind == "append":
        case["keys"] = rng.random() < 0.5
        case["block"] = rng.choice([16, 32, 64, 128, 256])
    return case


# ------------------------------------------------------------------- inputs
def generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def lengths(case):
    """A batch's prompt lengths: the longest, and others between a tenth of it and all of it; of each
    eight one has a single token and one, an empty place of the batch, none."""
    gen = torch.Generator().manual_seed(11)
    spread = torch.rand(case["requests"], generator=gen).tolist()
    out = [max(1, int(case["longest"] * (0.1 + 0.9 * u))) for u in spread]
    for i in range(len(out)):
        if i % 8 == 6:
            out[i] = 1
        elif i % 8 == 7:
            out[i] = 0
    out[0] = case["longest"]
    return out


def step_positions(case):
    """The rows' positions: requests of `new` rows each, the last one's cut off, behind contexts
    between a fifth of the case's and all of it; 0 for padding."""
    tokens, new = case["tokens"], case["new"]
    requests = -(-tokens // new)
    spread = torch.rand(requests, generator=torch.Generator().manual_seed(13))
    behind = (case["context"] * (0.2 + 0.8 * spread)).long()
    position = (behind[:, None] + torch.arange(new)).flatten()[:tokens]
    return torch.cat([position, torch.zeros(case["pad"], dtype=torch.long)]).to(torch.int32)


def rope_table(rotated, count):
    """[count, rotated]: cosines, then sines; angles in 64 bits."""
    half = rotated // 2
    frequency = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = torch.arange(count, dtype=torch.float64, device="cuda")[:, None] * frequency
    return torch.cat([angle.cos(), angle.sin()], -1).float()


def projected(gen, rows, heads, dim):
    """A projection's output [rows, heads, dim]: a few channels of every head are larger than the
    rest, as queries' and keys' are."""
    x = torch.randn(rows, heads, dim, generator=gen, device="cuda")
    x[:, :, torch.randperm(dim, generator=gen, device="cuda")[:dim // 16]] *= 4
    return x.to(torch.bfloat16)


def prepare(case, seed):
    gen = generator(seed)
    heads, kv_heads, dim = HEADS[case["model"]]
    if case["kind"] == "prompt":
        new = lengths(case)
        offsets = torch.zeros(len(new) + 1, dtype=torch.int32, device="cuda")
        offsets[1:] = ints(new).cumsum(0)
        rows = sum(new) + case["pad"]
        # queries and keys as the operator before leaves them; the values are a part of the projection's rows
        q = torch.randn(rows, heads, dim, generator=gen, device="cuda").to(torch.bfloat16)
        k = projected(gen, rows, kv_heads, dim)
        qkv = torch.randn(rows, heads + 2 * kv_heads, dim, generator=gen, device="cuda").to(torch.bfloat16)
        return {"case": case, "q": q, "k": k, "v": qkv[:, heads + kv_heads:], "offsets": offsets, "longest": max(new)}
    rows = case["tokens"] + case["pad"]
    position = step_positions(case)
    qkv = projected(gen, rows, heads + 2 * kv_heads, dim)
    state = {"case": case, "q": qkv[:, :heads], "k": qkv[:, heads:heads + kv_heads], "v": qkv[:, heads + kv_heads:],
             "positions": position.cuda(), "table": rope_table(case["rotated"], int(position.max()) + 1), "weights": (None, None)}
    if case["norm"]:
        state["weights"] = tuple((1 + 0.3 * torch.randn(dim, generator=gen, device="cuda")).to(torch.bfloat16)
                                 for _ in range(2))
    if case["kind"] == "append":
        block = case["block"]
        blocks = -(-case["tokens"] // block) + 4
        slots = torch.randperm(blocks, generator=gen, device="cuda")[:, None] * block
        slots = (slots + torch.arange(block, device="cuda")).flatten()[:case["tokens"]].to(torch.int32)
        state["slots"] = torch.cat([slots, ints([-1] * case["pad"])])
        state["cache"] = torch.zeros(blocks, kv_heads, block * (dim + 8), dtype=torch.uint8, device="cuda")
    return state


# ---------------------------------------------------------------------- run
def framework():
    """The framework, imported once as a user's program imports it."""
    if not hasattr(framework, "package"):
        framework.package = importlib.import_module("llm-serve_amd")
    return framework.package


def run(state):
    case = state["case"]
    if own:
        pkg = framework()
        if case["kind"] == "prompt":
            return {"out": pkg.attention_prompt(state["q"], state["k"], state["v"], state["offsets"],
                                                max_query_len=state["longest"])}
        q_weight, k_weight = state["weights"]
        if case["kind"] == "rope":
            q, k = pkg.qk_norm_rope(state["q"], state["k"], state["positions"], state["table"], q_weight=q_weight,
                                    k_weight=k_weight, eps=EPS)
            return {"q": q, "k": k}
        q = pkg.append_kv_int4(state["q"], state["k"], state["v"], state["cache"], state["slots"], state["positions"],
                               state["table"], block_size=case["block"], q_weight=q_weight, k_weight=k_weight, eps=EPS,
                               return_keys=case["keys"])
        outs = dict(zip(("q", "k"), q)) if case["keys"] else {"q": q}
        outs["cached_k"], outs["cached_v"] = pkg.load_kv_int4(state["cache"], state["slots"], block_size=case["block"])
        return outs
    if case["kind"] == "prompt":
        return {"out": plain_prompt(state["q"], state["k"], state["v"], state["offsets"], state["longest"])}
    cos, sin = (t[:, None] for t in state["table"][state["positions"].long()].chunk(2, -1))
    q, k = (turned(x, weight, cos, sin) for x, weight in zip((state["q"], state["k"]), state["weights"]))
    if case["kind"] == "rope":
        return {"q": q, "k": k}
    outs = {"q": q, "k": k} if case["keys"] else {"q": q}
    outs["cached_k"], outs["cached_v"] = plain_store(k, state["v"], state["cache"], state["slots"], case["block"])
    return outs


def turned(x, weight, cos, sin):
    """The rows normed (where there is a weight) and rotated in 32 bits, rounded once.  The sum of
    squares and the root are those of 64 bits: a key that is quantized afterwards may lie next to a
    border between two codes, which another last bit would move it across."""
    x = x.float()
    if weight is not None:
        mean = (x.double().square().sum(-1, keepdim=True) / x.shape[-1]).float()
        x = x * (mean + EPS).double().rsqrt().float() * weight.float()
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(torch.bfloat16)


def quantized(x):
    """(code words, meta word) of rows x [..., dim]: the range takes in zero."""
    x = x.float()
    low = x.amin(-1).clamp(max=0)
    scale = ((x.amax(-1).clamp(min=0) - low) / 15).to(torch.bfloat16)
    s = scale.float()
    zero = torch.where(s > 0, torch.round(-low / s), 0).clamp(0, 15)
    code = torch.where(s[..., None] > 0, torch.round(x / s[..., None]) + zero[..., None], 0).clamp(0, 15)
    shift = torch.tensor(SHIFTS, dtype=torch.int32, device="cuda")
    words = (code.to(torch.int32).unflatten(-1, (-1, 8)) << shift).sum(-1, dtype=torch.int32)
    return words, (scale.view(torch.int16).to(torch.int32) << 16) | 0x4300 | zero.to(torch.int32)


def values(words, meta):
    """scale * (code - zero) in 32 bits for code words [..., w] and meta words [...]."""
    shift = torch.tensor(SHIFTS, dtype=torch.int32, device="cuda")
    code = ((words[..., None] >> shift) & 15).flatten(-2).float()
    scale = (meta & -65536).view(torch.float32)
    zero = (meta << 16).view(torch.float32) - 128
    return scale[..., None] * (code - zero[..., None])


def plain_store(k, v, cache, slots, block):
    rows, kv_heads, dim = k.shape
    words = dim // 8
    pages = cache.view(torch.int32)
    live = slots >= 0
    at = slots[live].long()
    page, token = (at // block)[:, None, None], (at % block)[:, None, None]
    head = torch.arange(kv_heads, device="cuda")[:, None]
    word = torch.arange(words, device="cuda")
    where_k = (page, head, token * words + word)
    where_v = (page, head, (block + token // 4 * 4) * words + word * 4 + token % 4)
    meta_k = (page, head, 2 * block * words + token)
    meta_v = (page, head, 2 * block * words + block + token)
    k_words, k_meta = quantized(k[live])
    v_words, v_meta = quantized(v[live])
    pages[where_k] = k_words
    pages[where_v] = v_words
    pages[meta_k] = k_meta[..., None]
    pages[meta_v] = v_meta[..., None]
    out_k = torch.zeros(rows, kv_heads, dim, dtype=torch.bfloat16, device="cuda")
    out_v = torch.zeros_like(out_k)
    out_k[live] = values(pages[where_k], pages[meta_k].squeeze(-1)).to(torch.bfloat16)
    out_v[live] = values(pages[where_v], pages[meta_v].squeeze(-1)).to(torch.bfloat16)
    return out_k, out_v


def plain_prompt(q, k, v, offsets, longest):
    rows, heads, dim = q.shape
    kv_heads = k.shape[1]
    group = heads // kv_heads
    # the prompts' rows, padded to the longest: [requests, kv heads, rows of one kv head, dim]
    new = offsets[1:] - offsets[:-1]
    nth = torch.arange(longest, device="cuda")
    live = nth < new[:, None]
    row = torch.where(live, offsets[:-1, None] + nth, 0)
    queries = q[row].float().unflatten(2, (kv_heads, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    keys, vals = (torch.where(live[..., None, None], x[row].float(), 0).transpose(1, 2).contiguous() for x in (k, v))
    score = torch.matmul(queries, keys.transpose(2, 3)).mul_(dim ** -0.5)
    # row i of a prompt sees its first i + 1 tokens
    hidden = (nth > nth[:, None]).repeat_interleave(group, 0)
    score = score.masked_fill_(hidden, -math.inf)
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score, vals) / total
    out = out.unflatten(2, (longest, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    packed = torch.zeros(rows + 1, heads, dim, dtype=torch.bfloat16, device="cuda")
    packed[torch.where(live, row, rows)] = out.to(torch.bfloat16)
    return packed[:rows]


# --------------------------------------------------------------------- work
def work(case):
    """Each input read once and each output written once; for prompts two products over the
    pairs of rows and keys that causality leaves."""
    heads, kv_heads, dim = HEADS[case["model"]]
    if case["kind"] == "prompt":
        new = lengths(case)
        pairs = sum(n * (n + 1) // 2 for n in new)
        return {"bytes": (sum(new) * (heads + 2 * kv_heads) + (sum(new) + case["pad"]) * heads) * dim * 2,
                "flops": 4 * pairs * heads * dim}
    rows, tokens = case["tokens"] + case["pad"], case["tokens"]
    positions = step_positions(case)
    # queries read and written, positions, and each position's row of the table once
    size = 4 * rows * heads * dim + 4 * rows + int(positions.unique().numel()) * case["rotated"] * 4
    if case["kind"] == "rope":
        return {"bytes": size + 4 * rows * kv_heads * dim, "flops": 0}
    # keys and values read, packed rows written and read, values written
    size += 4 * tokens * kv_heads * dim + 2 * tokens * 2 * kv_heads * (dim // 2 + 4) + 4 * rows * kv_heads * dim
    return {"bytes": size + case["keys"] * 2 * rows * kv_heads * dim, "flops": 0}


# -------------------------------------------------------------------- exact
def turn64(x, weight, positions, rotated):
    """The definition, channel pairs as complex numbers."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(torch.mean(x * x, -1, keepdim=True) + EPS) * weight.double()
    half = rotated // 2
    exponent = torch.arange(half, dtype=torch.float64, device="cuda") / half
    angle = positions.double()[:, None, None] * torch.pow(torch.tensor(10000.0, dtype=torch.float64, device="cuda"), -exponent)
    pairs = torch.complex(x[..., :half], x[..., half:rotated]) * torch.polar(torch.ones_like(angle), angle)
    return torch.cat([pairs.real, pairs.imag, x[..., rotated:]], -1)


def stored64(x, slots):
    """What rows in bfloat16 stand for once they are in the cache."""
    x = x.to(torch.bfloat16).double()
    high, low = x.amax(-1, True).clamp(min=0), x.amin(-1, True).clamp(max=0)
    s = ((high - low) / 15).to(torch.bfloat16).double()
    zero = torch.round(-low / s)
    x = s * (torch.clamp(torch.round(x / s) + zero, 0, 15) - zero)
    x[slots < 0] = 0
    return x


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] != "prompt":
        outs = {name: turn64(state[name], weight, state["positions"], case["rotated"])
                for name, weight in zip(("q", "k"), state["weights"])}
        if case["kind"] == "append":
            outs["cached_k"], outs["cached_v"] = stored64(outs["k"], state["slots"]), stored64(state["v"], state["slots"])
            if not case["keys"]:
                del outs["k"]
        return outs
    q, k, v = (state[name].double() for name in ("q", "k", "v"))
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(rows, heads, dim, dtype=torch.float64, device="cuda")
    offsets = state["offsets"].tolist()
    for first, end in zip(offsets, offsets[1:]):
        for start in range(first, end, 1024):
            stop = min(end, start + 1024)
            later = torch.arange(first, stop, device="cuda") > torch.arange(start, stop, device="cuda")[:, None]
            for h in range(heads):
                s = q[start:stop, h] @ k[first:stop, h // group].t() / math.sqrt(dim)
                out[start:stop, h] = torch.softmax(s.masked_fill(later, -math.inf), -1) @ v[first:stop, h // group]
    return {"out": out}
