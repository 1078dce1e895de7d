"""Attention over a key/value cache held in 4 bits, in place of the reference's bf16 cache and
flash-attn calls (llmserve/layers/attention.py:21-133).

* ``new_kv_cache_int4``  a layer's cache, ``[blocks, kv heads, block_size * (head_dim + 8)]`` bytes
* ``kv_step``            one step's positions, slots, row offsets and block tables from the
                         request lengths, on the GPU (the host loops of the reference's
                         ``prepare_prefill`` / ``prepare_decode``, model_runner.py:279-333)
* ``store_kv_int4``      new rows quantized into the cache (``store_kvcache``, attention.py:21-57)
* ``load_kv_int4``       rows read back as the values they stand for
* ``attention_int4``     causal attention of packed rows over their sequences' pages: decode,
                         draft verification, chunks and prompts in one call (attention.py:118-132)
* ``Attention``          the layer between QKV and O: ``store_kv_int4``, then ``attention_int4``

A row of the cache (one token of one kv head) is a code c in 0..15 a channel, one bf16 scale s and
one zero point z, as a group of an AWQ weight is; a channel stands for s * (c - z).  With 128
channels that is 68 bytes for a row of 256.

Everything runs in the HIP library and raises without it or without a GPU; nothing synchronises
the host (but for the first ``attention_int4`` on a device, which sets up its counters, and one in
4096 captured calls), and every call may be captured in a HIP graph.  ``attention_int4`` takes its workspace and counters from
``SCRATCH``, one pair a stream and one a captured call, so calls on several streams, and several
graphs, share neither.
"""
from __future__ import annotations

import functools
import threading
from dataclasses import dataclass

import torch
from torch import nn

from .._lib import _current_device, _current_stream, lib

__all__ = ("Attention", "KVStep", "attention_int4", "kv_step", "load_kv_int4", "new_kv_cache_int4", "store_kv_int4")

_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None)  # None without GPU support
_BF16, _I32, _U8 = torch.bfloat16, torch.int32, torch.uint8

HEAD_DIMS = (64, 128)
BLOCK_SIZES = (16, 32, 64, 128, 256)
MAX_STEP_REQUESTS = 4096
MAX_STEP_TOKENS = 1 << 18
MAX_SCALE = 2.3e38  # times log2(e), the kernels' multiplier, it is finite in 32 bits


def _require_int32(device: torch.device, **tensors: torch.Tensor) -> None:
    for name, t in tensors.items():
        if t.dtype != torch.int32 or t.device != device:
            raise ValueError(f"KV {name} must be an int32 tensor on the cache's GPU")


def _check_block_size(block_size: int) -> None:
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"KV block_size must be one of {BLOCK_SIZES} (got {block_size})")


def new_kv_cache_int4(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                      device: torch.device | str = "cuda") -> torch.Tensor:
    """A layer's empty cache.  Its rows hold nothing to read until they are stored."""
    _check_block_size(block_size)
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"KV head_dim must be one of {HEAD_DIMS} (got {head_dim})")
    if num_blocks < 1 or num_kv_heads < 1:
        raise ValueError("a KV cache needs at least one block and one kv head")
    if num_blocks * block_size >= 1 << 31:
        raise ValueError("a KV cache holds fewer than 2^31 tokens")
    return torch.zeros(num_blocks, num_kv_heads, block_size * (head_dim + 8), dtype=torch.uint8, device=device)


def _cache_head_dim(cache: torch.Tensor, block_size: int) -> int:
    shape = cache.shape
    if (block_size in BLOCK_SIZES and cache.dtype is _U8 and len(shape) == 3 and cache.is_contiguous()
            and cache.get_device() >= 0 and shape[0] > 0 and shape[1] > 0 and shape[0] * block_size < 1 << 31
            and cache.data_ptr() % 16 == 0):
        head_dim = shape[2] // block_size - 8
        if head_dim in HEAD_DIMS and shape[2] == block_size * (head_dim + 8):
            return head_dim
    _check_block_size(block_size)
    if cache.dtype != torch.uint8 or cache.ndim != 3 or not cache.is_contiguous():
        raise ValueError("a KV cache is a contiguous uint8 tensor [blocks, kv heads, page bytes]")
    if cache.device.type != "cuda":
        raise ValueError("a KV cache must be on a GPU (HIP) device")
    if cache.shape[0] < 1 or cache.shape[1] < 1:
        raise ValueError("a KV cache needs at least one block and one kv head")
    if cache.shape[0] * block_size >= 1 << 31:
        raise ValueError("a KV cache holds fewer than 2^31 tokens")
    if cache.data_ptr() % 16:
        raise ValueError("a KV cache must be 16-byte aligned")
    raise ValueError(f"KV page size must be block_size * (head_dim + 8) with head_dim in {HEAD_DIMS}")


def _rows(name: str, t: torch.Tensor, heads: int | None, head_dim: int, cache: torch.Tensor) -> torch.Tensor:
    """t as the kernels read it: [T, heads, head_dim], 16-byte aligned rows at any strides."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != head_dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"KV {name} must be [tokens, {'heads' if heads is None else heads}, {head_dim}]")
    if t.dtype is not _BF16 or t.get_device() != cache.get_device():
        raise ValueError(f"KV {name} must be a bfloat16 tensor on the cache's GPU")
    s0, s1, s2 = t.stride()
    if s2 != 1 or (s0 | s1) % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


@dataclass(frozen=True)
class KVStep:
    """One step's bookkeeping, shared by all layers: int32 tensors on the GPU."""
    cu_query_lens: torch.Tensor  # [requests + 1]: the requests' offsets among the packed rows
    seq_lens: torch.Tensor       # [requests]: tokens in the cache once the step's rows are stored
    positions: torch.Tensor      # [rows]: each row's position in its sequence (0 behind the last request)
    slots: torch.Tensor          # [rows]: each row's cache slot (-1: none)
    block_tables: torch.Tensor   # [requests, width]: the argument, with the new blocks entered
    blocks_used: torch.Tensor    # [1]: how many of the free blocks the step needs


def kv_step(query_lens: torch.Tensor, context_lens: torch.Tensor, block_tables: torch.Tensor,
            free_blocks: torch.Tensor, *, block_size: int, num_tokens: int) -> KVStep:
    """Positions, cache slots, offsets and block tables of a step whose request r brings
    ``query_lens[r]`` new tokens behind ``context_lens[r]`` cached ones (int32 on the GPU; a padded
    request has zero of both).  ``block_tables`` [requests, width] holds the cached tokens' blocks
    and gets, in place, the blocks that the new tokens open: those of ``free_blocks``, in order of
    request and position.  ``num_tokens`` is the number of packed rows, at least the sum of
    ``query_lens``; rows behind the last request get position 0 and slot -1, which
    ``store_kv_int4`` skips.  (With fewer, the last tokens have no row to be stored from; offsets,
    lengths and block tables count them all the same.)

    The host takes the first ``blocks_used`` entries off its free list (it can count them from the
    lengths without reading the tensor).  A token for which the list or the table's width is too
    short gets slot -1, and -1 as its table entry; ``blocks_used`` then exceeds the list."""
    index, requests = query_lens.get_device(), query_lens.shape[0] if query_lens.ndim == 1 else 0
    shape = block_tables.shape
    if not (index >= 0 and 0 < requests <= MAX_STEP_REQUESTS and 0 <= num_tokens <= MAX_STEP_TOKENS
            and block_size in BLOCK_SIZES
            and query_lens.dtype is _I32 and query_lens.is_contiguous()
            and context_lens.dtype is _I32 and context_lens.get_device() == index
            and context_lens.is_contiguous() and context_lens.shape == (requests,)
            and free_blocks.dtype is _I32 and free_blocks.get_device() == index
            and free_blocks.is_contiguous() and free_blocks.ndim == 1
            and block_tables.dtype is _I32 and block_tables.get_device() == index
            and block_tables.is_contiguous() and len(shape) == 2 and shape[0] == requests and shape[1] > 0):
        query_lens, context_lens, block_tables, free_blocks = _check_step(query_lens, context_lens, block_tables,
                                                                          free_blocks, block_size, num_tokens)
    # one allocation: offsets, lengths, blocks used, positions, slots
    size = 2 * requests + 2 + 2 * num_tokens
    out = torch.empty_strided((size,), (1,), dtype=_I32, device=index)
    cu, seq, used, positions, slots = out.split_with_sizes((requests + 1, requests, 1, num_tokens, num_tokens))
    lib().kv_step(query_lens, context_lens, block_tables, free_blocks, cu, seq, positions, slots, used, block_size)
    return KVStep(cu, seq, positions, slots, block_tables, used)


def _check_step(query_lens, context_lens, block_tables, free_blocks, block_size, num_tokens):
    """The argument errors of ``kv_step``; its arguments as the kernel reads them."""
    _check_block_size(block_size)
    if query_lens.device.type != "cuda":
        raise ValueError("KV step lengths must be GPU (HIP) tensors")
    device = query_lens.device
    _require_int32(device, query_lens=query_lens, context_lens=context_lens, block_tables=block_tables,
                   free_blocks=free_blocks)
    requests = query_lens.shape[0] if query_lens.ndim == 1 else -1
    if requests < 0 or context_lens.shape != (requests,) or free_blocks.ndim != 1:
        raise ValueError("KV query_lens, context_lens [requests] and free_blocks must be one-dimensional")
    if block_tables.ndim != 2 or block_tables.shape[0] != requests or block_tables.shape[1] < 1:
        raise ValueError("KV block_tables must be [requests, width]")
    if requests < 1 or requests > MAX_STEP_REQUESTS:
        raise ValueError(f"a KV step takes 1 to {MAX_STEP_REQUESTS} requests (got {requests})")
    if num_tokens < 0 or num_tokens > MAX_STEP_TOKENS:
        raise ValueError(f"a KV step takes 0 to {MAX_STEP_TOKENS} rows (got {num_tokens})")
    width = block_tables.shape[1]  # a dimension of one entry may have any stride
    if (width > 1 and block_tables.stride(1) != 1) or (requests > 1 and block_tables.stride(0) < width):
        raise ValueError("KV block_tables rows must be contiguous and must not overlap")
    return query_lens.contiguous(), context_lens.contiguous(), block_tables, free_blocks.contiguous()


def store_kv_int4(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor, *,
                  block_size: int) -> None:
    """Quantizes the rows k, v [tokens, kv heads, head_dim] (bf16; views of the split QKV output
    are read in place) into the cache's ``slots`` [tokens] (int32).  Slots outside the cache (-1)
    are skipped; the others must differ from each other.

    Per row: s = bf16((max(x, 0) - min(x, 0)) / 15), z = round(-min(x, 0) / s),
    c = clamp(round(x / s) + z, 0, 15).  A row that holds a NaN or an infinity is stored as NaN."""
    head_dim = _cache_head_dim(cache, block_size)
    k = _rows("keys", k, cache.shape[1], head_dim, cache)
    v = _rows("values", v, cache.shape[1], head_dim, cache)
    if slots.dtype is not _I32 or slots.get_device() != cache.get_device():
        _require_int32(cache.device, slots=slots)
    if k.shape != v.shape or slots.shape != k.shape[:1]:
        raise ValueError("KV keys, values and slots must have one entry a token")
    if k.shape[0] > 0:
        lib().kv_store(k, v, cache, slots.contiguous(), head_dim, block_size)


def load_kv_int4(cache: torch.Tensor, slots: torch.Tensor, *, block_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows at ``slots`` [tokens] (int32): (k, v) [tokens, kv heads, head_dim], the values
    s * (c - z) rounded to bf16; zeros for a slot outside the cache."""
    head_dim = _cache_head_dim(cache, block_size)
    index, kv_heads = cache.get_device(), cache.shape[1]
    if slots.dtype is not _I32 or slots.get_device() != index:
        _require_int32(cache.device, slots=slots)
    if slots.ndim != 1:
        raise ValueError("KV slots must be one-dimensional")
    shape, stride = (slots.shape[0], kv_heads, head_dim), (kv_heads * head_dim, head_dim, 1)
    k = torch.empty_strided(shape, stride, dtype=_BF16, device=index)
    v = torch.empty_strided(shape, stride, dtype=_BF16, device=index)
    if slots.shape[0] > 0:
        lib().kv_load(cache, slots.contiguous(), k, v, head_dim, block_size)
    return k, v


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(*sizes: int) -> int:
    """The library's answer for these sizes, which depends on nothing else."""
    return lib().kv_attention_workspace(*sizes)


class _ScratchPool:
    """Workspaces and arrival counters of ``attention_int4``; a call's counters (1024 int32) are zero
    before and after it.

    Eager calls of one stream run in order and share one pair, whose workspace is as large as their
    largest (up to some 80 MB where prompts are among them) and stays with the stream.  A captured
    call takes its workspace from the graph's pool and a set of counters (4 KiB) of its own, for
    good: its graph may be replayed beside anything else, and nothing tells when it is destroyed.
    Counters come from a zeroed array a device (16 MiB: 4096 sets), made by the device's first eager
    call, which waits for the zeros, and again by the next eager call once captured ones have used
    it up.  A call captured while there is none takes a new zeroed tensor, which its graph clears on
    every replay."""

    SETS = 4096
    SIZE = 1024

    def __init__(self):
        self._lock = threading.Lock()
        self._free: dict[int, list[torch.Tensor]] = {}
        self._streams: dict[tuple[int, int], tuple[torch.Tensor, torch.Tensor]] = {}
        self._captured: list[torch.Tensor] = []

    def get(self, index: int, nbytes: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(workspace of at least nbytes, counters) for a call on GPU `index`'s current stream."""
        if _current_device() != index:
            with torch.cuda.device(index):
                return self.get(index, nbytes)
        if _capturing():
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=index)
            with self._lock:
                free = self._free.get(index)
                if free:
                    self._captured.append(free.pop())
                    return workspace, self._captured[-1]
            return workspace, torch.zeros(self.SIZE, dtype=_I32, device=index)
        key = (index, _current_stream(index))
        pair = self._streams.get(key)
        if pair is not None and pair[0].numel() >= nbytes and self._free.get(index):
            return pair
        with self._lock:
            if not self._free.get(index):
                array = torch.zeros(self.SETS, self.SIZE, dtype=_I32, device=index)
                torch.cuda.current_stream(index).synchronize()
                self._free[index] = list(array.unbind())
            pair = self._streams.get(key)  # another thread may have made or grown it since
            if pair is None or pair[0].numel() < nbytes:
                counters = self._free[index].pop() if pair is None else pair[1]
                pair = self._streams[key] = (torch.empty(nbytes, dtype=torch.uint8, device=index), counters)
            return pair


SCRATCH = _ScratchPool()


def attention_int4(q: torch.Tensor, cache: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                   cu_query_lens: torch.Tensor, *, block_size: int, scale: float | None = None,
                   max_query_len: int | None = None, tree_mask: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the packed rows q [rows, heads, head_dim] (bf16; a view of the split QKV
    output is read in place) over their sequences' cached keys and values, the rows' own included:
    request r's rows ``cu_query_lens[r]`` .. ``cu_query_lens[r + 1]`` are the last tokens of its
    ``seq_lens[r]``, on the pages ``block_tables[r]`` names.  Returns bf16 [rows, heads, head_dim].

    Offsets that decrease name no rows at all.  ``scale`` defaults to 1 / sqrt(head_dim).
    ``max_query_len``, the longest query of the batch if the caller knows it (1 for a decode step),
    picks kernels; results are right whatever it is, if not the same bits.
    ``tree_mask`` (int64 [rows]) replaces causality among a request's new rows: row t sees the
    cached tokens and those new ones j < 64 whose bit j is set.  A row that sees nothing is zero.
    Without ``out`` (contiguous, of q's shape), rows of no request (before the first one's, behind the
    last one's) are zero; in ``out`` they are left as they were.  ``out`` may be q itself, and overlaps no other operand."""
    # One expression accepts what all the checks accept; only what it does not goes through them.
    shape, tshape, index = q.shape, block_tables.shape, cache.get_device()
    head_dim = shape[2] if len(shape) == 3 else 0
    if not (index >= 0 and block_size in BLOCK_SIZES and head_dim in HEAD_DIMS
            and cache.dtype is _U8 and cache.is_contiguous() and len(cache.shape) == 3
            and cache.shape[2] == block_size * (head_dim + 8) and cache.shape[0] * block_size < 1 << 31
            and shape[1] > 0 and cache.shape[1] > 0 and shape[1] % cache.shape[1] == 0
            and q.dtype is _BF16 and q.get_device() == index
            and q.stride(2) == 1 and q.stride(1) % 8 == 0 and q.stride(0) % 8 == 0
            and (q.data_ptr() | cache.data_ptr()) % 16 == 0
            and len(tshape) == 2 and tshape[0] > 0 and tshape[1] > 0
            and block_tables.dtype is _I32 and block_tables.get_device() == index
            and block_tables.is_contiguous()
            and seq_lens.dtype is _I32 and seq_lens.get_device() == index and seq_lens.is_contiguous()
            and seq_lens.shape == (tshape[0],)
            and cu_query_lens.dtype is _I32 and cu_query_lens.get_device() == index
            and cu_query_lens.is_contiguous() and cu_query_lens.shape == (tshape[0] + 1,)):
        q, block_tables, seq_lens, cu_query_lens = _check_attention(q, cache, block_tables, seq_lens, cu_query_lens,
                                                                    block_size)
        shape, tshape, head_dim = q.shape, block_tables.shape, q.shape[2]
    rows, heads = shape[0], shape[1]
    if scale is None:
        scale = head_dim ** -0.5
    elif not 0.0 < scale < MAX_SCALE:
        raise ValueError(f"attention scale must be positive and below {MAX_SCALE} (got {scale})")
    if max_query_len is None:
        max_query_len = max(rows, 1)
    elif max_query_len < 1:
        raise ValueError(f"max_query_len must be at least 1 (got {max_query_len})")
    if tree_mask is not None:
        if tree_mask.dtype != torch.int64 or tree_mask.get_device() != index or tree_mask.shape != (rows,):
            raise ValueError("tree_mask must be an int64 [rows] tensor on the cache's GPU")
        tree_mask = tree_mask.contiguous()
    zero_tail = out is None
    if out is None:
        out = torch.empty_strided(shape, (heads * head_dim, head_dim, 1), dtype=_BF16, device=index)
    elif (out.shape != shape or out.dtype != torch.bfloat16 or out.get_device() != index or not out.is_contiguous()
          or out.data_ptr() % 16):
        raise ValueError("attention out must be a contiguous, 16-byte aligned bfloat16 tensor of q's shape")
    if rows > 0:
        size = _workspace_bytes(rows, tshape[0], heads, cache.shape[1], head_dim, block_size, tshape[1], max_query_len)
        workspace, counters = SCRATCH.get(index, size)
        lib().kv_attention(q, cache, block_tables, seq_lens, cu_query_lens, tree_mask, out, scale, block_size,
                           max_query_len, zero_tail, workspace, counters)
    return out


def _check_attention(q, cache, block_tables, seq_lens, cu_query_lens, block_size):
    """The argument errors of ``attention_int4``; its arguments as the kernels read them."""
    head_dim = _cache_head_dim(cache, block_size)
    q = _rows("queries", q, None, head_dim, cache)
    heads, kv_heads = q.shape[1], cache.shape[1]
    if heads < 1 or heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a multiple of the cache's kv heads ({kv_heads})")
    _require_int32(cache.device, block_tables=block_tables, seq_lens=seq_lens, cu_query_lens=cu_query_lens)
    requests = seq_lens.shape[0] if seq_lens.ndim == 1 else 0
    if requests < 1 or cu_query_lens.shape != (requests + 1,):
        raise ValueError("KV seq_lens must be [requests], at least one, and cu_query_lens [requests + 1]")
    width = block_tables.shape[1] if block_tables.ndim == 2 else 0
    if width < 1 or block_tables.shape[0] != requests:
        raise ValueError("KV block_tables must be [requests, width]")
    if (width > 1 and block_tables.stride(1) != 1) or (requests > 1 and block_tables.stride(0) < width):
        block_tables = block_tables.contiguous()
    return q, block_tables, seq_lens.contiguous(), cu_query_lens.contiguous()


class Attention(nn.Module):
    """The reference's ``Attention`` (attention.py:21-133) over a 4-bit cache: ``forward(q, k, v,
    step)`` stores the step's keys and values and attends.  ``kv_cache`` is the layer's cache
    (``new_kv_cache_int4``), set once by the engine as the reference sets ``k_cache`` and
    ``v_cache``."""

    def __init__(self, num_heads: int, head_dim: int, scale: float, num_kv_heads: int, block_size: int = 256):
        super().__init__()
        _check_block_size(block_size)
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"KV head_dim must be one of {HEAD_DIMS} (got {head_dim})")
        if num_kv_heads < 1 or num_heads < 1 or num_heads % num_kv_heads:
            raise ValueError(f"query heads ({num_heads}) must be a multiple of kv heads ({num_kv_heads})")
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.block_size = block_size
        self.kv_cache: torch.Tensor | None = None

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: KVStep, *,
                max_query_len: int | None = None, tree_mask: torch.Tensor | None = None) -> torch.Tensor:
        """q [rows, heads * head_dim], k and v [rows, kv heads * head_dim], flat or with the heads
        apart; returns [rows, heads * head_dim], O's input."""
        if self.kv_cache is None:
            raise RuntimeError("Attention.kv_cache must be set before the first step")
        rows = q.shape[0]
        q = q.view(rows, self.num_heads, self.head_dim)
        k = k.view(rows, self.num_kv_heads, self.head_dim)
        v = v.view(rows, self.num_kv_heads, self.head_dim)
        store_kv_int4(k, v, self.kv_cache, step.slots, block_size=self.block_size)
        out = attention_int4(q, self.kv_cache, step.block_tables, step.seq_lens, step.cu_query_lens,
                             block_size=self.block_size, scale=self.scale, max_query_len=max_query_len,
                             tree_mask=tree_mask)
        return out.view(rows, self.num_heads * self.head_dim)
