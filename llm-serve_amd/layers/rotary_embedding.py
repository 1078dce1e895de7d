"""Position rotation of queries and keys with their per-head norms, in place of the reference's
``RotaryEmbedding`` (llmserve/layers/rotary_embedding.py:6-59) and the ``q_norm`` / ``k_norm`` in
front of it (llmserve/models/qwen3.py:87-94).

* ``rotary_table``     cosines and sines of every position, made once at load
* ``qk_norm_rope``     both heads' norms and the rotation in one launch, from the QKV projection's output
* ``RotaryEmbedding``  the reference's layer: ``forward(positions, query, key)``

``append_kv_int4`` (layers/attention.py) does the same on the way into the 4-bit cache.  Everything
runs in the HIP library and raises without it or without a GPU; every call may be captured in a HIP
graph.
"""
from __future__ import annotations

import torch
from torch import nn

from .._lib import lib

__all__ = ("RotaryEmbedding", "qk_norm_rope", "rotary_table")

_BF16, _I32, _F32 = torch.bfloat16, torch.int32, torch.float32
HEAD_DIMS = (64, 128)
MAX_HEADS = 0xFFFF


def rotary_table(rotary_dim: int, max_position: int, base: float = 10000.0,
                 device: torch.device | str = "cuda") -> torch.Tensor:
    """fp32 [max_position, rotary_dim]: a position's rotary_dim / 2 cosines, then its sines, of the angles
    position * base^(-2 i / rotary_dim), which are formed in 64 bits (far positions' angles have no
    digits to spare in 32).  Tables of scaled frequencies have the same form."""
    if rotary_dim < 16 or rotary_dim % 16:
        raise ValueError(f"rotary_dim must be a multiple of 16 (got {rotary_dim})")
    if max_position < 1:
        raise ValueError(f"max_position must be at least 1 (got {max_position})")
    if not 0.0 < base < float("inf"):
        raise ValueError(f"the rotary base must be positive and finite (got {base})")
    half = rotary_dim // 2
    frequency = float(base) ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    angle = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * frequency
    return torch.cat((angle.cos(), angle.sin()), -1).float()


def _head_rows(name: str, t: torch.Tensor, heads: int | None, head_dim: int, index: int) -> torch.Tensor:
    """t as the kernels read it: [T, heads, head_dim], 16-byte aligned rows at any strides."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != head_dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, {head_dim}]")
    if t.dtype is not _BF16 or t.get_device() != index:
        raise ValueError(f"{name} must be a bfloat16 tensor on the queries' GPU")
    s0, s1, s2 = t.stride()
    if s2 != 1 or (s0 | s1) % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def rope_ready(q, k, positions, table, q_weight, k_weight, eps) -> bool:
    """Whether the kernel can read all operands as they are: one expression accepts what ``rope_operands``
    accepts, but for what it has to copy; a call with few rows is over in less time than its checks."""
    shape, kshape, tshape, index = q.shape, k.shape, table.shape, q.get_device()
    if not (index >= 0 and len(shape) == 3 and len(kshape) == 3 and len(tshape) == 2):
        return False
    tokens, heads, head_dim = shape
    count, rotary = tshape
    q0, q1, q2 = q.stride()
    k0, k1, k2 = k.stride()
    return (head_dim in HEAD_DIMS and kshape[2] == head_dim and kshape[0] == tokens
            and 0 < heads <= MAX_HEADS and 0 < kshape[1] <= MAX_HEADS
            and q.dtype is _BF16 and k.dtype is _BF16 and k.get_device() == index
            and q2 == 1 and k2 == 1 and (q0 | q1 | k0 | k1) % 8 == 0
            and (q.data_ptr() | k.data_ptr() | table.data_ptr()) % 16 == 0
            and positions.dtype is _I32 and positions.get_device() == index and positions.shape == (tokens,)
            and positions.is_contiguous()
            and table.dtype is _F32 and table.get_device() == index and table.is_contiguous()
            and 0 < count < 1 << 31 and 0 < rotary <= head_dim and rotary % 16 == 0
            and (q_weight is None or (q_weight.dtype is _BF16 and q_weight.get_device() == index
                                      and q_weight.shape == (head_dim,) and q_weight.is_contiguous()
                                      and q_weight.data_ptr() % 16 == 0))
            and (k_weight is None or (k_weight.dtype is _BF16 and k_weight.get_device() == index
                                      and k_weight.shape == (head_dim,) and k_weight.is_contiguous()
                                      and k_weight.data_ptr() % 16 == 0))
            and 0.0 <= eps <= 3.4e38)


def rope_operands(q, k, positions, table, q_weight, k_weight, eps):
    """The argument errors of the rotating calls; their operands as the kernel reads them."""
    index = q.get_device()
    if index < 0:
        raise ValueError("queries must be on a GPU (HIP) device")
    head_dim = q.shape[2] if q.ndim == 3 else 0
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"queries must be [tokens, heads, head_dim] with head_dim in {HEAD_DIMS}")
    q = _head_rows("queries", q, None, head_dim, index)
    k = _head_rows("keys", k, None, head_dim, index)
    tokens = q.shape[0]
    if k.shape[0] != tokens:
        raise ValueError("queries and keys must have one row a token")
    if not (0 < q.shape[1] <= MAX_HEADS and 0 < k.shape[1] <= MAX_HEADS):
        raise ValueError(f"queries and keys must have 1 to {MAX_HEADS} heads")
    if positions.dtype is not _I32 or positions.get_device() != index or positions.shape != (tokens,):
        raise ValueError("positions must be an int32 [tokens] tensor on the queries' GPU")
    if (table.dtype is not _F32 or table.get_device() != index or table.ndim != 2 or table.shape[0] < 1
            or table.shape[1] < 16 or table.shape[1] % 16 or table.shape[1] > head_dim):
        raise ValueError("the rotary table must be a float32 [positions, rotary_dim] tensor on the queries' GPU, rotary_dim "
                         "a multiple of 16 up to head_dim")
    if table.shape[0] >= 1 << 31:
        raise ValueError("the rotary table must have fewer than 2^31 positions")
    if not table.is_contiguous() or table.data_ptr() % 16:
        table = table.clone(memory_format=torch.contiguous_format)
    for w in (q_weight, k_weight):
        if w is not None and (w.dtype is not _BF16 or w.get_device() != index or w.shape != (head_dim,)):
            raise ValueError("norm weights must be bfloat16 [head_dim] tensors on the queries' GPU")
    if not 0.0 <= eps <= 3.4e38:
        raise ValueError(f"eps must be finite and not negative (got {eps})")
    return q, k, positions.contiguous(), table, _weight(q_weight), _weight(k_weight)


def _weight(w: torch.Tensor | None) -> torch.Tensor | None:
    if w is not None and (not w.is_contiguous() or w.data_ptr() % 16):
        w = w.clone(memory_format=torch.contiguous_format)
    return w


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, *,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                 eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """q [tokens, heads, head_dim] and k [tokens, kv heads, head_dim] (bf16; views of the split QKV output
    are read in place), each row normed by its root mean square (where there is a weight [head_dim])
    and rotated by its token's position (int32 [tokens]), as new contiguous bf16 tensors.

    ``table`` [max positions, rotary_dim] is ``rotary_table``'s; channel i turns with channel
    i + rotary_dim / 2, and channels from rotary_dim on keep their place.  A row whose position the table
    does not have becomes NaN.  All steps are fp32, each rounded by itself (the sum of squares is fp64),
    and the result is rounded to bf16 once, where the reference rounds after each norm's step too.  A row with
    a weight whose mean square passes fp32's range (sizes from 2^64 on) becomes zero."""
    if not rope_ready(q, k, positions, table, q_weight, k_weight, eps):
        q, k, positions, table, q_weight, k_weight = rope_operands(q, k, positions, table, q_weight, k_weight, eps)
    shape, kshape, index = q.shape, k.shape, q.get_device()
    head_dim = shape[2]
    q_out = torch.empty_strided(shape, (shape[1] * head_dim, head_dim, 1), dtype=_BF16, device=index)
    k_out = torch.empty_strided(kshape, (kshape[1] * head_dim, head_dim, 1), dtype=_BF16, device=index)
    if shape[0] > 0:
        lib().qk_norm_rope(q, k, positions, table, q_weight, k_weight, eps, q_out, k_out)
    return q_out, k_out


class RotaryEmbedding(nn.Module):
    """The reference's layer (rotary_embedding.py:37-48): ``forward(positions, query, key)`` rotates both,
    [tokens, heads, head_size], with the norms' weights where they are given.  ``cos_sin_cache`` is the
    table."""

    def __init__(self, head_size: int, rotary_dim: int, max_position_embeddings: int, base: float = 10000.0,
                 device: torch.device | str = "cuda"):
        super().__init__()
        if head_size not in HEAD_DIMS:
            raise ValueError(f"head_size must be one of {HEAD_DIMS} (got {head_size})")
        if rotary_dim > head_size:
            raise ValueError(f"rotary_dim ({rotary_dim}) must not exceed head_size ({head_size})")
        self.head_size = head_size
        self.register_buffer("cos_sin_cache", rotary_table(rotary_dim, max_position_embeddings, base, device),
                             persistent=False)

    def forward(self, positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, *,
                q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
        return qk_norm_rope(query, key, positions, self.cos_sin_cache, q_weight=q_weight, k_weight=k_weight, eps=eps)
