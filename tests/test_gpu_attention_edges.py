"""Attention over the 4-bit cache at the edges of what its lists, layouts and values may be, against
its definition in 64 bits (oracle/kv4_oracle.py)."""
import pytest
import torch

from test_gpu_attention import Batch, attn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hint", [1, 100])
@pytest.mark.parametrize("new", [[3], [90], [2, 80, 1]])
def test_rows_before_the_first_request(gpu_lib, hint, new):
    """Offsets that begin above 0: the rows before them belong to no request, as those behind the
    last one do -- zero in a new output, whatever its memory held, and left alone in `out`."""
    b = Batch(new, [n + 40 for n in new], 8, 2, 128, 16, seed=80 + sum(new), pad=9)
    b.offsets = [o + 5 for o in b.offsets]
    rows = b.q.shape[0]
    print("first rows", hint, new, flush=True)
    dirt = torch.full((rows, 8, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    del dirt  # the output's memory
    out = b.run(max_query_len=hint)
    b.check(out)
    assert not bool(out[:5].any()) and not bool(out[b.offsets[-1]:].any())
    mine = torch.full_like(out, 7.0)
    b.run(max_query_len=hint, out=mine)
    assert bool((mine[:5] == 7.0).all()) and bool((mine[b.offsets[-1]:] == 7.0).all())
    assert torch.equal(mine[5:b.offsets[-1]], out[5:b.offsets[-1]])
