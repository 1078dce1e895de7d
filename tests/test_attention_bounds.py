"""The bounds that the GPU's attention outputs are tested against (oracle/kv4_oracle.py,
attention_errors), on the CPU: they pass the kernels' own roundings, and fail coarser operands and
any 16 keys lost or counted twice."""
import pytest
import torch

from kv4_helpers import emulate, mark_values, marked_channel
from oracle import kv4_oracle as ora


class HostBatch:
    """As the GPU tests' batch, in order of pages and on the CPU."""

    def __init__(self, new, seq, heads, kv_heads, dim, block, seed):
        gen = torch.Generator().manual_seed(seed)
        self.new, self.seq, self.block, self.dim = new, seq, block, dim
        counts = [-(-n // block) for n in seq]
        self.tables, at = [], 0
        for n in counts:
            self.tables.append(list(range(at, at + n)))
            at += n
        self.cache = torch.zeros(at, kv_heads, block * (dim + 8), dtype=torch.uint8)
        for r, n in enumerate(seq):
            k, v = (torch.randn(n, kv_heads, dim, generator=gen).to(torch.bfloat16) for _ in range(2))
            slots = [self.tables[r][p // block] * block + p % block for p in range(n)]
            if n <= 1000:
                ora.store(k, v, self.cache, torch.tensor(slots), block)
        self.offsets = [0]
        for n in new:
            self.offsets.append(self.offsets[-1] + n)
        self.q = torch.randn(self.offsets[-1], heads, dim, generator=gen).to(torch.bfloat16)

    def args(self):
        return self.q, self.cache, self.tables, self.seq, self.offsets, self.block


@pytest.mark.parametrize("kernel,new,seq", [("split", [1, 4, 2], [1, 60, 200]), ("split", [1] * 4, [90, 300, 17, 128]),
                                            ("prompt", [70], [70]), ("prompt", [65, 80], [300, 90])])
@pytest.mark.parametrize("dim", [64, 128])
def test_own_roundings_pass(kernel, new, seq, dim):
    for seed in range(4):
        b = HostBatch(new, seq, 4, 2, dim, 16, seed)
        assert ora.check_errors(emulate(*b.args(), kernel), *ora.attention_errors(*b.args(), kernel)) is None


@pytest.mark.parametrize("dim", [64, 128])
def test_bf16_operands_fail_for_prompts(dim):
    """Keys, values and weights of 8 bits, in single elements and in the squared error of all (elements'
    bounds a hundred times as wide)."""
    b = HostBatch([70, 66], [200, 66], 4, 2, dim, 16, 5)
    got, (out, sigma, worst) = emulate(*b.args(), "bf16"), ora.attention_errors(*b.args(), "prompt")
    assert "elements" in ora.check_errors(got, out, sigma, worst)
    assert "squared" in ora.check_errors(got, out, sigma, 100 * worst)


@pytest.mark.parametrize("dim", [64, 128])
def test_bf16_weights_fail_for_decode_rows(dim):
    """Weights of 8 bits where the kernel's have 16, in the squared error of all elements."""
    b = HostBatch([1] * 4, [90, 300, 200, 128], 4, 2, dim, 16, 6)
    got, (out, sigma, worst) = emulate(*b.args(), "weights"), ora.attention_errors(*b.args(), "split")
    assert "squared" in ora.check_errors(got, out, sigma, worst)


@pytest.mark.parametrize("kernel", ["split", "prompt"])
@pytest.mark.parametrize("factor", [0, 2])
def test_any_lost_or_doubled_keys_fail(kernel, factor):
    """Long marked sequences as the GPU tests have them: each group of 16 keys, lost or counted twice, takes some
    element past its bound.  (Scores of zero: equal shares, the case where a group's is smallest.)"""
    dim, keys = 128, 20000 if kernel == "split" else 3000
    b = HostBatch([1], [keys], 1, 1, dim, 256, 8)
    words = b.cache.view(torch.int32)
    words[:, :, 256 * dim // 4:] = 0x3E804308  # scales of 0.25
    mark_values(b, dim)
    b.q.zero_()
    out, sigma, worst = ora.attention_errors(*b.args(), kernel)
    limit = worst + 2.0 ** -8 * (out.abs() + worst)
    assert ora.check_errors(out.bfloat16(), out, sigma, worst) is None
    for first in range(0, keys, 16):
        n = min(16, keys - first)
        channel = marked_channel(first, dim)
        moved = n / keys * 15 * 0.25
        changed = out[0, 0, channel] + (factor - 1) * moved
        if n == 16:
            assert abs(changed - out[0, 0, channel]) > 2 * limit[0, 0, channel], first


def test_marks_are_where_they_are_read():
    b = HostBatch([1], [100], 2, 2, 64, 32, 3)
    mark_values(b, 64)
    _, v, _, vs = ora.load(b.cache, list(range(100)), 32)
    for p in range(100):
        want = torch.zeros(2, 64, dtype=torch.float64)
        want[:, marked_channel(p, 64)] = 15 * vs[p]
        assert torch.equal(v[p], want)
