"""The workspaces and arrival counters that ``attention_int4`` keeps: one pair a stream whichever
thread asks first, and a supply that captured calls may use up."""
import threading

import pytest
import torch

from test_gpu_attention import Batch, attn

pytestmark = pytest.mark.gpu


class MeetAtFirstLook(dict):
    """The pool's streams, whose first look-up of each of two threads waits for the other's."""

    def __init__(self):
        super().__init__()
        self.barrier = threading.Barrier(2)
        self.seen = set()

    def get(self, key, default=None):
        found = super().get(key, default)
        me = threading.get_ident()
        if me not in self.seen:
            self.seen.add(me)
            self.barrier.wait(20)
        return found


def test_two_threads_first_call_on_a_stream(gpu_lib):
    """Both find no pair; one makes it, the other takes that one, and one set of counters is gone."""
    pool = attn._ScratchPool()
    pool._streams = MeetAtFirstLook()
    pairs = []
    threads = [threading.Thread(target=lambda: pairs.append(pool.get(0, 4096))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert len(pairs) == 2 and pairs[0][1] is pairs[1][1] and pairs[0][0] is pairs[1][0]
    assert len(pool._free[0]) == pool.SETS - 1


def test_grown_workspace_keeps_its_counters(gpu_lib):
    pool = attn._ScratchPool()
    small = pool.get(0, 256)
    large = pool.get(0, 1 << 20)
    assert small[1] is large[1] and large[0].numel() >= 1 << 20 and pool.get(0, 1000) is large


def test_used_up_counters_are_supplied_again(gpu_lib, monkeypatch):
    """Captured calls that use the last sets: the next eager call, on an old stream or a new one,
    makes new ones, keeps its pair, and later captures have sets of their own again."""
    pool = attn._ScratchPool()
    monkeypatch.setattr(attn, "SCRATCH", pool)
    b = Batch([1, 3], [2500, 700], 8, 2, 128, 16, seed=82)
    args = b.args()
    want = attn.attention_int4(*args, block_size=16)
    b.check(want)
    del pool._free[0][2:]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [attn.attention_int4(*args, block_size=16) for _ in range(3)]  # the last one has none left
    assert len(pool._captured) == 2 and not pool._free[0]
    assert torch.equal(attn.attention_int4(*args, block_size=16), want)
    assert len(pool._free[0]) == pool.SETS
    pool._free[0].clear()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        assert torch.equal(attn.attention_int4(*args, block_size=16), want)
        assert pool.get(0, 16) is pool.get(0, 16)
    assert len(pool._free[0]) == pool.SETS - 1
    torch.cuda.synchronize()
    again = torch.cuda.CUDAGraph()
    with torch.cuda.graph(again):
        outs.append(attn.attention_int4(*args, block_size=16))
    assert len(pool._captured) == 3
    sets = [c.data_ptr() for c in pool._captured] + [c.data_ptr() for _, c in pool._streams.values()]
    assert len(set(sets)) == len(sets)
    for _ in range(3):
        for o in outs:
            o.fill_(5)
        graph.replay()
        again.replay()
        assert torch.equal(attn.attention_int4(*args, block_size=16), want)
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
