"""Caches keyed by tensors' addresses forget a tensor that is gone: a new one at
its address, with the same version and size, holds other data.  An allocator
reuses addresses when it likes; here two tensors in turn lie over one array."""
import numpy as np
import torch


class Memory:
    """tensor(x): a new tensor object of x's data at this memory's address, version 0."""

    def __init__(self, *shape):
        self.data = np.zeros(shape, dtype=np.int64)

    def tensor(self, x):
        self.data[...] = x.numpy()
        return torch.from_numpy(self.data)


def test_index_copies():
    from trafficrl.models.fused import _idx32
    memory, x = Memory(2, 50), torch.arange(100).view(2, 50)
    t = memory.tensor(x)
    a = _idx32(t[0])
    assert torch.equal(a, x[0].int()) and torch.equal(_idx32(t[1]), x[1].int())
    assert _idx32(t[0]) is a             # found again while t lives, though t[0] is a new view
    del t
    t = memory.tensor(x.flip(0))
    assert torch.equal(_idx32(t[0]), x[1].int()) and torch.equal(_idx32(t[1]), x[0].int())


def test_views_of_one_memory():
    """The same address and count, another stride."""
    from trafficrl.models.fused import _idx32
    t = torch.arange(40)
    assert torch.equal(_idx32(t[:20]), t[:20].int()) and torch.equal(_idx32(t[::2]), t[::2].int())


B, N, M = 5, 24, 76


def batch(seed, order=range(B)):
    local = torch.randint(0, N, (2, M), generator=torch.Generator().manual_seed(seed))
    return local, local.repeat(1, B) + (torch.tensor(list(order)) * N).repeat_interleave(M)


def test_edge_layout():
    from trafficrl.rl import sac
    edges, graphs = Memory(2, B * M), torch.arange(B).repeat_interleave(N)
    ei = edges.tensor(batch(1)[1])
    assert sac.is_regular_edges(ei, graphs, B) and sac.is_regular_edges(ei, graphs, B)
    del ei
    assert not sac.is_regular_edges(edges.tensor(batch(1, reversed(range(B)))[1]), graphs, B)


def test_regular_layout():
    from trafficrl.rl import sac
    edges, graphs = Memory(2, B * M), torch.arange(B).repeat_interleave(N)
    for seed in (1, 2, 3):
        local, all_ = batch(seed)
        ei = edges.tensor(all_)
        r = sac.regular_layout(ei, graphs, B)
        assert r[0] == B and torch.equal(r[1], local[0]) and torch.equal(r[2], local[1])
        assert sac.regular_layout(ei, graphs, B) is r
        del ei
