"""The sharded decode step hands the heads' norms to the rank that appends and to the ranks that only rotate the
query alike, and asks nothing new of an engine whose model has none."""
from types import SimpleNamespace

import pytest
import torch

from oomllama_b200.shard import DecodeShardPlan, ShardedDecodeStep


class _Engine:
    def __init__(self):
        self.config = SimpleNamespace(n_heads=4)
        self.calls = []

    def set_position_offset(self, s, a):
        pass

    def rope_append(self, layer, seq_ids, q, k, v, *bias, **norms):
        self.calls.append(("append", len(seq_ids), norms))
        return torch.zeros(q.shape[0], 4, 128)

    def rope_q(self, positions, q, bq=None, **norms):
        self.calls.append(("rotate", len(positions), norms))
        return torch.zeros(q.shape[0], 4, 128)


@pytest.mark.parametrize("rank", [0, 1])
@pytest.mark.parametrize("normed", [True, False])
def test_norms_reach_every_rank(rank, normed):
    eng = _Engine()
    step = ShardedDecodeStep(eng, DecodeShardPlan(4, 1, 2, rank), 0, [0, 1], [40, 3])
    step.decoder = lambda layer, ids, q: q
    w = dict(q_norm=torch.ones(128), k_norm=2 * torch.ones(128), eps=1e-5) if normed else {}
    step(torch.zeros(2, 512), torch.zeros(2, 128), torch.zeros(2, 128), **w)
    kinds = [c[0] for c in eng.calls]
    assert kinds == (["rotate"] if rank == 0 else ["append"])  # the last slice stores the new tokens
    for kind, n, norms in eng.calls:
        assert n == 2
        if not normed:
            assert norms == {}
        else:
            assert norms["q_norm"] is w["q_norm"] and norms["eps"] == 1e-5
            assert kind == "rotate" or norms["k_norm"] is w["k_norm"]


def test_int_arrays_take_what_they_took():
    """Lists, ranges, generators, arrays and numbers that are no int."""
    import numpy as np
    from oomllama_b200._lib import int_array
    for v in ([3, 1], (3, 1), range(3, 1, -2), (x for x in (3, 1)), np.array([3, 1]), [3.0, 1.0], (x for x in (3.0, 1.0)),
              [np.int64(3), 1], torch.tensor([3, 1])):
        want = [3] if isinstance(v, range) else [3, 1]
        assert list(int_array(v)) == want
    assert list(int_array([])) == [0]
