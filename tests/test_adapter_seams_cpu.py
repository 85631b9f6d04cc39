"""CPU checks of the adapters where they meet the rest of the framework: graph
keys under an adapter scope."""
import torch
from torch.utils import _pytree as pytree

from actune_amd.graph import GraphReplay
from actune_amd.kernels.adapters import active_adapter_ids, adapter_scope


def _key(replay, *args):
    return replay._key(*pytree.tree_flatten((args, {})))


def test_a_graph_belongs_to_its_adapter_scope():
    """A graph that was captured without adapters is not replayed with them, nor the other way round, nor for ids that
    its buffer does not fit; ids of one shape share a graph, which reads each replay's values."""
    replay, x = GraphReplay(lambda x: x, {}), torch.zeros(2, 3)
    none = _key(replay, x)
    keys = []
    for ids in (torch.tensor([0, 1], dtype=torch.int32), torch.tensor([1, -1], dtype=torch.int32),
                torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)):
        with adapter_scope(ids):
            assert active_adapter_ids() is ids
            keys.append(_key(replay, x))
            with adapter_scope(None):
                assert _key(replay, x) == none
    assert keys[0] == keys[1]
    assert len({none, *keys}) == 4
    assert active_adapter_ids() is None and _key(replay, x) == none
