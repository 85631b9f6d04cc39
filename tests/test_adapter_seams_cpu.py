"""CPU checks of the adapters where they meet the rest of the framework: graph
keys under an adapter scope, codes held of a tensor that is written."""
import pytest
import torch
from torch.utils import _pytree as pytree

from actune_amd import _native
from actune_amd.graph import GraphReplay
from actune_amd.kernels import tokenwise
from actune_amd.kernels.adapters import active_adapter_ids, adapter_scope
from actune_amd.kernels.grouped import shared_activation_scope


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


def test_a_write_moves_the_version_counter():
    t = torch.zeros(4, 6)
    view, before = t[1:, ::2], t._version
    _native.written(view)
    assert t._version == view._version == before + 1
    with torch.no_grad():
        _native.written(t)
    assert view._version == before + 2


@pytest.mark.parametrize("written", ["source", "view", "other"])
def test_a_write_drops_the_codes_of_an_inference_tensor(written):
    """Inference tensors have no version counter: the caches forget what they hold of that memory, and only that."""
    with torch.inference_mode(), shared_activation_scope() as groups, tokenwise.shared_a8_cache_scope() as rows:
        source, other = torch.zeros(4, 6), torch.zeros(4, 6)
        groups.entries.append((source, (None, 0), source.shape, 8, None, other, other))
        for slot in ("entry", "a4_entry"):
            setattr(rows, slot, tokenwise._Codes(source, None, 0, 6, other, other))
        _native.written({"source": source, "view": source[1:, :3], "other": other}[written])
        kept = written == "other"
        assert (len(groups.entries), rows.entry is not None, rows.a4_entry is not None) == (kept, kept, kept)
