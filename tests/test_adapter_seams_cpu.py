"""CPU checks of the adapters where they meet the rest of the framework: graph
keys under an adapter scope, codes held of a tensor that is written, the
adapted linear in place of the linear."""
import copy

import pytest
import torch
from torch.utils import _pytree as pytree

from actune_amd import _native
from actune_amd.graph import GraphReplay
from actune_amd.kernels import tokenwise
from actune_amd.kernels.adapters import AdaptedLinear, active_adapter_ids, adapter_scope
from actune_amd.kernels.grouped import GroupedPaddedLinear, gated_down_forward, grouped_sibling_forward, shared_activation_scope


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


def _adapted(inputs, outputs, base=None):
    torch.manual_seed(inputs + outputs)
    base = base or GroupedPaddedLinear(torch.nn.Linear(inputs, outputs), {"q11": "w4a8", "q00": "w2a8"}, "q11",
                                       {"w4a8": None, "w2a8": None})
    return AdaptedLinear(base, torch.randn(2, 4, inputs), torch.randn(2, outputs, 4), torch.ones(2))


def test_an_adapted_linear_stands_in_for_its_linear():
    layer = _adapted(128, 64)
    base = layer.base
    assert layer.weight is base.weight and layer.weight.dtype == torch.float32
    assert layer.active_backend() is base.backends["w4a8"] and layer.assignments is base.assignments
    assert layer.padding == 0 and layer.default_profile == "q11"
    layer.calls += 2
    layer.input_elements = 7
    assert (base.calls, base.input_elements, layer.calls) == (2, 7, 2)
    assert [n for n, _ in layer.named_buffers() if "." not in n] == ["a", "b", "scaling"]
    with pytest.raises(AttributeError, match="no_such"):
        layer.no_such
    twin = copy.deepcopy(layer)
    twin.calls += 1
    assert (twin.calls, layer.calls) == (3, 2)
    # over another linear: what that one has, and no more
    plain = _adapted(8, 6, torch.nn.Linear(8, 6))
    assert plain.weight is plain.base.weight and plain.bias is plain.base.bias and not hasattr(plain, "calls")


class _Linear(GroupedPaddedLinear):
    """A packed linear whose call runs on the CPU."""

    def forward(self, x):
        self.calls += 1
        return x @ torch.ones(x.shape[-1], self.out_features)


def test_siblings_and_gated_products_take_adapted_linears(monkeypatch):
    """Adapters are added behind the linears' outputs, each once and to its own, nested ones too; the linears' counters
    advance as for separate calls."""
    from actune_amd.kernels import adapters
    linears = [_Linear(torch.nn.Linear(128, n), {"q11": "w4a8"}, "q11", {"w4a8": None}) for n in (64, 64, 128)]
    add = lambda y, x, a, b, scaling, ids, out=None: y + scaling[0] * x[..., :1] * ids  # noqa: E731
    monkeypatch.setattr(adapters, "adapter_add", add)
    once = _adapted(128, 64, linears[0])
    twice = _adapted(128, 64, _adapted(128, 64, linears[1]))
    x = torch.randn(3, 128)
    for ids in (None, 5):
        with adapter_scope(ids):
            got = grouped_sibling_forward(x, [once, linears[2], twice])
            want = [once(x), linears[2](x), twice(x)]
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    assert not torch.equal(got[0], linears[0](x)) and not torch.equal(got[2], got[0])
    assert (linears[0].calls, linears[1].calls, linears[2].calls) == (5, 4, 4)
    down = _adapted(64, 64, _Linear(torch.nn.Linear(64, 64), {"q11": "w4a8"}, "q11", {"w4a8": None}))
    act, gate, up = torch.nn.functional.silu, torch.randn(3, 64), torch.randn(3, 64)
    for ids in (None, 5):
        with adapter_scope(ids):
            assert torch.equal(gated_down_forward(down, gate, up, act), down(act(gate) * up))
    assert (down.calls, down.base.calls) == (4, 4)
