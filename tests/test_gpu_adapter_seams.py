"""The adapters where they meet the rest of the framework, on the GPU: graph
replay under an adapter scope."""
import pytest
import torch

from actune_amd.graph import GraphReplay
from actune_amd.kernels.adapters import AdaptedLinear, adapter_scope
from actune_amd.kernels.grouped import GroupedPaddedLinear

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _packed(inputs, outputs, mode="W4A8"):
    linear = torch.nn.Linear(inputs, outputs, bias=False, device=DEV, dtype=torch.bfloat16)
    return GroupedPaddedLinear(linear, {"q11": mode}, "q11", {mode: None})


def _adapted(base, adapters=3, rank=16):
    a = torch.randn(adapters, rank, base.in_features, device=DEV, dtype=torch.bfloat16) * base.in_features ** -0.5
    b = torch.randn(adapters, base.out_features, rank, device=DEV, dtype=torch.bfloat16)
    return AdaptedLinear(base, a, b, torch.rand(adapters, device=DEV) + 0.5)


def _ids(*values):
    return torch.tensor(values, device=DEV, dtype=torch.int32)


def test_replays_follow_the_adapter_scope():
    """Graphs with and without a scope, ids of requests and of tokens, other values and other tensors of the same shape:
    each replay gives what the eager call gives in the same scope."""
    torch.manual_seed(0)
    with torch.inference_mode():
        layer = _adapted(_packed(256, 384))
        replay = GraphReplay(layer, {"base": layer.base})
        replay.enabled = True
        x = torch.randn(4, 5, 256, device=DEV, dtype=torch.bfloat16)

        def check(ids):
            with adapter_scope(ids):
                want = layer(x)
                for _ in range(3):
                    got = replay(x)
                    torch.cuda.synchronize()
                    assert torch.equal(got, want)
            return want

        alone = check(None)
        first = check(_ids(0, 1, -1, 2))
        assert not torch.equal(first, alone) and torch.equal(first[2], alone[2])
        _ids(7, 7, 7, 7)  # (the freed ids' memory, if anything read it still)
        second = check(_ids(2, -1, 1, 0))
        assert not torch.equal(second, first)
        each = check(_ids(*range(20)).view(4, 5) % 4 - 1)
        assert torch.equal(each[0, 0], alone[0, 0]) and not torch.equal(each, second)
        assert torch.equal(check(None), alone)
        assert len(replay.graphs) == 3 and replay.replays == 15 and replay.fallbacks == 0
