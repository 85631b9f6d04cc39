"""The adapters where they meet the rest of the framework, on the GPU: graph
replay under an adapter scope, codes that linears share."""
import pytest
import torch

from actune_amd import _block, _native
from actune_amd.graph import GraphReplay
from actune_amd.kernels.adapters import AdaptedLinear, adapter_add, adapter_scope
from actune_amd.kernels.grouped import GroupedPaddedLinear, shared_activation_scope
from actune_amd.kernels.tokenwise import W4A8TritonLinear, shared_a8_cache_scope

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


@pytest.mark.parametrize("mode", [torch.inference_mode, torch.no_grad, torch.enable_grad])
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("kind", ["groups", "rows"])
def test_codes_of_a_written_tensor_are_not_used_again(mode, native, kind, monkeypatch):
    """lin(t), adapters added to t in place, lin2(t) in one scope of shared codes: lin2 reads what t holds then, also where
    the call wrote through a view; codes of a tensor that was not written are still shared."""
    if not native:
        monkeypatch.setattr(_block, "_FAST", _native._CtypesOnly())
    torch.manual_seed(1)
    with torch.no_grad():
        if kind == "groups":
            scope, (first, second) = shared_activation_scope, (_packed(512, 512), _packed(512, 128))
        else:
            scope = shared_a8_cache_scope
            first, second = (W4A8TritonLinear(torch.nn.Linear(512, n, dtype=torch.bfloat16, device=DEV)) for n in (512, 128))
    with mode():
        x, t = (torch.randn(48, 512, device=DEV, dtype=torch.bfloat16) for _ in range(2))
        a = torch.randn(2, 8, 512, device=DEV, dtype=torch.bfloat16)
        b = torch.randn(2, 512, 8, device=DEV, dtype=torch.bfloat16)
        scaling, ids = torch.ones(2, device=DEV), torch.arange(48, device=DEV, dtype=torch.int32) % 2
        for out in (t, t[:24], t.view(48, 512)):
            with torch.no_grad(), scope() as state:
                stale = second(t)
                first(t)
                n = out.shape[0]
                adapter_add(out, x[:n], a, b, scaling, ids[:n], out=out)
                got = second(t)
                before = state.hits
                first(t)
                assert state.hits == before + 1
            with torch.no_grad(), scope():
                assert torch.equal(got, second(t.clone()))
            assert not torch.equal(got, stale)
