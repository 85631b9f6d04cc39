"""The adapters where they meet the rest of the framework, on the GPU: graph
replay under an adapter scope, codes that linears share, adapted linears in
sibling and gated launches."""
import pytest
import torch

from actune_amd import _block, _native
from actune_amd.graph import GraphReplay
from actune_amd.kernels.adapters import AdaptedLinear, adapter_add, adapter_scope
from actune_amd.kernels.grouped import (GroupedPaddedLinear, grouped_sibling_forward, reuse_mlp_temporary,
                                        shared_activation_scope)
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


@pytest.mark.parametrize("m", [1, 50, 200])
def test_adapted_siblings_equal_separate_calls(m):
    """Sibling projections of which some carry adapters: one launch for the linears, the adapters behind it, in a scope
    and outside; counters as for separate calls."""
    torch.manual_seed(2)
    with torch.inference_mode():
        q, k, v = (_packed(1024, n) for n in (2048, 256, 256))
        q, v = _adapted(q), _adapted(v, rank=40)
        x = torch.randn(m, 1024, device=DEV, dtype=torch.bfloat16)
        for ids in (None, torch.arange(m, device=DEV, dtype=torch.int32) % 4 - 1):
            with adapter_scope(ids):
                want = [layer(x) for layer in (q, k, v)]
                before = [layer.calls for layer in (q, k, v)]
                got = grouped_sibling_forward(x, [q, k, v])
            assert all(torch.equal(g, w) for g, w in zip(got, want))
            assert [layer.calls for layer in (q, k, v)] == [n + 1 for n in before]


def test_an_adapted_mlp_keeps_its_launches(monkeypatch):
    """A GemmaMLP whose projections all carry adapters: patched as unpatched, bit for bit, in a scope and outside, and
    replayed; outside a scope gate and up share a launch and the product is formed in down's quantizer."""
    from transformers import GemmaConfig
    from transformers.models.gemma.modeling_gemma import GemmaMLP
    torch.manual_seed(3)
    cfg = GemmaConfig(hidden_size=1024, intermediate_size=4096, hidden_activation="gelu_pytorch_tanh")
    mlp = GemmaMLP(cfg).to(device=DEV, dtype=torch.bfloat16)
    with torch.inference_mode():
        for name in ("gate_proj", "up_proj", "down_proj"):
            linear = GroupedPaddedLinear(getattr(mlp, name), {"q11": "w4a8"}, "q11", {"w4a8": None})
            setattr(mlp, name, _adapted(linear))
        x = torch.randn(5, 10, 1024, device=DEV, dtype=torch.bfloat16)
        scopes = (None, _ids(0, 1, -1, 2, 0), _ids(2, 2, 1, -1, -1))

        def run(module, ids):
            with adapter_scope(ids):
                return module(x).clone()

        want = [run(mlp, ids) for ids in scopes]
        assert reuse_mlp_temporary(mlp) == 1
        gated, multi = [], []
        for name, seen in (("quantize_gated", gated), ("grouped_forward_multi", multi)):
            call = getattr(_native, name)
            monkeypatch.setattr(_native, name, lambda *a, _call=call, _seen=seen, **kw: (_seen.append(1), _call(*a, **kw))[1])
        for ids, w in zip(scopes, want):
            assert torch.equal(run(mlp, ids), w)
        assert len(multi) == 3 and len(gated) == 1
        replay = GraphReplay(mlp, {n: getattr(mlp, n) for n in ("gate_proj", "up_proj", "down_proj")}, shared_a8=True)
        replay.enabled = True
        for ids, w in (*zip(scopes, want), *zip(scopes, want)):
            assert torch.equal(run(replay, ids), w)
            torch.cuda.synchronize()
        assert len(replay.graphs) == 2
