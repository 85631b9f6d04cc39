"""Edges of the operators between the packed projections: layouts that are
copied or not read, sizes past one dispatch, values at the ends of their range. Tolerances are those of test_gpu_block.py."""
import pytest
import torch

import test_gpu_block as block
from actune_amd import _block, _native

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("native", [True, False])
def test_attention_token_strides_past_the_kernels(native, monkeypatch):
    """Caches whose tokens lie 2^23 elements apart and more, which the kernels' offsets do not take, are copied, through
    both bindings; one stride below is read in place."""
    from actune_amd.kernels.attention import shared_prefix_attention
    if not native:
        monkeypatch.setattr(_block, "_FAST", _native._CtypesOnly())
    gen, tokens, d = block._gen(21), 70, 64
    q = block._normal(gen, 2, 3, 4, d, dtype=torch.bfloat16)
    for stride in ((1 << 23) - 8, 1 << 23, (1 << 23) + 64):
        cache = torch.empty(tokens * stride, device=DEV, dtype=torch.bfloat16)  # 1.2 GB
        views = []
        for at in (0, 4 * d):  # keys and values of two heads: one sequence's tokens, or every second one of two
            rows = cache.as_strided((1, tokens, 2, d), (0, stride, d, 1), at)
            rows.copy_(block._normal(gen, 1, tokens, 2, d, dtype=torch.bfloat16))
            views.append(rows)
        own = [r.as_strided((2, tokens // 2, 2, d), (tokens // 2 * stride, stride, d, 1), r.storage_offset()) for r in views]
        dense = [r.contiguous() for r in (*views, *own)]
        want = shared_prefix_attention(q, *dense, causal=True, return_lse=True)
        for operands in ((*views, *own), (*views, *dense[2:]), (*dense[:2], *own)):
            got = shared_prefix_attention(q, *operands, causal=True, return_lse=True)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), stride


@pytest.mark.parametrize("native", [True, False])
def test_attention_empty_operands_of_any_layout(native, monkeypatch):
    """No own keys, or no prefix, cut from tensors whose strides no kernel reads."""
    from actune_amd.kernels.attention import shared_prefix_attention
    if not native:
        monkeypatch.setattr(_block, "_FAST", _native._CtypesOnly())
    q, pk, pv, k, v = block._attention_inputs(block._gen(22), 3, 2, 4, 2, 64, 40, 10, 1, torch.bfloat16)
    odd = lambda t: torch.cat([t, t[..., :1]], -1)[:, 1:1, :, 1:]  # noqa: E731
    none = odd(k)
    assert none.shape == (3, 0, 2, 64) and none.stride(0) % 8
    assert torch.equal(shared_prefix_attention(q, pk, pv, none, odd(v)), shared_prefix_attention(q, pk, pv))
    assert torch.equal(shared_prefix_attention(q, odd(pk), odd(pv), k, v),
                       shared_prefix_attention(q, pk[:, :0], pv[:, :0], k, v))
    assert not bool(shared_prefix_attention(q, odd(pk), odd(pv), none, odd(v)).any())


@pytest.mark.parametrize("behind", [False, True])
def test_block_norm_rows_past_a_dispatch(behind):
    """More rows of few columns than a dispatch has room for at one workgroup each."""
    from actune_amd.kernels.norms import block_norm
    dtype, rows, width = torch.bfloat16, (1 << 22) + 4099, 4
    gen = block._gen(23)
    x, y = block._normal(gen, rows, width, dtype=dtype), block._normal(gen, rows, width, dtype=dtype)
    w = block._normal(gen, width, dtype=dtype)
    bw = block._normal(gen, width, dtype=dtype) if behind else None
    hidden, normed = block_norm(x, y, weight=w, branch_weight=bw)
    h, n, size, nsize = block._norm64(x, y, w, bw, None, None, None, 1.0, 0.0, 1e-6)
    block._near(hidden, h, block.UNIT[dtype] * h.abs() + 2.0 ** -18 * size, "hidden")
    block._near(normed, n, block.UNIT[dtype] * n.abs() + 2.0 ** -18 * nsize, "normed")


@pytest.mark.parametrize("b,heads,p,s,g", [((1 << 18) + 1, 16, 5, 2, 1), ((1 << 20) + 1, 16, 12, 2, 1),
                                           ((1 << 21) + 5, 1, 3, 1, (1 << 21) + 5)])
def test_attention_batches_past_a_dispatch(b, heads, p, s, g):
    """More items, and more rows to join, than one dispatch takes."""
    from actune_amd.kernels.attention import shared_prefix_attention
    gen, d, dtype = block._gen(24), 8, torch.bfloat16
    q, pk, pv, k, v = block._attention_inputs(gen, b, 1, heads, heads, d, p, s, g, dtype)
    got, lse = shared_prefix_attention(q, pk, pv, k, v, return_lse=True)
    per = b // g
    for first in range(0, b, 1 << 17):
        rows = slice(first, min(b, first + (1 << 17)))
        keys, vals = (torch.cat([(x[rows] if per == 1 else x.expand(b, -1, -1, -1)[rows]), y[rows]], 1).double()
                      for x, y in ((pk, k), (pv, v)))
        scores = (q[rows].double() * keys).sum(-1) * d ** -0.5  # (one query: [B, keys, heads])
        pr = torch.softmax(scores, 1)[..., None]
        want, size = (pr * vals).sum(1), (pr * vals.abs()).sum(1)
        block._near(got[rows, 0], want, block.UNIT[dtype] * want.abs() + (block.UNIT[dtype] + 1e-4) * size, first)
        block._near(lse[rows, 0], torch.logsumexp(scores, 1), 1e-4, first)


# one launch, and the largest K of one with 16 ranks; two: a token a workgroup, tiles of 16, of 64 and (rank above 64) of
# 32 tokens
ADAPTER_FORMS = [(5, 512, 96, 16), (12, 6143, 1030, 16), (12, 6160, 1030, 16), (5, 512, 96, 40), (5, 512, 96, 100), (70, 512, 96, 16), (70, 520, 100, 128),
                 (2100, 8200, 2100, 16), (2100, 8200, 2100, 64), (2100, 8200, 1030, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("by", [2.0 ** -20, 1.0, 2.0 ** 9])
@pytest.mark.parametrize("m,k,n,r", ADAPTER_FORMS)
def test_adapter_low_products_keep_their_range_in_every_form(m, k, n, r, by, dtype):
    """Low-rank products far above and below f16's range, in each way to form them. The bound is that of
    test_gpu_block.py: 2^-15 of the largest |a| |x| times |b|, and the output's rounding."""
    from actune_amd.kernels.adapters import adapter_add
    gen = block._gen(25)
    x, y = block._normal(gen, m, k, dtype=dtype, by=min(by, 1.0) * 8), torch.zeros(m, n, device=DEV, dtype=dtype)
    a, b = block._normal(gen, 2, r, k, dtype=dtype, by=max(by, 1.0)), block._normal(gen, 2, n, r, dtype=dtype)
    scaling = torch.full((2,), 1.0 / (k * by), device=DEV)
    ids = torch.arange(m, device=DEV, dtype=torch.int32) // 3 % 2
    want, tol = block._adapter64(y, x, a, b, scaling, ids)
    block._near(adapter_add(y, x, a, b, scaling, ids), want, tol + block.UNIT[dtype] * want.abs() + 2.0 ** -25)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,r", ADAPTER_FORMS)
def test_adapter_infinities_and_nan_are_the_formulas(m, k, n, r, dtype):
    """Infinities and NaN in B, in A and in x, beside low-rank products beyond f16's range and of zero: each output is
    infinite, NaN or finite as the formula's is, and the rows of other adapters keep their bits."""
    from actune_amd.kernels.adapters import adapter_add
    gen, inf, nan = block._gen(26), float("inf"), float("nan")
    x, y = block._normal(gen, m, k, dtype=dtype, by=16.0), block._normal(gen, m, n, dtype=dtype)
    a, b = block._normal(gen, 3, r, k, dtype=dtype, by=32.0), block._normal(gen, 3, n, r, dtype=dtype)
    x[:, :8] = (x[:, :8].abs() + 1).to(dtype)
    a[:, 3] = 0                       # (a low-rank product of zero: 0 times an infinity is NaN)
    scaling = torch.tensor([1e-3, -1e-3, 1e-3], device=DEV)
    ids = torch.arange(m, device=DEV, dtype=torch.int32) % 4 - 1
    clean = adapter_add(y, x, a, b, scaling, ids)
    b[0, 5, 1], b[0, 17, 2], b[0, 30, 4], b[0, 40, 3] = inf, -inf, nan, inf
    b[0, 50, 1], b[0, 50, 2] = inf, -inf
    a[1, 2, 7] = inf                  # (x[:, 7] is at least 1: this product is infinite in every row of adapter 1)
    want, tol = block._adapter64(y, x, a, b, scaling, ids)
    got = adapter_add(y, x, a, b, scaling, ids)
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(kind(got), kind(want)), kind
    other = (ids != 0) & (ids != 1)
    assert torch.equal(got[other], clean[other])
    columns = [i for i in range(n) if i not in (5, 17, 30, 40, 50)]
    rows = ids == 0
    assert torch.equal(got[rows][:, columns], clean[rows][:, columns])
    x[2, 9] = inf                     # (ids[2] is 1; one row alone)
    again = adapter_add(y, x, a, b, scaling, ids)
    kept = torch.arange(m, device=DEV) != 2
    assert torch.equal(again[kept].nan_to_num(), got[kept].nan_to_num())


@pytest.mark.parametrize("m,k,n,r", ADAPTER_FORMS)
def test_adapter_factors_far_apart(m, k, n, r):
    """A large low-rank product, a small B and a scaling whose product with the first passes f32's range, and the other
    way round: the result is in range and stays so."""
    from actune_amd.kernels.adapters import adapter_add
    gen, dtype = block._gen(27), torch.bfloat16
    y = torch.zeros(m, n, device=DEV, dtype=dtype)
    ids = torch.zeros(m, device=DEV, dtype=torch.int32)
    for low, up, scale in ((2.0 ** 54, 2.0 ** -90, 2.0 ** 20), (2.0 ** -50, 2.0 ** 110, 2.0 ** -24), (2.0 ** -45, 2.0 ** 90, 2.0 ** -40)):
        x, a = block._normal(gen, m, k, dtype=dtype, by=low), block._normal(gen, 1, r, k, dtype=dtype, by=low)
        b = block._normal(gen, 1, n, r, dtype=dtype, by=up)
        scaling = torch.full((1,), scale, device=DEV)
        want, tol = block._adapter64(y, x, a, b, scaling, ids)
        assert bool(want.abs().max() < 3e38) and bool(want.abs().max() > 1e-30)
        block._near(adapter_add(y, x, a, b, scaling, ids), want, tol + block.UNIT[dtype] * want.abs())


@pytest.mark.parametrize("m,k,n,r", ADAPTER_FORMS)
def test_adapters_keep_to_their_rows_in_every_form(m, k, n, r):
    """A broken adapter, a broken scaling and a broken row reach the rows that name them and no others."""
    from actune_amd.kernels.adapters import adapter_add
    gen, dtype = block._gen(28), torch.float16
    x, y = block._normal(gen, m, k, dtype=dtype), block._normal(gen, m, n, dtype=dtype)
    a, b = block._normal(gen, 3, r, k, dtype=dtype), block._normal(gen, 3, n, r, dtype=dtype)
    scaling = torch.full((3,), 1.0 / k, device=DEV)
    ids = torch.arange(m, device=DEV, dtype=torch.int32) % 4 - 1
    want = adapter_add(y, x, a, b, scaling, ids)
    a[1, 3, 5], b[1, 7, 2], x[1, 9], scaling[1] = torch.inf, torch.nan, torch.nan, torch.inf
    got = adapter_add(y, x, a, b, scaling, ids)
    kept = (ids != 1) & (torch.arange(m, device=DEV) != 1)
    assert torch.equal(got[kept], want[kept])
    assert bool(got[ids == 1].isnan().any()) and bool(got[1].isnan().all())


# every layout of the rows (32 or 128, a sequence's or a group's) at head sizes that fill no padded one, and at full ones
@pytest.mark.parametrize("b,t,hq,hkv,d,p,s,causal", [
    (1, 3, 4, 2, 8, 70, 5, True), (1, 50, 8, 1, 40, 300, 50, False), (2, 5, 8, 2, 80, 500, 17, True),
    (1, 50, 8, 1, 200, 300, 50, False), (12, 3, 4, 4, 56, 2500, 40, True), (12, 3, 4, 4, 104, 2500, 40, True),
    (12, 3, 4, 4, 136, 2500, 40, True), (40, 64, 4, 4, 24, 130, 70, True), (40, 64, 4, 4, 120, 130, 70, True),
    (40, 64, 4, 4, 248, 130, 70, True), (130, 1, 8, 2, 48, 1500, 5, False), (130, 1, 8, 2, 88, 1500, 5, False),
    (130, 1, 8, 1, 152, 1500, 70, False), (40, 64, 4, 4, 128, 130, 70, True), (130, 1, 8, 1, 256, 1500, 70, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_keys_of_infinite_scores(b, t, hq, hkv, d, p, s, causal, dtype):
    """A key that its queries see with a score of minus infinity counts nothing, one of plus infinity gives NaN, at every
    head size: what stands for the columns past it is no part of the score."""
    from actune_amd.kernels.attention import shared_prefix_attention
    gen = block._gen(d + b)
    q, pk, pv, k, v = block._attention_inputs(gen, b, t, hq, hkv, d, p, s, 1, dtype)
    q[..., 0] = (q[..., 0].abs() + 1).to(dtype)
    q[..., d - 1] = (q[..., d - 1].abs() + 1).to(dtype)
    pk[:, ::3, :, 0] = -torch.inf
    pk[:, 1::5, :, d - 1] = -torch.inf
    k[:, 0::4, :, 0] = -torch.inf
    got = block._check_attention(q, pk, pv, k, v, dtype, causal=causal)
    pk[:, p // 2, 0, 0], pk[:, p // 2, 0, d - 1] = torch.inf, 0
    bad = shared_prefix_attention(q, pk, pv, k, v, causal=causal)
    share = hq // hkv
    assert bool(bad[:, :, :share].isnan().all()) and torch.equal(bad[:, :, share:], got[:, :, share:])
