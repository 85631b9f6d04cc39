"""Attention of a batch over a prefix that it shares.

A policy's samples of one observation, the denoising steps of its action
expert and the requests behind one prompt all attend to the same long run of
keys. ``shared_prefix_attention`` reads that run once for all of them and
each sequence's own keys beside it (csrc/attention.hip). No counterpart in the
reference, whose models run torch's attention between the packed linears.
"""
from __future__ import annotations

import torch

from .. import _block, _native

_TYPES = (torch.bfloat16, torch.float16)


def _operand(t, keys):
    """t with dense heads and strides and address in whole 16 bytes, and its
    strides {batch, token, head} (0 for dimensions of one element): a copy
    only where its layout is another, or a token's stride of keys or values too
    long."""
    def strides(t):
        return [t.stride(i) if t.shape[i] > 1 else 0 for i in range(3)]
    got = strides(t)
    if t.stride(3) != 1 or any(s % 8 for s in got) or keys and got[1] >= 1 << 23 or t.data_ptr() % 16:
        t = t.contiguous()
        t = t.clone() if t.data_ptr() % 16 else t
        got = strides(t)
    return t, (_block._I64 * 3)(*got)


def shared_prefix_attention(q, prefix_k, prefix_v, k=None, v=None, *, prefix_lengths=None, prefix_mask=None,
                            lengths=None, causal=False, scale=None, return_lse=False):
    """softmax(scale * q . keys) values over a shared prefix and own keys.

    q: [B, T, Hq, D]. prefix_k, prefix_v: [P, Hkv, D], shared by all B
    sequences, or [G, P, Hkv, D]: sequence b reads prefix b // (B / G).
    k, v: [B, S, Hkv, D], each sequence's own keys, or None. Query head h reads
    key head h // (Hq / Hkv). D is a multiple of 8 up to 256, all bf16 or all
    f16; heads and tokens may be strided (a cache with heads first, a slice of
    a longer one).

    prefix_lengths: int32 [G], prefix_mask: bool [G, P] (or [P]), True for keys
    that are seen; lengths: int32 [B], own keys of each sequence. All on the
    device; lengths outside their range are clamped. causal: query t is the
    own key lengths[b] - T + t and sees the whole prefix and the own keys up
    to itself. scale: D ** -0.5 by default, above zero.

    Returns out [B, T, Hq, D] and, with return_lse, the log of the softmax's
    sum, f32 [B, T, Hq], by which the result can be joined with attention over
    further keys. A query that sees no key gets 0 and -inf. What keys and
    values hold that a query does not see does not matter to it, NaN included.
    Scores, sums and the softmax's statistics are f32; its probabilities are
    rounded to q's type for the product with the values.
    """
    single = isinstance(prefix_k, torch.Tensor) and prefix_k.dim() == 3 and isinstance(prefix_v, torch.Tensor)
    if single:
        prefix_k = prefix_k[None]
        prefix_v = prefix_v[None]
    if isinstance(prefix_mask, torch.Tensor) and prefix_mask.dim() == 1:
        prefix_mask = prefix_mask[None]
    if scale is None and isinstance(q, torch.Tensor) and q.dim() == 4:
        scale = q.shape[3] ** -0.5 if q.shape[3] else 1.0
    done = _block.fast().prefix_attention(q, prefix_k, prefix_v, k, v, prefix_lengths, prefix_mask, lengths, causal,
                                          scale, return_lse)
    if done is not None:
        return done
    if (k is None) != (v is None):
        raise ValueError("k and v go together")
    _block.check_inputs([(n, t) for n, t in (("q", q), ("prefix_k", prefix_k), ("prefix_v", prefix_v), ("k", k), ("v", v))
                         if t is not None or n[0] in "qp"], _TYPES)
    if q.dim() != 4 or prefix_k.dim() != 4:
        raise ValueError("q must be [B, T, Hq, D] and the prefix [P, Hkv, D] or [G, P, Hkv, D]")
    b, t, hq, d = q.shape
    g, p, hkv, _ = prefix_k.shape
    if prefix_k.shape[3] != d or prefix_v.shape != prefix_k.shape:
        raise ValueError(f"prefix_k and prefix_v must both be [.., P, Hkv, {d}], got {list(prefix_k.shape)} and "
                         f"{list(prefix_v.shape)}")
    if k is not None and (k.dim() != 4 or (k.shape[0], k.shape[2], k.shape[3]) != (b, hkv, d) or v.shape != k.shape):
        raise ValueError(f"k and v must both be [{b}, S, {hkv}, {d}], got {list(k.shape)} and {list(v.shape)}")
    if d < 8 or d > 256 or d % 8:
        raise ValueError(f"head size must be a multiple of 8 up to 256, got {d}")
    if hkv < 1 or hq < 1 or hq % hkv:
        raise ValueError(f"query heads must be a multiple of key heads, got {hq} and {hkv}")
    if g < 1 or b % g:
        raise ValueError(f"a batch of {b} is not whole groups of {g} prefixes")
    for name, x, dtype, shape in (("prefix_lengths", prefix_lengths, torch.int32, (g,)),
                                  ("prefix_mask", prefix_mask, torch.bool, (g, p)),
                                  ("lengths", lengths, torch.int32, (b,))):
        if x is not None:
            _block.check_index(name, x, q.device, dtype, shape)
    out = torch.empty((b, t, hq, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((b, t, hq), dtype=torch.float32, device=q.device) if return_lse else None
    operands = {"q": q, "prefix_k": prefix_k, "prefix_v": prefix_v, "k": k, "v": v}
    args = _block.AttentionArgs(out=_block.ptr(out), lse=_block.ptr(lse), B=b, G=g, T=t, Hq=hq, Hkv=hkv, D=d, P=p,
                                S=0 if k is None else k.shape[1], scale=scale, causal=bool(causal),
                                dtype=_native.DTYPE_CODES[q.dtype])
    held = []  # copies live until the call is made
    for name, x in operands.items():
        if x is not None and x.numel():  # (none of an empty one is read: its layout does not matter)
            x, stride = _operand(x, name != "q")
            held.append(x)
            setattr(args, name, _block.ptr(x))
            setattr(args, name + "_stride", stride)
    for name, x in (("prefix_lengths", prefix_lengths), ("lengths", lengths)):
        if x is not None:
            held.append(x.contiguous())
            setattr(args, name, _block.ptr(held[-1]))
    if prefix_mask is not None:
        mask = prefix_mask if p <= 1 or prefix_mask.stride(1) == 1 else prefix_mask.contiguous()
        held.append(mask)
        args.prefix_mask = _block.ptr(mask)
        args.mask_stride = mask.stride(0) if g > 1 else 0
    need = _block.lib().actune_prefix_attention_workspace_bytes(args)
    if need < 0:
        raise ValueError("invalid dimensions")
    work = torch.empty(need, dtype=torch.uint8, device=q.device)
    args.workspace, args.workspace_bytes = _block.ptr(work), need
    _block.launch("actune_prefix_attention", args, q.device)
    return (out, lse) if return_lse else out
