"""Low-rank adapters of many requests beside a shared packed projection.

A batch of requests that share one resident bank, each with an adapter of its
own: ``adapter_add`` adds every row's adapter to the projection's output
(csrc/adapter.hip), ``AdaptedLinear`` does so behind a packed linear, and
``adapter_scope`` says which adapter each request of a forward uses. No
counterpart in the reference, which serves the bank's own weights only.
"""
from __future__ import annotations

from contextlib import contextmanager
from contextvars import ContextVar

import torch

from .. import _block, _native
from .norms import _rows

_TYPES = (torch.bfloat16, torch.float16)
_IDS: ContextVar[torch.Tensor | None] = ContextVar("actune_adapter_ids", default=None)


def adapter_add(y, x, a, b, scaling, ids, out=None):
    """y + scaling[id] * b[id] @ (a[id] @ x) for every row, id = the row's.

    x: [..., K] (what the projection read), y: [..., N] (its output), a: [L, R,
    K], b: [L, N, R], all bf16 or all f16; scaling: f32 [L]; ids: int32, one
    for each row or, with fewer dimensions, for each of the leading ones ([B]
    for x [B, T, K]). A row whose id is not in [0, L) (-1, say) keeps y.
    1 <= R <= 128; adapters of a lower rank are padded with zeros. out: a
    tensor to write to, y itself included; a new one by default (written as by
    torch's in-place operators: codes that a shared scope holds of it are not
    used again). Sums in f32, one rounding at the end.
    """
    done = _block.fast().adapter_add(y, x, a, b, scaling, ids, out)
    if done is not None:
        if out is not None:
            _native.written(out)
        return done
    _block.check_inputs([("x", x), ("y", y), ("a", a), ("b", b)] + ([] if out is None else [("out", out)]), _TYPES)
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
        raise ValueError(f"adapters must be a [L, R, K] and b [L, N, R], got {list(a.shape)} and {list(b.shape)}")
    count, rank, k = a.shape
    n = b.shape[1]
    if not 1 <= rank <= 128:
        raise ValueError(f"rank must be between 1 and 128, got {rank}")
    if k < 1 or n < 1 or x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"x must be [..., {k}], got {list(x.shape)}")
    if tuple(y.shape) != (*x.shape[:-1], n):
        raise ValueError(f"y must be {[*x.shape[:-1], n]}, got {list(y.shape)}")
    _block.check_index("scaling", scaling, x.device, torch.float32, (count,))
    if scaling.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("scaling requires grad: this operator has no backward")
    if not isinstance(ids, torch.Tensor):
        raise TypeError("ids must be a tensor")
    if ids.dim() > x.dim() - 1 or ids.shape != x.shape[:ids.dim()]:
        raise ValueError(f"ids must be leading dimensions of {list(x.shape[:-1])}, got {list(ids.shape)}")
    _block.check_index("ids", ids, x.device, torch.int32, ids.shape)
    if out is not None and (out.shape != y.shape or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous {list(y.shape)} tensor")
    rows_x, rows_y = _rows(x, k), _rows(y, n)
    a, b, scaling, ids = a.contiguous(), b.contiguous(), scaling.contiguous(), ids.contiguous()
    m = rows_x.shape[0]
    need = _block.lib().actune_adapter_workspace_bytes(m, n, k, rank)
    if need < 0:
        raise ValueError("invalid dimensions")
    given = out is not None
    if not given:
        out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    work = torch.empty(need, dtype=torch.uint8, device=x.device)
    args = _block.AdapterArgs(
        x=_block.ptr(rows_x), y=_block.ptr(rows_y), a=_block.ptr(a), b=_block.ptr(b), scaling=_block.ptr(scaling),
        ids=_block.ptr(ids), out=_block.ptr(out), workspace=_block.ptr(work), workspace_bytes=need,
        x_stride=rows_x.stride(0), y_stride=rows_y.stride(0), out_stride=n,
        ids_rows=m // ids.numel() if m and ids.numel() else 1, M=m, N=n, K=k, R=rank, L=count,
        dtype=_native.DTYPE_CODES[x.dtype])
    _block.launch("actune_adapter_add", args, x.device)
    if given:
        _native.written(out)
    return out


@contextmanager
def adapter_scope(ids):
    """The adapter of each request (int32, leading dimensions of the linears'
    inputs; None: no adapters) for the AdaptedLinears of one forward. The
    tensor is read when the launches run. Around a GraphReplay it is an input
    like the call's arguments: a graph belongs to a scope's shape of ids (or to
    none), and a replay reads the values that the scope has then. A scope
    inside the captured function reads the tensor that it was captured with:
    make that one an argument of the function."""
    token = _IDS.set(ids)
    try:
        yield
    finally:
        _IDS.reset(token)


def active_adapter_ids():
    """The ids of the innermost adapter_scope (None: no adapters)."""
    return _IDS.get()


class AdaptedLinear(torch.nn.Module):
    """A packed linear (any module with in_features and out_features) with L
    adapters of rank R beside it, in the dtype of the activations. Outside an
    adapter_scope it is the linear alone. It stands in for the linear: what it
    has no attribute of its own for (weight, active_backend, assignments, ..)
    is the linear's, the call counters among it, and sibling and gated
    launches (kernels.grouped) take it."""

    def __init__(self, base, a, b, scaling):
        super().__init__()
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] \
                or a.shape[2] != base.in_features or b.shape[1] != base.out_features:
            raise ValueError(f"adapters do not fit a {base.in_features} to {base.out_features} projection: "
                             f"{list(a.shape)}, {list(b.shape)}")
        if tuple(scaling.shape) != (a.shape[0],) or scaling.dtype != torch.float32:
            raise ValueError("scaling must be one float32 for each adapter")
        self.in_features, self.out_features = base.in_features, base.out_features
        self.register_buffer("a", a.detach().contiguous())
        self.register_buffer("b", b.detach().contiguous())
        self.register_buffer("scaling", scaling.detach().contiguous())
        self.base = base  # (behind the buffers: attributes are the base's from here on)

    def __getattr__(self, name):
        try:
            return super().__getattr__(name)
        except AttributeError:
            if name == "base" or name.startswith("__"):  # (not set yet; python's own)
                raise
            return getattr(self.base, name)

    @property
    def calls(self):
        return self.base.calls

    @calls.setter
    def calls(self, value):
        self.base.calls = value

    @property
    def input_elements(self):
        return self.base.input_elements

    @input_elements.setter
    def input_elements(self, value):
        self.base.input_elements = value

    def adapt(self, y, x):
        """y (the linear's output on x, which this may write) with the scope's
        adapters added: for outputs of a call that runs several linears."""
        ids = active_adapter_ids()
        if ids is None:
            return y
        return adapter_add(y, x, self.a, self.b, self.scaling, ids, out=y if y.is_contiguous() else None)

    def forward(self, x):
        return self.adapt(self.base(x), x)
