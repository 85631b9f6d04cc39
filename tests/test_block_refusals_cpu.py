"""Refusals of the operators' C ABI at the ends of their ranges."""
import pytest

from actune_amd import _block


@pytest.mark.parametrize("rank,most", [(1, 64 * (2**24 - 1)), (64, 64 * (2**24 - 1)), (65, 32 * (2**24 - 1)),
                                       (128, 32 * (2**24 - 1))])
def test_adapter_tokens_end_where_a_dispatch_ends(rank, most):
    """The second product's workgroups of 256 threads, 64 tokens each (32 above rank 64), stay below 2^32 threads."""
    size = _block.lib().actune_adapter_workspace_bytes
    assert size(most, 64, 64, rank) > 0
    assert size(most + 1, 64, 64, rank) == -1
    args = _block.AdapterArgs(x=16, y=16, a=16, b=16, scaling=16, ids=16, out=16, x_stride=64, y_stride=64, out_stride=64,
                              ids_rows=1, M=most + 1, N=64, K=64, R=rank, L=2, dtype=0)
    assert _block.lib().actune_adapter_add(args, None) == 1
    assert "dimensions" in _block.lib().actune_block_last_error().decode()


@pytest.mark.parametrize("tokens,out_stride,message", [(4, 64, "y's row stride"), (4, 80, "workspace"), (1, 64, "workspace")])
def test_adapter_out_on_y_takes_the_stride_of_y(tokens, out_stride, message):
    """Rows written over others of y would be read as y, and rows without an adapter would not be moved."""
    args = _block.AdapterArgs(x=16, y=1024, a=16, b=16, scaling=16, ids=16, out=1024, x_stride=64, y_stride=80,
                              out_stride=out_stride, ids_rows=1, M=tokens, N=64, K=64, R=8, L=2, dtype=0)
    assert _block.lib().actune_adapter_add(args, None) == 1
    assert message in _block.lib().actune_block_last_error().decode()
