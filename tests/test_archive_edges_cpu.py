"""Packed archives and tile lists without a GPU: sizes and refusals at the edges."""

import pytest

from rfsn_b200.archive import workspace_bytes


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("batch,q_heads,kv_heads,q_len", [
    (1, 32, 8, 4), (1, 32, 8, 1), (1, 8, 2, 1), (1, 8, 1, 1), (2, 40, 1, 3), (1, 4, 4, 64), (3, 6, 2, 2), (1, 32, 8, 64)])
@pytest.mark.parametrize("n_tiles,n_select", [(0, 1), (10, 4), (2048, 128), (1, 1 << 12)])
def test_a_selecting_workspace_serves_a_call_over_no_tiles(head_dim, batch, q_heads, kv_heads, q_len, n_tiles, n_select):
    """Up to n_tiles tiles includes none: such a call attends to the window through one list for all rows."""
    shape = (batch, q_heads, kv_heads, q_len, head_dim, 1 << 14)
    assert workspace_bytes(*shape, n_tiles, n_select) >= workspace_bytes(*shape, 0, 0)
