"""Packed archives and tile lists without a GPU: sizes and refusals at the edges."""

from types import SimpleNamespace

import pytest
import torch

from rfsn_b200.archive import workspace_bytes
from rfsn_b200.cache import _out_pointer


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("batch,q_heads,kv_heads,q_len", [
    (1, 32, 8, 4), (1, 32, 8, 1), (1, 8, 2, 1), (1, 8, 1, 1), (2, 40, 1, 3), (1, 4, 4, 64), (3, 6, 2, 2), (1, 32, 8, 64)])
@pytest.mark.parametrize("n_tiles,n_select", [(0, 1), (10, 4), (2048, 128), (1, 1 << 12)])
def test_a_selecting_workspace_serves_a_call_over_no_tiles(head_dim, batch, q_heads, kv_heads, q_len, n_tiles, n_select):
    """Up to n_tiles tiles includes none: such a call attends to the window through one list for all rows."""
    shape = (batch, q_heads, kv_heads, q_len, head_dim, 1 << 14)
    assert workspace_bytes(*shape, n_tiles, n_select) >= workspace_bytes(*shape, 0, 0)


class Placed:
    """A tensor's face on a device that need not exist here."""

    def __init__(self, device, shape=(1, 2, 1, 64)):
        self.device, self.dtype, self.shape = torch.device(device), torch.float32, torch.Size(shape)

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096


@pytest.mark.parametrize("named", ["cuda", "cuda:1"])
def test_results_are_refused_on_another_gpu(named):
    """Also where the cache's device is named without an index: its arena lies on one GPU."""
    cache = SimpleNamespace(device=torch.device(named), _arena_k=Placed("cuda:1"))
    assert _out_pointer(cache, Placed("cuda:1"), (1, 2, 1, 64)) == 4096
    for other in ("cuda:0", "cuda:2"):
        with pytest.raises(ValueError, match="out must be on cuda:1"):
            _out_pointer(cache, Placed(other), (1, 2, 1, 64))
