"""Packed archives and tile lists without a GPU: sizes and refusals at the edges."""

import ctypes
from types import SimpleNamespace

import pytest
import torch

from rfsn_b200 import _native as native
from rfsn_b200.archive import PackedArchive, PreparedCall, workspace_bytes
from rfsn_b200.cache import _out_pointer
from rfsn_b200.sharded import GraphedShardedDecodeStep, sharded_decode_step


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


def test_ring_tokens_outside_the_tensors_are_refused():
    """Before anything is launched: the kernel reads what it is told."""
    a = object.__new__(PackedArchive)
    a.device, a.groups, a.rows, a.head_dim, a.handle = torch.device("cpu"), 2, 128, 64, None
    k = torch.zeros(2, 100, 64)
    for offset, wrap, count in ((0, 101, 10), (100, 100, 1), (-1, 100, 1), (0, 100, 101), (0, 0, 1), (0, -5, 1),
                                (60, 50, 10), (0, 100, -1)):
        with pytest.raises(ValueError, match="ring of"):
            a.pack_ring(k, k, offset, wrap, 0, count)
    for bad in (k[:1], k[None], k[:, :, :32], k[:, :50], k.half(), k.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(ValueError, match="pack_ring needs"):
            a.pack_ring(k, bad, 0, 50, 0, 10)
        with pytest.raises(ValueError, match="pack_ring needs"):
            a.pack_ring(bad, k, 0, 50, 0, 10)
    a.device = torch.device("cuda:0")
    with pytest.raises(ValueError, match="must be on cuda:0"):
        a.pack_ring(k, k, 0, 100, 0, 10)
    a.handle = None  # nothing to destroy


@pytest.mark.parametrize("packed", [True, False])
def test_a_prepared_call_does_not_outlive_what_it_points_to(packed):
    """Prepared calls hold the handles of the arena and the archive by value: closed ones are refused."""
    arena = SimpleNamespace(handle=ctypes.c_void_p(4096))
    archive = SimpleNamespace(handle=ctypes.c_void_p(8192)) if packed else None
    cache = SimpleNamespace(arena=arena, archive=archive, tile_bounds=torch.zeros(16), batch_size=1, num_kv_heads=2,
                            config=SimpleNamespace(head_dim=64, hot_capacity=64), device=torch.device("cpu"))
    segments = SimpleNamespace(tile_list=(torch.zeros(4, 4, dtype=torch.int32), 4))

    def prepare():
        return PreparedCall(cache, segments, native.HotWindowC(), 8, 1, 2, 0)

    call = prepare()
    assert call.current(cache)
    closed = [arena, archive] if packed else [arena]
    for part in closed:
        saved, part.handle = part.handle, ctypes.c_void_p()
        assert not call.current(cache)
        with pytest.raises(ValueError, match="closed"):
            prepare()
        part.handle = saved
    assert call.current(cache)
    cache.arena = SimpleNamespace(handle=arena.handle)
    assert not call.current(cache)


def test_sharded_decode_refuses_a_cache_that_selects():
    """It reads every tile of each rank's shard; dropping the option in silence would be another result."""
    cache = SimpleNamespace(top_tiles=3)
    x = torch.zeros(1, 2, 1, 64)
    for owns_hot in (True, False):
        with pytest.raises(NotImplementedError, match="top_tiles"):
            sharded_decode_step(cache, x, x, x, 0, owns_hot=owns_hot)
        with pytest.raises(NotImplementedError, match="top_tiles"):
            GraphedShardedDecodeStep(cache, 2, owns_hot=owns_hot, peers=None)
