"""Packed (8-bit) archives, tile selection and attention over lists of tiles.

No counterpart in the reference: its archived blocks keep the cache dtype
(cache.py:324-339) and every query attends to all of them. Two opt-in
extensions of ``LayerKVCache`` live here:

* **Packed archive** (``archive_dtype="float8_e4m3fn"``): archived K/V are held
  as e4m3 codes with one power-of-two scale per (64-token tile, KV head), for K
  and for V, so an attention call reads half the bytes. The hot ring keeps the
  cache dtype. ``PackedArchive`` owns the codes; ``pack`` and ``unpack`` convert.
* **Tile selection** (``tile_index=True``): the cache keeps the channel-wise
  smallest and largest key of every archived tile. The selection bounds the
  logits of each tile with them and picks the ``top_tiles`` best for each query
  and KV head; attention then reads those tiles and the hot window only. The
  result is the exact softmax over the keys that are read; the tiles left out
  are the approximation.

Everything runs on ``librfsn_b200.so``; there is no CPU fallback.
"""

from __future__ import annotations

import ctypes
import struct
from functools import lru_cache
from typing import Optional

import torch

from . import _native as native

TILE = native.TILE_KEYS
ARCHIVE_DTYPES = {"float8_e4m3fn": torch.float8_e4m3fn}
# Query rows of one sparse call: every row reads tiles of its own.
SPARSE_MAX_ROWS = 64


def padded_rows(n: int) -> int:
    """Rows of a block of n tokens in an archive of whole tiles."""
    return (n + TILE - 1) // TILE * TILE


def check_archive_options(dtype: torch.dtype, head_dim: int, archive_dtype: Optional[str], tile_index: bool) -> None:
    if archive_dtype is not None and archive_dtype not in ARCHIVE_DTYPES:
        raise ValueError(f"archive_dtype must be None or one of {set(ARCHIVE_DTYPES)}, got {archive_dtype!r}")
    if (archive_dtype is not None or tile_index) and (
            dtype not in (torch.bfloat16, torch.float16) or head_dim not in (64, 128)):
        raise ValueError("a packed archive or a tile index needs a float16 or bfloat16 model_dtype and head_dim 64 or "
                         f"128, got {dtype} and {head_dim}")


_KV_ROWS = struct.Struct("@PPqqqqqqiiii")  # rfsn_kv_rows; packed bytes cost half of a ctypes structure


def kv_rows(k: torch.Tensor, v: torch.Tensor, offset: int = 0, wrap: int = 0) -> bytes:
    """``rfsn_kv_rows`` of K/V [B, Hkv, n, D] (innermost stride 1)."""
    kb, kh, kt, _ = k.stride()
    vb, vh, vt, _ = v.stride()
    return _KV_ROWS.pack(k.data_ptr(), v.data_ptr(), kb, kh, kt, vb, vh, vt, native.dtype_code(k.dtype), k.shape[1],
                         offset, wrap)


class PackedArchive:
    """e4m3 codes ``k``, ``v`` [groups, rows, head_dim] and float32 ``k_scale``,
    ``v_scale`` [groups, rows / 64] of one layer (groups = batch * kv_heads).

    A tile is 64 rows; value = code * scale of its tile. ``rows`` is rounded up
    to whole tiles."""

    def __init__(self, groups: int, rows: int, head_dim: int, *,
                 device: Optional[torch.device | str] = None) -> None:
        native.lib()
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if dev.type != "cuda":
            raise native.NativeUnavailable("a packed archive lives on a CUDA device (no CPU path)")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.device = dev
        self.groups, self.rows, self.head_dim = int(groups), padded_rows(int(rows)), int(head_dim)
        if self.groups <= 0 or self.rows <= 0:
            raise ValueError("a packed archive needs at least one head and one row")
        shape = (self.groups, self.rows, self.head_dim)
        self.k = torch.zeros(shape, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        self.v = torch.zeros(shape, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        # {K scale, V scale, mark of a V tile packed from zeros, 0} per tile
        self.scales = torch.zeros((self.groups, self.rows // TILE, 4), dtype=torch.float32, device=dev)
        self.scales[..., :2] = 1.0
        self.k_scale, self.v_scale = self.scales[..., 0], self.scales[..., 1]
        handle = ctypes.c_void_p()
        with native.on_device(dev):
            native.check(
                native.lib().rfsn_packed_archive_create(self.k.data_ptr(), self.v.data_ptr(), self.scales.data_ptr(),
                                                        self.groups, self.rows, self.head_dim, ctypes.byref(handle)),
                "rfsn_packed_archive_create",
            )
        self.handle = handle

    def close(self) -> None:
        if getattr(self, "handle", None):
            native.load_library().rfsn_packed_archive_destroy(self.handle)
            self.handle = ctypes.c_void_p()

    def __del__(self) -> None:  # pragma: no cover - interpreter shutdown order
        try:
            self.close()
        except Exception:
            pass

    def clear(self) -> None:
        """Zero codes and unit scales (the state of a new archive)."""
        self.k.view(torch.uint8).zero_()
        self.v.view(torch.uint8).zero_()
        self.scales.zero_()
        self.scales[..., :2] = 1.0

    def pack(self, k: torch.Tensor, v: torch.Tensor, row: int = 0, *,
             bounds: Optional[torch.Tensor] = None) -> None:
        """Pack the tokens of k, v [B, Hkv, n, D] (float32, float16 or bfloat16,
        any strides with a contiguous last dimension) into rows row .. row + n
        (``row`` a multiple of 64), in tiles of 64 from the first token on. The
        rest of the last tile is zeroed. ``bounds`` (uint8 [groups, rows / 64,
        2, D]) receives the channel-wise smallest and largest K codes."""
        shape, dtype = k.shape, k.dtype
        if len(shape) != 4 or v.shape != shape or v.dtype != dtype:
            raise ValueError("pack needs k and v of one shape [B, Hkv, n, D] and one dtype")
        if shape[0] * shape[1] != self.groups or shape[3] != self.head_dim:
            raise ValueError(f"K/V of shape {tuple(shape)} do not fit {self.groups} heads of {self.head_dim}")
        if k.device != self.device or v.device != self.device:
            raise ValueError(f"K/V must be on {self.device}")
        if bounds is not None:
            self._check_bounds(bounds)
        if k.stride(3) != 1:
            k = k.contiguous()
        if v.stride(3) != 1:
            v = v.contiguous()
        self._pack(kv_rows(k, v), int(row), shape[2], bounds)

    def pack_ring(self, k: torch.Tensor, v: torch.Tensor, offset: int, wrap: int, row: int, count: int, *,
                  bounds: Optional[torch.Tensor] = None) -> None:
        """``pack`` of ``count`` ring tokens: k, v [groups, rows, D], the ring in
        the first ``wrap`` rows, its oldest token at ``offset``."""
        shape = k.shape
        if len(shape) != 3 or v.shape != shape or v.dtype != k.dtype or shape[0] != self.groups \
                or shape[2] != self.head_dim or k.stride(2) != 1 or v.stride(2) != 1:
            raise ValueError(f"pack_ring needs k and v of one shape [{self.groups}, rows, {self.head_dim}] and one "
                             "dtype, contiguous along the last dimension")
        if k.device != self.device or v.device != self.device:
            raise ValueError(f"K/V must be on {self.device}")
        if not (0 < wrap <= shape[1] and 0 <= offset < wrap and 0 <= count <= wrap):
            raise ValueError(f"{count} tokens from {offset} on do not lie in a ring of {wrap} of {shape[1]} rows")
        if bounds is not None:
            self._check_bounds(bounds)
        self._pack(kv_rows(k[None], v[None], offset, wrap), row, count, bounds)

    def _check_bounds(self, bounds: torch.Tensor) -> None:
        shape = (self.groups, self.rows // TILE, 2, self.head_dim)
        if tuple(bounds.shape) != shape or bounds.dtype != torch.uint8 or bounds.device != self.device \
                or not bounds.is_contiguous():
            raise ValueError(f"bounds must be a contiguous uint8 tensor of shape {shape} on {self.device}")

    def _pack(self, rows: bytes, row: int, count: int, bounds: Optional[torch.Tensor]) -> None:
        with native.on_device(self.device):
            status = native.lib().rfsn_pack_rows(self.handle, row, rows, count,
                                                 bounds.data_ptr() if bounds is not None else None,
                                                 native.stream_ptr())
        if status:
            native.check(status, "rfsn_pack_rows")

    def unpack(self, row: int, n: int, dtype: torch.dtype, *, out: Optional[tuple] = None):
        """(k, v) [groups, n, D] of rows row .. row + n in ``dtype`` (exact in
        float32 and bfloat16; float16 rounds and saturates). ``out``: a pair of
        [groups, n, D] views with one stride between heads to write instead."""
        if out is None:
            shape = (self.groups, n, self.head_dim)
            out = (torch.empty(shape, dtype=dtype, device=self.device),
                   torch.empty(shape, dtype=dtype, device=self.device))
        k, v = out
        for t in (k, v):
            if tuple(t.shape) != (self.groups, n, self.head_dim) or t.dtype != dtype or t.device != self.device \
                    or t.stride() != k.stride() or (n > 0 and t.stride()[1:] != (self.head_dim, 1)):
                raise ValueError(f"out must be two [{self.groups}, {n}, {self.head_dim}] tensors of {dtype} with "
                                 "contiguous rows and one stride between heads")
        with native.on_device(self.device):
            native.check(
                native.lib().rfsn_unpack_rows(self.handle, int(row), int(n), k.data_ptr(), v.data_ptr(),
                                              native.dtype_code(dtype), k.stride(0), native.stream_ptr()),
                "rfsn_unpack_rows",
            )
        return k, v


@lru_cache(maxsize=4096)
def workspace_bytes(batch: int, q_heads: int, kv_heads: int, q_len: int, head_dim: int, hot_capacity: int,
                    n_tiles: int, n_select: int = 0) -> int:
    out = ctypes.c_size_t()
    native.check(
        native.load_library().rfsn_archive_workspace_size(batch, q_heads, kv_heads, q_len, head_dim, hot_capacity,
                                                          n_tiles, n_select, ctypes.byref(out)),
        "rfsn_archive_workspace_size",
    )
    return int(out.value)


class PreparedCall:
    """``rfsn_archive_call`` of a layer's segments for one query shape, and the
    buffers it points to (kept alive with it). ``select_only`` prepares a call
    of ``select`` (no hot window)."""

    __slots__ = ("ref", "nbytes", "numbers", "keep")

    def __init__(self, cache, segments, hot: native.HotWindowC, q_heads: int, q_len: int, top_tiles: int,
                 max_splits: int, select_only: bool = False) -> None:
        if (top_tiles or select_only) and cache.tile_bounds is None:
            raise ValueError("tile selection needs a cache built with tile_index=True")
        if not int(select_only) <= top_tiles <= 1 << 20:
            raise ValueError(f"top_tiles must be between {int(select_only)} and {1 << 20}, got {top_tiles}")
        if top_tiles and q_len > SPARSE_MAX_ROWS:
            raise ValueError(f"top_tiles takes up to {SPARSE_MAX_ROWS} query rows a call, got {q_len}")
        tiles_dev, n_tiles = segments.tile_list
        archive, bounds = cache.archive, cache.tile_bounds
        if not cache.arena.handle or (archive is not None and not archive.handle):
            raise ValueError("the cache's arena or packed archive has been closed")
        call = native.ArchiveCallC(
            cache.arena.handle, archive.handle if archive is not None else None,
            bounds.data_ptr() if top_tiles else None, native.TileListC(tiles_dev.data_ptr(), n_tiles, 0), hot,
            cache.batch_size, q_heads, cache.num_kv_heads, q_len, top_tiles, max_splits)
        self.ref = ctypes.byref(call)
        self.nbytes = workspace_bytes(cache.batch_size, q_heads, cache.num_kv_heads, q_len, cache.config.head_dim,
                                      cache.config.hot_capacity, n_tiles, top_tiles if n_tiles or select_only else 0)
        self.numbers = torch.empty((cache.batch_size, cache.num_kv_heads, q_len, top_tiles), dtype=torch.int32,
                                   device=cache.device) if select_only else None  # shape of a selection
        self.keep = (call, cache.arena, archive, bounds, tiles_dev)

    def current(self, cache) -> bool:
        """The cache's buffers are still the ones this call points to, and open."""
        arena, archive = self.keep[1], self.keep[2]
        return arena is cache.arena and archive is cache.archive and bool(arena.handle) \
            and (archive is None or bool(archive.handle))

    def __call__(self, cache, q_ptr: int, q_start_pos: int, out_ptr: int, lse_ptr: Optional[int],
                 workspace: Optional[native.Workspace]) -> None:
        ws = workspace if workspace is not None else native.default_workspace(cache.device)
        buf = ws.get(self.nbytes)
        status = native.lib().rfsn_archive_attend(self.ref, q_ptr, q_start_pos, out_ptr, lse_ptr, buf.data_ptr(),
                                                  buf.numel(), native.stream_ptr())
        if status:
            native.check(status, "rfsn_archive_attend")

    def select(self, cache, q_ptr: int, q_start_pos: int, workspace: Optional[native.Workspace]) -> torch.Tensor:
        """Numbers of the selected tiles, int32 [B, Hkv, q_len, top_tiles]."""
        out = torch.empty_like(self.numbers)
        ws = workspace if workspace is not None else native.default_workspace(cache.device)
        buf = ws.get(self.nbytes)
        status = native.lib().rfsn_archive_select(self.ref, q_ptr, q_start_pos, out.data_ptr(), buf.data_ptr(),
                                                  buf.numel(), native.stream_ptr())
        if status:
            native.check(status, "rfsn_archive_select")
        return out


__all__ = ["ARCHIVE_DTYPES", "PackedArchive", "PreparedCall", "workspace_bytes"]
