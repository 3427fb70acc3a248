"""Packed archives and tile lists at the edges of what callers may hand over."""

import pytest

from test_archive_gpu import check_out, held, make, queries

pytestmark = pytest.mark.gpu


def _torch():
    import torch

    return torch


# ------------------------------------------------------------------ tile entries
@pytest.mark.parametrize("row", [2 ** 31 - 64, 2 ** 31 - 1, 2 ** 31 - 33, -2 ** 31])
@pytest.mark.parametrize("packed,Lq,top", [(True, 1, 0), (True, 4, 0), (True, 128, 0), (True, 1, 81), (False, 1, 81)])
def test_a_row_near_the_end_of_32_bits_is_reported_and_skipped(packed, Lq, top, row):
    """Row + length of such an entry is no 32-bit number; the other tiles are read as before."""
    torch = _torch()
    import archive_ref as ref
    from rfsn_b200 import _native as native
    from rfsn_b200.cache import paged_attention

    lens = (64,) * 81
    cache, k, v = make("bfloat16", 1, 8, 2, 128, lens, 100, tile_index=True,
                       archive_dtype="float8_e4m3fn" if packed else None)
    q = queries(1, 8, Lq, 128)
    n = sum(lens) + 100
    segs = cache.get_attention_segments()
    cache._tiles_dev[5, 0] = row
    ws = native.Workspace(cache.device)
    out, lse = paged_attention(cache, q, n - Lq, segs, workspace=ws, top_tiles=top, want_lse=True)
    with pytest.raises(RuntimeError):
        ws.check()
    seen = torch.ones(1, 2, Lq, n, dtype=torch.bool)
    seen[..., 320:384] = False
    kk, vv = held(cache, k, v, lens)
    want, want_lse = ref.attention(q, kk, vv, torch.arange(n), n - Lq, seen)
    check_out(out, lse, want, want_lse, vv)
