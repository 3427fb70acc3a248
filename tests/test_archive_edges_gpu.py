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


# ------------------------------------------------------------------ launch order
def edge_types(fn, stream=None):
    """Captures ``fn``, a chain of kernels, and gives the type of its dependencies in order (0: the later kernel
    starts after the earlier one, 1: they overlap), from the driver's description of the graph."""
    import ctypes

    torch = _torch()
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g, stream=stream):
        fn()
    handle, n = ctypes.c_void_p(g.raw_cuda_graph()), ctypes.c_size_t(0)
    edges = ctypes.CDLL("libcuda.so.1").cuGraphGetEdges_v2
    assert edges(handle, None, None, None, ctypes.byref(n)) == 0
    src, dst = (ctypes.c_void_p * n.value)(), (ctypes.c_void_p * n.value)()
    data = (ctypes.c_uint8 * 8 * n.value)()  # {from port, to port, type, reserved[5]}
    assert edges(handle, src, dst, data, ctypes.byref(n)) == 0
    follow = {src[i]: (dst[i], data[i][2]) for i in range(n.value)}
    assert len(follow) == n.value  # a chain
    at, types = (set(src) - set(dst)).pop(), []
    while at in follow:
        at, kind = follow[at]
        types.append(kind)
    return types


@pytest.mark.parametrize("Lq", [1, 4])
@pytest.mark.parametrize("packed", [True, False])
def test_what_reads_ahead_does_not_overlap_with_what_wrote(packed, Lq):
    """Attention and selection read codes, scales and bounds before they wait for the kernel in front of them: the
    first call behind a kernel that wrote them starts after it, later ones overlap again."""
    torch = _torch()
    from rfsn_b200 import _native as native
    from rfsn_b200.cache import paged_attention

    cache, k, v = make("bfloat16", 1, 8, 2, 128, (64,) * 20, 10, tile_index=True,
                       archive_dtype="float8_e4m3fn" if packed else None)
    q = queries(1, 8, Lq, 128)
    segs = cache.get_attention_segments()
    ws = native.Workspace(cache.device)

    def attend(top):
        paged_attention(cache, q, 1290 - Lq, segs, workspace=ws, top_tiles=top)

    def write():
        if packed:
            cache.archive.pack(k[:, :, :64], v[:, :, :64], 0, bounds=cache.tile_bounds)
        else:
            cache._ops.tile_bounds(segs.spans[0][0], 64, cache.tile_bounds)

    tops = [3] + [0] * packed
    for top in tops:
        attend(top)  # the workspace is as large as it gets
    cache.select_tiles(q, 1290 - Lq, 3, segs, workspace=ws)
    select = lambda: cache.select_tiles(q, 1290 - Lq, 3, segs, workspace=ws)  # noqa: E731
    assert edge_types(lambda: (attend(3), attend(3))) == [1, 1, 1]  # selection and attention, twice
    assert edge_types(lambda: (write(), attend(3), attend(3))) == [0, 1, 1, 1]
    assert edge_types(lambda: (write(), select(), select())) == [0, 1]
    if packed:
        assert edge_types(lambda: (attend(0), attend(0))) == [1]
        assert edge_types(lambda: (write(), write(), attend(0), attend(0))) == [0, 0, 1]
        assert edge_types(lambda: (write(), attend(0), write(), attend(0), attend(3))) == [0, 0, 0, 1, 1]


def test_a_write_on_another_stream_is_not_forgotten():
    """A call on one stream does not forget what was written on another; writes on several streams stay."""
    torch = _torch()
    from rfsn_b200 import _native as native
    from rfsn_b200.cache import paged_attention

    cache, k, v = make("bfloat16", 1, 8, 2, 128, (64,) * 20, 10)
    q = queries(1, 8, 1, 128)
    segs = cache.get_attention_segments()
    ws = native.Workspace(cache.device)
    attend = lambda: paged_attention(cache, q, 1289, segs, workspace=ws)  # noqa: E731
    write = lambda: cache.archive.pack(k[:, :, :64], v[:, :, :64], 0)  # noqa: E731
    attend()
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (one, two):
        with torch.cuda.stream(s):
            attend()
    torch.cuda.synchronize()
    with torch.cuda.stream(one):
        write()
    torch.cuda.synchronize()
    assert edge_types(lambda: (attend(), attend()), two) == [1]
    assert edge_types(lambda: (write(), attend(), attend()), one) == [0, 1]
    for s in (one, two):
        with torch.cuda.stream(s):
            write()
        torch.cuda.synchronize()
    assert edge_types(lambda: (attend(), attend()), one) == [0]


# ------------------------------------------------------------------ workspaces
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("H,Hkv,Lq", [(32, 8, 4), (8, 2, 1), (16, 1, 2)])
def test_a_selecting_call_over_no_tiles_fits_its_workspace(H, Hkv, Lq, packed):
    """The C call with top_tiles > 0 and an empty list over a long window, in a workspace of the size asked for."""
    import ctypes

    torch = _torch()
    import archive_ref as ref
    from rfsn_b200 import _native as native
    from rfsn_b200.archive import workspace_bytes

    hot = 1 << 14
    cache, k, v = make("bfloat16", 1, H, Hkv, 128, (), hot, hot_cap=hot, tile_index=True,
                       archive_dtype="float8_e4m3fn" if packed else None)
    q = queries(1, H, Lq, 128)
    tiles = torch.zeros(64, 4, dtype=torch.int32, device="cuda")
    call = native.ArchiveCallC(cache.arena.handle, cache.archive.handle if packed else None,
                               cache.tile_bounds.data_ptr(), native.TileListC(tiles.data_ptr(), 0, 0),
                               native.HotWindowC(0, hot, 0, hot, 0, 0, None), 1, H, Hkv, Lq, 4, 0)
    nbytes = workspace_bytes(1, H, Hkv, Lq, 128, hot, 10, 4)
    ws = torch.zeros(nbytes, dtype=torch.uint8, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(1, H, Lq, device="cuda")
    native.check(native.lib().rfsn_archive_attend(ctypes.byref(call), q.data_ptr(), hot - Lq, out.data_ptr(),
                                                  lse.data_ptr(), ws.data_ptr(), nbytes, native.stream_ptr()), "attend")
    want, want_lse = ref.attention(q, k, v, torch.arange(hot), hot - Lq)
    check_out(out, lse, want, want_lse, v)


# ------------------------------------------------------------------ tiles of zeros
def with_values(lens, hot, D, change, Lq, dtype="bfloat16"):
    """A packed cache of 8 / 2 heads whose V went through ``change`` before it was packed, its K and V as held."""
    torch = _torch()
    cache, _, _ = make(dtype, 1, 8, 2, D, (), 0, hot_cap=max(hot, 1), pool_tokens=sum(lens) + 64 * len(lens))
    g = torch.Generator(device="cuda").manual_seed(Lq + D)
    n = sum(lens) + hot
    k, v = (torch.randn(1, 2, n, D, generator=g, device="cuda") for _ in range(2))
    k, v = k.to(cache.dtype), change(v).to(cache.dtype)
    at = 0
    for length in lens:
        cache.import_block(k[:, :, at:at + length], v[:, :, at:at + length], at)
        at += length
    cache.hot_start = at
    if hot:
        cache.append_exact(k[:, :, at:], v[:, :, at:])
    return cache, k, v, *held(cache, k, v, lens)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("level", [1.0, 1e-2, 1e-6, 1e-30])
@pytest.mark.parametrize("zero", [[0], [1], [2, 3], [0, 2, 4, 6, 8], [7], list(range(80)), [81], [82], [80, 81]])
def test_tiles_of_zero_values_do_not_cost_the_others_precision(zero, level, D):
    """Padded tokens: the V of whole tiles is zero, in the archive (tiles 0 to 80) or in the ring (81 and 82). Such a
    tile has a scale of 1, which is no size of its values: with it as the unit, V of 1e-6 would keep a few bits."""
    torch = _torch()
    import archive_ref as ref

    lens = (64,) * 81

    def change(v):
        v = v * level
        for t in zero:
            v[:, :, 64 * t:64 * t + 64] = 0
        return v

    for Lq in (1, 2, 4, 40, 128):  # the decode, rows and chunk kernels
        cache, k, v, kk, vv = with_values(lens, 140, D, change, Lq)
        q = queries(1, 8, Lq, D)
        want, want_lse = ref.attention(q, kk, vv, torch.arange(5324), 5324 - Lq)
        out, lse = cache.attend(q, 5324 - Lq, want_lse=True)
        check_out(out, lse, want, want_lse, vv)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Lq", [1, 4, 128])
@pytest.mark.parametrize("at", [70, 5184 + 70])
def test_nan_among_zero_values_is_seen(at, Lq, D):
    """NaN and infinities in a tile whose other values are zero reach their channel (an infinity is NaN in 8 bits)."""
    torch = _torch()
    lens = (64,) * 81
    for bad in (float("nan"), float("inf")):
        def change(v):
            v[:, :, at // 64 * 64:at // 64 * 64 + 64] = 0
            v[:, :, at, 5] = bad
            return v

        cache, *_ = with_values(lens, 140, D, change, Lq)
        out = cache.attend(queries(1, 8, Lq, D), 5324 - Lq)
        fine = torch.arange(D, device="cuda") != 5
        sees = 5324 - Lq + torch.arange(Lq, device="cuda") >= at
        assert bool(torch.isfinite(out[..., fine]).all()) and not bool(torch.isfinite(out[:, :, sees, 5]).any())


def test_the_mark_of_zero_values():
    """The third entry of a tile's scales: 1 for a V tile packed from zeros, 0 for any other and for K."""
    torch = _torch()
    from rfsn_b200 import PackedArchive

    a = PackedArchive(2, 256, 64)
    assert not a.scales[..., 2:].any() and bool((a.scales[..., :2] == 1).all())
    x = torch.ones(1, 2, 200, 64, device="cuda")
    y = x.clone()
    y[0, 1, 64:128] = 0
    y[0, 0, 192:] = 0
    y[0, 0, 195, 3] = float("nan")
    a.pack(y, x)
    assert not a.scales[..., 2].any()
    a.pack(x, y)
    want = torch.zeros(2, 4)
    want[1, 1] = want[0, 3] = 1
    assert torch.equal(a.scales[..., 2].cpu(), want)
    a.pack(x, x)
    assert not a.scales[..., 2:].any()
    a.pack(x, y)
    a.clear()
    assert not a.scales[..., 2:].any() and bool((a.scales[..., :2] == 1).all())
