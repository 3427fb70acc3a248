"""Packed archives and tile lists without a GPU: the plain forms themselves, the cache's bookkeeping on a host test
double, refusals, and the C ABI's argument checks."""

import ctypes
import math

import numpy as np
import pytest
import torch

import archive_ref as ref
from fake_ops import FakeDeviceOps
from rfsn_b200 import LayerKVCache, RFSNCache, RFSNConfig
from rfsn_b200 import _native as native
from rfsn_b200.archive import kv_rows, padded_rows, workspace_bytes

BAD, UNSUPPORTED, OVERFLOW = native.RFSN_ERR_INVALID_ARG, native.RFSN_ERR_UNSUPPORTED, native.RFSN_ERR_OVERFLOW
FAKE = 0x10000  # a non-NULL, 16-byte aligned address that is never dereferenced


# ------------------------------------------------------------------ the plain forms
def test_reference_rounding_is_the_e4m3_of_every_half_step():
    """Every e4m3 value, the middles between neighbours (ties to even) and their neighbourhoods."""
    codes = torch.arange(0, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    x = torch.cat([codes, mid, mid * (1 + 2.0 ** -30), mid * (1 - 2.0 ** -30)])
    x = torch.cat([x, -x])
    nearest = (x[:, None] - torch.cat([codes, -codes])[None]).abs().argmin(1)  # not for ties
    got = ref.e4m3(x)
    assert torch.equal(got.abs(), got.to(torch.float8_e4m3fn).double().abs())
    both = torch.cat([codes, -codes])
    assert ((got - x).abs() <= (both[nearest] - x).abs()).all()
    ties = ref.e4m3(mid)
    even = codes[(torch.arange(len(mid)) + 1) // 2 * 2]  # of codes i and i + 1 the even one
    assert torch.equal(ties, even)


@pytest.mark.parametrize("amax,scale", [(448.0, 1.0), (448.5, 2.0), (447.0, 1.0), (224.0, 0.5), (225.0, 1.0), (0.0, 1.0),
                                        (1.75, 2.0 ** -8), (2.0, 2.0 ** -7), (1e-45, 2.0 ** -126), (3.3e38, 2.0 ** 120)])
def test_reference_scale(amax, scale):
    assert ref.scale_of(amax) == scale


def test_reference_selection_and_attention_agree_with_dense():
    g = torch.Generator().manual_seed(0)
    lens = [100, 64, 3]
    k, v = (torch.randn(1, 2, 167, 64, generator=g, dtype=torch.float64) for _ in range(2))
    q = torch.randn(1, 4, 2, 64, generator=g, dtype=torch.float64)
    lo, hi, pos = ref.bounds(k, lens)
    assert pos.tolist() == [0, 64, 100, 164]
    tiles = ref.select(q, lo, hi, pos, 165, 4)
    assert tiles.tolist() == [[[[0, 1, 2, 3]] * 2] * 2]
    assert ref.select(q, lo, hi, pos, 98, 4)[0, 0, 1].tolist() == [0, 1, -1, -1]  # row 1 at 99: tile 2 begins at 100
    out, lse = ref.attention(q, k, v, torch.arange(167), 165)
    s = torch.einsum("bhrd,bhnd->bhrn", q, k.repeat_interleave(2, 1)) / 8
    s[:, :, 0, 166] = -math.inf
    assert torch.allclose(out, torch.softmax(s, -1) @ v.repeat_interleave(2, 1))
    assert torch.allclose(lse, torch.logsumexp(s, -1))


# ------------------------------------------------------------------ the cache on a host test double
class FakeArchive:
    def __init__(self, groups, rows, head_dim):
        self.groups, self.rows, self.head_dim = groups, padded_rows(rows), head_dim
        self.k = torch.zeros((groups, self.rows, head_dim), dtype=torch.uint8).view(torch.float8_e4m3fn)
        self.v = torch.zeros((groups, self.rows, head_dim), dtype=torch.uint8).view(torch.float8_e4m3fn)
        self.scales = torch.ones((groups, self.rows // 64, 4))
        self.handle = None

    def clear(self):
        self.k.view(torch.uint8).zero_()
        self.v.view(torch.uint8).zero_()
        self.scales.fill_(1.0)

    def pack(self, k, v, row=0, *, bounds=None):
        assert row % 64 == 0 and row + k.shape[2] <= self.rows
        n = k.shape[2]
        for dst, x, w in ((self.k, k, 0), (self.v, v, 1)):
            _, scales, codes = ref.pack(x.reshape(self.groups, n, self.head_dim))
            dst.view(torch.uint8)[:, row:row + padded_rows(n)] = 0
            dst.view(torch.uint8)[:, row:row + n] = codes.to(torch.float8_e4m3fn).view(torch.uint8)
            self.scales[:, row // 64:row // 64 + scales.shape[1], w] = scales.float()

    def pack_ring(self, k, v, offset, wrap, row, count, *, bounds=None):
        at = (offset + torch.arange(count)) % wrap
        self.pack(k[None][:, :, at], v[None][:, :, at], row, bounds=bounds)

    def unpack(self, row, n, dtype, *, out=None):
        s = self.scales.repeat_interleave(64, dim=1)[:, row:row + n]
        return ((self.k[:, row:row + n].float() * s[..., :1]).to(dtype),
                (self.v[:, row:row + n].float() * s[..., 1:2]).to(dtype))


class FakeOps(FakeDeviceOps):
    def new_archive(self, groups, rows, head_dim):
        self.archives = getattr(self, "archives", 0) + 1
        return FakeArchive(groups, rows, head_dim)

    def tile_bounds(self, row, count, bounds):
        assert row % 64 == 0
        self.calls.append(("tile_bounds", row, count))
        for t in range((count + 63) // 64):
            part = self.k[:, row + 64 * t:row + min(count, 64 * t + 64)]
            bounds[:, row // 64 + t, 0], bounds[:, row // 64 + t, 1] = part.amin(1), part.amax(1)


def config(tmp_path, **kw):
    base = dict(hidden_dim=4 * 64, num_heads=4, num_kv_heads=2, head_dim=64, num_layers=1, hot_capacity=100,
                warm_capacity=1000, cold_capacity=4000, block_size_seq=37, model_dtype="bfloat16",
                disk_cache_dir=str(tmp_path))
    base.update(kw)
    return RFSNConfig(**base)


def layer(tmp_path, *, packed=True, tile_index=False, pool_tokens=None, host_tier=False, **kw):
    return LayerKVCache(config(tmp_path, **kw), 1, 4, 2, session_id="s", ops=FakeOps(), pool_tokens=pool_tokens,
                        archive_dtype="float8_e4m3fn" if packed else None, tile_index=tile_index, host_tier=host_tier)


def tokens(n, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(1, 2, n, 64, generator=g).to(dtype)


def expect_tiles(cache):
    """The tile list against the page table, and the rows' alignment and disjointness."""
    segs = cache.get_attention_segments()
    want, used = [], set()
    for row, start, n in segs.spans[:segs.n_archived]:
        assert row % 64 == 0
        rows = set(range(row, row + padded_rows(n)))
        assert not rows & used
        used |= rows
        want += [[row + o, start + o, min(64, n - o), len(want) + o // 64] for o in range(0, n, 64)]
    want = [[r, p, n, i] for i, (r, p, n, _) in enumerate(want)]
    dev, n = segs.tile_list
    assert n == len(want) and dev[:n].tolist() == want
    limit = cache.archive.rows if cache.archive is not None else cache._arena_k.shape[1]
    first = 0 if cache.archive is not None else padded_rows(cache.config.hot_capacity)
    assert all(first <= r < limit for r in used)
    return segs


@pytest.mark.parametrize("packed", [True, False])
def test_seals_own_whole_tiles_and_the_tile_list_follows_the_page_table(tmp_path, packed):
    cache = layer(tmp_path, packed=packed, tile_index=True, pool_tokens=192)  # grows on the way
    k = tokens(700)
    at = 0
    for n in (100, 1, 1, 30, 100, 64, 99, 5, 100, 100, 100):
        cache.evict_for_append(n)
        cache.append_exact(k[:, :, at:at + n], -k[:, :, at:at + n])
        at += n
        expect_tiles(cache)
    segs = expect_tiles(cache)
    for kk, vv, start in list(segs)[:segs.n_archived]:
        part = k[:, :, start:start + kk.shape[2]]
        if packed:
            values = ref.pack(part[0])[0]
            assert torch.equal(kk[0].double(), values) and torch.equal(vv[0].double(), -values)
        else:
            assert torch.equal(kk, part) and torch.equal(vv, -part)
    hot = torch.cat([s[0] for s in list(segs)[segs.n_archived:]], dim=2)
    assert torch.equal(hot, k[:, :, cache.hot_start:at])
    if packed:
        assert cache._arena_k.shape[1] == 100  # the ring alone
    else:  # the bounds of every block were taken where it lies
        taken = [c for c in cache._ops.calls if c[0] == "tile_bounds"]
        assert len(taken) == segs.n_archived
        for row, start, n in segs.spans[:segs.n_archived]:
            lo, hi, _ = ref.bounds(k[:, :, start:start + n], [n])
            b = cache.tile_bounds[:, row // 64:row // 64 + lo.shape[2]].double()
            assert torch.equal(b[:, :, 0], lo[0]) and torch.equal(b[:, :, 1], hi[0])


def test_the_seal_rule_and_the_page_table_do_not_depend_on_the_archive(tmp_path):
    caches = [LayerKVCache(config(tmp_path / str(i)), 1, 4, 2, session_id="s", ops=FakeOps(), **kw)
              for i, kw in enumerate([{}, dict(archive_dtype="float8_e4m3fn"), dict(tile_index=True),
                                      dict(archive_dtype="float8_e4m3fn", top_tiles=3)])]
    rng = np.random.default_rng(0)
    at = 0
    for _ in range(25):
        n = int(rng.integers(1, 60))
        k = tokens(n, at)
        spans = []
        for c in caches:
            c.evict_for_append(n)
            c.append_exact(k, k)
            segs = c.get_attention_segments()
            spans.append([(s, m) for _, s, m in segs.spans] + [segs.hot_state, c.get_total_length()])
        at += n
        assert all(s == spans[0] for s in spans)


@pytest.mark.parametrize("host_tier", [False, True])
def test_demoted_blocks_return_with_the_same_values(tmp_path, host_tier):
    if host_tier:
        pytest.skip("pinned memory needs a GPU")
    cache = layer(tmp_path, pool_tokens=640)
    k = tokens(300)
    for i in range(3):
        cache.import_block(k[:, :, 100 * i:100 * i + 100], -k[:, :, 100 * i:100 * i + 100], 100 * i)
    before = [(a.clone(), b.clone()) for a, b, _ in cache.get_archived_attention_segments()]
    rows = dict(cache._resident_rows)
    for m in list(cache.block_manager.iter_blocks(layer_id=0))[:2]:
        cache.demote_manifest_to_cold(m)
    cache._flush_deferred_free()
    assert cache._alloc.allocate(128) is not None  # one freed range is taken: the blocks come back elsewhere
    cache.archive.clear()
    for m in list(cache.block_manager.iter_blocks(layer_id=0))[2:]:
        cache.archive.pack(k[:, :, 200:], -k[:, :, 200:], rows[m.block_id])
    after = list(expect_tiles(cache))
    for (a, b), (c, d, _) in zip(before, after):
        assert torch.equal(a, c) and torch.equal(b, d)


def test_session_restore_through_a_packed_cache(tmp_path):
    cache = layer(tmp_path)
    k = tokens(130)
    cache.import_block(k, -k, 0)
    cache.demote_manifest_to_cold(next(iter(cache.block_manager.iter_blocks(layer_id=0))))
    fresh = layer(tmp_path)
    fresh.restore_from_disk()
    kk, vv, start = fresh.get_archived_attention_segments()[0]
    values = ref.pack(k[0])[0]
    assert start == 0 and torch.equal(kk[0].double(), values) and torch.equal(vv[0].double(), -values)
    # the session also restores into an exact cache, which then holds the 8-bit values
    exact = layer(tmp_path, packed=False)
    exact.restore_from_disk()
    assert torch.equal(exact.get_archived_attention_segments()[0][0][0].double(), values)


def test_reset_empties_a_packed_cache(tmp_path):
    cache = layer(tmp_path, tile_index=True)
    cache.import_block(tokens(70), tokens(70), 0)
    assert cache.get_attention_segments().tile_list[1] == 2
    cache.reset()
    assert cache.get_attention_segments().tile_list[1] == 0 and len(cache.get_attention_segments()) == 0
    assert not cache.archive.k.view(torch.uint8).any()
    cache.import_block(tokens(64), tokens(64), 0)
    assert expect_tiles(cache).tile_list[1] == 1


def test_capture_key_changes_with_what_a_graph_holds(tmp_path):
    cache = layer(tmp_path, tile_index=True, pool_tokens=64)
    keys = {cache.capture_key()}
    cache.import_block(tokens(64), tokens(64), 0)
    cache.get_attention_segments()
    keys.add(cache.capture_key())
    cache.import_block(tokens(64), tokens(64), 64)  # the archive grows
    cache.get_attention_segments()
    keys.add(cache.capture_key())
    assert len(keys) == 3
    assert LayerKVCache(config(tmp_path), 1, 4, 2, session_id="s", ops=FakeOps()).capture_key() == ()


# ------------------------------------------------------------------ refusals
@pytest.mark.parametrize("kw,message", [
    (dict(archive_dtype="int8"), "archive_dtype"),
    (dict(archive_dtype="float8_e5m2"), "archive_dtype"),
    (dict(top_tiles=-1), "top_tiles"),
])
def test_unknown_options_are_refused(tmp_path, kw, message):
    with pytest.raises(ValueError, match=message):
        LayerKVCache(config(tmp_path), 1, 4, 2, session_id="s", ops=FakeOps(), **kw)
    with pytest.raises(ValueError, match=message):
        RFSNCache(config(tmp_path), 1, session_id="s", ops_factory=FakeOps, **kw)


@pytest.mark.parametrize("kw", [dict(archive_dtype="float8_e4m3fn"), dict(tile_index=True), dict(top_tiles=4)])
@pytest.mark.parametrize("cfg", [dict(model_dtype="float32"), dict(head_dim=32, hidden_dim=128),
                                 dict(head_dim=96, hidden_dim=384)])
def test_shapes_without_kernels_are_refused_at_construction(tmp_path, kw, cfg):
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        LayerKVCache(config(tmp_path, **cfg), 1, 4, 2, session_id="s", ops=FakeOps(), **kw)


def test_cli_passes_the_archive_options(monkeypatch):
    from rfsn_b200 import __main__ as cli

    args = cli.build_parser().parse_args(["bench", "--archive-dtype", "float8_e4m3fn", "--top-tiles", "32"])
    assert args.archive_dtype == "float8_e4m3fn" and args.top_tiles == 32
    args = cli.build_parser().parse_args(["bench"])
    assert args.archive_dtype == "" and args.top_tiles == 0
    with pytest.raises(SystemExit):
        cli.build_parser().parse_args(["bench", "--archive-dtype", "int8"])


# ------------------------------------------------------------------ C ABI
@pytest.fixture(scope="module")
def lib():
    return native.load_library()


def expect(status, code, fragment):
    assert status == code, (status, native.last_error())
    assert fragment in native.last_error()


def test_struct_layouts_match_header():
    assert ctypes.sizeof(native.KvRowsC) == 80
    k, v = torch.zeros(2, 3, 5, 64).transpose(1, 2), torch.ones(2, 5, 3, 64)
    rows = native.KvRowsC.from_buffer_copy(kv_rows(k, v, 4, 9))
    assert [getattr(rows, f) for f, _ in rows._fields_] == [k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3],
                                                            native.dtype_code(torch.float32), 5, 4, 9]
    assert ctypes.sizeof(native.TileListC) == 16
    assert ctypes.sizeof(native.ArchiveCallC) == 96


def test_archive_arguments(lib):
    out = ctypes.c_void_p()
    create = lib.rfsn_packed_archive_create
    expect(create(FAKE, FAKE, FAKE, 8, 64, 128, None), BAD, "out is NULL")
    expect(create(None, FAKE, FAKE, 8, 64, 128, ctypes.byref(out)), BAD, "NULL pointer")
    expect(create(FAKE + 4, FAKE, FAKE, 8, 64, 128, ctypes.byref(out)), BAD, "aligned")
    expect(create(FAKE, FAKE, FAKE + 8, 8, 64, 128, ctypes.byref(out)), BAD, "aligned")
    expect(create(FAKE, FAKE, FAKE, 8, 65, 128, ctypes.byref(out)), BAD, "multiple of 64")
    expect(create(FAKE, FAKE, FAKE, 0, 64, 128, ctypes.byref(out)), BAD, "batch_kv_heads")
    expect(create(FAKE, FAKE, FAKE, 65536, 64, 128, ctypes.byref(out)), BAD, "batch_kv_heads")
    expect(create(FAKE, FAKE, FAKE, 32768, 65536, 128, ctypes.byref(out)), BAD, "2^31")
    expect(create(FAKE, FAKE, FAKE, 8, 64, 96, ctypes.byref(out)), UNSUPPORTED, "head_dim 96")
    assert out.value is None
    assert lib.rfsn_packed_archive_destroy(None) == native.RFSN_OK
    rows = native.KvRowsC()
    expect(lib.rfsn_pack_rows(None, 0, ctypes.byref(rows), 1, None, None), BAD, "NULL archive")
    expect(lib.rfsn_unpack_rows(None, 0, 1, FAKE, FAKE, native.RFSN_F32, 64, None), BAD, "NULL archive")
    expect(lib.rfsn_tile_bounds(None, 0, 1, FAKE, None), BAD, "NULL")


def select(lib, *, bounds=FAKE, dtype=native.RFSN_BF16, scales=None, rows=640, q=FAKE, shape=(1, 8, 2, 1, 128),
           tiles=(FAKE, 10, 0), n=4, out=FAKE, ws=FAKE, nbytes=1 << 20):
    t = native.TileListC(*tiles)
    return lib.rfsn_select_tiles(bounds, dtype, scales, rows, q, *shape, 100, ctypes.byref(t), n, out, None, ws, nbytes,
                                 None)


def test_selection_arguments(lib):
    expect(select(lib, bounds=None), BAD, "bounds")
    expect(select(lib, bounds=FAKE + 2), BAD, "bounds")
    expect(select(lib, dtype=native.RFSN_F32), BAD, "f16, bf16 or e4m3")
    expect(select(lib, dtype=native.RFSN_E4M3), BAD, "scales")
    expect(select(lib, rows=100), BAD, "multiple of 64")
    expect(select(lib, q=None), BAD, "NULL")
    expect(select(lib, q=FAKE + 8), BAD, "misaligned")
    expect(select(lib, out=FAKE + 8), BAD, "misaligned")
    expect(select(lib, shape=(1, 7, 2, 1, 128)), BAD, "divisible")
    expect(select(lib, shape=(1, 8, 2, 0, 128)), BAD, "non-positive")
    expect(select(lib, shape=(1, 8, 2, 1, 80)), UNSUPPORTED, "head_dim 80")
    expect(select(lib, shape=(1, 8, 2, 40000, 128)), BAD, "tile lists")
    expect(select(lib, tiles=(None, 10, 0)), BAD, "tile list")
    expect(select(lib, tiles=(FAKE, -1, 0)), BAD, "tile list")
    expect(select(lib, tiles=(FAKE, 10, 1)), BAD, "one list")
    expect(select(lib, n=0), BAD, "n_select")
    expect(select(lib, nbytes=1000), OVERFLOW, "workspace too small")


def test_attention_arguments(lib):
    hot, tiles = native.HotWindowC(0, 64, 0, 10, 100), native.TileListC(FAKE, 2, 0)
    expect(lib.rfsn_archive_attention(None, None, FAKE, 1, 8, 2, 1, 0, ctypes.byref(tiles), ctypes.byref(hot), FAKE, None,
                                      FAKE, 1 << 20, 0, None), BAD, "NULL arena")
    expect(lib.rfsn_archive_attend(None, FAKE, 0, FAKE, None, FAKE, 1 << 20, None), BAD, "NULL call")
    expect(lib.rfsn_archive_select(None, FAKE, 0, FAKE, FAKE, 1 << 20, None), BAD, "NULL call")
    call = native.ArchiveCallC()
    expect(lib.rfsn_archive_select(ctypes.byref(call), FAKE, 0, FAKE, FAKE, 1 << 20, None), BAD, "NULL call")
    expect(lib.rfsn_archive_attend(ctypes.byref(call), FAKE, 0, FAKE, None, FAKE, 1 << 20, None), BAD, "NULL call")


def test_workspace_size(lib):
    small = workspace_bytes(1, 32, 8, 1, 128, 4096, 2000)
    assert 65536 < small < 2 << 20
    # selected lists and scores come on top
    assert workspace_bytes(1, 32, 8, 1, 128, 4096, 2000, 128) >= small + 8 * 128 * 16
    assert workspace_bytes(1, 32, 8, 1, 128, 4096, 200000, 128) >= 8 * 200000 * 4
    # a chunk: partials of four parts per SM and the float16 copy of the ring
    assert workspace_bytes(1, 32, 8, 512, 128, 4096, 2000) >= 4 * 148 * 128 * 128 * 4 + 2 * 8 * 4096 * 128 * 2
    assert workspace_bytes(1, 32, 8, 512, 64, 4096, 2000) < 64 << 20  # head_dim 64 has no such kernel
    for bad in ((1, 30, 8, 1, 128, 64, 1), (0, 8, 8, 1, 128, 64, 1), (1, 8, 8, 1, 128, 64, -1), (1, 8, 8, 1, 128, -1, 1)):
        with pytest.raises(ValueError):
            workspace_bytes(*bad)
    with pytest.raises(NotImplementedError):
        workspace_bytes(1, 8, 8, 1, 96, 64, 1)
