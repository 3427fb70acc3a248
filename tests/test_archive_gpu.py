"""Packed archives, tile selection and attention over tiles on the GPU, against plain 64-bit forms.

Tolerance of the attention outputs, by arithmetic: a logit is a sum of D / 16 tensor-core steps of products that carry
at least 22 significant bits of q (K enters exactly), so its error is below (D / 16 + 4) 2^-23 sum |q_d k_d| / sqrt(D).
With |q_d k_d| summing to at most ~2 D for N(0, 1) data (checked below through the data itself) that is 12 * 2^-23 * 2
* sqrt(128) < 2^-15 for D = 128; the probabilities get that relative error twice (p and its sum), the split of p 2^-21,
the exponentials 2^-22, and the sums over a split's keys at most N / 64 steps of 2^-23 each (N <= 2^14 here: 2^-15).
Together below 2^-13 of the largest |v|.
"""

import math
import tempfile

import pytest

pytestmark = pytest.mark.gpu
REL = 2.0 ** -13


def _torch():
    import torch

    return torch


def make(dtype="bfloat16", B=1, H=8, Hkv=2, D=128, lens=(100, 64, 1), hot=50, hot_cap=None, wrap=0, seed=0,
         archive_dtype="float8_e4m3fn", tile_index=False, top_tiles=0, scale=1.0, v_scale=1.0, **kw):
    """A layer cache with the given archived blocks and ``hot`` ring tokens (the ring's oldest at slot ``wrap``), and
    its keys and values [B, Hkv, N + hot, D]."""
    torch = _torch()
    from rfsn_b200 import LayerKVCache, RFSNConfig

    g = torch.Generator(device="cuda").manual_seed(seed)
    n, cap = sum(lens) + hot, hot_cap or max(hot + wrap, 1)
    room = max(cap, sum(lens), 1)
    cfg = RFSNConfig(hidden_dim=H * D, num_heads=H, num_kv_heads=Hkv, head_dim=D, num_layers=1, hot_capacity=cap,
                     warm_capacity=room, cold_capacity=room, block_size_seq=min(64, cap), model_dtype=dtype,
                     disk_cache_dir=tempfile.mkdtemp(prefix="rfsn_archive_"))
    cache = LayerKVCache(cfg, B, H, Hkv, session_id="t", archive_dtype=archive_dtype, tile_index=tile_index,
                         top_tiles=top_tiles, **kw)
    k = (torch.randn(B, Hkv, n, D, generator=g, device="cuda") * scale).to(cache.dtype)
    v = (torch.randn(B, Hkv, n, D, generator=g, device="cuda") * v_scale).to(cache.dtype)
    at = 0
    for length in lens:
        cache.import_block(k[:, :, at:at + length], v[:, :, at:at + length], at)
        at += length
    cache.hot_start, cache.hot_head_index = at, wrap % cap
    if hot:
        cache.append_exact(k[:, :, at:], v[:, :, at:])
    return cache, k, v


def held(cache, k, v, lens):
    """The keys and values as the cache holds them (float64), from the plain form of packing."""
    torch = _torch()
    import archive_ref as ref

    out = []
    for x in (k, v):
        x = x.double().cpu()
        if cache.archive is not None:
            B, Hkv, n, D = x.shape
            at = 0
            for length in lens:
                part = ref.pack(x[:, :, at:at + length].reshape(B * Hkv, length, D))[0]
                x[:, :, at:at + length] = part.reshape(B, Hkv, length, D)
                at += length
        out.append(x)
    return out


def same(a, b):
    """Equal values, NaN where the other has NaN (fp16 input of the packing tests overflows to infinity in places)."""
    torch = _torch()
    return a.shape == b.shape and torch.allclose(a.double(), b.double(), rtol=0, atol=0, equal_nan=True)


def queries(B, H, Lq, D, seed=7, scale=1.0):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(B, H, Lq, D, generator=g, device="cuda") * scale


def check_out(out, lse, want, want_lse, v):
    torch = _torch()
    tol = REL * float(v.abs().max())
    err = float((out.double().cpu() - want).abs().max())
    assert err <= tol
    if lse is not None:
        got, fine = lse.double().cpu(), torch.isfinite(want_lse)
        assert torch.equal(torch.isfinite(got), fine)
        assert float((got - want_lse)[fine].abs().max() if fine.any() else 0.0) <= REL * 4


# ------------------------------------------------------------------ packing
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,row", [(1, 0), (64, 64), (65, 128), (300, 0)])
def test_pack_gives_the_codes_scales_and_bounds_of_the_formula(dtype, D, n, row):
    torch = _torch()
    import archive_ref as ref
    from rfsn_b200 import PackedArchive

    g = torch.Generator().manual_seed(n + D)
    x = [torch.randn(2, 3, n, D, generator=g) * torch.exp(3 * torch.randn(2, 3, n, 1, generator=g)) for _ in range(2)]
    x = [t.to(getattr(torch, dtype)) for t in x]
    x[0][0, 0, 0, 0] = 0.0
    x[0][1, 1] = 0.0  # a tile of zeros
    a = PackedArchive(6, 512, D)
    a.k.view(torch.uint8).fill_(0x7f)  # NaN codes: what is not written stays, what belongs to the block is overwritten
    a.v.view(torch.uint8).fill_(0x7f)
    bounds = torch.zeros(6, 8, 2, D, dtype=torch.uint8, device="cuda")
    # token-major memory: [B, n, Hkv, D] seen as [B, Hkv, n, D]
    kv = [t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in x]
    a.pack(kv[0], kv[1], row, bounds=bounds)
    end = (n + 63) // 64 * 64
    for t, got, scale in ((x[0], a.k, a.k_scale), (x[1], a.v, a.v_scale)):
        values, scales, codes = ref.pack(t.reshape(6, n, D))
        assert same(scale[:, row // 64:(row + end) // 64].double().cpu(), scales)
        assert same(got[:, row:row + n].double().cpu(), codes)
        assert (got[:, row + n:row + end].view(torch.uint8) == 0).all()
        assert (got[:, row + end:].view(torch.uint8) == 0x7f).all() and (got[:, :row].view(torch.uint8) == 0x7f).all()
        if t is x[0]:
            lo, hi, _ = ref.bounds(codes.reshape(2, 3, n, D), [n])
            b = bounds[:, row // 64:(row + end) // 64].view(torch.float8_e4m3fn).double().cpu()
            assert same(b[:, :, 0], lo.reshape(6, -1, D)) and same(b[:, :, 1], hi.reshape(6, -1, D))
    for out_dtype in (torch.float32, torch.bfloat16, torch.float16):
        k, v = a.unpack(row, n, out_dtype)
        top = torch.finfo(out_dtype).max  # finite values saturate
        assert same(k.cpu(), ref.pack(x[0].reshape(6, n, D))[0].clamp(-top, top).to(out_dtype))
        assert same(v.cpu(), ref.pack(x[1].reshape(6, n, D))[0].clamp(-top, top).to(out_dtype))


def test_pack_of_unpacked_values_changes_nothing():
    torch = _torch()
    from rfsn_b200 import PackedArchive

    x = (torch.randn(1, 2, 640, 128, device="cuda") * 3).to(torch.bfloat16)
    a, b = PackedArchive(2, 640, 128), PackedArchive(2, 640, 128)
    a.pack(x, -x)
    k, v = a.unpack(0, 640, torch.bfloat16)
    b.pack(k[None], v[None])
    k2, v2 = b.unpack(0, 640, torch.bfloat16)
    assert torch.equal(k, k2) and torch.equal(v, v2)


def test_pack_extremes():
    """NaN stays, infinities become NaN and do not count for the scale; the smallest and largest magnitudes of each
    type; a maximum that just reaches the next scale."""
    torch = _torch()
    import archive_ref as ref
    from rfsn_b200 import PackedArchive

    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        info = torch.finfo(dtype)
        x = torch.zeros(1, 8, 64, 64)
        x[0, 0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 2.0])
        x[0, 1, 3, 5] = info.max
        x[0, 2, 3, 5] = info.smallest_normal
        x[0, 3, 3, :2] = torch.tensor([448.0, -1.0])
        x[0, 4, 3, :2] = torch.tensor([449.0 if dtype == torch.float32 else 452.0, 2.0 ** -9])
        x[0, 5, :, :] = math.inf
        x[0, 6, 9, 9] = 1.75
        x[0, 7, 9, 9] = 1.75 + 4 * info.eps
        x = x.to(dtype)
        a = PackedArchive(8, 64, 64)
        a.pack(x.cuda(), x.cuda())
        values, scales, codes = ref.pack(x[0])
        assert torch.equal(a.k_scale.double().cpu(), scales), dtype
        got = a.v.double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(codes)) and torch.equal(got.nan_to_num(), codes.nan_to_num())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("head,count", [(0, 40), (90, 70), (60, 100)])
def test_seal_of_a_wrapped_ring_packs_its_oldest_tokens(dtype, head, count):
    torch = _torch()
    import archive_ref as ref

    cache, k, v = make(dtype, lens=(), hot=100, hot_cap=100, wrap=head)
    cache._seal_hot_prefix(count)
    want = ref.pack(k[0, :, :count])[0]
    got = cache.get_archived_attention_segments()[0]
    assert torch.equal(got[0][0].double().cpu(), want) and got[2] == 0
    assert cache.hot_seq_len == 100 - count


# ------------------------------------------------------------------ attention
CASES = [
    # dtype, B, H, Hkv, D, lens, hot, wrap, Lq
    ("bfloat16", 1, 32, 8, 128, (256,) * 5, 200, 0, 1),
    ("float16", 1, 32, 8, 128, (256,) * 5, 200, 100, 1),
    ("bfloat16", 1, 8, 8, 64, (65, 1, 64, 130), 3, 2, 1),
    ("float16", 2, 8, 2, 64, (1000, 37), 129, 60, 3),
    ("bfloat16", 2, 12, 4, 128, (63, 64, 65), 33, 30, 5),
    ("bfloat16", 1, 16, 1, 128, (700,), 1, 0, 2),      # 32 slots of one KV head
    ("float16", 1, 6, 2, 128, (), 100, 40, 1),         # nothing archived
    ("bfloat16", 1, 4, 4, 128, (900, 130), 0, 0, 1),   # nothing hot
    ("float16", 3, 4, 2, 64, (1,), 1, 0, 1),
    # chunks of 64 query slots and more: the tcgen05 kernel
    ("bfloat16", 1, 32, 8, 128, (512,) * 20 + (77,), 500, 400, 20),
    ("float16", 1, 32, 8, 128, (512, 33), 256, 0, 200),
    ("bfloat16", 2, 6, 2, 128, (64, 1, 130), 100, 33, 41),            # 3 heads per KV head: 126 of 128 rows used
    ("bfloat16", 1, 4, 4, 128, (70,), 128, 100, 128),                 # no GQA
    ("float16", 1, 32, 1, 128, (1, 63), 1, 0, 2),                     # 32 heads per KV head
    ("bfloat16", 1, 8, 8, 128, (100,) * 3, 0, 0, 70),                 # nothing hot
    ("bfloat16", 1, 16, 2, 128, (900,) * 9, 2000, 700, 16),           # few units: the keys are split
    ("bfloat16", 1, 8, 4, 64, (300,), 64, 0, 50),
]


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dtype,B,H,Hkv,D,lens,hot,wrap,Lq", CASES)
def test_attention_over_the_archive_and_the_ring(dtype, B, H, Hkv, D, lens, hot, wrap, Lq, packed):
    torch = _torch()
    import archive_ref as ref

    cache, k, v = make(dtype, B, H, Hkv, D, lens, hot, wrap=wrap, hot_cap=max(1, hot), seed=Lq,
                       archive_dtype="float8_e4m3fn" if packed else None, tile_index=not packed)
    n = sum(lens) + hot
    q = queries(B, H, Lq, D)
    kk, vv = held(cache, k, v, lens)
    want, want_lse = ref.attention(q, kk, vv, torch.arange(n), n - Lq)
    if packed:
        out, lse = cache.attend(q, n - Lq, want_lse=True)
        check_out(out, lse, want, want_lse, vv)
    elif Lq <= 64:  # every tile selected: the exact archive through the tile kernel
        out, lse = cache.attend(q, n - Lq, want_lse=True, top_tiles=len(ref.tiles_of(lens)) + 3)
        check_out(out, lse, want, want_lse, vv)
    if packed and 0 < len(lens):  # any split count gives the same softmax
        for splits in (1, 3):
            out, lse = cache.attend(q, n - Lq, want_lse=True, max_splits=splits)
            check_out(out, lse, want, want_lse, vv)


@pytest.mark.parametrize("Lq", [3, 40])  # one and several passes of the rows kernel
@pytest.mark.parametrize("q_pos", [-1, 0, 63, 64, 100, 250])
def test_queries_among_the_keys_see_the_earlier_ones_only(q_pos, Lq):
    """Positions inside the archive mask part of a tile, whole tiles and the ring; a row before every key gives zeros
    and -inf."""
    torch = _torch()
    import archive_ref as ref

    lens = (100, 90)
    cache, k, v = make("float16", 1, 8, 2, 128, lens, 60)
    q = queries(1, 8, Lq, 128)
    kk, vv = held(cache, k, v, lens)
    want, want_lse = ref.attention(q, kk, vv, torch.arange(250), q_pos)
    out, lse = cache.attend(q, q_pos, want_lse=True)
    check_out(out, lse, want, want_lse, vv)
    if q_pos == -1:
        assert float(out[:, :, 0].abs().max()) == 0.0 and bool((lse[:, :, 0] == -math.inf).all())


@pytest.mark.parametrize("Lq", [1, 40])
def test_what_is_masked_or_behind_the_ends_does_not_reach_the_result(Lq):
    """NaN and infinity in ring slots outside the live window, in the tile rows behind a block's end (other than the
    zero codes that packing writes) and in keys after the query."""
    torch = _torch()

    lens = (70,)
    cache, k, v = make("bfloat16", 1, 4, 2, 128, lens, 40, hot_cap=100, wrap=30)
    q = queries(1, 4, Lq, 128)
    last = 110 - Lq
    want = cache.attend(q, last).clone()
    cache._arena_k[:, :30] = math.nan
    cache._arena_v[:, :30] = math.nan
    cache._arena_k[:, 70:] = math.inf
    cache._arena_v[:, 70:] = math.nan
    assert torch.equal(cache.attend(q, last), want)
    early = 60 - Lq  # queries inside the archive: the ring lies behind them
    before = cache.attend(q, early).clone()
    cache._arena_k[:, 30:70] = math.nan
    assert torch.equal(cache.attend(q, early), before)


@pytest.mark.parametrize("Lq", [1, 40])
def test_nan_keys_and_values_that_are_seen_reach_the_result(Lq):
    torch = _torch()
    cache, k, v = make("float16", 1, 4, 2, 128, (70, 64), 40)
    q = queries(1, 4, Lq, 128)
    row = cache.get_attention_segments().spans[0][0]
    kn, vn = k[:, :, :70].clone(), v[:, :, :70].clone()
    kn[0, 1, 3, 5] = math.inf  # packed as NaN: every row of KV head 1
    vn[0, 0, 4, 7] = math.nan  # channel 7 of KV head 0
    cache.archive.pack(kn, vn, row)
    out = cache.attend(q, 174 - Lq)
    assert bool(torch.isnan(out[0, 2:]).all())
    fine = torch.ones(128, dtype=torch.bool, device="cuda")
    fine[7] = False
    assert bool(torch.isfinite(out[0, :2][..., fine]).all()) and bool(torch.isnan(out[0, :2, :, 7]).all())


def test_values_of_very_different_size_and_large_logits():
    """V scales from 2^-20 to 2^12 from tile to tile, and logits of some hundreds."""
    torch = _torch()
    import archive_ref as ref
    from rfsn_b200 import LayerKVCache  # noqa: F401

    lens = (64,) * 12
    cache, k, v = make("bfloat16", 1, 4, 1, 128, (), 0, hot_cap=8)
    g = torch.Generator(device="cuda").manual_seed(3)
    k = (torch.randn(1, 1, 768, 128, generator=g, device="cuda")).to(torch.bfloat16)
    level = torch.exp2(torch.tensor([-8, 0, 12, -20, 3, 3, -9, 12, -1, 0, 5, 2.0], device="cuda"))
    v = (torch.randn(1, 1, 768, 128, generator=g, device="cuda") * level.repeat_interleave(64)[:, None]).to(torch.bfloat16)
    for i in range(12):
        cache.import_block(k[:, :, 64 * i:64 * i + 64], v[:, :, 64 * i:64 * i + 64], 64 * i)
    kk, vv = held(cache, k, v, lens)
    for scale, Lq in ((1.0, 1), (60.0, 1), (1e-30, 1), (0.0, 1), (1.0, 20), (60.0, 20), (0.0, 20)):
        q = queries(1, 4, Lq, 128, scale=scale)
        want, want_lse = ref.attention(q, kk, vv, torch.arange(768), 768 - Lq)
        out, lse = cache.attend(q, 768 - Lq, want_lse=True)
        # logits of `scale` times the usual size carry that many times the error
        tol = REL * max(1.0, scale) * float(vv.abs().max())
        assert float((out.double().cpu() - want).abs().max()) <= tol
        assert float((lse.double().cpu() - want_lse).abs().max()) <= REL * 4 * max(1.0, scale)


# ------------------------------------------------------------------ selection
SELECT = [
    # dtype, packed, B, H, Hkv, D, lens, hot, Lq, top
    ("bfloat16", False, 1, 32, 8, 128, (256,) * 6, 100, 1, 5),
    ("float16", False, 2, 8, 2, 64, (65, 1, 200), 10, 3, 2),
    ("bfloat16", True, 1, 32, 8, 128, (1000,) * 4 + (24,), 70, 1, 16),
    ("float16", True, 2, 4, 4, 64, (130, 64), 5, 2, 100),   # more than there are
    ("bfloat16", False, 1, 32, 1, 128, (500,), 3, 4, 3),     # 32 heads of one KV head
    ("bfloat16", True, 1, 4, 2, 128, (1,), 1, 1, 1),
    ("bfloat16", False, 1, 4, 2, 128, (64,) * 300, 1, 1, 37),
    ("float16", False, 1, 10, 2, 64, (64,) * 70, 1, 2, 9),   # head groups side by side: 5, 12, 24 and 40 q heads each
    ("bfloat16", True, 1, 24, 2, 128, (640, 33, 64), 7, 1, 5),
    ("bfloat16", False, 2, 24, 1, 64, (1000, 20), 7, 1, 6),
    ("bfloat16", True, 1, 40, 1, 128, (64,) * 40, 1, 3, 12),
]


@pytest.mark.parametrize("dtype,packed,B,H,Hkv,D,lens,hot,Lq,top", SELECT)
def test_selected_tiles_and_the_attention_over_them(dtype, packed, B, H, Hkv, D, lens, hot, Lq, top):
    torch = _torch()
    import archive_ref as ref

    cache, k, v = make(dtype, B, H, Hkv, D, lens, hot, seed=top, tile_index=True,
                       archive_dtype="float8_e4m3fn" if packed else None)
    N = sum(lens)
    n = N + hot
    q = queries(B, H, Lq, D, seed=top)
    kk, vv = held(cache, k, v, lens)
    lo, hi, pos = ref.bounds(kk[:, :, :N], lens)
    for q_pos in (n - Lq, N // 2):
        want = ref.select(q, lo, hi, pos, q_pos, top)
        got = cache.select_tiles(q, q_pos, top)
        assert got.dtype == torch.int32 and torch.equal(got.cpu().long(), want)
        tile_of = torch.cat([torch.full((c,), i) for i, (_, _, c) in enumerate(ref.tiles_of(lens))])
        T = len(ref.tiles_of(lens))
        chosen = torch.zeros(B, Hkv, Lq, T + 1, dtype=torch.bool).scatter(3, torch.where(want < 0, T, want), True)
        seen = torch.cat([chosen[..., tile_of], torch.ones(B, Hkv, Lq, hot, dtype=torch.bool)], 3)
        ref_out, ref_lse = ref.attention(q, kk, vv, torch.arange(n), q_pos, seen)
        out, lse = cache.attend(q, q_pos, want_lse=True, top_tiles=top)
        check_out(out, lse, ref_out, ref_lse, vv)


def test_equal_scores_go_to_the_lowest_tiles_and_nan_comes_first():
    torch = _torch()
    lens = (64,) * 50
    cache, k, v = make("bfloat16", 1, 4, 1, 64, lens, 1, archive_dtype=None, tile_index=True)
    row = cache._attended_spans or cache.get_attention_segments().spans
    cache._arena_k[:, 64:] = 1.0
    cache._ops.tile_bounds(64, 50 * 64, cache.tile_bounds)
    q = queries(1, 4, 1, 64)
    assert cache.select_tiles(q, 5000, 7)[0, 0, 0].tolist() == list(range(7))
    last = row[49][0]
    cache._arena_k[0, last + 3, 9] = math.nan
    cache._ops.tile_bounds(last, 64, cache.tile_bounds)
    assert cache.select_tiles(q, 5000, 3)[0, 0, 0].tolist() == [0, 1, 49]
    q[0, 2, 0, 3] = math.nan  # a NaN query: every score is NaN
    assert cache.select_tiles(q, 5000, 3)[0, 0, 0].tolist() == [0, 1, 2]


def test_selection_over_more_tiles_than_fit_registers():
    torch = _torch()
    lens = (64 * 13000,)
    cache, k, v = make("bfloat16", 1, 2, 1, 64, (), 0, hot_cap=8, archive_dtype=None, tile_index=True,
                       pool_tokens=64 * 13000)
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn(1, 1, lens[0], 64, generator=g, device="cuda").to(torch.bfloat16)
    cache.import_block(k, k, 0)
    q = queries(1, 2, 1, 64)
    t = k[0, 0].double().reshape(13000, 64, 64)
    x = q[0, :, 0].double()
    score = torch.maximum(x[:, None] * t.amin(1), x[:, None] * t.amax(1)).sum(-1).amax(0).float()
    want = torch.sort(torch.topk(score, 100).indices).values
    assert torch.equal(cache.select_tiles(q, lens[0], 100)[0, 0, 0].long(), want)


# ------------------------------------------------------------------ in the cache
@pytest.mark.parametrize("host_tier", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_blocks_that_went_cold_come_back_with_the_same_values(dtype, host_tier):
    torch = _torch()
    lens = (100, 64, 30)
    cache, k, v = make(dtype, 1, 8, 2, 128, lens, 20, tile_index=True, host_tier=host_tier)
    q = queries(1, 8, 1, 128)
    want = cache.attend(q, 213).clone()
    tiles = cache.select_tiles(q, 213, 2).clone()
    for m in list(cache.block_manager.iter_blocks(layer_id=0)):
        cache.demote_manifest_to_cold(m)
    cache._flush_deferred_free()
    cache.archive.clear()
    cache.tile_bounds.zero_()
    # the blocks return to other rows, in the same order
    assert torch.equal(cache.attend(q, 213), want)
    assert torch.equal(cache.select_tiles(q, 213, 2), tiles)


def test_the_archive_grows_and_keeps_its_blocks():
    torch = _torch()
    import archive_ref as ref

    lens = (100, 64, 30, 500, 70)
    cache, k, v = make("bfloat16", 1, 8, 2, 128, lens, 20, tile_index=True, pool_tokens=128)
    assert cache.archive.rows > 128
    q = queries(1, 8, 1, 128)
    kk, vv = held(cache, k, v, lens)
    want, lse = ref.attention(q, kk, vv, torch.arange(784), 783)
    check_out(cache.attend(q, 783), None, want, lse, vv)
    lo, hi, pos = ref.bounds(kk[:, :, :764], lens)
    assert torch.equal(cache.select_tiles(q, 783, 4).cpu().long(), ref.select(q, lo, hi, pos, 783, 4))


def test_a_tile_outside_the_archive_is_reported_and_skipped():
    torch = _torch()
    from rfsn_b200 import _native as native

    cache, k, v = make("bfloat16", 1, 4, 2, 128, (64, 64, 64), 20, tile_index=True)
    q = queries(1, 4, 1, 128)
    segs = cache.get_attention_segments()
    for bad in (-64, 1 << 20, 7):
        saved = cache._tiles_dev.clone()
        cache._tiles_dev[1, 0] = bad
        ws = native.Workspace(cache.device)
        from rfsn_b200.cache import paged_attention

        out = paged_attention(cache, q, 211, segs, workspace=ws)
        with pytest.raises(RuntimeError):
            ws.check()
        assert bool(torch.isfinite(out).all())
        paged_attention(cache, q, 211, segs, workspace=ws, top_tiles=2)
        with pytest.raises(RuntimeError):
            ws.check()
        cache._tiles_dev.copy_(saved)
        paged_attention(cache, q, 211, segs, workspace=ws)
        ws.check()


def test_calls_on_another_stream_and_back():
    torch = _torch()
    cache, k, v = make("bfloat16", 1, 8, 2, 128, (300,), 20, tile_index=True)
    q = queries(1, 8, 1, 128)
    want = cache.attend(q, 319).clone()
    from rfsn_b200 import _native as native
    from rfsn_b200.cache import paged_attention

    s = torch.cuda.Stream()
    ws = native.Workspace(cache.device)
    segs = cache.get_attention_segments()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = paged_attention(cache, q, 319, segs, workspace=ws)
        b = paged_attention(cache, q, 319, segs, workspace=ws, top_tiles=3)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, want) and torch.equal(b, cache.attend(q, 319, top_tiles=3))


@pytest.mark.parametrize("top_tiles", [0, 3])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("H,D", [(8, 128), (16, 128), (40, 128), (8, 64), (40, 64)])  # 4 to 20 query heads per KV head
def test_graphed_decode_step_equals_the_op_by_op_step(packed, top_tiles, H, D):
    """Tokens through the seal rule, captured steps against attention_step on a second cache."""
    torch = _torch()
    if not packed and not top_tiles:
        pytest.skip("the exact dense path has its own tests")
    from rfsn_b200.layer import GraphedDecodeStep, attention_step

    caches = [make("bfloat16", 1, H, 2, D, (), 0, hot_cap=96, wrap=0, top_tiles=top_tiles,
                   archive_dtype="float8_e4m3fn" if packed else None, pool_tokens=2048)[0] for _ in range(2)]
    step = GraphedDecodeStep(caches[0], H)
    g = torch.Generator().manual_seed(11)
    for pos in range(330):
        q, k, v = (torch.randn(1, h, 1, D, generator=g).to(torch.bfloat16) for h in (H, 2, 2))
        step.q_host.copy_(q)
        step.k_host.copy_(k)
        step.v_host.copy_(v)
        got = step.step(pos).clone()
        want = attention_step(q.cuda(), k.cuda(), v.cuda(), caches[1], pos)
        # the split plans differ (a graph plans for a full ring): the same softmax, rounded in another order
        assert float((got - want.cpu()).abs().max()) <= REL * 5.0, pos
    # blocks beyond the warm capacity of 96 tokens go cold: the steps that reload them run op by op
    assert step.replays > 100 and step.captures >= 2 and step.fallbacks > 0


@pytest.mark.parametrize("kw", [dict(archive_dtype="float8_e4m3fn"), dict(top_tiles=2),
                                dict(archive_dtype="float8_e4m3fn", top_tiles=2)])
def test_model_generates_through_a_packed_and_a_sparse_cache(kw):
    """The whole path: chunked prefill, seals, graphed and op-by-op decode give the same tokens and nearly the same
    logits."""
    torch = _torch()
    from rfsn_b200 import RFSNCache, RFSNConfig, RFSNModel

    cfg = RFSNConfig(hidden_dim=512, num_heads=4, num_kv_heads=2, head_dim=128, num_layers=2, vocab_size=300,
                     hot_capacity=64, warm_capacity=1024, cold_capacity=1024, block_size_seq=32, ffn_dim=256,
                     model_dtype="bfloat16", disk_cache_dir=tempfile.mkdtemp(prefix="rfsn_archive_"))
    model = RFSNModel(cfg, seed=3)
    prompt = torch.randint(0, 300, (1, 200), generator=torch.Generator().manual_seed(0))
    logits = []
    for graphs in (True, False):
        model.use_graphs, model._graph = graphs, None
        cache = RFSNCache(cfg, 1, **kw)
        out = [model.prefill(prompt, cache)[:, -1]]
        for i in range(60):
            tok = torch.tensor([(17 * i) % 300], dtype=torch.int32)
            out.append(model.decode_step(tok, cache, 200 + i))
        logits.append(torch.stack(out).float())
        assert cache.layer(0)._n_tiles >= 3
    assert torch.isfinite(logits[0]).all()
    # bf16 activations: the two runs differ by roundings of one bf16 step here and there
    scale = float(logits[0].abs().max())
    assert float((logits[0] - logits[1]).abs().max()) <= 16 * 2.0 ** -8 * scale


@pytest.mark.parametrize("packed", [True, False])
def test_offsets_past_32_bits(packed):
    """Heads whose rows lie more than 2^31 elements into the archive (or arena), and its bounds."""
    torch = _torch()
    import archive_ref as ref

    lens = (200,)
    cache, k, v = make("bfloat16", 1, 8, 8, 128, lens, 10, tile_index=True, pool_tokens=2_500_032,
                       archive_dtype="float8_e4m3fn" if packed else None)
    rows = cache.archive.rows if packed else cache._arena_k.shape[1]
    assert 7 * rows * 128 > 1 << 31
    q = queries(1, 8, 1, 128)
    kk, vv = held(cache, k, v, lens)
    want, lse = ref.attention(q, kk, vv, torch.arange(210), 209)
    out, got = cache.attend(q, 209, want_lse=True, top_tiles=4)
    check_out(out, got, want, lse, vv)
    if packed:
        check_out(cache.attend(q, 209), None, want, lse, vv)
        q = queries(1, 8, 70, 128)
        want, lse = ref.attention(q, kk, vv, torch.arange(210), 140)
        check_out(cache.attend(q, 140), None, want, lse, vv)
    lo, hi, pos = ref.bounds(kk[:, :, :200], lens)
    q = queries(1, 8, 1, 128)
    assert torch.equal(cache.select_tiles(q, 209, 2).cpu().long(), ref.select(q, lo, hi, pos, 209, 2))


def test_results_go_where_the_caller_says():
    torch = _torch()
    from rfsn_b200.cache import paged_attention

    cache, k, v = make("bfloat16", 1, 8, 2, 128, (300,), 20, tile_index=True)
    q = queries(1, 8, 1, 128)
    segs = cache.get_attention_segments()
    for top in (0, 2):
        want = cache.attend(q, 319, top_tiles=top)
        out = torch.empty_like(q)
        assert paged_attention(cache, q, 319, segs, out=out, top_tiles=top) is out and torch.equal(out, want)
        host = torch.empty(q.shape).pin_memory()
        paged_attention(cache, q, 319, segs, out=host, top_tiles=top)
        torch.cuda.synchronize()
        assert torch.equal(host, want.cpu())
        half = cache.attend(q.to(torch.bfloat16), 319, top_tiles=top)  # any float q is taken as float32
        assert half.dtype == torch.float32 and torch.equal(half, cache.attend(q.to(torch.bfloat16).float(), 319,
                                                                              top_tiles=top))
        strided = torch.empty(1, 1, 8, 128, device="cuda").transpose(1, 2)
        strided.copy_(q)
        assert torch.equal(cache.attend(strided, 319, top_tiles=top), want)


def test_segments_are_a_snapshot_of_the_window():
    """A prepared call keeps the window of its segments; new segments see the appended token."""
    torch = _torch()
    import archive_ref as ref

    cache, k, v = make("bfloat16", 1, 8, 2, 128, (300,), 20, hot_cap=64)
    q = queries(1, 8, 1, 128)
    old = cache.get_attention_segments()
    before = cache.attend(q, 1000, old).clone()
    extra = torch.randn(1, 2, 1, 128, device="cuda").to(torch.bfloat16)
    cache.append_exact(extra, extra)
    assert torch.equal(cache.attend(q, 1000, old), before)
    kk, vv = held(cache, k, v, (300,))
    kk, vv = (torch.cat([x, extra.double().cpu()], 2) for x in (kk, vv))
    want, lse = ref.attention(q, kk, vv, torch.arange(321), 1000)
    check_out(cache.attend(q, 1000), None, want, lse, vv)


def test_refusals():
    torch = _torch()
    from rfsn_b200 import PackedArchive
    from rfsn_b200.cache import paged_attention

    cache, k, v = make("bfloat16", 1, 8, 2, 128, (300,), 20, tile_index=True)
    plain, _, _ = make("bfloat16", 1, 8, 2, 128, (300,), 20, archive_dtype=None)
    q = queries(1, 8, 1, 128)
    for bad in (queries(2, 8, 1, 128), queries(1, 8, 1, 64), queries(1, 7, 1, 128)):
        with pytest.raises(ValueError):
            cache.attend(bad, 319)
        with pytest.raises(ValueError):
            cache.select_tiles(bad, 319, 2)
    with pytest.raises(ValueError, match="tile_index"):
        plain.attend(q, 319, top_tiles=2)
    with pytest.raises(ValueError, match="tile_index"):
        plain.select_tiles(q, 319, 2)
    for top in (-1, (1 << 20) + 1):
        with pytest.raises(ValueError):
            cache.attend(q, 319, top_tiles=top)
        with pytest.raises(ValueError):
            cache.select_tiles(q, 319, top)
    with pytest.raises(ValueError):
        cache.select_tiles(q, 319, 0)
    with pytest.raises(ValueError, match="64 query rows"):
        cache.attend(queries(1, 8, 65, 128), 319, top_tiles=2)
    with pytest.raises(ValueError, match="64 query rows"):
        cache.select_tiles(queries(1, 8, 65, 128), 319, 2)
    segs = cache.get_attention_segments()
    with pytest.raises(NotImplementedError):
        paged_attention(cache, q, 319, segs, peers=object())
    with pytest.raises(ValueError, match="out must"):
        paged_attention(cache, q, 319, segs, out=torch.empty(1, 8, 2, 128, device="cuda"))
    empty, _, _ = make("bfloat16", 1, 8, 2, 128, (), 0, hot_cap=8)
    with pytest.raises(RuntimeError):
        empty.attend(q, 0)
    a = PackedArchive(2, 128, 128)
    x = torch.zeros(1, 2, 64, 128, device="cuda")
    for bad in ((x[:, :, :, :64], x[:, :, :, :64]), (x[0], x[0]), (x, x[:, :, :32]), (x, x.half()), (x.cpu(), x.cpu()),
                (x.double(), x.double()), (x[:, :1], x[:, :1])):
        with pytest.raises(ValueError):
            a.pack(*bad)
    for row, n in ((1, 64), (128, 64), (-64, 64), (64, 128)):
        with pytest.raises(ValueError):
            a.pack(torch.zeros(1, 2, n, 128, device="cuda"), torch.zeros(1, 2, n, 128, device="cuda"), row)
    with pytest.raises(ValueError, match="bounds"):
        a.pack(x, x, bounds=torch.zeros(2, 2, 2, 128, device="cuda"))
    for row, n in ((0, 129), (-1, 4), (128, 1)):
        with pytest.raises(ValueError):
            a.unpack(row, n, torch.float32)
    with pytest.raises(ValueError):
        a.unpack(0, 4, torch.float64)
    with pytest.raises((ValueError, NotImplementedError)):
        PackedArchive(2, 64, 96)
    with pytest.raises(ValueError):
        PackedArchive(0, 64, 128)
    a.pack(x[:, :, :0], x[:, :, :0])  # nothing to do
    assert a.unpack(0, 0, torch.float32)[0].shape == (2, 0, 128)


def test_two_streams_with_workspaces_of_their_own():
    torch = _torch()
    from rfsn_b200 import _native as native
    from rfsn_b200.cache import paged_attention

    caches = [make("bfloat16", 1, 8, 2, 128, (3000,), 20, tile_index=True, seed=i)[0] for i in range(2)]
    q = queries(1, 8, 1, 128)
    want = [[c.attend(q, 3019, top_tiles=top).clone() for top in (0, 5)] for c in caches]
    tiles = [c.select_tiles(q, 3019, 5).clone() for c in caches]
    streams = [torch.cuda.Stream() for _ in caches]
    spaces = [native.Workspace(c.device) for c in caches]
    segs = [c.get_attention_segments() for c in caches]
    got = [[], []]
    lists = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, c in enumerate(caches):
            with torch.cuda.stream(streams[i]):
                got[i].append([paged_attention(c, q, 3019, segs[i], workspace=spaces[i], top_tiles=top)
                               for top in (0, 5)])
                lists[i].append(c.select_tiles(q, 3019, 5, segs[i], workspace=spaces[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for pair in got[i]:
            assert torch.equal(pair[0], want[i][0]) and torch.equal(pair[1], want[i][1])
        assert all(torch.equal(x, tiles[i]) for x in lists[i])


def test_the_same_call_gives_the_same_bits():
    torch = _torch()
    cache, k, v = make("bfloat16", 1, 32, 8, 128, (1000,) * 8, 200, tile_index=True)
    for Lq in (1, 4, 64):
        q = queries(1, 32, Lq, 128)
        want = cache.attend(q, 8200 - Lq).clone()
        sparse = cache.attend(q, 8200 - Lq, top_tiles=9).clone()
        for _ in range(5):
            assert torch.equal(cache.attend(q, 8200 - Lq), want)
            assert torch.equal(cache.attend(q, 8200 - Lq, top_tiles=9), sparse)


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("Lq", [1, 3, 40])
def test_keys_and_values_behind_the_queries_are_not_touched(packed, Lq):
    """NaN K and V at every position behind the last query, in its own tile too."""
    torch = _torch()
    lens = (130, 64)
    tops = (0, 9) if packed else (9,)  # without either option the call is that of an exact cache
    for last in (20, 129, 150, 200, 215):
        cache, k, v = make("bfloat16", 1, 4, 2, 128, lens, 40, tile_index=True,
                           archive_dtype="float8_e4m3fn" if packed else None)
        q = queries(1, 4, Lq, 128)
        first = last + 1 - Lq
        if first < 0:
            continue
        want = [cache.attend(q, first, top_tiles=top, want_lse=True) for top in tops]
        bad_k, bad_v = k.clone(), v.clone()
        for x in (bad_k, bad_v):
            x[:, :, last + 1:] = math.nan
        spans = cache.get_attention_segments().spans
        for (row, start, n) in spans[:2]:
            kk, vv = bad_k[:, :, start:start + n], bad_v[:, :, start:start + n]
            if packed:  # codes only: the scales are those of the finite tiles
                codes = cache.archive.k.view(torch.uint8), cache.archive.v.view(torch.uint8)
                for c in codes:
                    c[:, row:row + n][:, max(0, last + 1 - start):] = 0x7F
            else:
                cache._arena_k[:, row:row + n] = kk[0]
                cache._arena_v[:, row:row + n] = vv[0]
        ring = max(0, last + 1 - 194)
        cache._arena_k[:, ring:40] = math.nan
        cache._arena_v[:, ring:40] = math.nan
        for top, (out, lse) in zip(tops, want):
            got, got_lse = cache.attend(q, first, top_tiles=top, want_lse=True)
            assert torch.equal(got, out) and torch.equal(got_lse, lse), (last, top)


@pytest.mark.parametrize("Lq", [1, 40])
@pytest.mark.parametrize("v_scale", [1e-6, 1e-30, 1e30])
@pytest.mark.parametrize("lens", [(64,), (64, 64), (50, 64, 64), ()])
def test_small_and_large_values(Lq, v_scale, lens):
    """V far from 1, an odd number of tiles: the halves without keys and the ring do not set the unit."""
    torch = _torch()
    import archive_ref as ref

    n = sum(lens) + 70
    torch.manual_seed(5)
    cache, k, v = make("bfloat16", 1, 4, 1, 128, lens, 70, v_scale=v_scale)
    q = queries(1, 4, Lq, 128)
    kk, vv = held(cache, k, v, lens)
    want, lse = ref.attention(q, kk, vv, torch.arange(n), n - Lq)
    out, got = cache.attend(q, n - Lq, want_lse=True)
    check_out(out, got, want, lse, vv)


def test_a_vanishing_product_of_scales_masks_like_any_other():
    """q and K so small that their scales' product underflows: logits 0, masked keys still masked."""
    torch = _torch()
    import archive_ref as ref

    cache, k, v = make("bfloat16", 1, 4, 1, 128, (64, 30), 0, hot_cap=8, scale=1e-20)
    for Lq in (1, 40):
        q = queries(1, 4, Lq, 128, scale=1e-36)
        kk, vv = held(cache, k, v, (64, 30))
        want, lse = ref.attention(q, kk, vv, torch.arange(94), 94 - Lq)
        out, got = cache.attend(q, 94 - Lq, want_lse=True)
        check_out(out, got, want, lse, vv)


def test_a_selection_from_no_tiles_reports_nothing():
    torch = _torch()
    from rfsn_b200 import _native as native

    cache, _, _ = make("bfloat16", 1, 4, 2, 128, (), 20, hot_cap=32, tile_index=True)
    q = queries(1, 4, 1, 128)
    assert bool((cache.select_tiles(q, 19, 3) == -1).all())
    assert torch.equal(cache.attend(q, 19, top_tiles=3), cache.attend(q, 19))
    native.default_workspace(cache.device).check()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("H,Hkv,Lq", [(6, 1, 1), (8, 1, 1), (3, 1, 3), (9, 1, 1), (7, 1, 2), (16, 1, 1), (17, 1, 1),
                                      (5, 1, 7), (33, 1, 1), (130, 1, 1)])
@pytest.mark.parametrize("lens,hot,wrap", [((64,), 1, 0), ((1, 63, 64, 65, 130), 200, 90), ((1000,) * 5, 300, 299),
                                           ((), 40, 5)])
def test_every_count_of_query_slots(dtype, H, Hkv, Lq, lens, hot, wrap):
    """5 and more query slots of a packed cache, one or several CTAs deep, odd counts and rings that wrap."""
    torch = _torch()
    import archive_ref as ref

    cap = hot if wrap else max(hot, 64)
    cache, k, v = make(dtype, 1, H, Hkv, 128, lens, hot, hot_cap=cap, wrap=wrap % cap)
    n = sum(lens) + hot
    q = queries(1, H, Lq, 128)
    kk, vv = held(cache, k, v, lens)
    for last in (n - 1, n + 50, n // 2):
        first = last - Lq + 1
        if first < 0:
            continue
        want, lse = ref.attention(q, kk, vv, torch.arange(n), first)
        out, got = cache.attend(q, first, want_lse=True)
        check_out(out, got, want, lse, vv)


@pytest.mark.parametrize("Lq", [1, 2, 4, 9, 40])
def test_captured_calls_replay_on_new_queries(Lq):
    """A captured call of every kernel gives what the eager call gives, on queries written before each replay."""
    torch = _torch()
    cache, k, v = make("bfloat16", 1, 8, 2, 128, (1000, 500), 60, tile_index=True)
    segs = cache.get_attention_segments()
    q = queries(1, 8, Lq, 128)
    first = 1560 - Lq
    from rfsn_b200 import _native as native
    from rfsn_b200.cache import paged_attention

    ws = [native.Workspace(cache.device) for _ in range(2)]  # a graph keeps the workspace it was captured with
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for i, top in enumerate((0, 3)):
        with torch.cuda.stream(side):
            paged_attention(cache, q, first, segs, workspace=ws[i], top_tiles=top)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append([paged_attention(cache, q, first, segs, workspace=ws[i], top_tiles=top) for _ in range(2)])
        graphs.append(g)
    for seed in range(3):
        q.copy_(queries(1, 8, Lq, 128, seed=seed + 20))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i, top in enumerate((0, 3)):
            want = cache.attend(q, first, segs, top_tiles=top)
            assert all(torch.equal(o, want) for o in outs[i])


def test_values_of_very_different_size_in_one_call():
    """Tiles whose V scales are 2^20 apart: the error is measured against the largest value that is seen."""
    torch = _torch()
    import archive_ref as ref

    lens = (64, 64, 64, 64, 64)
    for Lq in (1, 4, 40):
        torch.manual_seed(3)
        cache, k, v = make("bfloat16", 1, 4, 1, 128, (), 0, hot_cap=64, pool_tokens=2048)
        v = torch.randn(1, 1, 320, 128, device="cuda")
        k = torch.randn(1, 1, 320, 128, device="cuda").to(torch.bfloat16)
        for i, s in enumerate((1.0, 2.0 ** 20, 2.0 ** -20, 1.0, 2.0 ** 10)):
            v[:, :, 64 * i:64 * i + 64] *= s
            cache.import_block(k[:, :, 64 * i:64 * i + 64], v[:, :, 64 * i:64 * i + 64].to(torch.bfloat16), 64 * i)
        v = v.to(torch.bfloat16)
        kk, vv = held(cache, k, v, lens)
        q = queries(1, 4, Lq, 128)
        for last in (63, 319):
            if last - Lq + 1 < 0:
                continue
            want, lse = ref.attention(q, kk, vv, torch.arange(320), last - Lq + 1)
            out, got = cache.attend(q, last - Lq + 1, want_lse=True)
            check_out(out, got, want, lse, vv[:, :, :last + 1])


# ------------------------------------------------------------------ chunks (128 query slots per CTA)
def in_chunks(cache, q, first, **kw):
    """``attend``, checked to run the chunk kernel: the ring's copy or the merge is a launch of its own."""
    from rfsn_b200 import _native as native

    before = native.launch_count()
    out = cache.attend(q, first, **kw)
    assert native.launch_count() - before >= 2
    return out


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("dtype,B,H,Hkv,lens,hot,wrap,Lq", [
    ("bfloat16", 1, 8, 2, (64,) * 81, 100, 0, 128),            # an odd number of tiles
    ("float16", 2, 8, 2, (70,) * 30 + (64,) * 2, 33, 20, 100),  # ragged tiles, a wrapped ring
    ("bfloat16", 1, 40, 1, (1000,) * 8, 64, 0, 77),             # 40 heads a row: 3 rows in a CTA, 8 slots idle
    ("bfloat16", 1, 4, 4, (6000,), 300, 0, 300),
    ("float16", 1, 128, 1, (5000,), 10, 0, 9),                  # a row per CTA
])
def test_chunks_of_queries(dtype, B, H, Hkv, lens, hot, wrap, Lq, D):
    torch = _torch()
    import archive_ref as ref

    cache, k, v = make(dtype, B, H, Hkv, D, lens, hot, hot_cap=max(hot, 64), wrap=wrap)
    n = sum(lens) + hot
    q = queries(B, H, Lq, D)
    kk, vv = held(cache, k, v, lens)
    for first in (n - Lq, n + 7, n // 2, 0, -5):
        want, lse = ref.attention(q, kk, vv, torch.arange(n), first)
        out, got = in_chunks(cache, q, first, want_lse=True)
        check_out(out, got, want, lse, vv)
    assert torch.equal(in_chunks(cache, q, n - Lq), in_chunks(cache, q, n - Lq))


@pytest.mark.parametrize("D", [128, 64])
def test_chunks_and_what_lies_behind_them(D):
    """NaN K and V behind the last query of a chunk, in its own tile too, in the archive and in the ring. (Against the
    64-bit form: the scale of a ring tile, and with it the roundings of p, depends on its finite values.)"""
    torch = _torch()
    import archive_ref as ref

    lens = (64,) * 81
    cache, k, v = make("bfloat16", 1, 8, 2, D, lens, 100)
    q = queries(1, 8, 128, D)
    kk, vv = held(cache, k, v, lens)
    spans = cache.get_attention_segments().spans
    for last in (5184 + 70, 5183, 5170, 5120, 3000):  # NaN stays from one to the next
        first = last + 1 - 128
        for codes in (cache.archive.k.view(torch.uint8), cache.archive.v.view(torch.uint8)):
            for row, start, n in spans[:81]:
                if start + n > last + 1:
                    codes[:, row + max(0, last + 1 - start):row + n] = 0x7F
        for arena in (cache._arena_k, cache._arena_v):
            arena[:, max(0, last + 1 - 5184):100] = math.nan
        want, want_lse = ref.attention(q, kk, vv, torch.arange(5284), first)
        out, lse = in_chunks(cache, q, first, want_lse=True)
        check_out(out, lse, want, want_lse, vv)


@pytest.mark.parametrize("D", [128, 64])
def test_chunks_with_nan_that_is_seen(D):
    torch = _torch()
    cache, k, v = make("bfloat16", 1, 8, 2, D, (64,) * 81, 100)
    q = queries(1, 8, 128, D)
    row = cache.get_attention_segments().spans[7][0]
    kn, vn = k[:, :, 448:512].clone(), v[:, :, 448:512].clone()
    kn[0, 1, 3, 5] = math.inf  # packed as NaN: every row of KV head 1
    vn[0, 0, 4, 7] = math.nan  # channel 7 of KV head 0
    cache.archive.pack(kn, vn, row)
    out = in_chunks(cache, q, 5284 - 128)
    assert bool(torch.isnan(out[0, 4:]).all())
    fine = torch.ones(D, dtype=torch.bool, device="cuda")
    fine[7] = False
    assert bool(torch.isfinite(out[0, :4][..., fine]).all()) and bool(torch.isnan(out[0, :4, :, 7]).all())


@pytest.mark.parametrize("v_scale,q_scale", [(1e-6, 1.0), (1e-30, 0.0), (1e30, 60.0), (1.0, 1e-30)])
@pytest.mark.parametrize("D", [128, 64])
def test_chunks_of_extreme_sizes(v_scale, q_scale, D):
    torch = _torch()
    import archive_ref as ref

    lens = (64,) * 81
    cache, k, v = make("bfloat16", 1, 8, 2, D, lens, 100, v_scale=v_scale)
    q = queries(1, 8, 128, D, scale=q_scale)
    kk, vv = held(cache, k, v, lens)
    want, lse = ref.attention(q, kk, vv, torch.arange(5284), 5284 - 128)
    out, got = in_chunks(cache, q, 5284 - 128, want_lse=True)
    tol = REL * max(1.0, q_scale)  # logits of q_scale times the usual size carry that many times the error
    assert float((out.double().cpu() - want).abs().max()) <= tol * float(vv.abs().max())
    assert float((got.double().cpu() - lse).abs().max()) <= tol * 4


def test_chunks_captured_and_on_two_streams():
    torch = _torch()
    from rfsn_b200 import _native as native
    from rfsn_b200.cache import paged_attention

    cache, k, v = make("bfloat16", 1, 8, 2, 128, (64,) * 81, 100)
    segs = cache.get_attention_segments()
    q = queries(1, 8, 128, 128)
    first = 5284 - 128
    spaces = [native.Workspace(cache.device) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for ws, s in zip(spaces, streams):
        with torch.cuda.stream(s):
            paged_attention(cache, q, first, segs, workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(paged_attention(cache, q, first, segs, workspace=ws))
        graphs.append(g)
    for seed in range(3):
        q.copy_(queries(1, 8, 128, 128, seed=seed + 3))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        want = in_chunks(cache, q, first, segments=segs)
        assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("packed", [True, False])
def test_a_device_without_an_index(packed):
    """device="cuda" names the current device, for the cache, its archive and results given by the caller."""
    torch = _torch()
    from rfsn_b200.cache import paged_attention

    kw = dict(archive_dtype="float8_e4m3fn" if packed else None, tile_index=True)
    caches = [make("bfloat16", 1, 8, 2, 128, (300,), 20, device=d, **kw)[0] for d in ("cuda", "cuda:0")]
    q = queries(1, 8, 1, 128)
    for top in (0, 2):
        outs = []
        for c in caches:
            segs = c.get_attention_segments()
            outs.append(c.attend(q, 319, segs, top_tiles=top))
            given = torch.empty_like(q)
            outs.append(paged_attention(c, q, 319, segs, out=given, top_tiles=top))
        assert all(torch.equal(o, outs[0]) for o in outs)
    assert torch.equal(caches[0].select_tiles(q, 319, 2), caches[1].select_tiles(q, 319, 2))


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("Lq", [1, 2, 4, 40, 128])
@pytest.mark.parametrize("lens,scale", [((64,) * 81, 1.0), ((64,), 0.01)])
def test_infinities_and_nan_in_queries_stay_in_their_rows(Lq, packed, D, lens, scale):
    """A query row with an infinity or a NaN becomes NaN, the others do not change beyond rounding."""
    torch = _torch()
    import archive_ref as ref

    if not packed and Lq > 64:
        pytest.skip("a selecting call takes up to 64 rows")
    cache, k, v = make("bfloat16", 1, 8, 2, D, lens, 100, tile_index=True, scale=scale,
                       archive_dtype="float8_e4m3fn" if packed else None)
    q = queries(1, 8, Lq, D)
    kk, vv = held(cache, k, v, lens)
    n = sum(lens) + 100
    first = n - Lq
    want, lse = ref.attention(q, kk, vv, torch.arange(n), first)
    bad = torch.zeros(8, Lq, dtype=torch.bool)
    for h, r, x in ((3, 0, math.inf), (6, Lq - 1, math.nan), (4, Lq // 2, -math.inf)):
        q[0, h, r, 5] = x
        bad[h, r] = True
    for top in ([0] if packed else []) + ([200] if Lq <= 64 else []):
        out, got = cache.attend(q, first, top_tiles=top, want_lse=True)
        out, got = out.cpu(), got.cpu()
        assert bool(torch.isnan(out[0][bad]).all()) and bool(torch.isnan(got[0][bad]).all())
        check_out(out[0][~bad], got[0][~bad], want[0][~bad], lse[0][~bad], vv)
