"""Tile selection where scores lie close together or are equal, against the order of exactly known scores.

The keys of a tile are 64 times one row that holds a leading value and the seven base-8 digits of an integer j; the
query weighs them so that the tile's score is ``lead + j * 2^-23``. Leads are powers of two, digits and leads are exact
in bfloat16, float16 and e4m3 (with a tile's power-of-two scale), every product and sum is exact in 64 bits, and scores
below 2 are exact in float32: the expected list follows from the integers alone, without rounding.
"""

import random

import pytest

from test_archive_gpu import check_out, make

pytestmark = pytest.mark.gpu

D = 64
DIGITS = 7  # j < 2^21: scores up to 25 % above their lead


def _torch():
    import torch

    return torch


def offsets(pattern, T, rng):
    """(lead, j) of each tile."""
    if pattern == "bucket":  # the last bucket is narrower than the keys just above it reach
        return [(8, 0), (1, 40)] + [(1, 0)] * (T - 2)
    if pattern == "steps":
        return [(1, 0)] * (T - 4) + [(1, 600), (1, 1200), (1, 1800), (1, 2 ** 19 - 8)]
    if pattern == "ties":  # many equal scores, with neighbours 1 to 1,000 steps above them, and one far away
        return [(4, 0)] + [(1, rng.choice([5, 5, 5, 5, 6, 9, 30, 100, 700, 1005])) for _ in range(T - 1)]
    if pattern == "twice":  # the same tiles two times
        half = [(1, rng.randrange(2 ** 18)) for _ in range((T + 1) // 2)]
        return (half + half)[:T]
    if pattern == "below":  # most tiles of a negative score, some of them equal to -1
        return [(rng.choice([-1, -2, 1]), 8 * rng.randrange(64)) for _ in range(T)]
    spread = int(pattern[:-1]) * 2 ** 23 // 1000  # "5m": within 0.5 %
    return [(1, rng.randrange(spread)) for _ in range(T)]


def rows(tiles):
    """One key row per tile, [T, D]."""
    torch = _torch()
    x = torch.zeros(len(tiles), D)
    for t, (lead, j) in enumerate(tiles):
        x[t, 0] = lead
        for i in range(DIGITS):
            x[t, 1 + i] = j >> 3 * i & 7
    return x


def query(H):
    """[1, H, 1, D]; the heads behind the first weigh everything half as much and decide nothing where a score is
    positive; a score of below 0 comes from the last head."""
    torch = _torch()
    q = torch.zeros(1, H, 1, D)
    q[:, :, :, 0] = 1.0
    for i in range(DIGITS):
        q[:, :, :, 1 + i] = 2.0 ** (3 * i - 23)
    return (q * torch.exp2(-torch.arange(H).float())[:, None, None]).cuda()


def best(tiles, n, H):
    """The n largest scores, equal ones by the lowest tile, in tile order; exact in integers of 2^-23."""
    s = [lead * 2 ** 23 + j for lead, j in tiles]
    s = [x if x > 0 else x / 2 ** (H - 1) for x in s]  # the head with the largest score
    order = sorted(range(len(s)), key=lambda t: (-s[t], t))[:n]
    return sorted(order) + [-1] * (n - len(order))


CASES = [("bucket", 4, 3), ("steps", 6, 5), ("ties", 96, 16), ("ties", 512, 333), ("twice", 512, 31), ("twice", 97, 49),
         ("below", 200, 150), ("5m", 96, 16), ("20m", 96, 95), ("5m", 2064, 128), ("20m", 2064, 1000),
         ("30m", 2064, 128), ("5m", 4096, 77), ("5m", 4097, 77), ("20m", 30000, 1000), ("5m", 30000, 64),
         ("twice", 30001, 333), ("ties", 5000, 1500), ("1m", 8, 8), ("1m", 8, 9), ("1m", 1, 1)]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("pattern,T,n", CASES)
def test_the_n_largest_of_close_and_equal_scores(pattern, T, n, packed):
    torch = _torch()
    import archive_ref as ref

    H = 2
    cache, _, _ = make("bfloat16", 1, H, 1, D, (), 0, hot_cap=8, tile_index=True, pool_tokens=64 * T,
                       archive_dtype="float8_e4m3fn" if packed else None)
    q = query(H)
    for seed in range(3):
        tiles = offsets(pattern, T, random.Random(1000 * T + n + seed))
        x = rows(tiles)
        g = torch.Generator().manual_seed(seed)
        y = torch.randint(-4, 5, (T, D), generator=g).float()  # exact in all types
        cache.reset()
        cache.import_block(x.repeat_interleave(64, 0)[None, None].to(torch.bfloat16).cuda(),
                           y.repeat_interleave(64, 0)[None, None].to(torch.bfloat16).cuda(), 0)
        want = best(tiles, n, H)
        if n < T:  # the list that lies in the workspace, and the memory of the numbers, are another query's
            cache.attend(-q, 64 * T, top_tiles=n)
            cache.select_tiles(-q, 64 * T, n)
        assert cache.select_tiles(q, 64 * T, n)[0, 0, 0].tolist() == want
        if T > 5000:
            continue
        chosen = [t for t in want if t >= 0]
        # every key of a tile is the same, and so is its value: a tile is one key
        out, lse = cache.attend(q, 64 * T, want_lse=True, top_tiles=n)
        ref_out, ref_lse = ref.attention(q, x[None, None, chosen], y[None, None, chosen], torch.arange(len(chosen)),
                                         len(chosen))
        check_out(out, lse - torch.log(torch.tensor(64.0)), ref_out, ref_lse, y)


@pytest.mark.parametrize("packed", [False, True])
def test_rows_heads_and_batches_select_for_themselves(packed):
    """Close scores in several lists at once, rows at different positions."""
    torch = _torch()
    B, Hkv, G, Lq, T, n = 2, 2, 3, 4, 300, 37
    cache, _, _ = make("float16", B, Hkv * G, Hkv, D, (), 0, hot_cap=8, tile_index=True, pool_tokens=64 * T,
                       archive_dtype="float8_e4m3fn" if packed else None)
    rng = random.Random(5)
    tiles = [[offsets("20m" if h else "ties", T, rng) for h in range(Hkv)] for _ in range(B)]
    x = torch.stack([torch.stack([rows(t) for t in per]) for per in tiles]).repeat_interleave(64, 2).half().cuda()
    cache.import_block(x, x, 0)
    q = query(G).repeat(B, Hkv, Lq, 1)
    first = 64 * 250 - 2  # rows 2 and 3 see a tile more than rows 0 and 1
    got = cache.select_tiles(q, first, n)
    for b in range(B):
        for h in range(Hkv):
            for r in range(Lq):
                seen = (first + r) // 64 + 1
                assert got[b, h, r].tolist() == best(tiles[b][h][:seen], n, G), (b, h, r)
