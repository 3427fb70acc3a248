"""Cases of the archive operators: packing archived K/V into 8 bits, attention over such an archive and the hot
window, selection of archived tiles by a bound on their logits, and attention over the selected tiles.

A tile is 64 consecutive tokens of an archived block (the last tile of a block may be shorter). One layer's context is
`blocks` archived blocks of `block` tokens (and one of `tail` tokens, if any) followed by `hot` tokens in the ring.

`own` false: the operators in elementary torch operations. `own` true: the framework's calls.
"""

import math
import os
import sys
import tempfile

import torch

own = False

TILE = 64
E4M3_MAX = 448.0


# ------------------------------------------------------------------ cases
def _case(name, op, **kw):
    c = dict(name=name, op=op, dtype="bfloat16", batch=1, heads=32, kv_heads=8, dim=128, block=256, blocks=24, tail=0,
             hot=2048, q_len=1, top=0, packed=True)
    c.update(kw)
    return c


def listed():
    return [
        # one block of 256 tokens leaves the ring: the seal of a decode step
        _case("pack seal 256", "pack", block=256, blocks=1, hot=0),
        # a prompt's K/V, token-major as the projections deliver it, enters the archive at once; ragged last tile
        _case("pack import 65501", "pack", block=65501, blocks=1, hot=0),
        # one decode token, 8,192-token fp16 context (24 blocks of 256, ring of 2,048)
        _case("packed decode 8k fp16", "attend", dtype="float16"),
        # one decode token, 132,120-token bf16 context (127 blocks of 1,000 and one of 1,024, ring of 4,096)
        _case("packed decode 132k", "attend", block=1000, blocks=127, tail=1024, hot=4096),
        # the default configuration's heads (8 x 64, no GQA), three sequences, ragged blocks
        _case("packed decode d64 batch 3", "attend", batch=3, heads=8, kv_heads=8, dim=64, block=65, blocks=77, tail=7,
              hot=511),
        # four draft tokens checked at once against 33K
        _case("packed verify 4x33k", "attend", block=1000, blocks=31, hot=2000, q_len=4),
        # a prompt chunk over a packed archive
        _case("packed chunk 512x16k", "attend", block=512, blocks=32, hot=1024, q_len=512),
        # tile choice for one decode token of a short and of a long context
        _case("select 16 of 8k, batch 2", "select", batch=2, top=16, packed=False),
        _case("select 128 of 132k", "select", block=1000, blocks=127, tail=1024, hot=4096, top=128, packed=False),
        # one decode token over its 16 best tiles of a short fp16 context, and the 128 best of a long one, from the
        # exact archive and from the packed one
        _case("sparse 16 of 8k fp16", "sparse", dtype="float16", hot=512, top=16, packed=False),
        _case("sparse 128 of 132k", "sparse", block=1000, blocks=127, tail=1024, hot=1024, top=128, packed=False),
        _case("sparse packed 128 of 132k", "sparse", block=1000, blocks=127, tail=1024, hot=1024, top=128),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["pack", "attend", "attend", "select", "sparse", "sparse"])
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (8, 8), (16, 2), (12, 4), (32, 1)])
    dim = rng.choice([128, 128, 64])
    dtype = rng.choice(["bfloat16", "float16"])
    batch = rng.choice([1, 1, 1, 2, 3])
    if op == "pack":
        return dict(op=op, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, block=log(1, 20000),
                    blocks=1, tail=0, hot=0, q_len=1, top=0, packed=True)
    block = log(33, 2100)
    tokens = log(300, 40000)
    blocks = max(1, tokens // block)
    q_len = rng.choice([1, 1, 1, 1, 2, 3, 5]) if op != "attend" else rng.choice([1, 1, 1, 2, 4, 7, log(16, 300)])
    hot = max(q_len, log(1, 4096))
    if q_len >= 16:  # a chunk: no more products than the listed one's
        batch, q_len = 1, max(16, min(q_len, 8_000_000 // (tokens + hot)))
    top = log(1, 200) if op in ("select", "sparse") else 0
    return dict(op=op, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, block=block, blocks=blocks,
                tail=rng.choice([0, 1, 40, 64, 129]), hot=hot, q_len=q_len, top=top,
                packed=op == "attend" or (op == "sparse" and rng.random() < 0.5))


# ------------------------------------------------------------------ layout
def _dtype(case):
    return {"bfloat16": torch.bfloat16, "float16": torch.float16}[case["dtype"]]


def _block_lens(case):
    return [case["block"]] * case["blocks"] + ([case["tail"]] if case["tail"] else [])


def _tile_of_token(case):
    """For each archived token the number of its tile (tiles are counted through the blocks in order)."""
    block = torch.arange(case["block"] * case["blocks"])
    per = -(-case["block"] // TILE)
    out = (block // case["block"]) * per + (block % case["block"]) // TILE
    if case["tail"]:
        out = torch.cat([out, case["blocks"] * per + torch.arange(case["tail"]) // TILE])
    return out.cuda()


def _n_tiles(case):
    return sum(-(-n // TILE) for n in _block_lens(case))


def _scale(amax):
    """The power of two s with amax / s in (224, 448], 1 where amax is 0."""
    m, e = torch.frexp(amax.float())  # amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    s = torch.exp2((e - 9 + (m > E4M3_MAX / 512).int()).double()).clamp(min=2.0 ** -126).float()
    return torch.where(amax > 0, s, torch.ones_like(s))


def _tile_amax(x, tile, n_tiles):
    """[B, Hkv, N, D] -> [B, Hkv, n_tiles]: the largest magnitude of each tile."""
    row = x.abs().amax(dim=-1).float()
    out = torch.zeros(row.shape[:2] + (n_tiles,), device=x.device)
    return out.scatter_reduce(2, tile.expand_as(row), row, "amax")


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, H, Hkv, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    dtype, lens = _dtype(case), _block_lens(case)
    N, hot, Lq = sum(lens), case["hot"], case["q_len"]
    n = N + hot

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    # keys: a topic that holds for about a hundred tokens, noise, and a few strong channels; values: noise with a level
    # that differs from head to head. Token-major memory, as a projection writes it.
    topics = randn(B, n // 96 + 1, Hkv, D)
    channel = torch.where(torch.rand(Hkv, D, generator=g, device="cuda") < 0.05, 4.0, 1.0)
    at = torch.arange(n, device="cuda") // 96
    k = torch.empty(B, n, Hkv, D, dtype=dtype, device="cuda")
    v = torch.empty(B, n, Hkv, D, dtype=dtype, device="cuda")
    level = torch.exp(randn(Hkv, 1))
    for t0 in range(0, n, 16384):
        t1 = min(n, t0 + 16384)
        k[:, t0:t1] = ((0.7 * topics[:, at[t0:t1]] + randn(B, t1 - t0, Hkv, D)) * channel).to(dtype)
        v[:, t0:t1] = (randn(B, t1 - t0, Hkv, D) * level).to(dtype)
    k, v = k.transpose(1, 2), v.transpose(1, 2)  # [B, Hkv, n, D] views
    s = {"case": case}
    if case["op"] == "pack":
        s.update(k=k, v=v, rows=-(-N // TILE) * TILE)
        if own:
            s["archive"] = _package().PackedArchive(B * Hkv, s["rows"], D, device="cuda")
        return s
    # queries: towards the topic of some place in the context, at the last Lq positions
    where = torch.randint(0, n // 96 + 1, (B,), generator=g, device="cuda")
    toward = topics[torch.arange(B, device="cuda"), where].repeat_interleave(H // Hkv, dim=1)[:, :, None]
    s["q"] = 0.5 * toward + 0.7 * randn(B, H, Lq, D)
    s["pos"] = n - Lq
    if own:
        cache = _cache(case)
        start = 0
        for length in lens:
            cache.import_block(k[:, :, start:start + length], v[:, :, start:start + length], start)
            start += length
        cache.hot_start = N
        cache.append_exact(k[:, :, N:], v[:, :, N:])
        s["cache"], s["segments"] = cache, cache.get_attention_segments()
        return s
    tile = _tile_of_token(case)
    tiles = _n_tiles(case)
    s.update(tile=tile, hot_k=k[:, :, N:], hot_v=v[:, :, N:])
    ka, va = k[:, :, :N], v[:, :, :N]
    if case["packed"]:
        for name, x in (("k", ka), ("v", va)):
            scale = _scale(_tile_amax(x, tile, tiles))
            codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device="cuda")
            for b in range(B):
                codes[b] = (x[b].float() / scale[b][:, tile][..., None]).to(torch.float8_e4m3fn)
            s[name], s[name + "_scale"] = codes, scale
    else:
        s.update(k=ka.contiguous(), v=va.contiguous())
    if case["top"]:
        keys = _values(s, "k") if case["packed"] else s["k"]
        index = tile[:, None].expand(N, D)
        lo = torch.full((B, Hkv, tiles, D), float("inf"), device="cuda")
        s["lo"] = torch.stack([torch.stack([lo[b, h].scatter_reduce(0, index, keys[b, h].float(), "amin")
                                            for h in range(Hkv)]) for b in range(B)])
        s["hi"] = torch.stack([torch.stack([(-lo[b, h]).scatter_reduce(0, index, keys[b, h].float(), "amax")
                                            for h in range(Hkv)]) for b in range(B)])
        s["tile_pos"] = torch.zeros(tiles, dtype=torch.long, device="cuda").scatter_reduce(
            0, tile, torch.arange(N, device="cuda"), "amin", include_self=False)
    return s


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rfsn-mlx_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import rfsn_b200

    return rfsn_b200


def _cache(case):
    """What a program keeps: one layer's cache (with its archive), here without a model around it."""
    rfsn = _package()
    padded = sum(-(-n // TILE) * TILE for n in _block_lens(case))
    hot = max(1, case["hot"])
    room = max(hot, padded)
    cfg = rfsn.RFSNConfig(hidden_dim=case["heads"] * case["dim"], num_heads=case["heads"], num_kv_heads=case["kv_heads"],
                          head_dim=case["dim"], num_layers=1, hot_capacity=hot, warm_capacity=room, cold_capacity=room,
                          block_size_seq=min(hot, case["block"]), model_dtype=case["dtype"],
                          disk_cache_dir=os.path.join(tempfile.gettempdir(), "rfsn_perf"))
    return rfsn.LayerKVCache(cfg, case["batch"], case["heads"], case["kv_heads"], session_id="perf",
                             pool_tokens=padded, archive_dtype="float8_e4m3fn" if case["packed"] else None,
                             tile_index=case["top"] > 0)


# ------------------------------------------------------------------ plain forms
def _values(s, name):
    """The archived keys or values in float32."""
    if not s["case"]["packed"]:
        return s[name].float()
    return s[name].float() * s[name + "_scale"][:, :, s["tile"]][..., None]


def _plain_pack(s):
    out = {}
    for name in ("k", "v"):
        x = s[name]
        B, Hkv, n, D = x.shape
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, s["rows"] - n)).reshape(B * Hkv, -1, TILE, D)
        scale = _scale(x.abs().amax(dim=(2, 3)))
        out[name] = (x / scale[:, :, None, None]).to(torch.float8_e4m3fn).reshape(B * Hkv, -1, D)
        out[name + "_scale"] = scale
    return out


def _plain_select(s):
    """Tiles with the `top` largest bounds, ascending, -1 behind them."""
    case = s["case"]
    B, Hkv, G, Lq, D = case["batch"], case["kv_heads"], case["heads"] // case["kv_heads"], case["q_len"], case["dim"]
    q = s["q"].double().reshape(B, Hkv, G * Lq, D)
    up = q.clamp(min=0) @ s["hi"].double().transpose(-1, -2) + q.clamp(max=0) @ s["lo"].double().transpose(-1, -2)
    score = up.reshape(B, Hkv, G, Lq, -1).amax(dim=2).float()
    row = s["pos"] + torch.arange(Lq, device="cuda")
    score = torch.where(s["tile_pos"] <= row[:, None], score, torch.full_like(score, float("-inf")))
    order = torch.sort(score, dim=-1, descending=True, stable=True)
    best = torch.where(order.values > float("-inf"), order.indices, order.indices.shape[-1])[..., :case["top"]]
    best = torch.sort(best, dim=-1).values
    best = torch.where(best == order.indices.shape[-1], -1, best)
    return torch.nn.functional.pad(best, (0, case["top"] - best.shape[-1]), value=-1).int()


def _plain_attend(s, tiles=None):
    case = s["case"]
    B, H, Hkv, Lq, D = case["batch"], case["heads"], case["kv_heads"], case["q_len"], case["dim"]
    k = torch.cat([_values(s, "k"), s["hot_k"].float()], dim=2)
    v = torch.cat([_values(s, "v"), s["hot_v"].float()], dim=2)
    q = s["q"].reshape(B, Hkv, -1, D)
    score = (q @ k.transpose(-1, -2) / math.sqrt(D)).reshape(B, Hkv, H // Hkv, Lq, -1)
    n = k.shape[2]
    seen = torch.arange(n, device="cuda") <= s["pos"] + torch.arange(Lq, device="cuda")[:, None]
    if tiles is not None:
        chosen = torch.zeros(B, Hkv, Lq, int(s["tile_pos"].shape[0]) + 1, dtype=torch.bool, device="cuda")
        chosen = chosen.scatter(3, torch.where(tiles < 0, chosen.shape[3] - 1, tiles).long(), True)
        chosen = torch.cat([chosen[..., s["tile"]], chosen.new_ones(B, Hkv, Lq, n - s["tile"].shape[0])], dim=3)
        seen = (seen & chosen)[:, :, None]
    p = torch.exp(score - torch.where(seen, score, float("-inf")).amax(dim=-1, keepdim=True)) * seen
    out = (p.reshape(B, Hkv, -1, n) @ v) / p.sum(dim=-1).reshape(B, Hkv, -1, 1)
    return out.reshape(B, H, Lq, D)


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    op, top = case["op"], case["top"]
    if own:
        if op == "pack":
            a = s["archive"]
            a.pack(s["k"], s["v"], 0)
            return {"k": a.k, "v": a.v, "k_scale": a.k_scale, "v_scale": a.v_scale}
        if op == "select":
            return s["cache"].select_tiles(s["q"], s["pos"], top, s["segments"])
        return s["cache"].attend(s["q"], s["pos"], s["segments"], top_tiles=top)
    if op == "pack":
        return _plain_pack(s)
    if op == "select":
        return _plain_select(s)
    return _plain_attend(s, _plain_select(s) if top else None)


def work(case):
    B, H, Hkv, D, Lq, hot = (case[x] for x in ("batch", "heads", "kv_heads", "dim", "q_len", "hot"))
    N, T = sum(_block_lens(case)), _n_tiles(case)
    if case["op"] == "pack":
        return {"bytes": B * Hkv * (N * D * 4 + T * TILE * D * 2 + T * 8), "flops": 0}
    q_out = B * H * Lq * D * 8
    select = B * Hkv * T * D * 4
    if case["op"] == "select":
        return {"bytes": select + q_out / 2 + B * Hkv * Lq * case["top"] * 4, "flops": 2 * B * H * Lq * T * D}
    keys = N if not case["top"] else min(N, case["top"] * TILE)
    row = 2 * D + 8 / TILE if case["packed"] else 4 * D  # bytes of one archived key and value
    return {"bytes": B * Hkv * (keys * row + hot * D * 4) + q_out + (select if case["top"] else 0),
            "flops": 4 * B * H * D * Lq * (keys + hot - (Lq - 1) / 2) + (2 * B * H * Lq * T * D if case["top"] else 0)}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    global own
    asked, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = asked
    B, H, Hkv, D, Lq = (case[x] for x in ("batch", "heads", "kv_heads", "dim", "q_len"))
    G = H // Hkv
    if case["op"] == "pack":
        out = {}
        for name in ("k", "v"):
            code = torch.zeros(B * Hkv, s["rows"], D, dtype=torch.float64, device="cuda")
            scale = torch.ones(B * Hkv, s["rows"] // TILE, dtype=torch.float64, device="cuda")
            for i in range(B * Hkv):
                x = s[name][i // Hkv, i % Hkv].double()
                for t, part in enumerate(x.split(TILE)):
                    top = part.abs().max()
                    if top > 0:  # the largest power of two p <= top: top / p <= 1.75 fits 448 at p / 256
                        below = 2.0 ** torch.floor(torch.log2(top))
                        scale[i, t] = torch.where(top <= 1.75 * below, below / 256, below / 128)
                code[i, :x.shape[0]] = x / scale[i].repeat_interleave(TILE)[:x.shape[0], None]
            out[name], out[name + "_scale"] = code, scale
        return out
    if case["op"] == "select":
        return None  # whole numbers: they have to be equal
    n = s["pos"] + Lq
    N = n - case["hot"]
    out = torch.empty(B, H, Lq, D, dtype=torch.float64, device="cuda")
    tile, tiles = s["tile"], _n_tiles(case)
    for b in range(B):
        for h in range(Hkv):
            parts = []
            for name in ("k", "v"):
                x = s[name][b, h].double()
                if case["packed"]:
                    x = x * s[name + "_scale"][b, h].double()[tile][:, None]
                parts.append(torch.cat([x, s["hot_" + name][b, h].double()]))
            k, v = parts
            q = s["q"][b, h * G:(h + 1) * G].double()
            for r in range(0, Lq, 64):
                rows = torch.arange(r, min(Lq, r + 64), device="cuda")
                logits = torch.einsum("grd,nd->grn", q[:, rows], k) / math.sqrt(D)
                hide = torch.arange(n, device="cuda")[None] > (s["pos"] + rows)[:, None]
                if case["top"]:
                    bound = torch.stack([torch.maximum(q[:, i, None] * s["lo"][b, h].double(),
                                                       q[:, i, None] * s["hi"][b, h].double()).sum(-1).amax(0)
                                         for i in rows.tolist()]).float()
                    bound = bound.masked_fill(s["tile_pos"][None] > (s["pos"] + rows)[:, None], float("-inf"))
                    rank = torch.argsort(torch.argsort(bound, dim=1, descending=True, stable=True), dim=1)
                    hide[:, :N] |= (rank >= min(case["top"], tiles))[:, tile]
                out[b, h * G:(h + 1) * G, rows] = torch.softmax(logits.masked_fill(hide, float("-inf")), -1) @ v
    return out
