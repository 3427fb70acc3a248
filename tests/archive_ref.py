"""Plain 64-bit forms of the packed archive, tile selection and attention over tiles (test infrastructure)."""

from __future__ import annotations

import math

import torch

TILE = 64


def scale_of(amax: float) -> float:
    """Smallest power of two s with amax / s <= 448 (1 for 0), exponent at least -126."""
    if amax == 0.0:
        return 1.0
    s = 2.0 ** math.floor(math.log2(amax) - 9)
    while amax / s > 448.0:
        s *= 2.0
    return max(s, 2.0 ** -126)


def pack(x: torch.Tensor):
    """x [G, n, D] -> (values [G, n, D] float64, scales [G, tiles], codes as float64): tiles of 64 from the first row."""
    G, n, D = x.shape
    x = x.double().cpu()
    codes = torch.zeros_like(x)
    scales = torch.ones(G, (n + TILE - 1) // TILE, dtype=torch.float64)
    for g in range(G):
        for t in range(scales.shape[1]):
            part = x[g, t * TILE:(t + 1) * TILE]
            finite = part[torch.isfinite(part)]
            s = scale_of(float(finite.abs().max()) if finite.numel() else 0.0)
            scales[g, t] = s
            y = torch.where(part.abs() == math.inf, torch.full_like(part, math.nan), part / s)
            codes[g, t * TILE:(t + 1) * TILE] = e4m3(y)
    return codes * scales.repeat_interleave(TILE, dim=1)[:, :n, None], scales, codes


def e4m3(y: torch.Tensor) -> torch.Tensor:
    """Round to nearest even among the e4m3 values (|y| <= 448): 3 mantissa bits, exponent at least -6."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))).clamp(max=8.0)
    step = torch.exp2(e - 3)
    return torch.where(torch.isnan(y), y, torch.round(y / step) * step)  # torch.round is to even


def tiles_of(lens):
    """[(block, first token in the block, tokens)] of the tiles."""
    return [(b, o, min(TILE, n - o)) for b, n in enumerate(lens) for o in range(0, n, TILE)]


def attention(q, k, v, key_pos, q_pos, seen=None):
    """q [B, H, Lq, D], k / v [B, Hkv, N, D], key_pos [N]; row r at q_pos + r sees key_pos <= it, and where given
    seen [B, Hkv, Lq, N]. -> (out, lse) float64; rows that see nothing give 0 and -inf."""
    B, H, Lq, D = q.shape
    Hkv = k.shape[1]
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    row = q_pos + torch.arange(Lq)
    ok = (key_pos[None] <= row[:, None])[None, None].expand(B, Hkv, Lq, -1)
    if seen is not None:
        ok = ok & seen.cpu()
    ok = ok.repeat_interleave(H // Hkv, dim=1)
    kk, vv = k.repeat_interleave(H // Hkv, dim=1), v.repeat_interleave(H // Hkv, dim=1)
    s = torch.einsum("bhrd,bhnd->bhrn", q, kk) / math.sqrt(D)
    s = torch.where(ok, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.where(ok, torch.exp(s - m), torch.zeros_like(s))
    l = p.sum(-1, keepdim=True)
    out = torch.einsum("bhrn,bhnd->bhrd", p, torch.where(ok.any(2)[..., None], vv, torch.zeros_like(vv)))
    out = torch.where(l > 0, out / l, torch.where(l == 0, torch.zeros_like(out), out / l))
    return out, (m + torch.log(l))[..., 0]


def select(q, lo, hi, tile_pos, q_pos, top):
    """lo, hi [B, Hkv, T, D] float64 -> int tensor [B, Hkv, Lq, top] of tile numbers, ascending, -1 behind them."""
    B, H, Lq, D = q.shape
    Hkv, T = lo.shape[1], lo.shape[2]
    q = q.double().cpu().reshape(B, Hkv, H // Hkv, Lq, D)
    out = torch.full((B, Hkv, Lq, top), -1, dtype=torch.int64)
    for b in range(B):
        for h in range(Hkv):
            for r in range(Lq):
                x = q[b, h, :, r][:, None]  # [G, 1, D]
                s = torch.maximum(x * lo[b, h].cpu(), x * hi[b, h].cpu()).sum(-1).amax(0).float()
                nan = torch.isnan(torch.maximum(x * lo[b, h].cpu(), x * hi[b, h].cpu()).sum(-1)).any(0)
                order = [(not bool(nan[t]), -float(s[t]) if not nan[t] else 0.0, t) for t in range(T)
                         if tile_pos[t] <= q_pos + r and (bool(nan[t]) or float(s[t]) > -math.inf)]
                best = sorted(t for _, _, t in sorted(order)[:top])
                out[b, h, r, :len(best)] = torch.tensor(best, dtype=torch.int64)
    return out


def bounds(keys, lens):
    """keys [B, Hkv, N, D] (archived, block after block) -> lo, hi [B, Hkv, T, D], first positions [T]."""
    lo, hi, pos, at = [], [], [], 0
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    for b, o, n in tiles_of(lens):
        at = starts[b] + o
        part = keys[:, :, at:at + n].double().cpu()
        lo.append(part.amin(2))
        hi.append(part.amax(2))
        pos.append(at)
    return torch.stack(lo, 2), torch.stack(hi, 2), torch.tensor(pos)
