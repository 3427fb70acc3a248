// Tile selection: for every (query row, KV head) the n tiles whose keys can
// reach the largest logit, by the channel-wise bounds lo, hi of each tile:
//   score(tile) = max over the group's q heads of
//                 sum_d max(q_d lo_d, q_d hi_d)  >=  q . k  for every key k of the tile
// Tiles that begin behind the query are not scored. The n largest scores win,
// equal scores by the lowest tile number; the list comes out in tile order.
//
// The choice must not hang on rounding: q (float32) times a 16- or 8-bit bound
// is exact in 64 bits and the sums are taken there, then rounded to float32
// once, so any order of summation gives the same scores (up to a chance of
// about 1e-9 per score) and the same lists. The B200's 64-bit rate (64 FMA per
// SM and clock) makes that cheaper than it sounds: 2,067 tiles x 32 heads x
// 128 channels are 8.5 M FMA, 0.5 us.
//
// One launch: each CTA scores a range of tiles of one list and the last CTA
// of the list to arrive selects. Bound by launch, arrival and the selection's
// chain of counts; the bounds (8.4 MB at 132K tokens) are 1.3 us of HBM time.
#include <math_constants.h>

#include "archive.cuh"

namespace rfsn {
namespace archive {

constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kHeadsPerPass = 4;

template <typename T> struct BoundVec;  // 8 bounds -> float
template <> struct BoundVec<__nv_bfloat16> {
    static constexpr int kBytes = 16;
    uint4 w;
    __device__ __forceinline__ void load(const void* p) { w = __ldg(static_cast<const uint4*>(p)); }
    __device__ __forceinline__ float get(int i) const {
        const uint32_t x = (&w.x)[i >> 1];
        return __uint_as_float((i & 1) ? (x & 0xffff0000u) : (x << 16));
    }
};
template <> struct BoundVec<__half> {
    static constexpr int kBytes = 16;
    uint4 w;
    __device__ __forceinline__ void load(const void* p) { w = __ldg(static_cast<const uint4*>(p)); }
    __device__ __forceinline__ float get(int i) const {
        const uint32_t x = (&w.x)[i >> 1];
        return __half2float(__ushort_as_half((unsigned short)((i & 1) ? (x >> 16) : (x & 0xffffu))));
    }
};
template <> struct BoundVec<uint8_t> {  // e4m3
    static constexpr int kBytes = 8;
    uint2 w;
    __device__ __forceinline__ void load(const void* p) { w = __ldg(static_cast<const uint2*>(p)); }
    __device__ __forceinline__ float get(int i) const {
        const uint32_t x = (&w.x)[i >> 2] >> (8 * (i & 3));
        return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)(x & 0xffu), __NV_E4M3)));
    }
};

// Order-preserving 32-bit key of a score; 0 for tiles that cannot be chosen
// (behind the query, or a bound of -inf); a NaN score comes first.
__device__ __forceinline__ uint32_t score_key(float s) {
    if (s != s) return 0xffffffffu;
    if (s == -CUDART_INF_F) return 0u;
    const uint32_t b = __float_as_uint(s);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Selection of one list by one CTA, up to kSelRegKeys * 256 tiles: the keys
// stay in registers (key i of a thread is tile 256 i + thread).
constexpr int kSelRegKeys = 16;

struct SelShared {
    int flag;
    int count[2][kSelWarps];
    uint32_t any[kSelWarps], all[kSelWarps];
    alignas(16) int tally[kSelRegKeys * kSelWarps];  // tiles above (low half) and at (high half) the threshold
};

// The n-th largest key by bisection over the key's bits, two bits a round: a
// count for each of three candidate thresholds (packed into one word per warp:
// a warp holds at most 512 keys), skipping the leading bits that all keys
// share and stopping as soon as a threshold holds exactly n keys.
__device__ __forceinline__ void select_in_registers(const SelectParams& p, const float* scores, int4* out,
                                                    SelShared& sh) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int T_ = p.n_tiles;
    uint32_t key[kSelRegKeys];
    uint32_t any = 0u, all = 0xffffffffu;
    int visible = 0;
#pragma unroll
    for (int i = 0; i < kSelRegKeys; ++i) {
        const int t = tid + kSelThreads * i;
        key[i] = t < T_ ? score_key(__ldcg(scores + t)) : 0u;
    }
#pragma unroll
    for (int i = 0; i < kSelRegKeys; ++i)
        if (key[i] != 0u) {
            ++visible;
            any |= key[i];
            all &= key[i];
        }
    any = __reduce_or_sync(0xffffffffu, any);
    all = __reduce_and_sync(0xffffffffu, all);
    visible = __reduce_add_sync(0xffffffffu, visible);
    if (lane == 0) {
        sh.any[warp] = any;
        sh.all[warp] = all;
        sh.count[1][warp] = visible;
    }
    __syncthreads();
    visible = 0;
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) {
        any |= sh.any[w];
        all &= sh.all[w];
        visible += sh.count[1][w];
    }
    const int n = min(p.n_select, visible);
    uint32_t thr = 1u;  // every visible tile
    if (n < visible) {
        const uint32_t differ = any ^ all;
        int bit = differ ? 31 - __clz(differ) : -1;
        if (bit >= 0 && !(bit & 1)) ++bit;  // bit pairs: (31, 30) .. (1, 0)
        thr = bit < 31 ? (any >> (bit + 1)) << (bit + 1) : 0u;  // the bits all keys share
        int round = 0;
        for (; bit >= 0; bit -= 2, round ^= 1) {
            const uint32_t step = 1u << (bit - 1);
            int c = 0;
#pragma unroll
            for (int i = 0; i < kSelRegKeys; ++i)
                if (i * kSelThreads < T_)
                    c += (int)(key[i] >= thr + step) + ((int)(key[i] >= thr + 2 * step) << 10) +
                         ((int)(key[i] >= thr + 3 * step) << 20);
            c = __reduce_add_sync(0xffffffffu, c);
            if (lane == 0) sh.count[round][warp] = c;
            __syncthreads();  // the other buffer is written only after every thread has passed here again
            int c1 = 0, c2 = 0, c3 = 0;
#pragma unroll
            for (int w = 0; w < kSelWarps; ++w) {
                const int x = sh.count[round][w];
                c1 += x & 1023;
                c2 += (x >> 10) & 1023;
                c3 += x >> 20;
            }
            const int up = c3 >= n ? 3 : c2 >= n ? 2 : c1 >= n ? 1 : 0;
            thr += up * step;
            if ((up == 3 && c3 == n) || (up == 2 && c2 == n) || (up == 1 && c1 == n)) break;
        }
    }
    // Write in tile order: keys above the threshold all, keys equal to it from the lowest tile on.
#pragma unroll
    for (int i = 0; i < kSelRegKeys; ++i) {
        const unsigned mg = __ballot_sync(0xffffffffu, key[i] > thr), me = __ballot_sync(0xffffffffu, key[i] == thr);
        if (lane == 0) sh.tally[i * kSelWarps + warp] = __popc(mg) | __popc(me) << 16;
    }
    __syncthreads();
    static_assert(kSelRegKeys * kSelWarps == 128, "four tallies per lane");
    const int4 four = reinterpret_cast<const int4*>(sh.tally)[lane];
    int incl = four.x + four.y + four.z + four.w;
    const int own = incl;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
    }
    const int need = n - (__shfl_sync(0xffffffffu, incl, 31) & 0xffff);  // tiles taken among those at the threshold
    const int part = (warp & 3) > 0 ? four.x + ((warp & 3) > 1 ? four.y : 0) + ((warp & 3) > 2 ? four.z : 0) : 0;
    const int mine = incl - own + part;  // tallies before (i, warp) when the lane holds that entry
    const unsigned below = (1u << lane) - 1u;
#pragma unroll
    for (int i = 0; i < kSelRegKeys; ++i) {
        if (i * kSelThreads >= T_) break;
        const int before = __shfl_sync(0xffffffffu, mine, 2 * i + (warp >> 2));
        const bool gt = key[i] > thr, eq = key[i] == thr;
        const unsigned mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
        const int g = (before & 0xffff) + __popc(mg & below), e = (before >> 16) + __popc(me & below);
        if (gt || (eq && e < need)) {
            const int t = tid + kSelThreads * i;
            int4 x = __ldg(p.tiles + t);
            x.w = t;
            out[g + min(e, need)] = x;
        }
    }
    for (int i = n + tid; i < p.n_select; i += kSelThreads) out[i] = make_int4(0, 0, 0, -1);
}

// The same for any number of tiles: a bit a round, the scores read again from
// the workspace (L2) for each.
__device__ __forceinline__ void select_in_memory(const SelectParams& p, const float* scores, int4* out, SelShared& sh) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int T_ = p.n_tiles;
    auto key_at = [&](int t) { return score_key(__ldcg(scores + t)); };
    auto block_sum = [&](int c) {
        c = __reduce_add_sync(0xffffffffu, c);
        __syncthreads();  // the previous sum has been read
        if (lane == 0) sh.count[0][warp] = c;
        __syncthreads();
        c = 0;
#pragma unroll
        for (int w = 0; w < kSelWarps; ++w) c += sh.count[0][w];
        return c;
    };
    int visible = 0;
    for (int t = tid; t < T_; t += kSelThreads) visible += key_at(t) != 0u;
    visible = block_sum(visible);
    const int n = min(p.n_select, visible);
    uint32_t thr = 1u;
    if (n < visible) {
        thr = 0u;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t cand = thr | (1u << bit);
            int c = 0;
            for (int t = tid; t < T_; t += kSelThreads) c += key_at(t) >= cand;
            c = block_sum(c);
            if (c >= n) thr = cand;
            if (c == n) break;
        }
    }
    // each warp owns a run of tiles
    const int run = ((T_ + kSelWarps - 1) / kSelWarps + 31) / 32 * 32;
    const int r0 = min(warp * run, T_), r1 = min(r0 + run, T_);
    int gt = 0, eq = 0;
    for (int t = r0 + lane; t < r1; t += 32) {
        const uint32_t k = key_at(t);
        gt += k > thr;
        eq += k == thr;
    }
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) {
        sh.tally[warp] = gt;
        sh.tally[kSelWarps + warp] = eq;
    }
    __syncthreads();
    int gt_before = 0, eq_before = 0, gt_all = 0;
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) {
        if (w < warp) {
            gt_before += sh.tally[w];
            eq_before += sh.tally[kSelWarps + w];
        }
        gt_all += sh.tally[w];
    }
    const int need = n - gt_all;
    const unsigned below = (1u << lane) - 1u;
    for (int t0 = r0; t0 < r1; t0 += 32) {
        const int t = t0 + lane;
        const uint32_t k = t < r1 ? key_at(t) : 0u;
        const bool is_gt = t < r1 && k > thr, is_eq = t < r1 && k == thr;
        const unsigned mg = __ballot_sync(0xffffffffu, is_gt), me = __ballot_sync(0xffffffffu, is_eq);
        const int g = gt_before + __popc(mg & below), e = eq_before + __popc(me & below);
        if (is_gt || (is_eq && e < need)) {
            int4 x = __ldg(p.tiles + t);
            x.w = t;
            out[g + min(e, need)] = x;
        }
        gt_before += __popc(mg);
        eq_before += __popc(me);
    }
    for (int i = n + tid; i < p.n_select; i += kSelThreads) out[i] = make_int4(0, 0, 0, -1);
}

// Eight lanes score a tile, 32 tiles at a time per CTA; the tile's bounds are
// requested before the wait for q (they never come from the kernel that this
// launch overlaps: packing and bounding are launched without that overlap).
template <typename T, int D>
__global__ void __launch_bounds__(kSelThreads) select_kernel(const SelectParams p) {
    constexpr int NV = D / 64;  // vectors of 8 channels per lane
    __shared__ double2 qs[kHeadsPerPass * D / 2];
    __shared__ SelShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int list = blockIdx.y;
    const int row = list % p.q_len, bh = list / p.q_len;
    const int b = bh / p.kv_heads, hk = bh % p.kv_heads;
    const int t_begin = blockIdx.x * p.tiles_per_cta;
    const int t_end = min(t_begin + p.tiles_per_cta, p.n_tiles);
    float* scores = p.scores + (size_t)list * p.n_tiles;
    const int sub = lane >> 3, l8 = lane & 7;

    struct Fetched {
        int4 e;
        BoundVec<T> lo[NV], hi[NV];
        float sk;
    };
    auto fetch = [&](int t) {
        Fetched f;
        f.e = make_int4(0, 0, 0, 0);
        f.sk = 1.f;
        if (t < t_end) f.e = __ldg(p.tiles + t);
        if ((f.e.x & (kTile - 1)) != 0 || f.e.x < 0 || f.e.x / kTile >= p.tile_slots) {
            atomicExch(p.error, kDevErrBadTable);
            f.e.z = 0;
        }
        if (f.e.z > 0) {
            const size_t slot = (size_t)bh * p.tile_slots + f.e.x / kTile;
            if (sizeof(T) == 1) f.sk = __ldg(p.scales + slot).x;
            const char* base = static_cast<const char*>(p.bounds) + slot * 2 * D * sizeof(T);
#pragma unroll
            for (int v = 0; v < NV; ++v) {  // lanes read consecutive vectors
                const int d0 = 8 * (l8 + 8 * v);
                f.lo[v].load(base + d0 * sizeof(T));
                f.hi[v].load(base + (D + d0) * sizeof(T));
            }
        }
        return f;
    };
    Fetched next = fetch(t_begin + 4 * warp + sub);

    griddep_wait();  // q, the step state and the workspace may belong to the kernel this one overlaps
    griddep_launch_dependents();
    const int qpos = (p.dyn != nullptr ? p.dyn[RFSN_STEP_POS] : p.q_pos0) + row;
    for (int g0 = 0; g0 < p.G; g0 += kHeadsPerPass) {
        const int heads = min(kHeadsPerPass, p.G - g0);
        if (g0 > 0) {
            __syncthreads();
            next = fetch(t_begin + 4 * warp + sub);
        }
        for (int i = tid; i < kHeadsPerPass * D / 2; i += kSelThreads) {
            // pairs of channels 8 (l8 + 8 v) + 2 j, + 1 of a head at [head][4 v + j][l8]: lanes side by side
            const int g = i / (D / 2), pr = i % (D / 2);
            const int d = 8 * ((pr & 7) + 8 * (pr >> 5)) + 2 * ((pr >> 3) & 3);
            float2 x = make_float2(0.f, 0.f);
            if (g < heads)
                x = *reinterpret_cast<const float2*>(
                    p.q + (((size_t)b * p.q_heads + hk * p.G + g0 + g) * p.q_len + row) * D + d);
            qs[i] = make_double2((double)x.x, (double)x.y);
        }
        __syncthreads();
        for (int t0 = t_begin; t0 < t_end; t0 += kSelWarps * 4) {
            const int t = t0 + 4 * warp + sub;
            const Fetched f = next;
            if (t0 + kSelWarps * 4 < t_end) next = fetch(t + kSelWarps * 4);
            const bool live = t < t_end && f.e.z > 0 && f.e.y <= qpos;
            double acc[kHeadsPerPass];
#pragma unroll
            for (int g = 0; g < kHeadsPerPass; ++g) acc[g] = 0.0;
            if (live) {
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const double l0 = (double)f.lo[v].get(2 * j), h0 = (double)f.hi[v].get(2 * j);
                        const double l1 = (double)f.lo[v].get(2 * j + 1), h1 = (double)f.hi[v].get(2 * j + 1);
#pragma unroll
                        for (int g = 0; g < kHeadsPerPass; ++g) {
                            const double2 q2 = qs[g * (D / 2) + (4 * v + j) * 8 + l8];
                            acc[g] += q2.x * (q2.x >= 0.0 ? h0 : l0);
                            acc[g] += q2.y * (q2.y >= 0.0 ? h1 : l1);
                        }
                    }
            }
            // Sums over the 8 lanes, halving the heads a lane carries: lanes end with head 2 (l8 / 4) + (l8 / 2) % 2.
            static_assert(kHeadsPerPass == 4, "two halvings");
            const bool up4 = l8 & 4, up2 = l8 & 2;
            const double s0 = __shfl_xor_sync(0xffffffffu, up4 ? acc[0] : acc[2], 4);
            const double s1 = __shfl_xor_sync(0xffffffffu, up4 ? acc[1] : acc[3], 4);
            const double a0 = (up4 ? acc[2] : acc[0]) + s0, a1 = (up4 ? acc[3] : acc[1]) + s1;
            double a = (up2 ? a1 : a0) + __shfl_xor_sync(0xffffffffu, up2 ? a0 : a1, 2);
            a += __shfl_xor_sync(0xffffffffu, a, 1);
            const int head = (up4 ? 2 : 0) + (up2 ? 1 : 0);
            float best = head < heads ? (float)(a * (double)f.sk) : -CUDART_INF_F;
            unsigned nan = __ballot_sync(0xffffffffu, best != best);
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 4));
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
            if (l8 == 0 && t < t_end) {
                if ((nan >> (8 * sub)) & 0xffu) best = CUDART_NAN_F;
                if (!live) best = -CUDART_INF_F;
                if (g0 > 0) {  // heads of the earlier passes
                    const float prev = scores[t];
                    best = (prev != prev || best != best) ? CUDART_NAN_F : fmaxf(prev, best);
                }
                scores[t] = best;
            }
        }
    }
    __syncthreads();
    if (gridDim.x > 1) {
        if (tid == 0) sh.flag = atom_add_acq_rel_gpu(&p.counters[list], 1) == (int)gridDim.x - 1;
        __syncthreads();
        if (!sh.flag) return;
    }
    int4* out = p.out + (size_t)list * p.n_select;
    if (p.n_tiles <= kSelRegKeys * kSelThreads)
        select_in_registers(p, scores, out, sh);
    else
        select_in_memory(p, scores, out, sh);
    if (gridDim.x > 1 && tid == 0) p.counters[list] = 0;
}

template <typename T, int D>
rfsn_status launch(const SelectParams& p, int lists, int chunks, cudaStream_t s) {
    RFSN_CUDA(launch_pdl(select_kernel<T, D>, dim3(chunks, lists), dim3(kSelThreads), 0, s, p));
    note_launch();
    return RFSN_OK;
}

template <typename T>
void preload() {
    cudaFuncAttributes a;
    cudaFuncGetAttributes(&a, select_kernel<T, 64>);
    cudaFuncGetAttributes(&a, select_kernel<T, 128>);
}

}  // namespace archive

void preload_select_kernels() {
    archive::preload<uint8_t>();
    archive::preload<__half>();
    archive::preload<__nv_bfloat16>();
}

rfsn_status select_tiles_launch(int bounds_dtype, int head_dim, const archive::SelectParams& p, int lists, int chunks,
                                cudaStream_t s) {
    using namespace archive;
    const bool d128 = head_dim == 128;
    if (bounds_dtype == RFSN_E4M3)
        return d128 ? launch<uint8_t, 128>(p, lists, chunks, s) : launch<uint8_t, 64>(p, lists, chunks, s);
    if (bounds_dtype == RFSN_F16)
        return d128 ? launch<__half, 128>(p, lists, chunks, s) : launch<__half, 64>(p, lists, chunks, s);
    return d128 ? launch<__nv_bfloat16, 128>(p, lists, chunks, s) : launch<__nv_bfloat16, 64>(p, lists, chunks, s);
}

}  // namespace rfsn
