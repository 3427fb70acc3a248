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
// of the list to arrive selects. Bound by the chain of launch, bounds, arrival
// and counts: 128 of 2,064 tiles 9.1 us, 16 of 96 6.6 us (32 q / 8 KV heads);
// the bounds (8.4 MB at 132K tokens) are 1.3 us of HBM time.
#include <math_constants.h>

#include "archive.cuh"

namespace rfsn {
namespace archive {

constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kHeadsPerPass = 4;  // of a warp

// Eight lanes score kTilesPerLane tiles side by side (each q pair fetched from
// shared memory serves all of them), kPassTiles at a time per CTA. With more
// than four q heads per KV head the warps are shared out over up to eight
// groups of four heads, and a CTA takes as many tiles less at a time (32 heads
// of 1 KV head, 78 tiles: 31.3 us with the groups one after the other in one
// CTA, 8.5 us side by side in five). The first pass's tiles and bounds are
// requested before the wait for q: a call whose bounds or scales may have been
// written by the kernel before it is launched without the overlap.
constexpr int kTilesPerLane = 2;
constexpr int kPassTiles = kSelWarps * 4 * kTilesPerLane;
constexpr int kMaxHeadGroups = 8;

template <typename T> struct BoundVec;  // 8 bounds -> float
template <> struct BoundVec<__nv_bfloat16> {
    uint4 w;
    __device__ __forceinline__ void clear() { w = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void load(const void* p) { w = __ldcg(static_cast<const uint4*>(p)); }
    __device__ __forceinline__ float get(int i) const {
        const uint32_t x = (&w.x)[i >> 1];
        return __uint_as_float((i & 1) ? (x & 0xffff0000u) : (x << 16));
    }
};
template <> struct BoundVec<__half> {
    uint4 w;
    __device__ __forceinline__ void clear() { w = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void load(const void* p) { w = __ldcg(static_cast<const uint4*>(p)); }
    __device__ __forceinline__ float get(int i) const {
        const uint32_t x = (&w.x)[i >> 1];
        return __half2float(__ushort_as_half((unsigned short)((i & 1) ? (x >> 16) : (x & 0xffffu))));
    }
};
template <> struct BoundVec<uint8_t> {  // e4m3
    uint2 w;
    __device__ __forceinline__ void clear() { w = make_uint2(0, 0); }
    __device__ __forceinline__ void load(const void* p) { w = __ldcg(static_cast<const uint2*>(p)); }
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

// Selection of one list by one CTA. Up to kSelRegKeys * kSelThreads tiles the
// keys stay in registers (key i of a thread is tile kSelThreads i + thread);
// longer lists read their scores again from the workspace (L2) in each pass.
constexpr int kSelRegKeys = 8;
constexpr int kBuckets = 2 * kSelThreads;

struct SelShared {
    int flag;
    uint32_t lo[kSelWarps], hi[kSelWarps];
    int visible[kSelWarps], total[kSelWarps];
    int bucket, above, inside;
    int hist[kBuckets];
    alignas(16) int tally[kSelRegKeys * kSelWarps];  // tiles above (low half) and at (high half) the threshold
    float part[kSelWarps * 4 * kTilesPerLane];       // scores by head group
};

// The n-th largest key by narrowing a key range [lo, lo + span]: a histogram of
// up to 1,024 equal buckets of 2^shift keys, the bucket in which the count from
// the top passes n becomes the range, and the keys above it, which are taken,
// are not counted again (a range of fewer than 1,024 keys has fewer buckets).
// Two passes as a rule (the first bucket holds a few scores, the second
// separates them), four at most; integer counts, so any order gives the same.
template <bool REGS>
__device__ __forceinline__ void select_list(const SelectParams& p, const float* scores, int list, SelShared& sh) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int T_ = p.n_tiles;
    uint32_t key[REGS ? kSelRegKeys : 1];
    if (REGS) {
#pragma unroll
        for (int i = 0; i < kSelRegKeys; ++i) {
            const int t = tid + kSelThreads * i;
            key[REGS ? i : 0] = t < T_ ? score_key(__ldcg(scores + t)) : 0u;
        }
    }
    auto each = [&](auto&& f) {  // f(key) for the thread's keys
        if (REGS) {
#pragma unroll
            for (int i = 0; i < kSelRegKeys; ++i)
                if (i * kSelThreads < T_) f(key[REGS ? i : 0]);
        } else {
            for (int t = tid; t < T_; t += kSelThreads) f(score_key(__ldcg(scores + t)));
        }
    };
    uint32_t lo = 0xffffffffu, hi = 0u;
    int visible = 0;
    each([&](uint32_t k) {
        if (k != 0u) {
            ++visible;
            lo = min(lo, k);
            hi = max(hi, k);
        }
    });
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    visible = __reduce_add_sync(0xffffffffu, visible);
    if (lane == 0) {
        sh.lo[warp] = lo;
        sh.hi[warp] = hi;
        sh.visible[warp] = visible;
    }
    sh.hist[tid] = sh.hist[tid + kSelThreads] = 0;
    __syncthreads();
    visible = 0;
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) {
        lo = min(lo, sh.lo[w]);
        hi = max(hi, sh.hi[w]);
        visible += sh.visible[w];
    }
    const int n = min(p.n_select, visible);
    uint32_t thr = 1u;  // every visible tile
    if (n < visible) {
        int need = n;
        uint32_t span = hi - lo;
        int shift = max(0, 32 - __clz(span) - 10);  // span + 1 keys in at most 1,024 buckets
        for (;;) {
            each([&](uint32_t k) {
                if (k - lo <= span) atomicAdd(&sh.hist[(k - lo) >> shift], 1);  // keys below lo wrap around
            });
            __syncthreads();
            // counts from the top: thread i has buckets 1023 - 2 i and 1022 - 2 i
            const int h1 = sh.hist[kBuckets - 1 - 2 * tid], h0 = sh.hist[kBuckets - 2 - 2 * tid];
            int incl = h0 + h1;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, off);
                if (lane >= off) incl += v;
            }
            if (lane == 31) sh.total[warp] = incl;
            __syncthreads();
            sh.hist[tid] = sh.hist[tid + kSelThreads] = 0;  // every thread has read its buckets
#pragma unroll
            for (int w = 0; w < kSelWarps; ++w)
                if (w < warp) incl += sh.total[w];
            const int before = incl - h0 - h1;
            if (before < need && incl >= need) {
                const bool first = before + h1 >= need;
                sh.bucket = kBuckets - (first ? 1 : 2) - 2 * tid;
                sh.above = before + (first ? 0 : h1);
                sh.inside = first ? h1 : h0;
            }
            __syncthreads();
            lo += (uint32_t)sh.bucket << shift;
            need -= sh.above;
            if (sh.inside == need || shift == 0) break;
            span = min((1u << shift) - 1u, hi - lo);  // the last bucket may reach beyond the largest key
            shift = max(0, shift - 10);
        }
        thr = lo;
    }
    // Write in tile order: keys above the threshold all, keys equal to it from
    // the lowest tile on (all of them, unless the bucket was one key). Entries
    // behind the ones written, by their own count, are filled.
    int written;
    const unsigned below = (1u << lane) - 1u;
    const size_t base = (size_t)list * p.n_select;
    auto put = [&](int i, int t) {
        if (p.numbers != nullptr) {
            p.numbers[base + i] = t;
            return;
        }
        int4 x = make_int4(0, 0, 0, -1);
        if (t >= 0) {
            x = __ldg(p.tiles + t);
            x.w = t;
        }
        p.out[base + i] = x;
    };
    if (REGS) {
#pragma unroll
        for (int i = 0; i < kSelRegKeys; ++i) {
            const uint32_t k = key[REGS ? i : 0];
            const unsigned mg = __ballot_sync(0xffffffffu, k > thr), me = __ballot_sync(0xffffffffu, k == thr);
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
        const int all = __shfl_sync(0xffffffffu, incl, 31);
        const int need = n - (all & 0xffff);  // taken among those at the threshold
        written = (all & 0xffff) + min(all >> 16, need);
        const int w3 = warp & 3;
        const int part = (w3 > 0 ? four.x : 0) + (w3 > 1 ? four.y : 0) + (w3 > 2 ? four.z : 0);
        const int mine = incl - own + part;  // tallies before (i, warp), in the lane that holds that entry
#pragma unroll
        for (int i = 0; i < kSelRegKeys; ++i) {
            if (i * kSelThreads >= T_) break;
            const uint32_t k = key[REGS ? i : 0];
            const int before = __shfl_sync(0xffffffffu, mine, (i * kSelWarps + warp) >> 2);
            const bool gt = k > thr, eq = k == thr;
            const unsigned mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
            const int g = (before & 0xffff) + __popc(mg & below), e = (before >> 16) + __popc(me & below);
            if (gt || (eq && e < need)) put(g + min(e, need), tid + kSelThreads * i);
        }
    } else {
        // each warp owns a run of tiles
        const int run = ((T_ + kSelWarps - 1) / kSelWarps + 31) / 32 * 32;
        const int r0 = min(warp * run, T_), r1 = min(r0 + run, T_);
        int gt = 0, eq = 0;
        for (int t = r0 + lane; t < r1; t += 32) {
            const uint32_t k = score_key(__ldcg(scores + t));
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
        int gt_before = 0, eq_before = 0, gt_all = 0, eq_all = 0;
#pragma unroll
        for (int w = 0; w < kSelWarps; ++w) {
            if (w < warp) {
                gt_before += sh.tally[w];
                eq_before += sh.tally[kSelWarps + w];
            }
            gt_all += sh.tally[w];
            eq_all += sh.tally[kSelWarps + w];
        }
        const int need = n - gt_all;
        written = gt_all + min(eq_all, need);
        for (int t0 = r0; t0 < r1; t0 += 32) {
            const int t = t0 + lane;
            const uint32_t k = t < r1 ? score_key(__ldcg(scores + t)) : 0u;
            const bool is_gt = t < r1 && k > thr, is_eq = t < r1 && k == thr;
            const unsigned mg = __ballot_sync(0xffffffffu, is_gt), me = __ballot_sync(0xffffffffu, is_eq);
            const int g = gt_before + __popc(mg & below), e = eq_before + __popc(me & below);
            if (is_gt || (is_eq && e < need)) put(g + min(e, need), t);
            gt_before += __popc(mg);
            eq_before += __popc(me);
        }
    }
    for (int i = written + tid; i < p.n_select; i += kSelThreads) put(i, -1);
}

// A bound as a double has an empty low word (8 or 11 significant bits), so the
// choice between lo and hi by the sign of q is one word.
__device__ __forceinline__ double pick(bool up, int hi_hi, int hi_lo) { return __hiloint2double(up ? hi_hi : hi_lo, 0); }

template <typename T, int D>
__global__ void __launch_bounds__(kSelThreads) select_kernel(const SelectParams p) {
    constexpr int NV = D / 64;  // vectors of 8 channels per lane
    constexpr int U = kTilesPerLane;
    __shared__ double2 qs[kMaxHeadGroups * kHeadsPerPass * D / 2];
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
        if (t < t_end) f.e = __ldcg(p.tiles + t);
        if (f.e.z > 0 && ((f.e.x & (kTile - 1)) != 0 || f.e.x < 0 || f.e.x / kTile >= p.tile_slots)) {
            atomicExch(p.error, kDevErrBadTable);
            f.e.z = 0;
        }
        const size_t slot = (size_t)bh * p.tile_slots + (f.e.z > 0 ? f.e.x / kTile : 0);
        const char* base = static_cast<const char*>(p.bounds) + slot * 2 * D * sizeof(T);
#pragma unroll
        for (int v = 0; v < NV; ++v) {  // lanes read consecutive vectors
            f.lo[v].clear();
            f.hi[v].clear();
        }
        if (f.e.z > 0) {
            if (sizeof(T) == 1) f.sk = __ldcg(p.scales + slot).x;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int d0 = 8 * (l8 + 8 * v);
                f.lo[v].load(base + d0 * sizeof(T));
                f.hi[v].load(base + (D + d0) * sizeof(T));
            }
        }
        return f;
    };
    const int groups = p.head_groups, group_warps = kSelWarps / groups, pass_tiles = kPassTiles / groups;
    const int group = warp / group_warps, slot = U * (4 * (warp % group_warps) + sub);  // of the pass's tiles
    const int t_lane = t_begin + slot;
    Fetched f[U];
#pragma unroll
    for (int u = 0; u < U; ++u) f[u] = fetch(t_lane + u);

    griddep_wait();  // q, the step state and the workspace may belong to the kernel this one overlaps
    griddep_launch_dependents();
    const int qpos = (p.dyn != nullptr ? p.dyn[RFSN_STEP_POS] : p.q_pos0) + row;
    for (int g0 = 0; g0 < p.G; g0 += kHeadsPerPass * groups) {
        const int heads = p.G - g0 - kHeadsPerPass * group;  // of the warp's group (and more)
        if (g0 > 0) __syncthreads();
        for (int i = tid; i < groups * kHeadsPerPass * D / 2; i += kSelThreads) {
            // pairs of channels 8 (l8 + 8 v) + 2 j, + 1 of a head at [head][4 v + j][l8]: lanes side by side
            const int g = i / (D / 2), pr = i % (D / 2);
            const int d = 8 * ((pr & 7) + 8 * (pr >> 5)) + 2 * ((pr >> 3) & 3);
            float2 x = make_float2(0.f, 0.f);
            if (g0 + g < p.G)
                x = *reinterpret_cast<const float2*>(
                    p.q + (((size_t)b * p.q_heads + hk * p.G + g0 + g) * p.q_len + row) * D + d);
            qs[i] = make_double2((double)x.x, (double)x.y);
        }
        __syncthreads();
        for (int t0 = 0; t_begin + t0 < t_end; t0 += pass_tiles) {
            if (t0 > 0 || g0 > 0) {
#pragma unroll
                for (int u = 0; u < U; ++u) f[u] = fetch(t_lane + t0 + u);
            }
            double acc[U][kHeadsPerPass];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int g = 0; g < kHeadsPerPass; ++g) acc[u][g] = 0.0;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    int lo0[U], hi0[U], lo1[U], hi1[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        lo0[u] = __double2hiint((double)f[u].lo[v].get(2 * j));
                        hi0[u] = __double2hiint((double)f[u].hi[v].get(2 * j));
                        lo1[u] = __double2hiint((double)f[u].lo[v].get(2 * j + 1));
                        hi1[u] = __double2hiint((double)f[u].hi[v].get(2 * j + 1));
                    }
#pragma unroll
                    for (int g = 0; g < kHeadsPerPass; ++g) {
                        const double2 q2 = qs[(kHeadsPerPass * group + g) * (D / 2) + (4 * v + j) * 8 + l8];
                        const bool up0 = q2.x >= 0.0, up1 = q2.y >= 0.0;
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            acc[u][g] += q2.x * pick(up0, hi0[u], lo0[u]);
                            acc[u][g] += q2.y * pick(up1, hi1[u], lo1[u]);
                        }
                    }
                }
            // Sums over the 8 lanes, halving the heads a lane carries: lanes end with head 2 (l8 / 4) + (l8 / 2) % 2.
            static_assert(kHeadsPerPass == 4, "two halvings");
            const bool up4 = l8 & 4, up2 = l8 & 2;
            const int head = (up4 ? 2 : 0) + (up2 ? 1 : 0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int t = t_lane + t0 + u;
                const double s0 = __shfl_xor_sync(0xffffffffu, up4 ? acc[u][0] : acc[u][2], 4);
                const double s1 = __shfl_xor_sync(0xffffffffu, up4 ? acc[u][1] : acc[u][3], 4);
                const double a0 = (up4 ? acc[u][2] : acc[u][0]) + s0, a1 = (up4 ? acc[u][3] : acc[u][1]) + s1;
                double a = (up2 ? a1 : a0) + __shfl_xor_sync(0xffffffffu, up2 ? a0 : a1, 2);
                a += __shfl_xor_sync(0xffffffffu, a, 1);
                float best = head < heads ? (float)(a * (double)f[u].sk) : -CUDART_INF_F;
                const unsigned nan = __ballot_sync(0xffffffffu, best != best);
                best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 4));
                best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
                if ((nan >> (8 * sub)) & 0xffu) best = CUDART_NAN_F;
                if (f[u].e.z <= 0 || f[u].e.y > qpos) best = -CUDART_INF_F;
                if (groups > 1) {
                    if (l8 == 0) sh.part[group * pass_tiles + slot + u] = best;
                } else if (l8 == 0 && t < t_end) {
                    scores[t] = best;
                }
            }
            if (groups > 1) {  // the head groups of this pass, and those of earlier ones
                __syncthreads();
                const int t = t_begin + t0 + tid;
                if (tid < pass_tiles && t < t_end) {
                    auto larger = [](float a, float b) { return a != a || b != b ? CUDART_NAN_F : fmaxf(a, b); };
                    float best = sh.part[tid];
                    for (int g = 1; g < groups; ++g) best = larger(best, sh.part[g * pass_tiles + tid]);
                    scores[t] = g0 > 0 ? larger(scores[t], best) : best;
                }
                __syncthreads();
            }
        }
    }
    __syncthreads();
    if (gridDim.x > 1) {
        if (tid == 0) sh.flag = atom_add_acq_rel_gpu(&p.counters[list], 1) == (int)gridDim.x - 1;
        __syncthreads();
        if (!sh.flag) return;
    }
    if (p.n_tiles <= kSelRegKeys * kSelThreads)
        select_list<true>(p, scores, list, sh);
    else
        select_list<false>(p, scores, list, sh);
    if (gridDim.x > 1 && tid == 0) p.counters[list] = 0;
}

template <typename T, int D>
rfsn_status launch(const SelectParams& p, int lists, int chunks, cudaStream_t s) {
    RFSN_CUDA(launch_kernel(p.overlap, select_kernel<T, D>, dim3(chunks, lists), dim3(kSelThreads), 0, s, p));
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
