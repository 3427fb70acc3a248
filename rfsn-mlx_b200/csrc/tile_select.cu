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
#include <algorithm>

#include <math_constants.h>

#include "archive.cuh"

namespace rfsn {
namespace archive {

constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelSmemKeys = 12288;  // lists up to this many tiles keep their keys in shared memory
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

template <typename T, int D>
__global__ void __launch_bounds__(kSelThreads) select_kernel(const SelectParams p) {
    constexpr int DL = D / 8;  // channels per lane (8 lanes per tile)
    extern __shared__ uint8_t smem_sel[];
    double* qs = reinterpret_cast<double*>(smem_sel);  // [kHeadsPerPass][D]; later the selection's keys
    __shared__ int s_flag, s_count[kSelWarps], s_gt[kSelWarps], s_eq[kSelWarps];
    __shared__ uint32_t s_or[kSelWarps], s_and[kSelWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int list = blockIdx.y;
    const int row = list % p.q_len, bh = list / p.q_len;
    const int b = bh / p.kv_heads, hk = bh % p.kv_heads;
    griddep_wait();  // q, the step state and the workspace may belong to the kernel this one overlaps
    const int qpos = (p.dyn != nullptr ? p.dyn[RFSN_STEP_POS] : p.q_pos0) + row;
    const int t_begin = blockIdx.x * p.tiles_per_cta;
    const int t_end = min(t_begin + p.tiles_per_cta, p.n_tiles);
    float* scores = p.scores + (size_t)list * p.n_tiles;
    const int sub = lane >> 3, l8 = lane & 7;
    for (int g0 = 0; g0 < p.G; g0 += kHeadsPerPass) {
        const int heads = min(kHeadsPerPass, p.G - g0);
        __syncthreads();
        for (int i = tid; i < kHeadsPerPass * D; i += kSelThreads) {
            // lanes' channel pairs side by side: [head][4 v + i / 2][l8] pairs of channels 8 (l8 + 8 v) + i, + 1
            const int g = i / D, w = i % D, pr = w >> 1;
            const int d = 8 * ((pr & 7) + 8 * (pr >> 5)) + 2 * ((pr >> 3) & 3) + (w & 1);
            qs[i] = g < heads ? (double)p.q[(((size_t)b * p.q_heads + hk * p.G + g0 + g) * p.q_len + row) * D + d] : 0.0;
        }
        __syncthreads();
        for (int t0 = t_begin + warp * 4; t0 < t_end; t0 += kSelWarps * 4) {
            const int t = t0 + sub;
            const bool in = t < t_end;
            int4 e = make_int4(0, 0, 0, -1);
            if (in) e = __ldg(p.tiles + t);
            const bool bad = in && ((e.x & (kTile - 1)) != 0 || e.x < 0 || e.x / kTile >= p.tile_slots);
            if (bad) atomicExch(p.error, kDevErrBadTable);
            const bool live = in && !bad && e.z > 0 && e.y <= qpos;
            double acc[kHeadsPerPass];
#pragma unroll
            for (int g = 0; g < kHeadsPerPass; ++g) acc[g] = 0.0;
            float sk = 1.f;
            if (live) {
                const size_t slot = (size_t)bh * p.tile_slots + e.x / kTile;
                if (sizeof(T) == 1) sk = __ldg(p.scales + slot).x;
                const char* base = static_cast<const char*>(p.bounds) + slot * 2 * D * sizeof(T);
#pragma unroll
                for (int v = 0; v < DL / 8; ++v) {
                    // channel blocks interleaved over the lanes: 8 lanes read consecutive vectors
                    const int d0 = 8 * (l8 + 8 * v);
                    BoundVec<T> lo, hi;
                    lo.load(base + d0 * sizeof(T));
                    hi.load(base + (D + d0) * sizeof(T));
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const double l0 = (double)lo.get(i), h0 = (double)hi.get(i);
                        const double l1 = (double)lo.get(i + 1), h1 = (double)hi.get(i + 1);
#pragma unroll
                        for (int g = 0; g < kHeadsPerPass; ++g) {
                            const double2 q2 = reinterpret_cast<const double2*>(qs)[g * (D / 2) + (4 * v + i / 2) * 8 + l8];
                            acc[g] += q2.x * (q2.x >= 0.0 ? h0 : l0);
                            acc[g] += q2.y * (q2.y >= 0.0 ? h1 : l1);
                        }
                    }
                }
            }
            float best = -CUDART_INF_F;
            bool nan = false;
#pragma unroll
            for (int g = 0; g < kHeadsPerPass; ++g) {
#pragma unroll
                for (int off = 4; off > 0; off >>= 1) acc[g] += __shfl_xor_sync(0xffffffffu, acc[g], off);
                if (g < heads) {
                    const float s = (float)(acc[g] * (double)sk);
                    best = fmaxf(best, s);
                    nan |= s != s;
                }
            }
            if (l8 == 0 && in) {
                if (!live) best = -CUDART_INF_F;
                if (nan && live) best = CUDART_NAN_F;
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
        if (tid == 0) s_flag = atom_add_acq_rel_gpu(&p.counters[list], 1) == (int)gridDim.x - 1;
        __syncthreads();
        if (!s_flag) return;
    }
    griddep_launch_dependents();

    // ---------------- selection: the last CTA of the list ----------------
    // The n-th largest key by bisection over its bits: a count per candidate
    // threshold, skipping the leading bits that all keys share and stopping
    // as soon as a threshold holds exactly n keys.
    const int T_ = p.n_tiles;
    const bool in_smem = T_ <= kSelSmemKeys;
    uint32_t* keys = reinterpret_cast<uint32_t*>(smem_sel);
    uint32_t k_or = 0u, k_and = 0xffffffffu;
    int visible = 0;
    for (int t = tid; t < T_; t += kSelThreads) {
        const uint32_t k = score_key(__ldcg(scores + t));
        if (in_smem) keys[t] = k;
        if (k != 0u) {
            ++visible;
            k_or |= k;
            k_and &= k;
        }
    }
    auto key_at = [&](int t) { return in_smem ? keys[t] : score_key(__ldcg(scores + t)); };
    k_or = __reduce_or_sync(0xffffffffu, k_or);
    k_and = __reduce_and_sync(0xffffffffu, k_and);
    visible = __reduce_add_sync(0xffffffffu, visible);
    if (lane == 0) {
        s_or[warp] = k_or;
        s_and[warp] = k_and;
        s_count[warp] = visible;
    }
    __syncthreads();
    k_or = 0u;
    k_and = 0xffffffffu;
    visible = 0;
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) {
        k_or |= s_or[w];
        k_and &= s_and[w];
        visible += s_count[w];
    }
    const int n = min(p.n_select, visible);
    uint32_t thr = 1u;  // every visible tile
    if (n < visible) {
        const uint32_t differ = k_or ^ k_and;
        const int top = differ ? 31 - __clz(differ) : -1;
        thr = top < 31 ? (k_or >> (top + 1)) << (top + 1) : 0u;  // the bits all keys share
        for (int bit = top; bit >= 0; --bit) {
            const uint32_t cand = thr | (1u << bit);
            int c = 0;
            for (int t = tid; t < T_; t += kSelThreads) c += key_at(t) >= cand;
            c = __reduce_add_sync(0xffffffffu, c);
            __syncthreads();  // the previous round's counts have been read
            if (lane == 0) s_count[warp] = c;
            __syncthreads();
            c = 0;
#pragma unroll
            for (int w = 0; w < kSelWarps; ++w) c += s_count[w];
            if (c >= n) thr = cand;
            if (c == n) break;
        }
    }
    // Each warp owns a run of tiles: count, then write in tile order. Keys
    // above the threshold are all taken, keys equal to it from the lowest tile on.
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
        s_gt[warp] = gt;
        s_eq[warp] = eq;
    }
    __syncthreads();
    int gt_before = 0, eq_before = 0, gt_all = 0;
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) {
        if (w < warp) {
            gt_before += s_gt[w];
            eq_before += s_eq[w];
        }
        gt_all += s_gt[w];
    }
    const int need = n - gt_all;  // tiles taken among those equal to the threshold
    int4* out = p.out + (size_t)list * p.n_select;
    const unsigned below = (1u << lane) - 1u;
    for (int t0 = r0; t0 < r1; t0 += 32) {
        const int t = t0 + lane;
        const uint32_t k = t < r1 ? key_at(t) : 0u;
        const bool is_gt = t < r1 && k > thr, is_eq = t < r1 && k == thr;
        const unsigned mg = __ballot_sync(0xffffffffu, is_gt), me = __ballot_sync(0xffffffffu, is_eq);
        const int g = gt_before + __popc(mg & below), q = eq_before + __popc(me & below);
        if (is_gt || (is_eq && q < need)) {
            int4 e = __ldg(p.tiles + t);
            e.w = t;
            out[g + min(q, need)] = e;
        }
        gt_before += __popc(mg);
        eq_before += __popc(me);
    }
    for (int i = n + tid; i < p.n_select; i += kSelThreads) out[i] = make_int4(0, 0, 0, -1);
    if (gridDim.x > 1 && tid == 0) p.counters[list] = 0;
}

template <typename T, int D>
rfsn_status launch(const SelectParams& p, int lists, int chunks, cudaStream_t s) {
    const size_t smem = std::max((size_t)kHeadsPerPass * D * sizeof(double),
                                 p.n_tiles <= kSelSmemKeys ? sizeof(uint32_t) * (size_t)p.n_tiles : (size_t)0);
    RFSN_CUDA(launch_pdl(select_kernel<T, D>, dim3(chunks, lists), dim3(kSelThreads), smem, s, p));
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
