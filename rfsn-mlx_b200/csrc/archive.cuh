// Packed (8-bit) archive, tile lists and tile selection: what the kernels of
// archive_pack.cu, tile_select.cu and archive_attn.cu share with their C entry
// points (archive_api.cu).
#pragma once

#include <cuda_fp8.h>

#include "attn_common.cuh"
#include "params.cuh"

// One layer's 8-bit archive (opaque to C ABI users).
struct rfsn_packed_archive {
    uint8_t* k;       // [groups][rows][head_dim] e4m3 codes
    uint8_t* v;
    float4* scales;   // [groups][rows / 64] {K scale, V scale, 1 for a V tile of zeros, 0}
    int groups;
    int rows;
    int head_dim;
    int device;
    CUtensorMap maps[4];  // K and V: boxes of one 64-token tile, boxes of 16 rows
    rfsn::FreshWrites fresh;  // codes, scales and key bounds
};

namespace rfsn {
namespace archive {

constexpr float kPScale = 128.f;  // p <= 2^8 (kLazy), p * 2^7 <= 2^15 fits float16
constexpr float kTiny = 1.17549435e-38f;  // 2^-126, the smallest scale
constexpr float kLazy = 8.f;      // log2 units the running maximum may be exceeded by before it moves
constexpr int kStageBytes = 16384;              // one item: 64 packed keys, or 32 (head_dim 64: 64) 16-bit keys
constexpr int kMaxSplits128 = 240, kMaxSplits64 = 120;  // bounded by the merge weights kept in shared memory

struct Params {
    const float* q;
    float* out;
    float* lse;
    const int4* tiles;      // {row, pos, len, tile}
    int n_tiles;            // entries per list
    int per_query;          // 0: one list for every head and query; 1: a list per (batch * kv head, query row)
    int ring_row0, capacity, head, hlen, hstart;
    int rows;               // arena rows per head
    int packed_rows;
    const float4* scales;
    int q_heads, kv_heads, q_len, q_pos0, G;
    int slots;              // query slots of one list: q_len * G, or G per query row
    int items_per_split, splits;
    int hot_items;          // archive_rows.cu: items of 128 ring keys, at most
    float qscale;           // 1/sqrt(D) * log2(e)
    WsView ws;
    const int* dyn;         // device step state (RFSN_STEP_*) or nullptr
    bool overlap;           // launched with programmatic overlap (FreshWrites)
};

struct SelectParams {
    const void* bounds;     // [groups][slots][2][D]: smallest and largest key of each channel of a tile
    const float4* scales;   // e4m3 bounds: the archive's scales
    int tile_slots;         // tile slots per group (rows / 64)
    const float* q;
    int q_heads, kv_heads, q_len, q_pos0, G;
    const int4* tiles;
    int n_tiles, n_select, tiles_per_cta;
    int head_groups;        // of four q heads, scored side by side: 1, 2, 4 or 8
    int4* out;              // [groups * q_len][n_select] tiles, or
    int* numbers;           // their numbers only (out is nullptr)
    float* scores;          // workspace [groups * q_len][n_tiles]
    int* counters;
    int* error;
    const int* dyn;
    bool overlap;           // as in Params
};

// Paired float32 arithmetic (PTX .f32x2): two results per issue slot, each rounded as the scalar operation.
__device__ __forceinline__ uint64_t pair(float2 a) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t r) {
    float2 a;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(r));
    return a;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair(a)), "l"(pair(b)), "l"(pair(c)));
    return unpair(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair(a)), "l"(pair(b)));
    return unpair(r);
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b) {
    uint64_t r;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair(a)), "l"(pair(b)));
    return unpair(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair(a)), "l"(pair(b)));
    return unpair(r);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Split merge by the last CTA of a list (and block of SL query slots) to
// arrive; called by threads 0 .. nthreads - 1 of the CTA after they wrote its
// partials (named barrier 1 is theirs). The partials of all splits are
// contiguous runs (m, l, O) and come by asynchronous copies through `stage`:
// m and l with as many splits' O as fit in one round trip, the rest in further
// ones. Reading them one by one took 13 us for 240 splits of 4 slots. wts: room
// for SL * splits floats.
template <int D>
__device__ __forceinline__ void merge_splits(const Params& p, const OutMap& om, int bh, int slot0, int nslots, int SL,
                                             int counter, uint8_t* stage, int stage_bytes, float* wts, float* inv,
                                             int* flag, int nthreads) {
    constexpr int V4 = D / 4;   // float4 per row
    constexpr int kOwn = 2;     // float4 of the result per thread, at most
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    named_barrier_sync(1, nthreads);  // the CTA's partials before thread 0's release
    if (threadIdx.x == 0) *flag = atom_add_acq_rel_gpu(&p.ws.counters[counter], 1) == p.splits - 1;
    named_barrier_sync(1, nthreads);
    if (!*flag) return;
    const size_t part_base = (size_t)counter * p.splits * SL;
    const int parts = p.splits * SL;
    float4* st_ml = reinterpret_cast<float4*>(stage);
    float4* st_o = st_ml + parts / 2;
    const int round = min(p.splits, (stage_bytes - parts * 8) / (SL * D * 4));  // splits per round trip
    const float* gm = p.ws.m + part_base;
    const float* gl = p.ws.l + part_base;
    const float4* go = reinterpret_cast<const float4*>(p.ws.o + part_base * D);
    for (int i = threadIdx.x; i < parts / 2; i += nthreads)
        cp_async_16(st_ml + i, i < parts / 4 ? gm + 4 * i : gl + 4 * (i - parts / 4));
    cp_async_commit();
    float4 acc[kOwn];
#pragma unroll
    for (int k = 0; k < kOwn; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < p.splits; s0 += round) {
        const int n = min(round, p.splits - s0);
        if (s0 > 0) named_barrier_sync(1, nthreads);  // the stage has been read
        for (int i = threadIdx.x; i < n * SL * V4; i += nthreads) cp_async_16(st_o + i, go + (size_t)s0 * SL * V4 + i);
        cp_async_commit();
        if (s0 == 0) {  // the weights while O is on its way
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            named_barrier_sync(1, nthreads);
            const float* src_m = reinterpret_cast<const float*>(st_ml);
            const float* src_l = src_m + parts;
            for (int sl = warp; sl < nslots; sl += nthreads / 32) {
                float M = -INFINITY, L = 0.f;
                for (int s = lane; s < p.splits; s += 32) M = fmaxf(M, src_m[s * SL + sl]);
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
                for (int s = lane; s < p.splits; s += 32) {
                    const float wt = M == -INFINITY ? 1.f : ex2_approx(src_m[s * SL + sl] - M);
                    L += wt * src_l[s * SL + sl];
                    wts[sl * p.splits + s] = wt;
                }
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
                if (lane == 0) {
                    const bool any = L > 0.f || L != L;
                    inv[sl] = any ? 1.f / L : 0.f;
                    if (p.lse != nullptr)
                        p.lse[om.row(bh, slot0 + sl)] = any ? (M + log2f(L)) * 0.69314718055994531f : -INFINITY;
                }
            }
        }
        cp_async_wait_all();
        named_barrier_sync(1, nthreads);
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            const int i = threadIdx.x + k * nthreads, sl = i / V4;
            if (i >= nslots * V4) break;
            const float4* from = st_o + i;
            const float* w = wts + sl * p.splits + s0;
#pragma unroll 8
            for (int s = 0; s < n; ++s) {
                const float4 o = from[s * SL * V4];
                const float wt = w[s];
                acc[k].x += wt * o.x;
                acc[k].y += wt * o.y;
                acc[k].z += wt * o.z;
                acc[k].w += wt * o.w;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
        const int i = threadIdx.x + k * nthreads, sl = i / V4;
        if (i >= nslots * V4) break;
        const float r = inv[sl];
        *reinterpret_cast<float4*>(p.out + om.row(bh, slot0 + sl) * D + 4 * (i % V4)) =
            make_float4(acc[k].x * r, acc[k].y * r, acc[k].z * r, acc[k].w * r);
    }
    if (threadIdx.x == 0) p.ws.counters[counter] = 0;
}

}  // namespace archive

// archive_pack.cu
rfsn_status pack_rows_launch(const rfsn_packed_archive* a, int dst_row0, const rfsn_kv_rows* src, int count,
                             void* bounds, cudaStream_t stream);
rfsn_status unpack_rows_launch(const rfsn_packed_archive* a, int row0, int count, void* k_out, void* v_out, int dtype,
                               long long group_stride, cudaStream_t stream);
rfsn_status tile_bounds_launch(const rfsn_arena* arena, int row0, int count, void* bounds, cudaStream_t stream);
void preload_pack_kernels();
// tile_select.cu
void preload_select_kernels();
rfsn_status select_tiles_launch(int bounds_dtype, int head_dim, const archive::SelectParams& p, int lists, int chunks,
                                cudaStream_t stream);
// archive_attn.cu: nb = column blocks of 4 query slots per CTA (1 or 2); CTAs per SM of that variant
int archive_attn_ctas(int nb);
rfsn_status archive_attn_launch(const rfsn_arena* arena, const rfsn_packed_archive* packed, const archive::Params& p,
                                int lists, int nb, int zblocks, cudaStream_t stream);
// archive_rows.cu: 5 to 16 query slots per CTA (slots 8 or 16) over a packed archive, head_dim 128
rfsn_status archive_rows_launch(const rfsn_arena* arena, const rfsn_packed_archive* packed, const archive::Params& p,
                                int lists, int slots, int zblocks, cudaStream_t stream);
void preload_rows_kernels();

// archive_chunk.cu: chunks of queries over a packed archive. Workspace: partials and a copy of the ring.
bool archive_chunk_fits(int G);
size_t archive_chunk_ws(int groups, int hot_capacity, int head_dim);
rfsn_status archive_chunk_launch(const rfsn_arena* arena, const rfsn_packed_archive* packed, const archive::Params& a,
                                 int batch, void* workspace, size_t workspace_bytes, int max_splits,
                                 cudaStream_t stream);
void preload_chunk_kernels();

}  // namespace rfsn
