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
    float4* scales;   // [groups][rows / 64] {K scale, V scale, 0, 0}
    int groups;
    int rows;
    int head_dim;
    int device;
    CUtensorMap maps[2];  // K and V, boxes of one 64-token tile
};

namespace rfsn {
namespace archive {

constexpr float kPScale = 128.f;  // p <= 2^8 (kLazy), p * 2^7 <= 2^15 fits float16
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
    float qscale;           // 1/sqrt(D) * log2(e)
    WsView ws;
    const int* dyn;         // device step state (RFSN_STEP_*) or nullptr
};

struct SelectParams {
    const void* bounds;     // [groups][slots][2][D]: smallest and largest key of each channel of a tile
    const float4* scales;   // e4m3 bounds: the archive's scales
    int tile_slots;         // tile slots per group (rows / 64)
    const float* q;
    int q_heads, kv_heads, q_len, q_pos0, G;
    const int4* tiles;
    int n_tiles, n_select, tiles_per_cta;
    int4* out;              // [groups * q_len][n_select] tiles, or
    int* numbers;           // their numbers only (out is nullptr)
    float* scores;          // workspace [groups * q_len][n_tiles]
    int* counters;
    int* error;
    const int* dyn;
};

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

// archive_chunk.cu: chunks of queries over a packed archive, head_dim 128. Workspace: partials and a copy of the ring.
bool archive_chunk_fits(int G);
size_t archive_chunk_ws(int groups, int hot_capacity);
rfsn_status archive_chunk_launch(const rfsn_arena* arena, const rfsn_packed_archive* packed, const archive::Params& a,
                                 int batch, void* workspace, size_t workspace_bytes, int max_splits,
                                 cudaStream_t stream);
void preload_chunk_kernels();

}  // namespace rfsn
