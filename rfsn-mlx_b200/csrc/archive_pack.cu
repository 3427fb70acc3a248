// Packing of archived K/V rows into 8 bits and back, and the per-tile key
// bounds that tile selection scores.
//
// A tile is 64 consecutive tokens of a block. For each (tile, KV head), K and
// V apart, with a = the largest finite |x| of the tile:
//   s = 2^e, the smallest power of two with a / s <= 448 (1 when a = 0)
//   code = round-to-nearest-even e4m3(x / s)
// A power of two makes x / s exact, so packing rounds once (at most half an
// e4m3 step, 2^-4 of the value, or 2^-10 * s below e4m3's normal range), a
// packed value is exact in bfloat16, and packing an unpacked tile again gives
// the same values. It costs no precision against a / 448: the codes are
// floating-point numbers, only the point where they turn subnormal moves.
// NaN stays NaN, infinities become NaN (e4m3 has none, and saturating them
// would hide them).
#include <algorithm>
#include <cstring>

#include <math_constants.h>

#include "archive.cuh"

namespace rfsn {
namespace archive {

constexpr int kPackThreads = 256;
constexpr int kPackCtas = 8;  // per SM: 65,501 tokens of 8 heads 67.8 us (3: 74.5, 4: 72.1, 6: 77.6, not in order)

struct RowSource {
    const void* p;
    long long sb, sh, st;  // strides in elements: batch, head, token
    int kv_heads, offset, wrap;
    int vec;               // rows may be read as 16-byte vectors
};

// 8 elements as they are in memory, and their values
template <typename T> struct Vec8 {
    uint4 w[8 * sizeof(T) / 16];
    __device__ __forceinline__ void load(const T* p, int vec) {
        if (vec) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(w) / 16; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
        } else {
            T* e = reinterpret_cast<T*>(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = p[i];
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(w) / 16; ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ float get(int i) const { return to_f32<T>(reinterpret_cast<const T*>(w)[i]); }
    __device__ __forceinline__ void drop_infinities() {  // to NaN
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (fabsf(get(i)) == CUDART_INF_F) reinterpret_cast<T*>(w)[i] = from_f32<T>(CUDART_NAN_F);
    }
    // Largest |x| so far as bit patterns (they order like the magnitudes, infinities and NaN above all numbers): one
    // per word, two per word for 16-bit types.
    __device__ __forceinline__ uint32_t abs_max(uint32_t acc) const {
#pragma unroll
        for (int i = 0; i < (int)sizeof(w) / 4; ++i) {
            const uint32_t x = (&w[i / 4].x)[i % 4];
            acc = sizeof(T) == 4 ? max(acc, x & 0x7fffffffu) : __vmaxu2(acc, x & 0x7fff7fffu);
        }
        return acc;
    }
};
// The pattern of abs_max as a number, infinite for infinities and NaN alike.
template <typename T> __device__ __forceinline__ float pattern_value(uint32_t m) {
    if (sizeof(T) == 4) return m >= 0x7f800000u ? CUDART_INF_F : __uint_as_float(m);
    const uint16_t h = (uint16_t)m;
    T x;
    memcpy(&x, &h, 2);
    const float f = to_f32<T>(x);
    return f != f ? CUDART_INF_F : f;
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ __half2 half2_of_e4m3x2(uint32_t x) {
    return __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)x, __NV_E4M3));
}

// The scale of a tile whose largest finite magnitude is a: from the exponent
// and mantissa of a = m * 2^e, m in [1, 2): 448 = 1.75 * 2^8.
__device__ __forceinline__ float tile_scale(float a) {
    if (!(a > 0.f)) return 1.f;
    const uint32_t b = __float_as_uint(a);
    int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    if (e < -126) e = -126;  // also subnormal a
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// A CTA's work item is a (tile, KV head, K or V); the tile stays in registers
// between the maximum and the conversion, so it is read once, and the next
// item's tile is requested before this one is converted. Items are numbered K
// and V fastest, then the heads, so that the CTAs that run together read
// neighbouring rows of token-major sources. Bound by memory (65,501 tokens of 8
// heads 67 us, 93 % of the copy rate); with key bounds by their reduction through
// shared memory (99 us; 256 tokens 2.5 against 2.1). Rows of the tile
// behind `count` become zero codes (the attention kernels read whole tiles and
// multiply them by zero weights).
template <typename T, int D, bool BOUNDS>
__global__ void __launch_bounds__(kPackThreads) pack_kernel(RowSource ks, RowSource vs, uint8_t* __restrict__ kd,
                                                            uint8_t* __restrict__ vd, float* __restrict__ scales,
                                                            uint8_t* __restrict__ bounds, int rows, int dst_row0,
                                                            int count, uint32_t groups, uint32_t items) {
    constexpr int VPR = D / 8;                    // 8-element vectors per row
    constexpr int RPP = kPackThreads / VPR;       // rows per pass
    constexpr int PASSES = kTile / RPP;
    const int c8 = threadIdx.x % VPR, r0 = threadIdx.x / VPR;
    __shared__ uint32_t part[2][kPackThreads / 32];
    __shared__ __half2 red[BOUNDS ? 2 : 1][BOUNDS ? RPP : 1][D / 2];
    struct Place {
        int is_v, bh, tile;
    };
    auto fetch = [&](uint32_t item, Vec8<T> (&x)[PASSES]) {
        const uint32_t pair = item >> 1, tile_ = pair / groups;
        const Place at{(int)(item & 1), (int)(pair - tile_ * groups), (int)tile_};
        const RowSource& src = at.is_v ? vs : ks;
        const uint32_t b = (uint32_t)at.bh / (uint32_t)src.kv_heads, h = (uint32_t)at.bh - b * src.kv_heads;
        const T* base = static_cast<const T*>(src.p) + b * src.sb + h * src.sh + 8 * c8;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r = at.tile * kTile + r0 + i * RPP;
            x[i].clear();
            if (r < count) {
                long long t = (long long)src.offset + r;
                if (src.wrap > 0 && t >= src.wrap) t -= src.wrap;
                x[i].load(base + t * src.st, src.vec);
            }
        }
        return at;
    };
    Vec8<T> next[PASSES];
    uint32_t item = blockIdx.x;
    Place next_at = fetch(item, next);  // the grid has at most `items` CTAs
    for (int turn = 0; item < items; item += gridDim.x, turn ^= 1) {
        Vec8<T> x[PASSES];
#pragma unroll
        for (int i = 0; i < PASSES; ++i) x[i] = next[i];
        const int is_v = next_at.is_v, bh = next_at.bh, tile = next_at.tile;
        if (item + gridDim.x < items) next_at = fetch(item + gridDim.x, next);
        const int len = min(kTile, count - tile * kTile);
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) m = x[i].abs_max(m);
        if (sizeof(T) == 2) m = max(m & 0xffffu, m >> 16);
        m = __reduce_max_sync(0xffffffffu, m);
        if ((threadIdx.x & 31) == 0) part[turn][threadIdx.x >> 5] = m;
        __syncthreads();  // also: the previous item's bounds have been reduced
        m = part[turn][0];
#pragma unroll
        for (int i = 1; i < kPackThreads / 32; ++i) m = max(m, part[turn][i]);
        float a = pattern_value<T>(m);
        if (a == CUDART_INF_F) {  // infinities or NaN in the tile (all threads agree): the maximum of the rest
            a = 0.f;
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                x[i].drop_infinities();
#pragma unroll
                for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(x[i].get(e)));  // NaN loses
            }
            const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(a));
            __syncthreads();
            if ((threadIdx.x & 31) == 0) part[turn][threadIdx.x >> 5] = bits;
            __syncthreads();
            m = part[turn][0];
#pragma unroll
            for (int i = 1; i < kPackThreads / 32; ++i) m = max(m, part[turn][i]);
            a = __uint_as_float(m);
        }
        const float s = tile_scale(a), inv = 1.f / s;  // both powers of two
        const int row0 = dst_row0 + tile * kTile;
        uint8_t* dst = (is_v ? vd : kd) + ((size_t)bh * rows + row0) * D + 8 * c8;
        const bool bound = BOUNDS && !is_v;
        __half2 lo[4], hi[4];
        const __half2 top = __half2half2(__ushort_as_half(0x7c00)), bottom = __half2half2(__ushort_as_half(0xfc00));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            lo[j] = top;
            hi[j] = bottom;
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r = r0 + i * RPP;
            uint32_t c[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                c[j] = e4m3x2(x[i].get(2 * j) * inv, x[i].get(2 * j + 1) * inv);
                if (BOUNDS && bound && r < len) {
                    const __half2 h = half2_of_e4m3x2(c[j]);
                    lo[j] = __hmin2_nan(lo[j], h);
                    hi[j] = __hmax2_nan(hi[j], h);
                }
            }
            *reinterpret_cast<uint2*>(dst + (size_t)r * D) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
        }
        const size_t slot = (size_t)bh * (rows / kTile) + row0 / kTile;
        if (threadIdx.x == 0) {
            scales[4 * slot + is_v] = s;
            // its scale of 1 says nothing about the size of V: the attention kernels leave it out of their units
            if (is_v) scales[4 * slot + 2] = a > 0.f ? 0.f : 1.f;
        }
        if constexpr (BOUNDS) {
            if (!bound) continue;
            // channel-wise smallest and largest code of the tile's keys
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                red[0][r0][4 * c8 + j] = lo[j];
                red[1][r0][4 * c8 + j] = hi[j];
            }
            __syncthreads();
            if (threadIdx.x < D) {  // 2 bounds x D / 2 channel pairs
                const int w = threadIdx.x / (D / 2), j = threadIdx.x % (D / 2);
                __half2 m = red[w][0][j];
#pragma unroll 4
                for (int r = 1; r < RPP; ++r)
                    m = w ? __hmax2_nan(m, red[w][r][j]) : __hmin2_nan(m, red[w][r][j]);
                const float2 f = __half22float2(m);
                reinterpret_cast<uint16_t*>(bounds)[(slot * 2 + w) * (D / 2) + j] = (uint16_t)e4m3x2(f.x, f.y);
            }
        }
    }
}

// value = code * scale, rounded once to T (exact for float32 and bfloat16;
// finite values saturate at float16's largest number).
template <typename T> __device__ __forceinline__ T unpacked(float x) { return from_f32<T>(x); }
template <> __device__ __forceinline__ __half unpacked<__half>(float x) {
    if (fabsf(x) > 65504.f) x = copysignf(65504.f, x);
    return __float2half_rn(x);
}

// 16 codes per thread: one 16-byte load, 32 (64) bytes stored. Bound by memory:
// 65,501 tokens of 8 heads to bf16 69.7 us, 89 % of the copy rate.
template <typename T, int D>
__global__ void __launch_bounds__(256) unpack_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                     const float4* __restrict__ scales, T* __restrict__ ko,
                                                     T* __restrict__ vo, int rows, int row0, int count,
                                                     long long group_stride) {
    constexpr int VPR = D / 16;
    const int bh = blockIdx.y, is_v = blockIdx.z;
    const long long total = (long long)count * VPR;
    const uint8_t* src = (is_v ? vc : kc) + ((size_t)bh * rows + row0) * D;
    T* dst = (is_v ? vo : ko) + (size_t)bh * group_stride;
    const float4* sc = scales + (size_t)bh * (rows / kTile);
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
        const int r = (int)(i / VPR);
        const float4 s4 = __ldg(sc + (row0 + r) / kTile);
        const float s = is_v ? s4.y : s4.x;
        const uint4 c = __ldg(reinterpret_cast<const uint4*>(src) + i);
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
        alignas(16) T o[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 f = __half22float2(half2_of_e4m3x2((w[j >> 1] >> (16 * (j & 1))) & 0xffffu));
            o[2 * j] = unpacked<T>(f.x * s);
            o[2 * j + 1] = unpacked<T>(f.y * s);
        }
#pragma unroll
        for (int j = 0; j < (int)sizeof(T); ++j) reinterpret_cast<uint4*>(dst + 16 * i)[j] = reinterpret_cast<uint4*>(o)[j];
    }
}

// Channel-wise smallest and largest key of each tile of an exact (16-bit)
// block: one CTA per (tile, KV head); NaN keys give NaN bounds. Bound by the
// chain load, reduction, barrier of each CTA: 65,536 tokens of 8 heads 56 us (21 at
// the copy rate), 256 tokens 3.3.
template <typename T, int D>
__global__ void __launch_bounds__(256) bounds_kernel(const T* __restrict__ k, T* __restrict__ bounds, int rows,
                                                     int row0, int count) {
    constexpr int VPR = D / 8, RPP = 256 / VPR;
    const int tile = blockIdx.x, bh = blockIdx.y;
    const int len = min(kTile, count - tile * kTile);
    const int c8 = threadIdx.x % VPR, r0 = threadIdx.x / VPR;
    const T* src = k + ((size_t)bh * rows + row0 + tile * kTile) * D + 8 * c8;
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        lo[e] = CUDART_INF_F;
        hi[e] = -CUDART_INF_F;
    }
#pragma unroll
    for (int i = 0; i < kTile / RPP; ++i) {
        const int r = r0 + i * RPP;
        if (r < len) {
            Vec8<T> x;
            x.load(src + (size_t)r * D, 1);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = x.get(e);
                lo[e] = (y < lo[e] || y != y) ? y : lo[e];
                hi[e] = (y > hi[e] || y != y) ? y : hi[e];
            }
        }
    }
    __shared__ float red[2][RPP][D];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        red[0][r0][8 * c8 + e] = lo[e];
        red[1][r0][8 * c8 + e] = hi[e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += 256) {
        const int w = i / D, d = i % D;
        float m = red[w][0][d];
        for (int r = 1; r < RPP; ++r) {
            const float x = red[w][r][d];
            // a NaN met first stays (comparisons with it are false), one met later replaces m
            m = ((w ? x > m : x < m) || x != x) ? x : m;
        }
        bounds[(((size_t)bh * (rows / kTile) + (row0 + tile * kTile) / kTile) * 2 + w) * D + d] = from_f32<T>(m);
    }
}

template <typename T, int D>
rfsn_status pack_launch(const rfsn_packed_archive* a, int dst_row0, const RowSource& ks, const RowSource& vs,
                        int count, void* bounds, cudaStream_t s) {
    // groups * rows < 2^31, so the count fits 32 bits
    const uint32_t items = 2u * (uint32_t)a->groups * (uint32_t)((count + kTile - 1) / kTile);
    const uint32_t ctas = std::min(items, (uint32_t)(kPackCtas * device_sms()));
    if (bounds != nullptr)
        pack_kernel<T, D, true><<<ctas, kPackThreads, 0, s>>>(ks, vs, a->k, a->v, reinterpret_cast<float*>(a->scales),
                                                              static_cast<uint8_t*>(bounds), a->rows, dst_row0, count,
                                                              a->groups, items);
    else
        pack_kernel<T, D, false><<<ctas, kPackThreads, 0, s>>>(ks, vs, a->k, a->v, reinterpret_cast<float*>(a->scales),
                                                               nullptr, a->rows, dst_row0, count, a->groups, items);
    RFSN_CUDA(cudaGetLastError());
    note_launch();
    return RFSN_OK;
}

template <typename T, int D>
rfsn_status unpack_launch(const rfsn_packed_archive* a, int row0, int count, void* k, void* v, long long gs,
                          cudaStream_t s) {
    const long long per = ((long long)count * (D / 16) + 255) / 256;
    const dim3 grid((unsigned)(per < 2048 ? per : 2048), a->groups, 2);
    unpack_kernel<T, D><<<grid, 256, 0, s>>>(a->k, a->v, a->scales, static_cast<T*>(k), static_cast<T*>(v), a->rows,
                                             row0, count, gs);
    RFSN_CUDA(cudaGetLastError());
    note_launch();
    return RFSN_OK;
}

template <typename T, int D>
rfsn_status bounds_launch(const rfsn_arena* a, int row0, int count, void* bounds, cudaStream_t s) {
    const dim3 grid((count + kTile - 1) / kTile, a->groups);
    bounds_kernel<T, D><<<grid, 256, 0, s>>>(static_cast<const T*>(a->k), static_cast<T*>(bounds), a->rows, row0,
                                             count);
    RFSN_CUDA(cudaGetLastError());
    note_launch();
    return RFSN_OK;
}

template <typename T, int D>
void preload() {
    cudaFuncAttributes a;
    cudaFuncGetAttributes(&a, pack_kernel<T, D, false>);
    cudaFuncGetAttributes(&a, pack_kernel<T, D, true>);
    cudaFuncGetAttributes(&a, unpack_kernel<T, D>);
    if constexpr (sizeof(T) == 2) cudaFuncGetAttributes(&a, bounds_kernel<T, D>);
}

}  // namespace archive

void preload_pack_kernels() {
    using namespace archive;
    preload<float, 64>();
    preload<float, 128>();
    preload<__half, 64>();
    preload<__half, 128>();
    preload<__nv_bfloat16, 64>();
    preload<__nv_bfloat16, 128>();
}

rfsn_status pack_rows_launch(const rfsn_packed_archive* a, int dst_row0, const rfsn_kv_rows* src, int count,
                             void* bounds, cudaStream_t s) {
    using namespace archive;
    const int es = dtype_size(src->dtype);
    auto make = [&](const void* p, int64_t sb, int64_t sh, int64_t st) {
        const bool vec = ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(sb * es) | (uintptr_t)(sh * es) |
                           (uintptr_t)(st * es)) & 15) == 0;
        return RowSource{p, sb, sh, st, src->kv_heads, src->offset, src->wrap, vec ? 1 : 0};
    };
    const RowSource ks = make(src->k, src->k_stride_b, src->k_stride_h, src->k_stride_t);
    const RowSource vs = make(src->v, src->v_stride_b, src->v_stride_h, src->v_stride_t);
    const bool d128 = a->head_dim == 128;
    if (src->dtype == RFSN_F32)
        return d128 ? pack_launch<float, 128>(a, dst_row0, ks, vs, count, bounds, s)
                    : pack_launch<float, 64>(a, dst_row0, ks, vs, count, bounds, s);
    if (src->dtype == RFSN_F16)
        return d128 ? pack_launch<__half, 128>(a, dst_row0, ks, vs, count, bounds, s)
                    : pack_launch<__half, 64>(a, dst_row0, ks, vs, count, bounds, s);
    return d128 ? pack_launch<__nv_bfloat16, 128>(a, dst_row0, ks, vs, count, bounds, s)
                : pack_launch<__nv_bfloat16, 64>(a, dst_row0, ks, vs, count, bounds, s);
}

rfsn_status unpack_rows_launch(const rfsn_packed_archive* a, int row0, int count, void* k, void* v, int dtype,
                               long long gs, cudaStream_t s) {
    using namespace archive;
    const bool d128 = a->head_dim == 128;
    if (dtype == RFSN_F32)
        return d128 ? unpack_launch<float, 128>(a, row0, count, k, v, gs, s)
                    : unpack_launch<float, 64>(a, row0, count, k, v, gs, s);
    if (dtype == RFSN_F16)
        return d128 ? unpack_launch<__half, 128>(a, row0, count, k, v, gs, s)
                    : unpack_launch<__half, 64>(a, row0, count, k, v, gs, s);
    return d128 ? unpack_launch<__nv_bfloat16, 128>(a, row0, count, k, v, gs, s)
                : unpack_launch<__nv_bfloat16, 64>(a, row0, count, k, v, gs, s);
}

rfsn_status tile_bounds_launch(const rfsn_arena* a, int row0, int count, void* bounds, cudaStream_t s) {
    using namespace archive;
    const bool d128 = a->head_dim == 128;
    if (a->dtype == RFSN_F16)
        return d128 ? bounds_launch<__half, 128>(a, row0, count, bounds, s)
                    : bounds_launch<__half, 64>(a, row0, count, bounds, s);
    return d128 ? bounds_launch<__nv_bfloat16, 128>(a, row0, count, bounds, s)
                : bounds_launch<__nv_bfloat16, 64>(a, row0, count, bounds, s);
}

}  // namespace rfsn
