// Split-KV attention over a list of archived tiles and the hot window, the
// tiles in 8 bits (packed archive) or in the cache's 16-bit type.
//
//   out = softmax(q K^T / sqrt(D) + causal) V,   K = code * s_k(tile), V = code * s_v(tile)
//
// The keys of one (batch, kv head) are given as a list of 64-token tiles
// {row, pos, len}: the archived blocks of the page table (one list for all
// heads and queries), or the tiles selected for each query and KV head. A
// producer warp streams them (and then the hot window) with TMA as 16 KB
// items: 64 packed keys, or 32 16-bit keys (64 with head_dim 64). Consumer
// warps in groups of four take items in turn, a 16-key strip each:
//   S^T[16 keys x 8] = K[16 x D] . Q^T[D x 8]       (mma.sync m16n8k16)
//   O^T[D x 8]      += V^T[D x 16] . P^T[16 x 8]
// A column pair (2s, 2s + 1) is query slot s twice: the 16-bit head and the
// 16-bit remainder of the float32 operand. Tensor instructions are not the
// bound here (HBM is), and this transposed form wastes none of their columns
// for GQA groups of 4.
//
// Packed tiles. An e4m3 code is exact in float16, so codes are widened two at
// a time (cvt.rn.f16x2.e4m3x2) on their way from shared memory to the operand
// registers and the scales stay outside the products: s_k multiplies the
// logit, s_v the probability. q and p are split into two float16 (22
// significant bits); q is first scaled by a power of two per query slot, and
// p by 2^7 s_v / u with u the largest s_v met so far, so neither leaves
// float16's range. No ldmatrix: the order of keys and channels inside a
// product is free as long as both operands agree, so a lane reads 16
// consecutive codes of a key and takes them as channels of four k-steps.
//
// 16-bit tiles come through ldmatrix. float16 ones use the same two-way split;
// bfloat16 ones a three-way split (24 bits) in a second column block, since
// two bfloat16 hold 16 bits only.
//
// The softmax keeps a reference maximum per query slot that moves only when a
// logit exceeds it by more than 2^8 (in powers of two), so most strips need
// one vote instead of a reduction over the lanes and a rescale.
//
// Measured, 32 q / 8 KV heads, head_dim 128: 128K packed tokens and 4K ring
// 48.7 us (5.7 TB/s; 43.2 at the copy rate), 6K and 2K fp16 9.2 us, where the
// wait for the SMs, q, one round of tiles and the merge are 1 to 2 us each. 8
// and 16 consumer warps per SM take the same time as 8 (two CTAs of four).
#include <atomic>

#include <math_constants.h>

#include "archive.cuh"

namespace rfsn {
namespace archive {

template <int D> struct Geometry {
    static constexpr int kHotKeys = D == 128 ? 32 : 64;   // 16-bit keys per item
    static constexpr int kItemsPerTile16 = kTile / kHotKeys;
    static constexpr int kHalves = D / 64;                // 64-element column boxes of a 16-bit row
    static constexpr int kV16 = kStageBytes / 2;          // V offset inside a 16-bit item
    static constexpr int kVPacked = kTile * D;            // V offset inside a packed item
};

template <int D, int NB, int GROUPS, int STAGES, bool PACKED, bool BF16>
struct Smem {
    static constexpr int SL = 4 * NB;
    static constexpr int kNCW = 4 * GROUPS;
    static constexpr int kRow = D + 8;  // row stride of red_o: the slots' rows start in different banks
    uint8_t stage[STAGES][kStageBytes];
    alignas(16) float4 meta[STAGES];  // scales of a packed tile, by bulk copy with the tile
    int4 info[STAGES];                // {packed, position of the first key, valid keys, 0}
    alignas(16) float red_o[kNCW][SL][kRow];
    float red_m[kNCW][SL], red_l[kNCW][SL], red_u[kNCW];
    int red_packed[kNCW];             // order of red_o's channels (packed_pos)
    // With several column blocks the Q^T fragments of all warps live here (16-bit tiles: head and remainder, third
    // terms of bfloat16; packed tiles), with one in each warp's registers.
    static constexpr int kSets = (BF16 ? 2 : 1) + (PACKED ? 1 : 0);
    uint2 qf[NB > 1 ? kSets : 1][NB > 1 ? NB : 1][D / 16][32];
    uint64_t full[STAGES], empty[STAGES];
    int flag, abort;
};

__device__ __forceinline__ uint32_t f16x2_of_e4m3x2(uint32_t x) {  // low 16 bits of x
    uint32_t y;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t f16x2_of_e4m3x2_hi(uint32_t x) {  // high 16 bits of x
    uint32_t y;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;\n\t}" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint4 lds_u4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint2 lds_u2(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
// Untiled bulk copy global -> shared (16-byte aligned on both sides), completion on an mbarrier.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
        "l"(src), "r"(bytes), "r"(smem_u32(bar))
        : "memory");
}

// Channel group (D / 8 consecutive channels, 16-byte chunk or half of one) that
// lane group g takes of a packed V row, and, for head_dim 128, the key of a
// strip's row g: a permutation that spreads a shared-memory phase over all banks.
template <int D> __device__ __forceinline__ int spread(int g) { return D == 128 ? ((g & 1) << 2 | g >> 1) : g; }
template <int D> __device__ __forceinline__ int unspread(int c) { return D == 128 ? ((c & 3) << 1 | c >> 2) : c; }

// Place of channels c, c + 1 (c even) in a row of red_o written in the order of
// packed tiles' accumulators: lane group major, so that a warp's stores meet all banks.
template <int D> __device__ __forceinline__ int packed_pos(int c) {
    return (((c & (D / 8 - 1)) >> 1) * 8 + unspread<D>(c / (D / 8))) * 2;
}

// A warp's Q^T operand fragments: column n = lane / 4 is query slot
// 4 nb + n / 2, the head (n even) or the remainder (n odd) of q times a power
// of two that puts the row's largest magnitude into [2^4, 2^5). a: k-steps of
// head and remainder, c: third terms (bfloat16). mul[nb]: for the lane's own
// softmax slot 4 nb + lane % 4, what turns products into log2 units.
template <int D, int NB>
struct QFrag {
    uint32_t a[NB][D / 16][2], c[NB][D / 16][2];
    float mul[NB];
};

// Fragments of one set (a or c) of all column blocks -> shared memory.
template <int D, int NB>
__device__ __forceinline__ void store_q(uint2 (*dst)[D / 16][32], const uint32_t (&f)[NB][D / 16][2]) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) dst[nb][kk][threadIdx.x & 31] = make_uint2(f[nb][kk][0], f[nb][kk][1]);
}

// Channels of k-step kk, register h, of lane t: packed tiles 64 (kk / 4) + 16 t + 4 (kk % 4) + 2 h (the lane's 16
// consecutive codes), 16-bit tiles 16 kk + 2 t + 8 h (ldmatrix).
template <typename T, int D, int NB, bool PACKED_TILE, bool THIRD>
__device__ __forceinline__ void load_q(QFrag<D, NB>& q, const float* __restrict__ base, const OutMap& om, int bh,
                                       int slot0, int nslots, float qscale) {
    const int lane = threadIdx.x & 31, n = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int sl = 4 * nb + (n >> 1);
        const bool live = sl < nslots;
        const float* row = base + om.row(bh, live ? slot0 + sl : slot0) * D;
        float x[D / 16][4];
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            const int d0 = PACKED_TILE ? 64 * (kk >> 2) + 16 * t + 4 * (kk & 3) : 16 * kk + 2 * t;
            const int d1 = PACKED_TILE ? d0 + 2 : d0 + 8;
            const float2 u = *reinterpret_cast<const float2*>(row + d0), v = *reinterpret_cast<const float2*>(row + d1);
            x[kk][0] = live ? u.x : 0.f;
            x[kk][1] = live ? u.y : 0.f;
            x[kk][2] = live ? v.x : 0.f;
            x[kk][3] = live ? v.y : 0.f;
        }
        float a = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int j = 0; j < 4; ++j) a = fmaxf(a, fabsf(x[kk][j]));
        a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
        a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
        int e = a > 0.f ? 4 + 127 - (int)(__float_as_uint(a) >> 23) : 0;  // a infinite: 2^-124, q stays infinite
        e = max(-126, min(126, e));
        const float up = __uint_as_float((uint32_t)(e + 127) << 23);
        q.mul[nb] = __shfl_sync(0xffffffffu, qscale * __uint_as_float((uint32_t)(127 - e) << 23), 8 * t);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float x0 = x[kk][2 * h] * up, x1 = x[kk][2 * h + 1] * up;
                const float h0 = round16<T>(x0), h1 = round16<T>(x1);
                const float r0 = x0 - h0, r1 = x1 - h1;
                q.a[nb][kk][h] = (n & 1) ? pack2<T>(r0, r1) : pack2<T>(h0, h1);
                if (THIRD) q.c[nb][kk][h] = (n & 1) ? 0u : pack2<T>(r0 - round16<T>(r0), r1 - round16<T>(r1));
            }
    }
}

// Online-softmax state of a warp, one value per lane and column block: lane
// (g, t) = (lane / 4, lane % 4) holds keys g and g + 8 of a strip for query
// slot 4 nb + t.
template <int D, int NB>
struct State {
    float acc[NB][D / 16][4];
    float m[NB], l[NB];
    float u, inv_u;  // largest V scale met so far; O is in units of u * 2^-7
};

// One strip's logits -> P^T operand fragments (b: head|remainder, b3: third
// terms of bfloat16); s0, s1 in log2 units, -inf where masked.
template <typename T, int D, int NB, bool THIRD>
__device__ __forceinline__ void softmax_strip(State<D, NB>& st, const float (&s0)[NB], const float (&s1)[NB], float sv,
                                              uint32_t (&b)[NB][2], uint32_t (&b3)[NB][2]) {
    bool up = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) up |= fmaxf(s0[nb], s1[nb]) > st.m[nb] + kLazy;
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float tm = fmaxf(s0[nb], s1[nb]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, off));
            const float mn = fmaxf(st.m[nb], tm);
            const float al = mn == -CUDART_INF_F ? 1.f : ex2_approx(st.m[nb] - mn);
            st.m[nb] = mn;
            st.l[nb] *= al;
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                for (int j = 0; j < 4; ++j) st.acc[nb][dt][j] *= al;
        }
    }
    if (sv > st.u) {  // the same for the whole warp
        const float r = st.u / sv;
        st.u = sv;
        st.inv_u = 1.f / sv;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                for (int j = 0; j < 4; ++j) st.acc[nb][dt][j] *= r;
    }
    const float f = sv * st.inv_u * kPScale;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const float ms = st.m[nb] == -CUDART_INF_F ? 0.f : st.m[nb];
        const float p0 = ex2_approx(s0[nb] - ms), p1 = ex2_approx(s1[nb] - ms);
        st.l[nb] += p0 + p1;
        const float x0 = p0 * f, x1 = p1 * f;
        const float h0 = round16<T>(x0), h1 = round16<T>(x1);
        const float r0 = x0 - h0, r1 = x1 - h1;
        b[nb][0] = movmatrix_trans(pack2<T>(h0, r0));
        b[nb][1] = movmatrix_trans(pack2<T>(h1, r1));
        if (THIRD) {
            b3[nb][0] = movmatrix_trans(pack2<T>(r0 - round16<T>(r0), 0.f));
            b3[nb][1] = movmatrix_trans(pack2<T>(r1 - round16<T>(r1), 0.f));
        }
    }
}

// Consumer warps come in GROUPS of four; item i of a split belongs to group
// i % GROUPS (a divisor of STAGES, so each stage has one group of its own).
template <typename T, int D, int NB, int GROUPS, int STAGES, int CTAS, bool PACKED>
__global__ void __launch_bounds__((4 * GROUPS + 1) * 32, CTAS)
archive_attn_kernel(const __grid_constant__ CUtensorMap mapK16, const __grid_constant__ CUtensorMap mapV16,
                    const __grid_constant__ CUtensorMap mapK8, const __grid_constant__ CUtensorMap mapV8,
                    const __grid_constant__ CUtensorMap stripK8, const __grid_constant__ CUtensorMap stripV8,
                    const Params p) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    using Geo = Geometry<D>;
    using Sm = Smem<D, NB, GROUPS, STAGES, PACKED, BF16>;
    static_assert(STAGES % GROUPS == 0, "a stage belongs to one group");
    constexpr int kNCW = Sm::kNCW;
    constexpr int SL = Sm::SL;
    constexpr int HK = Geo::kHotKeys;
    extern __shared__ uint8_t smem_raw[];
    Sm& sm = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int list = blockIdx.x, split = blockIdx.y, zb = blockIdx.z;
    const int row0 = p.per_query ? list % p.q_len : 0;             // query row of a list of its own
    const int bh = p.per_query ? list / p.q_len : list;
    const int slot0 = (p.per_query ? row0 * p.G : 0) + zb * SL;    // first query slot handled: slot = row * G + head
    const int nslots = min(SL, (p.per_query ? row0 * p.G : 0) + p.slots - slot0);
    const int4* tiles = p.tiles + (p.per_query ? (size_t)list * p.n_tiles : 0);
    constexpr int kPer = PACKED ? 1 : Geo::kItemsPerTile16;        // items per archived tile
    const int arch_items = p.n_tiles * kPer;
    const int item0 = split * p.items_per_split;

    int q_pos0 = p.q_pos0, head = p.head, hlen = p.hlen, hstart = p.hstart;
    int first = 0, total = 0;
    auto plan = [&]() {
        first = min(hlen, p.capacity - head);
        total = arch_items + (first + HK - 1) / HK + (hlen - first + HK - 1) / HK;
    };
    auto read_state = [&](bool report) {
        q_pos0 = p.dyn[RFSN_STEP_POS];
        head = p.dyn[RFSN_STEP_HEAD];
        hlen = p.dyn[RFSN_STEP_LENGTH];
        hstart = p.dyn[RFSN_STEP_START];
        if (head < 0 || head >= p.capacity || hlen < 0 || hlen > p.capacity) {  // malformed: attend to no hot key
            if (report) atomicExch(p.ws.error, kDevErrBadTable);
            head = 0;
            hlen = 0;
        }
        plan();
    };
    plan();

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 4);
        }
        sm.abort = 0;
        fence_mbar_init();
    }
    __syncthreads();

    if (warp == kNCW) {
        // ---------------- producer ----------------
        // The descriptors of 32 items are fetched by the 32 lanes together;
        // lane 0 issues the copies. A list written by the kernel this one
        // overlaps, the step state and the ring rows are read after the
        // dependency wait; the tiles of the page table before it.
        bool waited = false;
        auto wait_dep = [&]() {
            if (!waited) {
                griddep_wait();
                waited = true;
                if (p.dyn != nullptr) read_state(false);
            }
        };
        if (p.per_query) wait_dep();
        const int arch_end = min(item0 + p.items_per_split, arch_items);
        int it = 0;
        bool stop = false;
        auto issue = [&](int4 d, int packed) {  // d = {arena row, position, valid keys, scale slot}
            if (lane == 0) {
                const int s = it % STAGES;
                if (it >= STAGES && !mbar_wait_bounded(&sm.empty[s], ((it / STAGES) + 1) & 1, &sm.abort)) {
                    atomicExch(&sm.abort, 1);
                    atomicExch(p.ws.error, kDevErrTimeout);
                    stop = true;
                } else {
                    sm.info[s] = make_int4(packed, d.y, d.z, 0);
                    uint8_t* st = sm.stage[s];
                    if (d.z <= 0) {
                        mbar_arrive(&sm.full[s]);  // nothing to load
                    } else if (PACKED && packed) {
                        // of a tile at a block's end only the strips of 16 keys that it has
                        const int strips = (d.z + 15) / 16, r = bh * p.packed_rows + d.x;
                        mbar_arrive_expect_tx(&sm.full[s], strips * 32 * D + 16);
                        if (strips == 4) {
                            tma_load_2d(st, &mapK8, 0, r, &sm.full[s]);
                            tma_load_2d(st + Geo::kVPacked, &mapV8, 0, r, &sm.full[s]);
                        } else {
                            for (int i = 0; i < strips; ++i) {
                                tma_load_2d(st + 16 * D * i, &stripK8, 0, r + 16 * i, &sm.full[s]);
                                tma_load_2d(st + Geo::kVPacked + 16 * D * i, &stripV8, 0, r + 16 * i, &sm.full[s]);
                            }
                        }
                        bulk_load(&sm.meta[s], p.scales + (size_t)bh * (p.packed_rows / kTile) + d.x / kTile, 16,
                                  &sm.full[s]);
                    } else {
                        mbar_arrive_expect_tx(&sm.full[s], kStageBytes);
                        const int r = bh * p.rows + d.x;
#pragma unroll
                        for (int h = 0; h < Geo::kHalves; ++h) {
                            tma_load_2d(st + h * HK * 128, &mapK16, 64 * h, r, &sm.full[s]);
                            tma_load_2d(st + Geo::kV16 + h * HK * 128, &mapV16, 64 * h, r, &sm.full[s]);
                        }
                    }
                }
            }
            stop = __shfl_sync(0xffffffffu, stop, 0);
            ++it;
        };
        for (int base = item0; base < arch_end && !stop; base += 32) {
            const int i = base + lane;
            int4 d = make_int4(0, 0, 0, 0);
            if (i < arch_end) {
                d = __ldcg(tiles + i / kPer);
                const int rows = PACKED ? p.packed_rows : p.rows;
                if (d.x < 0 || d.z < 0 || d.z > kTile || d.x > rows - d.z || (PACKED && (d.x & (kTile - 1)) != 0)) {
                    atomicExch(p.ws.error, kDevErrBadTable);  // a tile outside the arena: skipped
                    d = make_int4(0, 0, 0, 0);
                }
                if (kPer > 1) {
                    const int off = (i % kPer) * HK;
                    d.x += off;
                    d.y += off;
                    d.z = max(0, min(HK, d.z - off));
                }
            }
            const int n = min(32, arch_end - base);
            for (int j = 0; j < n && !stop; ++j) {
                const int4 e = make_int4(__shfl_sync(0xffffffffu, d.x, j), __shfl_sync(0xffffffffu, d.y, j),
                                         __shfl_sync(0xffffffffu, d.z, j), 0);
                issue(e, PACKED ? 1 : 0);
            }
        }
        if (!stop && item0 + p.items_per_split > arch_items) {
            wait_dep();
            const int end = min(item0 + p.items_per_split, total);
            const int items_a = (first + HK - 1) / HK;
            for (int i = max(item0, arch_items); i < end && !stop; ++i) {
                int h = i - arch_items;
                int4 d;
                if (h < items_a) {
                    d = make_int4(p.ring_row0 + head + h * HK, hstart + h * HK, min(HK, first - h * HK), 0);
                } else {
                    h -= items_a;
                    d = make_int4(p.ring_row0 + h * HK, hstart + first + h * HK, min(HK, hlen - first - h * HK), 0);
                }
                issue(d, 0);
            }
        }
        return;
    }

    // ---------------- consumers ----------------
    const int g = lane >> 2, t4 = lane & 3;
    const OutMap om{p.q_heads, p.kv_heads, p.q_len, D, p.G};
    // q, the step state and the workspace may belong to the kernel this one overlaps
    griddep_wait();
    if (p.dyn != nullptr) read_state(threadIdx.x == 0 && split == 0 && list == 0 && zb == 0);
    const int nitems = min(p.items_per_split, total - item0);

    QFrag<D, NB> q;
    bool packed_order = PACKED && nitems > 0 && item0 < arch_items;
    constexpr bool QS = NB > 1;
    constexpr int kPackedSet = Sm::kSets - 1;
    if constexpr (QS) {
        if (!PACKED || warp != 1) load_q<T, D, NB, false, BF16>(q, p.q, om, bh, slot0, nslots, p.qscale);
        if (warp == 0) {
            store_q<D, NB>(sm.qf[0], q.a);
            if constexpr (BF16) store_q<D, NB>(sm.qf[1], q.c);
        }
        if (PACKED && warp == 1) {
            load_q<__half, D, NB, true, false>(q, p.q, om, bh, slot0, nslots, p.qscale);
            store_q<D, NB>(sm.qf[kPackedSet], q.a);
        }
        named_barrier_sync(1, kNCW * 32);
    } else {
        if (PACKED && packed_order)
            load_q<__half, D, NB, true, false>(q, p.q, om, bh, slot0, nslots, p.qscale);
        else
            load_q<T, D, NB, false, BF16>(q, p.q, om, bh, slot0, nslots, p.qscale);
    }
    // operand of k-step kk: set 0 head and remainder, 1 third terms (16-bit tiles), kPackedSet packed tiles
    auto qop = [&](int set, int nb, int kk) {
        if constexpr (QS) return sm.qf[set][nb][kk][lane];
        if (BF16 && set == 1 && !(PACKED && kPackedSet == 1)) return make_uint2(q.c[nb][kk][0], q.c[nb][kk][1]);
        return make_uint2(q.a[nb][kk][0], q.a[nb][kk][1]);
    };
    int qp[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) qp[nb] = q_pos0 + (slot0 + 4 * nb + t4) / p.G;
    const int qlast = q_pos0 + (slot0 + nslots - 1) / p.G;  // keys behind it reach no slot of the CTA: neither K nor V is used
    State<D, NB> st;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        st.m[nb] = -CUDART_INF_F;
        st.l[nb] = 0.f;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j) st.acc[nb][dt][j] = 0.f;
    }
    st.u = 0.f;
    st.inv_u = 0.f;
    // Channel of accumulator row g (+ 8 h) of strip dt: packed tiles
    // chan0 + 2 dt + h, 16-bit tiles 16 dt + 8 h + g.
    const int cg = spread<D>(g);
    const int chan0 = cg * (D / 8);

    const int mi = lane >> 3, ri = lane & 7;
    const int group = warp >> 2, gwarp = warp & 3;
    int next = group;  // first item of this group not consumed yet
    for (int it = group; it < nitems; it += GROUPS) {
        const int s = it % STAGES;
        if (!mbar_wait_bounded(&sm.full[s], (it / STAGES) & 1, &sm.abort)) {
            atomicExch(&sm.abort, 1);
            atomicExch(p.ws.error, kDevErrTimeout);
            break;
        }
        next = it + GROUPS;
        const int4 inf = sm.info[s];
        const uint32_t sb = smem_u32(sm.stage[s]);
        if (PACKED && inf.x) {
            const int k_strip = 16 * ((gwarp + it / GROUPS) & 3);  // in turn: a block's short last tile is not always warp 0's
            const int seen = min(inf.z, qlast - inf.y + 1) - k_strip;
            const bool mine = seen > 0;
            if (mine) {
                const float4 sc = sm.meta[s];
                const int ka = k_strip + (D == 128 ? cg : g), kb = ka + 8;  // rows ka and kb share the swizzle pattern
                uint32_t wa[D / 16], wb[D / 16];
#pragma unroll
                for (int half = 0; half < D / 64; ++half) {
                    const int ch = t4 + 4 * half;
                    const uint32_t swz = D == 128 ? (ch ^ (ka & 7)) : (ch ^ ((ka >> 1) & 3));
                    const uint4 xa = lds_u4(sb + ka * D + (swz << 4)), xb = lds_u4(sb + kb * D + (swz << 4));
                    wa[4 * half] = xa.x, wa[4 * half + 1] = xa.y, wa[4 * half + 2] = xa.z, wa[4 * half + 3] = xa.w;
                    wb[4 * half] = xb.x, wb[4 * half + 1] = xb.y, wb[4 * half + 2] = xb.z, wb[4 * half + 3] = xb.w;
                }
                // V: keys of P^T rows 2t, 2t + 1 and 2t + 8, 2t + 9; D / 8 consecutive channels per lane.
                // With one column block they are fetched before the logits are needed and free the stage early;
                // with more there are no registers to hold them through the softmax.
                const int v0 = k_strip + (D == 128 ? t4 : 2 * t4), v1 = D == 128 ? v0 + 4 : v0 + 1;
                const uint32_t vb = sb + Geo::kVPacked;
                uint32_t x0[D / 32], x1[D / 32], x2[D / 32], x3[D / 32];
                auto fetch_v = [&]() {
                    if constexpr (D == 128) {
                        const uint4 y0 = lds_u4(vb + v0 * D + ((cg ^ (v0 & 7)) << 4));
                        const uint4 y1 = lds_u4(vb + v1 * D + ((cg ^ (v1 & 7)) << 4));
                        const uint4 y2 = lds_u4(vb + (v0 + 8) * D + ((cg ^ (v0 & 7)) << 4));
                        const uint4 y3 = lds_u4(vb + (v1 + 8) * D + ((cg ^ (v1 & 7)) << 4));
                        x0[0] = y0.x, x0[1] = y0.y, x0[2] = y0.z, x0[3] = y0.w;
                        x1[0] = y1.x, x1[1] = y1.y, x1[2] = y1.z, x1[3] = y1.w;
                        x2[0] = y2.x, x2[1] = y2.y, x2[2] = y2.z, x2[3] = y2.w;
                        x3[0] = y3.x, x3[1] = y3.y, x3[2] = y3.z, x3[3] = y3.w;
                    } else {
                        const int ch = g >> 1, lo = (g & 1) * 8;
                        auto at = [&](int key) { return lds_u2(vb + key * D + ((ch ^ ((key >> 1) & 3)) << 4) + lo); };
                        const uint2 y0 = at(v0), y1 = at(v1), y2 = at(v0 + 8), y3 = at(v1 + 8);
                        x0[0] = y0.x, x0[1] = y0.y, x1[0] = y1.x, x1[1] = y1.y;
                        x2[0] = y2.x, x2[1] = y2.y, x3[0] = y3.x, x3[1] = y3.y;
                    }
                    if (seen < 16) {
                        const int k0 = v0 - k_strip, k1 = v1 - k_strip;
#pragma unroll
                        for (int w = 0; w < D / 32; ++w) {
                            x0[w] = k0 < seen ? x0[w] : 0u;
                            x1[w] = k1 < seen ? x1[w] : 0u;
                            x2[w] = k0 + 8 < seen ? x2[w] : 0u;
                            x3[w] = k1 + 8 < seen ? x3[w] : 0u;
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.empty[s]);
                };
                if (NB == 1) fetch_v();
                float c[NB][2][4];  // two chains of dependent products
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[nb][0][j] = c[nb][1][j] = 0.f;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t a[4] = {f16x2_of_e4m3x2(wa[kk]), f16x2_of_e4m3x2(wb[kk]), f16x2_of_e4m3x2_hi(wa[kk]),
                                           f16x2_of_e4m3x2_hi(wb[kk])};
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const uint2 o = qop(kPackedSet, nb, kk);
                        MmaOp<__half>::run(c[nb][kk & 1], a, o.x, o.y);
                    }
                }
                float s0[NB], s1[NB];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const float f = q.mul[nb] * sc.x;
                    s0[nb] = (ka < inf.z && inf.y + ka <= qp[nb])
                                 ? ((c[nb][0][0] + c[nb][1][0]) + (c[nb][0][1] + c[nb][1][1])) * f : -CUDART_INF_F;
                    s1[nb] = (kb < inf.z && inf.y + kb <= qp[nb])
                                 ? ((c[nb][0][2] + c[nb][1][2]) + (c[nb][0][3] + c[nb][1][3])) * f : -CUDART_INF_F;
                }
                uint32_t b[NB][2], b3[NB][2];
                softmax_strip<__half, D, NB, false>(st, s0, s1, sc.z == 0.f ? sc.y : kTiny, b, b3);  // z: V all zero
                if (NB > 1) fetch_v();
#pragma unroll
                for (int w = 0; w < D / 32; ++w) {
                    // interleave the two keys' bytes: each half word is one channel of both
                    const uint32_t lo01 = __byte_perm(x0[w], x1[w], 0x5140), hi01 = __byte_perm(x0[w], x1[w], 0x7362);
                    const uint32_t lo23 = __byte_perm(x2[w], x3[w], 0x5140), hi23 = __byte_perm(x2[w], x3[w], 0x7362);
                    const uint32_t a0[4] = {f16x2_of_e4m3x2(lo01), f16x2_of_e4m3x2_hi(lo01), f16x2_of_e4m3x2(lo23),
                                            f16x2_of_e4m3x2_hi(lo23)};
                    const uint32_t a1[4] = {f16x2_of_e4m3x2(hi01), f16x2_of_e4m3x2_hi(hi01), f16x2_of_e4m3x2(hi23),
                                            f16x2_of_e4m3x2_hi(hi23)};
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        MmaOp<__half>::run(st.acc[nb][2 * w], a0, b[nb][0], b[nb][1]);
                        MmaOp<__half>::run(st.acc[nb][2 * w + 1], a1, b[nb][0], b[nb][1]);
                    }
                }
            } else {
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.empty[s]);
            }
        } else {
            // 16-bit item: HK / 16 strips; with two strips the group's warp pairs take turns
            const int strip = HK == 64 ? (gwarp + it / GROUPS) & 3 : (gwarp & 1);
            const bool mine = HK == 64 || (gwarp >> 1) == ((it / GROUPS) & 1);
            const int sv = min(inf.z, qlast - inf.y + 1) - 16 * strip;  // keys of the strip that some slot sees
            if (mine && sv > 0) {
                if (PACKED && packed_order) {  // first 16-bit strip after packed ones: reorder O's channels, q's fragments
                    packed_order = false;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int dt = 0; dt < D / 16; ++dt) {
                            float* o = &sm.red_o[warp][4 * nb + t4][chan0 + 2 * dt];
                            o[0] = st.acc[nb][dt][0] + st.acc[nb][dt][1];
                            o[1] = st.acc[nb][dt][2] + st.acc[nb][dt][3];
                        }
                    __syncwarp();
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int dt = 0; dt < D / 16; ++dt) {
                            const float* o = &sm.red_o[warp][4 * nb + t4][16 * dt + g];
                            st.acc[nb][dt][0] = o[0];
                            st.acc[nb][dt][2] = o[8];
                            st.acc[nb][dt][1] = st.acc[nb][dt][3] = 0.f;
                        }
                    __syncwarp();
                    if (!QS) load_q<T, D, NB, false, BF16>(q, p.q, om, bh, slot0, nslots, p.qscale);
                }
                float c[NB][2][4];  // two chains of dependent products
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[nb][0][j] = c[nb][1][j] = 0.f;
                const int kkey = 16 * strip + ri + 8 * (mi & 1);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const int chunk = (kk & 3) * 2 + (mi >> 1);
                    uint32_t a[4];
                    ldmatrix_x4(a, sb + (kk >> 2) * HK * 128 + kkey * 128 + ((chunk ^ (kkey & 7)) << 4));
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const uint2 o = qop(0, nb, kk);
                        MmaOp<T>::run(c[nb][BF16 ? 0 : kk & 1], a, o.x, o.y);
                        if (BF16) {
                            const uint2 o3 = qop(1, nb, kk);
                            MmaOp<T>::run(c[nb][1], a, o3.x, o3.y);
                        }
                    }
                }
                const int ka = 16 * strip + g, kb = ka + 8;
                float s0[NB], s1[NB];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    s0[nb] = (ka < inf.z && inf.y + ka <= qp[nb])
                                 ? ((c[nb][0][0] + c[nb][1][0]) + (c[nb][0][1] + c[nb][1][1])) * q.mul[nb] : -CUDART_INF_F;
                    s1[nb] = (kb < inf.z && inf.y + kb <= qp[nb])
                                 ? ((c[nb][0][2] + c[nb][1][2]) + (c[nb][0][3] + c[nb][1][3])) * q.mul[nb] : -CUDART_INF_F;
                }
                uint32_t b[NB][2], b3[NB][2];
                softmax_strip<T, D, NB, BF16>(st, s0, s1, 1.f, b, b3);
                uint32_t m01 = 0xffffffffu, m23 = 0xffffffffu;  // rows that no slot sees hold anything: zero them
                if (sv < 16) {
                    const int k2 = 2 * t4;
                    m01 = (k2 < sv ? 0x0000ffffu : 0u) | (k2 + 1 < sv ? 0xffff0000u : 0u);
                    m23 = (k2 + 8 < sv ? 0x0000ffffu : 0u) | (k2 + 9 < sv ? 0xffff0000u : 0u);
                }
                const int vkey = 16 * strip + ri + 8 * (mi >> 1);
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt) {
                    const int chunk = (dt & 3) * 2 + (mi & 1);
                    uint32_t a[4];
                    ldmatrix_x4_trans(a, sb + Geo::kV16 + (dt >> 2) * HK * 128 + vkey * 128 + ((chunk ^ (vkey & 7)) << 4));
                    a[0] &= m01;
                    a[1] &= m01;
                    a[2] &= m23;
                    a[3] &= m23;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        MmaOp<T>::run(st.acc[nb][dt], a, b[nb][0], b[nb][1]);
                        if (BF16) MmaOp<T>::run(st.acc[nb][dt], a, b3[nb][0], b3[nb][1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.empty[s]);
        }
    }

    griddep_launch_dependents();
    if (sm.abort) {
        // Drain: wait (bounded) for loads already issued into stages we did not consume.
        for (int it = next; it < min(nitems, next + STAGES); it += GROUPS)
            mbar_wait_bounded(&sm.full[it % STAGES], (it / STAGES) & 1, nullptr);
    }

    // ---------------- warp -> CTA merge ----------------
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) st.l[nb] += __shfl_xor_sync(0xffffffffu, st.l[nb], off);
        const int sl = 4 * nb + t4;
        float* row = sm.red_o[warp][sl];
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
            const float o0 = st.acc[nb][dt][0] + st.acc[nb][dt][1], o1 = st.acc[nb][dt][2] + st.acc[nb][dt][3];
            if (PACKED && packed_order) {
                *reinterpret_cast<float2*>(row + (dt * 8 + g) * 2) = make_float2(o0, o1);
            } else {
                row[16 * dt + g] = o0;
                row[16 * dt + 8 + g] = o1;
            }
        }
        if (g == 0) {
            sm.red_m[warp][sl] = st.m[nb];
            sm.red_l[warp][sl] = st.l[nb];
        }
    }
    if (lane == 0) {
        sm.red_u[warp] = st.u * (1.f / kPScale);
        sm.red_packed[warp] = packed_order;
    }
    named_barrier_sync(1, kNCW * 32);

    const int counter = list * gridDim.z + zb;
    const size_t part_base = (size_t)counter * p.splits * SL;
    constexpr int V4 = D / 4;  // float4 per row
    for (int i = threadIdx.x; i < nslots * V4; i += kNCW * 32) {
        const int sl = i / V4, d4 = i % V4;
        float M = -CUDART_INF_F, L = 0.f;
#pragma unroll
        for (int w = 0; w < kNCW; ++w) M = fmaxf(M, sm.red_m[w][sl]);
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kNCW; ++w) {
            const float mw = sm.red_m[w][sl];
            // a warp without keys has weight 0; NaN maxima cannot occur (fmaxf drops them), NaN sums stay
            const float wt = M == -CUDART_INF_F ? 1.f : ex2_approx(mw - M);
            const float wo = wt * sm.red_u[w];
            float4 o;
            if (PACKED && sm.red_packed[w]) {
                const float* r = sm.red_o[w][sl] + packed_pos<D>(4 * d4);
                const float2 a = *reinterpret_cast<const float2*>(r), b = *reinterpret_cast<const float2*>(r + 16);
                o = make_float4(a.x, a.y, b.x, b.y);
            } else {
                o = reinterpret_cast<const float4*>(sm.red_o[w][sl])[d4];
            }
            L += wt * sm.red_l[w][sl];
            O.x += wo * o.x;
            O.y += wo * o.y;
            O.z += wo * o.z;
            O.w += wo * o.w;
        }
        if (p.splits == 1) {
            const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
            const size_t r = om.row(bh, slot0 + sl);
            *reinterpret_cast<float4*>(p.out + r * D + 4 * d4) = make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv);
            if (p.lse != nullptr && d4 == 0)
                p.lse[r] = L > 0.f || L != L ? (M + log2f(L)) * 0.69314718055994531f : -CUDART_INF_F;
        } else {
            const size_t part = part_base + (size_t)split * SL + sl;
            reinterpret_cast<float4*>(p.ws.o + part * D)[d4] = O;
            if (d4 == 0) {
                p.ws.m[part] = M;
                p.ws.l[part] = L;
            }
        }
    }
    if (p.splits == 1) return;

    static_assert(SL * (D / 4) <= 2 * kNCW * 32, "two float4 of the result per thread");
    merge_splits<D>(p, om, bh, slot0, nslots, SL, counter, &sm.stage[0][0], STAGES * kStageBytes, &sm.red_o[0][0][0],
                    sm.red_l[0], &sm.flag, kNCW * 32);
}

// Launch shape by column blocks: consumer groups, stages and CTAs per SM. With two column blocks a CTA needs the
// registers of a whole SM's share; two CTAs of four warps with one block are 50 us at 128K, one of eight 53.
template <int NB> struct Shape;
template <> struct Shape<1> { static constexpr int kGroups = 1, kStages = 6, kCtas = 2; };
template <> struct Shape<2> { static constexpr int kGroups = 2, kStages = 8, kCtas = 1; };

template <typename T, int D, int NB, bool PACKED>
rfsn_status launch(const rfsn_arena* arena, const rfsn_packed_archive* packed, const Params& p, int lists, int zblocks,
                   cudaStream_t s) {
    using Sh = Shape<NB>;
    const size_t smem = sizeof(Smem<D, NB, Sh::kGroups, Sh::kStages, PACKED, std::is_same<T, __nv_bfloat16>::value>) + 1024;
    auto kern = archive_attn_kernel<T, D, NB, Sh::kGroups, Sh::kStages, Sh::kCtas, PACKED>;
    static std::atomic<bool> ready[64];  // the attribute stays with the kernel on each device
    const int dev = arena->device;
    if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
        RFSN_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_relaxed);
    }
    const CUtensorMap& k8 = PACKED ? packed->maps[0] : arena->item_maps[0];
    const CUtensorMap& v8 = PACKED ? packed->maps[1] : arena->item_maps[1];
    const CUtensorMap& ks = PACKED ? packed->maps[2] : arena->item_maps[0];
    const CUtensorMap& vs = PACKED ? packed->maps[3] : arena->item_maps[1];
    RFSN_CUDA(launch_kernel(p.overlap, kern, dim3(lists, p.splits, zblocks), dim3((4 * Sh::kGroups + 1) * 32), smem, s,
                         arena->item_maps[0], arena->item_maps[1], k8, v8, ks, vs, p));
    note_launch();
    return RFSN_OK;
}

template <typename T, int D, int NB>
rfsn_status launch_packed(const rfsn_arena* a, const rfsn_packed_archive* pk, const Params& p, int lists, int zb,
                          cudaStream_t s) {
    return pk != nullptr ? launch<T, D, NB, true>(a, pk, p, lists, zb, s) : launch<T, D, NB, false>(a, pk, p, lists, zb, s);
}

template <typename T, int D>
rfsn_status launch_nb(const rfsn_arena* a, const rfsn_packed_archive* pk, const Params& p, int lists, int nb, int zb,
                      cudaStream_t s) {
    if (nb == 1) return launch_packed<T, D, 1>(a, pk, p, lists, zb, s);
    return launch_packed<T, D, 2>(a, pk, p, lists, zb, s);
}

template <typename T, int D, int NB>
void preload_nb() {
    using Sh = Shape<NB>;
    cudaFuncAttributes a;
    cudaFuncGetAttributes(&a, archive_attn_kernel<T, D, NB, Sh::kGroups, Sh::kStages, Sh::kCtas, true>);
    cudaFuncGetAttributes(&a, archive_attn_kernel<T, D, NB, Sh::kGroups, Sh::kStages, Sh::kCtas, false>);
}

template <typename T, int D>
void preload() {
    preload_nb<T, D, 1>();
    preload_nb<T, D, 2>();
}

}  // namespace archive

int archive_attn_ctas(int nb) {
    using namespace archive;
    return nb == 1 ? Shape<1>::kCtas : Shape<2>::kCtas;
}

rfsn_status archive_attn_launch(const rfsn_arena* arena, const rfsn_packed_archive* packed, const archive::Params& p,
                                int lists, int nb, int zblocks, cudaStream_t s) {
    using namespace archive;
    const bool d128 = arena->head_dim == 128;
    if (arena->dtype == RFSN_BF16)
        return d128 ? launch_nb<__nv_bfloat16, 128>(arena, packed, p, lists, nb, zblocks, s)
                    : launch_nb<__nv_bfloat16, 64>(arena, packed, p, lists, nb, zblocks, s);
    return d128 ? launch_nb<__half, 128>(arena, packed, p, lists, nb, zblocks, s)
                : launch_nb<__half, 64>(arena, packed, p, lists, nb, zblocks, s);
}

void preload_archive_kernels() {
    using namespace archive;
    preload_pack_kernels();
    preload_select_kernels();
    preload_rows_kernels();
    preload_chunk_kernels();
    preload<__nv_bfloat16, 128>();
    preload<__nv_bfloat16, 64>();
    preload<__half, 128>();
    preload<__half, 64>();
}

}  // namespace rfsn
