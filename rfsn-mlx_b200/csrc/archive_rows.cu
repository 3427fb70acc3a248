// Attention of a few query rows (5 to 16 query slots at a time) over a packed
// archive and the hot window on tcgen05 tensor cores, head_dim 128.
//
//   out = softmax(q K^T / sqrt(D) + causal) V,  K = code * s_k(tile), V = code * s_v(tile)
//
// The tensor core takes the e4m3 codes as they arrive: with the keys (then the
// channels) as the 128 rows of the product,
//   S^T[128 keys x N] = K[128 x D] . Q^T[D x N]        (kind::f8f6f4)
//   O^T[D x N]        = V^T[D x 128] . P^T[128 x N]
// nothing has to be widened or moved. The float32 operand becomes five e4m3
// terms, each the rounded remainder of the one before times 2^5: x = sum_j
// 2^-5j t_j + e with |e| <= 2^-24 |x| (a term rounds to 4 bits, the remainder
// begins 5 bits lower), 2^-30 for x below e4m3's normal range (q is scaled to a
// row maximum of 2^8, p is at most 2^8 and mostly about 1). Term j of slot s is column j SL + s of the product, so
// terms never meet in an accumulator and the 2^-5j are applied to the sums, in
// float32. N is 80 for 16 slots: 52 cycles per instruction, 420 per tile of
// 128 keys, where HBM needs about 1,400; accumulation over the 128 products of
// a column measured 3e-8 of their magnitudes.
//
// P V of one tile is a fresh accumulation; the softmax warps add the tiles in
// registers (acc = acc + u O_t), so each tile has its own unit u of V, the
// larger scale of its two 64-token halves. The reference maximum of the
// softmax is lazy (kLazy), so p <= 2^8 fits e4m3's range.
//
// The hot window (16-bit ring) takes the same way with kind::f16: 128 ring
// keys, their K and V in two stages, q and p in two float16 or three bfloat16
// terms of weight 1.
//
// Measured, 32 q / 8 KV heads: 4 rows (16 slots) over 31K packed tokens and 2K
// ring 23.3 us (two passes of the tile kernel 33.8; 11.1 at the copy rate), 131K
// 59.5 (107); 2 rows over 131K 53.4 (59). About 11 us of it (16 slots; 8.5 with
// 8) is there without keys: q, the first item, the merge. Above that an item of
// 128 keys takes 0.85 us of a CTA (0.66 of HBM time): the softmax warps' issue
// slots. Four groups of 8 slots in 640 threads took 29.8 us.
//
// Warps: 0-3 and 4-7 two softmax groups that take tiles in turn (thread = key
// of S^T, then channel of O^T) and merge at the end; 8 producer (TMA); 9 MMA
// issuer: S(t), then O(t - 2).
#include <math_constants.h>

#include <atomic>

#include "archive.cuh"
#include "tcgen05.cuh"

namespace rfsn {
namespace archive {
namespace rows {

constexpr int D = 128;
constexpr int BN = 128;                  // keys per item
constexpr int kStages = 5;
constexpr int kItemBytes = 2 * BN * D;   // K and V codes of an item, or K or V of a hot item
constexpr int kInfo = 8;                 // posted at most kStages items ahead
constexpr int kTerms = 5;
constexpr int kSoftmaxThreads = 256, kThreads = 320;
constexpr int kProducerWarp = 8, kMmaWarp = 9;
constexpr uint32_t kTmemCols = 512, kBuf = 80;  // four S and two O buffers of up to 80 columns
constexpr uint32_t kTmemS = 0, kTmemO = 4 * kBuf;
constexpr float kMinF = 7.8886091e-31f;   // 2^-100

struct Info {
    int pos[2], len[2];
    float sk[2], sv[2];
};

constexpr int round16up(int n) { return (n + 15) / 16 * 16; }

template <int SL, bool BF16>
struct Smem {
    static constexpr int kN8 = round16up(kTerms * SL);
    static constexpr int kTerms16 = BF16 ? 3 : 2;
    static constexpr int kN16 = round16up(kTerms16 * SL);
    static constexpr int kRow = D + 4;
    uint8_t stage[kStages][kItemBytes];
    uint8_t q8[kN8 * D];          // Q^T terms, 128-byte-swizzled rows (term, slot)
    uint8_t q16[2][kN16 * 128];   // the same in 16 bits, by channel half
    uint8_t p[2][BN * 128];       // P^T terms of the two groups, a row of columns per key; at the end the merge's weights
    uint64_t full[kStages], empty[kStages];
    uint64_t s_full[4], p_full[2], o_full[2], mma_done;
    Info info[kInfo];
    alignas(16) float qmul[SL];   // what turns products into log2 units
    int row[SL];                  // query row of a slot, relative to the call's first; unused slots see nothing
    alignas(16) float red[2][4][SL];
    int bad[2][4];
    float m[2][SL], l[2][SL], inv[SL];
    uint32_t tmem;
    int abort, flag;
};

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* abort_flag) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag));
}
__device__ __forceinline__ void fail(int* abort_flag, const Params& p) {
    atomicExch(abort_flag, 1);
    atomicExch(p.ws.error, kDevErrTimeout);
}
// Two floats -> two e4m3 codes (low byte a), rounded to nearest.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
// -32 times the values of two codes (exact in float16).
__device__ __forceinline__ float2 minus32(uint32_t codes) {
    uint32_t y;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(y) : "r"(codes));
    return __half22float2(__hmul2(*reinterpret_cast<const __half2*>(&y), __float2half2_rn(-32.f)));
}
__device__ __forceinline__ void sts_v2(uint32_t addr, uint2 v) {
    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ void sts_v4(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
}
// Barrier of a softmax group: does any of its threads raise its hand?
__device__ __forceinline__ bool group_any(int group, bool hand) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)hand), "r"(2 + group)
        : "memory");
    return r != 0;
}

// SL values per lane reduced over the warp's lanes, each step halving the values a lane carries (SL instead of
// 5 SL shuffles). The result of slot `slot` comes out in every lane with own_slot(lane) == slot.
template <int SL, typename Op>
__device__ __forceinline__ float reduce_slots(const float2 (&x)[SL / 2], Op op) {
    const int lane = threadIdx.x & 31;
    float v[SL];
#pragma unroll
    for (int s = 0; s < SL; ++s) v[s] = (s & 1) ? x[s / 2].y : x[s / 2].x;
#pragma unroll
    for (int n = SL / 2, bit = 16; n > 0; n >>= 1, bit >>= 1) {
        const bool up = lane & bit;
#pragma unroll
        for (int s = 0; s < n; ++s) {
            const float other = __shfl_xor_sync(0xffffffffu, up ? v[s] : v[s + n], bit);
            v[s] = op(up ? v[s + n] : v[s], other);
        }
    }
#pragma unroll
    for (int bit = 16 / SL; bit > 0; bit >>= 1) v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], bit));
    return v[0];
}
template <int SL> __device__ __forceinline__ int own_slot(int lane) {  // bits of the lane from the highest down
    return SL == 16 ? lane >> 1 : lane >> 2;
}

// A row of SL * terms sums from TMEM, the terms joined: e4m3 terms by their weights (in two loads: the registers of
// all five at once would not stay in place), 16-bit ones as they are.
template <int SL, int TERMS16>
__device__ __forceinline__ void load_joined(uint32_t taddr, bool codes, float2 (&x)[SL / 2]) {
    static_assert(kTerms == 5 && TERMS16 <= 3, "columns");
    uint32_t r[2 * SL], r4[SL];
    auto two = [](const uint32_t* w) { return make_float2(__uint_as_float(w[0]), __uint_as_float(w[1])); };
    auto pair_of_terms = [&](uint32_t at) {
        if constexpr (SL == 16) tc::ld_32x32b_x32_sync(at, r);
        else tc::ld_32x32b_x16_sync(at, r);
    };
    auto term = [&](uint32_t at) {
        if constexpr (SL == 16) tc::ld_32x32b_x16_sync(at, r4);
        else tc::ld_32x32b_x8_sync(at, r4);
    };
    const float2 down = both(0.03125f);
    if (codes) {
        term(taddr + 4 * SL);
        pair_of_terms(taddr + 2 * SL);
#pragma unroll
        for (int s = 0; s < SL / 2; ++s)
            x[s] = fma2(fma2(two(r4 + 2 * s), down, two(r + SL + 2 * s)), down, two(r + 2 * s));
        pair_of_terms(taddr);
#pragma unroll
        for (int s = 0; s < SL / 2; ++s) x[s] = fma2(fma2(x[s], down, two(r + SL + 2 * s)), down, two(r + 2 * s));
    } else {
        pair_of_terms(taddr);
        if (TERMS16 == 3) term(taddr + 2 * SL);
#pragma unroll
        for (int s = 0; s < SL / 2; ++s) {
            const float2 low = TERMS16 == 3 ? add2(two(r4 + 2 * s), two(r + SL + 2 * s)) : two(r + SL + 2 * s);
            x[s] = add2(low, two(r + 2 * s));
        }
    }
}

template <typename T, int SL>
__global__ void __launch_bounds__(kThreads, 1)
rows_kernel(const __grid_constant__ CUtensorMap mapK8, const __grid_constant__ CUtensorMap mapV8,
            const __grid_constant__ CUtensorMap stripK8, const __grid_constant__ CUtensorMap stripV8,
            const __grid_constant__ CUtensorMap mapK16, const __grid_constant__ CUtensorMap mapV16, const Params p) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    using Sm = Smem<SL, BF16>;
    constexpr int kTerms16 = Sm::kTerms16, kN8 = Sm::kN8, kN16 = Sm::kN16;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    if ((smem_u32(smem_raw) & 1023u) != 0) {  // the swizzled tiles need 1024-byte alignment
        if (threadIdx.x == 0) atomicExch(p.ws.error, kDevErrBadTable);
        return;
    }
    Sm& sm = *reinterpret_cast<Sm*>(smem_raw);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int bh = blockIdx.x, split = blockIdx.y, zb = blockIdx.z;
    const int slot0 = zb * SL, nslots = min(SL, p.slots - slot0);

    // Items: two tiles of the list, then 128 ring keys, of twice the bytes. A split has its share of the ring items,
    // and archived items up to its share of the whole. (That count is fixed on the host from the longest window where
    // the window is only known now: the loads of archived tiles begin before.)
    auto share = [&](int items, int s) { return (int)((long long)items * s / p.splits); };
    const int arch_items = (p.n_tiles + 1) / 2;
    auto arch_before = [&](int s) {
        const int fair = share(arch_items + 2 * p.hot_items, s) - 2 * share(p.hot_items, s);
        return arch_items >= 2 * p.splits ? max(0, min(arch_items, fair)) : share(arch_items, s);
    };
    const int a0 = arch_before(split), na = arch_before(split + 1) - a0;
    int q_pos0 = p.q_pos0, head = p.head, hlen = p.hlen, hstart = p.hstart;
    int first = 0, h0 = 0, nh = 0;
    auto plan = [&]() {
        first = min(hlen, p.capacity - head);
        const int items = (first + BN - 1) / BN + (hlen - first + BN - 1) / BN;
        h0 = share(items, split);
        nh = share(items, split + 1) - h0;
    };
    auto read_state = [&](bool report) {
        if (p.dyn != nullptr) {
            q_pos0 = p.dyn[RFSN_STEP_POS];
            head = p.dyn[RFSN_STEP_HEAD];
            hlen = p.dyn[RFSN_STEP_LENGTH];
            hstart = p.dyn[RFSN_STEP_START];
            if (head < 0 || head >= p.capacity || hlen < 0 || hlen > p.capacity) {  // malformed: attend to no hot key
                if (report) atomicExch(p.ws.error, kDevErrBadTable);
                head = 0;
                hlen = 0;
            }
        }
        plan();
    };

    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&sm.s_full[i], 1);
        for (int w = 0; w < 2; ++w) {
            mbar_init(&sm.p_full[w], 128);
            mbar_init(&sm.o_full[w], 1);
        }
        mbar_init(&sm.mma_done, 1);
        sm.abort = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        tc::tmem_alloc(&sm.tmem, kTmemCols);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = sm.tmem;

    if (warp == kProducerWarp) {
        // ---------------- producer ----------------
        // The archived tiles come before the dependency wait, the step state and the ring after it.
        int slot = 0, it = 0;
        bool stop = false;
        auto acquire = [&]() {
            if (slot < kStages || mbar_wait_bounded(&sm.empty[slot % kStages], (slot / kStages + 1) & 1, &sm.abort))
                return true;
            fail(&sm.abort, p);
            return false;
        };
        for (int base = 0; base < na && !stop; base += 16) {
            // lanes 2 j, 2 j + 1 fetch the two halves of item base + j
            const int i = 2 * (a0 + base) + lane;
            int4 e = make_int4(0, 0, 0, 0);
            float sk = 1.f, sv = kTiny;  // a half without keys or of zero V leaves the unit to the other one
            if (base + (lane >> 1) < na && i < p.n_tiles) {
                e = __ldcg(p.tiles + i);
                if (e.x < 0 || e.z < 0 || e.z > kTile || (e.x & (kTile - 1)) != 0 || e.x > p.packed_rows - e.z) {
                    atomicExch(p.ws.error, kDevErrBadTable);  // a tile outside the archive: skipped
                    e = make_int4(0, 0, 0, 0);
                } else if (e.z > 0) {
                    const float4 sc = __ldcg(p.scales + (size_t)bh * (p.packed_rows / kTile) + e.x / kTile);
                    sk = sc.x;
                    if (sc.z == 0.f) sv = sc.y;  // else a tile of zeros
                }
            }
            const int n = min(16, na - base);
            for (int j = 0; j < n && !stop; ++j) {
                int r[2];
                Info inf;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    r[h] = __shfl_sync(0xffffffffu, e.x, 2 * j + h);
                    inf.pos[h] = __shfl_sync(0xffffffffu, e.y, 2 * j + h);
                    inf.len[h] = __shfl_sync(0xffffffffu, e.z, 2 * j + h);
                    inf.sk[h] = __shfl_sync(0xffffffffu, sk, 2 * j + h);
                    inf.sv[h] = __shfl_sync(0xffffffffu, sv, 2 * j + h);
                }
                if (lane == 0) {
                    if (!acquire()) {
                        stop = true;
                    } else {
                        sm.info[it % kInfo] = inf;
                        uint64_t* full = &sm.full[slot % kStages];
                        uint8_t* dst = sm.stage[slot % kStages];
                        // of a tile at a block's end only the strips of 16 keys that it has
                        const int strips[2] = {(inf.len[0] + 15) / 16, (inf.len[1] + 15) / 16};
                        if (strips[0] + strips[1] > 0)
                            mbar_arrive_expect_tx(full, (strips[0] + strips[1]) * 32 * D);
                        else
                            mbar_arrive(full);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int g = bh * p.packed_rows + r[h];
                            uint8_t* k = dst + h * kTile * D;
                            if (strips[h] == 4) {
                                tma_load_2d(k, &mapK8, 0, g, full);
                                tma_load_2d(k + BN * D, &mapV8, 0, g, full);
                            } else {
                                for (int i = 0; i < strips[h]; ++i) {
                                    tma_load_2d(k + 16 * D * i, &stripK8, 0, g + 16 * i, full);
                                    tma_load_2d(k + BN * D + 16 * D * i, &stripV8, 0, g + 16 * i, full);
                                }
                            }
                        }
                    }
                }
                ++slot;
                ++it;
                stop = __shfl_sync(0xffffffffu, stop, 0);
            }
        }
        if (!stop && (p.dyn != nullptr || p.hlen > 0)) {
            griddep_wait();
            read_state(false);
            const int items_a = (first + BN - 1) / BN;
            for (int j = 0; j < nh && !stop; ++j) {
                const int h = h0 + j;
                const bool a = h < items_a;
                const int off = (a ? h : h - items_a) * BN;
                const int len = min(BN, (a ? first : hlen - first) - off);
                if (lane == 0) {
                    const int pos = hstart + (a ? 0 : first) + off;
                    const int g = bh * p.rows + p.ring_row0 + (a ? head : 0) + off;
                    for (int w = 0; w < 2 && !stop; ++w) {  // K, then V
                        if (!acquire()) {
                            stop = true;
                            break;
                        }
                        if (w == 0) {
                            Info inf;
                            inf.pos[0] = pos;
                            inf.pos[1] = pos + kTile;
                            inf.len[0] = min(kTile, len);
                            inf.len[1] = len - inf.len[0];
                            inf.sk[0] = inf.sk[1] = inf.sv[0] = inf.sv[1] = 1.f;
                            sm.info[it % kInfo] = inf;
                        }
                        uint64_t* full = &sm.full[slot % kStages];
                        uint8_t* dst = sm.stage[slot % kStages];
                        const int boxes = len > kTile ? 2 : 1;  // of 64 keys
                        mbar_arrive_expect_tx(full, boxes * 2 * kTile * 128);
                        for (int c = 0; c < 2; ++c)
                            for (int b = 0; b < boxes; ++b)
                                tma_load_2d(dst + c * BN * 128 + b * kTile * 128, w ? &mapV16 : &mapK16, 64 * c,
                                            g + b * kTile, full);
                        ++slot;
                    }
                }
                ++it;
                stop = __shfl_sync(0xffffffffu, stop, 0);
            }
        }
        // copies in flight land before the CTA exits (on success the tensor core has consumed them all)
        if (lane == 0 && sm.abort)
            for (int i = max(0, slot - kStages); i < slot; ++i)
                mbar_wait_bounded(&sm.full[i % kStages], (i / kStages) & 1, nullptr);
    } else if (warp == kMmaWarp) {
        // ---------------- MMA issuer ----------------
        griddep_wait();
        read_state(false);
        named_barrier_sync(4, kSoftmaxThreads + 32);  // q is in shared memory
        const bool leader = tc::elect_leader();  // the whole warp waits and counts, one lane issues
        constexpr uint32_t id_s8 = tc::idesc_e4m3(false, false, BN, kN8), id_o8 = tc::idesc_e4m3(true, true, D, kN8);
        constexpr uint32_t id_s16 = tc::idesc_f16(BF16, false, false, BN, kN16);
        constexpr uint32_t id_o16 = tc::idesc_f16(BF16, true, true, D, kN16);
        const int n = na + nh;
        auto k_slot = [&](int t) { return t < na ? t : na + 2 * (t - na); };
        bool ok = true;
        for (int t = 0; t < n + 2 && ok; ++t) {
            if (t < n) {
                const int ks = k_slot(t);
                // S buffer t % 4: the sums of t - 4 were read before P(t - 4), waited for below, was posted
                ok = warp_wait(&sm.full[ks % kStages], (ks / kStages) & 1, &sm.abort);
                if (!ok) break;
                tc::fence_after_sync();
                const uint32_t tS = tmem + kTmemS + kBuf * (t & 3), k = smem_u32(sm.stage[ks % kStages]);
                if (t < na) {
#pragma unroll
                    for (int kk = 0; kk < D / 32; ++kk)
                        tc::mma_e4m3_ss(leader, tS, tc::smem_desc_sw128(k + 32 * kk, 16, 1024),
                                        tc::smem_desc_sw128(smem_u32(sm.q8) + 32 * kk, 16, 1024), id_s8, kk > 0);
                } else {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        tc::mma_f16_ss(leader, tS, tc::smem_desc_sw128(k + (kk >> 2) * BN * 128 + 32 * (kk & 3), 16, 1024),
                                       tc::smem_desc_sw128(smem_u32(sm.q16[kk >> 2]) + 32 * (kk & 3), 16, 1024),
                                       id_s16, kk > 0);
                }
                tc::commit(leader, &sm.s_full[t & 3]);
            }
            if (t > 1) {
                const int u = t - 2, w = u & 1, ks = k_slot(u), vs = u < na ? ks : ks + 1;
                ok = warp_wait(&sm.full[vs % kStages], (vs / kStages) & 1, &sm.abort) &&
                     warp_wait(&sm.p_full[w], (u >> 1) & 1, &sm.abort);  // O(u - 2) read out as well
                if (!ok) break;
                tc::fence_after_sync();
                const uint32_t tO = tmem + kTmemO + kBuf * w, pb = smem_u32(sm.p[w]);
                const uint32_t v = smem_u32(sm.stage[vs % kStages]);
                if (u < na) {
#pragma unroll
                    for (int kk = 0; kk < BN / 32; ++kk)
                        tc::mma_e4m3_ss(leader, tO, tc::smem_desc_sw128(v + BN * D + 32 * 128 * kk, 16, 1024),
                                        tc::smem_desc_sw128(pb + 32 * 128 * kk, 16, 1024), id_o8, kk > 0);
                } else {
#pragma unroll
                    for (int kk = 0; kk < BN / 16; ++kk)
                        tc::mma_f16_ss(leader, tO, tc::smem_desc_sw128(v + 16 * 128 * kk, BN * 128, 1024),
                                       tc::smem_desc_sw128(pb + 16 * 128 * kk, 16, 1024),
                                       id_o16, kk > 0);
                }
                tc::commit(leader, &sm.o_full[w]);
                tc::commit(leader, &sm.empty[ks % kStages]);
                if (vs != ks) tc::commit(leader, &sm.empty[vs % kStages]);
            }
        }
        if (!ok && lane == 0) fail(&sm.abort, p);
        // no tensor-core work may be in flight when TMEM is released
        tc::commit(leader, &sm.mma_done);
        mbar_wait_bounded(&sm.mma_done, 0, nullptr);
    } else {
        // ---------------- softmax groups ----------------
        griddep_wait();  // q, the step state and the workspace may belong to the kernel this one overlaps
        read_state(tid == 0 && split == 0 && bh == 0 && zb == 0);
        const OutMap om{p.q_heads, p.kv_heads, p.q_len, D, p.G};
        if (tid < 16 * SL) {  // 16 threads per slot, 8 channels each
            const int s = tid >> 4, c = 8 * (tid & 15);
            const bool live = s < nslots;
            const float* src = p.q + om.row(bh, slot0 + (live ? s : 0)) * D + c;
            float x[8];
            float a = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const float4 y = *reinterpret_cast<const float4*>(src + i);
                x[i] = live ? y.x : 0.f, x[i + 1] = live ? y.y : 0.f;
                x[i + 2] = live ? y.z : 0.f, x[i + 3] = live ? y.w : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(x[i]));
#pragma unroll
            for (int off = 8; off > 0; off >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, off));
            // the slot's largest magnitude to [2^7, 2^8)
            int e = a > 0.f ? 7 + 127 - (int)(__float_as_uint(a) >> 23) : 0;
            e = max(-126, min(126, e));
            const float up = __uint_as_float((uint32_t)(e + 127) << 23);
            if (c == 0) {
                sm.qmul[s] = p.qscale * __uint_as_float((uint32_t)(127 - e) << 23);
                sm.row[s] = live ? (slot0 + s) / p.G : INT_MIN;
            }
            // an infinity makes every logit of the row infinite or NaN; e4m3 has none
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = a == CUDART_INF_F ? CUDART_NAN_F : x[i] * up;
            if (na > 0) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[i];
#pragma unroll
                for (int j = 0; j < kTerms; ++j) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        w[i] = e4m3x2(y[2 * i], y[2 * i + 1]);
                        const float2 t = minus32(w[i]);
                        y[2 * i] = fmaf(y[2 * i], 32.f, t.x);
                        y[2 * i + 1] = fmaf(y[2 * i + 1], 32.f, t.y);
                    }
                    const int r = j * SL + s;
                    *reinterpret_cast<uint2*>(sm.q8 + r * 128 + (c ^ ((r & 7) << 4))) =
                        make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
                }
            }
            if (nh > 0) {
#pragma unroll
                for (int j = 0; j < kTerms16; ++j) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float t0 = round16<T>(x[2 * i]), t1 = round16<T>(x[2 * i + 1]);
                        w[i] = pack2<T>(t0, t1);
                        x[2 * i] -= t0;
                        x[2 * i + 1] -= t1;
                    }
                    const int r = j * SL + s;
                    *reinterpret_cast<uint4*>(sm.q16[c >> 6] + r * 128 + ((2 * (c & 63)) ^ ((r & 7) << 4))) =
                        make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        tc::fence_proxy_async_smem();
        named_barrier_sync(4, kSoftmaxThreads + 32);

        const int w = warp >> 2, gw = warp & 3, r = tid & 127;
        const int half = r >> 6, ki = r & 63;  // key of the item: half and place in it
        const uint32_t lane_base = (uint32_t)(32 * gw) << 16;
        const uint32_t tS = tmem + kTmemS + lane_base, tO = tmem + kTmemO + kBuf * w + lane_base;
        const uint32_t pb = smem_u32(sm.p[w]);
        const int row_first = slot0 / p.G, qlast = q_pos0 + (slot0 + nslots - 1) / p.G;
        const int n = na + nh;
        constexpr int H = SL / 2;  // slots in pairs
        float2 acc[H], nm[H], l[H], qm[H];  // O of channel r, minus the reference maximum, sums of the thread's keys
        uint32_t fresh = (1u << nslots) - 1u;  // slots that have seen no key yet (their reference is 0)
#pragma unroll
        for (int s = 0; s < H; ++s) {
            acc[s] = l[s] = nm[s] = both(0.f);
            qm[s] = *reinterpret_cast<const float2*>(sm.qmul + 2 * s);
        }
        float unit = 0.f;    // of the O buffer not added yet
        bool codes = true;   // its terms
        bool ok = true;
        auto drain = [&]() {
            float2 o[H];
            tc::fence_after_sync();
            load_joined<SL, kTerms16>(tO, codes, o);
#pragma unroll
            for (int s = 0; s < H; ++s) acc[s] = fma2(o[s], both(unit), acc[s]);
        };
        int t = w;
        for (; t < n; t += 2) {
            const bool arch = t < na;
            const int ks = arch ? t : na + 2 * (t - na), vs = arch ? ks : ks + 1, k = t >> 1;
            ok = warp_wait(&sm.full[ks % kStages], (ks / kStages) & 1, &sm.abort) &&
                 warp_wait(&sm.s_full[t & 3], (t >> 2) & 1, &sm.abort) && (k == 0 || warp_wait(&sm.o_full[w], (k - 1) & 1, &sm.abort));
            float2 x[H];
            if (ok) {
                tc::fence_after_sync();
                load_joined<SL, kTerms16>(tS + kBuf * (t & 3), arch, x);
                if (k > 0) drain();
            } else {
#pragma unroll
                for (int s = 0; s < H; ++s) x[s] = both(0.f);
            }
            const Info& inf = sm.info[t % kInfo];
            const int len = inf.len[half], pos = inf.pos[half];
            const float sk = inf.sk[half];
            // the item's unit: the larger scale of the halves that some slot sees
            const float u = fmaxf(inf.pos[0] <= qlast ? inf.sv[0] : kTiny, inf.pos[1] <= qlast ? inf.sv[1] : kTiny);
            // p times f: the key's share of the unit, nothing to a half behind it (16-bit items: a power of two that
            // fits float16)
            const float f = arch ? fminf(fmaxf(inf.sv[half] / u, kMinF), 1.f) : kPScale;
            // logits in log2 units below the reference maximum
#pragma unroll
            for (int s = 0; s < H; ++s) x[s] = fma2(x[s], mul2(qm[s], both(sk)), nm[s]);
            const int seen = min(len, qlast - pos + 1);  // keys of this half that some slot sees
            if (len < kTile || pos + kTile - 1 > q_pos0 + row_first) {  // the same for the whole warp
                const int rel = ki < len ? pos + ki - q_pos0 : INT_MAX;
#pragma unroll
                for (int s = 0; s < H; ++s) {
                    if (rel > sm.row[2 * s]) x[s].x = -CUDART_INF_F;
                    if (rel > sm.row[2 * s + 1]) x[s].y = -CUDART_INF_F;
                }
            }
            float top = -CUDART_INF_F;
#pragma unroll
            for (int s = 0; s < H; ++s) top = fmaxf(top, fmaxf(x[s].x, x[s].y));
            if (group_any(w, top > kLazy || fresh != 0 || !ok)) {  // a maximum moves, or a wait gave up
                const float tm = reduce_slots<SL>(x, [](float a, float b) { return fmaxf(a, b); });
                if ((lane & (32 / SL - 1)) == 0) sm.red[w][gw][own_slot<SL>(lane)] = tm;
                if (lane == 0) sm.bad[w][gw] = !ok;
                named_barrier_sync(2 + w, 128);
                if (sm.bad[w][0] | sm.bad[w][1] | sm.bad[w][2] | sm.bad[w][3]) {
                    ok = false;
                    break;  // the whole group
                }
#pragma unroll
                for (int s = 0; s < SL; ++s) {
                    float& nms = (s & 1) ? nm[s / 2].y : nm[s / 2].x;
                    float& xs = (s & 1) ? x[s / 2].y : x[s / 2].x;
                    float& ls = (s & 1) ? l[s / 2].y : l[s / 2].x;
                    float& as = (s & 1) ? acc[s / 2].y : acc[s / 2].x;
                    const float up = fmaxf(fmaxf(sm.red[w][0][s], sm.red[w][1][s]), fmaxf(sm.red[w][2][s], sm.red[w][3][s]));
                    // a slot's first maximum replaces 0, later ones only rise
                    const bool first_key = (fresh >> s) & 1;
                    if (up > (first_key ? -CUDART_INF_F : 0.f)) {
                        fresh &= ~(1u << s);
                        const float next = nms - up, d = next - nms;  // what the rounded maximum moved by
                        const float al = first_key ? 1.f : tc::ex2(d);
                        nms = next;
                        xs += d;
                        ls *= al;
                        as *= al;
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < H; ++s) {
                const float2 pr = make_float2(tc::ex2(x[s].x), tc::ex2(x[s].y));
                l[s] = add2(l[s], pr);
                x[s] = mul2(pr, both(f));
            }
            // P^T, N-major: the key's row of columns (term, slot)
            const uint32_t prow = pb + r * 128;
            auto chunk = [&](int c) { return prow + ((c ^ (r & 7)) << 4); };
            if (arch) {
#pragma unroll
                for (int j = 0; j < kTerms; ++j) {
                    uint32_t c[H];
#pragma unroll
                    for (int s = 0; s < H; ++s) {
                        c[s] = e4m3x2(x[s].x, x[s].y);
                        if (j < kTerms - 1) x[s] = fma2(x[s], both(32.f), minus32(c[s]));
                    }
                    if constexpr (SL == 16)
                        sts_v4(chunk(j), make_uint4(c[0] | c[1] << 16, c[2] | c[3] << 16, c[4] | c[5] << 16, c[6] | c[7] << 16));
                    else
                        sts_v2(chunk(j >> 1) + 8 * (j & 1), make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16));
                }
            } else {
#pragma unroll
                for (int j = 0; j < kTerms16; ++j) {
                    uint32_t c[H];
#pragma unroll
                    for (int s = 0; s < H; ++s) {
                        const float2 y = make_float2(round16<T>(x[s].x), round16<T>(x[s].y));
                        c[s] = pack2<T>(y.x, y.y);
                        x[s] = sub2(x[s], y);
                    }
#pragma unroll
                    for (int i = 0; i < H / 4; ++i)
                        sts_v4(chunk(j * (H / 4) + i), make_uint4(c[4 * i], c[4 * i + 1], c[4 * i + 2], c[4 * i + 3]));
                }
            }
            if (seen < kTile && ki >= seen) {  // V of keys that no slot sees may hold anything: zeroed
                // a hot item's V comes behind its K: the copy must have landed
                if (!arch && !mbar_wait_bounded(&sm.full[vs % kStages], (vs / kStages) & 1, &sm.abort)) fail(&sm.abort, p);
                const uint32_t v = smem_u32(sm.stage[vs % kStages]) + (arch ? BN * D : 0) + r * 128;
#pragma unroll
                for (int i = 0; i < 8; ++i) sts_v4(v + ((16 * i) ^ ((r & 7) << 4)), make_uint4(0, 0, 0, 0));
                if (!arch) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) sts_v4(v + BN * 128 + ((16 * i) ^ ((r & 7) << 4)), make_uint4(0, 0, 0, 0));
                }
            }
            unit = arch ? u : 1.f / kPScale;
            codes = arch;
            tc::fence_proxy_async_smem();
            tc::fence_before_sync();
            mbar_arrive(&sm.p_full[w]);
        }
        if (!ok) fail(&sm.abort, p);
        if (ok && t > w) {  // the group's last product
            ok = warp_wait(&sm.o_full[w], ((t - 2) >> 1) & 1, &sm.abort);
            if (ok)
                drain();
            else
                fail(&sm.abort, p);
        }
        griddep_launch_dependents();
        // row sums over the group's keys
        const float sum = reduce_slots<SL>(l, [](float a, float b) { return a + b; });
        if ((lane & (32 / SL - 1)) == 0) sm.red[w][gw][own_slot<SL>(lane)] = sum;
        if (r == 0) {
#pragma unroll
            for (int s = 0; s < SL; ++s)
                sm.m[w][s] = (fresh >> s) & 1 ? -CUDART_INF_F : -((s & 1) ? nm[s / 2].y : nm[s / 2].x);
        }
        tc::fence_before_sync();
        named_barrier_sync(1, kSoftmaxThreads);
        float* red = reinterpret_cast<float*>(sm.stage[0]);  // [2][SL][kRow]
#pragma unroll
        for (int s = 0; s < SL; ++s) red[(w * SL + s) * Sm::kRow + r] = (s & 1) ? acc[s / 2].y : acc[s / 2].x;
        if (r < SL) sm.l[w][r] = sm.red[w][0][r] + sm.red[w][1][r] + sm.red[w][2][r] + sm.red[w][3][r];
    }
    __syncthreads();
    if (warp == kMmaWarp) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
    if (warp >= kProducerWarp) return;

    // ---------------- both groups -> the CTA's partial ----------------
    const OutMap om{p.q_heads, p.kv_heads, p.q_len, D, p.G};
    const float* red = reinterpret_cast<const float*>(sm.stage[0]);
    const int counter = bh * gridDim.z + zb;
    constexpr int V4 = D / 4;
    for (int i = tid; i < nslots * V4; i += kSoftmaxThreads) {
        const int s = i / V4, d4 = i % V4;
        const float M = fmaxf(sm.m[0][s], sm.m[1][s]);
        float L = 0.f;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const float wt = M == -CUDART_INF_F ? 1.f : ex2_approx(sm.m[w][s] - M);
            const float4 o = *reinterpret_cast<const float4*>(red + (w * SL + s) * Sm::kRow + 4 * d4);
            L += wt * sm.l[w][s];
            O.x += wt * o.x;
            O.y += wt * o.y;
            O.z += wt * o.z;
            O.w += wt * o.w;
        }
        if (p.splits == 1) {
            const bool any = L > 0.f || L != L;
            const float inv = any ? 1.f / L : 0.f;
            const size_t row = om.row(bh, slot0 + s);
            *reinterpret_cast<float4*>(p.out + row * D + 4 * d4) = make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv);
            if (p.lse != nullptr && d4 == 0)
                p.lse[row] = any ? (M + log2f(L)) * 0.69314718055994531f : -CUDART_INF_F;
        } else {
            const size_t part = ((size_t)counter * p.splits + split) * SL + s;
            reinterpret_cast<float4*>(p.ws.o + part * D)[d4] = O;
            if (d4 == 0) {
                p.ws.m[part] = M;
                p.ws.l[part] = L;
            }
        }
    }
    if (p.splits == 1) return;
    static_assert(sizeof(sm.p) >= SL * kMaxSplits128 * sizeof(float), "room for the merge's weights");
    static_assert(SL * V4 <= 2 * kSoftmaxThreads, "two float4 of the result per thread");
    merge_splits<D>(p, om, bh, slot0, nslots, SL, counter, &sm.stage[0][0], sizeof(sm.stage),
                    reinterpret_cast<float*>(sm.p[0]), sm.inv, &sm.flag, kSoftmaxThreads);
}

template <typename T, int SL>
rfsn_status launch(const rfsn_arena* arena, const rfsn_packed_archive* packed, const Params& p, int lists, int zblocks,
                   cudaStream_t s) {
    using Sm = Smem<SL, std::is_same<T, __nv_bfloat16>::value>;
    static std::atomic<bool> ready[64];  // the attribute stays with the kernel on each device
    const int dev = arena->device;
    if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
        RFSN_CUDA(cudaFuncSetAttribute(rows_kernel<T, SL>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Sm)));
        if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_relaxed);
    }
    RFSN_CUDA(launch_kernel(p.overlap, rows_kernel<T, SL>, dim3(lists, p.splits, zblocks), dim3(kThreads), sizeof(Sm), s,
                            packed->maps[0], packed->maps[1], packed->maps[2], packed->maps[3], arena->maps[0],
                            arena->maps[1], p));
    note_launch();
    return RFSN_OK;
}

}  // namespace rows
}  // namespace archive

rfsn_status archive_rows_launch(const rfsn_arena* arena, const rfsn_packed_archive* packed, const archive::Params& p,
                                int lists, int slots, int zblocks, cudaStream_t s) {
    using namespace archive::rows;
    if (arena->dtype == RFSN_BF16)
        return slots == 8 ? launch<__nv_bfloat16, 8>(arena, packed, p, lists, zblocks, s)
                          : launch<__nv_bfloat16, 16>(arena, packed, p, lists, zblocks, s);
    return slots == 8 ? launch<__half, 8>(arena, packed, p, lists, zblocks, s)
                      : launch<__half, 16>(arena, packed, p, lists, zblocks, s);
}

void preload_rows_kernels() {
    using namespace archive::rows;
    cudaFuncAttributes a;
    cudaFuncGetAttributes(&a, rows_kernel<__nv_bfloat16, 8>);
    cudaFuncGetAttributes(&a, rows_kernel<__nv_bfloat16, 16>);
    cudaFuncGetAttributes(&a, rows_kernel<__half, 8>);
    cudaFuncGetAttributes(&a, rows_kernel<__half, 16>);
}

}  // namespace rfsn
