// Attention of a chunk of queries over a packed archive and the hot window on
// tcgen05 tensor cores.
//
//   out = softmax(q K^T / sqrt(D) + causal) V,  K = code * s_k(tile), V = code * s_v(tile)
//
// A chunk is bound by its products, so the e4m3 codes are widened to float16
// (exact) once per CTA and tile on their way into the operand buffers, and the
// scales stay outside: s_k multiplies the logit, s_v the probability. CTA =
// one KV head x 128 query rows packed GQA-style (row r: head r % G at chunk
// position r / G), keys in tiles of 128 = two 64-token tiles of the list, each
// with its own position, length and scales.
//
// Accuracy. q (times a power of two per row) and P (times 2^7 s_v / u, u the
// larger s_v of the two halves) are split into two float16 each: 22 bits. The
// tensor core adds into its float32 accumulator with truncation, an error
// that grows with the number of additions; P V of one tile is therefore a
// fresh accumulation of 16 steps, and the tiles are added in registers by the
// softmax warps (acc = acc + w O_t, rounded to nearest). That also makes the
// softmax's rescale a register multiplication, and lets every tile have its
// own unit u.
//
// The hot window (bf16 or f16 ring) is first copied by hot_half_kernel into
// float16 tiles of 64 tokens with a power-of-two scale each (the smallest for a
// tile of zeros): an element keeps its 8 or 11 bits unless it is 2^-29 of its
// tile's maximum, so the main kernel sees one kind of operand.
//
// Measured: 512 rows over 16K packed tokens and 1K ring, 32 q / 8 KV heads, 249
// us back to back = 580 TFLOP/s useful, 1,160 executed (273 us and 527 with other
// work between the calls); a tile of 128 keys takes 3,300 cycles of which the
// products are 2,050 at full rate. They are issued by a converged warp and its
// elected lane: from a one-lane branch the same kernel took 287 us.
// head_dim 64, 256 rows of 32 heads over 16K: 116 us (743 in passes of 8 slots).
//
// Warps (512 threads, registers shifted to the softmax warps by setmaxnreg):
//   0-7   softmax: warp w owns TMEM lane quarter w % 4 (thread = row) and key
//         half w / 4 of a tile; then O's channel half w / 4
//   8-11  converters: staged codes (or float16 hot tiles) -> operand buffers in
//         the 128-byte-swizzle layout
//   12    producer: TMA into the staging slots, tile info
//   13    MMA issuer: S(t) = Q K(t)^T, then O(t - 1) = P(t - 1) V(t - 1)
// TMEM: two S/P buffers [0, 256), O [256, 384), q hi/lo [384, 512).
// Every wait is bounded and reports through the workspace's error word.
#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <cstring>

#include "archive.cuh"
#include "tcgen05.cuh"

namespace rfsn {
namespace archive {
namespace chunk {

constexpr int BM = 128;               // query rows per CTA
constexpr int BN = 128;               // keys per tile
constexpr int kHalfBytes = BN * 128;  // 64 channels of a float16 operand tile
constexpr int kStages = 2;            // staging, operand and S/P buffers alike
// Tile infos in flight. Tile t + 8 is posted when the staging slot two before its own is free, at the earliest after
// K(t + 7) was copied: S(t + 5) was done then, which needs P V (t + 3) and so the softmax of tile t to be over.
constexpr int kInfo = 8;
constexpr int kSoftmaxThreads = 256, kThreads = 512;
// registers per thread of the two softmax warpgroups and of the two others: together the 512 x 128 of the launch
constexpr int kSoftmaxRegs = 192, kOtherRegs = 64;
constexpr int kConvWarp = 8, kProducerWarp = 12, kMmaWarp = 13;
constexpr int kMaxSplit = 32;  // key ranges of a unit
constexpr float kMinF = 7.8886091e-31f;   // 2^-100
constexpr uint32_t kTmemCols = 512, kColO = 256, kColQ = 384;  // q: hi, then lo, head_dim / 2 columns each

struct Info {
    int pos[2], len[2];
    float sk[2], sv[2];
};

template <int D>
struct Smem {
    static constexpr int kCodeBytes = BN * D;  // codes of K or V of a tile
    uint8_t k[kStages][D / 64][kHalfBytes];   // float16 operands
    uint8_t v[kStages][D / 64][kHalfBytes];
    uint8_t staged[kStages][2 * kCodeBytes];  // codes of K and V of a tile, or K or V of a float16 hot tile
    uint64_t c_full[kStages], c_empty[kStages];
    uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint64_t info_full[kInfo];
    uint64_t s_full[kStages], p_full[kStages], pv_done[kStages];
    uint64_t o_empty, mma_done;
    uint64_t pair[4][2];
    uint64_t pair_l[4];
    float red[2][2][BM];
    Info info[kInfo];
    uint32_t tmem;
    int abort, n_arch, n_hot;
};

struct Params {
    const float* q;
    float* out;
    float* lse;
    const int4* tiles;
    int n_tiles;
    int packed_rows;
    const float4* scales;
    const float2* hot_scales;  // [groups][hot_rows / 64] {K, V}
    int hot_rows;              // rows of the float16 hot copy per head (a multiple of 128)
    int hlen, hstart;
    int q_heads, kv_heads, q_len, q_pos0, G, groups;
    int units, nsplit;
    float qscale;
    WsView ws;
};

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* abort_flag) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag));
}
__device__ __forceinline__ void fail(int* abort_flag, const Params& p) {
    atomicExch(abort_flag, 1);
    atomicExch(p.ws.error, kDevErrTimeout);
}
__device__ __forceinline__ uint32_t widen(uint32_t x) {  // two e4m3 codes in the low half
    uint32_t y;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t widen_hi(uint32_t x) {
    uint32_t y;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;\n\t}" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint4 lds_u4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void sts_u4(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
}
// (a, b) -> two float16 high parts and two float16 remainders. The high part
// is the value cut to 11 significant bits (exact in float16, and no
// conversion back is needed for the remainder), the remainder is exact in
// float32 and rounded to 11 bits: 21 to 22 bits together. Below float16's
// normal range bits are lost at 2^-25, 2^-32 of the largest p.
__device__ __forceinline__ void split_half(float2 x, uint32_t& hi, uint32_t& lo) {
    const float2 h = make_float2(__uint_as_float(__float_as_uint(x.x) & 0xffffe000u),
                                 __uint_as_float(__float_as_uint(x.y) & 0xffffe000u));
    const float2 r = sub2(x, h);
    hi = pack2<__half>(h.x, h.y);
    lo = pack2<__half>(r.x, r.y);
}

// The same rounded to nearest: 24 bits. For q, which is split once per CTA: an error of q moves every logit of its row.
__device__ __forceinline__ void split_half_rn(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack2<__half>(a, b);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    lo = pack2<__half>(a - f.x, b - f.y);
}

// Codes of 128 keys -> float16 operand tile: a thread widens 16 codes (one
// 16-byte chunk of a row) at a time. The lanes of a phase cover whole rows of
// codes; with head_dim 128 those of the upper channel half store their two
// chunks in the other order, so that both the load and the stores meet every
// bank once. Rows from first (second) of the two 64-key halves on are zeroed: a
// half without keys (its staging holds an earlier tile), and V of keys that no
// query row of the CTA sees.
template <int D>
__device__ __forceinline__ void convert_tile(uint32_t codes, uint32_t op, int first, int second) {
    constexpr int kChunks = D / 16, kRows = 128 / kChunks;  // chunks of a row, rows at a time
    const int th = threadIdx.x & 127, c = th % kChunks, r0 = th / kChunks;
    const int c0 = (2 * c) & 7, half = c >> 2, swap = D == 128 ? half : 0;
    // rows r0 + kRows i share r & 7, so the swizzled chunk offsets are the thread's own
    const uint32_t from = codes + r0 * D + ((D == 128 ? c ^ (r0 & 7) : c ^ ((r0 >> 1) & 3)) << 4);
    const uint32_t to = op + half * kHalfBytes + r0 * 128;
    const uint32_t to0 = to + (((c0 + swap) ^ (r0 & 7)) << 4), to1 = to + (((c0 + 1 - swap) ^ (r0 & 7)) << 4);
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // the two 64-key halves, their loads in flight together
        constexpr int kLoads = kTile / kRows;
        uint4 x[kLoads];
        const int live = (h ? second : first) - r0;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            x[i] = kRows * i < live ? lds_u4(from + (64 * h + kRows * i) * D) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint4 a = make_uint4(widen(x[i].x), widen_hi(x[i].x), widen(x[i].y), widen_hi(x[i].y));
            const uint4 b = make_uint4(widen(x[i].z), widen_hi(x[i].z), widen(x[i].w), widen_hi(x[i].w));
            sts_u4(to0 + (64 * h + kRows * i) * 128, swap ? b : a);
            sts_u4(to1 + (64 * h + kRows * i) * 128, swap ? a : b);
        }
    }
}

// A float16 tile that is already in the operand's layout; rows zeroed as above.
template <int D>
__device__ __forceinline__ void copy_tile(uint32_t from, uint32_t op, int first, int second) {
    const int th = threadIdx.x & 127;
#pragma unroll
    for (int i = 0; i < D / 64 * kHalfBytes / 16 / 128; i += 8) {
        uint4 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = (16 * (i + j) + (th >> 3)) & (BN - 1);
            x[j] = (r & 63) < (r < 64 ? first : second) ? lds_u4(from + (128 * (i + j) + th) * 16) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sts_u4(op + (128 * (i + j) + th) * 16, x[j]);
    }
}

// This warp's generic-proxy writes to an operand buffer are done: visible to
// the tensor core for whoever waits on the barrier.
__device__ __forceinline__ void publish(uint64_t* bar) {
    tc::fence_proxy_async_smem();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
chunk_kernel(const __grid_constant__ CUtensorMap mapK8, const __grid_constant__ CUtensorMap mapV8,
             const __grid_constant__ CUtensorMap mapKh, const __grid_constant__ CUtensorMap mapVh, const Params p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    if ((smem_u32(smem_raw) & 1023u) != 0) {  // the swizzled tiles need 1024-byte alignment
        if (threadIdx.x == 0) atomicExch(p.ws.error, kDevErrBadTable);
        return;
    }
    constexpr int kCodeBytes = Smem<D>::kCodeBytes;
    constexpr uint32_t kColQlo = kColQ + D / 2;
    Smem<D>& sm = *reinterpret_cast<Smem<D>*>(smem_raw);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int G = p.G, ppc = BM / G;
    // Units (query block, KV head): latest query blocks first, the heads
    // interleaved; the splits of a unit's keys are consecutive CTAs.
    const int unit = blockIdx.x / p.nsplit, split = blockIdx.x % p.nsplit;
    const int nqb = p.units / p.groups;
    const int qb = nqb - 1 - unit / p.groups, bh = unit % p.groups;
    const int b = bh / p.kv_heads, hk = bh % p.kv_heads;
    const int pos_base = qb * ppc;
    const int qlast = p.q_pos0 + min(pos_base + ppc, p.q_len) - 1;  // causal limit

    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sm.c_full[s], 1);
            mbar_init(&sm.c_empty[s], 4);
            mbar_init(&sm.k_full[s], 4);
            mbar_init(&sm.k_empty[s], 1);
            mbar_init(&sm.v_full[s], 4);
            mbar_init(&sm.v_empty[s], 1);
            mbar_init(&sm.s_full[s], 1);
            mbar_init(&sm.p_full[s], kSoftmaxThreads);
            mbar_init(&sm.pv_done[s], 1);
        }
        for (int i = 0; i < kInfo; ++i) mbar_init(&sm.info_full[i], 1);
        mbar_init(&sm.o_empty, kSoftmaxThreads);
        mbar_init(&sm.mma_done, 1);
        for (int qd = 0; qd < 4; ++qd) {
            mbar_init(&sm.pair[qd][0], 64);
            mbar_init(&sm.pair[qd][1], 64);
            mbar_init(&sm.pair_l[qd], 64);
        }
        sm.abort = 0;
        // 64-token tiles up to the causal limit (positions ascend through the list)
        int lo = 0, hi = p.n_tiles;
        if (hi > 0 && __ldcg(p.tiles + hi - 1).y <= qlast) lo = hi;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (__ldcg(p.tiles + mid).y <= qlast) lo = mid + 1; else hi = mid;
        }
        sm.n_arch = lo;
        const int seen = max(0, min(p.hlen, qlast - p.hstart + 1));
        sm.n_hot = (seen + kTile - 1) / kTile;
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
    griddep_wait();  // q, the hot copy and the workspace belong to the kernels before
    griddep_launch_dependents();
    // Tiles of 128 keys: archived pairs, then hot pairs; this split's share [t_lo, t_hi).
    const int arch_tiles = (sm.n_arch + 1) / 2, all_tiles = arch_tiles + (sm.n_hot + 1) / 2;
    const int t_lo = (int)((long long)split * all_tiles / p.nsplit);
    const int nt = (int)((long long)(split + 1) * all_tiles / p.nsplit) - t_lo;

    if (warp >= kConvWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp < kProducerWarp) {
            // ---------------- converters ----------------
            // Staging slots in order: one for an archived tile, two (K, V) for a hot one.
            int slot = 0;
            bool ok = true;
            for (int t = 0; t < nt; ++t) {
                const int s = t & 1;
                const uint32_t ph = (t >> 1) & 1;
                const bool arch = t_lo + t < arch_tiles;
                ok = warp_wait(&sm.info_full[t % kInfo], (t / kInfo) & 1, &sm.abort) &&
                     warp_wait(&sm.c_full[slot & 1], (slot >> 1) & 1, &sm.abort) &&
                     (t < kStages || warp_wait(&sm.k_empty[s], ph ^ 1, &sm.abort));
                if (!ok) break;
                const Info& inf = sm.info[t % kInfo];
                const int first = inf.len[0] > 0 ? 64 : 0, second = inf.len[1] > 0 ? 64 : 0;
                const int v_first = min(inf.len[0], qlast - inf.pos[0] + 1), v_second = min(inf.len[1], qlast - inf.pos[1] + 1);
                const uint32_t k_op = smem_u32(sm.k[s][0]), v_op = smem_u32(sm.v[s][0]);
                if (arch) {
                    convert_tile<D>(smem_u32(sm.staged[slot & 1]), k_op, first, second);
                } else {
                    copy_tile<D>(smem_u32(sm.staged[slot & 1]), k_op, first, second);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.c_empty[slot & 1]);
                    ++slot;
                }
                publish(&sm.k_full[s]);
                ok = (arch || warp_wait(&sm.c_full[slot & 1], (slot >> 1) & 1, &sm.abort)) &&
                     (t < kStages || warp_wait(&sm.v_empty[s], ph ^ 1, &sm.abort));
                if (!ok) break;
                if (arch)
                    convert_tile<D>(smem_u32(sm.staged[slot & 1]) + kCodeBytes, v_op, v_first, v_second);
                else
                    copy_tile<D>(smem_u32(sm.staged[slot & 1]), v_op, v_first, v_second);
                publish(&sm.v_full[s]);
                if (lane == 0) mbar_arrive(&sm.c_empty[slot & 1]);
                ++slot;
            }
            if (!ok) fail(&sm.abort, p);
        } else if (warp == kProducerWarp) {
            // ---------------- producer ----------------
            if (lane == 0) {
                prefetch_tmap(&mapK8);
                prefetch_tmap(&mapV8);
            }
            bool stop = false;
            int slot = 0;  // staging slots filled so far
            for (int base = 0; base < nt && !stop; base += 16) {
                // lanes 2 j, 2 j + 1 fetch the two halves of tile base + j
                const int t_mine = base + (lane >> 1), gt = t_lo + t_mine, half = lane & 1;
                int row = 0, pos = 0, len = 0;
                float sk = 1.f, sv = kTiny;  // a half without keys or of zero V leaves the unit to the other one
                if (t_mine < nt) {
                    if (gt < arch_tiles) {
                        const int i = 2 * gt + half;
                        if (i < sm.n_arch) {
                            const int4 e = __ldcg(p.tiles + i);
                            if (e.x < 0 || e.z < 0 || e.z > kTile || (e.x & (kTile - 1)) != 0 ||
                                e.x > p.packed_rows - e.z) {
                                atomicExch(p.ws.error, kDevErrBadTable);  // outside the archive: skipped
                            } else {
                                row = e.x;
                                pos = e.y;
                                len = e.z;
                                const float4 sc = __ldcg(p.scales + (size_t)bh * (p.packed_rows / kTile) + row / kTile);
                                sk = sc.x;
                                if (sc.z == 0.f) sv = sc.y;  // else a tile of zeros
                            }
                        }
                    } else {
                        const int i = 2 * (gt - arch_tiles) + half;
                        row = i * kTile;
                        pos = p.hstart + row;
                        len = max(0, min(kTile, p.hlen - row));
                        if (len > 0) {
                            const float2 sc = p.hot_scales[(size_t)bh * (p.hot_rows / kTile) + i];
                            sk = sc.x;
                            sv = sc.y;
                        }
                    }
                }
                const int n = min(16, nt - base);
                for (int j = 0; j < n && !stop; ++j) {
                    const int t = base + j;
                    int r[2];
                    Info inf;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        r[h] = __shfl_sync(0xffffffffu, row, 2 * j + h);
                        inf.pos[h] = __shfl_sync(0xffffffffu, pos, 2 * j + h);
                        inf.len[h] = __shfl_sync(0xffffffffu, len, 2 * j + h);
                        inf.sk[h] = __shfl_sync(0xffffffffu, sk, 2 * j + h);
                        inf.sv[h] = __shfl_sync(0xffffffffu, sv, 2 * j + h);
                    }
                    if (lane == 0) {
                        const bool arch = t_lo + t < arch_tiles;
                        // a staging slot is free after its conversion; the info slot then is too (kInfo)
                        auto acquire = [&]() {
                            return slot < kStages ||
                                   mbar_wait_bounded(&sm.c_empty[slot & 1], ((slot >> 1) & 1) ^ 1, &sm.abort);
                        };
                        if (!acquire()) {
                            stop = true;
                        } else {
                            sm.info[t % kInfo] = inf;
                            mbar_arrive(&sm.info_full[t % kInfo]);
                            uint64_t* full = &sm.c_full[slot & 1];
                            uint8_t* dst = sm.staged[slot & 1];
                            if (arch) {
                                const int parts = (inf.len[0] > 0) + (inf.len[1] > 0);
                                if (parts > 0)
                                    mbar_arrive_expect_tx(full, parts * 2 * kTile * D);
                                else
                                    mbar_arrive(full);
                                for (int h = 0; h < 2; ++h)
                                    if (inf.len[h] > 0) {
                                        const int g = bh * p.packed_rows + r[h];
                                        tma_load_2d(dst + h * kTile * D, &mapK8, 0, g, full);
                                        tma_load_2d(dst + kCodeBytes + h * kTile * D, &mapV8, 0, g, full);
                                    }
                                ++slot;
                            } else {
                                const int g = bh * p.hot_rows + r[0];
                                for (int w = 0; w < 2 && !stop; ++w) {  // K, then V
                                    if (w == 1) {
                                        if (!acquire()) {
                                            stop = true;
                                            break;
                                        }
                                        full = &sm.c_full[slot & 1];
                                        dst = sm.staged[slot & 1];
                                    }
                                    mbar_arrive_expect_tx(full, D / 64 * kHalfBytes);
                                    for (int c = 0; c < D / 64; ++c)
                                        for (int h = 0; h < 2; ++h)
                                            tma_load_2d(dst + c * kHalfBytes + h * kTile * 128, w ? &mapVh : &mapKh,
                                                        64 * c, g + h * kTile, full);
                                    ++slot;
                                }
                            }
                        }
                        if (stop) fail(&sm.abort, p);
                    }
                    stop = __shfl_sync(0xffffffffu, stop, 0);
                }
            }
            // copies in flight land before the CTA exits (on success the converters have consumed them all)
            if (lane == 0 && sm.abort)
                for (int i = max(0, slot - kStages); i < slot; ++i)
                    mbar_wait_bounded(&sm.c_full[i & 1], (i >> 1) & 1, nullptr);
        } else if (warp == kMmaWarp) {
            // ---------------- MMA issuer ----------------
            named_barrier_sync(1, kSoftmaxThreads + 32);  // q is in TMEM
            tc::fence_after_sync();
            if (nt > 0) {  // the whole warp waits and counts, one lane issues
                const bool leader = tc::elect_leader();
                const uint32_t id_qk = tc::idesc_f16(false, false, false, BM, BN);
                const uint32_t id_pv = tc::idesc_f16(false, false, true, BM, D);
                const uint32_t tO = tmem + kColO;
                bool ok = true;
                for (int t = 0; t <= nt && ok; ++t) {
                    const int s = t & 1;
                    const uint32_t ph = (t >> 1) & 1;
                    if (t < nt) {
                        // S buffer t % 2 last held P(t - 2)
                        ok = warp_wait(&sm.k_full[s], ph, &sm.abort) &&
                             (t < kStages || warp_wait(&sm.pv_done[s], ph ^ 1, &sm.abort));
                        if (!ok) break;
                        tc::fence_after_sync();
                        const uint32_t tS = tmem + 128 * s;
#pragma unroll 1
                        for (int part = 0; part < 2; ++part) {
                            const uint32_t tQ = tmem + (part ? kColQlo : kColQ);
#pragma unroll
                            for (int kk = 0; kk < D / 16; ++kk)
                                tc::mma_f16_ts(leader, tS, tQ + 8 * kk,
                                               tc::smem_desc_sw128(smem_u32(sm.k[s][kk >> 2]) + (kk & 3) * 32, 16, 1024),
                                               id_qk, part > 0 || kk > 0);
                        }
                        tc::commit(leader, &sm.s_full[s]);
                        tc::commit(leader, &sm.k_empty[s]);
                    }
                    if (t > 0) {
                        const int u = t - 1, us = u & 1;
                        const uint32_t uph = (u >> 1) & 1;
                        // P(u) written, V(u) there, O(u - 1) read out
                        ok = warp_wait(&sm.p_full[us], uph, &sm.abort) &&
                             warp_wait(&sm.v_full[us], uph, &sm.abort) &&
                             (u == 0 || warp_wait(&sm.o_empty, (u - 1) & 1, &sm.abort));
                        if (!ok) break;
                        tc::fence_after_sync();
                        const uint32_t tP = tmem + 128 * us;
#pragma unroll 1
                        for (int part = 0; part < 2; ++part) {
#pragma unroll
                            for (int kk = 0; kk < 8; ++kk)
                                tc::mma_f16_ts(leader, tO, tP + 64 * part + 8 * kk,
                                               tc::smem_desc_sw128(smem_u32(sm.v[us][0]) + kk * 16 * 128, kHalfBytes, 1024),
                                               id_pv, part > 0 || kk > 0);
                        }
                        tc::commit(leader, &sm.pv_done[us]);
                        tc::commit(leader, &sm.v_empty[us]);
                    }
                }
                if (!ok && lane == 0) fail(&sm.abort, p);
                // no tensor-core work may be in flight when TMEM is released
                tc::commit(leader, &sm.mma_done);
                mbar_wait_bounded(&sm.mma_done, 0, nullptr);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ---------------- softmax warps ----------------
        const int qd = warp & 3, ch = warp >> 2;
        const int r = 32 * qd + lane;  // row = TMEM lane
        const int g = r % G, j = r / G, qrow = pos_base + j;
        const bool row_ok = j < ppc && qrow < p.q_len;
        const uint32_t lane_base = (uint32_t)(32 * qd) << 16;
        float qmul;
        {
            const float* src =
                p.q + (((size_t)b * p.q_heads + hk * G + g) * p.q_len + (row_ok ? qrow : 0)) * D + D / 2 * ch;
            float4 x[D / 8];
            float a = 0.f;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                x[c] = row_ok ? *reinterpret_cast<const float4*>(src + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
                a = fmaxf(a, fmaxf(fmaxf(fabsf(x[c].x), fabsf(x[c].y)), fmaxf(fabsf(x[c].z), fabsf(x[c].w))));
            }
            sm.red[0][ch][r] = a;
            named_barrier_sync(3, kSoftmaxThreads);
            a = fmaxf(a, sm.red[0][ch ^ 1][r]);
            // the row's largest magnitude to [2^4, 2^5)
            int e = a > 0.f ? 4 + 127 - (int)(__float_as_uint(a) >> 23) : 0;
            e = max(-126, min(126, e));
            const float up = __uint_as_float((uint32_t)(e + 127) << 23);
            qmul = p.qscale * __uint_as_float((uint32_t)(127 - e) << 23);
            uint32_t hi[D / 4], lo[D / 4];
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                split_half_rn(x[c].x * up, x[c].y * up, hi[2 * c], lo[2 * c]);
                split_half_rn(x[c].z * up, x[c].w * up, hi[2 * c + 1], lo[2 * c + 1]);
            }
            if constexpr (D == 128) {
                tc::st_32x32b_x32(tmem + lane_base + kColQ + 32 * ch, hi);
                tc::st_32x32b_x32(tmem + lane_base + kColQlo + 32 * ch, lo);
            } else {
                tc::st_32x32b_x16(tmem + lane_base + kColQ + 16 * ch, hi);
                tc::st_32x32b_x16(tmem + lane_base + kColQlo + 16 * ch, lo);
            }
            tc::wait_st();
        }
        tc::fence_before_sync();
        named_barrier_sync(1, kSoftmaxThreads + 32);

        const int qpos = p.q_pos0 + qrow;
        const uint32_t tO = tmem + kColO + lane_base + D / 2 * ch;
        float2 acc[D / 4];  // O of the row's channel half ch
#pragma unroll
        for (int i = 0; i < D / 4; ++i) acc[i] = make_float2(0.f, 0.f);
        float m = -CUDART_INF_F, l = 0.f, w_prev = 0.f;
        bool failed = false;
        // acc += w O(t): P V of tile t out of TMEM, 32 columns at a time
        auto drain = [&](int t, float w) {
            if (!warp_wait(&sm.pv_done[t & 1], (t >> 1) & 1, &sm.abort)) return false;
            tc::fence_after_sync();
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                uint32_t o[32];
                tc::ld_32x32b_x32_sync(tO + 32 * c, o);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    acc[16 * c + i] = fma2(make_float2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])),
                                           make_float2(w, w), acc[16 * c + i]);
            }
            tc::fence_before_sync();
            mbar_arrive(&sm.o_empty);
            return true;
        };
        for (int t = 0; t < nt; ++t) {
            const int s = t & 1;
            if (!warp_wait(&sm.info_full[t % kInfo], (t / kInfo) & 1, &sm.abort)) { failed = true; break; }
            const Info& inf = sm.info[t % kInfo];
            const int pos = inf.pos[ch], len = inf.len[ch];
            // the larger scale of the halves that some row of the CTA sees
            const float u = fmaxf(inf.pos[0] <= qlast ? inf.sv[0] : kTiny, inf.pos[1] <= qlast ? inf.sv[1] : kTiny);
            // p comes out of the exponential times f = 2^7 s_v / u; the row sum takes f off again once per tile. Both
            // factors stay normal numbers: a product below them is lost beside the other half (f) or a logit of 0 (c).
            const float f = fminf(fmaxf(inf.sv[ch] / u, kMinF), 1.f) * kPScale, c = fmaxf(qmul * inf.sk[ch], kTiny);
            const float lf = log2f(f);
            if (!warp_wait(&sm.s_full[s], (t >> 1) & 1, &sm.abort)) { failed = true; break; }
            tc::fence_after_sync();
            const uint32_t tS = tmem + 128 * s + lane_base;
            uint32_t sr[64];
            tc::ld_32x32b_x64_sync(tS + 64 * ch, sr);
            const int lim = min(len, qpos - pos + 1);  // keys of this half that the row sees
            float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
            if (__all_sync(0xffffffffu, lim >= 64)) {
#pragma unroll
                for (int i = 0; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(sr[i]));
            } else {
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    const float x = i < lim ? __uint_as_float(sr[i]) : -CUDART_INF_F;
                    sr[i] = __float_as_uint(x);
                    mx[i & 3] = fmaxf(mx[i & 3], x);
                }
            }
            float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;  // c > 0
            sm.red[s][ch][r] = tmax;
            mbar_arrive(&sm.pair[qd][s]);
            if (!warp_wait(&sm.pair[qd][s], (t >> 1) & 1, &sm.abort)) { failed = true; break; }
            tmax = fmaxf(tmax, sm.red[s][ch ^ 1][r]);
            // the reference maximum moves when it is exceeded by more than 2^8; both warps of a row decide alike
            const float mn = fmaxf(m, tmax);
            float alpha = 1.f;
            if (mn > m + kLazy) {
                alpha = m == -CUDART_INF_F ? 0.f : tc::ex2(m - mn);
                m = mn;
            }
            const float ms = m == -CUDART_INF_F ? 0.f : m;
            const float2 c2 = make_float2(c, c), b2 = make_float2(lf - ms, lf - ms);
            float2 rs[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            uint32_t hi[32], lo[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                const float2 x =
                    fma2(make_float2(__uint_as_float(sr[2 * e]), __uint_as_float(sr[2 * e + 1])), c2, b2);
                const float2 pp = make_float2(tc::ex2(x.x), tc::ex2(x.y));
                rs[e & 1] = add2(rs[e & 1], pp);
                split_half(pp, hi[e], lo[e]);
            }
            tc::st_32x32b_x32(tS + 32 * ch, hi);
            tc::st_32x32b_x32(tS + 64 + 32 * ch, lo);
            const float2 sum = add2(rs[0], rs[1]);
            l = l * alpha + (sum.x + sum.y) * (1.f / f);
            tc::wait_st();
            tc::fence_before_sync();
            mbar_arrive(&sm.p_full[s]);
            // O(t - 1) was made with the previous reference maximum: added before the rescale
            if (t > 0 && !drain(t - 1, w_prev)) { failed = true; break; }
            w_prev = u * (1.f / kPScale);
            if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
                for (int i = 0; i < D / 4; ++i) acc[i] = make_float2(acc[i].x * alpha, acc[i].y * alpha);
            }
        }
        if (!failed && nt > 0 && !drain(nt - 1, w_prev)) failed = true;
        if (failed) fail(&sm.abort, p);
        // row sum over both key halves (every maximum posted in red[0] has been read:
        // the partner read it before it published the P of a product that is done)
        bool ok = !failed;
        if (ok) {
            sm.red[0][ch][r] = l;
            mbar_arrive(&sm.pair_l[qd]);
            ok = warp_wait(&sm.pair_l[qd], 0, &sm.abort);
        }
        ok = ok && __all_sync(0xffffffffu, *(volatile int*)&sm.abort == 0);
        const float lt = ok ? l + sm.red[0][ch ^ 1][r] : 0.f;
        const bool any = lt > 0.f || lt != lt;
        const float inv = any ? 1.f / lt : 0.f;
        const float lse = any ? (m + log2f(lt)) * 0.69314718055994531f : -CUDART_INF_F;
        // the call's output, or this split's normalised output and log-sum-exp for chunk_merge_kernel
        const bool whole = p.nsplit == 1;
        const size_t orow = whole ? ((size_t)b * p.q_heads + hk * G + g) * p.q_len + qrow : (size_t)blockIdx.x * BM + r;
        float* dst = (whole ? p.out : p.ws.o) + (!whole || row_ok ? orow : 0) * D + D / 2 * ch;
        float* dst_lse = whole ? p.lse : p.ws.m;
        if (!whole || row_ok) {
#pragma unroll
            for (int i = 0; i < D / 4; i += 2)
                *reinterpret_cast<float4*>(dst + 2 * i) =
                    make_float4(acc[i].x * inv, acc[i].y * inv, acc[i + 1].x * inv, acc[i + 1].y * inv);
            if (ch == 0 && dst_lse != nullptr) dst_lse[orow] = lse;
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == kMmaWarp) {
        __syncwarp();
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
}

// out = sum_s e^(lse_s - M) O_s / sum_s e^(lse_s - M) over the splits of a unit's
// keys: one warp per query row, a lane holding 4 channels. Bound by the
// partials' bytes (64 KB per part, from L2).
template <int D>
__global__ void __launch_bounds__(256) chunk_merge_kernel(const Params p) {
    griddep_wait();
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int unit = row / BM, r = row % BM;
    if (unit >= p.units) return;
    const int nqb = p.units / p.groups, ppc = BM / p.G;
    const int qb = nqb - 1 - unit / p.groups, bh = unit % p.groups;
    const int g = r % p.G, j = r / p.G, qrow = qb * ppc + j;
    if (j >= ppc || qrow >= p.q_len) return;
    const size_t base = (size_t)unit * p.nsplit * BM + r;
    static_assert(kMaxSplit == 32, "a lane per split");
    const float ls = lane < p.nsplit ? __ldcg(p.ws.m + base + (size_t)lane * BM) : -CUDART_INF_F;
    float M = ls;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    const float wl = ls == -CUDART_INF_F ? 0.f : expf(ls - M);
    float L = wl;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const int c = lane % (D / 4);  // with head_dim 64 the upper half of the lanes repeats the lower one
    const float4* src = reinterpret_cast<const float4*>(p.ws.o + base * D) + c;
#pragma unroll 8
    for (int s = 0; s < p.nsplit; ++s) {
        const float4 o = __ldcg(src + (size_t)s * BM * (D / 4));
        const float wt = __shfl_sync(0xffffffffu, wl, s);
        acc.x += wt * o.x;
        acc.y += wt * o.y;
        acc.z += wt * o.z;
        acc.w += wt * o.w;
    }
    const bool some = L > 0.f || L != L;
    const float inv = some ? 1.f / L : 0.f;
    const size_t orow = ((size_t)(bh / p.kv_heads) * p.q_heads + (bh % p.kv_heads) * p.G + g) * p.q_len + qrow;
    if (lane < D / 4)
        reinterpret_cast<float4*>(p.out + orow * D)[c] = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    if (lane == 0 && p.lse != nullptr) p.lse[orow] = some ? M + logf(L) : -CUDART_INF_F;
}

// The live ring tokens as float16 tiles of 64 with a power-of-two scale s each
// (largest magnitude / s in [2^14, 2^15)), zero rows behind the last token.
// One CTA per (tile, KV head, K or V).
template <typename T, int D>
__global__ void __launch_bounds__(256) hot_half_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                       __half* __restrict__ kh, __half* __restrict__ vh,
                                                       float* __restrict__ scales, int rows, int ring_row0,
                                                       int capacity, int head, int hlen, int hot_rows) {
    const int tile = blockIdx.x, bh = blockIdx.y, is_v = blockIdx.z;
    constexpr int kPerRow = D / 8, kRows = 256 / kPerRow, kIters = kTile / kRows;
    const int c8 = threadIdx.x % kPerRow, r0 = threadIdx.x / kPerRow;
    const T* src = (is_v ? v : k) + (size_t)bh * rows * D + 8 * c8;
    float x[kIters][8];
    float a = 0.f;
    bool number = true;
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
        const int t = tile * kTile + r0 + kRows * i;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (t < hlen) w = *reinterpret_cast<const uint4*>(src + (size_t)(ring_row0 + (head + t) % capacity) * D);
        const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[i][j] = to_f32<T>(e[j]);
            const float y = fabsf(x[i][j]);
            a = fmaxf(a, y < CUDART_INF_F ? y : 0.f);
            number &= y < CUDART_INF_F;
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, off));
    __shared__ float part[8];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
    number = __syncthreads_and(number);
    a = part[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) a = fmaxf(a, part[i]);
    // a tile of zeros leaves the unit of V to the tile beside it
    const int e = a > 0.f ? max((int)(__float_as_uint(a) >> 23) - 127 - 14, -126) : (number ? -126 : 0);
    const float s = __uint_as_float((uint32_t)(e + 127) << 23), inv = 1.f / s;
    __half* dst = (is_v ? vh : kh) + ((size_t)bh * hot_rows + tile * kTile) * D + 8 * c8;
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack2<__half>(x[i][2 * j] * inv, x[i][2 * j + 1] * inv);
        *reinterpret_cast<uint4*>(dst + (size_t)(r0 + kRows * i) * D) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (threadIdx.x == 0) scales[2 * ((size_t)bh * (hot_rows / kTile) + tile) + is_v] = s;
}

// Splits of each unit's keys: the count (of at most kMaxParts parts per SM)
// with the shortest run of waves, a part costing its share of the tiles plus
// about four tiles' time of set-up, partial output and merge.
constexpr int kMaxParts = 4;
constexpr double kPartTiles = 4.0;

int choose_split(int units, double tiles, int sms, int max_splits) {
    int best = 1;
    double best_t = 1e300;
    for (int s = 1; s <= kMaxSplit; ++s) {
        if (max_splits > 0 && s > max_splits) break;
        if (s > 1 && ((long long)units * s > (long long)kMaxParts * sms || tiles / s < 4.0)) break;
        const double waves = (double)((units * (long long)s + sms - 1) / sms);
        const double t = waves * (tiles / s + kPartTiles * (s > 1 ? 2.0 : 1.0));
        if (t < 0.97 * best_t) {
            best_t = t;
            best = s;
        }
    }
    return best;
}

size_t hot_offset(int sms, int head_dim) {
    return align_up(ws_layout(1, 1, kMaxParts * sms, BM, head_dim).total, 1024);
}
int hot_rows_for(int tokens) { return (tokens + BN - 1) / BN * BN; }
size_t hot_bytes(int groups, int tokens, int head_dim) {
    const size_t rows = (size_t)groups * hot_rows_for(tokens);
    return 2 * rows * head_dim * 2 + rows / kTile * sizeof(float2);
}

template <typename T, int D>
void launch_hot_half(const rfsn_arena* arena, const archive::Params& a, int groups, int hot_rows, __half* kh, __half* vh,
                     float* scales, cudaStream_t s) {
    hot_half_kernel<T, D><<<dim3(hot_rows / kTile, groups, 2), 256, 0, s>>>(
        static_cast<const T*>(arena->k), static_cast<const T*>(arena->v), kh, vh, scales, a.rows, a.ring_row0, a.capacity,
        a.head, a.hlen, hot_rows);
}

template <int D>
rfsn_status launch(const rfsn_arena* arena, const rfsn_packed_archive* packed, const archive::Params& a,
                                 int batch, void* workspace, size_t workspace_bytes, int max_splits, cudaStream_t s) {
    const int groups = batch * a.kv_heads;
    const int sms = std::max(device_sms(), 148);
    const size_t off = hot_offset(sms, D), need = off + hot_bytes(groups, a.hlen, D);
    if (workspace_bytes < need) {
        set_error("rfsn_archive_attention: workspace too small: need %zu bytes, have %zu", need, workspace_bytes);
        return RFSN_ERR_OVERFLOW;
    }
    Params p;
    memset(&p, 0, sizeof(p));
    p.q = a.q;
    p.out = a.out;
    p.lse = a.lse;
    p.tiles = a.tiles;
    p.n_tiles = a.n_tiles;
    p.packed_rows = a.packed_rows;
    p.scales = a.scales;
    p.hot_rows = std::max(hot_rows_for(a.hlen), BN);
    p.hlen = a.hlen;
    p.hstart = a.hstart;
    p.q_heads = a.q_heads;
    p.kv_heads = a.kv_heads;
    p.q_len = a.q_len;
    p.q_pos0 = a.q_pos0;
    p.G = a.G;
    p.groups = groups;
    p.qscale = a.qscale;
    const int ppc = BM / a.G, nqb = (a.q_len + ppc - 1) / ppc;
    p.units = nqb * groups;
    p.nsplit = choose_split(p.units, (a.n_tiles + 1) / 2 + p.hot_rows / (double)BN, device_sms(), max_splits);
    // partials of all parts: outputs [parts][128][128] and log-sum-exps [parts][128] (in the layout's m)
    p.ws = ws_view(workspace, ws_layout(1, 1, p.nsplit > 1 ? p.units * p.nsplit : 1, BM, D));
    static std::atomic<bool> ready[64];
    const int dev = arena->device;
    if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
        // setmaxnreg moves registers between the warpgroups of what the block was launched with
        cudaFuncAttributes attr;
        RFSN_CUDA(cudaFuncGetAttributes(&attr, chunk_kernel<D>));
        if (attr.numRegs * kThreads < 256 * (kSoftmaxRegs + kOtherRegs)) {
            set_error("rfsn_archive_attention: built with %d registers per thread, the chunk kernel needs %d",
                      attr.numRegs, 256 * (kSoftmaxRegs + kOtherRegs) / kThreads);
            return RFSN_ERR_UNSUPPORTED;
        }
        RFSN_CUDA(cudaFuncSetAttribute(chunk_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem<D>)));
        // the small kernels around it with the same split of the SM's memory, or each change of split drains the SMs
        for (const void* f : {reinterpret_cast<const void*>(hot_half_kernel<__half, D>),
                              reinterpret_cast<const void*>(hot_half_kernel<__nv_bfloat16, D>),
                              reinterpret_cast<const void*>(chunk_merge_kernel<D>)})
            RFSN_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributePreferredSharedMemoryCarveout,
                                           cudaSharedmemCarveoutMaxShared));
        if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_relaxed);
    }
    char* hot = static_cast<char*>(workspace) + off;
    const size_t rows = (size_t)groups * p.hot_rows;
    CUtensorMap mk, mv;
    if (a.hlen > 0) {
        __half* kh = reinterpret_cast<__half*>(hot);
        __half* vh = kh + rows * D;
        float* hs = reinterpret_cast<float*>(vh + rows * D);
        p.hot_scales = reinterpret_cast<const float2*>(hs);
        if (arena->dtype == RFSN_BF16)
            launch_hot_half<__nv_bfloat16, D>(arena, a, groups, p.hot_rows, kh, vh, hs, s);
        else
            launch_hot_half<__half, D>(arena, a, groups, p.hot_rows, kh, vh, hs, s);
        RFSN_CUDA(cudaGetLastError());
        note_launch();
        rfsn_status st = encode_rows_map(&mk, kh, RFSN_F16, groups, p.hot_rows, D, kTile);
        if (st == RFSN_OK) st = encode_rows_map(&mv, vh, RFSN_F16, groups, p.hot_rows, D, kTile);
        if (st != RFSN_OK) return st;
    } else {
        mk = arena->item_maps[0];  // not used
        mv = arena->item_maps[1];
    }
    RFSN_CUDA(launch_pdl(chunk_kernel<D>, dim3(p.units * p.nsplit), dim3(kThreads), sizeof(Smem<D>), s,
                         packed->maps[0], packed->maps[1], mk, mv, p));
    note_launch();
    if (p.nsplit > 1) {
        RFSN_CUDA(launch_pdl(chunk_merge_kernel<D>, dim3(p.units * (BM / 8)), dim3(256), 0, s, p));
        note_launch();
    }
    return RFSN_OK;
}

template <int D>
void preload() {
    cudaFuncAttributes a;
    cudaFuncGetAttributes(&a, chunk_kernel<D>);
    cudaFuncGetAttributes(&a, chunk_merge_kernel<D>);
    cudaFuncGetAttributes(&a, hot_half_kernel<__half, D>);
    cudaFuncGetAttributes(&a, hot_half_kernel<__nv_bfloat16, D>);
}

}  // namespace chunk
}  // namespace archive

size_t archive_chunk_ws(int groups, int hot_capacity, int head_dim) {
    using namespace archive::chunk;
    return hot_offset(std::max(device_sms(), 148), head_dim) + hot_bytes(groups, hot_capacity, head_dim);
}

bool archive_chunk_fits(int G) { return G <= archive::chunk::BM; }

rfsn_status archive_chunk_launch(const rfsn_arena* arena, const rfsn_packed_archive* packed, const archive::Params& a,
                                 int batch, void* workspace, size_t workspace_bytes, int max_splits, cudaStream_t s) {
    using namespace archive::chunk;
    return arena->head_dim == 128 ? launch<128>(arena, packed, a, batch, workspace, workspace_bytes, max_splits, s)
                                  : launch<64>(arena, packed, a, batch, workspace, workspace_bytes, max_splits, s);
}

void preload_chunk_kernels() {
    archive::chunk::preload<128>();
    archive::chunk::preload<64>();
}

}  // namespace rfsn
