// C entry points of the packed archive, tile selection and the attention over
// tile lists (include/rfsn_b200.h): argument checks and launch plans.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>

#include "archive.cuh"

using namespace rfsn;

namespace {

constexpr int kMaxLists = 65535;  // grid dimension y

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

rfsn_status check_device(int device, const char* what) {
    int dev = 0;
    RFSN_CUDA(cudaGetDevice(&dev));
    RFSN_CHECK_ARG(dev == device, "%s: called with device %d current, the buffers are on device %d", what, dev, device);
    return RFSN_OK;
}

// Query slots of one list, slots per CTA, CTAs (z) per list, and the kernel: rows (archive_rows.cu) or tiles
// (archive_attn.cu, 4 or 8 slots per CTA).
struct SlotPlan {
    int lists, slots, per_cta, zblocks;
    bool rows;
};

SlotPlan make_plan(int batch, int q_heads, int kv_heads, int q_len, bool per_query, int per_cta, bool rows) {
    SlotPlan s;
    const int G = q_heads / kv_heads;
    s.lists = batch * kv_heads * (per_query ? q_len : 1);
    s.slots = per_query ? G : G * q_len;
    s.per_cta = per_cta;
    s.zblocks = (s.slots + per_cta - 1) / per_cta;
    s.rows = rows;
    return s;
}

int ctas_per_sm(const SlotPlan& sp) { return sp.rows ? 1 : archive_attn_ctas(sp.per_cta / 4); }

// Splits of a list's items: the CTAs that are resident at once, over all lists.
int split_limit(const SlotPlan& sp, int head_dim, int max_splits) {
    const int sms = std::max(device_sms(), 1);
    int s = std::max(1, ctas_per_sm(sp) * sms / std::max(1, sp.lists * sp.zblocks));
    s = std::min(s, head_dim == 128 ? archive::kMaxSplits128 : archive::kMaxSplits64);
    if (max_splits > 0) s = std::min(s, max_splits);
    return s;
}

// The rows kernel runs from 5 slots on (8 slots, 8 heads: 33K keys 20 us, the tile kernel 23; 131K 53 / 59). It takes 8
// or 16 slots a CTA: 16 halve the passes over K/V, but their merge reads twice the partials. Measured (us, 8 / 16
// slots): 16 slots, 8 heads (18 splits of 16): 4K keys 10.7 / 13.3, 16K 18.5 / 17.8, 33K 29 / 25, 131K 88 / 61;
// 32 slots: 4K 13.8 / 13.9, 16K 31 / 24; 1 head (74 splits): 33K 14 / 23. units: a split's work, below.
SlotPlan slot_plan(int batch, int q_heads, int kv_heads, int q_len, int head_dim, bool packed, bool per_query,
                   long long units) {
    const int slots = q_heads / kv_heads * (per_query ? 1 : q_len);
    auto plan = [&](int per_cta, bool rows) {
        return make_plan(batch, q_heads, kv_heads, q_len, per_query, per_cta, rows);
    };
    if (slots <= 4) return plan(4, false);
    if (!packed || per_query || head_dim != 128) return plan(8, false);
    const SlotPlan wide = plan(16, true);
    const long long splits = std::min<long long>(split_limit(wide, head_dim, 0), std::max(units, 1LL));
    return slots > 8 && units > splits * (2 + splits / 4) ? wide : plan(8, true);
}

WsLayout attention_ws(const SlotPlan& sp, int splits, int head_dim) {
    return ws_layout(splits > 1 ? sp.lists * sp.zblocks : 0, 1, splits, sp.per_cta, head_dim);
}

// Largest attention workspace of a shape: every split count it may choose (at
// least 148 SMs are assumed, so a size computed without a device serves a B200).
size_t attention_ws_limit(const SlotPlan& sp, int head_dim) {
    const int units = std::max(1, sp.lists * sp.zblocks);
    const int limit = std::max(split_limit(sp, head_dim, 0),
                               std::min(head_dim == 128 ? archive::kMaxSplits128 : archive::kMaxSplits64,
                                        std::max(1, ctas_per_sm(sp) * 148 / units)));
    return attention_ws(sp, limit, head_dim).total;
}

// Packed archives: the rows kernel (head_dim 128) reads K/V again for every 16
// query slots, the tile kernel (head_dim 64) for every 8, the chunk kernel for
// every 128, at about 2.1 (1.95) times the cost of a pass, and 9 us more to
// begin with. Measured (8 KV heads, us, rows / chunk kernel): 32 slots over 16K
// keys 24 / 35, 131K 107 / 125; 48 slots over 16K 30 / 35, 33K 49 / 52, 131K 155 /
// 126; 64 slots over 4K 18 / 22, 16K 39 / 36, 33K 69 / 53; 1 KV head: 96 slots over
// 33K 22 / 35. head_dim 64 (tile / chunk kernel): 24 slots over 16K 23 / 26, 33K 41 /
// 39; 64 over 4K 19 / 18, 16K 57 / 27; 1,024 over 16K 743 / 116; 1 KV head: 128 over
// 16K 17 / 23, 256 31 / 23.
// With fewer than 5 units of 128 slots (times 32 key ranges) it leaves SMs idle and a unit's pass costs as much as 5's.
bool chunk_shape(int head_dim, int groups, int G, int q_len, int n_tiles) {
    const long long slots = q_len * (long long)G, units = std::max(5LL, (slots + 127) / 128 * groups);
    const long long saved = head_dim == 128 ? 20 * ((slots + 15) / 16) * groups - 42 * units   // 20 * passes of a head
                                            : 20 * ((slots + 7) / 8) * groups - 39 * units;
    return archive_chunk_fits(G) && saved * n_tiles > 76000;  // * 64-token tiles
}

size_t select_scores_offset();

// Selected lists of rfsn_archive_attend: behind everything its two kernels write.
size_t lists_offset(const SlotPlan& sp, int head_dim, int n_tiles) {
    return align_up(std::max(attention_ws_limit(sp, head_dim),
                             select_scores_offset() + sizeof(float) * (size_t)sp.lists * n_tiles), 256);
}

size_t select_scores_offset() { return align_up(256 + sizeof(int) * (size_t)kMaxCounters, 256); }

rfsn_status check_shape(int batch, int q_heads, int kv_heads, int q_len, int head_dim, bool per_query,
                        const char* what) {
    RFSN_CHECK_ARG(batch > 0 && q_heads > 0 && kv_heads > 0 && q_len > 0, "%s: non-positive shape", what);
    RFSN_CHECK_ARG(q_heads % kv_heads == 0, "num_heads (%d) must be divisible by num_kv_heads (%d)", q_heads, kv_heads);
    if (head_dim != 64 && head_dim != 128) {
        set_error("%s: head_dim %d is not supported (64 or 128)", what, head_dim);
        return RFSN_ERR_UNSUPPORTED;
    }
    RFSN_CHECK_ARG((long long)batch * kv_heads * (per_query ? q_len : 1) <= kMaxLists, "%s: more than %d tile lists", what,
                   kMaxLists);
    RFSN_CHECK_ARG((long long)batch * q_heads * q_len < (1LL << 30), "%s: too many query rows", what);
    return RFSN_OK;
}

rfsn_status check_tiles(const rfsn_tile_list* t, const char* what) {
    RFSN_CHECK_ARG(t != nullptr && t->n >= 0 && t->n <= (1 << 25) && (t->n == 0 || t->tiles != nullptr) &&
                       aligned16(t->tiles) && (t->per_query == 0 || t->per_query == 1),
                   "%s: bad tile list", what);
    return RFSN_OK;
}

// check_only: every argument check of the call, without a launch
rfsn_status attention(const rfsn_arena* arena, const rfsn_packed_archive* packed, const float* q, int batch, int q_heads,
                      int kv_heads, int q_len, int q_pos0, const rfsn_tile_list* tiles, const rfsn_hot_window* hot,
                      float* out, float* lse, void* workspace, size_t workspace_bytes, int max_splits, void* stream,
                      bool check_only) {
    const char* what = "rfsn_archive_attention";
    RFSN_CHECK_ARG(arena != nullptr && hot != nullptr, "%s: NULL arena or hot window", what);
    rfsn_status st = check_tiles(tiles, what);
    if (st == RFSN_OK)
        st = check_shape(batch, q_heads, kv_heads, q_len, arena->head_dim, tiles->per_query != 0, what);
    if (st != RFSN_OK) return st;
    if (!arena->has_items) {
        set_error("%s: needs a bf16/f16 arena with head_dim 64 or 128", what);
        return RFSN_ERR_UNSUPPORTED;
    }
    const int groups = batch * kv_heads;
    RFSN_CHECK_ARG(groups == arena->groups, "%s: batch*kv_heads %d != arena groups %d", what, groups, arena->groups);
    RFSN_CHECK_ARG(packed == nullptr || (packed->groups == groups && packed->head_dim == arena->head_dim &&
                                         packed->device == arena->device),
                   "%s: the packed archive's heads, head_dim or device differ from the arena's", what);
    RFSN_CHECK_ARG(q != nullptr && aligned16(q) && out != nullptr && aligned16(out) && workspace != nullptr &&
                       aligned16(workspace), "%s: NULL or misaligned pointer (q, out and workspace: 16 bytes)", what);
    RFSN_CHECK_ARG(hot->length >= 0 && hot->length <= hot->capacity && hot->head_index >= 0 &&
                       hot->head_index < (hot->capacity > 0 ? hot->capacity : 1) && hot->ring_row0 >= 0 &&
                       hot->ring_row0 <= arena->rows && hot->capacity <= arena->rows - hot->ring_row0,
                   "%s: bad hot window", what);
    const bool stepped = hot->step_state != nullptr;
    if (tiles->n == 0 && hot->length == 0 && !stepped) {
        set_error("run_segmented_attention requires at least one KV segment");
        return RFSN_ERR_INVALID_ARG;
    }
    st = check_device(arena->device, what);
    if (st != RFSN_OK) return st;
    const bool chunk = packed != nullptr && tiles->per_query == 0 && !stepped && tiles->n > 0 &&
                       chunk_shape(arena->head_dim, groups, q_heads / kv_heads, q_len, tiles->n);
    const int first = std::min(hot->length, hot->capacity - hot->head_index);
    // with a device step state the window is only known when the kernel runs: planned for the largest
    auto hot_of = [&](int keys) {  // items of that many ring keys
        return stepped ? (hot->capacity + keys - 1) / keys + 1
                       : (first + keys - 1) / keys + (hot->length - first + keys - 1) / keys;
    };
    // rows kernel: an item of two tiles is one unit, one of 128 ring keys (twice the bytes) two
    const SlotPlan sp = slot_plan(batch, q_heads, kv_heads, q_len, arena->head_dim, packed != nullptr,
                                  tiles->per_query != 0, (tiles->n + 1) / 2 + 2LL * hot_of(128));
    RFSN_CHECK_ARG(chunk || sp.zblocks <= kMaxLists, "%s: too many query rows", what);
    const int hk = sp.rows ? 128 : (arena->head_dim == 128 ? 32 : 64);
    const int per_tile = packed != nullptr ? 1 : kTile / hk;
    RFSN_CHECK_ARG((long long)tiles->n * per_tile < (1LL << 30), "%s: too many tiles", what);
    const int hot_items = hot_of(hk);
    const int total = std::max(1, sp.rows ? (tiles->n + 1) / 2 + 2 * hot_items : tiles->n * per_tile + hot_items);
    int splits = std::min(split_limit(sp, arena->head_dim, max_splits), total);
    // The last CTA reads every split's partials: with few lists, more splits than about sqrt(c items / slots) cost more
    // there than they save. Measured (1 KV head, 4 slots, 49K keys, us): 32 splits 18.5, 64 14.0, 96 13.3, 240 17.1;
    // 5K keys: 16 8.0, 48 7.5, 80 9.3; two heads of 8 slots, 43 tiles: 8 20.1, 24 19.0, 43 20.6.
    splits = std::min(splits, std::max(1, (int)std::sqrt((sp.rows ? 72.0 : 50.0) * total / sp.per_cta)));
    const int per = (total + splits - 1) / splits;
    splits = (total + per - 1) / per;
    // more than one split only where all lists leave SMs idle: far fewer lists than arrival counters
    RFSN_CHECK_ARG(splits == 1 || (long long)sp.lists * sp.zblocks <= kMaxCounters, "%s: too many lists", what);
    const WsLayout w = attention_ws(sp, splits, arena->head_dim);
    if (!chunk && w.total > workspace_bytes) {
        set_error("%s: workspace too small: need %zu bytes, have %zu", what, w.total, workspace_bytes);
        return RFSN_ERR_OVERFLOW;
    }
    if (check_only) return RFSN_OK;
    archive::Params p;
    memset(&p, 0, sizeof(p));
    p.q = q;
    p.out = out;
    p.lse = lse;
    p.tiles = reinterpret_cast<const int4*>(tiles->tiles);
    p.n_tiles = tiles->n;
    p.per_query = tiles->per_query;
    p.ring_row0 = hot->ring_row0;
    p.capacity = hot->capacity;
    p.head = hot->head_index;
    p.hlen = hot->length;
    p.hstart = hot->start_pos;
    p.rows = arena->rows;
    p.packed_rows = packed != nullptr ? packed->rows : 0;
    p.scales = packed != nullptr ? packed->scales : nullptr;
    p.q_heads = q_heads;
    p.kv_heads = kv_heads;
    p.q_len = q_len;
    p.q_pos0 = q_pos0;
    p.G = q_heads / kv_heads;
    p.slots = sp.slots;
    p.items_per_split = per;
    p.splits = splits;
    p.hot_items = hot_items;
    p.qscale = (float)(1.0 / std::sqrt((double)arena->head_dim)) * 1.4426950408889634f;
    p.ws = ws_view(workspace, w);
    p.dyn = hot->step_state;
    // the chunk kernel reads no archived row ahead of the kernel before it, the others do
    p.overlap = chunk || (packed != nullptr ? packed->fresh : arena->fresh).overlap(static_cast<cudaStream_t>(stream));
    if (chunk)
        return archive_chunk_launch(arena, packed, p, batch, workspace, workspace_bytes, max_splits,
                                    static_cast<cudaStream_t>(stream));
    if (sp.rows)
        return archive_rows_launch(arena, packed, p, sp.lists, sp.per_cta, sp.zblocks, static_cast<cudaStream_t>(stream));
    return archive_attn_launch(arena, packed, p, sp.lists, sp.per_cta / 4, sp.zblocks, static_cast<cudaStream_t>(stream));
}

// numbers: out receives the tiles' numbers ([lists][n_select]) instead of their entries; fresh: of the owner of the
// bounds and scales, unless it is not known (then nothing is read ahead of the kernel before)
rfsn_status select(const char* what, const void* bounds, int bounds_dtype, const float* scales, int rows, const float* q,
                   int batch, int q_heads, int kv_heads, int q_len, int head_dim, int q_pos0,
                   const rfsn_tile_list* tiles, int n_select, int32_t* out, bool numbers, const int32_t* step_state,
                   void* workspace, size_t workspace_bytes, void* stream, const FreshWrites* fresh) {
    rfsn_status st = check_shape(batch, q_heads, kv_heads, q_len, head_dim, true, what);
    if (st == RFSN_OK) st = check_tiles(tiles, what);
    if (st != RFSN_OK) return st;
    RFSN_CHECK_ARG(tiles->per_query == 0, "%s: selects from one list for all heads and queries", what);
    RFSN_CHECK_ARG(q != nullptr && aligned16(q) && out != nullptr && aligned16(out) && workspace != nullptr &&
                       aligned16(workspace), "%s: NULL or misaligned pointer (q, out and workspace: 16 bytes)", what);
    RFSN_CHECK_ARG(bounds_dtype == RFSN_F16 || bounds_dtype == RFSN_BF16 || bounds_dtype == RFSN_E4M3,
                   "%s: bounds must be f16, bf16 or e4m3", what);
    RFSN_CHECK_ARG(tiles->n == 0 || (bounds != nullptr && aligned16(bounds)), "%s: NULL or misaligned bounds", what);
    RFSN_CHECK_ARG(tiles->n == 0 || bounds_dtype != RFSN_E4M3 || (scales != nullptr && aligned16(scales)),
                   "%s: e4m3 bounds need the archive's scales", what);
    RFSN_CHECK_ARG(rows >= 0 && rows % kTile == 0, "%s: rows (%d) must be a multiple of %d", what, rows, kTile);
    RFSN_CHECK_ARG(n_select > 0 && n_select <= (1 << 20), "%s: n_select %d outside [1, %d]", what, n_select, 1 << 20);
    const int lists = batch * kv_heads * q_len;
    RFSN_CHECK_ARG(lists <= kMaxCounters, "%s: batch * kv_heads * q_len above %d", what, kMaxCounters);
    const size_t off = select_scores_offset(), need = off + sizeof(float) * (size_t)lists * tiles->n;
    if (workspace_bytes < need) {
        set_error("%s: workspace too small: need %zu bytes, have %zu", what, need, workspace_bytes);
        return RFSN_ERR_OVERFLOW;
    }
    char* ws = static_cast<char*>(workspace);
    archive::SelectParams p;
    memset(&p, 0, sizeof(p));
    p.bounds = bounds;
    p.scales = reinterpret_cast<const float4*>(scales);
    p.tile_slots = rows / kTile;
    p.q = q;
    p.q_heads = q_heads;
    p.kv_heads = kv_heads;
    p.q_len = q_len;
    p.q_pos0 = q_pos0;
    p.G = q_heads / kv_heads;
    p.tiles = reinterpret_cast<const int4*>(tiles->tiles);
    p.n_tiles = tiles->n;
    p.n_select = n_select;
    p.out = numbers ? nullptr : reinterpret_cast<int4*>(out);
    p.numbers = numbers ? out : nullptr;
    p.scores = reinterpret_cast<float*>(ws + off);
    p.counters = reinterpret_cast<int*>(ws + 256);
    p.error = reinterpret_cast<int*>(ws);
    p.dyn = step_state;
    p.overlap = fresh != nullptr && fresh->overlap(static_cast<cudaStream_t>(stream));
    // one CTA per SM over all lists, in steps of the tiles that a CTA scores at once (128 over the head groups)
    p.head_groups = p.G <= 4 ? 1 : (p.G <= 8 ? 2 : (p.G <= 16 ? 4 : 8));
    const int want = std::max(1, device_sms() / lists), step = 128 / p.head_groups;
    p.tiles_per_cta = std::max(step, ((tiles->n + want - 1) / want + step - 1) / step * step);
    const int chunks = std::max(1, (tiles->n + p.tiles_per_cta - 1) / p.tiles_per_cta);
    return select_tiles_launch(bounds_dtype, head_dim, p, lists, chunks, static_cast<cudaStream_t>(stream));
}

rfsn_status select_call(const char* what, const rfsn_archive_call* c, const float* q, int q_pos0, int32_t* out,
                        bool numbers, void* workspace, size_t workspace_bytes, void* stream) {
    const rfsn_packed_archive* pk = c->packed;
    return select(what, c->bounds, pk != nullptr ? RFSN_E4M3 : c->arena->dtype,
                  pk != nullptr ? reinterpret_cast<const float*>(pk->scales) : nullptr,
                  pk != nullptr ? pk->rows : c->arena->rows, q, c->batch, c->q_heads, c->kv_heads, c->q_len,
                  c->arena->head_dim, q_pos0, &c->tiles, c->top_tiles, out, numbers, c->hot.step_state, workspace,
                  workspace_bytes, stream, pk != nullptr ? &pk->fresh : &c->arena->fresh);
}

}  // namespace

extern "C" {

rfsn_status rfsn_packed_archive_create(void* k_codes, void* v_codes, float* scales, int batch_kv_heads, int rows,
                                       int head_dim, rfsn_packed_archive** out) {
    RFSN_CHECK_ARG(out != nullptr, "rfsn_packed_archive_create: out is NULL");
    RFSN_CHECK_ARG(k_codes != nullptr && v_codes != nullptr && scales != nullptr,
                   "rfsn_packed_archive_create: NULL pointer");
    RFSN_CHECK_ARG(aligned16(k_codes) && aligned16(v_codes) && aligned16(scales),
                   "rfsn_packed_archive_create: pointers must be 16-byte aligned");
    RFSN_CHECK_ARG(batch_kv_heads > 0 && batch_kv_heads <= kMaxLists && rows > 0 && rows % kTile == 0,
                   "rfsn_packed_archive_create: rows (%d) must be a positive multiple of %d, batch_kv_heads (%d) in "
                   "1..%d", rows, kTile, batch_kv_heads, kMaxLists);
    RFSN_CHECK_ARG((long long)batch_kv_heads * rows < (1LL << 31),
                   "rfsn_packed_archive_create: batch_kv_heads * rows above 2^31 - 1");
    if (head_dim != 64 && head_dim != 128) {
        set_error("rfsn_packed_archive_create: head_dim %d is not supported (64 or 128)", head_dim);
        return RFSN_ERR_UNSUPPORTED;
    }
    rfsn_packed_archive* a = new (std::nothrow) rfsn_packed_archive();
    if (a == nullptr) {
        set_error("rfsn_packed_archive_create: out of host memory");
        return RFSN_ERR_OVERFLOW;
    }
    a->k = static_cast<uint8_t*>(k_codes);
    a->v = static_cast<uint8_t*>(v_codes);
    a->scales = reinterpret_cast<float4*>(scales);
    a->groups = batch_kv_heads;
    a->rows = rows;
    a->head_dim = head_dim;
    a->device = 0;
    cudaGetDevice(&a->device);
    rfsn_status st = encode_rows_map(&a->maps[0], k_codes, RFSN_E4M3, batch_kv_heads, rows, head_dim, kTile);
    if (st == RFSN_OK) st = encode_rows_map(&a->maps[1], v_codes, RFSN_E4M3, batch_kv_heads, rows, head_dim, kTile);
    if (st == RFSN_OK) st = encode_rows_map(&a->maps[2], k_codes, RFSN_E4M3, batch_kv_heads, rows, head_dim, 16);
    if (st == RFSN_OK) st = encode_rows_map(&a->maps[3], v_codes, RFSN_E4M3, batch_kv_heads, rows, head_dim, 16);
    if (st != RFSN_OK) {
        delete a;
        return st;
    }
    *out = a;
    return RFSN_OK;
}

rfsn_status rfsn_packed_archive_destroy(rfsn_packed_archive* archive) {
    delete archive;
    return RFSN_OK;
}

rfsn_status rfsn_pack_rows(const rfsn_packed_archive* a, int dst_row0, const rfsn_kv_rows* src, int count,
                           void* bounds, void* stream) {
    RFSN_CHECK_ARG(a != nullptr && src != nullptr, "rfsn_pack_rows: NULL archive or source");
    RFSN_CHECK_ARG(count >= 0 && dst_row0 >= 0 && dst_row0 % kTile == 0 && dst_row0 <= a->rows &&
                       count <= a->rows - dst_row0,
                   "rfsn_pack_rows: rows [%d, +%d) must start at a multiple of %d inside the archive (%d rows)",
                   dst_row0, count, kTile, a->rows);
    RFSN_CHECK_ARG(src->dtype == RFSN_F32 || src->dtype == RFSN_F16 || src->dtype == RFSN_BF16,
                   "rfsn_pack_rows: unknown dtype %d", src->dtype);
    RFSN_CHECK_ARG(src->kv_heads > 0 && a->groups % src->kv_heads == 0,
                   "rfsn_pack_rows: %d KV heads do not divide the archive's %d", src->kv_heads, a->groups);
    RFSN_CHECK_ARG(src->offset >= 0 && src->wrap >= 0 &&
                       (src->wrap == 0 || (src->offset < src->wrap && count <= src->wrap)),
                   "rfsn_pack_rows: bad offset or wrap");
    RFSN_CHECK_ARG(bounds == nullptr || aligned16(bounds), "rfsn_pack_rows: bounds must be 16-byte aligned");
    if (count == 0) return RFSN_OK;
    RFSN_CHECK_ARG(src->k != nullptr && src->v != nullptr, "rfsn_pack_rows: NULL K or V");
    rfsn_status st = check_device(a->device, "rfsn_pack_rows");
    if (st != RFSN_OK) return st;
    a->fresh.note(static_cast<cudaStream_t>(stream));
    return pack_rows_launch(a, dst_row0, src, count, bounds, static_cast<cudaStream_t>(stream));
}

rfsn_status rfsn_unpack_rows(const rfsn_packed_archive* a, int src_row0, int count, void* k_out, void* v_out,
                             int out_dtype, int64_t out_stride, void* stream) {
    RFSN_CHECK_ARG(a != nullptr, "rfsn_unpack_rows: NULL archive");
    RFSN_CHECK_ARG(count >= 0 && src_row0 >= 0 && src_row0 <= a->rows && count <= a->rows - src_row0,
                   "rfsn_unpack_rows: rows [%d, +%d) outside the archive (%d rows)", src_row0, count, a->rows);
    RFSN_CHECK_ARG(out_dtype == RFSN_F32 || out_dtype == RFSN_F16 || out_dtype == RFSN_BF16,
                   "rfsn_unpack_rows: unknown dtype %d", out_dtype);
    if (count == 0) return RFSN_OK;
    RFSN_CHECK_ARG(k_out != nullptr && v_out != nullptr && aligned16(k_out) && aligned16(v_out) &&
                       out_stride * dtype_size(out_dtype) % 16 == 0 && out_stride >= 0,
                   "rfsn_unpack_rows: outputs and their stride must be 16-byte aligned");
    RFSN_CHECK_ARG(a->groups == 1 || out_stride >= (int64_t)count * a->head_dim,
                   "rfsn_unpack_rows: out_stride %lld overlaps rows of the next head", (long long)out_stride);
    rfsn_status st = check_device(a->device, "rfsn_unpack_rows");
    if (st != RFSN_OK) return st;
    return unpack_rows_launch(a, src_row0, count, k_out, v_out, out_dtype, out_stride, static_cast<cudaStream_t>(stream));
}

rfsn_status rfsn_tile_bounds(const rfsn_arena* arena, int row0, int count, void* bounds, void* stream) {
    RFSN_CHECK_ARG(arena != nullptr && bounds != nullptr && aligned16(bounds), "rfsn_tile_bounds: NULL or misaligned pointer");
    if (!arena->has_items) {
        set_error("rfsn_tile_bounds: needs a bf16/f16 arena with head_dim 64 or 128");
        return RFSN_ERR_UNSUPPORTED;
    }
    RFSN_CHECK_ARG(count >= 0 && row0 >= 0 && row0 % kTile == 0 && row0 <= arena->rows && count <= arena->rows - row0,
                   "rfsn_tile_bounds: rows [%d, +%d) must start at a multiple of %d inside the arena (%d rows)", row0,
                   count, kTile, arena->rows);
    RFSN_CHECK_ARG(arena->rows % kTile == 0, "rfsn_tile_bounds: the arena's rows (%d) must be a multiple of %d",
                   arena->rows, kTile);
    RFSN_CHECK_ARG(arena->groups <= kMaxLists, "rfsn_tile_bounds: more than %d heads", kMaxLists);
    if (count == 0) return RFSN_OK;
    rfsn_status st = check_device(arena->device, "rfsn_tile_bounds");
    if (st != RFSN_OK) return st;
    arena->fresh.note(static_cast<cudaStream_t>(stream));
    return tile_bounds_launch(arena, row0, count, bounds, static_cast<cudaStream_t>(stream));
}

rfsn_status rfsn_archive_workspace_size(int batch, int q_heads, int kv_heads, int q_len, int head_dim,
                                        int hot_capacity, int n_tiles, int n_select, size_t* bytes) {
    RFSN_CHECK_ARG(bytes != nullptr, "rfsn_archive_workspace_size: bytes is NULL");
    rfsn_status st = check_shape(batch, q_heads, kv_heads, q_len, head_dim, n_select > 0, "rfsn_archive_workspace_size");
    if (st != RFSN_OK) return st;
    RFSN_CHECK_ARG(n_tiles >= 0 && n_select >= 0 && hot_capacity >= 0,
                   "rfsn_archive_workspace_size: negative count");
    // every plan that a call over up to that many tiles may take; a selecting call over none attends to a shared list
    const SlotPlan shared = slot_plan(batch, q_heads, kv_heads, q_len, head_dim, false, false, 0);
    size_t need = attention_ws_limit(shared, head_dim);
    if (shared.slots > 4 && head_dim == 128)
        for (int per_cta = 8; per_cta <= 16; per_cta += 8)
            need = std::max(need, attention_ws_limit(make_plan(batch, q_heads, kv_heads, q_len, false, per_cta, true),
                                                     head_dim));
    if (n_select > 0) {
        const SlotPlan sp = slot_plan(batch, q_heads, kv_heads, q_len, head_dim, false, true, 0);
        need = std::max(need, lists_offset(sp, head_dim, n_tiles) + sizeof(int4) * (size_t)sp.lists * n_select);
    } else if (chunk_shape(head_dim, batch * kv_heads, q_heads / kv_heads, q_len, n_tiles))
        need = std::max(need, archive_chunk_ws(batch * kv_heads, hot_capacity, head_dim));
    *bytes = need;
    return RFSN_OK;
}

rfsn_status rfsn_select_tiles(const void* bounds, int bounds_dtype, const float* scales, int rows, const float* q,
                              int batch, int q_heads, int kv_heads, int q_len, int head_dim, int q_pos0,
                              const rfsn_tile_list* tiles, int n_select, int32_t* out, const int32_t* step_state,
                              void* workspace, size_t workspace_bytes, void* stream) {
    return select("rfsn_select_tiles", bounds, bounds_dtype, scales, rows, q, batch, q_heads, kv_heads, q_len, head_dim,
                  q_pos0, tiles, n_select, out, false, step_state, workspace, workspace_bytes, stream, nullptr);
}

rfsn_status rfsn_archive_attention(const rfsn_arena* arena, const rfsn_packed_archive* packed, const float* q,
                                   int batch, int q_heads, int kv_heads, int q_len, int q_pos0,
                                   const rfsn_tile_list* tiles, const rfsn_hot_window* hot, float* out, float* lse,
                                   void* workspace, size_t workspace_bytes, int max_splits, void* stream) {
    return attention(arena, packed, q, batch, q_heads, kv_heads, q_len, q_pos0, tiles, hot, out, lse, workspace,
                     workspace_bytes, max_splits, stream, false);
}

rfsn_status rfsn_archive_attend(const rfsn_archive_call* c, const float* q, int q_pos0, float* out, float* lse,
                                void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "rfsn_archive_attend";
    RFSN_CHECK_ARG(c != nullptr && c->arena != nullptr && c->top_tiles >= 0, "%s: NULL call or negative top_tiles", what);
    if (c->top_tiles == 0 || c->tiles.n == 0)
        return rfsn_archive_attention(c->arena, c->packed, q, c->batch, c->q_heads, c->kv_heads, c->q_len, q_pos0,
                                      &c->tiles, &c->hot, out, lse, workspace, workspace_bytes, c->max_splits, stream);
    const int head_dim = c->arena->head_dim;
    rfsn_status st = check_shape(c->batch, c->q_heads, c->kv_heads, c->q_len, head_dim, true, what);
    if (st != RFSN_OK) return st;
    RFSN_CHECK_ARG(c->tiles.n > 0 && c->tiles.per_query == 0 && c->top_tiles <= (1 << 20), "%s: bad tile list", what);
    const SlotPlan sp = slot_plan(c->batch, c->q_heads, c->kv_heads, c->q_len, head_dim, c->packed != nullptr, true, 0);
    const size_t off = lists_offset(sp, head_dim, c->tiles.n);
    const size_t need = off + sizeof(int4) * (size_t)sp.lists * c->top_tiles;
    if (workspace == nullptr || workspace_bytes < need) {
        set_error("%s: workspace too small: need %zu bytes, have %zu", what, need,
                  workspace == nullptr ? (size_t)0 : workspace_bytes);
        return RFSN_ERR_OVERFLOW;
    }
    rfsn_tile_list chosen;
    chosen.tiles = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + off);
    chosen.n = c->top_tiles;
    chosen.per_query = 1;
    // Everything the attention would refuse is refused before the selection is launched.
    st = attention(c->arena, c->packed, q, c->batch, c->q_heads, c->kv_heads, c->q_len, q_pos0, &chosen, &c->hot, out,
                   lse, workspace, off, c->max_splits, stream, true);
    if (st != RFSN_OK) return st;
    st = select_call(what, c, q, q_pos0, const_cast<int32_t*>(chosen.tiles), false, workspace, off, stream);
    if (st != RFSN_OK) return st;
    return attention(c->arena, c->packed, q, c->batch, c->q_heads, c->kv_heads, c->q_len, q_pos0, &chosen, &c->hot, out,
                     lse, workspace, off, c->max_splits, stream, false);
}

rfsn_status rfsn_archive_select(const rfsn_archive_call* c, const float* q, int q_pos0, int32_t* numbers,
                                void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "rfsn_archive_select";
    RFSN_CHECK_ARG(c != nullptr && c->arena != nullptr, "%s: NULL call", what);
    RFSN_CHECK_ARG(c->batch > 0 && c->kv_heads > 0 && c->batch * c->kv_heads == c->arena->groups &&
                       (c->packed == nullptr || (c->packed->groups == c->arena->groups &&
                                                 c->packed->head_dim == c->arena->head_dim)),
                   "%s: heads or head_dim differ from the arena's", what);
    rfsn_status st = check_device(c->arena->device, what);
    if (st != RFSN_OK) return st;
    return select_call(what, c, q, q_pos0, numbers, true, workspace, workspace_bytes, stream);
}

}  // extern "C"
