// Caches in pages: the C entry points, how an attention launch is laid out, and the join of its splits.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "tq_attn_rows.h"
#include "tq_check.h"
#include "tq_paged_attn.h"

int tqk_paged_attn_k2(const tqpaged::PagedAttnArgs &a, int vb, tqpaged::PagedKind kind, unsigned grid, hipStream_t s);
int tqk_paged_attn_k3(const tqpaged::PagedAttnArgs &a, int vb, tqpaged::PagedKind kind, unsigned grid, hipStream_t s);
int tqk_paged_attn_k4(const tqpaged::PagedAttnArgs &a, int vb, tqpaged::PagedKind kind, unsigned grid, hipStream_t s);
int tqk_paged_attn_k8(const tqpaged::PagedAttnArgs &a, int vb, tqpaged::PagedKind kind, unsigned grid, hipStream_t s);

namespace {

using namespace tqpaged;

constexpr int MERGE_THREADS = 256;

// The splits' partial results of a row -> its output: two dims per lane, a wavefront has HEADS query heads of a row with their reads in
// flight together: it waits for the tables first (4 x 448 rows x 16 heads, two splits: one head each 15.5 us, four 11.8; 80 rows x 64 heads,
// two splits: 4.9, 5.5).
constexpr int MERGE_HEADS = 4;
__global__ __launch_bounds__(MERGE_THREADS) void k_paged_merge(PagedAttnArgs a) {
    const int lane = threadIdx.x & 63, heads = a.r.p.n_kv_heads * a.group, sets = (heads + MERGE_HEADS - 1) / MERGE_HEADS;
    const int64_t at = (int64_t)blockIdx.x * (MERGE_THREADS / 64) + (threadIdx.x >> 6);
    const int64_t row = at / sets;
    const int head0 = (int)(at - row * sets) * MERGE_HEADS;
    if (row >= a.r.rows) return;
    int b, nth;
    PagedSeq seq;
    if (!paged_item(a.r, (int)row, [&](const PagedSeq &q) { return q.n; }, b, nth, seq)) return;
    const PagedSpan span = paged_span(a, seq);
    if (span.splits <= 1 || nth >= a.max_new) return;
    const int64_t out_row = (int64_t)(seq.row0 + nth) * heads;
    int64_t place[MERGE_HEADS];
    float top[MERGE_HEADS];
#pragma unroll
    for (int h = 0; h < MERGE_HEADS; ++h) {   // heads past the last one repeat it
        place[h] = (out_row + min(head0 + h, heads - 1)) * a.n_splits;
        top[h] = -INFINITY;
    }
    for (int s = lane; s < span.splits; s += 64)
#pragma unroll
        for (int h = 0; h < MERGE_HEADS; ++h) top[h] = fmaxf(top[h], a.part_ml[2 * (place[h] + s)]);
#pragma unroll
    for (int h = 0; h < MERGE_HEADS; ++h) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top[h] = fmaxf(top[h], __shfl_xor(top[h], o));
        top[h] = top[h] == -INFINITY ? 0.0f : top[h];
    }
    float l[MERGE_HEADS] = {}, o0[MERGE_HEADS] = {}, o1[MERGE_HEADS] = {};
#pragma unroll 2
    for (int s = 0; s < span.splits; ++s) {
        float2 ml[MERGE_HEADS], v[MERGE_HEADS];
#pragma unroll
        for (int h = 0; h < MERGE_HEADS; ++h) {
            ml[h] = *reinterpret_cast<const float2 *>(a.part_ml + 2 * (place[h] + s));
            v[h] = *reinterpret_cast<const float2 *>(a.part_o + (place[h] + s) * 128 + 2 * lane);
        }
#pragma unroll
        for (int h = 0; h < MERGE_HEADS; ++h) {
            const float f = __builtin_amdgcn_exp2f(ml[h].x - top[h]);
            l[h] = fmaf(ml[h].y, f, l[h]);
            o0[h] = fmaf(v[h].x, f, o0[h]);
            o1[h] = fmaf(v[h].y, f, o1[h]);
        }
    }
    float2 s1 = make_float2(1.0f, 1.0f), s2 = s1;
    if (a.vs1) {
        s1 = *reinterpret_cast<const float2 *>(a.vs1 + 2 * lane);
        s2 = *reinterpret_cast<const float2 *>(a.vs2 + 2 * lane);
    }
#pragma unroll
    for (int h = 0; h < MERGE_HEADS; ++h) {
        if (head0 + h >= heads) return;
        float inv = l[h] > 0.0f ? a.v_unscale / l[h] : l[h] == 0.0f ? 0.0f : l[h], x0 = o0[h], x1 = o1[h];
        if (a.vs1) {
            x0 *= s2.x;
            x1 *= s2.y;
            wht128_wave(x0, x1, lane);
            x0 *= s1.x;
            x1 *= s1.y;
            inv *= RSQRT128;
        }
        x0 *= inv;
        x1 *= inv;
        const uint32_t lo = a.bf16 ? __builtin_bit_cast(uint16_t, (__bf16)x0) : __builtin_bit_cast(uint16_t, (_Float16)x0);
        const uint32_t hi = a.bf16 ? __builtin_bit_cast(uint16_t, (__bf16)x1) : __builtin_bit_cast(uint16_t, (_Float16)x1);
        reinterpret_cast<uint32_t *>(a.out)[(out_row + head0 + h) * 64 + lane] = lo | (hi << 16);
    }
}

struct Plan {
    PagedKind kind;
    int kw, n_splits, split_tiles, max_context, max_new;
    int64_t items;   // row blocks of all sequences, an upper bound
    unsigned grid;
    // few rows: k_decode_attn and k_decode_turbo
    bool few, lane_tables;
    int hg, wpw, gpw, parts, passes, wg_tiles, splits;
};
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t merge_groups(const tq_paged_attn_params *p) { return ceil_div(p->rows * ceil_div(p->n_q_heads, MERGE_HEADS), MERGE_THREADS / 64); }
struct Formats {
    int kb, vb;    // code widths, 8 for 8-bit rows
    bool share;    // one codebook
};
// The decode kernels: four rows per pass, or eight, and as many wavefronts as the chip holds at once, each with two tiles at least (16 x 8
// groups at 32K, turbo3, us: 93; twice as many wavefronts 102, four times 125; 32 ragged sequences 117, 126, 147).  Workgroups are
// shared among groups, cut to make one for every CU, and run by k_decode_turbo with its larger tables as in a step over contiguous
// caches.  A workgroup's share of the tiles follows from max_context: sequences that are shorter leave workgroups idle, which end
// at once, and none has more to do than another.
bool plan_few(const tq_paged_attn_params *p, const Formats &f, int64_t most, Plan &pl) {
    const bool turbo_k = f.kb != 8, turbo_v = f.vb != 8;
    pl.hg = most > 4 ? 2 : 1;
    pl.passes = (int)ceil_div(most, 4 * pl.hg);
    const int64_t groups = (int64_t)p->pages.batch * p->pages.n_kv_heads, units = groups * pl.passes, tiles = std::max<int64_t>(1, ceil_div(pl.max_context, 64));
    const int wmax = tqattn::max_waves_per_workgroup(turbo_v ? 0 : 8, pl.hg), resident = pl.hg == 1 && turbo_v ? 16 : 8;
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(256ll * resident / units, ceil_div(tiles, 2)));
    pl.gpw = 1;
    if (want <= wmax / 2) {   // several groups to a workgroup
        int64_t s = 1;
        while (2 * s <= want) s *= 2;
        int64_t g = wmax / s;
        while (g > 1 && (groups % g != 0 || units / g < 256)) g /= 2;
        if (g > 1) {
            pl.gpw = (int)g;
            pl.wpw = (int)(g * s);
            pl.splits = (int)s;
            pl.parts = 1;
            pl.wg_tiles = (int)tiles;
        }
    }
    if (pl.gpw == 1) {
        pl.wpw = wmax;
        if (pl.hg == 2 && turbo_k && turbo_v && want % 12 == 0) pl.wpw = 12;
        while (pl.wpw > 1 && pl.wpw > want) pl.wpw /= 2;
        while (pl.wpw > 4 && pl.wpw % 2 == 0 && units * ceil_div(want, pl.wpw) < 256) pl.wpw /= 2;
        pl.wg_tiles = (int)ceil_div(tiles, ceil_div(want, pl.wpw));
        pl.parts = (int)ceil_div(tiles, pl.wg_tiles);
        pl.splits = pl.parts * pl.wpw;
    }
    const int tables = tqk_decode_turbo_lds(f.kb, f.vb, f.share) + pl.gpw * 1024 * pl.hg;
    const int64_t wgs = units * pl.parts / pl.gpw, per_cu = std::min<int64_t>(ceil_div(wgs, 256), std::max(1, (pl.hg == 2 ? 12 : 16) / pl.wpw));
    pl.lane_tables = turbo_k && turbo_v && (f.kb == 4 || f.vb == 4) && per_cu * tables <= 160 * 1024 && ceil_div(tiles, pl.splits) >= 3 && pl.wpw >= 4;
    if (wgs / pl.passes > 0x7FFFFFFF || pl.passes > 65535) return false;
    pl.grid = (unsigned)(wgs / pl.passes);
    pl.n_splits = 1;
    return true;
}
bool make_plan(const tq_paged_attn_params *p, const Formats &f, Plan &pl) {
    const int64_t group = p->n_q_heads / p->pages.n_kv_heads, rows = p->rows;
    const int64_t max_new = p->pages.cu_new ? (p->max_new > 0 ? std::min<int64_t>(p->max_new, rows) : rows) : 1;
    pl.max_new = (int)max_new;
    const int64_t most = max_new * group, space = (int64_t)p->pages.max_blocks * TQ_ROWS_PER_BLOCK;
    pl.max_context = (int)(p->max_context > 0 ? std::min<int64_t>(p->max_context, space) : space);
    // Up to two passes of eight rows the decode kernels are ahead, whose loads are a row to a lane (16 ragged sequences of up to 8000
    // positions, 8 KV heads, turbo3, us: 16 rows 47; 24 rows three passes 68, ROWS_32 59, CHUNK_128 107).  Then a wavefront
    // that decodes for itself (40 rows ROWS_48 80, CHUNK_128 115), then shared operands (64 rows CHUNK_64 96, CHUNK_128 113; 128 rows
    // CHUNK_64 162, CHUNK_128 125; 448 rows over 1500 positions, 64 heads, CHUNK_128 81, CHUNK_256 75; 800 rows over 32K 279, 213;
    // 8192 rows 1414, 1290).
    pl.few = most <= 16;
    if (pl.few) return plan_few(p, f, most, pl);
    pl.kind = most <= 32 ? ROWS_32 : most <= 48 ? ROWS_48 : most <= 64 ? CHUNK_64 : most < 256 ? CHUNK_128 : CHUNK_256;
    const int64_t tile = rows_of(pl.kind);
    pl.items = std::min(p->pages.batch * ceil_div(most, tile), rows * group / tile + p->pages.batch);
    const int64_t tiles = std::max<int64_t>(1, ceil_div(pl.max_context, 64)), blocks = pl.items * p->pages.n_kv_heads;
    // wavefronts (chunks: workgroups) that the chip holds at once, and the tiles that one is given at least.  More rounds of smaller parts
    // even out ragged batches but pay for it in partial results (6 prompts of up to 2501 tokens 321 us, 626 with four times the parts).
    const int w = pl.kind == ROWS_32 || pl.kind == ROWS_48 ? ROWS_WAVES : 1;   // wavefronts that can share a row block
    const int64_t want = pl.kind == ROWS_32 ? 2048 : pl.kind == ROWS_48 ? 1024 : pl.kind == CHUNK_256 ? 256 : 512, least = w > 1 ? 2 : 8;
    pl.kw = 1;
    while (pl.kw < w && blocks * pl.kw < want && tiles >= 2 * pl.kw) pl.kw *= 2;
    const int64_t splits = std::max<int64_t>(1, std::min(ceil_div(want, blocks * pl.kw), tiles / (least * pl.kw)));
    pl.split_tiles = (int)ceil_div(tiles, splits);
    pl.n_splits = (int)ceil_div(tiles, pl.split_tiles);
    const int64_t grid = ceil_div(pl.items, w / pl.kw) * pl.n_splits * p->pages.n_kv_heads;
    if (grid > 0x7FFFFFFF || rows * group > 0x7FFFFFFF || merge_groups(p) > 0x7FFFFFFF) return false;
    pl.grid = (unsigned)grid;
    return true;
}
// partial results, of a row's 128 sums, maximum and sum of weights each
int64_t part_values(const tq_paged_attn_params *p, const Plan &pl) {
    // few rows: a partial has places for whole sets of four; one more per group holds its counter of finished workgroups
    if (pl.few) return pl.parts > 1 ? (int64_t)p->pages.batch * p->pages.n_kv_heads * pl.passes * (pl.parts + 1) * 4 * pl.hg : 0;
    return pl.n_splits > 1 ? p->rows * p->n_q_heads * (int64_t)pl.n_splits : 0;
}
// most bytes that the call needs with any formats
int64_t workspace_bytes_of(const tq_paged_attn_params *p, bool &ok) {
    int64_t most = 0;
    ok = true;
    for (const Formats &f : {Formats{3, 3, true}, Formats{3, 8, false}, Formats{8, 3, false}}) {
        Plan pl;
        ok = ok && make_plan(p, f, pl);
        if (ok) most = std::max(most, part_values(p, pl));
    }
    return most * 130 * 4 + 16;
}
int attend_few(const tq_handle *hk, const tq_handle *hv, const tq_paged_attn_params *p, const Plan &pl, const Formats &f, const void *q, const void *k,
               const void *v, void *out, void *ws, int max_context, hipStream_t s) {
    const int64_t groups = (int64_t)p->pages.batch * p->pages.n_kv_heads, partials = groups * pl.passes * pl.parts;
    tqattn::AttnArgs a{};
    a.q = q; a.k = (const uint8_t *)k; a.v = (const uint8_t *)v; a.out = (float *)out;
    a.scale_log2e = p->scale * 1.4426950408889634f;
    a.pg.v_unscale = 1.0f;
    if (hk) { a.klut = hk->scaled_lut; a.ks1 = hk->s1_32; a.ks2 = hk->s2_32; a.scale_log2e /= hk->value_scale; }
    if (hv) { a.vlut = hv->scaled_lut; a.vs1 = hv->s1_32; a.vs2 = hv->s2_32; a.pg.v_unscale = 1.0f / hv->value_scale; }
    a.part_o = (float *)ws;
    a.part_ml = a.part_o + partials * 4 * pl.hg * 128;
    a.flags = (unsigned long long *)(a.part_ml + partials * 4 * pl.hg * 2);
    a.nonce = tqk_attn_nonce();
    a.n_groups = (int)groups;
    a.n_splits = pl.splits;
    a.q_group = pl.max_new * (p->n_q_heads / p->pages.n_kv_heads);
    a.pass_heads = 4 * pl.hg;
    a.gpw = pl.gpw;
    while ((1 << a.gw_shift) < pl.splits) ++a.gw_shift;
    a.wgs_per_group = pl.parts;
    a.pg.r = PagedRows{p->pages, p->rows, tqd::make_fast_div((uint32_t)p->pages.n_kv_heads)};
    a.pg.heads_div = tqd::make_fast_div((uint32_t)(p->n_q_heads / p->pages.n_kv_heads));
    a.pg.q_token = p->q_token; a.pg.q_head = p->q_head;
    a.pg.max_context = max_context; a.pg.max_new = pl.max_new;
    a.pg.causal = p->causal != 0; a.pg.bf16 = p->dtype == TQ_BF16;
    a.pg.wg_tiles = pl.wg_tiles;
    a.pg.wg_div = tqd::make_fast_div((uint32_t)pl.wg_tiles);
    a.pg.wave_div = tqd::make_fast_div((uint32_t)pl.wpw);
    const dim3 grid(pl.grid, (unsigned)pl.passes);
    const size_t lds = (size_t)pl.wpw * pl.hg * tqattn::MERGE_FLOATS * sizeof(float) + (size_t)pl.gpw * 1024 * pl.hg;
    const bool built = pl.lane_tables ? tqk_launch_paged_turbo(a, f.kb, f.vb, f.share, 4 * pl.hg, grid, pl.wpw, s)
                                      : tqk_launch_paged(a, f.kb, f.vb, f.share, pl.hg, grid, 64u * (unsigned)pl.wpw, lds, s);
    if (!built) {
        tq_set_error("tq_paged_attention: K of %d bits with V of %d bits is not built", f.kb, f.vb);
        return TQ_ERR_UNSUPPORTED;
    }
    return tq_check_launch("paged_attention");
}

int check_pages(const tq_pages *p, int64_t rows, const char *who) {
    REQUIRE(p, TQ_ERR_ARG, "%s: null pages", who);
    REQUIRE(p->batch >= 0 && p->n_kv_heads >= 1 && p->n_pages >= 0 && p->max_blocks >= 0 && rows >= 0, TQ_ERR_ARG, "%s: negative size", who);
    REQUIRE(p->n_kv_heads <= 65536 && (int64_t)p->batch * p->n_kv_heads <= 0x7FFFFFFF, TQ_ERR_UNSUPPORTED,
            "%s: over 65536 KV heads, or over 2^31 - 1 of all sequences", who);
    REQUIRE(p->max_blocks < (1 << 24) && rows <= 0x7FFFFFFF, TQ_ERR_UNSUPPORTED, "%s: positions and rows have to fit 32 bits", who);
    REQUIRE(p->table_stride >= p->max_blocks || p->batch <= 1, TQ_ERR_ARG, "%s: table_stride %lld is under max_blocks %d", who,
            (long long)p->table_stride, p->max_blocks);
    REQUIRE(p->cu_new || rows >= p->batch, TQ_ERR_ARG, "%s: %lld rows for %d sequences", who, (long long)rows, p->batch);
    const uintptr_t at = reinterpret_cast<uintptr_t>(p->block_table) | reinterpret_cast<uintptr_t>(p->cu_new) | reinterpret_cast<uintptr_t>(p->lens);
    REQUIRE(at % 4 == 0, TQ_ERR_ALIGN, "%s: a table is not aligned to its type", who);
    if (p->batch == 0 || rows == 0) return TQ_OK;
    REQUIRE(p->lens && (p->block_table || p->max_blocks == 0), TQ_ERR_ARG, "%s: null table", who);
    return TQ_OK;
}
int check_sides(const tq_handle *hk, const tq_handle *hv, const char *who) {
    const int rc = hk ? check_fast(hk, who) : TQ_OK;
    return rc ? rc : hv ? check_fast(hv, who) : TQ_OK;
}
int check_attn(const tq_paged_attn_params *p) {
    REQUIRE(p, TQ_ERR_ARG, "tq_paged_attention: null parameters");
    const int rc = check_pages(&p->pages, p->rows, "tq_paged_attention");
    if (rc) return rc;
    REQUIRE(p->n_q_heads >= 1 && p->n_q_heads % p->pages.n_kv_heads == 0, TQ_ERR_ARG,
            "tq_paged_attention: %d query heads are not a multiple of the KV head count (%d)", p->n_q_heads, p->pages.n_kv_heads);
    REQUIRE(p->scale > 1e-18f && p->scale < 1e18f, TQ_ERR_ARG, "tq_paged_attention: scale %g is not positive and finite", (double)p->scale);
    REQUIRE(p->dtype == TQ_F16 || p->dtype == TQ_BF16, TQ_ERR_ARG, "tq_paged_attention: dtype %d is neither float16 nor bfloat16", p->dtype);
    REQUIRE(p->max_context >= 0 && p->max_new >= 0, TQ_ERR_ARG, "tq_paged_attention: negative size");
    return TQ_OK;
}

}  // namespace

extern "C" {

int tq_append_paged(const tq_handle *hk, const tq_handle *hv, const tq_pages *pages, const void *k, const void *v, int64_t rows,
                    int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head, int in_dtype, void *k_pages, void *v_pages,
                    uint32_t *overrun_dev, void *stream) {
    int rc = check_sides(hk, hv, "tq_append_paged");
    rc = rc ? rc : check_pages(pages, rows, "tq_append_paged");
    if (rc) return rc;
    REQUIRE(in_dtype == TQ_F16 || in_dtype == TQ_BF16 || in_dtype == TQ_F32, TQ_ERR_ARG, "tq_append_paged: dtype %d is none of float16, bfloat16, float32",
            in_dtype);
    if (pages->batch == 0 || rows == 0) return TQ_OK;
    REQUIRE(k && v && ((k_pages && v_pages) || pages->n_pages == 0), TQ_ERR_ARG, "tq_append_paged: null pointer");
    const int each = in_dtype == TQ_F32 ? 4 : 2;
    auto steps_ok = [&](const void *x, int64_t token, int64_t head) { return aligned16(x) && token * each % 16 == 0 && head * each % 16 == 0; };
    REQUIRE((!hk || steps_ok(k, k_token, k_head)) && (!hv || steps_ok(v, v_token, v_head)) && aligned16(k_pages) && aligned16(v_pages) &&
                reinterpret_cast<uintptr_t>(k) % each == 0 && reinterpret_cast<uintptr_t>(v) % each == 0,
            TQ_ERR_ALIGN, "tq_append_paged: pages, and rows and strides of turbo formats, must be multiples of 16 bytes");
    REQUIRE((reinterpret_cast<uintptr_t>(overrun_dev) & 3u) == 0, TQ_ERR_ALIGN, "tq_append_paged: overrun_dev must be 4-byte aligned");
    return tqk_append_paged(hk, hv, pages, k, v, rows, k_token, k_head, v_token, v_head, in_dtype, k_pages, v_pages, overrun_dev, (hipStream_t)stream);
}

int tq_load_paged(const tq_handle *hk, const tq_handle *hv, const tq_pages *pages, const void *k_pages, const void *v_pages, int64_t rows,
                  void *out_k, void *out_v, void *stream) {
    int rc = check_sides(hk, hv, "tq_load_paged");
    rc = rc ? rc : check_pages(pages, rows, "tq_load_paged");
    if (rc) return rc;
    if (pages->batch == 0 || rows == 0) return TQ_OK;
    REQUIRE(out_k && out_v && ((k_pages && v_pages) || pages->n_pages == 0), TQ_ERR_ARG, "tq_load_paged: null pointer");
    REQUIRE(aligned16(out_k) && aligned16(out_v) && aligned16(k_pages) && aligned16(v_pages), TQ_ERR_ALIGN,
            "tq_load_paged: pages and outputs must be 16-byte aligned");
    return tqk_load_paged(hk, hv, pages, k_pages, v_pages, rows, out_k, out_v, (hipStream_t)stream);
}

int64_t tq_paged_attn_workspace_bytes(const tq_paged_attn_params *p) {
    if (check_attn(p)) return -1;
    if (p->pages.batch == 0 || p->rows == 0) return 16;
    bool ok;
    const int64_t need = workspace_bytes_of(p, ok);
    if (!ok) tq_set_error("tq_paged_attention: %lld rows are more than a launch takes", (long long)p->rows);
    return ok ? need : -1;
}

int tq_paged_attention(const tq_handle *hk, const tq_handle *hv, const tq_paged_attn_params *p, const void *q, const void *k_pages,
                       const void *v_pages, void *out, void *workspace, int64_t workspace_bytes, void *stream) {
    int rc = check_sides(hk, hv, "tq_paged_attention");
    rc = rc ? rc : check_attn(p);
    if (rc) return rc;
    if (p->pages.batch == 0 || p->rows == 0) return TQ_OK;
    const bool no_pages = p->pages.n_pages == 0 || p->pages.max_blocks == 0;
    REQUIRE(q && out && workspace && (no_pages || (k_pages && v_pages)), TQ_ERR_ARG, "tq_paged_attention: null pointer");
    REQUIRE(aligned16(q) && aligned16(out) && aligned16(workspace) && aligned16(k_pages) && aligned16(v_pages) && p->q_token % 8 == 0 && p->q_head % 8 == 0,
            TQ_ERR_ALIGN, "tq_paged_attention: q, its strides, out, pages and workspace must be multiples of 16 bytes");
    const int kb = hk ? hk->bits : 8, vb = hv ? hv->bits : 8;
    const bool share = hk && hv && kb == vb && std::memcmp(hk->centroids_host, hv->centroids_host, sizeof(double) << kb) == 0;
    bool ok;
    const int64_t need = workspace_bytes_of(p, ok);
    Plan pl;
    const Formats f{kb, vb, share};
    if (!ok || !make_plan(p, f, pl)) {
        tq_set_error("tq_paged_attention: %lld rows are more than a launch takes", (long long)p->rows);
        return TQ_ERR_UNSUPPORTED;
    }
    REQUIRE(workspace_bytes >= need, TQ_ERR_ARG, "tq_paged_attention: the workspace holds %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)need);
    if (pl.few) return attend_few(hk, hv, p, pl, f, q, k_pages, v_pages, out, workspace, no_pages ? 0 : pl.max_context, (hipStream_t)stream);
    PagedAttnArgs a{};
    a.r = PagedRows{p->pages, p->rows, tqd::make_fast_div((uint32_t)p->pages.n_kv_heads)};
    a.q = q; a.out = out; a.q_token = p->q_token; a.q_head = p->q_head;
    a.bf16 = p->dtype == TQ_BF16; a.causal = p->causal != 0;
    a.max_context = no_pages ? 0 : pl.max_context;   // nothing is read then
    a.max_new = pl.max_new;
    a.blocks_each = p->pages.cu_new ? 0 : (int)ceil_div(p->n_q_heads / p->pages.n_kv_heads, rows_of(pl.kind));
    a.group = p->n_q_heads / p->pages.n_kv_heads;
    a.group_div = tqd::make_fast_div((uint32_t)a.group); a.heads_div = a.r.heads_div;
    a.k = (const uint8_t *)k_pages; a.v = (const uint8_t *)v_pages;
    a.scale = p->scale * 1.4426950408889634f;
    a.v_unscale = 1.0f;
    if (hk) {
        a.klut = hk->scaled_lut;
        a.scale /= hk->value_scale;
        for (int i = 0; i < 4; ++i) { a.ks1neg[i] = hk->s1neg_host[i]; a.ks2neg[i] = hk->s2neg_host[i]; }
    }
    if (hv) { a.vlut = hv->scaled_lut; a.vs1 = hv->s1_32; a.vs2 = hv->s2_32; a.v_unscale = 1.0f / hv->value_scale; }
    a.n_splits = pl.n_splits; a.split_tiles = pl.split_tiles; a.kw = pl.kw;
    a.part_o = (float *)workspace;
    a.part_ml = a.part_o + part_values(p, pl) * 128;
    a.share = share;
    hipStream_t s = (hipStream_t)stream;
    switch (kb) {
    case 2: rc = tqk_paged_attn_k2(a, vb, pl.kind, pl.grid, s); break;
    case 3: rc = tqk_paged_attn_k3(a, vb, pl.kind, pl.grid, s); break;
    case 4: rc = tqk_paged_attn_k4(a, vb, pl.kind, pl.grid, s); break;
    default: rc = tqk_paged_attn_k8(a, vb, pl.kind, pl.grid, s); break;
    }
    if (rc || pl.n_splits == 1) return rc;
    k_paged_merge<<<(unsigned)merge_groups(p), MERGE_THREADS, 0, s>>>(a);
    return tq_check_launch("paged_merge");
}

}  // extern "C"
