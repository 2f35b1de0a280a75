// Attention of several new tokens over a paged cache of packed rows (tq_paged_attention): k_paged_rows for 17 to 48 rows of a KV
// head (a row: one new token under one query head), k_paged_chunk for more; fewer run on k_decode_attn and k_decode_turbo.
//
// Both walk tiles of 64 positions.  Codes become fp16 operands of 16x16x32 matrix instructions through decode tables in LDS, and
// each operand serves several blocks of 16 rows: what a tile costs to decode is paid once for all of them.
//   S^T = K Q^T.  A = K: lane (m = lane % 16, kq = lane / 16) holds dims 32 kq .. 32 kq + 31 of a token, which are BITS dwords of its
//     row (one pair group), 8 of them per step; B = Q likewise, so Q is loaded, rotated and scaled in the layout in which it is
//     used.  Row m of unit u is token 16 (m / 4) + 4 u + m % 4 of the tile: the result then gives lane (n, kq) the logits of
//     row n for the tokens 16 kq + 4 u + i.
//   softmax: running maximum and sum per lane and row block in 32 bits; the maximum goes over the four lanes of a row.  A token's norm of
//     K multiplies the logits in 32 bits (as fp16 operands they would double the error of the result).
//   O^T = V^T P^T.  B = P: the lane's own 16 weights, rounded to fp16 with the tokens' norms in them (|error| <= 2^-11 of a weight, of
//     either sign, so a sum of them is as good as its rounding to 16 bits); A = V: rows are dims, lane (m, kq) takes the pair group kq =
//     tokens 16 kq .. 16 kq + 15 of dims m and 64 + m of a 16-row block.  No exchange between lanes anywhere in the loop but the
//     maximum.
// A query's rounding to fp16 is the largest error of a result (5e-4 of its size over 4000 to 32K positions).
// The result of a lane is 32 dims of a row, and the transposed rotation of V is a butterfly of five stages in registers and two
// across lanes.  Where rows are few, n_splits workgroups share the positions and join through partial results in memory (32
// bits) and k_paged_merge.
// One MI355X.  17 to 48 rows are bound by the decoding: 16 ragged sequences of up to 8000 positions, 8 KV heads, turbo3: 24 rows 59 us
// (k_paged_chunk 107), 40 rows 75 us (115).  Many rows are bound by the matrix instructions with the softmax between them: 2048
// tokens x 32 heads at the end of 32K positions 1.28 ms, 834 TFLOP/s where a product of 8192^3 fp16 matrices reaches 1159 (vector unit
// 55 %, matrix unit 35 %, LDS 35 % busy before two tiles of logits were in flight).
#pragma once
#include <type_traits>

#include "tq_device.h"
#include "tq_paged.h"

namespace tqpaged {

using namespace tqd;

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr float RSQRT128 = 0.08838834764831845f;

// How rows are dealt out, by a sequence's most: 32 or 48 to a wavefront that decodes for itself, 64, 128 or 256 to a workgroup
enum PagedKind { ROWS_32, ROWS_48, CHUNK_64, CHUNK_128, CHUNK_256 };
__host__ __device__ constexpr int rows_of(PagedKind k) { return k == ROWS_32 ? 32 : k == ROWS_48 ? 48 : k == CHUNK_64 ? 64 : k == CHUNK_128 ? 128 : 256; }

struct PagedAttnArgs {
    PagedRows r;
    const void *q;
    void *out;
    int64_t q_token, q_head;
    int bf16, causal, max_context, max_new;
    int group;                   // query heads per KV head
    int blocks_each;             // 0, or the row blocks that every sequence has
    FastDiv group_div, heads_div;
    const uint8_t *k, *v;
    const uint32_t *klut, *vlut; // pair tables of value_scale times the codebook
    uint32_t ks1neg[4], ks2neg[4];   // negative signs of K's rotation, 32 dims to a word
    const float *vs1, *vs2;
    float scale;                 // logits' scale * log2(e) / value_scale of K
    float v_unscale;             // 1 / value_scale of V
    int share;                   // K's table is V's
    int n_splits, split_tiles;   // of the positions, and 64-position tiles of each
    int kw;                      // wavefronts that share a row block's positions
    float *part_o, *part_ml;     // [row][query head][split]: 128 sums; maximum (log2 units), sum of weights
};

__device__ __forceinline__ float load_value(const void *p, int64_t i, int bf16) {
    return bf16 ? (float)reinterpret_cast<const __bf16 *>(p)[i] : (float)reinterpret_cast<const _Float16 *>(p)[i];
}

// what a sequence's launch covers: tokens that count, and splits that have any
struct PagedSpan {
    int ctx, splits;
};
__device__ __forceinline__ PagedSpan paged_span(const PagedAttnArgs &a, const PagedSeq &q) {
    PagedSpan s;
    s.ctx = (int)(q.start < 0 ? 0 : q.start > a.max_context ? a.max_context : q.start);
    const int tiles = (s.ctx + 63) >> 6;
    s.splits = a.n_splits == 1 ? 1 : (tiles + a.split_tiles - 1) / a.split_tiles;
    return s;
}

// ---- decode tables ---------------------------------------------------------------------------------
// Two fp16 values per entry, indexed by a pair code, with C copies next to each other: lanes read their own copy, so that
// look-ups of a wavefront meet in few banks.
__host__ __device__ constexpr int pair_table_bytes(int bits, int copies) { return bits == 8 ? 0 : (4 << (2 * bits)) * copies; }
template <int BITS, int C> __device__ __forceinline__ void build_pair_table(char *dst, const uint32_t *pairs, int tid, int threads) {
    for (int e = tid; e < (C << (2 * BITS)) / 4; e += threads) {
        const uint32_t p = pairs[4 * e / C];
        reinterpret_cast<uint4 *>(dst)[e] = make_uint4(p, p, p, p);
    }
}
template <int BITS> __device__ __forceinline__ uint32_t group_tail(const uint32_t (&w)[BITS]) {
    if constexpr (BITS == 3) return (w[0] >> 24) | ((w[1] >> 24) << 8) | ((w[2] >> 24) << 16);
    else return 0u;
}
constexpr int log2_of(int x) { return x <= 1 ? 0 : 1 + log2_of(x >> 1); }
// the two values of pair P = 0 .. 15 of a pair group; copy: 4 (lane % C)
template <int BITS, int C> __device__ __forceinline__ uint32_t group_pair(const uint32_t (&w)[BITS], uint32_t tail, const char *lut, uint32_t copy, int P) {
    constexpr int SCALE = 2 + log2_of(C);
    uint32_t at;
    if constexpr (BITS == 4) at = field_offset<SCALE>(w[P >> 2], 8 * (P & 3), 8);
    else if constexpr (BITS == 2) at = field_offset<SCALE>(w[P >> 3], 4 * (P & 7), 4);
    else at = P < 12 ? field_offset<SCALE>(w[P < 12 ? P >> 2 : 0], 6 * (P & 3), 6) : field_offset<SCALE>(tail, 6 * (P - 12), 6);
    return *reinterpret_cast<const uint32_t *>(lut + (at | copy));
}
// the four values of quad Q = 0 .. 7
template <int BITS, int C> __device__ __forceinline__ uint2 group_quad(const uint32_t (&w)[BITS], uint32_t tail, const char *lut, uint32_t copy, int Q) {
    return make_uint2(group_pair<BITS, C>(w, tail, lut, copy, 2 * Q), group_pair<BITS, C>(w, tail, lut, copy, 2 * Q + 1));
}
__device__ __forceinline__ half8_t join(uint2 a, uint2 b) { return __builtin_bit_cast(half8_t, make_uint4(a.x, a.y, b.x, b.y)); }

// four int8 of a dword as fp16 times `s`, in the order 0, 2, 1, 3: 0x6400 | (x + 128) is the fp16 number 1152 + x
__device__ __forceinline__ uint2 int8x4_times(uint32_t w, half2_t s02, half2_t s13) {
    const uint32_t u = w ^ 0x80808080u;
    const half2_t bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    const half2_t h02 = (__builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04020400u)) - bias) * s02;
    const half2_t h13 = (__builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030401u)) - bias) * s13;
    return make_uint2(__builtin_bit_cast(uint32_t, h02), __builtin_bit_cast(uint32_t, h13));
}

__device__ __forceinline__ float half_of(uint32_t w, int i) { return __half2float(__ushort_as_half((unsigned short)(i ? w >> 16 : w & 0xffff))); }
__device__ __forceinline__ float over_row_max(float v) {
    v = fmaxf(v, xor_lane<16>(v));
    return fmaxf(v, xor_lane<32>(v));
}
__device__ __forceinline__ float over_row_sum(float v) {
    v += xor_lane<16>(v);
    return v + xor_lane<32>(v);
}

// 128-point butterfly over values that four lanes (kq = lane / 16) hold 32 each of; which of their dims' bits is a lane's does not
// matter to it
__device__ __forceinline__ void butterfly32x4(float (&x)[32], int lane) {
#pragma unroll
    for (int h = 1; h < 32; h <<= 1)
#pragma unroll
        for (int e = 0; e < 32; ++e)
            if ((e & h) == 0) {
                const float s = x[e], d = x[e + h];
                x[e] = s + d;
                x[e + h] = s - d;
            }
    const float s16 = lane & 16 ? -1.0f : 1.0f, s32 = lane & 32 ? -1.0f : 1.0f;
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e] = bfly<16>(x[e], s16);
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e] = bfly<32>(x[e], s32);
}

// dim of output register e of lane quarter kq: e = 16 hf + 4 block + i
__device__ __forceinline__ int out_dim(int e, int kq) { return 64 * (e >> 4) + 16 * ((e >> 2) & 3) + 4 * kq + (e & 3); }

// a row's sums -> its output: over the weights' sum, V's rotation undone, rounded to the type
__device__ __forceinline__ void write_out(const PagedAttnArgs &a, float (&o)[32], float inv_l, int64_t row, int head, bool there, int lane) {
    const int kq = lane >> 4;
    if (a.vs1) {
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
            const float4 s = *reinterpret_cast<const float4 *>(a.vs2 + out_dim(e, kq));
            o[e] *= s.x; o[e + 1] *= s.y; o[e + 2] *= s.z; o[e + 3] *= s.w;
        }
        butterfly32x4(o, lane);
        inv_l *= RSQRT128;
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
            const float4 s = *reinterpret_cast<const float4 *>(a.vs1 + out_dim(e, kq));
            o[e] *= s.x; o[e + 1] *= s.y; o[e + 2] *= s.z; o[e + 3] *= s.w;
        }
    }
    if (!there) return;
    uint16_t *to = reinterpret_cast<uint16_t *>(a.out) + (row * (a.r.p.n_kv_heads * a.group) + head) * 128;
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
        uint16_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = o[e + i] * inv_l;
            h[i] = a.bf16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
        }
        *reinterpret_cast<uint2 *>(to + out_dim(e, kq)) = make_uint2(h[0] | ((uint32_t)h[1] << 16), h[2] | ((uint32_t)h[3] << 16));
    }
}

// Rows r0 .. of a sequence, RB blocks of 16 of them to a wavefront: which they are, their queries, and what the walk leaves.
struct PagedBlock {
    PagedSeq seq;
    PagedSpan span;
    int n_rows, r0;    // rows of the sequence (tokens times query heads); the block's first
    bool active;       // it has rows, and positions in this split (the first split also if there are none)
};
// Row block `item` (of `rows` rows each) of all sequences
__device__ __forceinline__ PagedBlock paged_block(const PagedAttnArgs &a, int item, int rows, int split, int &b) {
    PagedBlock k{{0, 0, 0}, {0, 0}, 0, 0, false};
    int nth = 0;
    bool some;
    b = 0;
    if (a.blocks_each) {    // one row per sequence: every one has as many row blocks
        b = item / a.blocks_each;
        nth = item - b * a.blocks_each;
        some = b < a.r.p.batch;
        if (!some) b = 0;
        k.seq = paged_seq(a.r, b);
    } else some = paged_item(a.r, item, [&](const PagedSeq &q) { return (min(q.n, a.max_new) * a.group + rows - 1) / rows; }, b, nth, k.seq);
    if (some) {
        k.span = paged_span(a, k.seq);
        k.n_rows = min(k.seq.n, a.max_new) * a.group;
        // the last block first, which sees the most: short ones are left for the launch's end (8000 new tokens x 32 heads: 865 -> 727 us)
        k.r0 = (a.causal ? (k.n_rows + rows - 1) / rows - 1 - nth : nth) * rows;
        k.active = k.r0 >= 0 && k.r0 < k.n_rows && (split < k.span.splits || split == 0);
    }
    return k;
}
// positions that row r sees
__device__ __forceinline__ int row_limit(const PagedAttnArgs &a, const PagedBlock &k, int r) {
    const int t = (int)a.group_div.div((uint32_t)r), seen = a.causal ? k.span.ctx - k.seq.n + t + 1 : k.span.ctx;
    return seen < 0 ? 0 : seen;
}

// Queries of RB blocks from row `first` on: 32 values of row n16 of each block, rotated as K's rows are, as fp16 of their size up to
// a power of two, which joins the logits' scale.  Rows past the last one repeat it.
// The rotation goes through the matrix cores, whose products with +-1 are exact for either type.  Dim 32 kq + 8 ks + j in and dim
// 32 kq' + 8 c + 4 h + i out: H's sign is that of (kq' & kq), (c & ks) and (4 h + i) & j together, so two +-1 operands (h) serve the four
// steps ks, and the sums over ks are a butterfly of four: a quarter of the vector instructions of one of 128 values (40 rows of 16 ragged
// sequences 84 -> 79 us, 256 x 64 new tokens over themselves 188 -> 162 with the second tile's K requested beside the first's).
template <int KB, int RB>
__device__ __forceinline__ void load_queries(const PagedAttnArgs &a, const PagedBlock &k, int first, int head, int lane, half8_t (&qf)[RB][4],
                                             float (&scale)[RB], int (&seen)[RB]) {
    const int n16 = lane & 15, kq = lane >> 4;
    uint4 w[RB][4];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int r = min(first + 16 * rb + n16, max(k.n_rows - 1, 0));
        const int t = (int)a.group_div.div((uint32_t)r), g = r - t * a.group;
        seen[rb] = row_limit(a, k, r);
        const int64_t at = (int64_t)(k.seq.row0 + t) * a.q_token + (int64_t)(head * a.group + g) * a.q_head + 32 * kq;
        const uint4 *p = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(a.q) + (k.active ? at : 0));
#pragma unroll
        for (int c = 0; c < 4; ++c) w[rb][c] = p[c];
    }
    auto of_quarter = [&](const uint32_t (&x)[4]) { return kq < 2 ? (kq == 0 ? x[0] : x[1]) : (kq == 2 ? x[2] : x[3]); };
    const uint32_t neg1 = KB != 8 ? of_quarter(a.ks1neg) : 0u, neg2 = KB != 8 ? of_quarter(a.ks2neg) : 0u;
    uint4 f[2];
    if constexpr (KB != 8) {
        const uint32_t one = a.bf16 ? 0x3F803F80u : 0x3C003C00u;
        const uint32_t d0 = one ^ (__builtin_popcount((n16 >> 2) & kq) & 1 ? 0x80008000u : 0u) ^ (n16 & 1 ? 0x80000000u : 0u);
        const uint32_t d1 = d0 ^ (n16 & 2 ? 0x80008000u : 0u);
        f[0] = make_uint4(d0, d1, d0, d1);
        f[1] = make_uint4(d0, d1, d0 ^ 0x80008000u, d1 ^ 0x80008000u);
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        float x[32];
        if constexpr (KB != 8) {
            float4_t z[4][2];
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                auto flipped = [&](uint32_t v, int j) {   // the signs of dims 8 ks + 2 j and the next
                    const int e = 8 * ks + 2 * j;
                    return v ^ (((neg1 >> e) & 1u) << 15) ^ (((neg1 >> (e + 1)) & 1u) << 31);
                };
                const uint4 v = make_uint4(flipped(w[rb][ks].x, 0), flipped(w[rb][ks].y, 1), flipped(w[rb][ks].z, 2), flipped(w[rb][ks].w, 3));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float4_t none = {0.f, 0.f, 0.f, 0.f};
                    if (a.bf16) z[ks][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, f[h]), __builtin_bit_cast(bf16x8_t, v), none, 0, 0, 0);
                    else z[ks][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, f[h]), __builtin_bit_cast(half8_t, v), none, 0, 0, 0);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float s01 = z[0][h][i] + z[1][h][i], d01 = z[0][h][i] - z[1][h][i], s23 = z[2][h][i] + z[3][h][i], d23 = z[2][h][i] - z[3][h][i];
                    x[4 * h + i] = s01 + s23;
                    x[8 + 4 * h + i] = d01 + d23;
                    x[16 + 4 * h + i] = s01 - s23;
                    x[24 + 4 * h + i] = d01 - d23;
                }
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = __uint_as_float(__float_as_uint(x[e]) ^ (((neg2 >> e) & 1u) << 31));
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t u[4] = {w[rb][c].x, w[rb][c].y, w[rb][c].z, w[rb][c].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[8 * c + 2 * j] = a.bf16 ? __uint_as_float(u[j] << 16) : half_of(u[j], 0);
                    x[8 * c + 2 * j + 1] = a.bf16 ? __uint_as_float(u[j] & 0xFFFF0000u) : half_of(u[j], 1);
                }
            }
        }
        float most = 0.0f;
#pragma unroll
        for (int e = 0; e < 32; ++e) most = fmaxf(most, fabsf(x[e]));
        most = over_row_max(most);
        int ex = most > 0.0f && most < INFINITY ? __builtin_amdgcn_frexp_expf(most) : 0;
        ex = min(max(ex, -100), 120);
        scale[rb] = __builtin_amdgcn_ldexpf(KB != 8 ? a.scale * RSQRT128 : a.scale, ex);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // int8 rows hand their values over in the order 0, 2, 1, 3
                const int from = KB == 8 ? (e & 4) | ((e & 1) << 1) | ((e >> 1) & 1) : e;
                qf[rb][ks][e] = (_Float16)__builtin_amdgcn_ldexpf(x[8 * ks + from], -ex);
            }
    }
}

// One tile's logits of a row block, in three steps.  (1) times the tokens' norms, places that do not count out (MASKED: the lane's 16
// tokens of which the first `sees` do); the row's new maximum.
template <int KB, bool MASKED, class KNorm>
__device__ __forceinline__ float logits_max(float4_t (&s)[4], KNorm kn, int sees, float scale, float m) {
    float most = -INFINITY;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v = s[u][i];
            if constexpr (KB != 8) v *= kn(4 * u + i);
            if constexpr (MASKED) v = 4 * u + i < sees ? v : -INFINITY;
            s[u][i] = v;
            most = fmaxf(most, v);
        }
    return fmaxf(m, over_row_max(most) * scale);
}
// (2) the sums of all of a wavefront's row blocks shrink to the new maxima, which they rarely have to
template <int RB, typename L> __device__ __forceinline__ void move_max(const float (&m_new)[RB], float (&m)[RB], L (&l)[RB], float4_t (&o)[RB][2][4]) {
    bool moved = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) moved = moved || m_new[rb] != m[rb];
    if (__builtin_amdgcn_ballot_w64(moved) != 0ull) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const float shrink = m_new[rb] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[rb] - m_new[rb]);
            l[rb] *= shrink;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[rb][e >> 2][e & 3] *= shrink;
            m[rb] = m_new[rb];
        }
    }
}
// (3) the weights 2^(s scale - m), their sum, and the weights times the tokens' norms as fp16.  The product in a fused multiply-add is
// exact and m is one that was rounded: they differ by up to half a step of m, which is nothing below 2^20 but lets a weight
// overflow where logits are beyond 2^31.  So rows with logits past 2^20 have their products rounded.  FAST: there are none, and every
// row sees the whole tile; what a row gets does not depend on which of the two it goes through.
template <int VB, bool FAST, class VNorm>
__device__ __forceinline__ void weights(const float4_t (&s)[4], VNorm vn, int sees, float m, float scale, float &l, half8_t (&pf)[2]) {
    const float off = FAST || m != -INFINITY ? m : 0.0f;
    const bool near = fabsf(m) <= 0x1p20f;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x = fmaf(s[u][i], scale, -off);
            if constexpr (!FAST) {
#pragma clang fp contract(off)
                const float rounded = s[u][i] * scale - off;
                x = near ? x : rounded;
            }
            const float w = __builtin_amdgcn_exp2f(x);
            l += w;
            float p = w;
            if constexpr (VB != 8) {
                p = w * vn(4 * u + i);
                asm("" : "+v"(p));   // rounded to 32 bits before 16, FAST or not: the compiler makes one instruction with one rounding of some
                if constexpr (!FAST) p = 4 * u + i < sees ? p : 0.0f;   // what a masked place holds may be no number
            }
            // int8 rows: the order 0, 2, 1, 3
            const int to = VB == 8 ? ((i & 1) << 1) | (i >> 1) : i;
            pf[u >> 1][4 * (u & 1) + to] = (_Float16)p;
        }
}
// whether some row's logits are beyond what FAST weights are for
template <int RB> __device__ __forceinline__ bool far_logits(const float (&m)[RB]) {
    bool far = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) far = far || fabsf(m[rb]) > 0x1p20f;   // of -inf, too: nothing was seen so far
    return __builtin_amdgcn_ballot_w64(far) != 0ull;
}

// What a walk leaves of a row block (o, m and the sum of weights over the row): the output, or this split's partial result
template <int RB>
__device__ __forceinline__ void leave_rows(const PagedAttnArgs &a, const PagedBlock &k, int first, int head, int split, int lane, const float4_t (&o)[RB][2][4],
                                           const float (&m)[RB], const float (&l)[RB]) {
    const int n16 = lane & 15, kq = lane >> 4;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int r = first + 16 * rb + n16;
        const bool there = r < k.n_rows;
        const int t = (int)a.group_div.div((uint32_t)(there ? r : 0)), hq = head * a.group + (there ? r : 0) - t * a.group;
        float x[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = o[rb][e >> 4][(e >> 2) & 3][e & 3];
        if (k.span.splits <= 1) {
            write_out(a, x, l[rb] > 0.0f ? a.v_unscale / l[rb] : l[rb] == 0.0f ? 0.0f : l[rb], k.seq.row0 + t, hq, there, lane);
        } else if (there) {
            const int64_t at = ((int64_t)(k.seq.row0 + t) * (a.r.p.n_kv_heads * a.group) + hq) * a.n_splits + split;
#pragma unroll
            for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4 *>(a.part_o + at * 128 + out_dim(e, kq)) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
            if (kq == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * at) = make_float2(m[rb], l[rb]);
        }
    }
}

// This workgroup's KV head, split and number among the row blocks.  Neighbouring workgroups have the KV heads of the same rows:
// with eight of them each die keeps to one head's pages.
struct PagedTurn {
    int head, split, turn;
};
__device__ __forceinline__ PagedTurn paged_turn(const PagedAttnArgs &a) {
    const uint32_t rest = a.heads_div.div(blockIdx.x);
    PagedTurn p;
    p.head = (int)(blockIdx.x - rest * a.heads_div.d);
    p.split = a.n_splits == 1 ? 0 : (int)(rest % (uint32_t)a.n_splits);
    p.turn = a.n_splits == 1 ? (int)rest : (int)(rest / (uint32_t)a.n_splits);
    return p;
}

// ---- 17 to 48 rows: every wavefront decodes for itself ---------------------------------------------------
constexpr int ROWS_WAVES = 4;   // wavefronts of a workgroup
// floats that a wavefront leaves behind for another one to join: 32 RB sums, RB maxima and sums of weights per lane
__host__ __device__ constexpr int join_floats(int rb) { return 64 * 34 * rb; }
__host__ __device__ constexpr int rows_copies(int bits) { return bits == 4 ? 16 : 32; }
__host__ __device__ constexpr int rows_lds(int kb, int vb, int rb, bool share) {
    const int tables = pair_table_bytes(kb, rows_copies(kb)) + (share ? 0 : pair_table_bytes(vb, rows_copies(vb))), join = ROWS_WAVES / 2 * join_floats(rb) * 4;
    return tables > join ? tables : join;
}

// KB, VB: code widths, 8 for q8_0-style rows; RB: blocks of 16 rows per wavefront; SHARE: one table for K and V
template <int KB, int VB, int RB, bool SHARE>
__global__ __launch_bounds__(64 * ROWS_WAVES, RB == 2 ? 2 : 1) void k_paged_rows(PagedAttnArgs a) {
    constexpr int W = ROWS_WAVES, TILE = 16 * RB;
    constexpr int KBLOCK = KB == 8 ? TQ_ROWS_PER_BLOCK * 136 : block_bytes(KB), VBLOCK = VB == 8 ? TQ_ROWS_PER_BLOCK * 136 : block_bytes(VB);
    __shared__ __attribute__((aligned(16))) char smem[rows_lds(KB, VB, RB, SHARE)];
    __shared__ __attribute__((aligned(16))) uint4 q_s[W][RB][4][64];
    __shared__ float scale_s[W][RB][64];
    constexpr int KC = rows_copies(KB), VC = rows_copies(VB), V_TABLE = SHARE ? 0 : pair_table_bytes(KB, KC);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, kq = lane >> 4;
    const PagedTurn p = paged_turn(a);
    const int head = p.head, split = p.split, kw = a.kw, part = wave & (kw - 1);
    int b;
    const PagedBlock rows = paged_block(a, p.turn * (W / kw) + wave / kw, TILE, split, b);
    if (kw == W && !rows.active) return;    // all of the workgroup
    int t_begin = 0, t_end = 0, least = 0;
    if (rows.active) {
        least = row_limit(a, rows, rows.r0);
        t_begin = split * a.split_tiles;
        t_end = min((row_limit(a, rows, min(rows.r0 + TILE, rows.n_rows) - 1) + 63) >> 6, t_begin + a.split_tiles);
        const int each = (max(t_end - t_begin, 0) + kw - 1) / kw;
        t_begin += part * each;
        t_end = min(t_end, t_begin + each);
    }
    // ---- A tile's codes and norms are requested a tile ahead into the registers that its predecessor has just been read from: K's
    // after the logits, V's after the values; the first one's before anything else.
    const int32_t *table = a.r.p.block_table + (int64_t)__builtin_amdgcn_readfirstlane(b) * a.r.p.table_stride;
    auto page_of = [&](int tile) { return scalar_entry(table, __builtin_amdgcn_readfirstlane(tile >> 1)); };
    auto is_page = [&](int page) { return page >= 0 && page < a.r.p.n_pages; };
    auto block_at = [&](int page) { return (int64_t)(is_page(page) ? page : 0) * a.r.p.n_kv_heads + head; };
    uint32_t kw_[4][KB == 8 ? 8 : KB], vw[4][VB == 8 ? 8 : VB];
    uint32_t kn[8], vn[VB == 8 ? 32 : 8];   // norms of the lane's 16 tokens; 8-bit K: a scale per unit, 8-bit V: [32-dim block] of them
    const int k_row = 16 * (n16 >> 2) + (n16 & 3);
    auto load_k = [&](int tile, int page) {
        const uint8_t *kb = a.k + block_at(page) * KBLOCK;
        const int half = tile & 1;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int row = 64 * half + k_row + 4 * u;
            if constexpr (KB == 8) {
                const uint4 lo = *reinterpret_cast<const uint4 *>(kb + (2 * kq) * 2048 + row * 16);
                const uint4 hi = *reinterpret_cast<const uint4 *>(kb + (2 * kq + 1) * 2048 + row * 16);
                kw_[u][0] = lo.x; kw_[u][1] = lo.y; kw_[u][2] = lo.z; kw_[u][3] = lo.w;
                kw_[u][4] = hi.x; kw_[u][5] = hi.y; kw_[u][6] = hi.z; kw_[u][7] = hi.w;
                kn[u] = reinterpret_cast<const uint16_t *>(kb + 8 * 2048)[4 * row + kq];
            } else {
#pragma unroll
                for (int j = 0; j < KB; ++j) kw_[u][j] = *reinterpret_cast<const uint32_t *>(kb + j * 2048 + row * 16 + kq * 4);
            }
        }
        if constexpr (KB != 8) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint4 n = *reinterpret_cast<const uint4 *>(kb + block_code_bytes(KB) + 2 * (64 * half + 16 * kq) + 16 * c);
                kn[4 * c] = n.x; kn[4 * c + 1] = n.y; kn[4 * c + 2] = n.z; kn[4 * c + 3] = n.w;
            }
        }
    };
    auto load_v = [&](int tile, int page) {
        const uint8_t *vb = a.v + block_at(page) * VBLOCK;
        const int half = tile & 1;
#pragma unroll
        for (int blk = 0; blk < 4; ++blk) {
            const int row = 64 * half + 16 * blk + n16;
            if constexpr (VB == 8) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(vb + (4 * hf + kq) * 2048 + row * 16);
                    vw[blk][4 * hf] = w.x; vw[blk][4 * hf + 1] = w.y; vw[blk][4 * hf + 2] = w.z; vw[blk][4 * hf + 3] = w.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < VB; ++j) vw[blk][j] = *reinterpret_cast<const uint32_t *>(vb + j * 2048 + row * 16 + kq * 4);
            }
        }
#pragma unroll
        for (int c = 0; c < (VB == 8 ? 8 : 2); ++c) {
            const uint8_t *side = VB == 8 ? vb + 8 * 2048 + 2 * ((half * 4 + (c >> 1)) * 64 + 16 * kq) + 16 * (c & 1)
                                          : vb + 128 * 16 * VB + 2 * (64 * half + 16 * kq) + 16 * c;
            const uint4 n = *reinterpret_cast<const uint4 *>(side);
            vn[4 * c] = n.x; vn[4 * c + 1] = n.y; vn[4 * c + 2] = n.z; vn[4 * c + 3] = n.w;
        }
    };

    int page = 0, page_next = 0;
    if (t_begin < t_end) {
        page = page_of(t_begin);
        page_next = page_of(min(t_begin + 1, t_end - 1));
        load_k(t_begin, page);
        load_v(t_begin, page);
    }
    // queries: rotated by one wavefront of those that share the rows
    if (part == 0) {
        half8_t q0[RB][4];
        float s0[RB];
        int n0[RB];
        load_queries<KB, RB>(a, rows, rows.r0, head, lane, q0, s0, n0);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) q_s[wave / kw][rb][ks][lane] = __builtin_bit_cast(uint4, q0[rb][ks]);
            scale_s[wave / kw][rb][lane] = s0[rb];
        }
    }
    if constexpr (KB != 8) build_pair_table<KB, KC>(smem, a.klut, tid, 64 * W);
    if constexpr (VB != 8 && !SHARE) build_pair_table<VB, VC>(smem + V_TABLE, a.vlut, tid, 64 * W);
    const uint32_t k_copy = 4 * (lane & (KC - 1)), v_copy = 4 * (lane & (VC - 1));
    __syncthreads();   // the tables and the queries
    half8_t qf[RB][4];
    float scale[RB], m[RB], l[RB];
    int seen[RB];
    float4_t o[RB][2][4];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) qf[rb][ks] = __builtin_bit_cast(half8_t, q_s[wave / kw][rb][ks][lane]);
        scale[rb] = scale_s[wave / kw][rb][lane];
        seen[rb] = row_limit(a, rows, min(rows.r0 + 16 * rb + n16, max(rows.n_rows - 1, 0)));
#pragma unroll
        for (int e = 0; e < 8; ++e) o[rb][e >> 2][e & 3] = float4_t{0.f, 0.f, 0.f, 0.f};
        m[rb] = -INFINITY;
        l[rb] = 0.0f;
    }

    // one tile; masked_t: some row does not see all of it, or its page is none
    auto do_tile = [&](auto masked_t, int tile, bool real, int page_next) {
        constexpr bool MASKED = decltype(masked_t)::value;
        const int first = 64 * tile + 16 * kq;     // this lane's tokens: first + 4 u + i
        const int next = min(tile + 1, t_end - 1);
        // ---- logits
        float4_t s[RB][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            half8_t kf[4];
            if constexpr (KB == 8) {
                const _Float16 d = __builtin_bit_cast(_Float16, (uint16_t)kn[u]);
                const half2_t dd = {d, d};
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) kf[ks] = join(int8x4_times(kw_[u][2 * ks], dd, dd), int8x4_times(kw_[u][2 * ks + 1], dd, dd));
            } else {
                const uint32_t tail = group_tail<KB>(kw_[u]);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) kf[ks] = join(group_quad<KB, KC>(kw_[u], tail, smem, k_copy, 2 * ks), group_quad<KB, KC>(kw_[u], tail, smem, k_copy, 2 * ks + 1));
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                s[rb][u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) s[rb][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[ks], qf[rb][ks], s[rb][u], 0, 0, 0);
            }
        }
        float knf[16];
        if constexpr (KB != 8) {
#pragma unroll
            for (int e = 0; e < 16; ++e) knf[e] = half_of(kn[e >> 1], e & 1);
        }
        load_k(next, page_next);
        __builtin_amdgcn_sched_barrier(0);   // the scheduler otherwise has all look-ups in flight and spills
        // ---- softmax
        half8_t pf[RB][2];
        float m_new[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
            m_new[rb] = logits_max<KB, MASKED>(s[rb], [&](int e) { return knf[e]; }, real ? seen[rb] - first : 0, scale[rb], m[rb]);
        move_max<RB>(m_new, m, l, o);
        auto all_weights = [&](auto fast_t) __attribute__((always_inline)) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
                weights<VB, decltype(fast_t)::value>(s[rb], [&](int e) { return half_of(vn[e >> 1], e & 1); }, real ? seen[rb] - first : 0, m[rb], scale[rb],
                                                     l[rb], pf[rb]);
        };
        if constexpr (MASKED) all_weights(std::false_type{});
        else if (far_logits<RB>(m)) all_weights(std::false_type{});
        else all_weights(std::true_type{});
        __builtin_amdgcn_sched_barrier(0);
        // ---- values
#pragma unroll
        for (int blk = 0; blk < 4; ++blk) {
            half8_t vf[2][2];   // [dims' half][step]
            if constexpr (VB == 8) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t d[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) d[j] = vn[8 * (2 * hf + (blk >> 1)) + j];
                    // In a tile that some row does not see whole, a scale that is no finite number (of rows that held none, or of a
                    // place that nothing was written to) must not reach the rows that do not see its token, and 0 times
                    // it would: it is replaced, and the rows that see it are marked.
                    if constexpr (MASKED) {
                        uint32_t bad = 0;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const bool lo = (d[j] & 0x7C00u) == 0x7C00u, hi = (d[j] & 0x7C000000u) == 0x7C000000u;
                            bad |= (lo ? 1u << (2 * j) : 0u) | (hi ? 2u << (2 * j) : 0u);
                            d[j] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
                        }
                        if (__builtin_amdgcn_ballot_w64(bad != 0u) != 0ull) {
#pragma unroll
                            for (int rb = 0; rb < RB; ++rb) {
                                const int sees = real ? min(max(seen[rb] - first, 0), 16) : 0;
                                const float mark = (bad & ((1u << sees) - 1u)) ? 1.0f : 0.0f;
                                if (over_row_max(mark) > 0.0f) o[rb][hf][blk] = float4_t{NAN, NAN, NAN, NAN};
                            }
                        }
                    }
                    uint2 q4[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t d02 = __builtin_amdgcn_perm(d[2 * u + 1], d[2 * u], 0x05040100u), d13 = __builtin_amdgcn_perm(d[2 * u + 1], d[2 * u], 0x07060302u);
                        q4[u] = int8x4_times(vw[blk][4 * hf + u], __builtin_bit_cast(half2_t, d02), __builtin_bit_cast(half2_t, d13));
                    }
                    vf[hf][0] = join(q4[0], q4[1]);
                    vf[hf][1] = join(q4[2], q4[3]);
                }
            } else {
                const uint32_t tail = group_tail<VB>(vw[blk]);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int st = 0; st < 2; ++st)
                        vf[hf][st] = join(group_quad<VB, VC>(vw[blk], tail, smem + V_TABLE, v_copy, 4 * st + hf), group_quad<VB, VC>(vw[blk], tail, smem + V_TABLE, v_copy, 4 * st + 2 + hf));
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int st = 0; st < 2; ++st)
                        o[rb][hf][blk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[hf][st], pf[rb][st], o[rb][hf][blk], 0, 0, 0);
        }
        load_v(next, page_next);
        __builtin_amdgcn_sched_barrier(0);
    };
    if (t_begin < t_end) {
        const int whole = min(max(least >> 6, t_begin), t_end);     // tiles that every row sees
        int tile = t_begin;
#pragma unroll 1
        for (; tile < whole && is_page(page); ++tile) {
            const int after = page_of(min(tile + 2, t_end - 1));
            do_tile(std::false_type{}, tile, true, page_next);
            page = page_next;
            page_next = after;
        }
#pragma unroll 1
        for (; tile < t_end; ++tile) {
            const int after = page_of(min(tile + 2, t_end - 1));
            do_tile(std::true_type{}, tile, is_page(page), page_next);
            page = page_next;
            page_next = after;
        }
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) l[rb] = over_row_sum(l[rb]);

    // ---- the wavefronts of a row block join, in halves: the upper ones leave their results in LDS, the lower ones take them in
    float *joint = reinterpret_cast<float *>(smem);
    for (int step = kw >> 1; step >= 1; step >>= 1) {
        __syncthreads();
        if (part >= step && part < 2 * step) {
            float *to = joint + ((wave / kw) * step + part - step) * join_floats(RB);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
                for (int e = 0; e < 32; ++e) to[(34 * rb + e) * 64 + lane] = o[rb][e >> 4][(e >> 2) & 3][e & 3];
                to[(34 * rb + 32) * 64 + lane] = m[rb];
                to[(34 * rb + 33) * 64 + lane] = l[rb];
            }
        }
        __syncthreads();
        if (part < step) {
            const float *from = joint + ((wave / kw) * step + part) * join_floats(RB);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const float m2 = from[(34 * rb + 32) * 64 + lane], l2 = from[(34 * rb + 33) * 64 + lane];
                const float top = fmaxf(m[rb], m2), off = top == -INFINITY ? 0.0f : top;
                const float f1 = __builtin_amdgcn_exp2f(m[rb] - off), f2 = __builtin_amdgcn_exp2f(m2 - off);
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const float x = o[rb][e >> 4][(e >> 2) & 3][e & 3];
                    o[rb][e >> 4][(e >> 2) & 3][e & 3] = fmaf(from[(34 * rb + e) * 64 + lane], f2, x * f1);
                }
                l[rb] = fmaf(l2, f2, l[rb] * f1);
                m[rb] = top;
            }
        }
    }
    if (part == 0 && rows.active) leave_rows<RB>(a, rows, rows.r0, head, split, lane, o, m, l);
}

// ---- many rows: a workgroup decodes a tile once for all of its wavefronts ------------------------------------
// 16 RB rows per wavefront (RB 1: 64 rows, else 128 or 256 per workgroup).  Every tile's operands are decoded by the wavefronts in
// turns of a 16-token unit of K or a 16-dim block of V and lie in LDS as the matrix instructions take them (a lane's 16 bytes next
// to its neighbour's), ahead of their use, behind one barrier per tile: K's two tiles and V's one, so that the next tile's
// logits are multiplied while this one's weights are worked out (chunk of 2048 at 32K: 3.07 -> 1.33 ms with the shared decoding,
// wider loads and this order).
// copies of a decode table: a workgroup looks each pair up once, and two of its size share a CU's LDS
__host__ __device__ constexpr int chunk_copies(int bits) { return bits == 4 ? 4 : 16; }
template <int KB, int VB, int W, int RB>
__global__ __launch_bounds__(64 * W, 2) void k_paged_chunk(PagedAttnArgs a) {
    constexpr int TILE = 16 * RB * W, KC = chunk_copies(KB), VC = chunk_copies(VB);
    constexpr int KBLOCK = KB == 8 ? TQ_ROWS_PER_BLOCK * 136 : block_bytes(KB), VBLOCK = VB == 8 ? TQ_ROWS_PER_BLOCK * 136 : block_bytes(VB);
    __shared__ __attribute__((aligned(16))) uint4 kf_s[2][4][4][64], vf_s[2][4][4][64];   // [buffer][unit][step], [block][half of the dims, step]
    __shared__ __attribute__((aligned(16))) char lut_s[pair_table_bytes(KB, KC) + pair_table_bytes(VB, VC) + 16];
    __shared__ __attribute__((aligned(16))) float kn_s[2][64], vn_s[2][64];
    __shared__ uint32_t bad_s[2][16];     // 8-bit V: [32-dim block][quarter]: tokens whose scale is no finite number
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, kq = lane >> 4;
    const PagedTurn p = paged_turn(a);
    const int head = p.head, split = p.split;
    int b;
    const PagedBlock rows = paged_block(a, p.turn, TILE, split, b);
    if (!rows.active) return;    // all of the workgroup
    const int first_row = rows.r0 + 16 * RB * wave;
    const bool computes = first_row < rows.n_rows;
    const int t_begin = split * a.split_tiles;
    const int t_end = min((row_limit(a, rows, min(rows.r0 + TILE, rows.n_rows) - 1) + 63) >> 6, t_begin + a.split_tiles);
    // of this wavefront's rows: the tiles that all of them see, and those that any does
    const int whole = computes ? min(t_end, row_limit(a, rows, first_row) >> 6) : 0;
    const int upto = computes ? min(t_end, (row_limit(a, rows, min(first_row + 16 * RB, rows.n_rows) - 1) + 63) >> 6) : 0;

    // ---- decoding: wavefronts 0 .. 3 have K units, the last four (W = 4: the same ones) V blocks
    constexpr bool BOTH = W == 4;
    const int32_t *table = a.r.p.block_table + (int64_t)__builtin_amdgcn_readfirstlane(b) * a.r.p.table_stride;
    auto page_of = [&](int tile) { return scalar_entry(table, __builtin_amdgcn_readfirstlane(min(tile, t_end - 1) >> 1)); };
    auto is_page = [&](int page) { return page >= 0 && page < a.r.p.n_pages; };
    const bool does_k = BOTH || wave < 4, does_v = BOTH || wave >= 4;
    const int unit = wave & 3, k_token = 16 * (n16 >> 2) + 4 * unit + (n16 & 3), v_row = 16 * unit + n16;
    uint32_t kw[KB == 8 ? 8 : KB], vw[VB == 8 ? 8 : VB], vsc[VB == 8 ? 16 : 1];
    uint16_t kn = 0, vn = 0;
    auto request_k = [&](int tile, int page, auto &kw, uint16_t &kn) __attribute__((always_inline)) {
        const uint8_t *kb = a.k + ((int64_t)(is_page(page) ? page : 0) * a.r.p.n_kv_heads + head) * KBLOCK;
        const int base = 64 * (min(tile, t_end - 1) & 1);
        if (does_k) {
            const int row = base + k_token;
            if constexpr (KB == 8) {
                const uint4 lo = *reinterpret_cast<const uint4 *>(kb + (2 * kq) * 2048 + row * 16), hi = *reinterpret_cast<const uint4 *>(kb + (2 * kq + 1) * 2048 + row * 16);
                kw[0] = lo.x; kw[1] = lo.y; kw[2] = lo.z; kw[3] = lo.w;
                kw[4] = hi.x; kw[5] = hi.y; kw[6] = hi.z; kw[7] = hi.w;
                kn = reinterpret_cast<const uint16_t *>(kb + 8 * 2048)[4 * row + kq];
            } else {
#pragma unroll
                for (int j = 0; j < KB; ++j) kw[j] = *reinterpret_cast<const uint32_t *>(kb + j * 2048 + row * 16 + kq * 4);
                kn = reinterpret_cast<const uint16_t *>(kb + block_code_bytes(KB))[row];
            }
        }
    };
    auto request_v = [&](int tile, int page) __attribute__((always_inline)) {
        const uint8_t *vb = a.v + ((int64_t)(is_page(page) ? page : 0) * a.r.p.n_kv_heads + head) * VBLOCK;
        const int base = 64 * (min(tile, t_end - 1) & 1);
        if (does_v) {
            const int row = base + v_row;
            if constexpr (VB == 8) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(vb + (4 * hf + kq) * 2048 + row * 16);
                    vw[4 * hf] = w.x; vw[4 * hf + 1] = w.y; vw[4 * hf + 2] = w.z; vw[4 * hf + 3] = w.w;
                    const uint4 *d = reinterpret_cast<const uint4 *>(vb + 8 * 2048 + 2 * ((4 * (base >> 6) + 2 * hf + (unit >> 1)) * 64 + 16 * kq));
                    const uint4 d0 = d[0], d1 = d[1];
                    vsc[8 * hf] = d0.x; vsc[8 * hf + 1] = d0.y; vsc[8 * hf + 2] = d0.z; vsc[8 * hf + 3] = d0.w;
                    vsc[8 * hf + 4] = d1.x; vsc[8 * hf + 5] = d1.y; vsc[8 * hf + 6] = d1.z; vsc[8 * hf + 7] = d1.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < VB; ++j) vw[j] = *reinterpret_cast<const uint32_t *>(vb + j * 2048 + row * 16 + kq * 4);
                vn = reinterpret_cast<const uint16_t *>(vb + block_code_bytes(VB))[row];   // of token 16 unit + n16
            }
        }
    };
    const char *vlut = lut_s + (a.share ? 0 : pair_table_bytes(KB, KC));
    const uint32_t k_copy = 4 * (lane & (KC - 1)), v_copy = 4 * (lane & (VC - 1));
    auto decode_k = [&](int buf) __attribute__((always_inline)) {
        if (does_k) {
            if constexpr (KB == 8) {
                const _Float16 d = __builtin_bit_cast(_Float16, kn);
                const half2_t dd = {d, d};
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    kf_s[buf][unit][ks][lane] = __builtin_bit_cast(uint4, join(int8x4_times(kw[2 * ks], dd, dd), int8x4_times(kw[2 * ks + 1], dd, dd)));
            } else {
                const uint32_t tail = group_tail<KB>(kw);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    kf_s[buf][unit][ks][lane] = make_uint4(group_pair<KB, KC>(kw, tail, lut_s, k_copy, 4 * ks), group_pair<KB, KC>(kw, tail, lut_s, k_copy, 4 * ks + 1),
                                                           group_pair<KB, KC>(kw, tail, lut_s, k_copy, 4 * ks + 2), group_pair<KB, KC>(kw, tail, lut_s, k_copy, 4 * ks + 3));
                if (kq == 0) kn_s[buf][k_token] = __half2float(__ushort_as_half(kn));
            }
        }
    };
    auto decode_v = [&](int buf) __attribute__((always_inline)) {
        if (does_v) {
            if constexpr (VB == 8) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    // a scale that is no finite number would reach rows that do not see its token, as 0 times it: it is replaced, and the
                    // rows that see it are marked
                    uint32_t d[8], bad = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        d[j] = vsc[8 * hf + j];
                        const bool lo = (d[j] & 0x7C00u) == 0x7C00u, hi = (d[j] & 0x7C000000u) == 0x7C000000u;
                        bad |= (lo ? 1u << (2 * j) : 0u) | (hi ? 2u << (2 * j) : 0u);
                        d[j] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
                    }
                    if ((unit & 1) == 0 && n16 == 0) bad_s[buf][4 * (2 * hf + (unit >> 1)) + kq] = bad;
                    uint2 q4[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t d02 = __builtin_amdgcn_perm(d[2 * u + 1], d[2 * u], 0x05040100u), d13 = __builtin_amdgcn_perm(d[2 * u + 1], d[2 * u], 0x07060302u);
                        q4[u] = int8x4_times(vw[4 * hf + u], __builtin_bit_cast(half2_t, d02), __builtin_bit_cast(half2_t, d13));
                    }
                    vf_s[buf][unit][2 * hf][lane] = __builtin_bit_cast(uint4, join(q4[0], q4[1]));
                    vf_s[buf][unit][2 * hf + 1][lane] = __builtin_bit_cast(uint4, join(q4[2], q4[3]));
                }
            } else {
                const uint32_t tail = group_tail<VB>(vw);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        const int p0 = 2 * (4 * st + hf);   // quads 4 st + hf and two further
                        vf_s[buf][unit][2 * hf + st][lane] = make_uint4(group_pair<VB, VC>(vw, tail, vlut, v_copy, p0), group_pair<VB, VC>(vw, tail, vlut, v_copy, p0 + 1),
                                                                        group_pair<VB, VC>(vw, tail, vlut, v_copy, p0 + 4), group_pair<VB, VC>(vw, tail, vlut, v_copy, p0 + 5));
                    }
                if (kq == 0) vn_s[buf][v_row] = __half2float(__ushort_as_half(vn));
            }
        }
    };

    uint32_t kw1[KB == 8 ? 8 : KB];    // the second tile's K, requested with the first
    uint16_t kn1 = 0;
    int page = 0, page1 = 0, page2 = 0;    // of this tile and the next two
    if (t_begin < t_end) {
        page = page_of(t_begin);
        page1 = page_of(t_begin + 1);
        page2 = page_of(t_begin + 2);
        request_k(t_begin, page, kw, kn);
        request_v(t_begin, page);
        request_k(t_begin + 1, page1, kw1, kn1);
    }
    if constexpr (KB != 8) build_pair_table<KB, KC>(lut_s, a.klut, tid, 64 * W);
    if constexpr (VB != 8)
        if (!a.share) build_pair_table<VB, VC>(lut_s + pair_table_bytes(KB, KC), a.vlut, tid, 64 * W);
    half8_t qf[RB][4];
    float scale[RB], m[RB], l[RB];
    int seen[RB];
    load_queries<KB, RB>(a, rows, first_row, head, lane, qf, scale, seen);
    float4_t o[RB][2][4];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[rb][e >> 2][e & 3] = float4_t{0.f, 0.f, 0.f, 0.f};
        m[rb] = -INFINITY;
        l[rb] = 0.0f;
    }
    __syncthreads();   // the tables
    // The logits of the next tile are multiplied while this one's weights are worked out, and the next one's maximum is found while
    // this one's values are multiplied: K is decoded two tiles ahead, V one.
    if (t_begin < t_end) {
        decode_k(t_begin & 1);
        decode_v(t_begin & 1);
        request_v(t_begin + 1, page1);
#pragma unroll
        for (int j = 0; j < (int)(sizeof(kw) / sizeof(kw[0])); ++j) kw[j] = kw1[j];
        kn = kn1;
        decode_k((t_begin + 1) & 1);
        request_k(t_begin + 2, page2, kw, kn);
    }
    __syncthreads();

    auto logits = [&](int tile, float4_t (&s)[RB][4]) __attribute__((always_inline)) {
        const int buf = tile & 1;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) s[rb][u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                const half8_t kf = __builtin_bit_cast(half8_t, kf_s[buf][u][ks][lane]);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) s[rb][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[rb][ks], s[rb][u], 0, 0, 0);
            }
        }
    };
    float m_new[RB];
    auto maxima = [&](auto fast_t, int tile, bool real, float4_t (&s)[RB][4]) __attribute__((always_inline)) {
        constexpr bool FAST = decltype(fast_t)::value;
        const int buf = tile & 1, first = 64 * tile + 16 * kq;     // this lane's tokens: first + 4 u + i
        float4_t knf[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if constexpr (KB != 8) knf[u] = *reinterpret_cast<const float4_t *>(&kn_s[buf][16 * kq + 4 * u]);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
            m_new[rb] = logits_max<KB, !FAST>(s[rb], [&](int e) { return knf[e >> 2][e & 3]; }, real ? seen[rb] - first : 0, scale[rb], m[rb]);
    };
    auto values = [&](int tile, const half8_t (&pf)[RB][2]) __attribute__((always_inline)) {
        const int buf = tile & 1;
#pragma unroll
        for (int blk = 0; blk < 4; ++blk)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    const half8_t vf = __builtin_bit_cast(half8_t, vf_s[buf][blk][2 * hf + st][lane]);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) o[rb][hf][blk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[rb][st], o[rb][hf][blk], 0, 0, 0);
                }
    };
    auto all_weights = [&](auto fast_t, int tile, bool real, const float4_t (&s)[RB][4], half8_t (&pf)[RB][2]) __attribute__((always_inline)) {
        constexpr bool FAST = decltype(fast_t)::value;
        const int buf = tile & 1, first = 64 * tile + 16 * kq;
        float4_t vnf[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if constexpr (VB != 8) vnf[u] = *reinterpret_cast<const float4_t *>(&vn_s[buf][16 * kq + 4 * u]);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
            weights<VB, FAST>(s[rb], [&](int e) { return vnf[e >> 2][e & 3]; }, real ? seen[rb] - first : 0, m[rb], scale[rb], l[rb], pf[rb]);
        if constexpr (VB == 8) {
            const uint32_t bad = bad_s[buf][n16];
            if (__builtin_amdgcn_ballot_w64(bad != 0u) != 0ull) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t mine = bad_s[buf][4 * j + kq];
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        const int sees = real ? min(max(seen[rb] - first, 0), 16) : 0;
                        if (over_row_max((mine & ((1u << sees) - 1u)) ? 1.0f : 0.0f) > 0.0f)
                            o[rb][j >> 1][2 * (j & 1)] = o[rb][j >> 1][2 * (j & 1) + 1] = float4_t{NAN, NAN, NAN, NAN};
                    }
                }
            }
        }
    };
    auto decode_next = [&](int tile) __attribute__((always_inline)) {
        decode_v((tile + 1) & 1);
        decode_k(tile & 1);
        page = page1;
        page1 = page2;
        page2 = page_of(tile + 3);
        request_v(tile + 2, page1);
        request_k(tile + 3, page2, kw, kn);
        __syncthreads();
    };
    float4_t s[RB][4];     // this tile's logits, with norms and masks
    if (upto > t_begin) {
        logits(t_begin, s);
        maxima(std::false_type{}, t_begin, is_page(page), s);
    }
    __syncthreads();
    int tile = t_begin;
#pragma unroll 1
    for (; tile + 1 < whole && is_page(page) && is_page(page1) && !far_logits<RB>(m_new); ++tile) {
        move_max<RB>(m_new, m, l, o);
        float4_t next[RB][4];
        half8_t pf[RB][2];
        logits(tile + 1, next);
        all_weights(std::true_type{}, tile, true, s, pf);
        values(tile, pf);
        maxima(std::true_type{}, tile + 1, true, next);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int u = 0; u < 4; ++u) s[rb][u] = next[rb][u];
        decode_next(tile);
    }
#pragma unroll 1
    for (; tile < t_end; ++tile) {
        if (tile < upto) {
            half8_t pf[RB][2];
            move_max<RB>(m_new, m, l, o);
            all_weights(std::false_type{}, tile, is_page(page), s, pf);
            values(tile, pf);
            logits(tile + 1, s);
            maxima(std::false_type{}, tile + 1, is_page(page1), s);
        }
        decode_next(tile);
    }
    if (!computes) return;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) l[rb] = over_row_sum(l[rb]);
    leave_rows<RB>(a, rows, first_row, head, split, lane, o, m, l);
}

}  // namespace tqpaged
