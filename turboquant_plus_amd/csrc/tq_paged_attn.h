// Attention of new tokens over a paged cache of packed rows: k_paged_attn and k_paged_merge.
//
// A wavefront takes 16 RB rows (a row: one new token under one query head of a KV head) and walks tiles of 64 positions; it
// needs nobody else until its end.  Codes become fp16 operands of 16x16x32 matrix instructions in its own registers, through
// decode tables in LDS, and each operand serves the RB row blocks: what a tile costs to decode is paid once per 16 RB rows.
//   S^T = K Q^T.  A = K: lane (m = lane % 16, kq = lane / 16) holds dims 32 kq .. 32 kq + 31 of a token, which are BITS dwords of its
//     row (one pair group), 8 of them per step; B = Q likewise, so Q is loaded, rotated and scaled in the layout in which it is
//     used.  Row m of unit u is token 16 (m / 4) + 4 u + m % 4 of the tile: the result then gives lane (n, kq) the logits of
//     row n for the tokens 16 kq + 4 u + i.
//   softmax: running maximum and sum per lane and row block in 32 bits; the maximum goes over the four lanes of a row.
//   O^T = V^T P^T.  B = P: the lane's own 16 weights, rounded to fp16 with the tokens' norms in them (|error| <= 2^-11 of a weight, of
//     either sign, so a sum of them is as good as its rounding to 16 bits); A = V: rows are dims, lane (m, kq) takes the pair group kq =
//     tokens 16 kq .. 16 kq + 15 of dims m and 64 + m of a 16-row block.  No exchange between lanes anywhere in the loop but the
//     maximum.
// The result of a lane is 32 dims of a row, and the transposed rotation of V is a butterfly of five stages in registers and two
// across lanes.  `kw` wavefronts of a workgroup share the positions of one row block and join through LDS at the end;
// n_splits workgroups share them where rows are few, through partial results in memory (32 bits) and k_paged_merge.
#pragma once
#include "tq_device.h"
#include "tq_paged.h"

namespace tqpaged {

using namespace tqd;

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

constexpr float RSQRT128 = 0.08838834764831845f;

struct PagedAttnArgs {
    PagedRows r;
    const void *q;
    void *out;
    int64_t q_token, q_head;
    int bf16, causal, max_context, max_new;
    int group;                   // query heads per KV head
    FastDiv group_div, heads_div;
    const uint8_t *k, *v;
    const uint32_t *klut, *vlut; // pair tables of value_scale times the codebook
    const float *ks1, *ks2, *vs1, *vs2;
    float scale;                 // logits' scale * log2(e) / value_scale of K
    float v_unscale;             // 1 / value_scale of V
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
// 2 and 3 bits: four values per entry (8 bytes), indexed by two neighbouring pair codes; 4 bits: two values per entry
__host__ __device__ constexpr int table_bytes(int bits) { return bits == 8 ? 0 : bits == 4 ? 1024 : 8 << (4 * bits); }
template <int BITS> __device__ __forceinline__ void build_table(char *dst, const uint32_t *pairs, int tid, int threads) {
    if constexpr (BITS == 4) {
        for (int e = tid; e < 256; e += threads) reinterpret_cast<uint32_t *>(dst)[e] = pairs[e];
    } else {
        constexpr int NP = 1 << (2 * BITS);
        for (int e = tid; e < NP * NP; e += threads) reinterpret_cast<uint2 *>(dst)[e] = make_uint2(pairs[e & (NP - 1)], pairs[e / NP]);
    }
}
template <int BITS> __device__ __forceinline__ uint32_t group_tail(const uint32_t (&w)[BITS]) {
    if constexpr (BITS == 3) return (w[0] >> 24) | ((w[1] >> 24) << 8) | ((w[2] >> 24) << 16);
    else return 0u;
}
// the four values of quad Q = 0 .. 7 of a pair group
template <int BITS> __device__ __forceinline__ uint2 group_quad(const uint32_t (&w)[BITS], uint32_t tail, const char *lut, int Q) {
    if constexpr (BITS == 4) {
        const uint32_t x = w[Q >> 1];
        return make_uint2(*reinterpret_cast<const uint32_t *>(lut + field_offset<2>(x, 16 * (Q & 1), 8)),
                          *reinterpret_cast<const uint32_t *>(lut + field_offset<2>(x, 16 * (Q & 1) + 8, 8)));
    } else if constexpr (BITS == 2) {
        return *reinterpret_cast<const uint2 *>(lut + field_offset<3>(w[Q >> 2], 8 * (Q & 3), 8));
    } else {
        return *reinterpret_cast<const uint2 *>(lut + (Q < 6 ? field_offset<3>(w[Q >> 1], 12 * (Q & 1), 12) : field_offset<3>(tail, 12 * (Q - 6), 12)));
    }
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

__host__ __device__ constexpr int paged_waves(int rb) { return rb == 1 ? 8 : 4; }
// floats that a wavefront leaves behind for another one to join: 32 RB sums, RB maxima and sums of weights per lane
__host__ __device__ constexpr int join_floats(int rb) { return 64 * 34 * rb; }
__host__ __device__ constexpr int paged_lds(int kb, int vb, int rb, bool share) {
    const int tables = table_bytes(kb) + (share ? 0 : table_bytes(vb)), join = paged_waves(rb) / 2 * join_floats(rb) * 4;
    return tables > join ? tables : join;
}

// KB, VB: code widths, 8 for q8_0-style rows; RB: blocks of 16 rows per wavefront; SHARE: one table for K and V
template <int KB, int VB, int RB, bool SHARE>
__global__ __launch_bounds__(64 * paged_waves(RB)) void k_paged_attn(PagedAttnArgs a) {
    constexpr int W = paged_waves(RB), TILE = 16 * RB;
    constexpr int KBLOCK = KB == 8 ? TQ_ROWS_PER_BLOCK * 136 : block_bytes(KB), VBLOCK = VB == 8 ? TQ_ROWS_PER_BLOCK * 136 : block_bytes(VB);
    __shared__ __attribute__((aligned(16))) char smem[paged_lds(KB, VB, RB, SHARE)];
    const char *klut = smem, *vlut = SHARE ? smem : smem + table_bytes(KB);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, kq = lane >> 4;
    // neighbouring workgroups have the KV heads of the same rows: with eight of them each die keeps to one head's pages
    const uint32_t rest = a.heads_div.div(blockIdx.x);
    const int head = (int)(blockIdx.x - rest * a.heads_div.d);
    const int split = a.n_splits == 1 ? 0 : (int)(rest % (uint32_t)a.n_splits);
    const int turn = a.n_splits == 1 ? (int)rest : (int)(rest / (uint32_t)a.n_splits);
    const int kw = a.kw, part = wave & (kw - 1);
    const int item = turn * (W / kw) + wave / kw;
    int b = 0, nth = 0;
    const bool some = paged_item(a.r, item, [&](int s) { return (min(paged_seq(a.r, s).n, a.max_new) * a.group + TILE - 1) / TILE; }, b, nth);
    PagedSeq seq{0, 0, 0};
    PagedSpan span{0, 0};
    if (some) {
        seq = paged_seq(a.r, b);
        span = paged_span(a, seq);
    }
    const int n_rows = min(seq.n, a.max_new) * a.group, r0 = nth * TILE;
    const bool active = some && (split < span.splits || split == 0);
    // positions that the block's last and first rows see
    auto limit = [&](int r) {
        const int t = (int)a.group_div.div((uint32_t)r), seen = a.causal ? span.ctx - seq.n + t + 1 : span.ctx;
        return seen < 0 ? 0 : seen;
    };
    int t_begin = 0, t_end = 0, least = 0;
    if (active) {
        least = limit(r0);
        t_begin = split * a.split_tiles;
        t_end = min((limit(min(r0 + TILE, n_rows) - 1) + 63) >> 6, t_begin + a.split_tiles);
        const int each = (max(t_end - t_begin, 0) + kw - 1) / kw;
        t_begin += part * each;
        t_end = min(t_end, t_begin + each);
    }
    if constexpr (KB != 8) build_table<KB>(smem, a.klut, tid, 64 * W);
    if constexpr (VB != 8 && !SHARE) build_table<VB>(smem + table_bytes(KB), a.vlut, tid, 64 * W);

    // queries: 32 values of row n16 of each block, rotated as K's rows are, as fp16 of their size up to a power of two
    half8_t qf[RB][4];
    float scale[RB];   // of the logits, with that power of two
    int seen[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int r = min(r0 + 16 * rb + n16, max(n_rows - 1, 0));   // rows past the last one repeat it
        const int t = (int)a.group_div.div((uint32_t)r), g = r - t * a.group;
        seen[rb] = limit(r);
        float x[32];
        const int64_t at = (seq.row0 + t) * a.q_token + (int64_t)(head * a.group + g) * a.q_head + 32 * kq;
        if (active) {
            const uint4 *p = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(a.q) + at);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint4 u = p[c];
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[8 * c + 2 * j] = a.bf16 ? __uint_as_float(w[j] << 16) : half_of(w[j], 0);
                    x[8 * c + 2 * j + 1] = a.bf16 ? __uint_as_float(w[j] & 0xFFFF0000u) : half_of(w[j], 1);
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = 0.0f;
        }
        if constexpr (KB != 8) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                const float4 s = *reinterpret_cast<const float4 *>(a.ks1 + 32 * kq + e);
                x[e] *= s.x; x[e + 1] *= s.y; x[e + 2] *= s.z; x[e + 3] *= s.w;
            }
            butterfly32x4(x, lane);
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                const float4 s = *reinterpret_cast<const float4 *>(a.ks2 + 32 * kq + e);
                x[e] *= s.x * RSQRT128; x[e + 1] *= s.y * RSQRT128; x[e + 2] *= s.z * RSQRT128; x[e + 3] *= s.w * RSQRT128;
            }
        }
        float most = 0.0f;
#pragma unroll
        for (int e = 0; e < 32; ++e) most = fmaxf(most, fabsf(x[e]));
        most = over_row_max(most);
        int ex = most > 0.0f && most < INFINITY ? __builtin_amdgcn_frexp_expf(most) : 0;
        ex = min(max(ex, -100), 120);
        scale[rb] = __builtin_amdgcn_ldexpf(a.scale, ex);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // int8 rows hand their values over in the order 0, 2, 1, 3
                const int from = KB == 8 ? (e & 4) | ((e & 1) << 1) | ((e >> 1) & 1) : e;
                qf[rb][ks][e] = (_Float16)__builtin_amdgcn_ldexpf(x[8 * ks + from], -ex);
            }
    }

    float4_t o[RB][2][4];
    float m[RB], l[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[rb][e >> 2][e & 3] = float4_t{0.f, 0.f, 0.f, 0.f};
        m[rb] = -INFINITY;
        l[rb] = 0.0f;
    }
    __syncthreads();   // the tables

    const int32_t *table = a.r.p.block_table + (int64_t)b * a.r.p.table_stride;
    auto page_of = [&](int tile) { return __builtin_amdgcn_readfirstlane(table[tile >> 1]); };
    int page = t_begin < t_end ? page_of(t_begin) : 0;
#pragma unroll 1
    for (int tile = t_begin; tile < t_end; ++tile) {
        const bool real = page >= 0 && page < a.r.p.n_pages;
        const int64_t at = (int64_t)(real ? page : 0) * a.r.p.n_kv_heads + head;
        const uint8_t *kb = a.k + at * KBLOCK, *vb = a.v + at * VBLOCK;
        const int half = tile & 1, first = 64 * tile + 16 * kq;     // this lane's tokens: first + 4 u + i
        if (tile + 1 < t_end) page = page_of(tile + 1);
        const bool masked = !real || 64 * tile + 64 > least;   // some row does not see all of the tile
        // ---- logits
        float4_t s[RB][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int row = 64 * half + 16 * (n16 >> 2) + 4 * u + (n16 & 3);
            half8_t kf[4];
            if constexpr (KB == 8) {
                const uint4 lo = *reinterpret_cast<const uint4 *>(kb + (2 * kq) * 2048 + row * 16);
                const uint4 hi = *reinterpret_cast<const uint4 *>(kb + (2 * kq + 1) * 2048 + row * 16);
                const _Float16 d = reinterpret_cast<const _Float16 *>(kb + 8 * 2048)[4 * row + kq];
                const half2_t dd = {d, d};
                kf[0] = join(int8x4_times(lo.x, dd, dd), int8x4_times(lo.y, dd, dd));
                kf[1] = join(int8x4_times(lo.z, dd, dd), int8x4_times(lo.w, dd, dd));
                kf[2] = join(int8x4_times(hi.x, dd, dd), int8x4_times(hi.y, dd, dd));
                kf[3] = join(int8x4_times(hi.z, dd, dd), int8x4_times(hi.w, dd, dd));
            } else {
                uint32_t w[KB];
#pragma unroll
                for (int j = 0; j < KB; ++j) w[j] = *reinterpret_cast<const uint32_t *>(kb + j * 2048 + row * 16 + kq * 4);
                const uint32_t tail = group_tail<KB>(w);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) kf[ks] = join(group_quad<KB>(w, tail, klut, 2 * ks), group_quad<KB>(w, tail, klut, 2 * ks + 1));
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                s[rb][u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) s[rb][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[ks], qf[rb][ks], s[rb][u], 0, 0, 0);
            }
        }
        // the tokens' norms; 0 where the page is none, so that nothing it may hold gets in
        uint32_t kn[8], vn[8];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if constexpr (KB != 8) {
                const uint4 n = *reinterpret_cast<const uint4 *>(kb + block_code_bytes(KB) + 2 * (64 * half + 16 * kq) + 16 * c);
                kn[4 * c] = n.x; kn[4 * c + 1] = n.y; kn[4 * c + 2] = n.z; kn[4 * c + 3] = n.w;
            }
            if constexpr (VB != 8) {
                const uint4 n = *reinterpret_cast<const uint4 *>(vb + block_code_bytes(VB) + 2 * (64 * half + 16 * kq) + 16 * c);
                vn[4 * c] = n.x; vn[4 * c + 1] = n.y; vn[4 * c + 2] = n.z; vn[4 * c + 3] = n.w;
            }
        }
        // ---- softmax
        half8_t pf[RB][2];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            float most = -INFINITY;
            const int sees = real ? seen[rb] - first : 0;    // this lane's tokens 0 .. sees - 1 count
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = s[rb][u][i];
                    if constexpr (KB != 8) v *= half_of(kn[2 * u + (i >> 1)], i & 1);
                    if (masked) v = 4 * u + i < sees ? v : -INFINITY;
                    s[rb][u][i] = v;
                    most = fmaxf(most, v);
                }
            const float m_new = fmaxf(m[rb], over_row_max(most) * scale[rb]);
            if (__builtin_amdgcn_ballot_w64(m_new != m[rb]) != 0ull) {
                const float shrink = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[rb] - m_new);
                l[rb] *= shrink;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[rb][e >> 2][e & 3] *= shrink;
                m[rb] = m_new;
            }
            float off = m[rb] == -INFINITY ? 0.0f : m[rb], by = scale[rb];
            // The product in a fused multiply-add is exact and m is one that was rounded: they differ by up to half a step of m, which
            // is nothing below 2^20 but lets a weight overflow where logits are beyond 2^31.
            if (__builtin_amdgcn_ballot_w64(fabsf(off) > 0x1p20f) != 0ull) {
#pragma clang fp contract(off)
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[rb][u][i] = s[rb][u][i] * by - off;
                off = 0.0f;
                by = 1.0f;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(s[rb][u][i], by, -off));
                    l[rb] += w;
                    float p = w;
                    if constexpr (VB != 8) {
                        p *= half_of(vn[2 * u + (i >> 1)], i & 1);
                        if (masked) p = 4 * u + i < sees ? p : 0.0f;   // what a masked place holds may be no number
                    }
                    // int8 rows: the order 0, 2, 1, 3
                    const int to = VB == 8 ? ((i & 1) << 1) | (i >> 1) : i;
                    pf[rb][u >> 1][4 * (u & 1) + to] = (_Float16)p;
                }
        }
        // ---- values
#pragma unroll
        for (int blk = 0; blk < 4; ++blk) {
            const int row = 64 * half + 16 * blk + n16;
            half8_t vf[2][2];   // [dims' half][step]
            if constexpr (VB == 8) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(vb + (4 * hf + kq) * 2048 + row * 16);
                    const uint4 *d4 = reinterpret_cast<const uint4 *>(vb + 8 * 2048 + 2 * ((half * 4 + 2 * hf + (blk >> 1)) * 64 + 16 * kq));
                    const uint4 d0 = d4[0], d1 = d4[1];
                    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
                    uint32_t d[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
                    // In a tile that some row does not see whole, a scale that is no finite number (of rows that held none, or of a
                    // place that nothing was written to) must not reach the rows that do not see its token, and 0 times
                    // it would: it is replaced, and the rows that see it are marked.
                    if (masked) {
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
                        q4[u] = int8x4_times(ww[u], __builtin_bit_cast(half2_t, d02), __builtin_bit_cast(half2_t, d13));
                    }
                    vf[hf][0] = join(q4[0], q4[1]);
                    vf[hf][1] = join(q4[2], q4[3]);
                }
            } else {
                uint32_t w[VB];
#pragma unroll
                for (int j = 0; j < VB; ++j) w[j] = *reinterpret_cast<const uint32_t *>(vb + j * 2048 + row * 16 + kq * 4);
                const uint32_t tail = group_tail<VB>(w);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int st = 0; st < 2; ++st)
                        vf[hf][st] = join(group_quad<VB>(w, tail, vlut, 4 * st + hf), group_quad<VB>(w, tail, vlut, 4 * st + 2 + hf));
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int st = 0; st < 2; ++st)
                        o[rb][hf][blk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[hf][st], pf[rb][st], o[rb][hf][blk], 0, 0, 0);
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
    if (part != 0 || !active) return;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int r = r0 + 16 * rb + n16;
        const bool there = r < n_rows;
        const int t = (int)a.group_div.div((uint32_t)(there ? r : 0)), hq = head * a.group + (there ? r : 0) - t * a.group;
        float x[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = o[rb][e >> 4][(e >> 2) & 3][e & 3];
        if (span.splits <= 1) {
            write_out(a, x, l[rb] > 0.0f ? a.v_unscale / l[rb] : l[rb] == 0.0f ? 0.0f : l[rb], seq.row0 + t, hq, there, lane);
        } else if (there) {
            const int64_t at = ((seq.row0 + t) * (a.r.p.n_kv_heads * a.group) + hq) * a.n_splits + split;
#pragma unroll
            for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4 *>(a.part_o + at * 128 + out_dim(e, kq)) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
            if (kq == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * at) = make_float2(m[rb], l[rb]);
        }
    }
}

}  // namespace tqpaged
