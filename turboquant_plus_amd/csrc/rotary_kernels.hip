// Rotary positions of queries and keys.
//
// k_rotary: pair (u, w) of a head -> (u cos a - w sin a, w cos a + u sin a), a = position * frequency.  A workgroup takes a few
//   tokens with all their heads: it works out the cosines and sines of those tokens once (64-bit turns, reduced to a fraction of
//   one, so that far positions lose nothing), keeps them in LDS and streams the heads past them, 16 bytes of each half of a
//   pair at a time.  Bound by memory: 32768 tokens of 32 + 8 heads of 128, fp16, 671 MB in 123.6 us (5.4 TB/s, 128 in a loop of its own);
//   value by value, where rows do not begin at 16 bytes, 255 us (interleaved 235).
#include "tq_check.h"
#include "tq_layout.h"

namespace {

using tqd::FastDiv;
using tqd::make_fast_div;

struct RotaryArgs {
    const void *x[2];
    void *y[2];
    int64_t x_token[2], x_head[2], y_token[2], y_head[2];
    const double *turns;
    const void *positions;
    int64_t tokens;
    int positions_64, inverse;
    float magnitude;
    int half;                    // rotated pairs of a head
    int per_wg;                  // tokens of a workgroup
    uint32_t q_heads;
    uint32_t turned, pieces;     // pieces of a head that are turned, and all that are written (VEC values, or VEC pairs of halves)
    FastDiv pieces_div, heads_div;
};

template <typename T, int VEC> struct Piece {
    typedef T type __attribute__((ext_vector_type(VEC)));
};
template <typename T> struct Piece<T, 1> {
    typedef T type;
};
template <typename T, int VEC> __device__ __forceinline__ float value(const typename Piece<T, VEC>::type &p, int i) {
    if constexpr (VEC == 1) return (float)p;
    else return (float)p[i];
}
template <typename T, int VEC> __device__ __forceinline__ void put(typename Piece<T, VEC>::type &p, int i, float v) {
    if constexpr (VEC == 1) p = (T)v;
    else p[i] = (T)v;
}

constexpr int ROTARY_THREADS = 256, ROTARY_BATCH = 4;

// VEC: values of a load, 16 bytes of them, or 1 where strides, pointers or sizes do not allow that
template <typename T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(ROTARY_THREADS) void k_rotary(RotaryArgs a) {
    typedef typename Piece<T, VEC>::type piece_t;
    constexpr bool PAIRS = INTERLEAVED && VEC > 1;   // a piece holds whole pairs
    extern __shared__ float2 turn_s[];               // [token of the workgroup][pair]: cosine, sine
    const int tid = threadIdx.x;
    const int64_t first = (int64_t)blockIdx.x * a.per_wg;
    const uint32_t here = (uint32_t)(a.tokens - first < a.per_wg ? a.tokens - first : a.per_wg);
    const uint32_t heads = a.heads_div.d, n = here * heads * a.pieces;

    piece_t lo[ROTARY_BATCH], hi[ROTARY_BATCH];
    struct Place {
        const T *from;
        T *to;
        uint32_t token, piece;
        int second;              // from a pair's first value to its other one
        bool turned;
    };
    auto place = [&](uint32_t item) {
        const uint32_t row = a.pieces_div.div(item), piece = item - row * a.pieces;
        const uint32_t token = a.heads_div.div(row), head = row - token * heads;
        const int side = head >= a.q_heads;
        const int64_t h = side ? head - a.q_heads : head;
        Place p;
        p.turned = piece < a.turned;
        p.token = token;
        p.piece = piece;
        p.second = INTERLEAVED ? 1 : a.half;
        const int at = p.turned ? (PAIRS ? VEC : INTERLEAVED ? 2 : VEC) * (int)piece : 2 * a.half + VEC * (int)(piece - a.turned);
        // selects, not indexing: an index into kernel arguments goes through scratch memory
        p.from = reinterpret_cast<const T *>(side ? a.x[1] : a.x[0]) + (first + token) * (side ? a.x_token[1] : a.x_token[0]) +
                 h * (side ? a.x_head[1] : a.x_head[0]) + at;
        p.to = reinterpret_cast<T *>(side ? a.y[1] : a.y[0]) + (first + token) * (side ? a.y_token[1] : a.y_token[0]) +
               h * (side ? a.y_head[1] : a.y_head[0]) + at;
        return p;
    };
    auto load = [&](uint32_t item0) {
#pragma unroll
        for (int b = 0; b < ROTARY_BATCH; ++b) {
            const uint32_t item = item0 + b * ROTARY_THREADS;
            if (item < n) {
                const Place p = place(item);
                lo[b] = *reinterpret_cast<const piece_t *>(p.from);
                if (!PAIRS && p.turned) hi[b] = *reinterpret_cast<const piece_t *>(p.from + p.second);
            }
        }
    };
    // the first batch is on its way while the angles are worked out
    load(tid);
    for (uint32_t e = tid; e < here * (uint32_t)a.half; e += ROTARY_THREADS) {
        const uint32_t t = e / (uint32_t)a.half, i = e - t * (uint32_t)a.half;
        const int64_t pos = a.positions_64 ? reinterpret_cast<const int64_t *>(a.positions)[first + t]
                                           : (int64_t) reinterpret_cast<const int32_t *>(a.positions)[first + t];
        double turns = (double)pos * a.turns[i];
        turns -= rint(turns);
        float s, c;
        sincospif((float)(2.0 * turns), &s, &c);
        turn_s[e] = make_float2(c * a.magnitude, (a.inverse ? -s : s) * a.magnitude);
    }
    __syncthreads();
    for (uint32_t item0 = tid; item0 < n; item0 += ROTARY_BATCH * ROTARY_THREADS) {
        if (item0 != (uint32_t)tid) load(item0);
#pragma unroll
        for (int b = 0; b < ROTARY_BATCH; ++b) {
            const uint32_t item = item0 + b * ROTARY_THREADS;
            if (item >= n) break;
            const Place p = place(item);
            if (p.turned) {
                const float2 *turn = turn_s + p.token * (uint32_t)a.half + (PAIRS ? VEC / 2 : VEC) * p.piece;
                if constexpr (PAIRS) {
                    piece_t r;
#pragma unroll
                    for (int i = 0; i < VEC; i += 2) {
                        const float u = value<T, VEC>(lo[b], i), w = value<T, VEC>(lo[b], i + 1);
                        put<T, VEC>(r, i, u * turn[i / 2].x - w * turn[i / 2].y);
                        put<T, VEC>(r, i + 1, w * turn[i / 2].x + u * turn[i / 2].y);
                    }
                    lo[b] = r;
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float u = value<T, VEC>(lo[b], i), w = value<T, VEC>(hi[b], i);
                        put<T, VEC>(lo[b], i, u * turn[i].x - w * turn[i].y);
                        put<T, VEC>(hi[b], i, w * turn[i].x + u * turn[i].y);
                    }
                    *reinterpret_cast<piece_t *>(p.to + p.second) = hi[b];
                }
            }
            *reinterpret_cast<piece_t *>(p.to) = lo[b];
        }
    }
}

template <typename T> int launch(RotaryArgs a, const tq_rotary_params *p, bool wide, hipStream_t s) {
    constexpr int WIDE = 16 / sizeof(T);
    const int vec = wide ? WIDE : 1;
    const bool pairs = p->interleaved && wide;
    a.turned = (uint32_t)(pairs ? p->rotary_dim / vec : p->rotary_dim / 2 / vec);
    // in place nothing but the turned values is written
    const bool moved = (p->n_q_heads && a.x[0] != a.y[0]) || (p->n_k_heads && a.x[1] != a.y[1]);
    a.pieces = a.turned + (moved ? (uint32_t)((p->head_dim - p->rotary_dim) / vec) : 0u);
    a.pieces_div = make_fast_div(a.pieces);
    a.heads_div = make_fast_div((uint32_t)(p->n_q_heads + p->n_k_heads));
    // several tokens to a workgroup, so that every thread works out a cosine, as long as that leaves the chip full
    int per = 1;
    while (per < 16 && per * a.half < ROTARY_THREADS && p->tokens / (2 * per) >= 1024) per *= 2;
    a.per_wg = per;
    const int64_t grid = (p->tokens + per - 1) / per;
    if ((int64_t)per * a.pieces * a.heads_div.d > (1u << 31) || grid > 0x7FFFFFFF) {
        tq_set_error("tq_rotary: %lld tokens of %u heads are more than a launch takes", (long long)p->tokens, a.heads_div.d);
        return TQ_ERR_UNSUPPORTED;
    }
    const size_t lds = (size_t)per * a.half * sizeof(float2);
#define TQ_ROTARY(V, I) k_rotary<T, V, I><<<(unsigned)grid, ROTARY_THREADS, lds, s>>>(a)
    if (wide && p->interleaved) TQ_ROTARY(WIDE, true);
    else if (wide) TQ_ROTARY(WIDE, false);
    else if (p->interleaved) TQ_ROTARY(1, true);
    else TQ_ROTARY(1, false);
#undef TQ_ROTARY
    return tq_check_launch("rotary");
}

}  // namespace

extern "C" int tq_rotary(const tq_rotary_params *p, const void *q, void *q_out, const void *k, void *k_out, const void *positions,
                         const double *turns, void *stream) {
    REQUIRE(p, TQ_ERR_ARG, "tq_rotary: null parameters");
    REQUIRE(p->tokens >= 0 && p->n_q_heads >= 0 && p->n_k_heads >= 0, TQ_ERR_ARG, "tq_rotary: negative size");
    REQUIRE(p->head_dim >= 1 && p->head_dim <= 65536, TQ_ERR_ARG, "tq_rotary: head_dim %d is not in 1..65536", p->head_dim);
    REQUIRE(p->rotary_dim >= 2 && p->rotary_dim % 2 == 0 && p->rotary_dim <= p->head_dim, TQ_ERR_ARG,
            "tq_rotary: rotary_dim %d must be even and in 2..head_dim (%d)", p->rotary_dim, p->head_dim);
    REQUIRE(p->rotary_dim <= 1024, TQ_ERR_UNSUPPORTED, "tq_rotary: rotary_dim %d is over 1024", p->rotary_dim);
    REQUIRE((int64_t)p->n_q_heads + p->n_k_heads <= 65536, TQ_ERR_UNSUPPORTED, "tq_rotary: over 65536 heads");
    REQUIRE(p->dtype == TQ_F16 || p->dtype == TQ_F32 || p->dtype == TQ_BF16, TQ_ERR_ARG, "tq_rotary: dtype %d is none of float16, float32, bfloat16",
            p->dtype);
    const bool has_q = p->n_q_heads > 0, has_k = p->n_k_heads > 0;
    if (p->tokens == 0 || !(has_q || has_k)) return TQ_OK;
    REQUIRE((!has_q || (q && q_out)) && (!has_k || (k && k_out)) && positions && turns, TQ_ERR_ARG, "tq_rotary: null pointer");
    const unsigned size = p->dtype == TQ_F32 ? 4 : 2;
    const uintptr_t at = (has_q ? reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) : 0) |
                         (has_k ? reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out) : 0);
    REQUIRE(at % size == 0 && reinterpret_cast<uintptr_t>(turns) % 8 == 0 && reinterpret_cast<uintptr_t>(positions) % (p->positions_64 ? 8 : 4) == 0,
            TQ_ERR_ALIGN, "tq_rotary: a pointer is not aligned to its type");
    RotaryArgs a;
    a.x[0] = q; a.x[1] = k; a.y[0] = q_out; a.y[1] = k_out;
    const int64_t strides[8] = {p->q_token, p->q_head, p->q_out_token, p->q_out_head, p->k_token, p->k_head, p->k_out_token, p->k_out_head};
    for (int i = 0; i < 2; ++i) {
        a.x_token[i] = strides[4 * i]; a.x_head[i] = strides[4 * i + 1];
        a.y_token[i] = strides[4 * i + 2]; a.y_head[i] = strides[4 * i + 3];
    }
    a.turns = turns; a.positions = positions; a.tokens = p->tokens; a.positions_64 = p->positions_64; a.inverse = p->inverse;
    a.magnitude = p->magnitude; a.half = p->rotary_dim / 2; a.q_heads = (uint32_t)p->n_q_heads;
    // 16 bytes at a time: every stride, pointer and size is a multiple of that
    const int vec = 16 / (int)size;
    bool wide = at % 16 == 0 && p->head_dim % vec == 0 && (p->interleaved ? p->rotary_dim : p->rotary_dim / 2) % vec == 0;
    for (int i = 0; i < 8; ++i) wide = wide && (!(i < 4 ? has_q : has_k) || strides[i] % vec == 0);
    hipStream_t s = (hipStream_t)stream;
    if (p->dtype == TQ_F16) return launch<_Float16>(a, p, wide, s);
    if (p->dtype == TQ_BF16) return launch<__bf16>(a, p, wide, s);
    return launch<float>(a, p, wide, s);
}
