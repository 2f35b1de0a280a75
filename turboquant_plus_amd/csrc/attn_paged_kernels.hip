// Decode attention over a paged cache: k_decode_attn with BIAS_PAGED (tq_attn_rows.h), for steps of one or a few new tokens.
#include "tq_attn_rows.h"

using namespace tqattn;

bool tqk_launch_paged(const AttnArgs &a, int kb, int vb, bool share, int hg, dim3 grid, unsigned wg, size_t lds, hipStream_t s) {
#define TQ_PAIR(KF, K, V, SH)                                                                                 \
    if (kb == (KF == KFMT_Q8 ? 8 : K) && vb == V && share == SH) {                                            \
        if (hg == 2) k_decode_attn<KF, K, V, false, SH, 2, BIAS_PAGED><<<grid, wg, lds, s>>>(a);              \
        else k_decode_attn<KF, K, V, false, SH, 1, BIAS_PAGED><<<grid, wg, lds, s>>>(a);                      \
        return true;                                                                                         \
    }
    TQ_PAIR(KFMT_TURBO, 3, 3, true) TQ_PAIR(KFMT_TURBO, 4, 4, true) TQ_PAIR(KFMT_TURBO, 2, 2, true)
    TQ_PAIR(KFMT_TURBO, 3, 3, false) TQ_PAIR(KFMT_TURBO, 4, 4, false) TQ_PAIR(KFMT_TURBO, 2, 2, false)
    TQ_PAIR(KFMT_TURBO, 4, 2, false) TQ_PAIR(KFMT_TURBO, 3, 2, false) TQ_PAIR(KFMT_TURBO, 3, 4, false)
    TQ_PAIR(KFMT_TURBO, 4, 3, false) TQ_PAIR(KFMT_TURBO, 2, 3, false) TQ_PAIR(KFMT_TURBO, 2, 4, false)
    TQ_PAIR(KFMT_Q8, 3, 2, false) TQ_PAIR(KFMT_Q8, 3, 3, false) TQ_PAIR(KFMT_Q8, 3, 4, false) TQ_PAIR(KFMT_Q8, 3, 8, false)
    TQ_PAIR(KFMT_TURBO, 2, 8, false) TQ_PAIR(KFMT_TURBO, 3, 8, false) TQ_PAIR(KFMT_TURBO, 4, 8, false)
#undef TQ_PAIR
    return false;
}
