// Attention over a paged cache, K rows of 8 bits (tq_paged_attn.h).
#include "tq_paged_launch.h"

int tqk_paged_attn_k8(const tqpaged::PagedAttnArgs &a, int vb, tqpaged::PagedKind kind, unsigned grid, hipStream_t s) {
    return tqpaged::launch_k<8>(a, vb, kind, grid, s);
}
