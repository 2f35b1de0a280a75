// Attention over a paged cache, K rows of 3-bit codes (tq_paged_attn.h).
#include "tq_paged_launch.h"

int tqk_paged_attn_k3(const tqpaged::PagedAttnArgs &a, int vb, tqpaged::PagedKind kind, unsigned grid, hipStream_t s) {
    return tqpaged::launch_k<3>(a, vb, kind, grid, s);
}
