// The kernels of one K width, by V's width, shared table and row blocks.
#pragma once
#include "tq_paged_attn.h"

namespace tqpaged {

template <int KB, int VB, bool SHARE> int launch_rows(const PagedAttnArgs &a, int rb, unsigned grid, hipStream_t s) {
    switch (rb) {
    case 1: k_paged_attn<KB, VB, 1, SHARE><<<grid, 64 * paged_waves(1), 0, s>>>(a); break;
    case 2: k_paged_attn<KB, VB, 2, SHARE><<<grid, 64 * paged_waves(2), 0, s>>>(a); break;
    default: k_paged_attn<KB, VB, 4, SHARE><<<grid, 64 * paged_waves(4), 0, s>>>(a); break;
    }
    return tq_check_launch("paged_attn");
}

template <int KB> int launch_k(const PagedAttnArgs &a, int vb, bool share, int rb, unsigned grid, hipStream_t s) {
    if constexpr (KB != 8) {
        if (share && vb == KB) return launch_rows<KB, KB, true>(a, rb, grid, s);
    }
    switch (vb) {
    case 2: return launch_rows<KB, 2, false>(a, rb, grid, s);
    case 3: return launch_rows<KB, 3, false>(a, rb, grid, s);
    case 4: return launch_rows<KB, 4, false>(a, rb, grid, s);
    default: return launch_rows<KB, 8, false>(a, rb, grid, s);
    }
}

}  // namespace tqpaged
