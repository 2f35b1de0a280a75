// The kernels of one K width, by V's width and the number of rows.
#pragma once
#include "tq_paged_attn.h"

namespace tqpaged {

template <int KB, int VB, int RB> void launch_rows(const PagedAttnArgs &a, unsigned grid, hipStream_t s) {
    if constexpr (KB == VB && KB != 8) {
        if (a.share) {
            k_paged_rows<KB, VB, RB, true><<<grid, 64 * ROWS_WAVES, 0, s>>>(a);
            return;
        }
    }
    k_paged_rows<KB, VB, RB, false><<<grid, 64 * ROWS_WAVES, 0, s>>>(a);
}
template <int KB, int VB> int launch_kind(const PagedAttnArgs &a, PagedKind kind, unsigned grid, hipStream_t s) {
    switch (kind) {
    case ROWS_32: launch_rows<KB, VB, 2>(a, grid, s); break;
    case ROWS_48: launch_rows<KB, VB, 3>(a, grid, s); break;
    case CHUNK_64: k_paged_chunk<KB, VB, 4, 1><<<grid, 256, 0, s>>>(a); break;
    case CHUNK_128: k_paged_chunk<KB, VB, 4, 2><<<grid, 256, 0, s>>>(a); break;
    default: k_paged_chunk<KB, VB, 8, 2><<<grid, 512, 0, s>>>(a); break;
    }
    return tq_check_launch("paged_attn");
}

template <int KB> int launch_k(const PagedAttnArgs &a, int vb, PagedKind kind, unsigned grid, hipStream_t s) {
    switch (vb) {
    case 2: return launch_kind<KB, 2>(a, kind, grid, s);
    case 3: return launch_kind<KB, 3>(a, kind, grid, s);
    case 4: return launch_kind<KB, 4>(a, kind, grid, s);
    default: return launch_kind<KB, 8>(a, kind, grid, s);
    }
}

}  // namespace tqpaged
