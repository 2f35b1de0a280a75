// Which sequence, block or rows a workgroup has in a launch over a paged cache.
#pragma once
#include "tq_internal.h"
#include "tq_layout.h"

// An entry of a table that no running launch changes, at an index that is the same in all lanes: by a scalar load.  As a vector
// load it would return behind the rows requested before it, and the wavefront, which needs it at once, would wait for them all.
__device__ __forceinline__ int32_t scalar_entry(const int32_t *table, int64_t i) {
    typedef const int32_t __attribute__((address_space(4))) *constant_ptr;
    return *(constant_ptr)(uintptr_t)(table + i);
}

struct PagedRows {
    tq_pages p;
    int64_t rows;           // of the new tokens' tensors
    tqd::FastDiv heads_div; // division by n_kv_heads
};

struct PagedSeq {
    int row0;       // its first row in the new tokens' tensors
    int n;          // its rows; 0 where the tables give rows outside of the tensors
    int start;      // lens[b]
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedRows &r, int b) {
    PagedSeq q;
    const int32_t lo = r.p.cu_new ? r.p.cu_new[b] : b, hi = r.p.cu_new ? r.p.cu_new[b + 1] : b + 1;
    q.row0 = lo;
    q.n = lo >= 0 && hi > lo && hi <= r.rows ? hi - lo : 0;
    q.start = r.p.lens[b];
    return q;
}
// whether an append at lens[b] has a place for the sequence's rows
__device__ __forceinline__ bool paged_room(const PagedRows &r, const PagedSeq &q) {
    return q.start >= 0 && (int64_t)q.start + q.n <= (int64_t)r.p.max_blocks * TQ_ROWS_PER_BLOCK;
}
// blocks that hold rows of a sequence
__device__ __forceinline__ int paged_blocks(const PagedRows &r, const PagedSeq &q) {
    if (q.n == 0 || !paged_room(r, q)) return 0;
    return (q.start + q.n - 1) / TQ_ROWS_PER_BLOCK - q.start / TQ_ROWS_PER_BLOCK + 1;
}
// One workgroup's look at every sequence: why an append leaves some out.
__device__ __forceinline__ void paged_report(const PagedRows &r, uint32_t *overrun) {
    for (int b = threadIdx.x; b < r.p.batch; b += blockDim.x) {
        const PagedSeq q = paged_seq(r, b);
        const int32_t lo = r.p.cu_new ? r.p.cu_new[b] : b, hi = r.p.cu_new ? r.p.cu_new[b + 1] : b + 1;
        uint32_t why = 0;
        if (q.n == 0) why = lo == hi && lo >= 0 && hi <= r.rows ? 0u : TQ_OVERRUN_NO_PAGE;
        else if (q.start < 0) why = TQ_OVERRUN_NEGATIVE;
        else if (!paged_room(r, q)) why = TQ_OVERRUN_NO_ROOM;
        if (why) atomicOr(overrun, why);
    }
}

// sum over the lanes up to this one
__device__ __forceinline__ int sum_upto_lane(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // from one, two, four, eight lanes down in a row of sixteen
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // the rows' sums: rows 0 and 2 to 1 and 3, then row 1's to 2 and 3
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
}
// Item `item` of the sequences' items laid end to end, count(sequence) of them to each: its sequence and its number there, the
// same in every lane; false behind the last one.  Every wavefront of a workgroup calls it and works it out for itself: 64
// sequences at a time, a sum over the lanes.
template <class Count> __device__ __forceinline__ bool paged_item(const PagedRows &r, int item, Count count, int &b, int &nth, PagedSeq &seq) {
    const int lane = (int)(threadIdx.x & 63);
    if (!r.p.cu_new) {   // one row each, and no more than one item
        if (item >= r.p.batch) return false;
        b = item;
        nth = 0;
        seq = PagedSeq{item, 1, scalar_entry(r.p.lens, item)};
        return count(seq) > 0;
    }
    for (int b0 = 0; b0 < r.p.batch; b0 += 64) {
        PagedSeq q{0, 0, 0};
        int c = 0;
        if (b0 + lane < r.p.batch) {
            q = paged_seq(r, b0 + lane);
            c = count(q);
        }
        const int upto = sum_upto_lane(c);
        const unsigned long long behind = __builtin_amdgcn_ballot_w64(upto > item);
        if (behind) {
            const int at = __builtin_ctzll(behind);
            b = b0 + at;
            nth = item - __builtin_amdgcn_readlane(upto - c, at);
            seq = PagedSeq{__builtin_amdgcn_readlane(q.row0, at), __builtin_amdgcn_readlane(q.n, at), __builtin_amdgcn_readlane(q.start, at)};
            return true;
        }
        item -= __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}
