// What the kernels of the attention over a shared prefix (attention_shared.cu, attention_shared_tc.cu) have in common: the launch's
// arguments, which rows form a group, and which keys of a row are taken with the group's and which with the row's own.
#pragma once
#include "common.cuh"

namespace imparo {
namespace sp {

struct Args {
    const void* q;
    const void* k;
    const void* v;
    const int* positions;
    const int* item_of_token;
    const int* table;
    const int* group_start;        // [n_groups + 1]
    const int* shared;             // [n_groups]
    float* part_acc;
    float* part_ml;
    int* status;
    long long q_stride;            // elements between rows of q
    int n_rows, n_items, n_groups, max_blocks, page_size, n_pages, window, nh, nkv, hd;
    int chunk_shared, n_shared, chunk_own, n_own;
    int most_pos;                  // the first position that the table has no block for: later ones are taken for it
    float scale;
};

// The rows [start, end) of a group and its shared positions, in range whatever the arrays hold.
__device__ __forceinline__ void group_rows(const Args& a, int g, int& start, int& end) {
    start = min(max(a.group_start[g], 0), a.n_rows);
    end = min(max(a.group_start[g + 1], start), a.n_rows);
}
// the group a row belongs to, -1: none (the row then shares nothing)
__device__ __forceinline__ int group_of(const Args& a, int t) {
    int lo = 0, hi = a.n_groups;                                   // the last group that starts at or before t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.group_start[mid] <= t) lo = mid + 1; else hi = mid;
    }
    const int g = lo - 1;
    return g >= 0 && t < a.group_start[g + 1] ? g : -1;
}
// The same by a warp that is together: few groups are looked at all at once, one trip to memory instead of a search's.
__device__ __forceinline__ int group_of_warp(const Args& a, int t) {
    if (a.n_groups > 128) return group_of(a, t);
    for (int base = 0; base < a.n_groups; base += 32) {
        const int g = base + (threadIdx.x & 31);
        const unsigned found = __ballot_sync(0xffffffffu, g < a.n_groups && a.group_start[min(g, a.n_groups - 1)] <= t && t < a.group_start[min(g, a.n_groups - 1) + 1]);
        if (found) return base + __ffs(found) - 1;
    }
    return -1;
}
__device__ __forceinline__ const int* table_row(const Args& a, int t, int kernel) {
    const int item = a.item_of_token[t];
    if (item < 0 || item >= a.n_items) {
        report(a.status, IMPARO_ST_PAGE_RANGE, kernel, t, item);
        return nullptr;
    }
    return a.table + (size_t)item * a.max_blocks;
}
__device__ __forceinline__ int first_seen(const Args& a, int pos) { return a.window > 0 && pos + 1 > a.window ? pos + 1 - a.window : 0; }

// The keys [first, end) that the shared stretches take for a group: those of its shared positions that every row of it sees (rows
// without a position, pos < 0, aside).  Each row takes the rest of what it sees, on both sides of them, with its own ones, so the
// shared stretches need no mask by row and whatever a row does not see never meets its weights.  The pages are those that the first row
// with a position lists: one without may have ended and its pages be gone, and a group of nothing but such rows has no shared keys.
// Every warp finds all this by itself (no barrier); the result is the same for every launch of the same arrays.
struct Span { int first, end, row; };
__device__ __forceinline__ Span shared_span(const Args& a, int g) {
    if (g < 0) return Span{0, 0, 0};
    int start, end;
    group_rows(a, g, start, end);
    int lo = 0, hi = max(0, a.shared[g]), row = a.n_rows;
#pragma unroll 4
    for (int t = start + (threadIdx.x & 31); t < end; t += 32) {
        const int pos = min(a.positions[t], a.most_pos);
        if (pos >= 0) { lo = max(lo, first_seen(a, pos)); hi = min(hi, pos + 1); row = min(row, t); }
    }
    lo = __reduce_max_sync(0xffffffffu, lo);
    hi = __reduce_min_sync(0xffffffffu, hi);
    row = __reduce_min_sync(0xffffffffu, row);
    return row < a.n_rows && lo < hi ? Span{lo, hi, row} : Span{0, 0, 0};
}
// A row's own keys, counted through: the first `before` of them lie before the shared ones.  (A position far beyond the table is an
// error that the first key without a block reports; without the bound the row would look up every one of up to 2^31 keys.)
struct Own {
    int lo, before, skip, count;
    __device__ __forceinline__ int key(int i) const { return lo + i + (i < before ? 0 : skip); }
};
__device__ __forceinline__ Own own_keys(const Args& a, int pos, Span s) {
    Own o;
    pos = min(pos, a.most_pos);
    o.lo = first_seen(a, pos);
    o.before = s.first < s.end ? s.first - o.lo : 0x7fffffff;      // (a row sees all of the span: lo <= first, end <= pos + 1)
    o.skip = s.end - s.first;
    o.count = pos < 0 ? 0 : pos + 1 - o.lo - o.skip;
    return o;
}

// The tensor-core path (attention_shared_tc.cu): bfloat16, head size 64 or 128.  -8: it does not take these sizes.
int launch_tc(const Args& a, void* out, const float* sinks, cudaStream_t stream);

}  // namespace sp
}  // namespace imparo
