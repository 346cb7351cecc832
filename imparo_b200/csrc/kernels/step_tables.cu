// The description of a step over the paged cache, made on the device from the requests' lengths.
//
// Item r holds lengths[r] positions and brings counts[r] new tokens.  Its row of the step's block table is the row it holds (or, for
// the first shared[r] / page whole pages, the row its parent holds), and every block of its new positions that has no page yet takes
// the next one of the free list: items in order, blocks in order, the order in which the cache manager of the host hands pages out
// when requests reserve one after another (csrc/host/cache_manager.cpp).  The token arrays follow: an item's first token is the sum
// of the counts before it, a token's slot is page * page_size + place in the page (64-bit: rows of a large arena pass 32 bits in
// bytes long before, but slots are multiplied by a row's width by whoever uses them).
//
// One launch makes it: a CTA owns some items and sums the counts and the pages taken over all items before them by itself; for the item
// counts of a step (hundreds) that is one or two loads per thread, less than a launch before it or a wait between CTAs costs.
//
// A second, empty launch completes it: the engine's kernels read the description before they wait for the kernels ahead of them
// (common.cuh), so nothing may start before it is there.  Both on a B200: 4.0 us for 8 decode rows of 2,048 positions, 7.4 for 256 items
// of 32,768 (3.7 MB), 11.1 for 500 portions of 200 tokens, where every CTA looks at the 13 blocks of each item before its own.  The
// empty launch adds about 1 us to the first two.
#include "common.cuh"

namespace imparo {
namespace st {

constexpr int THREADS = 256;

struct Args {
    const int* lengths;
    const int* counts;
    const int* free_pages;
    const int* held;
    const int* parent;             // or null
    const int* shared;             // with parent
    int* table;
    int* positions;
    int* item_of_token;
    int* row_start;
    long long* slots;
    int* taken;
    int* status;
    int n_items, n_free, held_width, width, page_size, n_pages, n_tokens, items_per_cta;
};

// An item's numbers, brought into range (what is out of range is reported by its own CTA).
struct Item {
    int length, count, first, last;      // blocks [first, last) hold its new positions
    int from;                            // the row that gives the first `shared_blocks` blocks
    int shared_blocks;
};

__device__ __forceinline__ Item read_item(const Args& a, int r) {
    Item it;
    it.length = max(0, a.lengths[r]);
    it.count = max(0, min(a.counts[r], 0x7fffffff - it.length - a.page_size));
    it.first = min(it.length / a.page_size, a.width);
    it.last = it.count > 0 ? min((it.length + it.count + a.page_size - 1) / a.page_size, a.width) : it.first;
    it.from = r;
    it.shared_blocks = 0;
    if (a.parent) {
        const int p = a.parent[r];
        if (p >= 0 && p < a.n_items) {
            it.from = p;
            it.shared_blocks = min(max(0, a.shared[r]), it.length) / a.page_size;           // (new positions never go to a parent's page)
        }
    }
    return it;
}

__device__ __forceinline__ int held_page(const Args& a, const Item& it, int r, int block) {
    if (block >= a.held_width) return -1;
    return a.held[(size_t)(block < it.shared_blocks ? it.from : r) * a.held_width + block];
}

__device__ __forceinline__ long long warp_sum64(long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__global__ void __launch_bounds__(THREADS)
step_tables_kernel(const Args a) {
    __shared__ long long part[2][THREADS / 32];
    timeline_begin();                                          // (lets nothing start early: the launch behind it waits for all of it)
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r0 = blockIdx.x * a.items_per_cta, r1 = min(a.n_items, r0 + a.items_per_cta);

    // tokens and new pages of all items before this CTA's
    long long tokens = 0, pages = 0;
    for (int r = tid; r < r0; r += THREADS) {
        const Item it = read_item(a, r);
        tokens += it.count;
        for (int b = it.first; b < it.last; ++b) pages += held_page(a, it, r, b) < 0 ? 1 : 0;
    }
    tokens = warp_sum64(tokens);
    pages = warp_sum64(pages);
    if (lane == 0) { part[0][warp] = tokens; part[1][warp] = pages; }
    __syncthreads();
    tokens = pages = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) { tokens += part[0][i]; pages += part[1][i]; }

    // a page that is held: none where the arena has no such page
    auto listed = [&](int page, int r) -> int {
        if (page >= a.n_pages) report(a.status, IMPARO_ST_PAGE_RANGE, 64, r, page);
        return page < 0 || page >= a.n_pages ? -1 : page;
    };
    for (int r = r0; r < r1; ++r) {
        const Item it = read_item(a, r);
        int* row = a.table + (size_t)r * a.width;
        if (tid == 0) {
            a.row_start[r] = (int)min(tokens, (long long)0x7fffffff);
            if (a.lengths[r] < 0 || a.counts[r] < 0 || a.counts[r] != it.count) report(a.status, IMPARO_ST_STEP_SIZE, 60, r, a.counts[r]);
            if (it.count > 0 && it.last < (it.length + it.count + a.page_size - 1) / a.page_size)
                report(a.status, IMPARO_ST_STEP_SIZE, 61, r, it.length + it.count);
            if (a.parent && a.parent[r] >= a.n_items) report(a.status, IMPARO_ST_STEP_SIZE, 62, r, a.parent[r]);
            if (it.from != r && a.shared[r] / a.page_size > it.shared_blocks) report(a.status, IMPARO_ST_STEP_SIZE, 66, r, a.shared[r]);
        }
        // blocks without new positions: as held
        for (int b = tid; b < a.width; b += THREADS)
            if (b < it.first || b >= it.last) row[b] = listed(held_page(a, it, r, b), r);
        // blocks with new positions: the missing pages from the free list, in order; every warp counts, one writes
        long long next = pages;
        for (int b0 = it.first; b0 < it.last; b0 += 32) {
            const int b = b0 + lane;
            int page = b < it.last ? held_page(a, it, r, b) : 0;
            const bool missing = page < 0;
            const unsigned mask = __ballot_sync(0xffffffffu, missing);
            if (missing) {
                const long long at = next + __popc(mask & ((1u << lane) - 1u));
                page = at < a.n_free ? a.free_pages[at] : -1;
                if (warp == 0 && (page < 0 || page >= a.n_pages))
                    report(a.status, at < a.n_free ? IMPARO_ST_PAGE_RANGE : IMPARO_ST_STEP_SIZE, 63, r, page);
                if (page < 0 || page >= a.n_pages) page = -1;
            }
            if (warp == 0 && b < it.last) row[b] = listed(page, r);
            next += __popc(mask);
        }
        __syncthreads();                                       // the row is written: the tokens read it
        for (int i = tid; i < it.count; i += THREADS) {
            const long long t = tokens + i;
            if (t >= a.n_tokens) break;
            const int pos = it.length + i, b = pos / a.page_size;
            const int page = b < a.width ? row[b] : -1;
            a.positions[t] = pos;
            a.item_of_token[t] = r;
            a.slots[t] = page >= 0 ? (long long)page * a.page_size + pos % a.page_size : -1;
        }
        tokens += it.count;
        pages = next;
    }
    if (r1 == a.n_items) {                                     // the last CTA: the totals, and the tokens behind the last item's
        if (tid == 0) {
            a.row_start[a.n_items] = (int)min(tokens, (long long)0x7fffffff);
            a.taken[0] = (int)min(pages, (long long)0x7fffffff);
            if (tokens > a.n_tokens) report(a.status, IMPARO_ST_STEP_SIZE, 65, a.n_items, (int)min(tokens, (long long)0x7fffffff));
        }
        for (long long t = tokens + tid; t < a.n_tokens; t += THREADS) {
            a.positions[t] = -1;
            a.item_of_token[t] = 0;
            a.slots[t] = -1;
        }
    }
}

// Does nothing.  The engine's kernels read the description of the step before they wait for the kernels ahead of them, so none may
// start before the description is complete: this one is launched without that freedom, and they come behind it.
__global__ void step_tables_complete_kernel() {
    pdl_trigger();
    pdl_wait();
}

}  // namespace st
}  // namespace imparo

using namespace imparo;

extern "C" int imparo_step_tables(const int* lengths, const int* counts, const int* free_pages, int n_free, const int* held,
                                  int held_width, const int* parent, const int* shared, int n_items, int page_size, int n_pages,
                                  int* table, int width, int* positions, int* item_of_token, int n_tokens, int* row_start,
                                  long long* slots, int* taken, int* status, cudaStream_t stream) {
    if (n_items < 1 || n_items > (1 << 24) || page_size < 1 || n_pages < 1 || width < 1 || held_width < 0 || n_free < 0 || n_tokens < 0)
        return -2;
    if (parent && !shared) return -2;
    st::Args a;
    a.lengths = lengths; a.counts = counts; a.free_pages = free_pages; a.held = held; a.parent = parent; a.shared = shared;
    a.table = table; a.positions = positions; a.item_of_token = item_of_token; a.row_start = row_start; a.slots = slots;
    a.taken = taken; a.status = status; a.n_items = n_items; a.n_free = n_free; a.held_width = held_width; a.width = width;
    a.page_size = page_size; a.n_pages = n_pages; a.n_tokens = n_tokens;
    a.items_per_cta = (n_items + 1183) / 1184;                 // up to eight CTAs per SM
    const int ctas = (n_items + a.items_per_cta - 1) / a.items_per_cta;
    cudaError_t e = launch(st::step_tables_kernel, dim3(ctas), dim3(st::THREADS), 0, stream, a);
    if (e == cudaSuccess) e = launch_after(st::step_tables_complete_kernel, dim3(1), dim3(32), 0, stream);
    return e == cudaSuccess ? 0 : (int)e;
}
