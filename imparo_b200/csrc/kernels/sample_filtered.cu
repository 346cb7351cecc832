// Picking a token per row of logits under a temperature, top-k, top-p and min-p, from a given random number per row.
//
// With m the largest logit of the row, T its temperature and w_i = exp((v_i - m) / T), the entries ordered by falling logit (equal
// ones by rising index):
//   K  the first top_k of the order (top_k <= 0: all)          P  the shortest beginning of K whose weight reaches top_p w(K)
//   M  those of P with w_i >= min_p                            pick: the first index, in vocabulary order over M, at which the
//                                                              running sum of w passes u w(M)
// Every filter keeps a beginning of the same order, so the kept set is a cut (logit, index) and one more bound on the logit.
//
// Weights are whole numbers, w_i rounded to a multiple of 2^-shift (2^-45 for 131,072 entries), summed in 64 bits: sums are the
// same whatever the order of their terms, so counts and sums may be gathered by atomics, part by part, and the picked index is the
// one that 64-bit arithmetic gives except where a border lies within some 2^-40 of the drawn number.  In 32-bit sums, neighbours
// with weights of 1e-5 of the total each were told apart wrongly once in some hundred rows.
//
// A cluster of CTAs owns a row, each CTA a contiguous stretch of it, which it keeps in shared memory where it fits; with many rows a
// row has one CTA, which reads a long row several times, from the L2 but for the first.  The cut is found by histograms (the cluster's
// CTAs exchange them through distributed shared memory): 1,024 bins of equal width in (m - v) / T.  Where the order up to the cut's
// bin fits a list of 1,024 entries, the first CTA does the rest with that list alone; otherwise the entries of the cut's bin are
// sorted, and a bin with more entries than the list holds is cut further by ten bits of the ordered logit at a time.
//
// What bounds it, on a B200: with few rows the chain of looks and barriers (one row of 65,536 under top-k 40 and top-p 0.95 10.5 us, eight
// under top-p 32); with many, reading (256 greedy rows of 131,072 34 us, 3.9 TB/s), then the 64-bit operations of the weights (256 rows
// at a temperature alone 112 us) and, where a border is found by a histogram, shared-memory atomics at some 12 cycles a warp (top-p
// 0.9 300 us).  A top-k of up to some 500 needs no histogram: the k-th largest of the groups' largest entries bounds it (k 50: 79 us).
#include "common.cuh"
#include <cooperative_groups.h>
#include <type_traits>
#include <utility>

namespace imparo {
namespace sf {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int BINS = 1024;                     // two per thread
constexpr int LIST = 1024;                     // entries of a bin that are sorted at once
constexpr int STAGED_MOST = 16384;             // entries of a stretch kept in shared memory (64 KB: two CTAs per SM)
constexpr int MOST_RANKS = 8;                  // CTAs of a cluster
constexpr int FEW = 256;                       // listed entries that are compared each with each
constexpr int LOG_STEPS = 10, STEPS = 1 << LOG_STEPS;           // of the exponential's table to a factor of two
constexpr float BIN_RANGE = 24.0f;             // (m - v) / T covered by the bins; the last one takes all beyond
static_assert(BINS == 2 * THREADS && LIST == 2 * THREADS, "two bins and two list entries per thread");

struct Args {
    const void* logits;
    const float* temperature;
    const float* uniform;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    int* out;
    int* kept;
    long long ld;
    int vocab, per, shift;
};

struct Shared {
    uint32_t n[BINS], lo[BINS], hi[BINS];                          // this CTA's histogram: counts, weights in two halves
    uint32_t all_n[BINS];                                          // the cluster's, written share by share by its CTAs
    u64 all_w[BINS];
    u64 list[LIST];                                                // entries that are sorted
    double table[STEPS];                                           // 2^(i / STEPS)
    u64 warp_w[WARPS + 1];
    uint32_t warp_n[WARPS + 1];
    u64 part_w;                                                    // read by the other CTAs
    uint32_t part_n, list_n, gathered[2];      // (the first: the same in every CTA)
    u64 before_w, found_cut, total_w;
    uint32_t before_n, bin, found, total_n;
};

// a logit as a whole number of the same order, and back; equal logits have equal numbers (the zero's sign is dropped on loading)
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
// an entry's place in the order as one number: the larger comes first
__device__ __forceinline__ u64 entry(float v, int index) { return ((u64)ordered(v) << 32) | (uint32_t)~index; }

// the place in the order at or above which every number above minus infinity lies
constexpr u64 ALL = (u64)0x00800000u << 32;

// NaN is no number: it is taken for minus infinity, which no filter keeps
__device__ __forceinline__ float clean(float v) { return v == v ? v + 0.0f : -INFINITY; }

struct Weights {
    double top, rate;          // the row's largest logit; STEPS log2(e) / T
    const double* table;       // 2^(i / STEPS)
    float topf, least;         // below `least` a weight is 0
    int shift;
    // exp((v - top) / T), v above minus infinity, as a multiple of 2^-shift.  Table-driven exponential (P. T. P. Tang, 1989): t =
    // STEPS log2(e) (v - top) / T is split into a whole number n and a rest f of at most 1/2; 2^(n / STEPS) from the table and the
    // exponent, 2^(f / STEPS) by its series in f: with 1,024 steps the first four terms leave out less than 2^-50.
    __device__ __forceinline__ u64 operator()(float v) const {
        const double t = ((double)v - top) * rate;
        const double whole = 6755399441055744.0;                   // 1.5 2^52: adding it rounds to a whole number
        const double tn = t + whole;
        const int n = __double2loint(tn);
        const double f = t - (tn - whole);
        constexpr double c = 0.69314718055994530942 / STEPS;
        const double p = table[n & (STEPS - 1)] * fma(f, fma(f, fma(f, c * c * c / 6.0, c * c / 2.0), c), 1.0);
        // times 2^(n / STEPS) and 2^shift, by the exponent (from 2^-63 2^38 on: a normal number), then + 2^52: rounded to a whole one
        const double scaled = __hiloint2double(__double2hiint(p) + (((n >> LOG_STEPS) + shift) << 20), __double2loint(p));
        const u64 w = __double_as_longlong(scaled + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
        return v == topf ? 1ull << shift : v < least ? 0 : w;      // (the largest may be infinite)
    }
};

// x times num for a float 0 <= x < 1, rounded down / up to a whole number
__device__ __forceinline__ u64 part_of(float x, u64 num, bool up) {
    const uint32_t bits = __float_as_uint(x);
    const int e = (int)(bits >> 23);
    const u64 mant = (bits & 0x7FFFFFu) | (e ? 0x800000u : 0u);
    const int right = 150 - (e ? e : 1);                           // x = mant 2^-right, right >= 24 for x < 1
    const u64 low = mant * num, high = __umul64hi(mant, num);
    u64 q, rest;
    if (right < 64) {
        q = (high << (64 - right)) | (low >> right);               // high < 2^24 <= 2^right
        rest = low & ((1ull << right) - 1);
    } else if (right < 128) {
        q = right == 64 ? high : high >> (right - 64);
        rest = low | (right == 64 ? 0 : high & ((1ull << (right - 64)) - 1));
    } else {
        q = 0;
        rest = low | high;
    }
    return q + (up && rest != 0 ? 1 : 0);
}

// The weight that the running sum has to pass for the pick.  (The largest entry always stays: total >= 1.)
__device__ __forceinline__ u64 target_of(float u, u64 total) { return u < 1.f ? (u > 0.f ? part_of(u, total, false) : 0) : total - 1; }

// where four logits lie
struct Places {
    int first, step;
    __device__ __forceinline__ int operator()(int e) const { return first + e * step; }
};
template <typename T> struct Four;
template <> struct Four<float> { using type = uint4; };
template <> struct Four<__nv_bfloat16> { using type = uint2; };

template <typename T>
__device__ __forceinline__ float load1(const T* p) { return clean(to_f32(*p)); }

template <typename V>
__device__ __forceinline__ V warp_total(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ u64 warp_largest(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// What comes before a thread's (n, w) in thread order.  All threads call it.
__device__ __forceinline__ void block_before(Shared& s, uint32_t n, u64 w, uint32_t& before_n, u64& before_w) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t in = n;
    u64 iw = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t un = __shfl_up_sync(0xffffffffu, in, o);
        const u64 uw = __shfl_up_sync(0xffffffffu, iw, o);
        if (lane >= o) { in += un; iw += uw; }
    }
    __syncthreads();
    if (lane == 31) { s.warp_n[warp] = in; s.warp_w[warp] = iw; }
    __syncthreads();
    before_n = in - n;
    before_w = iw - w;
    for (int i = 0; i < warp; ++i) { before_n += s.warp_n[i]; before_w += s.warp_w[i]; }
}

// Sorts list[0 .. size) falling, size a power of two of 64 to LIST.  A bitonic network with two neighbouring entries per thread: the
// strides within a thread or a warp are exchanged by registers, only those of 64 and more go through shared memory and a barrier.
__device__ __forceinline__ void sort_list(u64* list, int size) {
    const int i0 = 2 * threadIdx.x;
    const bool active = i0 < size;                                 // (whole warps)
    __syncthreads();
    u64 x0 = active ? list[i0] : 0, x1 = active ? list[i0 + 1] : 0;
    for (int k = 2; k <= size; k <<= 1) {
        const bool falling = (i0 & k) == 0;
        for (int j = k >> 1; j >= 64; j >>= 1) {
            __syncthreads();
            if (active) { list[i0] = x0; list[i0 + 1] = x1; }
            __syncthreads();
            if (active) {
                const u64 y0 = list[i0 ^ j], y1 = list[(i0 ^ j) + 1];
                const bool larger = ((i0 & j) == 0) == falling;
                x0 = larger ? max(x0, y0) : min(x0, y0);
                x1 = larger ? max(x1, y1) : min(x1, y1);
            }
        }
        if (active) {
            for (int j = min(k >> 1, 32); j > 1; j >>= 1) {
                const u64 y0 = __shfl_xor_sync(0xffffffffu, x0, j >> 1), y1 = __shfl_xor_sync(0xffffffffu, x1, j >> 1);
                const bool larger = ((i0 & j) == 0) == falling;
                x0 = larger ? max(x0, y0) : min(x0, y0);
                x1 = larger ? max(x1, y1) : min(x1, y1);
            }
            const u64 hi = max(x0, x1), lo = min(x0, x1);
            x0 = falling ? hi : lo;
            x1 = falling ? lo : hi;
        }
    }
    __syncthreads();
    if (active) { list[i0] = x0; list[i0 + 1] = x1; }
    __syncthreads();
}

template <typename T, bool STAGED>
__global__ void __launch_bounds__(THREADS, 2)
sample_filtered_kernel(const Args a) {
    extern __shared__ __align__(16) uint8_t sf_smem[];
    Shared& s = *reinterpret_cast<Shared*>(sf_smem);
    float* staged = reinterpret_cast<float*>(sf_smem + ((sizeof(Shared) + 15) & ~(size_t)15));
    cg::cluster_group cluster = cg::this_cluster();
    // A CTA's shared memory may be touched by the others only once it runs: each says so here, and waits for all of them before its first
    // store to another.  What lies between, the load of the stretch, hides the barrier.
    auto started = cluster.barrier_arrive();
    pdl_trigger();
    pdl_wait();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int r = blockIdx.x / ranks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int lo = min(a.vocab, rank * a.per), count = min(a.vocab, lo + a.per) - lo;
    const T* row = reinterpret_cast<const T*>(a.logits) + (size_t)r * a.ld + lo;
    // A warp owns a contiguous part of the stretch, so the warps' sums are in the order of the vocabulary.
    constexpr int VEC = 16 / sizeof(T);
    const int seg = ((count + WARPS - 1) / WARPS + 7) / 8 * 8, s0 = min(count, warp * seg), s1 = min(count, s0 + seg);
    const bool aligned = ((uintptr_t)row & 15) == 0;
    auto value = [&](int i) -> float { return STAGED ? staged[i] : load1(row + i); };
    // f(four logits, their places in the stretch) over a part of it by one warp, the next four on their way meanwhile; places at or
    // beyond `to` come as minus infinity.
    auto visit = [&](int from, int to, auto f) __attribute__((always_inline)) {
        if (STAGED) {
            for (int i = from + 4 * lane; i < to; i += 128) {      // (from is a multiple of 8; behind the stretch lie minus infinities)
                const float4 x = *reinterpret_cast<const float4*>(staged + i);
                const float v[4] = {x.x, i + 1 < to ? x.y : -INFINITY, i + 2 < to ? x.z : -INFINITY, i + 3 < to ? x.w : -INFINITY};
                f(v, Places{i, 1});
            }
        } else if (aligned) {
            using Raw = typename Four<T>::type;
            const int whole = to & ~3;                             // (from is a multiple of 8)
            int i = from + 4 * lane;
            Raw raw{}, next{};
            if (i < whole) raw = *reinterpret_cast<const Raw*>(row + i);
            for (; i < whole; i += 128) {
                if (i + 128 < whole) next = *reinterpret_cast<const Raw*>(row + i + 128);
                const T* x = reinterpret_cast<const T*>(&raw);
                const float v[4] = {clean(to_f32(x[0])), clean(to_f32(x[1])), clean(to_f32(x[2])), clean(to_f32(x[3]))};
                f(v, Places{i, 1});
                raw = next;
            }
            if (from <= whole && whole < to) {                     // the last ones, by the first lanes (an empty part has none)
                const float v[4] = {whole + lane < to ? load1(row + whole + lane) : -INFINITY, -INFINITY, -INFINITY, -INFINITY};
                f(v, Places{whole + lane, 32});
            }
        } else {
            for (int i = from + lane; i < to; i += 128) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = i + 32 * e < to ? load1(row + i + 32 * e) : -INFINITY;
                f(v, Places{i, 32});
            }
        }
    };
    // f(logit, place) for those of a part that `pick` takes: few
    auto visit_some = [&](int from, int to, auto pick, auto f) __attribute__((always_inline)) {
        visit(from, to, [&](const float (&v)[4], Places at) {
            uint32_t hits = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) hits |= pick(v[e], at(e)) ? 1u << e : 0u;
            for (; hits; hits &= hits - 1) {
                const int i = at(__ffs(hits) - 1);
                f(value(i), i);
            }
        });
    };

    for (int i = tid; i < STEPS; i += THREADS) s.table[i] = exp2((double)i / STEPS);
    if (tid < 2) s.gathered[tid] = 0;

    // ---- the stretch into shared memory, every thread's first largest entry ----
    u64 mine = 0;                                                  // (0: no number above minus infinity)
    {
        float most = -INFINITY;
        int place = 0;
        auto look = [&](float v, int i) {
            if (v > most) { most = v; place = i; }
        };
        int done = 0;
        if (aligned) {
            const int vecs = count / VEC;
            const uint4* src = reinterpret_cast<const uint4*>(row);
            for (int i = tid; i < vecs; i += 4 * THREADS) {
                uint4 raw[4];                                      // 64 bytes a thread on their way at once
#pragma unroll
                for (int u = 0; u < 4; ++u) raw[u] = i + u * THREADS < vecs ? src[i + u * THREADS] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (i + u * THREADS >= vecs) break;
                    const T* x = reinterpret_cast<const T*>(&raw[u]);
                    const int at = (i + u * THREADS) * VEC;
#pragma unroll
                    for (int e = 0; e < VEC; e += 4) {
                        float4 v;
                        v.x = clean(to_f32(x[e])); v.y = clean(to_f32(x[e + 1])); v.z = clean(to_f32(x[e + 2])); v.w = clean(to_f32(x[e + 3]));
                        look(v.x, at + e); look(v.y, at + e + 1); look(v.z, at + e + 2); look(v.w, at + e + 3);
                        if (STAGED) *reinterpret_cast<float4*>(staged + at + e) = v;
                    }
                }
            }
            done = vecs * VEC;
        }
        for (int i = done + tid; i < (STAGED ? a.per : count); i += THREADS) {
            const float v = i < count ? load1(row + i) : -INFINITY;
            if (STAGED) staged[i] = v;
            look(v, i);
        }
        if (most > -INFINITY) mine = entry(most, lo + place);
    }
    // The largest entries of 512 to 1,024 groups that share no entry, in every CTA: the k-th largest of them is a place at or above
    // which at least k entries of the row lie, and not many more while k is well below the number of groups.
    u64* largest = reinterpret_cast<u64*>(s.n);                    // (before the first histogram)
    const int groups = ranks == 1 ? THREADS : 2 * THREADS;
    {
        const int group = ranks > 2 ? ranks / 2 : 1;               // threads that share one
        for (int o = 1; o < group; o <<= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
        cluster.barrier_wait(std::move(started));
        if (tid % group == 0)
            for (int k = 0; k < ranks; ++k) *cluster.map_shared_rank(&largest[rank * (groups / ranks) + tid / group], k) = mine;
    }
    cluster.sync();
    const float temp = a.temperature[r];
    const int top_k = a.top_k && a.top_k[r] > 0 && a.top_k[r] < a.vocab ? a.top_k[r] : 0;          // 0: all
    const float top_p = a.top_p && a.top_p[r] < 1.f ? fmaxf(a.top_p[r], 0.f) : 1.f;                // 1: all
    u64 top = 0, from = 0;                                         // the row's first largest entry; where a list of candidates begins
    for (int i = tid; i < groups; i += THREADS) top = max(top, largest[i]);
    top = warp_largest(top);
    if (lane == 0) s.warp_w[warp] = top;
    __syncthreads();
    top = warp_largest(lane < WARPS ? s.warp_w[lane] : 0);
    // About -groups log(1 - k / groups) entries of rows without order lie at or above the k-th of the groups' largest: 720 at 386 of
    // 512 and 516 of 1,024, which the list takes with room to spare.
    const int likely = ranks == 1 ? 386 : 516;
    if (temp > 0.f && top_k > 0 && top_k <= groups) {
        // the upper 22 bits of its logit are enough, the lowest logit of those bits is below it by less than 2^-13 of itself
        const uint32_t x0 = (uint32_t)(largest[tid] >> 32), x1 = ranks == 1 ? 0 : (uint32_t)(largest[tid + THREADS] >> 32);
        uint32_t key = 0;
        for (uint32_t bit = 1u << 31; bit >= 1u << 10; bit >>= 1) {
            const uint32_t trial = key | bit;
            const int n = __syncthreads_count(x0 >= trial) + (ranks == 1 ? 0 : __syncthreads_count(x1 >= trial));
            if (n >= top_k) key = trial;
        }
        from = (u64)key << 32;                                     // (0: fewer groups than top_k have an entry)
    }
    if (temp > 0.f && top_p >= 1.f && top_k == 0 && a.min_p && a.min_p[r] > 0.f) from = ALL;       // (min_p alone)
    if (a.vocab <= LIST && (top_k > 0 || top_p < 1.f)) from = max(from, ALL);
    __syncthreads();                                               // (the histograms take the groups' place)

    if (top == 0 || !(temp > 0.f)) {                               // nothing to pick from, or greedy
        if (rank == 0 && tid == 0) {
            a.out[r] = top == 0 ? 0 : (int)~(uint32_t)top;
            if (a.kept) a.kept[r] = top == 0 ? 0 : 1;
        }
        return;                                                    // (no CTA looks into another from here on)
    }
    const float topf = unordered((uint32_t)(top >> 32));
    Weights weight;
    weight.top = topf; weight.topf = topf; weight.rate = STEPS * 1.4426950408889634074 / (double)temp; weight.least = topf < INFINITY ? topf - 43.5f * temp : INFINITY; weight.table = s.table;
    weight.shift = a.shift;
    // Entries below floor_v lie beyond every cut: the last bin is theirs.
    float floor_v = from > ALL ? unordered((uint32_t)(from >> 32)) : -INFINITY;
    if (top_k == 0 && top_p < 1.f) {
        // all weigh at least what the groups' largest weigh, M; entries of at most (1 - top_p) M / vocab weigh at most (1 - top_p) of
        // all together, so top_p is reached before them
        u64 w = 0;
        for (int i = tid; i < groups; i += THREADS) w += largest[i] ? weight(unordered((uint32_t)(largest[i] >> 32))) : 0;
        w = warp_total(w);
        __syncthreads();
        if (lane == 0) s.warp_w[warp] = w;
        __syncthreads();
        w = warp_total(lane < WARPS ? s.warp_w[lane] : 0);
        const double least_w = (double)((w - part_of(top_p, w, true)) / (u64)a.vocab) * exp2(-(double)a.shift);
        // (less by far more than the logarithm's and the product's rounding)
        floor_v = __double2float_rd((double)topf + (double)temp * (log(least_w) - 1e-9) - 1e-9 * fabs((double)topf));
        if (!(floor_v <= topf)) floor_v = -INFINITY;
        __syncthreads();                                           // (the histograms take the groups' place)
    }
    const float per_bin = floor_v > -INFINITY && floor_v < topf && topf < INFINITY ? (float)(BINS - 1) / (topf - floor_v) : (float)BINS / (BIN_RANGE * temp);
    // the bin of a logit: never falls as the logit falls, whatever the rounding
    auto bin_of = [&](float v) -> int {                            // (rounded down by adding 2^23)
        const int b = __float_as_int(__fadd_rz(fminf((topf - v) * per_bin, (float)(BINS - 1)), 8388608.0f)) & (BINS - 1);
        return v == topf ? 0 : v < floor_v ? BINS - 1 : b;
    };
    // whether an entry lies at or above a place in the order
    auto at_least = [&](float v, int index, u64 place) -> bool {
        const float pv = unordered((uint32_t)(place >> 32));
        return v > pv || (v == pv && (uint32_t)index <= ~(uint32_t)place);
    };

    auto kept_weight = [&](float v, int i, u64 cut) -> u64 { return v > -INFINITY && at_least(v, lo + i, cut) ? weight(v) : 0; };

    // The cluster's histogram over the entries that `take` maps to a bin (-1: none): a thread gets its two bins' sums.
    bool first_histogram = true;
    auto histogram = [&](auto weighed, auto take, uint32_t (&n)[2], u64 (&w)[2]) __attribute__((always_inline)) {
        constexpr bool weights = decltype(weighed)::value;
        if (!first_histogram) cluster.sync();                      // the others have read the one before
        first_histogram = false;
        for (int i = tid; i < BINS; i += THREADS) { s.n[i] = 0; s.lo[i] = 0; s.hi[i] = 0; }
        __syncthreads();
        auto add_weight = [&](int b, u64 x) {
            const uint32_t low = (uint32_t)x, old = atomicAdd(&s.lo[b], low);
            const uint32_t high = (uint32_t)(x >> 32) + (old + low < old ? 1u : 0u);
            if (high) atomicAdd(&s.hi[b], high);
        };
        // (the last bin, where the many unlikely entries fall, is counted apart: atomics on one place go one after the other)
        uint32_t last_n = 0;
        u64 last_w = 0;
        visit(s0, s1, [&](const float (&v)[4], Places at) {
            int b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                b[e] = take(v[e], lo + at(e));
                if (b[e] == BINS - 1) ++last_n;
                else if (b[e] >= 0) atomicAdd(&s.n[b[e]], 1u);
            }
            if (weights) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const u64 x = weight(v[e]);
                    if (b[e] == BINS - 1) last_w += x;
                    else if (b[e] >= 0) add_weight(b[e], x);
                }
            }
        });
        last_n = warp_total(last_n);
        if (weights) last_w = warp_total(last_w);
        if (lane == 0 && last_n) {
            atomicAdd(&s.n[BINS - 1], last_n);
            if (weights) add_weight(BINS - 1, last_w);
        }
        cluster.sync();
        if (ranks == 1) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                n[i] = s.n[2 * tid + i];
                w[i] = weights ? ((u64)s.hi[2 * tid + i] << 32) + s.lo[2 * tid + i] : 0;
            }
            return;
        }
        // a CTA sums its share of the bins and gives the sums to all (each summing all bins reads eight times as much from the others)
        const int share = BINS / ranks;
        for (int i = rank * share + tid; i < (rank + 1) * share; i += THREADS) {
            uint32_t sum_n = 0;
            u64 sum_w = 0;
            uint32_t x[MOST_RANKS];                                // all on their way at once
#pragma unroll
            for (int k = 0; k < MOST_RANKS; ++k) x[k] = k < ranks ? cluster.map_shared_rank(&s, k)->n[i] : 0;
#pragma unroll
            for (int k = 0; k < MOST_RANKS; ++k) sum_n += x[k];
            if (weights) {
                uint32_t y[MOST_RANKS];
#pragma unroll
                for (int k = 0; k < MOST_RANKS; ++k) {
                    x[k] = k < ranks ? cluster.map_shared_rank(&s, k)->lo[i] : 0;
                    y[k] = k < ranks ? cluster.map_shared_rank(&s, k)->hi[i] : 0;
                }
#pragma unroll
                for (int k = 0; k < MOST_RANKS; ++k) sum_w += ((u64)y[k] << 32) + x[k];
            }
            for (int k = 0; k < ranks; ++k) {
                Shared* other = cluster.map_shared_rank(&s, k);
                other->all_n[i] = sum_n;
                if (weights) other->all_w[i] = sum_w;
            }
        }
        cluster.sync();
#pragma unroll
        for (int i = 0; i < 2; ++i) { n[i] = s.all_n[2 * tid + i]; w[i] = weights ? s.all_w[2 * tid + i] : 0; }
    };
    // The entries that `in` takes, LIST at most, into the first CTA's list, in any order.
    auto gather = [&](auto in) {
        Shared* first = cluster.map_shared_rank(&s, 0);
        visit_some(s0, s1, [&](float v, int i) { return in(v, lo + i); }, [&](float v, int i) {
            const unsigned here = __activemask();                  // (the lanes that are here together ask once)
            const int leader = __ffs(here) - 1;
            uint32_t place = 0;
            if (lane == leader) place = atomicAdd(&first->gathered[1], (uint32_t)__popc(here));
            place = __shfl_sync(here, place, leader) + __popc(here & ((1u << lane) - 1u));
            first->list[place] = entry(v, lo + i);
        });
        cluster.sync();
    };
    auto kept_bound = [&]() -> u64 {                               // min_p as a bound on the logit: w >= min_p
        if (!a.min_p || !(a.min_p[r] > 0.f)) return ALL;
        const float p = a.min_p[r];
        if (p > 1.f) return top;                                   // only the first largest entry stays
        // (what is below an infinite logit weighs nothing, at an infinite temperature too)
        const float bound = topf < INFINITY ? __double2float_ru((double)topf + (double)temp * log((double)p)) : topf;
        return bound > -INFINITY ? (u64)ordered(bound + 0.0f) << 32 : ALL;
    };

    // All that is left to do, by the first CTA alone, where the list holds a beginning of the order that reaches beyond every cut:
    // sorts it, cuts it, and picks from what stays in the order of the vocabulary.  need: the weight before which entries stay, 0:
    // top_p of the first top_k's weight, which the list holds.
    auto finish = [&](int size, u64 need) {
        if (size <= FEW) {
            // each entry with each: what comes before it in the order, then in the vocabulary (a sort of so few waits at its barriers
            // for longer)
            u64* ws = reinterpret_cast<u64*>(s.n);                 // (the histograms have been read)
            const u64 e = tid < size ? s.list[tid] : 0;
            const u64 x = e ? weight(unordered((uint32_t)(e >> 32))) : 0;
            if (tid < FEW) ws[tid] = x;
            __syncthreads();
            uint32_t ahead = 0;
            u64 ahead_w = 0;
            if (warp * 32 < size) {
#pragma unroll 4
                for (int j = 0; j < size; ++j)
                    if (s.list[j] > e) { ++ahead; ahead_w += ws[j]; }
            }
            const bool among = e != 0 && (top_k == 0 || ahead < (uint32_t)top_k);
            uint32_t bn;
            u64 bw;
            if (need == 0) {
                if (top_p < 1.f) {
                    block_before(s, 0, among ? x : 0, bn, bw);
                    if (tid == THREADS - 1) s.total_w = bw + (among ? x : 0);
                    __syncthreads();
                    need = max(part_of(top_p, s.total_w, true), 1ull);
                } else need = ~0ull;
            }
            const bool stays = among && (ahead == 0 || (ahead_w < need && e >= kept_bound()));
            __syncthreads();
            if (tid < FEW) ws[tid] = stays ? x : 0;
            const int stay = __syncthreads_count(stays);
            if (stays) {
                u64 before = 0, whole = 0;
#pragma unroll 4
                for (int j = 0; j < size; ++j) {
                    const u64 y = ws[j];
                    whole += y;
                    if ((uint32_t)s.list[j] > (uint32_t)e) before += y;                    // (the larger is the smaller index)
                }
                const u64 target = target_of(a.uniform[r], whole);
                if (before <= target && target < before + x) {
                    a.out[r] = (int)~(uint32_t)e;
                    if (a.kept) a.kept[r] = stay;
                }
            }
            return;
        }
        int pow2 = 64;
        while (pow2 < size) pow2 <<= 1;
        for (int i = size + tid; i < pow2; i += THREADS) s.list[i] = 0;
        sort_list(s.list, pow2);
        const int stay_k = top_k > 0 ? min(size, top_k) : size, i0 = 2 * tid;
        const u64 e[2] = {i0 < stay_k ? s.list[i0] : 0, i0 + 1 < stay_k ? s.list[i0 + 1] : 0};
        u64 x[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) x[i] = e[i] ? weight(unordered((uint32_t)(e[i] >> 32))) : 0;
        uint32_t bn;
        u64 bw;
        block_before(s, 0, x[0] + x[1], bn, bw);
        if (tid == THREADS - 1) s.total_w = bw + x[0] + x[1];
        if (tid == 0) s.found = 0;
        __syncthreads();
        if (need == 0) need = top_p < 1.f ? max(part_of(top_p, s.total_w, true), 1ull) : ~0ull;
        const u64 bound = kept_bound();
        if (e[0] && bw < need && e[0] >= bound) atomicMax(&s.found, (uint32_t)i0 + 1);
        if (e[1] && bw + x[0] < need && e[1] >= bound) atomicMax(&s.found, (uint32_t)i0 + 2);
        __syncthreads();
        const int stay = max(1, (int)s.found);                     // (the first entry always stays)
        // The pick: the smallest index up to which more than the target weighs, bit by bit of its complement (which e holds), from
        // the top: entries whose complement is at least `trial` are those up to an index.
        const bool in0 = i0 < stay, in1 = i0 + 1 < stay;
        const uint32_t c0 = (uint32_t)e[0], c1 = (uint32_t)e[1];
        auto weight_from = [&](uint32_t least) -> u64 {
            u64 w = warp_total((in0 && c0 >= least ? x[0] : 0) + (in1 && c1 >= least ? x[1] : 0));
            __syncthreads();
            if (lane == 0) s.warp_w[warp] = w;
            __syncthreads();
            return warp_total(lane < WARPS ? s.warp_w[lane] : 0);
        };
        const u64 target = target_of(a.uniform[r], weight_from(0));
        uint32_t least = 0xff000000u;                              // (indexes have 24 bits)
        for (uint32_t bit = 1u << 23; bit != 0; bit >>= 1)
            if (weight_from(least | bit) > target) least |= bit;   // the largest complement from which on enough weighs
        if ((in0 && c0 == least) || (in1 && c1 == least)) {
            a.out[r] = (int)~least;
            if (a.kept) a.kept[r] = stay;
        }
    };

    // The cut behind the last entry kept: entries are counted (by_rank: the first top_k of the order stay) or weighed (those stay before
    // which less than top_p of the total weighs), over the entries at or above `least`.  Returns 0 where the first CTA has finished
    // the row: the beginning of the order up to the cut's bin fits the list.
    auto find_cut = [&](auto counted, u64 least) __attribute__((always_inline)) -> u64 {
        constexpr bool by_rank = decltype(counted)::value;
        u64 need = by_rank ? (u64)top_k : 0;
        uint32_t before_n = 0;
        u64 before_w = 0;
        int chosen_bin = -1;                                       // the bin of equal width, then the prefix of the ordered logit
        uint32_t prefix = 0;
        for (int level = 0; ; ++level) {
            // level 0: bins of equal width; levels 1 to 4: the next 10, 10, 10 and 2 bits of the ordered logit
            const int down = level == 0 ? 32 : level < 4 ? 32 - 10 * level : 0, up = level == 1 ? 0 : 42 - 10 * level;
            uint32_t hn[2];
            u64 hw[2];
            histogram(std::bool_constant<!by_rank>{}, [&](float v, int index) -> int {
                if (!(v > -INFINITY) || !at_least(v, index, least)) return -1;
                const int b = bin_of(v);
                if (level == 0) return b;
                const uint32_t k = ordered(v);
                if (b != chosen_bin || (level > 1 && (k >> (level == 4 ? 2 : up)) != prefix)) return -1;
                return BINS - 1 - (int)((k >> down) & (level == 4 ? 3u : 1023u));
            }, hn, hw);
            uint32_t bn;
            u64 bw;
            block_before(s, hn[0] + hn[1], hw[0] + hw[1], bn, bw);
            if (level == 0) {
                if (tid == THREADS - 1) { s.total_n = bn + hn[0] + hn[1]; s.total_w = bw + hw[0] + hw[1]; }
                __syncthreads();
                if (by_rank) {
                    if (need >= s.total_n) return least;           // there are no more than top_k
                } else {
                    need = max(part_of(top_p, s.total_w, true), 1ull);               // (the first entry always stays)
                }
            }
            // the first bin at whose end the count or the weight has been reached
            bn += before_n;
            bw += before_w;
            const u64 at = by_rank ? bn : bw, x0 = by_rank ? hn[0] : hw[0], x1 = by_rank ? hn[1] : hw[1];
            if (at < need && at + x0 >= need) { s.bin = 2 * tid; s.before_n = bn; s.before_w = bw; s.found = hn[0]; }
            else if (at + x0 < need && at + x0 + x1 >= need) { s.bin = 2 * tid + 1; s.before_n = bn + hn[0]; s.before_w = bw + hw[0]; s.found = hn[1]; }
            __syncthreads();
            before_n = s.before_n;
            before_w = s.before_w;
            const int bin = (int)s.bin;
            const uint32_t found = s.found;
            if (level == 0 && before_n + found <= LIST) {
                gather([&](float v, int index) { return v > -INFINITY && bin_of(v) <= bin && at_least(v, index, least); });
                if (rank == 0) finish((int)(before_n + found), by_rank ? 0 : need);
                return 0;
            }
            if (level == 0) chosen_bin = bin;
            else prefix = level == 4 ? prefix : (level == 1 ? 0u : prefix << 10) | (uint32_t)(BINS - 1 - bin);
            const uint32_t last_digit = level == 4 ? (uint32_t)(BINS - 1 - bin) : 0u;
            auto in_set = [&](float v, int index) -> bool {
                if (!(v > -INFINITY) || !at_least(v, index, least) || bin_of(v) != chosen_bin) return false;
                const uint32_t k = ordered(v);
                if (level == 4) return k == ((prefix << 2) | last_digit);
                return level == 0 || (k >> down) == prefix;
            };
            if (found <= LIST) {
                // the bin's entries to every CTA of the cluster, sorted there
                uint32_t mine = s.n[bin], first = 0;
                for (int k = 0; k < rank; ++k) first += cluster.map_shared_rank(&s, k)->n[bin];
                if (tid == 0) s.list_n = first;
                int size = 64;
                while (size < (int)found) size <<= 1;
                for (int i = (int)found + tid; i < size; i += THREADS) s.list[i] = 0;
                __syncthreads();
                if (mine) {
                    visit_some(s0, s1, [&](float v, int i) { return in_set(v, lo + i); }, [&](float v, int i) {
                        const uint32_t at_list = atomicAdd(&s.list_n, 1u);
                        for (int k = 0; k < ranks; ++k) cluster.map_shared_rank(&s, k)->list[at_list] = entry(v, lo + i);
                    });
                }
                cluster.sync();
                sort_list(s.list, size);
                if (by_rank) return s.list[need - before_n - 1];
                const int i0 = 2 * tid;
                const u64 e0 = i0 < (int)found ? s.list[i0] : 0, e1 = i0 + 1 < (int)found ? s.list[i0 + 1] : 0;
                const u64 v0 = e0 ? weight(unordered((uint32_t)(e0 >> 32))) : 0, v1 = e1 ? weight(unordered((uint32_t)(e1 >> 32))) : 0;
                block_before(s, 0, v0 + v1, bn, bw);
                bw += before_w;
                // the last one before which less than `need` weighs
                if (e1 && bw + v0 < need) atomicMax(&s.found, (uint32_t)(i0 + 1) + 0x40000000u);
                else if (e0 && bw < need) atomicMax(&s.found, (uint32_t)i0 + 0x40000000u);
                __syncthreads();
                return s.list[s.found - 0x40000000u];
            }
            if (level == 4) {
                // more equal logits than the list holds: the first so many by index
                const float v = unordered((prefix << 2) | last_digit);
                u64 stay;
                if (by_rank) stay = need - before_n;
                else {
                    const u64 w = weight(v);
                    stay = w ? min((u64)found, (need - before_w + w - 1) / w) : found;
                }
                uint32_t n = 0;
                visit(s0, s1, [&](const float (&v)[4], Places at) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) n += in_set(v[e], lo + at(e)) ? 1u : 0u;
                });
                n = warp_total(n);
                __syncthreads();
                if (lane == 0) s.warp_n[warp] = n;
                __syncthreads();
                if (tid == 0) {
                    uint32_t total = 0;
                    for (int i = 0; i < WARPS; ++i) total += s.warp_n[i];
                    s.part_n = total;
                    s.found_cut = 0;
                }
                cluster.sync();
                u64 first = 0;
                for (int k = 0; k < rank; ++k) first += cluster.map_shared_rank(&s, k)->part_n;
                for (int i = 0; i < warp; ++i) first += s.warp_n[i];
                if (first < stay && stay <= first + n) {           // this warp holds the last one that stays (warp-uniform)
                    for (int i = s0 + lane; i - lane < s1; i += 32) {
                        const bool is = i < s1 && in_set(value(i), lo + i);
                        const unsigned mask = __ballot_sync(0xffffffffu, is);
                        if (is && first + __popc(mask & ((2u << lane) - 1u)) == stay)
                            for (int k = 0; k < ranks; ++k) cluster.map_shared_rank(&s, k)->found_cut = entry(v, lo + i);
                        first += __popc(mask);
                    }
                }
                cluster.sync();
                return s.found_cut;
            }
        }
    };

    // ---- a list of candidates: a beginning of the order that reaches beyond every cut, if it is short enough ----
    if (from != 0 && (top_k <= likely || a.vocab <= LIST)) {
        from = max(from, top_p >= 1.f ? kept_bound() : ALL);       // (top_p is of all that top_k leaves)
        Shared* first = cluster.map_shared_rank(&s, 0);
        visit_some(s0, s1, [&](float v, int i) { return at_least(v, lo + i, from); }, [&](float v, int i) {
            if (*reinterpret_cast<volatile uint32_t*>(&s.gathered[0]) > LIST) return;          // (too many: every CTA will find so)
            const unsigned here = __activemask();                  // (the lanes that are here together ask once)
            const int leader = __ffs(here) - 1;
            uint32_t place = 0;
            if (lane == leader) {
                place = atomicAdd(&first->gathered[0], (uint32_t)__popc(here));
                for (int k = 1; k < ranks; ++k) atomicAdd(&cluster.map_shared_rank(&s, k)->gathered[0], (uint32_t)__popc(here));
            }
            place = __shfl_sync(here, place, leader) + __popc(here & ((1u << lane) - 1u));
            if (place < LIST) first->list[place] = entry(v, lo + i);
        });
        cluster.sync();
        if (s.gathered[0] <= LIST) {
            if (rank == 0) finish((int)s.gathered[0], 0);
            return;
        }
    }

    // ---- cuts that lie further down: by histograms ----
    u64 cut = ALL;
    if (top_k > 0 && (cut = find_cut(std::true_type{}, cut)) == 0) return;
    if (top_p < 1.f && (cut = find_cut(std::false_type{}, cut)) == 0) return;
    cut = max(cut, kept_bound());

    // ---- the kept weights in vocabulary order: warps own contiguous parts, whose sums are whole numbers ----
    u64 w = 0;
    uint32_t n = 0;
    visit(s0, s1, [&](const float (&v)[4], Places at) {
        bool stays[4], any = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            stays[e] = v[e] > -INFINITY && at_least(v[e], lo + at(e), cut);
            any |= stays[e];
        }
        if (any) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u64 x = weight(v[e]);
                if (stays[e]) { w += x; ++n; }
            }
        }
    });
    w = warp_total(w);
    n = warp_total(n);
    __syncthreads();
    if (lane == 0) { s.warp_w[warp] = w; s.warp_n[warp] = n; }
    __syncthreads();
    if (warp == 0) {
        const u64 tw = warp_total(lane < WARPS ? s.warp_w[lane] : 0);
        const uint32_t tn = warp_total(lane < WARPS ? s.warp_n[lane] : 0);
        if (lane == 0) { s.part_w = tw; s.part_n = tn; }
    }
    cluster.sync();
    const u64 his_w = lane < ranks ? cluster.map_shared_rank(&s, lane)->part_w : 0;
    const uint32_t his_n = lane < ranks ? cluster.map_shared_rank(&s, lane)->part_n : 0;
    const u64 whole = warp_total(his_w), before_cta = warp_total(lane < rank ? his_w : 0);
    const uint32_t kept = warp_total(his_n);
    const u64 target = target_of(a.uniform[r], whole);
    const u64 cta_w = __shfl_sync(0xffffffffu, his_w, rank);
    if (before_cta <= target && target < before_cta + cta_w) {     // (the whole CTA) the pick lies in this stretch
        // the warp's part that holds it, cut into parts for all warps once more
        u64 before = before_cta;
        int part = 0;
        while (part < WARPS - 1 && target >= before + s.warp_w[part]) before += s.warp_w[part++];
        const int p0 = min(count, part * seg), p1 = min(count, p0 + seg), sub = ((seg + WARPS - 1) / WARPS + 7) / 8 * 8;
        const int q0 = min(p1, p0 + warp * sub), q1 = min(p1, q0 + sub);
        u64 x = 0;
        visit(q0, q1, [&](const float (&v)[4], Places at) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x += kept_weight(v[e], at(e), cut);
        });
        x = warp_total(x);
        __syncthreads();                                           // (the parts' sums have been read)
        if (lane == 0) s.warp_w[warp] = x;
        __syncthreads();
        before += warp_total(lane < warp ? s.warp_w[lane] : 0);
        if (before <= target && target < before + x) {             // (warp-uniform)
            for (int i = q0 + lane; i - lane < q1; i += 32) {
                const u64 mine = i < q1 ? kept_weight(value(i), i, cut) : 0;
                u64 incl = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 up = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += up;
                }
                const unsigned past = __ballot_sync(0xffffffffu, before + incl > target);
                if (past) {
                    if (lane == __ffs(past) - 1) {
                        a.out[r] = lo + i;
                        if (a.kept) a.kept[r] = (int)kept;
                    }
                    break;
                }
                before += __shfl_sync(0xffffffffu, incl, 31);
            }
        }
    }
    cluster.sync();
}

template <typename T>
static int launch_sample(const Args& a, int n_rows, int ranks, bool staged, cudaStream_t stream) {
    constexpr size_t fixed = (sizeof(Shared) + 15) & ~(size_t)15;
    const size_t smem = fixed + (staged ? (size_t)a.per * sizeof(float) : 0);
    auto kern = staged ? sample_filtered_kernel<T, true> : sample_filtered_kernel<T, false>;
    // the attribute is the device's: set once on each
    static bool configured[64][2] = {};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    if (device < 0 || device >= 64 || !configured[device][staged]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(fixed + (staged ? STAGED_MOST * sizeof(float) : 0)));
        if (e != cudaSuccess) return (int)e;
        if (device >= 0 && device < 64) configured[device][staged] = true;
    }
    e = timeline_note(reinterpret_cast<const void*>(kern));
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n_rows * ranks);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = imparo_pdl_enabled() ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kern, a);
    return e == cudaSuccess ? 0 : (int)e;
}

}  // namespace sf
}  // namespace imparo

using namespace imparo;

// logits [n_rows, vocab] with row stride ld, float32 or bfloat16; temperature and uniform [n_rows]; top_k, top_p, min_p [n_rows] or
// null; out [n_rows]; kept [n_rows] (how many entries the filters left) or null.
extern "C" int imparo_sample_filtered(const void* logits, int dtype, long long ld, const float* temperature, const float* uniform,
                                      const int* top_k, const float* top_p, const float* min_p, int* out, int* kept, int n_rows,
                                      int vocab, cudaStream_t stream) {
    if (n_rows <= 0) return 0;
    if (!temperature || !uniform) return -7;
    if (vocab < 1 || vocab > (1 << 24) || n_rows > (1 << 20) || ld < vocab) return -2;
    if (dtype != IMPARO_DT_F32 && dtype != IMPARO_DT_BF16) return -1;
    sf::Args a;
    a.logits = logits; a.temperature = temperature; a.uniform = uniform; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
    a.out = out; a.kept = kept; a.ld = ld; a.vocab = vocab;
    // As many CTAs per row as fill the chip about twice (two CTAs per SM), as long as each has 2,048 entries: a row's CTAs wait for one
    // another a few times, so more of them pay only where SMs would have nothing to do or a long row would hold up the end.
    int ranks = 1;
    while (ranks < sf::MOST_RANKS && vocab > 2048 * ranks && (long long)n_rows * ranks < 592) ranks <<= 1;
    a.per = ((vocab + ranks - 1) / ranks + 7) / 8 * 8;
    // sums of vocab weights of at most 2^shift stay below 2^62
    a.shift = 62;
    while ((1ll << (62 - a.shift)) < vocab) --a.shift;
    if (a.shift > 46) a.shift = 46;                                // (a weight is made as the low bits of a 52-bit number)
    const bool staged = a.per <= sf::STAGED_MOST;
    return dtype == IMPARO_DT_F32 ? sf::launch_sample<float>(a, n_rows, ranks, staged, stream)
                                  : sf::launch_sample<__nv_bfloat16>(a, n_rows, ranks, staged, stream);
}
