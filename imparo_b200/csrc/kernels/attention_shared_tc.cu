// The attention over a shared prefix on the 5th-generation tensor cores: bfloat16, head size 64 or 128, pages of 16, 32 or a
// multiple of 64 positions (attention_shared.cu says what is computed; it takes all other cases).
//
// Two kernels.  The first takes the shared keys: a CTA owns one stretch of keys and up to 512 rows (tokens of a group x query heads
// of one kv head) as four tiles of 128 rows, with head size 128 up to 256 rows as two, and leaves each row's partial result.  The
// second takes each row's own keys, and joins them with the partial results of the shared ones.
//
// Scores, the softmax's max and sum and all accumulators are 32-bit.  The weights exp(s - max) are rounded to bfloat16 for the second
// product (by 2^-8 of each at most), as in the engine's other bfloat16 attention kernels: the tensor cores take both operands in one
// 16-bit type, and the values are bfloat16.  Over prefixes of 8,000 to 100,000 positions the results are off by 2.2e-3 to 2.3e-3 of
// their root mean square from the formula in 64 bits; rounding the result alone gives 1.7e-3.
//
// On a B200, bfloat16, 32 heads in 8 groups of 64: 256 rows over 100,000 shared and up to 200 own positions 278 us (the first kernel about 260:
// 0.8 PFLOP/s of products, the exponential units busy for two thirds of it), 64 rows over 32,768 and up to 256 own ones 49 us.
#include "attention_shared.cuh"
#include "tcgen05.cuh"

namespace imparo {
namespace sp {

using namespace tc;

// ---- the shared keys ---------------------------------------------------------------------------------------------------
// One CTA per SM, 64 keys a step, TILES tiles of 128 rows (four with head size 64, two with 128: what tensor memory holds):
//   4 warps a tile  the softmax, one thread per row (= tensor-memory lane): the row's 64 scores of the step go into registers at once,
//                   P = exp2(s - max) goes back to the first half of their columns as bfloat16, where the second product reads it
//   1 warp          TMA: keys and values page by page (lane p fetches page p of a step) into rings with barriers of their own
//   2 warps         tcgen05.mma, each for every other tile: S = Q K^T (both from shared memory), O += P V (P from tensor memory)
// The output stays in tensor memory; it is scaled down only when a row's max has grown by more than 8 (in log2 units) since the max
// in use was taken, which leaves every term below 2^8 and the result the same.
// Rows that fill one or two tiles only are given to all of them: of P tiles with the same rows, each takes every P-th step, and the
// first one adds the others' results at the end.
constexpr int TILE = 128, STEP = 64;               // rows per tile, keys per step
constexpr uint32_t REGION = TILE * 128;            // [128 rows][64 dims] of queries in shared memory
constexpr uint32_t KEY_REGION = STEP * 128;        // [64 keys][64 dims] of keys or values
constexpr float GROW = 8.0f;
constexpr float LN2 = 0.69314718055994530942f, LOG2E = 1.4426950408889634074f;

template <int HD> struct Shape {
    static constexpr int NB = HD / 64;                       // 64-dim blocks of a head
    static constexpr int TILES = HD == 64 ? 4 : 2;
    static constexpr int S_BUFS = HD == 64 ? 1 : 2;          // steps whose scores a tile holds at once
    static constexpr int STAGES = HD == 64 ? 8 : 4;          // a multiple of TILES: a buffer always holds steps of the same tiles
    static constexpr int LOAD_WARP = 4 * TILES, MMA_WARP = LOAD_WARP + 1, THREADS = 32 * (LOAD_WARP + 3);
    static constexpr uint32_t Q_BYTES = NB * REGION, KEY_BYTES = NB * KEY_REGION;
    static constexpr uint32_t O_COL = TILES * S_BUFS * STEP;                 // tensor memory: scores (and P) first, then outputs
    static_assert(O_COL + TILES * HD == 512 && STAGES % TILES == 0, "tensor memory and stages");
    static constexpr int PAGES = 4096, REFILL = 1024;        // the copies' rows of the cache: a ring, filled so many at a time
    static constexpr size_t SMEM = 1024 + TILES * Q_BYTES + (size_t)STAGES * 2 * KEY_BYTES + 512 + PAGES * 4;
};

__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {           // values: [key][dim], the dims contiguous (MN-major)
    uint64_t d = 0;
    d |= (uint64_t)((addr & 0x3FFFF) >> 4);
    d |= (uint64_t)((KEY_REGION >> 4) & 0x3FFF) << 16;                 // 64-dim blocks
    d |= (uint64_t)(1024 >> 4) << 32;                                  // groups of 8 keys
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ uint32_t idesc(int n, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24);
}
// the product with its first operand in tensor memory (lane = row, two bfloat16 of K per column)
__device__ __forceinline__ void umma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
                 ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(accumulate) : "memory");
}
// One lane of a warp that is together.  The instructions of the tensor cores take their operands from registers that the whole warp
// shares: in the branch of an elected lane the compiler knows that there is one such value, in one on the lane's number it does not.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// the largest of three; no number if one of them is none
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ void arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// false when the wait ran out
__device__ __forceinline__ bool wait_at(uint32_t bar, uint32_t parity) {
    for (uint32_t it = 0; it < WAIT_LIMIT; ++it) {
        uint32_t done;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.b32 %0, 1, 0, p;\n}"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ void commit_at(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int HD>
__global__ void __launch_bounds__(Shape<HD>::THREADS, 1)
shared_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Args a, const int n_splits) {
    using C = Shape<HD>;
    constexpr int NB = C::NB, ST = C::STAGES, NT = C::TILES, SB = C::S_BUFS;
    extern __shared__ __align__(1024) uint8_t tc_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)tc_smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* q_s = smem;                                     // [NT][Q_BYTES]
    uint8_t* k_s = q_s + NT * C::Q_BYTES;                    // [ST][KEY_BYTES]
    uint8_t* v_s = k_s + ST * C::KEY_BYTES;                  // [ST][KEY_BYTES]
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + ST * C::KEY_BYTES);
    uint64_t* k_full = bars;                                 // [ST]
    uint64_t* k_empty = k_full + ST;
    uint64_t* v_full = k_empty + ST;
    uint64_t* v_empty = v_full + ST;
    uint64_t* q_ready = v_empty + ST;                        // [NT]
    uint64_t* s_ready = q_ready + NT;                        // [NT][SB] the tile's scores of a step are complete
    uint64_t* p_ready = s_ready + NT * SB;                   // [NT] the step's weights are written, the output is scaled
    uint64_t* o_done = p_ready + NT;                         // [NT] P V of the step is accumulated (with one buffer of scores: of the last step)
    uint64_t* drained = o_done + NT;                         // [2]  every product of an issuing warp has run
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert((4 * ST + NT * (3 + SB) + 2) * 8 + 8 <= 512, "barriers");

    timeline_begin();
    pdl_wait();
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int G = a.nh / a.nkv, TQ = TILE / G;               // tokens per tile
    const int kvh = blockIdx.x, chunk = blockIdx.y;
    int group = 0, unit = blockIdx.z, start = 0, end = 0;
    for (; group < a.n_groups; ++group) {
        group_rows(a, group, start, end);
        const int units = (end - start + NT * TQ - 1) / (NT * TQ);
        if (unit < units) break;
        unit -= units;
    }
    if (group >= a.n_groups) return;                         // the grid is an upper bound (uniform per CTA)
    const int row0 = start + unit * NT * TQ, n_tok = min(NT * TQ, end - row0);
    const int row_tiles = (n_tok + TQ - 1) / TQ;
    const int log_r = row_tiles > 2 ? 2 : row_tiles - 1, R = 1 << log_r;   // tile x: rows x % R, every phases-th step from x / R on
    const int phases = NT >> log_r;
    const int n_tiles = R > 2 ? row_tiles : NT;              // (a fourth tile without rows does nothing)
    const Span span = shared_span(a, group);
    const int per_chunk = a.chunk_shared / STEP;
    const int first_step = span.first / STEP + chunk * per_chunk;
    const int all_steps = (span.end + STEP - 1) / STEP;
    const int n_steps = span.first < span.end ? max(0, (chunk + 1 < a.n_shared ? min(all_steps, first_step + per_chunk) : all_steps) - first_step) : 0;
    if (n_steps == 0) {
        for (int i = threadIdx.x; i < n_tok * G; i += C::THREADS) {
            float* ml = a.part_ml + (((size_t)(row0 + i / G) * a.nh + kvh * G + i % G) * n_splits + chunk) * 2;
            ml[0] = -INFINITY;
            ml[1] = 0.f;
        }
        return;
    }

    if (threadIdx.x == 0) {
        const int readers = min(R, row_tiles);               // a step's keys and values are free when all tiles that use them have read them
        for (int s = 0; s < ST; ++s) {
            mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], readers);
            mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], readers);
        }
        for (int x = 0; x < NT; ++x) {
            mbar_init(&q_ready[x], 128); mbar_init(&p_ready[x], 128); mbar_init(&o_done[x], 1);
            for (int i = 0; i < SB; ++i) mbar_init(&s_ready[x * SB + i], 1);
        }
        mbar_init(&drained[0], 1);
        mbar_init(&drained[1], 1);
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == C::MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    // The next kernel may start now: everything before this one is complete (it reads what those wrote before it waits for this
    // one), and this CTA has its tensor memory, which no later kernel's CTA can hold any more while it waits for this one.
    pdl_trigger_late();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    // tile x works on the steps at(x, 0), at(x, 1), ... of the CTA's
    auto steps_of = [&](int x) { return x < n_tiles ? (n_steps - (x >> log_r) + phases - 1) / phases : 0; };
    auto at = [&](int x, int j) { return j * phases + (x >> log_r); };

    if (warp == C::LOAD_WARP) {
        // Keys and values are fetched as their buffers come free, whichever first.  Where the copies' rows lie is looked up a
        // thousand copies at a time: a lookup per copy is a trip to memory that every step then waits for.
        int* where = reinterpret_cast<int*>(bars + 64);      // [PAGES] first cache row of copy c of the CTA's, at c % PAGES
        const int* tab = table_row(a, span.row, 72);
        const int box = min(a.page_size, STEP), log_copies = box == 16 ? 2 : box == 32 ? 1 : 0, copies = 1 << log_copies;
        const int first_blk = span.first / a.page_size, last_blk = (span.end - 1) / a.page_size;
        int known = 0;
        auto look_up = [&]() {
            const int until = min(known + C::REFILL, n_steps << log_copies);
            for (int c = known + lane; c < until; c += 32) {
                // blocks in which nothing is seen: a page that is seen stands in for them (its values are cleared below)
                const int key = first_step * STEP + c * box, blk = min(max(key / a.page_size, first_blk), last_blk);
                int page = tab != nullptr && blk < a.max_blocks ? tab[blk] : -1;
                if (page < 0 || page >= a.n_pages) {
                    report(a.status, IMPARO_ST_PAGE_RANGE, 73, span.row, page);
                    page = 0;
                }
                where[c % C::PAGES] = page * a.page_size + key % a.page_size;
            }
            known = until;
            __syncwarp();
        };
        look_up();
        auto load = [&](int i, bool values) {                // warp-uniform call
            const int s = i % ST;
            uint8_t* dst = (values ? v_s : k_s) + s * C::KEY_BYTES;
            uint64_t* bar = values ? &v_full[s] : &k_full[s];
            if (!values && (i + 1) << log_copies > known) look_up();         // (values follow their keys by a few steps)
            if (lane == 0) mbar_expect_tx(bar, C::KEY_BYTES);
            __syncwarp();
            if (lane < copies) {
                const int y = where[((i << log_copies) + lane) % C::PAGES];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    tma_load_2d(dst + nb * KEY_REGION + (uint32_t)lane * box * 128, values ? &map_v : &map_k, bar, kvh * HD + nb * 64, y);
            }
        };
        int k_next = 0, v_next = 0;
        uint32_t idle = 0;
        while (k_next < n_steps || v_next < n_steps) {
            int what = 0;                                    // bit 0: the next keys' buffer is free, bit 1: the next values', bit 2: stop
            if (lane == 0) {
                if (k_next < n_steps && (k_next < ST || mbar_test(&k_empty[k_next % ST], ((k_next / ST) - 1) & 1))) what |= 1;
                if (v_next < k_next && (v_next < ST || mbar_test(&v_empty[v_next % ST], ((v_next / ST) - 1) & 1))) what |= 2;
                if (*gave_up) what = 4;
                if (what == 0 && ++idle > WAIT_LIMIT / 16) {
                    report(a.status, IMPARO_ST_WAIT_LIMIT, 74, k_next, v_next);
                    *gave_up = 1;
                    what = 4;
                }
            }
            what = __shfl_sync(0xffffffffu, what, 0);
            if (what & 4) break;
            if (what & 1) load(k_next++, false);
            if (what & 2) load(v_next++, true);
            if (what != 0) idle = 0; else __nanosleep(64);
        }
        // no CTA ends with a copy on its way (where nothing gave up, the products have waited for all of them)
        if (lane == 0) {
            for (int i = max(0, k_next - ST); i < k_next; ++i) mbar_wait(&k_full[i % ST], (i / ST) & 1);
            for (int i = max(0, v_next - ST); i < v_next; ++i) mbar_wait(&v_full[i % ST], (i / ST) & 1);
        }
    } else if (warp >= C::MMA_WARP) {
        constexpr int MINE = NT / 2;                         // this warp's tiles: w, w + 2
        const int w = warp - C::MMA_WARP;
        const uint64_t qd0 = smem_desc(smem_u32(q_s)), kd0 = smem_desc(smem_u32(k_s)), vd0 = desc_mn(smem_u32(v_s));
        const uint32_t id_s = idesc(STEP, false), id_o = idesc(HD, true);
        const uint32_t b_kf = smem_u32(k_full), b_ke = smem_u32(k_empty), b_vf = smem_u32(v_full), b_ve = smem_u32(v_empty),
                       b_s = smem_u32(s_ready), b_p = smem_u32(p_ready), b_o = smem_u32(o_done);
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity, int code, int j) {                // the whole warp
            if (!wait_at(bar, parity)) {
                report(a.status, IMPARO_ST_WAIT_LIMIT, code, j, w);
                *gave_up = 1;
                ok = false;
            }
            ok = __all_sync(0xffffffffu, ok);
        };
        int k_seen = -1, v_seen = -1;                        // the last step whose keys / values this warp has waited for
        auto scores = [&](int x, int j) {                    // S = Q K^T of the tile's step j
            const int i = at(x, j), s = i % ST;
            if (i != k_seen) { wait(b_kf + s * 8, (i / ST) & 1, 76, i); k_seen = i; }
            if (!ok) return;
            if (elect_one()) {
                const uint64_t qd = qd0 + (uint64_t)(((x & (R - 1)) * C::Q_BYTES) >> 4), kd = kd0 + (uint64_t)((s * C::KEY_BYTES) >> 4);
                const uint32_t t_s = tmem + (x * SB + j % SB) * STEP;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int k = 0; k < BK / UMMA_K; ++k)
                        umma(t_s, qd + (uint64_t)((nb * REGION + k * 32) >> 4), kd + (uint64_t)((nb * KEY_REGION + k * 32) >> 4), id_s,
                             (nb > 0 || k > 0) ? 1u : 0u);
                commit_at(b_s + (x * SB + j % SB) * 8);
                commit_at(b_ke + s * 8);
            }
            __syncwarp();
        };
        // values outside the span are cleared: their weights are 0, and what lies there may be infinite or no number
        const int clear_first = span.first % STEP != 0 && chunk == 0 ? 0 : -1;
        const int clear_last = span.end % STEP != 0 && first_step + n_steps == all_steps ? n_steps - 1 : -1;
        auto clear_values = [&](int i) {
            const int key0 = (first_step + i) * STEP, lo = max(0, span.first - key0), hi = min(STEP, span.end - key0);
            uint8_t* v = v_s + (i % ST) * C::KEY_BYTES;
            for (int c = lane; c < STEP * NB * 8; c += 32) {
                const int row = (c >> 3) % STEP, nb = (c >> 3) / STEP;
                if (row < lo || row >= hi) *reinterpret_cast<uint4*>(v + nb * KEY_REGION + row * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        int n_x[MINE];
#pragma unroll
        for (int u = 0; u < MINE; ++u) {
            const int x = w + 2 * u;
            n_x[u] = steps_of(x);
            if (n_x[u] > 0 && ok) {
                wait(smem_u32(&q_ready[x & (R - 1)]), 0, 75, x);
                fence_after();
            }
            for (int j = 0; j < SB && j < n_x[u] && ok; ++j) scores(x, j);
        }
        for (int j = 0; j < n_x[0] && ok; ++j) {             // (a later tile has no more steps than an earlier one)
#pragma unroll
            for (int u = 0; u < MINE; ++u) {
                const int x = w + 2 * u, i = at(x, j), s = i % ST;
                if (j >= n_x[u] || !ok) continue;
                if (i != v_seen) {
                    wait(b_vf + s * 8, (i / ST) & 1, 78, i);
                    if (!ok) continue;
                    v_seen = i;
                    if (i == clear_first || i == clear_last) clear_values(i);
                }
                wait(b_p + x * 8, j & 1, 79, j);
                if (!ok) continue;
                fence_after();
                if (elect_one()) {                           // O += P V
                    const uint64_t vd = vd0 + (uint64_t)((s * C::KEY_BYTES) >> 4);
                    const uint32_t t_p = tmem + (x * SB + j % SB) * STEP, t_o = tmem + C::O_COL + x * HD;
#pragma unroll
                    for (int kk = 0; kk < STEP / UMMA_K; ++kk)
                        umma_ta(t_o, t_p + kk * 8, vd + (uint64_t)((kk * (UMMA_K * 128)) >> 4), id_o, (kk > 0 || j > 0) ? 1u : 0u);
                    if (SB > 1 || j + 1 == n_x[u]) commit_at(b_o + x * 8);
                    commit_at(b_ve + s * 8);
                }
                __syncwarp();
                if (j + SB < n_x[u]) scores(x, j + SB);      // (behind P V in the tensor cores' order, which reads the same columns)
            }
        }
        if (elect_one()) {                                   // tensor memory is given back only when nothing uses it any more
            commit_at(smem_u32(&drained[w]));
            mbar_wait(&drained[w], 0);
        }
        __syncwarp();
    } else {
        const int x = warp >> 2, r = (warp & 3) * 32 + lane, n_x = steps_of(x);
        const int tok0 = row0 + (x & (R - 1)) * TQ, toks = min(TQ, max(0, n_tok - (x & (R - 1)) * TQ));
        const bool valid = r < toks * G;
        const bool warp_valid = (warp & 3) * 32 < toks * G;
        const int t = tok0 + (valid ? r / G : 0), head = kvh * G + r % G;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_o = tmem + lanes + C::O_COL + x * HD;
        if (x < R) {
            const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)t * a.q_stride + (size_t)head * HD);
            uint8_t* dst = q_s + x * C::Q_BYTES + r * 128;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c)
                *reinterpret_cast<uint4*>(dst + (c >> 3) * REGION + (((c & 7) ^ (r & 7)) << 4)) = valid ? src[c] : make_uint4(0u, 0u, 0u, 0u);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            arrive(smem_u32(&q_ready[x]));
        }
        const float sl2 = a.scale * LOG2E;                   // scores in units of log2(e)
        float m = -INFINITY;                                 // the max in use, scaled
        float2 l2 = make_float2(0.f, 0.f);
        bool ok = true;
        const uint32_t b_s = smem_u32(&s_ready[x * SB]), b_p = smem_u32(&p_ready[x]), b_o = smem_u32(&o_done[x]);
        auto wait = [&](uint32_t bar, uint32_t parity, int code, int j) {
            if (!wait_at(bar, parity)) { report(a.status, IMPARO_ST_WAIT_LIMIT, code, j, r); *gave_up = 1; ok = false; }
            ok = __all_sync(0xffffffffu, ok);
            fence_after();
        };
        const int key_first = (first_step + at(x, 0)) * STEP, key_step = phases * STEP;
        for (int j = 0; j < n_x; ++j) {
            const uint32_t t_s = tmem + lanes + (x * SB + j % SB) * STEP;
            wait(b_s + j % SB * 8, (j / SB) & 1, 81, j);
            if (!ok) break;
            float sv[STEP];
            float corr = 1.f;
            if (warp_valid) {
                uint32_t raw[STEP];
                tmem_ld32(t_s, raw); tmem_ld32(t_s + 32, raw + 32);
                wait_ld();
#pragma unroll
                for (int i = 0; i < STEP; ++i) { asm volatile("" : "+r"(raw[i]) :: "memory"); sv[i] = __uint_as_float(raw[i]); }
                const int key0 = key_first + j * key_step, lo = span.first - key0, hi = span.end - key0;
                if (lo > 0 || hi < STEP) {
#pragma unroll
                    for (int i = 0; i < STEP; ++i)
                        if (i < lo || i >= hi) sv[i] = -INFINITY;
                }
                float mx[4];                                 // four running maxima: no long dependent chain
#pragma unroll
                for (int i = 0; i < 4; ++i) mx[i] = max3(sv[3 * i], sv[3 * i + 1], sv[3 * i + 2]);
#pragma unroll
                for (int i = 12; i < 60; i += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], sv[i + 2 * e], sv[i + 2 * e + 1]);
                mx[0] = max3(max3(mx[0], sv[60], sv[61]), sv[62], sv[63]);
                const float mx0 = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * sl2;         // (scale > 0: the max commutes with it)
                // (true for m = -inf and a finite max, and for a max that is no number: a row with such a score has no result, nor
                // has one with an infinite score)
                const bool grow = !(mx0 <= m + GROW);
                const float m_new = grow ? (mx0 == INFINITY ? __int_as_float(0x7fffffff) : mx0) : m;
                corr = m == -INFINITY ? 0.f : ex2(m - m_new);
                m = m_new;
                if (__any_sync(0xffffffffu, grow && j > 0)) {                // the accumulated output of this warp's rows, in place
                    // (one buffer of scores: these scores were made behind the P V of the step before)
                    if (SB > 1) wait(b_o, (j - 1) & 1, 82, j);
                    if (!ok) break;
#pragma unroll 1
                    for (int c = 0; c < HD; c += 16) {
                        float ov[16];
                        tmem_ld16(t_o + c, ov);
                        uint32_t ow[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) ow[e] = __float_as_uint(ov[e] * corr);
                        tmem_st16(t_o + c, ow);
                    }
                    l2.x *= corr;
                    l2.y *= corr;
                }
            }
            if (warp_valid) {
                const float nb = m == -INFINITY ? 0.f : -m;
                const float2 sl = make_float2(sl2, sl2), base = make_float2(nb, nb);
                float2 sum[2] = {l2, make_float2(0.f, 0.f)};
#pragma unroll
                for (int c = 0; c < 2; ++c) {                // 32 keys = 16 columns of P
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float2 e = __ffma2_rn(make_float2(sv[c * 32 + 2 * i], sv[c * 32 + 2 * i + 1]), sl, base);
                        e.x = ex2(e.x);
                        e.y = ex2(e.y);
                        sum[i & 1] = __fadd2_rn(sum[i & 1], e);
                        p[i] = pack_bf16(e.x, e.y);
                    }
                    tmem_st16(t_s + c * 16, p);
                }
                l2 = __fadd2_rn(sum[0], sum[1]);
                wait_st();
            }
            // every phase is waited for, so that a wait by parity cannot take an earlier one for the one it means
            if (SB > 1 && j > 0) {
                wait(b_o, (j - 1) & 1, 84, j);
                if (!ok) break;
            }
            fence_before();
            arrive(b_p);
        }
        if (ok && n_x > 0) wait(b_o, SB > 1 ? (n_x - 1) & 1 : 0, 83, n_x);
        float l = l2.x + l2.y;
        const size_t part = ((size_t)t * a.nh + head) * n_splits + chunk;
        // the results of the tiles with the same rows, for the first of them to add: [tile][dims, max, sum][row], where keys and values were
        float* other = reinterpret_cast<float*>(k_s);
        constexpr int OTHER = (HD + 2) * TILE;
        static_assert((size_t)(NT - 1) * OTHER * 4 <= (size_t)ST * 2 * C::KEY_BYTES && (size_t)NT / 2 * TILE * HD * 4 <= (size_t)NT * C::Q_BYTES &&
                      (size_t)NT * TILE * HD * 4 <= (size_t)NT * C::Q_BYTES + (size_t)ST * 2 * C::KEY_BYTES, "results in shared memory");
        asm volatile("bar.sync 1, %0;" ::"n"(NT * 128) : "memory");                          // all tiles' products have run
        if (phases > 1) {
            if (x >= R && ok) {
                float* mine = other + (x - R) * OTHER + r;
                if (n_x > 0 && warp_valid) {
#pragma unroll 1
                    for (int c = 0; c < HD; c += 16) {
                        float o[16];
                        tmem_ld16(t_o + c, o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) mine[(c + e) * TILE] = o[e];
                    }
                }
                mine[HD * TILE] = n_x > 0 ? m : -INFINITY;
                mine[(HD + 1) * TILE] = n_x > 0 ? l : 0.f;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(NT * 128) : "memory");
        }
        if (ok && !__any_sync(0xffffffffu, *gave_up) && x < R && warp_valid) {
            float m_all = m, f[NT];                          // the factor of each result
#pragma unroll
            for (int i = 1; i < NT; ++i)
                if (i < phases && other[(x + (i - 1) * R) * OTHER + (HD + 1) * TILE + r] != 0.f)
                    m_all = fmaxf(m_all, other[(x + (i - 1) * R) * OTHER + HD * TILE + r]);
            f[0] = m == -INFINITY ? 0.f : ex2(m - m_all);
            l *= f[0];
#pragma unroll
            for (int i = 1; i < NT; ++i) {
                f[i] = 0.f;
                if (i < phases) {
                    const float* his = other + (x + (i - 1) * R) * OTHER + r;
                    if (his[(HD + 1) * TILE] != 0.f) {
                        f[i] = ex2(his[HD * TILE] - m_all);
                        l += his[(HD + 1) * TILE] * f[i];
                    }
                }
            }
            // by way of shared memory (where the queries were, and with four tiles of rows the keys): a thread has a row, which alone
            // it would write 16 bytes at a time, far from its neighbours'
            float4* rows = reinterpret_cast<float4*>(q_s) + (size_t)(x * TILE + (warp & 3) * 32) * (HD / 4);
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
                float o[16];
                tmem_ld16(t_o + c, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] *= f[0];
#pragma unroll
                for (int i = 1; i < NT; ++i)
                    if (i < phases && f[i] != 0.f) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] += other[(x + (i - 1) * R) * OTHER + (c + e) * TILE + r] * f[i];
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    rows[lane * (HD / 4) + ((c / 4 + e) ^ (lane & 7))] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
            __syncwarp();
            constexpr int LANES = HD / 4;                    // 16 bytes each to a row
            for (int i = lane / LANES; i < 32; i += 32 / LANES) {
                const size_t his = __shfl_sync(0xffffffffu, part, i);
                if ((warp & 3) * 32 + i < toks * G)
                    reinterpret_cast<float4*>(a.part_acc)[his * (HD / 4) + lane % LANES] = rows[i * (HD / 4) + ((lane % LANES) ^ (i & 7))];
            }
            if (valid) {
                const bool sees = a.positions[t] >= 0;       // (a row without a position sees nothing)
                a.part_ml[part * 2] = sees && m_all != -INFINITY ? m_all * LN2 : -INFINITY;
                a.part_ml[part * 2 + 1] = sees ? l : 0.f;
            }
        }
    }
    fence_before();
    __syncthreads();
    if (warp == C::MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ---- a row's own keys, and the join ----------------------------------------------------------------------------------
// One CTA per (stretch of own keys, kv head x tile of 16 query heads, token).  A warp takes 16 or 32 keys at a time on mma.sync: the heads
// are the rows of the tile, keys and values go from the cache to registers as 16-byte loads, whole 64- or 128-byte stretches of a
// row at a time.  The products' inner index may run in any order that both operands share, and so may the outer one of P V: a lane's
// eight neighbouring dims are four steps' fragments of the first product and its own column of eight output tiles of the second
// (no exchange through shared memory; the memory is what bounds it).  With one stretch the CTA joins the shared keys' partial results
// to its own after it has waited for the kernel that makes them: its own keys are read while that kernel runs.
constexpr int OWN_WARPS = 4;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// WIDE: up to 16 heads; otherwise at most eight, the lower half of the tile stays empty and costs no registers.
template <int HD, bool JOIN, bool WIDE>
__global__ void __launch_bounds__(OWN_WARPS * 32, HD == 64 ? 4 : (WIDE ? 2 : 3))
own_tc_kernel(const Args a, __nv_bfloat16* __restrict__ out, const float* __restrict__ sinks, const int n_splits) {
    constexpr int NB = HD / 64, KB = HD / 32;                // 64-dim blocks (values), 32-dim blocks (keys)
    constexpr int HEADS = WIDE ? 16 : 8, SLABS = HD == 64 && !WIDE ? 2 : 1;      // 16 keys each, all loads of a turn at once
    __shared__ float w_m[OWN_WARPS][HEADS], w_l[OWN_WARPS][HEADS];
    __shared__ __align__(16) float w_o[OWN_WARPS][HEADS][HD + 4];
    pdl_trigger();
    pdl_no_wait();                                           // (what this reads before its wait was complete before the kernel ahead let it start)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tg = lane & 3;
    const int G = a.nh / a.nkv, head_tiles = (G + 15) / 16;
    const int kvh = blockIdx.x / head_tiles, head0 = kvh * G + blockIdx.x % head_tiles * 16, n_heads = min(16, kvh * G + G - head0);
    const int t = blockIdx.y, split = blockIdx.z;
    const int pos = a.positions[t], item = a.item_of_token[t];           // (on their way while the group is found)
    const int group = group_of_warp(a, t);
    const Span span = shared_span(a, group);
    const Own own = own_keys(a, pos, span);
    const int k0 = (int)min((long long)split * a.chunk_own, (long long)own.count);
    const int k1 = split + 1 == a.n_own ? own.count : (int)min((long long)k0 + a.chunk_own, (long long)own.count);
    if (k0 < k1 && (item < 0 || item >= a.n_items) && tid == 0) report(a.status, IMPARO_ST_PAGE_RANGE, 84, t, item);
    const int* tab = k0 < k1 && item >= 0 && item < a.n_items ? a.table + (size_t)item * a.max_blocks : nullptr;
    const size_t kvw = (size_t)a.nkv * HD;
    const __nv_bfloat16* kc = reinterpret_cast<const __nv_bfloat16*>(a.k) + (size_t)kvh * HD;
    const __nv_bfloat16* vc = reinterpret_cast<const __nv_bfloat16*>(a.v) + (size_t)kvh * HD;
    // the queries: heads g and g + 8, dims 32 b + 8 tg .. + 7
    uint4 qa[KB], qb[WIDE ? KB : 1];
    if (!WIDE) qb[0] = make_uint4(0u, 0u, 0u, 0u);
    {
        const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)t * a.q_stride + (size_t)head0 * HD + tg * 8;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            qa[b] = g < n_heads ? *reinterpret_cast<const uint4*>(q + (size_t)g * HD + b * 32) : make_uint4(0u, 0u, 0u, 0u);
            if (WIDE) qb[b] = g + 8 < n_heads ? *reinterpret_cast<const uint4*>(q + (size_t)(g + 8) * HD + b * 32) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    float o[NB * 8][WIDE ? 4 : 2];                           // output tile nb * 8 + i: dims 64 nb + 8 column + i
#pragma unroll
    for (int i = 0; i < NB * 8; ++i)
#pragma unroll
        for (int e = 0; e < (WIDE ? 4 : 2); ++e) o[i][e] = 0.f;
    float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;
    const float sl2 = a.scale * LOG2E;
    if (tab != nullptr) {
        auto look_up = [&](int base) -> int {                // lane i: where key base + i lies
            if (lane >= 16 * SLABS || base + lane >= k1) return -1;
            const int key = own.key(base + lane), block = key / a.page_size;
            const int page = block < a.max_blocks ? tab[block] : -1;
            if (page >= 0 && page < a.n_pages) return page * a.page_size + key % a.page_size;
            report(a.status, IMPARO_ST_PAGE_RANGE, 85, t, page);
            return -1;
        };
        int next_row = look_up(k0 + warp * 16 * SLABS);
        for (int base = k0 + warp * 16 * SLABS; base < k1; base += OWN_WARPS * 16 * SLABS) {
            const int row = next_row;
            uint4 kf[SLABS][2][KB], vf[SLABS][4][NB];
#pragma unroll
            for (int slab = 0; slab < SLABS; ++slab) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int at = __shfl_sync(0xffffffffu, row, slab * 16 + n * 8 + g);
#pragma unroll
                    for (int b = 0; b < KB; ++b)
                        kf[slab][n][b] = __ldg(reinterpret_cast<const uint4*>(kc + (size_t)max(at, 0) * kvw + b * 32 + tg * 8));
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {                // keys 2 tg, 2 tg + 1, 2 tg + 8, 2 tg + 9
                    const int at = __shfl_sync(0xffffffffu, row, slab * 16 + 2 * tg + (u & 1) + (u >> 1) * 8);
#pragma unroll
                    for (int b = 0; b < NB; ++b)
                        vf[slab][u][b] = __ldg(reinterpret_cast<const uint4*>(vc + (size_t)max(at, 0) * kvw + b * 64 + g * 8));
                }
            }
            next_row = look_up(base + OWN_WARPS * 16 * SLABS);            // (a turn ahead: its keys need not wait for the table)
            const unsigned there = __ballot_sync(0xffffffffu, row >= 0);
            // (places without a key read the cache's first row: their scores are left out, their values must be finite)
            if (there != (SLABS == 2 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
                for (int slab = 0; slab < SLABS; ++slab)
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (!((there >> (slab * 16 + 2 * tg + (u & 1) + (u >> 1) * 8)) & 1u)) {
#pragma unroll
                            for (int b = 0; b < NB; ++b) vf[slab][u][b] = make_uint4(0u, 0u, 0u, 0u);
                        }
            }
#pragma unroll
            for (int slab = 0; slab < SLABS; ++slab) {
            float s[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    const uint4 q2 = qb[WIDE ? b : 0];
                    mma16816(s[n], qa[b].x, q2.x, qa[b].y, q2.y, kf[slab][n][b].x, kf[slab][n][b].y);
                    mma16816(s[n], qa[b].z, q2.z, qa[b].w, q2.w, kf[slab][n][b].z, kf[slab][n][b].w);
                }
            }
            float mx_a = -INFINITY, mx_b = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool seen = (there >> (slab * 16 + n * 8 + 2 * tg + e)) & 1u;
                    s[n][e] = seen ? s[n][e] * sl2 : -INFINITY;
                    s[n][2 + e] = seen ? s[n][2 + e] * sl2 : -INFINITY;
                    mx_a = fmaxf(mx_a, s[n][e]);
                    mx_b = fmaxf(mx_b, s[n][2 + e]);
                }
            mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 1));
            mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 2));
            mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 1));
            mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 2));
            const float mn_a = fmaxf(m_a, mx_a), mn_b = fmaxf(m_b, mx_b);
            const float ca = m_a == -INFINITY ? 0.f : ex2(m_a - mn_a), cb = m_b == -INFINITY ? 0.f : ex2(m_b - mn_b);
            const float ba = mn_a == -INFINITY ? 0.f : mn_a, bb = mn_b == -INFINITY ? 0.f : mn_b;
            m_a = mn_a;
            m_b = mn_b;
            l_a *= ca;
            l_b *= cb;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[n][e] = ex2(s[n][e] - ba);
                    s[n][2 + e] = ex2(s[n][2 + e] - bb);
                    l_a += s[n][e];
                    l_b += s[n][2 + e];
                }
#pragma unroll
            for (int i = 0; i < NB * 8; ++i) {
                o[i][0] *= ca;
                o[i][1] *= ca;
                if (WIDE) { o[i][WIDE ? 2 : 0] *= cb; o[i][WIDE ? 3 : 1] *= cb; }
            }
            const uint32_t p0 = pack_bf16(s[0][0], s[0][1]), p1 = pack_bf16(s[0][2], s[0][3]), p2 = pack_bf16(s[1][0], s[1][1]),
                           p3 = pack_bf16(s[1][2], s[1][3]);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const uint32_t x0[4] = {vf[slab][0][b].x, vf[slab][0][b].y, vf[slab][0][b].z, vf[slab][0][b].w}, x1[4] = {vf[slab][1][b].x, vf[slab][1][b].y, vf[slab][1][b].z, vf[slab][1][b].w};
                const uint32_t x2[4] = {vf[slab][2][b].x, vf[slab][2][b].y, vf[slab][2][b].z, vf[slab][2][b].w}, x3[4] = {vf[slab][3][b].x, vf[slab][3][b].y, vf[slab][3][b].z, vf[slab][3][b].w};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t pick = i & 1 ? 0x7632u : 0x5410u;
                    float (&acc)[WIDE ? 4 : 2] = o[b * 8 + i];
                    float c[4] = {acc[0], acc[1], WIDE ? acc[WIDE ? 2 : 0] : 0.f, WIDE ? acc[WIDE ? 3 : 1] : 0.f};
                    mma16816(c, p0, WIDE ? p1 : 0u, p2, WIDE ? p3 : 0u, __byte_perm(x0[i >> 1], x1[i >> 1], pick), __byte_perm(x2[i >> 1], x3[i >> 1], pick));
                    acc[0] = c[0];
                    acc[1] = c[1];
                    if (WIDE) { acc[WIDE ? 2 : 0] = c[2]; acc[WIDE ? 3 : 1] = c[3]; }
                }
            }
            }
        }
        l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
        l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
        l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
        l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
    }
    if (tg == 0) { w_m[warp][g] = m_a; w_l[warp][g] = l_a; }
    if (WIDE && tg == 0) { w_m[warp][g + 8] = m_b; w_l[warp][g + 8] = l_b; }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        // a lane's columns of the eight tiles are 2 tg and 2 tg + 1: dims 8 (2 tg) .. + 7 and the eight behind them
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float* dst = &w_o[warp][g][b * 64 + 8 * (2 * tg + e) + 4 * h];
                *reinterpret_cast<float4*>(dst) = make_float4(o[b * 8 + 4 * h][e], o[b * 8 + 4 * h + 1][e], o[b * 8 + 4 * h + 2][e], o[b * 8 + 4 * h + 3][e]);
                if (WIDE) {
                    constexpr int LOW = WIDE ? 2 : 0;
                    dst = &w_o[warp][WIDE ? g + 8 : 0][b * 64 + 8 * (2 * tg + e) + 4 * h];
                    *reinterpret_cast<float4*>(dst) = make_float4(o[b * 8 + 4 * h][LOW + e], o[b * 8 + 4 * h + 1][LOW + e],
                                                                  o[b * 8 + 4 * h + 2][LOW + e], o[b * 8 + 4 * h + 3][LOW + e]);
                }
            }
        }
    }
    __syncthreads();
    // the shared stretches that hold anything for this row's group
    int live = 0;
    if (JOIN && span.first < span.end) {
        const int per_chunk = a.chunk_shared / STEP, steps = (span.end + STEP - 1) / STEP - span.first / STEP;
        live = min(a.n_shared, (steps + per_chunk - 1) / per_chunk);
    }
    if (JOIN) pdl_wait();                                    // the kernel that makes the partial results is complete
    // a warp a head: the lanes are the partial results (their largest score and sum) first, then the dims
    constexpr int PER = HD / 32;
    for (int h = warp; h < n_heads; h += OWN_WARPS) {
        const size_t row = (size_t)t * a.nh + head0 + h;
        float m = lane < OWN_WARPS ? w_m[lane][h] : -INFINITY, l = 0.f, acc[PER];
        m = warp_max(m);
        const float own_f = lane < OWN_WARPS && w_l[lane][h] != 0.f ? ex2(w_m[lane][h] - m) : 0.f;
        l = warp_sum(lane < OWN_WARPS ? w_l[lane][h] * own_f : 0.f);
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll
        for (int w = 0; w < OWN_WARPS; ++w) {
            const float f = __shfl_sync(0xffffffffu, own_f, w);
            if (f != 0.f) {
#pragma unroll
                for (int e = 0; e < PER; ++e) acc[e] += w_o[w][h][lane * PER + e] * f;
            }
        }
        if (JOIN) {
            const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + row * n_splits;
            const float* part = a.part_acc + row * n_splits * HD + lane * PER;
            for (int s0 = 0; s0 < live; s0 += 32) {
                const float2 v = s0 + lane < live ? __ldcg(ml + s0 + lane) : make_float2(-INFINITY, 0.f);
                const float m_new = fmaxf(m, warp_max(v.y != 0.f ? v.x * LOG2E : -INFINITY));
                const float f = v.y != 0.f ? ex2(v.x * LOG2E - m_new) : 0.f;
                const float corr = m == -INFINITY ? 0.f : ex2(m - m_new);
                m = m_new;
                l = l * corr + warp_sum(v.y * f);
#pragma unroll
                for (int e = 0; e < PER; ++e) acc[e] *= corr;
                const int n = min(32, live - s0);
                for (int s = 0; s < n; s += 8) {
                    float x[8][PER];                         // eight partial results on their way at once
#pragma unroll
                    for (int u = 0; u < 8; ++u)
#pragma unroll
                        for (int e = 0; e < PER; ++e) x[u][e] = s + u < n ? __ldcg(part + (size_t)(s0 + s + u) * HD + e) : 0.f;
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const float fs = __shfl_sync(0xffffffffu, f, (s + u) & 31);
                        if (s + u < n && fs != 0.f) {        // (a result of sum 0 has no values)
#pragma unroll
                            for (int e = 0; e < PER; ++e) acc[e] += x[u][e] * fs;
                        }
                    }
                }
            }
            if (sinks) {
                const float sink = sinks[head0 + h] * LOG2E, m_new = fmaxf(m, sink), corr = m == -INFINITY ? 0.f : ex2(m - m_new);
                l = l * corr + (sink == -INFINITY ? 0.f : ex2(sink - m_new));        // (minus infinity: no sink, for a row of nothing too)
#pragma unroll
                for (int e = 0; e < PER; ++e) acc[e] *= corr;
            }
            const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
            for (int e = 0; e < PER; e += 2)
                *reinterpret_cast<uint32_t*>(out + row * HD + lane * PER + e) = pack_bf16(acc[e] * inv, acc[e + 1] * inv);
        } else {
            const size_t mine = row * n_splits + a.n_shared + split;
#pragma unroll
            for (int e = 0; e < PER; ++e) a.part_acc[mine * HD + lane * PER + e] = acc[e];
            if (lane == 0) {
                a.part_ml[mine * 2] = m == -INFINITY ? -INFINITY : m * LN2;
                a.part_ml[mine * 2 + 1] = l;
            }
            // a row of no group has no part in the shared stretches
            if (split == 0 && group < 0)
                for (int s = lane; s < a.n_shared; s += 32) {
                    a.part_ml[(row * n_splits + s) * 2] = -INFINITY;
                    a.part_ml[(row * n_splits + s) * 2 + 1] = 0.f;
                }
        }
    }
    if (!JOIN && tid == 0) pdl_wait_at_end();                // this kernel completes after the one it ran beside
}

// The same for up to eight query heads to a kv head, joined at once: a CTA takes a token and `per` of its kv heads, one to a warp.  A warp
// copies its keys and values into a ring of its own, up to RING turns of 16 keys ahead, so that the memory's latency is paid once and not a
// turn; no result leaves it: the partial results of the shared keys are read by the lanes that hold the same dims.  132 rows of 8 kv heads of
// 128 over 8,000 shared positions and up to 200 own ones 59 us with the kernel before, of which this one about 20 (39 by a CTA per kv head).
constexpr int OWN_DIMS = 512, TURN = 16, LOOKED = 1024;      // dims of a CTA's heads; LOOKED keys' places are looked up at once

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

constexpr size_t own_ring_bytes(int turns, int dims) { return (size_t)turns * TURN * dims * 4; }

template <int HD, int RING>
__global__ void __launch_bounds__(OWN_DIMS / HD * 32, 2)
own_ring_kernel(const Args a, __nv_bfloat16* __restrict__ out, const float* __restrict__ sinks, const int n_splits) {
    constexpr int NB = HD / 64, KB = HD / 32;
    constexpr uint32_t ROW = HD * 2, SLAB = TURN * ROW;
    extern __shared__ __align__(128) uint8_t ring[];         // [warp][RING][keys, values][TURN][ROW]
    __shared__ int where[LOOKED];
    pdl_trigger();
    pdl_no_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tg = lane & 3;
    const int G = a.nh / a.nkv, t = blockIdx.y, kvh = blockIdx.x * (blockDim.x >> 5) + warp;
    const int pos = a.positions[t], item = a.item_of_token[t];
    const int group = group_of_warp(a, t);
    const Span span = shared_span(a, group);
    const Own own = own_keys(a, pos, span);
    const bool there_is_a_row = item >= 0 && item < a.n_items;
    if (own.count > 0 && !there_is_a_row && threadIdx.x == 0) report(a.status, IMPARO_ST_PAGE_RANGE, 84, t, item);
    const int count = there_is_a_row ? own.count : 0;
    const int* tab = a.table + (size_t)(there_is_a_row ? item : 0) * a.max_blocks;
    const size_t kvw = (size_t)a.nkv * HD;
    const uint8_t* mine = ring + warp * (RING * 2 * SLAB);
    // copies: lane >> 3 is the key (and every fourth from it), lane & 7 the 16 bytes of each 128; their places in shared memory are such that
    // neither the copies nor the fragments' reads meet a bank twice
    const __nv_bfloat16* kc = reinterpret_cast<const __nv_bfloat16*>(a.k) + (size_t)kvh * HD + (lane & 7) * 8;
    const __nv_bfloat16* vc = reinterpret_cast<const __nv_bfloat16*>(a.v) + (size_t)kvh * HD + (lane & 7) * 8;
    auto fetch = [&](int turn) {                             // a turn of the LOOKED keys
        const uint32_t to = smem_u32(mine) + turn % RING * (2 * SLAB);
#pragma unroll
        for (int c = 0; c < TURN / 4; ++c) {
            const int key = (lane >> 3) + 4 * c, row = where[turn * TURN + key];
            if (row >= 0) {
#pragma unroll
                for (int d = 0; d < NB; ++d) {
                    copy16(to + key * ROW + d * 128 + (((lane & 7) ^ ((key & 1) << 2)) << 4), kc + (size_t)row * kvw + d * 64);
                    copy16(to + SLAB + key * ROW + d * 128 + (((lane & 7) ^ (key & 6)) << 4), vc + (size_t)row * kvw + d * 64);
                }
            }
        }
    };
    const int head0 = kvh * G;
    uint4 qa[KB];                                            // the queries: head g, dims 32 b + 8 tg .. + 7
    {
        const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)t * a.q_stride + (size_t)head0 * HD + tg * 8;
#pragma unroll
        for (int b = 0; b < KB; ++b) qa[b] = g < G ? *reinterpret_cast<const uint4*>(q + (size_t)g * HD + b * 32) : make_uint4(0u, 0u, 0u, 0u);
    }
    float o[NB * 8][2];                                      // head g, dims 64 nb + 8 (2 tg + e) + i at [nb * 8 + i][e]
#pragma unroll
    for (int i = 0; i < NB * 8; ++i) o[i][0] = o[i][1] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float sl2 = a.scale * LOG2E;
    for (int done = 0; done < count; done += LOOKED) {
    const int known = min(LOOKED, count - done), turns = (known + TURN - 1) / TURN;
    if (done > 0) __syncthreads();                           // (every warp is through with the places before)
    for (int i = threadIdx.x; i < turns * TURN; i += blockDim.x) {
        int row = -1;
        if (i < known) {
            const int key = own.key(done + i), block = key / a.page_size;
            const int page = block < a.max_blocks ? tab[block] : -1;
            if (page >= 0 && page < a.n_pages) row = page * a.page_size + key % a.page_size;
            else report(a.status, IMPARO_ST_PAGE_RANGE, 85, t, page);
        }
        where[i] = row;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) {
        if (i < turns) fetch(i);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    for (int turn = 0; turn < turns; ++turn) {
        __syncwarp();                                        // (the turn whose place the next one takes has been read by all lanes)
        if (turn + RING - 1 < turns) fetch(turn + RING - 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
        const unsigned there = __ballot_sync(0xffffffffu, where[turn * TURN + (lane & 15)] >= 0) & 0xffffu;
        __syncwarp();                                        // every lane's copies of this turn have arrived
        const uint8_t* ks = mine + turn % RING * (2 * SLAB);
        const uint8_t* vs = ks + SLAB;
        float s[2][2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < KB; ++d) {
                const uint4 kf = *reinterpret_cast<const uint4*>(ks + (n * 8 + g) * ROW + (d >> 1) * 128 + ((((d & 1) << 2 | tg) ^ ((g & 1) << 2)) << 4));
                mma16816(c, qa[d].x, 0u, qa[d].y, 0u, kf.x, kf.y);
                mma16816(c, qa[d].z, 0u, qa[d].w, 0u, kf.z, kf.w);
            }
            s[n][0] = c[0];
            s[n][1] = c[1];
        }
        uint4 vf[4][NB];                                     // keys 2 tg, 2 tg + 1, 2 tg + 8, 2 tg + 9
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int key = 2 * tg + (u & 1) + (u >> 1) * 8;
#pragma unroll
            for (int d = 0; d < NB; ++d) {
                vf[u][d] = *reinterpret_cast<const uint4*>(vs + key * ROW + d * 128 + ((g ^ (key & 6)) << 4));
                if (there != 0xffffu && !((there >> key) & 1u)) vf[u][d] = make_uint4(0u, 0u, 0u, 0u);       // (nothing was copied)
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[n][e] = (there >> (n * 8 + 2 * tg + e)) & 1u ? s[n][e] * sl2 : -INFINITY;
                mx = fmaxf(mx, s[n][e]);
            }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m, mx), corr = m == -INFINITY ? 0.f : ex2(m - m_new), base = m_new == -INFINITY ? 0.f : m_new;
        m = m_new;
        l *= corr;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) { s[n][e] = ex2(s[n][e] - base); l += s[n][e]; }
#pragma unroll
        for (int i = 0; i < NB * 8; ++i) { o[i][0] *= corr; o[i][1] *= corr; }
        const uint32_t p0 = pack_bf16(s[0][0], s[0][1]), p2 = pack_bf16(s[1][0], s[1][1]);
#pragma unroll
        for (int d = 0; d < NB; ++d) {
            const uint32_t x0[4] = {vf[0][d].x, vf[0][d].y, vf[0][d].z, vf[0][d].w}, x1[4] = {vf[1][d].x, vf[1][d].y, vf[1][d].z, vf[1][d].w};
            const uint32_t x2[4] = {vf[2][d].x, vf[2][d].y, vf[2][d].z, vf[2][d].w}, x3[4] = {vf[3][d].x, vf[3][d].y, vf[3][d].z, vf[3][d].w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t pick = i & 1 ? 0x7632u : 0x5410u;
                float c[4] = {o[d * 8 + i][0], o[d * 8 + i][1], 0.f, 0.f};
                mma16816(c, p0, 0u, p2, 0u, __byte_perm(x0[i >> 1], x1[i >> 1], pick), __byte_perm(x2[i >> 1], x3[i >> 1], pick));
                o[d * 8 + i][0] = c[0];
                o[d * 8 + i][1] = c[1];
            }
        }
    }
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    // the shared stretches that hold anything for this row's group
    int live = 0;
    if (span.first < span.end) {
        const int per_chunk = a.chunk_shared / STEP, steps = (span.end + STEP - 1) / STEP - span.first / STEP;
        live = min(a.n_shared, (steps + per_chunk - 1) / per_chunk);
    }
    pdl_wait();                                              // the kernel that makes the partial results is complete
    if (g >= G) return;
    const size_t row = (size_t)t * a.nh + head0 + g;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + row * n_splits;
    const float* part = a.part_acc + row * n_splits * HD + tg * 16;
    constexpr int AHEAD = 2;                                 // partial results on their way at once
    for (int s0 = 0; s0 < live; s0 += AHEAD) {
        float2 v[AHEAD];
        float4 x[AHEAD][NB][4];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            v[u] = s0 + u < live ? __ldcg(ml + s0 + u) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int d = 0; d < NB; ++d)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    x[u][d][c] = s0 + u < live ? __ldcg(reinterpret_cast<const float4*>(part + (size_t)(s0 + u) * HD + d * 64) + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float m_new = m;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) m_new = fmaxf(m_new, v[u].y != 0.f ? v[u].x * LOG2E : -INFINITY);
        const float corr = m == -INFINITY ? 0.f : ex2(m - m_new);
        m = m_new;
        l *= corr;
#pragma unroll
        for (int i = 0; i < NB * 8; ++i) { o[i][0] *= corr; o[i][1] *= corr; }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (v[u].y == 0.f) continue;                     // (a result of sum 0 has no values)
            const float f = ex2(v[u].x * LOG2E - m);
            l += v[u].y * f;
#pragma unroll
            for (int d = 0; d < NB; ++d)
#pragma unroll
                for (int c = 0; c < 4; ++c) {                // dims 64 d + 16 tg + 4 c ..: e = c / 2, i from 4 (c % 2) on
                    o[d * 8 + 4 * (c & 1)][c >> 1] += x[u][d][c].x * f;
                    o[d * 8 + 4 * (c & 1) + 1][c >> 1] += x[u][d][c].y * f;
                    o[d * 8 + 4 * (c & 1) + 2][c >> 1] += x[u][d][c].z * f;
                    o[d * 8 + 4 * (c & 1) + 3][c >> 1] += x[u][d][c].w * f;
                }
        }
    }
    if (sinks) {
        const float sink = sinks[head0 + g] * LOG2E, m_new = fmaxf(m, sink), corr = m == -INFINITY ? 0.f : ex2(m - m_new);
        l = l * corr + (sink == -INFINITY ? 0.f : ex2(sink - m_new));        // (minus infinity: no sink, for a row of nothing too)
#pragma unroll
        for (int i = 0; i < NB * 8; ++i) { o[i][0] *= corr; o[i][1] *= corr; }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            uint4 w;
            w.x = pack_bf16(o[d * 8][e] * inv, o[d * 8 + 1][e] * inv);
            w.y = pack_bf16(o[d * 8 + 2][e] * inv, o[d * 8 + 3][e] * inv);
            w.z = pack_bf16(o[d * 8 + 4][e] * inv, o[d * 8 + 5][e] * inv);
            w.w = pack_bf16(o[d * 8 + 6][e] * inv, o[d * 8 + 7][e] * inv);
            *reinterpret_cast<uint4*>(out + row * HD + d * 64 + 8 * (2 * tg + e)) = w;
        }
}

// A [rows, cols] bfloat16 matrix without gaps, tiles of box_rows x 64 elements, 128-byte swizzle.
static int encode(const void* ptr, uint64_t rows, uint64_t cols, uint32_t box_rows, CUtensorMap* out) {
    static PFN_cuTensorMapEncodeTiled fn = nullptr;          // (found once; two threads that look at the same time find the same)
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
        if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !p) return -20;
        fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled>(p);
    }
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {cols * 2};
    const cuuint32_t box[2] = {64, box_rows}, estr[2] = {1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -21;
}

template <int HD>
static int launch_hd(const Args& a, __nv_bfloat16* out, const float* sinks, cudaStream_t stream) {
    const int G = a.nh / a.nkv, TQ = TILE / G, head_tiles = (G + 15) / 16;
    const int box = a.page_size < STEP ? a.page_size : STEP;
    CUtensorMap mk, mv;
    const uint64_t rows = (uint64_t)a.n_pages * a.page_size, cols = (uint64_t)a.nkv * HD;
    int rc = encode(a.k, rows, cols, (uint32_t)box, &mk);
    if (rc) return rc;
    rc = encode(a.v, rows, cols, (uint32_t)box, &mv);
    if (rc) return rc;
    constexpr int DEEP = 4, SHALLOW = 3;                     // turns of a ring: a CTA per SM, two CTAs per SM
    static int sms[65] = {};                                 // by device; the attributes below are the device's too
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    const int slot = device >= 0 && device < 64 ? device : 64;
    if (slot == 64 || sms[slot] == 0) {
        e = cudaFuncSetAttribute(shared_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<HD>::SMEM);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(own_ring_kernel<HD, DEEP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)own_ring_bytes(DEEP, OWN_DIMS));
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(own_ring_kernel<HD, SHALLOW>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)own_ring_bytes(SHALLOW, OWN_DIMS));
        int n = 0;
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
        if (e != cudaSuccess) return (int)e;
        sms[slot] = n;
    }
    const int n_splits = a.n_own == 1 ? a.n_shared : a.n_shared + a.n_own;
    const int tokens = Shape<HD>::TILES * TQ;
    const long long units = (a.n_rows + tokens - 1) / tokens + a.n_groups - 1;       // every group may end a tile early
    e = launch(shared_tc_kernel<HD>, dim3(a.nkv, a.n_shared, (unsigned)units), dim3(Shape<HD>::THREADS), Shape<HD>::SMEM, stream, mk, mv, a, n_splits);
    if (e != cudaSuccess) return (int)e;
    int per = OWN_DIMS / HD;                                 // kv heads of a CTA that takes a row's own keys by rings
    while (a.nkv % per != 0) --per;
    const long long ctas = (long long)a.nkv / per * a.n_rows;
    // Rings, as soon as a CTA per token and 512 dims gives half of the SMs something to do: 256 rows of 8 kv heads of 64 over 20,000 shared
    // positions and up to 200 own ones 92 us (109 by a CTA per kv head), 128 rows 56 (64), 80 rows 48 (47); below, one warp's turns
    // take longer than four warps' (64 rows over 32,768: 51 against 48, 40 rows over 8,000: 30 against 25).  Up to a CTA per SM the
    // shared memory is such that no two come to the same SM (128 rows: 56; with two to an SM, where they would go first, 65).
    if (G <= 8 && a.n_own == 1 && 2 * ctas > sms[slot]) {
        const bool few = ctas <= sms[slot];
        const size_t smem = own_ring_bytes(few ? DEEP : SHALLOW, few ? OWN_DIMS : per * HD);
        e = launch(few ? own_ring_kernel<HD, DEEP> : own_ring_kernel<HD, SHALLOW>, dim3(a.nkv / per, a.n_rows), dim3(32 * per), smem, stream, a,
                   out, sinks, n_splits);
        return e == cudaSuccess ? 0 : (int)e;
    }
    const dim3 grid(a.nkv * head_tiles, a.n_rows, a.n_own);
    auto own = G > 8 ? (a.n_own == 1 ? own_tc_kernel<HD, true, true> : own_tc_kernel<HD, false, true>)
                     : (a.n_own == 1 ? own_tc_kernel<HD, true, false> : own_tc_kernel<HD, false, false>);
    e = launch(own, grid, dim3(OWN_WARPS * 32), 0, stream, a, out, sinks, n_splits);
    return e == cudaSuccess ? 0 : (int)e;
}

int launch_tc(const Args& a, void* out, const float* sinks, cudaStream_t stream) {
    const int G = a.nh / a.nkv;
    if ((a.hd != 64 && a.hd != 128) || G > TILE || !(a.scale > 0.f)) return -8;
    if (a.page_size != 16 && a.page_size != 32 && a.page_size != 64 && a.page_size % STEP != 0) return -8;
    if (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)out | (uintptr_t)a.part_acc | (uintptr_t)a.part_ml) & 15) return -8;
    if (a.q_stride % 8 != 0 || a.chunk_shared % STEP != 0) return -8;
    if (a.n_rows > 65535 || a.n_own > 65535 || a.n_rows + a.n_groups > 65535) return -8;
    return a.hd == 64 ? launch_hd<64>(a, (__nv_bfloat16*)out, sinks, stream) : launch_hd<128>(a, (__nv_bfloat16*)out, sinks, stream);
}

}  // namespace sp
}  // namespace imparo
