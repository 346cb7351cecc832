// The attention over a shared prefix on the 5th-generation tensor cores: bfloat16, head size 64 or 128, pages of 16, 32, 64 or a
// multiple of 128 positions (attention_shared.cu says what is computed; it takes all other cases).
//
// Two kernels.  The first takes the shared keys: a CTA owns one stretch of keys and up to 256 rows (tokens of a group x query heads
// of one kv head) as two tiles of 128 rows, and leaves each row's partial result.  The second takes each row's own keys, and joins
// them with the partial results of the shared ones.
#include "attention_shared.cuh"
#include "tcgen05.cuh"

namespace imparo {
namespace sp {

using namespace tc;

// ---- the shared keys ---------------------------------------------------------------------------------------------------
// One CTA per SM, 128 keys a step:
//   warps 0-3, 4-7  the softmax of tile A and B, one thread per row (= tensor-memory lane): the row's 128 scores of the step go into
//                   registers at once, P = exp2(s - max) goes back to tensor memory as bfloat16, where the second product reads it
//   warp 8          TMA: keys and values page by page (lane p fetches page p of a step) into rings with barriers of their own
//   warps 9, 10     tcgen05.mma, one issuing thread per tile: S = Q K^T (both from shared memory), O += P V (P from tensor memory)
// The output stays in tensor memory; it is scaled down only when a row's max has grown by more than 8 (in log2 units) since the max
// in use was taken, which leaves every term below 2^8 and the result the same.
// With head size 64 P has columns of its own, and the next step's scores are computed while this step's are weighted.  With 128 the
// scores' own columns take P; the other tile's softmax runs while this tile's products do.
// A group's rows that fill one tile at most are given to both: A takes the even steps, B the odd ones, and A adds B's result at the
// end (otherwise the SM's exponential units would wait for one tile's products every step).
constexpr int TILE = 128, STEP = 128;              // rows per tile, keys per step
constexpr int TC_THREADS = 384, LOAD_WARP = 8, MMA_WARP = 9;
constexpr uint32_t REGION = 128 * 128;             // a [128 rows][64 dims] block in shared memory
constexpr float GROW = 8.0f;
constexpr float LN2 = 0.69314718055994530942f, LOG2E = 1.4426950408889634074f;

template <int HD> struct Shape {
    static constexpr int NB = HD / 64;                       // 64-dim blocks of a head
    static constexpr int STAGES = HD == 64 ? 4 : 2;          // even: where the tiles take turns at the steps, a buffer is always the same tile's
    static constexpr bool ALIAS = HD == 128;                 // P in the scores' columns
    static constexpr uint32_t BLOCK = NB * REGION;           // a tile of queries, a step's keys or its values
    static constexpr uint32_t S_COL = 0, O_COL = 256, P_COL = ALIAS ? 0 : 384, P_STRIDE = ALIAS ? 128 : 64;
    static constexpr size_t SMEM = 1024 + 2 * BLOCK + (size_t)STAGES * 2 * BLOCK + 512;
};

__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {           // values: [key][dim], the dims contiguous (MN-major)
    uint64_t d = 0;
    d |= (uint64_t)((addr & 0x3FFFF) >> 4);
    d |= (uint64_t)((REGION >> 4) & 0x3FFF) << 16;                     // 64-dim blocks
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
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
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
__global__ void __launch_bounds__(TC_THREADS, 1)
shared_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Args a, const int n_splits) {
    using C = Shape<HD>;
    constexpr int NB = C::NB, ST = C::STAGES;
    extern __shared__ __align__(1024) uint8_t tc_smem_raw[];
    __shared__ int span_scratch[2];
    uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)tc_smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* q_s = smem;                                     // [2][BLOCK]
    uint8_t* k_s = q_s + 2 * C::BLOCK;                       // [ST][BLOCK]
    uint8_t* v_s = k_s + ST * C::BLOCK;                      // [ST][BLOCK]
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + ST * C::BLOCK);
    uint64_t* k_full = bars;                                 // [ST]
    uint64_t* k_empty = k_full + ST;
    uint64_t* v_full = k_empty + ST;
    uint64_t* v_empty = v_full + ST;
    uint64_t* q_ready = v_empty + ST;                        // [2]
    uint64_t* s_ready = q_ready + 2;                         // [2]  the tile's scores of a step are complete
    uint64_t* s_free = s_ready + 2;                          // [2]  ... and have been read into registers
    uint64_t* p_half = s_free + 2;                           // [2]  the first 64 keys' weights are written, the output is scaled
    uint64_t* p_ready = p_half + 2;                          // [2]  all are
    uint64_t* o_done = p_ready + 2;                          // [2]  P V of the step is accumulated
    uint64_t* drained = o_done + 2;                          // [2]  every product of the tile has run
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert((4 * 5 + 14) * 8 + 8 <= 512, "barriers");

    timeline_begin();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.nh / a.nkv, TQ = TILE / G;               // tokens per tile
    const int kvh = blockIdx.x, chunk = blockIdx.y;
    int group = 0, unit = blockIdx.z, start = 0, end = 0;
    for (; group < a.n_groups; ++group) {
        group_rows(a, group, start, end);
        const int units = (end - start + 2 * TQ - 1) / (2 * TQ);
        if (unit < units) break;
        unit -= units;
    }
    if (group >= a.n_groups) return;                         // the grid is an upper bound (uniform per CTA)
    const int row0 = start + unit * 2 * TQ, n_tok = min(2 * TQ, end - row0);
    const bool both = n_tok <= TQ;                           // one tile of rows, which both halves of the CTA work on
    const Span span = shared_span(a, group, span_scratch);
    const int per_chunk = a.chunk_shared / STEP;
    const int first_step = span.first / STEP + chunk * per_chunk;
    const int all_steps = (span.end + STEP - 1) / STEP;
    const int n_steps = span.first < span.end ? max(0, (chunk + 1 < a.n_shared ? min(all_steps, first_step + per_chunk) : all_steps) - first_step) : 0;
    if (n_steps == 0) {
        for (int i = threadIdx.x; i < n_tok * G; i += TC_THREADS) {
            float* ml = a.part_ml + (((size_t)(row0 + i / G) * a.nh + kvh * G + i % G) * n_splits + chunk) * 2;
            ml[0] = -INFINITY;
            ml[1] = 0.f;
        }
        return;
    }

    if (threadIdx.x == 0) {
        const int readers = both ? 1 : 2;                    // a step's keys and values are free when every tile that uses them has read them
        for (int s = 0; s < ST; ++s) {
            mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], readers);
            mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], readers);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(&q_ready[x], 128); mbar_init(&s_ready[x], 1); mbar_init(&s_free[x], 128);
            mbar_init(&p_half[x], 128); mbar_init(&p_ready[x], 128); mbar_init(&o_done[x], 1); mbar_init(&drained[x], 1);
        }
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    // The next kernel may start now: everything before this one is complete (it reads what those wrote before it waits for this
    // one), and this CTA has its tensor memory, which no later kernel's CTA can hold any more while it waits for this one.
    pdl_trigger_late();
    const uint32_t tmem = *tmem_slot;
    // tile x works on steps at(0), at(1), ... of the CTA's
    auto steps_of = [&](int x) { return both ? (n_steps + 1 - x) >> 1 : n_steps; };
    auto at = [&](int x, int j) { return both ? 2 * j + x : j; };

    if (warp == LOAD_WARP) {
        // keys and values are fetched as their buffers come free, whichever first
        const int* tab = table_row(a, start, 72);
        const int box = min(a.page_size, STEP), copies = STEP / box;
        const int first_blk = span.first / a.page_size, last_blk = (span.end - 1) / a.page_size;
        auto load = [&](int i, bool values) {                // warp-uniform call
            const int s = i % ST;
            uint8_t* dst = (values ? v_s : k_s) + s * C::BLOCK;
            uint64_t* bar = values ? &v_full[s] : &k_full[s];
            if (lane == 0) mbar_expect_tx(bar, C::BLOCK);
            __syncwarp();
            for (int c = lane; c < copies; c += 32) {
                // blocks in which nothing is seen: a page that is seen stands in for them (its values are cleared below)
                const int key = (first_step + i) * STEP + c * box, blk = min(max(key / a.page_size, first_blk), last_blk);
                int page = tab != nullptr && blk < a.max_blocks ? tab[blk] : -1;
                if (page < 0 || page >= a.n_pages) {
                    report(a.status, IMPARO_ST_PAGE_RANGE, 73, start, page);
                    page = 0;
                }
                const int y = page * a.page_size + key % a.page_size;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    tma_load_2d(dst + nb * REGION + (uint32_t)c * box * 128, values ? &map_v : &map_k, bar, kvh * HD + nb * 64, y);
            }
        };
        int k_next = 0, v_next = 0;
        uint32_t idle = 0;
        while (k_next < n_steps || v_next < n_steps) {
            int what = 0;                                    // bit 0: the next keys' buffer is free, bit 1: the next values', bit 2: stop
            if (lane == 0) {
                if (k_next < n_steps && (k_next < ST || mbar_test(&k_empty[k_next % ST], ((k_next / ST) - 1) & 1))) what |= 1;
                if (v_next < n_steps && (v_next < ST || mbar_test(&v_empty[v_next % ST], ((v_next / ST) - 1) & 1))) what |= 2;
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
    } else if (warp == MMA_WARP || warp == MMA_WARP + 1) {
        const int x = warp - MMA_WARP, n_x = steps_of(x);
        const uint64_t qd = smem_desc(smem_u32(q_s + x * C::BLOCK)), kd0 = smem_desc(smem_u32(k_s)), vd0 = desc_mn(smem_u32(v_s));
        const uint32_t id_s = idesc(STEP, false), id_o = idesc(HD, true);
        const uint32_t t_s = tmem + C::S_COL + x * 128, t_o = tmem + C::O_COL + x * HD, t_p = tmem + C::P_COL + x * C::P_STRIDE;
        auto wait = [&](uint64_t* bar, uint32_t parity, int code, int j) -> bool {       // the whole warp
            int good = 1;
            if (lane == 0 && !mbar_wait(bar, parity)) {
                report(a.status, IMPARO_ST_WAIT_LIMIT, code, j, x);
                *gave_up = 1;
                good = 0;
            }
            good = __shfl_sync(0xffffffffu, good, 0);
            fence_after();
            return good != 0;
        };
        auto issue_s = [&](int j) {                          // S = Q K^T of the tile's step j
            if (lane == 0) {
                const int s = at(x, j) % ST;
                const uint64_t kd = kd0 + (uint64_t)((s * C::BLOCK) >> 4);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int k = 0; k < BK / UMMA_K; ++k)
                        umma(t_s, qd + (uint64_t)((nb * REGION + k * 32) >> 4), kd + (uint64_t)((nb * REGION + k * 32) >> 4), id_s,
                             (nb > 0 || k > 0) ? 1u : 0u);
                umma_commit(&s_ready[x]);
                umma_commit(&k_empty[s]);
            }
            __syncwarp();
        };
        auto issue_pv = [&](int j, int half) {               // O += P V over 64 keys of the step
            if (lane == 0) {
                const int s = at(x, j) % ST;
                const uint64_t vd = vd0 + (uint64_t)((s * C::BLOCK) >> 4);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int kk = half * 4 + u;
                    umma_ta(t_o, t_p + kk * 8, vd + (uint64_t)((kk * (UMMA_K * 128)) >> 4), id_o, (kk > 0 || j > 0) ? 1u : 0u);
                }
                if (half == 1) {
                    umma_commit(&o_done[x]);
                    umma_commit(&v_empty[s]);
                }
            }
            __syncwarp();
        };
        // values outside the span are cleared: their weights are 0, and what lies there may be infinite or no number
        auto clear_values = [&](int j) {
            const int key0 = (first_step + at(x, j)) * STEP, lo = max(0, span.first - key0), hi = min(STEP, span.end - key0);
            if (lo == 0 && hi == STEP) return;
            uint8_t* v = v_s + (at(x, j) % ST) * C::BLOCK;
            for (int i = lane; i < STEP * NB * 8; i += 32) {
                const int row = (i >> 3) % STEP, nb = (i >> 3) / STEP;
                if (row < lo || row >= hi) *reinterpret_cast<uint4*>(v + nb * REGION + row * 128 + (i & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        auto full = [&](uint64_t* bar, int j, int code) { const int i = at(x, j); return wait(&bar[i % ST], (i / ST) & 1, code, j); };
        bool ok = n_x > 0 && wait(&q_ready[x], 0, 75, 0) && full(k_full, 0, 76);
        if (ok) issue_s(0);
        for (int j = 0; j < n_x && ok; ++j) {
            if (!C::ALIAS && j + 1 < n_x) {
                ok = wait(&s_free[x], j & 1, 77, j) && full(k_full, j + 1, 76);
                if (!ok) break;
                issue_s(j + 1);
            }
            ok = full(v_full, j, 78);
            if (!ok) break;
            clear_values(j);
            ok = wait(&p_half[x], j & 1, 79, j);
            if (!ok) break;
            issue_pv(j, 0);
            ok = wait(&p_ready[x], j & 1, 80, j);
            if (!ok) break;
            issue_pv(j, 1);
            if (C::ALIAS && j + 1 < n_x) {                   // (behind P V in the tensor cores' order, which reads the same columns)
                ok = full(k_full, j + 1, 76);
                if (!ok) break;
                issue_s(j + 1);
            }
        }
        if (lane == 0) {                                     // tensor memory is given back only when nothing uses it any more
            umma_commit(&drained[x]);
            mbar_wait(&drained[x], 0);
        }
        __syncwarp();
    } else if (warp < 8) {
        const int x = warp >> 2, r = (warp & 3) * 32 + lane, n_x = steps_of(x);
        const int tok0 = row0 + (both ? 0 : x * TQ), toks = both ? n_tok : min(TQ, max(0, n_tok - x * TQ));
        const bool valid = r < toks * G;
        const bool warp_valid = (warp & 3) * 32 < toks * G;
        const int t = tok0 + (valid ? r / G : 0), head = kvh * G + r % G;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + lanes + C::S_COL + x * 128, t_o = tmem + lanes + C::O_COL + x * HD, t_p = tmem + lanes + C::P_COL + x * C::P_STRIDE;
        {
            const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)t * a.q_stride + (size_t)head * HD);
            uint8_t* dst = q_s + x * C::BLOCK + r * 128;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c)
                *reinterpret_cast<uint4*>(dst + (c >> 3) * REGION + (((c & 7) ^ (r & 7)) << 4)) = valid ? src[c] : make_uint4(0u, 0u, 0u, 0u);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            arrive(&q_ready[x]);
        }
        const float sl2 = a.scale * LOG2E;                   // scores in units of log2(e)
        float m = -INFINITY;                                 // the max in use, scaled
        float2 l2 = make_float2(0.f, 0.f);
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, int code, int j) {
            if (!mbar_wait(bar, parity)) { report(a.status, IMPARO_ST_WAIT_LIMIT, code, j, r); *gave_up = 1; ok = false; }
            ok = __all_sync(0xffffffffu, ok);
            fence_after();
        };
        for (int j = 0; j < n_x; ++j) {
            wait(&s_ready[x], j & 1, 81, j);
            if (!ok) break;
            uint32_t sv[128];
            float corr = 1.f, m_new = m;
            if (warp_valid) {
                tmem_ld32(t_s, sv); tmem_ld32(t_s + 32, sv + 32); tmem_ld32(t_s + 64, sv + 64); tmem_ld32(t_s + 96, sv + 96);
                wait_ld();
#pragma unroll
                for (int i = 0; i < 128; ++i) asm volatile("" : "+r"(sv[i]) :: "memory");
            }
            fence_before();
            arrive(&s_free[x]);                              // the score columns may take the next step's product
            bool rescale = false;
            if (warp_valid) {
                const int key0 = (first_step + at(x, j)) * STEP, lo = span.first - key0, hi = span.end - key0;
                if (lo > 0 || hi < STEP) {
#pragma unroll
                    for (int i = 0; i < 128; ++i)
                        if (i < lo || i >= hi) sv[i] = __float_as_uint(-INFINITY);
                }
                float mx0 = __uint_as_float(sv[0]), mx1 = __uint_as_float(sv[1]);
#pragma unroll
                for (int i = 2; i < 126; i += 4) {
                    mx0 = max3(mx0, __uint_as_float(sv[i]), __uint_as_float(sv[i + 1]));
                    mx1 = max3(mx1, __uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3]));
                }
                mx0 = fmaxf(max3(mx0, __uint_as_float(sv[126]), __uint_as_float(sv[127])), mx1) * sl2;     // (a rising function: scale > 0)
                const bool grow = mx0 > m + GROW;            // (true for m = -inf and a finite max)
                rescale = __any_sync(0xffffffffu, grow && j > 0);
                m_new = grow ? mx0 : m;
                corr = m == -INFINITY ? 0.f : ex2(m - m_new);
            }
            if (j > 0) wait(&o_done[x], (j - 1) & 1, 82, j);
            if (!ok) break;
            if (rescale) {                                   // the accumulated output of this warp's rows, in place
#pragma unroll 1
                for (int c = 0; c < HD; c += 16) {
                    float ov[16];
                    tmem_ld16(t_o + c, ov);
                    uint32_t ow[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) ow[e] = __float_as_uint(ov[e] * corr);
                    tmem_st16(t_o + c, ow);
                }
            }
            if (warp_valid) {
                l2.x *= corr; l2.y *= corr;
                m = m_new;
                const float nb = m == -INFINITY ? 0.f : -m;
                const float2 sl = make_float2(sl2, sl2), base = make_float2(nb, nb);
#pragma unroll
                for (int c = 0; c < 4; ++c) {                // 32 keys = 16 columns of P
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float2 e = __ffma2_rn(make_float2(__uint_as_float(sv[c * 32 + 2 * i]), __uint_as_float(sv[c * 32 + 2 * i + 1])), sl, base);
                        e.x = ex2(e.x);
                        e.y = ex2(e.y);
                        l2 = __fadd2_rn(l2, e);
                        w[i] = pack_bf16(e.x, e.y);
                    }
                    tmem_st16(t_p + c * 16, w);
                    if (c == 1) { wait_st(); fence_before(); arrive(&p_half[x]); }
                }
                wait_st();
                fence_before();
            } else {
                arrive(&p_half[x]);
            }
            arrive(&p_ready[x]);
        }
        if (ok && n_x > 0) wait(&o_done[x], (n_x - 1) & 1, 83, n_x);
        float l = l2.x + l2.y;
        const size_t part = ((size_t)t * a.nh + head) * n_splits + chunk;
        // the second half's results for the first one to add: [dim][row] and (max, sum) per row, where keys and values were
        float* other = reinterpret_cast<float*>(k_s);
        if (both) {
            asm volatile("bar.sync 1, 256;" ::: "memory");   // both tiles' products have run
            if (x == 1 && ok) {
                if (n_x > 0 && warp_valid) {
#pragma unroll 1
                    for (int c = 0; c < HD; c += 16) {
                        float o[16];
                        tmem_ld16(t_o + c, o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) other[(c + e) * TILE + r] = o[e];
                    }
                }
                other[HD * TILE + r] = n_x > 0 ? m : -INFINITY;
                other[(HD + 1) * TILE + r] = n_x > 0 ? l : 0.f;
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        if (ok && !__any_sync(0xffffffffu, *gave_up) && (x == 0 || !both) && warp_valid) {
            float f = 1.f, g = 0.f, m_all = m;
            if (both) {
                const float m2 = other[HD * TILE + r], l_2 = other[(HD + 1) * TILE + r];
                if (l_2 > 0.f) {
                    m_all = fmaxf(m, m2);
                    f = m == -INFINITY ? 0.f : ex2(m - m_all);
                    g = ex2(m2 - m_all);
                    l = l * f + l_2 * g;
                }
            }
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
                float o[16];
                tmem_ld16(t_o + c, o);
                if (g != 0.f) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = o[e] * f + other[(c + e) * TILE + r] * g;
                }
                if (valid) {
                    float4* dst = reinterpret_cast<float4*>(a.part_acc + part * HD + c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dst[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                }
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
    if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ---- a row's own keys, and the join ----------------------------------------------------------------------------------
// One CTA per (stretch of own keys, kv head x tile of 16 query heads, token).  A warp takes 16 keys at a time on mma.sync: the heads
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

template <int HD, bool JOIN>
__global__ void __launch_bounds__(OWN_WARPS * 32)
own_tc_kernel(const Args a, __nv_bfloat16* __restrict__ out, const float* __restrict__ sinks, const int n_splits) {
    constexpr int NB = HD / 64, KB = HD / 32;                // 64-dim blocks (values), 32-dim blocks (keys)
    __shared__ int span_scratch[2];
    __shared__ float w_m[OWN_WARPS][16], w_l[OWN_WARPS][16];
    __shared__ __align__(16) float w_o[OWN_WARPS][16][HD + 4];
    pdl_trigger();
    pdl_no_wait();                                           // (what this reads before its wait was complete before the kernel ahead let it start)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tg = lane & 3;
    const int G = a.nh / a.nkv, head_tiles = (G + 15) / 16;
    const int kvh = blockIdx.x / head_tiles, head0 = kvh * G + blockIdx.x % head_tiles * 16, n_heads = min(16, kvh * G + G - head0);
    const int t = blockIdx.y, split = blockIdx.z;
    const int group = group_of(a, t);
    const Span span = shared_span(a, group, span_scratch);
    const Own own = own_keys(a, a.positions[t], span);
    const int k0 = (int)min((long long)split * a.chunk_own, (long long)own.count);
    const int k1 = split + 1 == a.n_own ? own.count : (int)min((long long)k0 + a.chunk_own, (long long)own.count);
    const int* tab = k0 < k1 ? table_row(a, t, 84) : nullptr;
    const size_t kvw = (size_t)a.nkv * HD;
    const __nv_bfloat16* kc = reinterpret_cast<const __nv_bfloat16*>(a.k) + (size_t)kvh * HD;
    const __nv_bfloat16* vc = reinterpret_cast<const __nv_bfloat16*>(a.v) + (size_t)kvh * HD;
    // the queries: heads g and g + 8, dims 32 b + 8 tg .. + 7
    uint4 qa[KB], qb[KB];
    {
        const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)t * a.q_stride + (size_t)head0 * HD + tg * 8;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            qa[b] = g < n_heads ? *reinterpret_cast<const uint4*>(q + (size_t)g * HD + b * 32) : make_uint4(0u, 0u, 0u, 0u);
            qb[b] = g + 8 < n_heads ? *reinterpret_cast<const uint4*>(q + (size_t)(g + 8) * HD + b * 32) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    float o[NB * 8][4];                                      // output tile nb * 8 + i: dims 64 nb + 8 column + i
#pragma unroll
    for (int i = 0; i < NB * 8; ++i) { o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f; }
    float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;
    const float sl2 = a.scale * LOG2E;
    if (tab != nullptr) {
        for (int base = k0 + warp * 16; base < k1; base += OWN_WARPS * 16) {
            int row = -1;                                    // lane i < 16: where key base + i lies
            if (lane < 16 && base + lane < k1) {
                const int key = own.key(base + lane), block = key / a.page_size;
                const int page = block < a.max_blocks ? tab[block] : -1;
                if (page < 0 || page >= a.n_pages) report(a.status, IMPARO_ST_PAGE_RANGE, 85, t, page);
                else row = page * a.page_size + key % a.page_size;
            }
            const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
            uint4 kf[2][KB], vf[4][NB];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int at = __shfl_sync(0xffffffffu, row, n * 8 + g);
#pragma unroll
                for (int b = 0; b < KB; ++b)
                    kf[n][b] = at >= 0 ? __ldg(reinterpret_cast<const uint4*>(kc + (size_t)at * kvw + b * 32 + tg * 8)) : zero;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {                    // keys 2 tg, 2 tg + 1, 2 tg + 8, 2 tg + 9
                const int at = __shfl_sync(0xffffffffu, row, 2 * tg + (u & 1) + (u >> 1) * 8);
#pragma unroll
                for (int b = 0; b < NB; ++b)
                    vf[u][b] = at >= 0 ? __ldg(reinterpret_cast<const uint4*>(vc + (size_t)at * kvw + b * 64 + g * 8)) : zero;
            }
            const unsigned there = __ballot_sync(0xffffffffu, row >= 0);
            float s[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    mma16816(s[n], qa[b].x, qb[b].x, qa[b].y, qb[b].y, kf[n][b].x, kf[n][b].y);
                    mma16816(s[n], qa[b].z, qb[b].z, qa[b].w, qb[b].w, kf[n][b].z, kf[n][b].w);
                }
            }
            float mx_a = -INFINITY, mx_b = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool seen = (there >> (n * 8 + 2 * tg + e)) & 1u;
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
            for (int i = 0; i < NB * 8; ++i) { o[i][0] *= ca; o[i][1] *= ca; o[i][2] *= cb; o[i][3] *= cb; }
            const uint32_t p0 = pack_bf16(s[0][0], s[0][1]), p1 = pack_bf16(s[0][2], s[0][3]), p2 = pack_bf16(s[1][0], s[1][1]),
                           p3 = pack_bf16(s[1][2], s[1][3]);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const uint32_t x0[4] = {vf[0][b].x, vf[0][b].y, vf[0][b].z, vf[0][b].w}, x1[4] = {vf[1][b].x, vf[1][b].y, vf[1][b].z, vf[1][b].w};
                const uint32_t x2[4] = {vf[2][b].x, vf[2][b].y, vf[2][b].z, vf[2][b].w}, x3[4] = {vf[3][b].x, vf[3][b].y, vf[3][b].z, vf[3][b].w};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t pick = i & 1 ? 0x7632u : 0x5410u;
                    mma16816(o[b * 8 + i], p0, p1, p2, p3, __byte_perm(x0[i >> 1], x1[i >> 1], pick), __byte_perm(x2[i >> 1], x3[i >> 1], pick));
                }
            }
        }
        l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
        l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
        l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
        l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
    }
    if (tg == 0) { w_m[warp][g] = m_a; w_l[warp][g] = l_a; w_m[warp][g + 8] = m_b; w_l[warp][g + 8] = l_b; }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        // a lane's columns of the eight tiles are 2 tg and 2 tg + 1: dims 8 (2 tg) .. + 7 and the eight behind them
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float* dst = &w_o[warp][g][b * 64 + 8 * (2 * tg + e) + 4 * h];
                *reinterpret_cast<float4*>(dst) = make_float4(o[b * 8 + 4 * h][e], o[b * 8 + 4 * h + 1][e], o[b * 8 + 4 * h + 2][e], o[b * 8 + 4 * h + 3][e]);
                dst = &w_o[warp][g + 8][b * 64 + 8 * (2 * tg + e) + 4 * h];
                *reinterpret_cast<float4*>(dst) = make_float4(o[b * 8 + 4 * h][2 + e], o[b * 8 + 4 * h + 1][2 + e], o[b * 8 + 4 * h + 2][2 + e],
                                                              o[b * 8 + 4 * h + 3][2 + e]);
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
    for (int i = tid; i < n_heads * (HD / 4); i += OWN_WARPS * 32) {
        const int h = i / (HD / 4), d = i % (HD / 4) * 4;
        const size_t row = (size_t)t * a.nh + head0 + h;
        const float* ml = a.part_ml + row * n_splits * 2;
        float m = -INFINITY;
        for (int w = 0; w < OWN_WARPS; ++w) m = fmaxf(m, w_m[w][h]);
        if (JOIN) {
            for (int s = 0; s < live; ++s) if (__ldcg(ml + 2 * s + 1) != 0.f) m = fmaxf(m, __ldcg(ml + 2 * s) * LOG2E);
            if (sinks) m = fmaxf(m, sinks[head0 + h] * LOG2E);
        }
        float l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < OWN_WARPS; ++w) {
            if (w_l[w][h] == 0.f) continue;
            const float f = ex2(w_m[w][h] - m);
            const float4 x = *reinterpret_cast<const float4*>(&w_o[w][h][d]);
            l += w_l[w][h] * f;
            acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
        }
        if (JOIN) {
            const float4* part = reinterpret_cast<const float4*>(a.part_acc + row * n_splits * HD + d);
#pragma unroll 4
            for (int s = 0; s < live; ++s) {
                const float4 x = __ldcg(part + (size_t)s * (HD / 4));
                const float ls = __ldcg(ml + 2 * s + 1);
                if (ls != 0.f) {
                    const float f = ex2(__ldcg(ml + 2 * s) * LOG2E - m);
                    l += ls * f;
                    acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
                }
            }
            if (sinks) l += ex2(sinks[head0 + h] * LOG2E - m);
            const float inv = l > 0.f ? 1.0f / l : 0.f;
            *reinterpret_cast<uint2*>(out + row * HD + d) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
        } else {
            *reinterpret_cast<float4*>(a.part_acc + (row * n_splits + a.n_shared + split) * HD + d) = acc;
            if (d == 0) {
                float* mine = a.part_ml + (row * n_splits + a.n_shared + split) * 2;
                mine[0] = m == -INFINITY ? -INFINITY : m * LN2;
                mine[1] = l;
            }
            // a row of no group has no part in the shared stretches
            if (d == 0 && split == 0 && group < 0)
                for (int s = 0; s < a.n_shared; ++s) {
                    a.part_ml[(row * n_splits + s) * 2] = -INFINITY;
                    a.part_ml[(row * n_splits + s) * 2 + 1] = 0.f;
                }
        }
    }
    if (!JOIN && tid == 0) pdl_wait_at_end();                // this kernel completes after the one it ran beside
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
    static bool configured[64] = {};                         // the attribute is the device's
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    if (device < 0 || device >= 64 || !configured[device]) {
        e = cudaFuncSetAttribute(shared_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<HD>::SMEM);
        if (e != cudaSuccess) return (int)e;
        if (device >= 0 && device < 64) configured[device] = true;
    }
    const int n_splits = a.n_own == 1 ? a.n_shared : a.n_shared + a.n_own;
    const long long units = (a.n_rows + 2 * TQ - 1) / (2 * TQ) + a.n_groups - 1;       // every group may end a tile early
    e = launch(shared_tc_kernel<HD>, dim3(a.nkv, a.n_shared, (unsigned)units), dim3(TC_THREADS), Shape<HD>::SMEM, stream, mk, mv, a, n_splits);
    if (e != cudaSuccess) return (int)e;
    const dim3 grid(a.nkv * head_tiles, a.n_rows, a.n_own);
    e = a.n_own == 1 ? launch(own_tc_kernel<HD, true>, grid, dim3(OWN_WARPS * 32), 0, stream, a, out, sinks, n_splits)
                     : launch(own_tc_kernel<HD, false>, grid, dim3(OWN_WARPS * 32), 0, stream, a, out, sinks, n_splits);
    return e == cudaSuccess ? 0 : (int)e;
}

int launch_tc(const Args& a, void* out, const float* sinks, cudaStream_t stream) {
    const int G = a.nh / a.nkv;
    if ((a.hd != 64 && a.hd != 128) || G > TILE || !(a.scale > 0.f)) return -8;
    if (a.page_size != 16 && a.page_size != 32 && a.page_size != 64 && a.page_size % STEP != 0) return -8;
    if (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)out | (uintptr_t)a.part_acc) & 15) return -8;
    if (a.q_stride % 8 != 0 || a.chunk_shared % STEP != 0) return -8;
    if (a.n_rows > 65535 || a.n_own > 65535 || a.n_rows + a.n_groups > 65535) return -8;
    return a.hd == 64 ? launch_hd<64>(a, (__nv_bfloat16*)out, sinks, stream) : launch_hd<128>(a, (__nv_bfloat16*)out, sinks, stream);
}

}  // namespace sp
}  // namespace imparo
