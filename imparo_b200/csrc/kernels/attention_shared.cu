// Attention of single-token rows whose first positions are the same pages of the cache: continuations of one prompt, or questions
// behind one document.  The rows are cut into groups; the positions 0 .. shared - 1 of a group's rows are read by the block table of
// its first row that has a position, once for all of its rows, the rest of each row by its own table.
//
//   o_t = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q_t . k_j),  lo_t <= j <= pos_t        (lo_t = 0, or pos_t + 1 - window)
//
// The keys are cut: the shared ones into n_shared stretches of chunk_shared, a row's own ones into n_own stretches of chunk_own (the
// last stretch of either takes all that is left, so every key is seen whatever the lengths the launch was planned for).  Each
// stretch leaves, per row and head, the largest score, the sum of exp(score - largest) and the sum of the weighted values in 32-bit
// (part_ml [rows, heads, splits, 2], part_acc [rows, heads, splits, head size], splits = n_shared + n_own), which the ordered combine
// of attention_split.cu joins.
#include "attention_shared.cuh"

namespace imparo {
namespace sp {

// ---- any head size, 32-bit or bfloat16 -------------------------------------------------------------------------------
// A CTA takes up to 16 rows (tokens of one group x query heads of one kv head) and one stretch of keys, 32 keys at a time in shared
// memory; eight threads per row make four scores each, then an eighth of the row's output each.  What bounds it is the chain of a
// stretch's few tiles (page lookup, keys and values, scores, weights): short stretches on many CTAs, up to four per SM.  5 rows of 16
// heads in 8 groups of 64 over 1,001 shared positions in 32-bit: 18 us with the join, of which the caches' bytes would need 0.7.
constexpr int ROWS = 16, KEYS = 32, THREADS = 128;
constexpr int MOST_HEAD = 256;

// 16 bytes of a cache row as 32-bit numbers
__device__ __forceinline__ void unpack16(const uint4& x, const float*, float (&v)[4]) {
    v[0] = __uint_as_float(x.x); v[1] = __uint_as_float(x.y); v[2] = __uint_as_float(x.z); v[3] = __uint_as_float(x.w);
}
__device__ __forceinline__ void unpack16(const uint4& x, const __nv_bfloat16*, float (&v)[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}

// HM: the head size rounded up to 64, 128 or 256.  aligned: the caches start on 16 bytes (their rows then do too).
template <typename T, int HM>
__global__ void __launch_bounds__(THREADS)
shared_any_kernel(const Args a, const int aligned) {
    extern __shared__ __align__(16) float sp_smem[];
    __shared__ int key_row[KEYS];
    const int hd = a.hd, ks_stride = hd + 4;
    float* qs = sp_smem;                                           // [ROWS][hd]
    float* ks = qs + ROWS * hd;                                    // [KEYS][hd + 4]
    float* vs = ks + KEYS * ks_stride;                             // [KEYS][hd]
    float* ps = vs + KEYS * hd;                                    // [ROWS][KEYS + 1]
    pdl_trigger();
    pdl_wait();
    const int G = a.nh / a.nkv, n_splits = a.n_shared + a.n_own;
    const int heads_per = min(G, ROWS), head_tiles = (G + ROWS - 1) / ROWS, tokens_per = max(1, ROWS / G);
    const int split = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x;
    const bool is_own = split >= a.n_shared;
    int unit = blockIdx.z;
    const int head0 = unit % head_tiles * ROWS;
    unit /= head_tiles;
    int row0, n_tok, group;                                        // the tokens of this tile
    if (is_own) {
        if (unit >= a.n_rows) return;
        row0 = unit;
        n_tok = 1;
        group = group_of_warp(a, row0);
    } else {
        group = 0;
        n_tok = 0;
        row0 = 0;
        for (; group < a.n_groups; ++group) {
            int start, end;
            group_rows(a, group, start, end);
            const int tiles = (end - start + tokens_per - 1) / tokens_per;
            if (unit < tiles) {
                row0 = start + unit * tokens_per;
                n_tok = min(tokens_per, end - row0);
                break;
            }
            unit -= tiles;
        }
        if (group >= a.n_groups) return;
    }
    const int n_heads = min(heads_per, G - head0), n_rows = n_tok * n_heads;
    // a row of no group has no part in the shared stretches
    if (is_own && group < 0 && split == a.n_shared)
        for (int i = tid; i < n_heads * a.n_shared; i += THREADS) {
            float* ml = a.part_ml + (((size_t)row0 * a.nh + kvh * G + head0 + i / a.n_shared) * n_splits + i % a.n_shared) * 2;
            ml[0] = -INFINITY;
            ml[1] = 0.f;
        }
    const Span span = shared_span(a, group);

    // this thread's row: eight threads each
    const int r = tid >> 3, sub = tid & 7;
    const bool written = r < n_rows;
    const int t = row0 + (written ? r / n_heads : 0), head = kvh * G + head0 + (written ? r % n_heads : 0);
    const bool valid = written && a.positions[t] >= 0;
    // the stretch: keys counted through from the first shared or own one
    const int chunk = is_own ? a.chunk_own : a.chunk_shared, at = is_own ? split - a.n_shared : split;
    const bool last = at + 1 == (is_own ? a.n_own : a.n_shared);
    const Own own = own_keys(a, a.positions[row0], span);
    const int total = is_own ? own.count : span.end - span.first;
    const int k0 = (int)min((long long)at * chunk, (long long)total), k1 = last ? total : (int)min((long long)k0 + chunk, (long long)total);
    const int tab_of = is_own ? row0 : span.row;                   // the row whose table gives the pages
    const int* tab = k0 < k1 ? table_row(a, tab_of, 70) : nullptr;

    const size_t kvw = (size_t)a.nkv * hd;
    const T* q = reinterpret_cast<const T*>(a.q);
    const T* kc = reinterpret_cast<const T*>(a.k) + (size_t)kvh * hd;
    const T* vc = reinterpret_cast<const T*>(a.v) + (size_t)kvh * hd;
    // (eight threads a row in every loop: no division by the head size)
    if (written) {
        const T* src = q + (size_t)t * a.q_stride + (size_t)head * hd;
        for (int d = sub; d < hd; d += 8) qs[r * hd + d] = to_f32(src[d]);
    }
    constexpr int OUT = HM / 32, VEC = 16 / sizeof(T);             // outputs of a thread: four dims from 4 sub on, every 32
    float4 o[OUT];
#pragma unroll
    for (int i = 0; i < OUT; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    for (int key0 = k0; tab != nullptr && key0 < k1; key0 += KEYS) {
        const int n = min(KEYS, k1 - key0);
        __syncthreads();                                           // the tile before is no longer read
        if (tid < KEYS) {
            int at_row = -1;
            if (tid < n) {
                const int key = is_own ? own.key(key0 + tid) : span.first + key0 + tid, block = key / a.page_size;
                const int page = block < a.max_blocks ? tab[block] : -1;
                if (page < 0 || page >= a.n_pages) report(a.status, IMPARO_ST_PAGE_RANGE, 71, tab_of, page);
                else at_row = page * a.page_size + key % a.page_size;
            }
            key_row[tid] = at_row;
        }
        __syncthreads();
        if (aligned) {
            // both tiles' loads of a thread are on their way before the first is used
            constexpr int TURNS = KEYS / ROWS, MOST = HM / VEC / 8 > 0 ? HM / VEC / 8 : 1;
#pragma unroll
            for (int c = 0; c < MOST; ++c) {
                const int at = (sub + 8 * c) * VEC;
                uint4 x[TURNS][2];
#pragma unroll
                for (int u = 0; u < TURNS; ++u) {
                    const int at_row = key_row[r + u * ROWS];
                    const bool there = at_row >= 0 && at < hd;
                    x[u][0] = there ? *reinterpret_cast<const uint4*>(kc + (size_t)at_row * kvw + at) : make_uint4(0u, 0u, 0u, 0u);
                    x[u][1] = there ? *reinterpret_cast<const uint4*>(vc + (size_t)at_row * kvw + at) : make_uint4(0u, 0u, 0u, 0u);
                }
                if (at < hd) {
#pragma unroll
                    for (int u = 0; u < TURNS; ++u) {
                        const int j = r + u * ROWS;
                        float v[VEC];
                        unpack16(x[u][0], kc, v);
#pragma unroll
                        for (int e = 0; e < VEC; e += 4) *reinterpret_cast<float4*>(ks + j * ks_stride + at + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                        unpack16(x[u][1], vc, v);
#pragma unroll
                        for (int e = 0; e < VEC; e += 4) *reinterpret_cast<float4*>(vs + j * hd + at + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                    }
                }
            }
        } else {
            for (int j = r; j < KEYS; j += ROWS) {
                const int at_row = key_row[j];
                for (int d = sub; d < hd; d += 8) {
                    ks[j * ks_stride + d] = at_row >= 0 ? to_f32(kc[(size_t)at_row * kvw + d]) : 0.f;
                    vs[j * hd + d] = at_row >= 0 ? to_f32(vc[(size_t)at_row * kvw + d]) : 0.f;
                }
            }
        }
        __syncthreads();
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        if (valid) {
            for (int d = 0; d < hd; d += 4) {
                const float4 x = *reinterpret_cast<const float4*>(qs + r * hd + d);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 y = *reinterpret_cast<const float4*>(ks + (sub + 8 * i) * ks_stride + d);
                    s[i] += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
                }
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = sub + 8 * i;
            s[i] = valid && j < n && key_row[j] >= 0 ? s[i] * a.scale : -INFINITY;
            top = fmaxf(top, s[i]);
        }
#pragma unroll
        for (int w = 4; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const float m_new = fmaxf(m, top);
        const float corr = m == -INFINITY ? 0.f : expf(m - m_new);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = s[i] == -INFINITY ? 0.f : expf(s[i] - m_new);
            sum += p;
            ps[r * (KEYS + 1) + sub + 8 * i] = p;
        }
#pragma unroll
        for (int w = 4; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        l = l * corr + sum;
        m = m_new;
        __syncwarp();                                              // a row's probabilities are written and read by one warp
#pragma unroll
        for (int i = 0; i < OUT; ++i) { o[i].x *= corr; o[i].y *= corr; o[i].z *= corr; o[i].w *= corr; }
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const float p = ps[r * (KEYS + 1) + j];
#pragma unroll
            for (int i = 0; i < OUT; ++i) {
                if (4 * sub + 32 * i < hd) {
                    const float4 x = *reinterpret_cast<const float4*>(vs + j * hd + 4 * sub + 32 * i);
                    o[i].x += p * x.x; o[i].y += p * x.y; o[i].z += p * x.z; o[i].w += p * x.w;
                }
            }
        }
    }
    if (written) {
        const size_t at_part = ((size_t)t * a.nh + head) * n_splits + split;
        if (sub == 0) { a.part_ml[at_part * 2] = m; a.part_ml[at_part * 2 + 1] = l; }
        if (l != 0.f) {                                            // (a sum that is no number counts: the row has no result)
#pragma unroll
            for (int i = 0; i < OUT; ++i)
                if (4 * sub + 32 * i < hd) {
                    float* dst = a.part_acc + at_part * hd + 4 * sub + 32 * i;       // (the scratch may start anywhere)
                    dst[0] = o[i].x; dst[1] = o[i].y; dst[2] = o[i].z; dst[3] = o[i].w;
                }
        }
    }
}

template <typename T>
static int launch_any(const Args& a, cudaStream_t stream) {
    const int G = a.nh / a.nkv, head_tiles = (G + ROWS - 1) / ROWS, tokens_per = G >= ROWS ? 1 : ROWS / G;
    const long long tiles = (a.n_rows + tokens_per - 1) / tokens_per + a.n_groups;      // every group may end a tile early
    const long long units = (tiles > a.n_rows ? tiles : a.n_rows) * head_tiles;
    if (units > 65535 || a.nkv > 65535) return -2;
    const size_t smem = sizeof(float) * (ROWS * a.hd + KEYS * (a.hd + 4) + KEYS * a.hd + ROWS * (KEYS + 1));
    auto kern = a.hd <= 64 ? shared_any_kernel<T, 64> : a.hd <= 128 ? shared_any_kernel<T, 128> : shared_any_kernel<T, 256>;
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
    }
    const int aligned = (((uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0;
    cudaError_t e = launch(kern, dim3(a.n_shared + a.n_own, a.nkv, (unsigned)units), dim3(THREADS), smem, stream, a, aligned);
    return e == cudaSuccess ? 0 : (int)e;
}

}  // namespace sp
}  // namespace imparo

using namespace imparo;

extern "C" int imparo_attention_split_combine_any_sum(const float* part_acc, const float* part_ml, void* out, int dtype, int n_rows, int hd,
                                                      int n_splits, const float* sink_values, int nh, cudaStream_t stream);

extern "C" int imparo_attention_shared(const void* q, long long q_stride, const void* k_cache, const void* v_cache, int dtype,
                                       const int* positions, const int* item_of_token, const int* table, int n_items, int max_blocks,
                                       int page_size, int n_pages, const int* group_start, const int* shared, int n_groups, int window,
                                       float scale, const float* sink_values, void* out, float* part_acc, float* part_ml, int n_rows,
                                       int nh, int nkv, int hd, int chunk_shared, int n_shared, int chunk_own, int n_own, int* status,
                                       cudaStream_t stream) {
    if (n_rows <= 0) return 0;
    if (hd < 16 || hd > sp::MOST_HEAD || hd % 16 != 0) return -3;
    if (nkv <= 0 || nh <= 0 || nh % nkv != 0) return -5;
    if (n_groups < 1 || n_items < 1 || max_blocks < 1 || page_size < 1 || n_pages < 1 || (long long)n_pages * page_size > 0x7fffffffll)
        return -2;
    if (chunk_shared < 1 || n_shared < 1 || chunk_own < 1 || n_own < 1 || n_shared + n_own > 2048) return -2;
    if ((long long)n_rows * nh > 0x7fffffffll) return -2;
    if (dtype != IMPARO_DT_F32 && dtype != IMPARO_DT_BF16) return -1;
    sp::Args a;
    a.q = q; a.k = k_cache; a.v = v_cache; a.positions = positions; a.item_of_token = item_of_token; a.table = table;
    a.group_start = group_start; a.shared = shared; a.part_acc = part_acc; a.part_ml = part_ml; a.status = status; a.q_stride = q_stride;
    a.n_rows = n_rows; a.n_items = n_items; a.n_groups = n_groups; a.max_blocks = max_blocks; a.page_size = page_size;
    a.n_pages = n_pages; a.window = window; a.nh = nh; a.nkv = nkv; a.hd = hd;
    a.chunk_shared = chunk_shared; a.n_shared = n_shared; a.chunk_own = chunk_own; a.n_own = n_own; a.scale = scale;
    const long long positions_of_table = (long long)max_blocks * page_size;
    a.most_pos = (int)(positions_of_table < 0x7ffffffell ? positions_of_table : 0x7ffffffell);
    int rc = dtype == IMPARO_DT_BF16 ? sp::launch_tc(a, out, sink_values, stream) : -8;
    if (rc == 0 && n_own == 1) return 0;                     // its second kernel has joined everything
    if (rc == -8) rc = dtype == IMPARO_DT_F32 ? sp::launch_any<float>(a, stream) : sp::launch_any<__nv_bfloat16>(a, stream);
    if (rc != 0) return rc;
    return imparo_attention_split_combine_any_sum(part_acc, part_ml, out, dtype, n_rows * nh, hd, n_shared + n_own, sink_values, nh, stream);
}
