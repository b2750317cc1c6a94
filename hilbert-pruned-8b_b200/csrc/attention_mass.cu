// Causal grouped attention over the paged cache that also adds up how much weight every cached row got: the kernels that take
// every head size up to 256, every group and both types, and the second half of steps of few tokens.
//
// For a token t of a sequence, a query head h of kv head g and a row j the token sees (lo..p, as in attention_general.cu):
//   s = scale q_th . k_jg,  lse_th = log sum_j exp(s),  w = exp(s - lse_th),  out_th = sum_j w v_jg,
//   mass_jg = (j appended by this step ? 0 : before_jg) + sum over the sequence's tokens t of the step and the heads h of g of w.
// A row's weight is known only once the token has seen all its keys, and then the scores are gone.  Two ways:
//   steps of few tokens   (memory-bound) the scores themselves are written beside the partial results, 4 bytes per (head, row) against
//                         the 2 head sizes of a key and a value; one more launch joins the partial results and turns the scores into
//                         weights (short sequences: the same block does it).  Keys and values are read once for a block of (token, head) pairs.
//   steps of many tokens  (bound by arithmetic) the tokens' log-sums are kept and a second kernel, a block per tile of keys,
//                         computes its keys' scores with all queries once more: half as much arithmetic again instead of
//                         writing and reading a weight for every (token, head, row).  Every key's sum belongs to one thread from
//                         beginning to end, so the order of the additions is fixed.
// Softmax statistics, scores, sums and mass are float32; lse is in units of log 2.
#include <type_traits>

#include "api.h"
#include "attention_mass.cuh"
#include "mma.cuh"

// ------------------------------------------------------------------------------------------- many tokens, every head size
// Tiles of 64 queries (of one head) x 64 keys, 256 threads, 4 x 4 scores a thread (rows ty + 16 i, keys tx + 16 j), operands
// widened to float32 in shared memory, products on the FP32 pipe: the true 32-bit path has no other.  NC: value columns a thread
// holds (head size up to 16 NC).
#define AM_ROWS 64
#define AM_KEYS 64
#define AM_THREADS 256

// 64 rows of a tensor as float32 in shared memory, `ld` apart (a multiple of 4), in two halves so that the loads can be in flight while
// something else is computed: registers (up to 4 NC numbers a thread), then shared memory.  Rows outside [from, rows) and columns
// behind hd are zero.  vec: rows are aligned for four elements at a time.
template <typename T, int NC>
struct AmTile {
    float4 x[NC];
    __device__ __forceinline__ void load(const T* src, long long stride, int hd, int rows, bool vec, int tid, int from = 0) {
        const int per = (hd + 3) >> 2;
#pragma unroll
        for (int u = 0; u < NC; u++) {
            const int i = tid + u * AM_THREADS, r = i / per, d = (i - r * per) * 4;
            x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (r >= from && r < rows) {
                const T* p = src + (size_t)r * stride + d;
                if (vec) {
                    float v[4];
                    load4(p, v);
                    x[u] = make_float4(v[0], v[1], v[2], v[3]);
                } else {
                    x[u].x = to_f32(p[0]);
                    if (d + 1 < hd) x[u].y = to_f32(p[1]);
                    if (d + 2 < hd) x[u].z = to_f32(p[2]);
                    if (d + 3 < hd) x[u].w = to_f32(p[3]);
                }
            }
        }
    }
    __device__ __forceinline__ void store(float* dst, int hd, int ld, int tid) const {
        const int per = (hd + 3) >> 2;
#pragma unroll
        for (int u = 0; u < NC; u++) {
            const int i = tid + u * AM_THREADS, r = i / per, d = (i - r * per) * 4;
            if (r < 64) *reinterpret_cast<float4*>(dst + r * ld + d) = x[u];
        }
    }
};

// s[i][j] = sum_d a[ty + 16 i][d] b[tx + 16 j][d]
__device__ __forceinline__ void am_scores(float (&s)[4][4], const float* a, const float* b, int ld, int tx, int ty) {
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[i][j] = 0.0f;
    for (int d = 0; d < ld - 4; d += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = *reinterpret_cast<const float4*>(a + (ty + 16 * i) * ld + d);
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * ld + d);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s[i][j] = fmaf(x[i].x, y[j].x, s[i][j]);
                s[i][j] = fmaf(x[i].y, y[j].y, s[i][j]);
                s[i][j] = fmaf(x[i].z, y[j].z, s[i][j]);
                s[i][j] = fmaf(x[i].w, y[j].w, s[i][j]);
            }
    }
}

static __host__ __device__ constexpr int am_ld(int hd) { return ((hd + 3) & ~3) + 4; }      // 4 more: rows start in different banks

template <typename T, int NC>
__global__ void __launch_bounds__(AM_THREADS)
attention_rows_kernel(const T* __restrict__ q, long long q_stride, const T* __restrict__ kc, const T* __restrict__ vc,
                      const int* __restrict__ page_table, int pt_width, const int* __restrict__ seq_start, const int* __restrict__ seq_pos0,
                      T* __restrict__ out, long long out_stride, float* __restrict__ lse, Shares sh, int n_tokens, int n_seqs, int nh, int nkv,
                      int hd, float scale_log2e, int window, int n_pages, int vec_q, int vec_kv, int* status) {
    extern __shared__ __align__(16) float am_smem[];
    pdl_trigger();
    pdl_wait();
    mass_fresh(page_table, seq_start, seq_pos0);
    q = pdl_fresh(q);
    kc = pdl_fresh(kc);
    vc = pdl_fresh(vc);
    const int ld = am_ld(hd);
    float* qs = am_smem;                                 // [64][ld]
    float* ks = qs + AM_ROWS * ld;                       // [64][ld]
    float* vs = ks + AM_KEYS * ld;                       // [64][ld]
    float* ps = vs + AM_KEYS * ld;                       // [64 rows][68]: weights
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int head = blockIdx.x, g = head / (nh / nkv), z = blockIdx.z;
    int b, blk, place0;
    if (!mass_find_block(seq_start, n_seqs, gridDim.y - 1 - blockIdx.y, AM_ROWS, b, blk, place0)) return;
    const int t0 = seq_start[b] + blk * AM_ROWS;
    const int rows = min(AM_ROWS, seq_start[b + 1] - t0);
    const int p0 = seq_pos0[b] + blk * AM_ROWS, p_last = p0 + rows - 1, oldest = hb_oldest_visible(p0, window, 0);
    int page0;
    const int n_all = key_tiles_of(p0, p_last, window, HB_PAGE_TOKENS, page0), S = shares_of(sh, n_all);
    if (z >= S) return;
    const int page1 = page0 + (int)((long long)n_all * (z + 1) / S);
    page0 += (int)((long long)n_all * z / S);
    const int* pt = page_table + (size_t)b * pt_width;
    AmTile<T, NC> tile;
    // rows of the cache that page pi holds of this sequence, and where; a page that is missing counts as no keys
    auto page_of = [&](int pi, size_t& row0) -> int {
        const int page = pi < pt_width ? pt[pi] : -1;
        const bool held = page >= 0 && page < n_pages;
        row0 = ((size_t)(held ? page : 0) * nkv + g) * HB_PAGE_TOKENS;
        return held ? min(HB_PAGE_TOKENS, p_last + 1 - pi * HB_PAGE_TOKENS) : 0;
    };
    tile.load(q + (size_t)t0 * q_stride + (size_t)head * hd, q_stride, hd, rows, vec_q, tid);
    tile.store(qs, hd, ld, tid);
    size_t row0;
    int held = page_of(page0, row0);
    tile.load(kc + row0 * hd, hd, hd, held, vec_kv, tid);
    tile.store(ks, hd, ld, tid);
    float m[4], l[4], acc[4][NC];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++) acc[i][c] = 0.0f;
    }
    for (int pi = page0; pi < page1; pi++) {
        if (held == 0 && tid == 0) hb_note(status, HB_STATUS_PAGE, 1 + b);
        __syncthreads();                                 // the keys are there; values and weights of the page before are used up
        // (values in front of the oldest key that the first row sees may be anything, and 0 * NaN is NaN)
        tile.load(vc + row0 * hd, hd, hd, held, vec_kv, tid, oldest - pi * HB_PAGE_TOKENS);
        float s[4][4];
        am_scores(s, qs, ks, ld, tx, ty);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = ty + 16 * i, p = p0 + r, lo = hb_oldest_visible(p, window, 0);
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int key = pi * HB_PAGE_TOKENS + tx + 16 * j;
                s[i][j] = (held > 0 && r < rows && key >= lo && key <= p) ? s[i][j] * scale_log2e : -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float m_new = fmaxf(m[i], top), m_safe = m_new == -INFINITY ? 0.0f : m_new;
            const float corr = exp2f(m[i] - m_safe);
            m[i] = m_new;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float w = exp2f(s[i][j] - m_safe);
                ps[r * 68 + tx + 16 * j] = w;
                sum += w;
            }
            l[i] = l[i] * corr + sum;                     // this thread's columns only
#pragma unroll
            for (int c = 0; c < NC; c++) acc[i][c] *= corr;
        }
        tile.store(vs, hd, ld, tid);
        __syncthreads();                                 // values and weights are there; the keys are used up
        if (pi + 1 < page1) {
            held = page_of(pi + 1, row0);
            tile.load(kc + row0 * hd, hd, hd, held, vec_kv, tid);
        }
        for (int e = 0; e < AM_KEYS; e += 4) {
            float4 w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = *reinterpret_cast<const float4*>(ps + (ty + 16 * i) * 68 + e);
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const int d = tx + 16 * c;
                if (d >= hd) break;
                const float v0 = vs[e * ld + d], v1 = vs[(e + 1) * ld + d], v2 = vs[(e + 2) * ld + d], v3 = vs[(e + 3) * ld + d];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    acc[i][c] = fmaf(w[i].x, v0, acc[i][c]);
                    acc[i][c] = fmaf(w[i].y, v1, acc[i][c]);
                    acc[i][c] = fmaf(w[i].z, v2, acc[i][c]);
                    acc[i][c] = fmaf(w[i].w, v3, acc[i][c]);
                }
            }
        }
        if (pi + 1 < page1) tile.store(ks, hd, ld, tid);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = ty + 16 * i;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
        if (r >= rows) continue;
        if (S > 1) {
            const size_t at = ((size_t)z * nh + head) * n_tokens + t0 + r;
#pragma unroll
            for (int c = 0; c < NC; c++)
                if (tx + 16 * c < hd) sh.o[at * hd + tx + 16 * c] = acc[i][c];
            if (tx == 0) {
                sh.ml[at * 2] = m[i];
                sh.ml[at * 2 + 1] = l[i];
            }
            continue;
        }
        const float inv = l[i] > 0.0f ? 1.0f / l[i] : 0.0f;
        T* o = out + (size_t)(t0 + r) * out_stride + (size_t)head * hd;
#pragma unroll
        for (int c = 0; c < NC; c++)
            if (tx + 16 * c < hd) o[tx + 16 * c] = from_f32<T>(acc[i][c] * inv);
        if (tx == 0) lse[(size_t)head * n_tokens + t0 + r] = l[i] > 0.0f ? m[i] + log2f(l[i]) : INFINITY;
    }
}

// out = sum_z o_z 2^(m_z - M) / sum_z l_z 2^(m_z - M), lse = M + log2 of that sum, for the rows whose block has several shares; a
// warp per (token, head)
template <typename T>
__global__ void __launch_bounds__(256)
shares_join_kernel(Shares sh, T* __restrict__ out, long long out_stride, float* __restrict__ lse, long long lse_ld, int rounded,
                   const int* __restrict__ seq_start, const int* __restrict__ seq_pos0, int span, int keys, int window, int n_tokens, int n_seqs,
                   int nh, int hd) {
    __shared__ float ws[8][32];
    pdl_trigger();
    pdl_wait();
    seq_start = pdl_fresh(seq_start);
    seq_pos0 = pdl_fresh(seq_pos0);
    const int lane = threadIdx.x & 31;
    int b, i, place0;
    if (!mass_find(n_seqs, blockIdx.x,
                   [&](int s) {
                       const int n = seq_start[s + 1] - seq_start[s];
                       return shares_may_cut(sh, seq_pos0[s] + n, span, window, keys) ? n : 0;
                   },
                   [&](int s) { return mass_round128(seq_start[s + 1] - seq_start[s]); }, b, i, place0))
        return;
    const int t = seq_start[b] + i, place = rounded ? place0 + i : t;
    const int n_new = seq_start[b + 1] - seq_start[b], row0 = i / span * span;
    int tile0;
    const int S = shares_of(sh, key_tiles_of(seq_pos0[b] + row0, seq_pos0[b] + min(row0 + span, n_new) - 1, window, keys, tile0));
    if (S == 1) return;
    float* mine = ws[threadIdx.x >> 5];
    const int head = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (head < nh) {
        const size_t at = (size_t)head * n_tokens + t, step = (size_t)nh * n_tokens;
        float2 ml = make_float2(-INFINITY, 0.0f);              // of share `lane` (at most 32)
        if (lane < S) ml = __ldcg(reinterpret_cast<const float2*>(sh.ml) + at + lane * step);
        const float M = warp_max(ml.x);
        const float w = ml.x != -INFINITY ? exp2f(ml.x - M) : 0.0f;
        const float L = warp_sum(ml.y * w), inv = L > 0.0f ? 1.0f / L : 0.0f;
        mine[lane] = w;
        __syncwarp();
        for (int d = lane; d < hd; d += 32) {
            float acc = 0.0f;
#pragma unroll 4
            for (int z = 0; z < S; z++) acc = fmaf(__ldcg(sh.o + (at + z * step) * hd + d), mine[z], acc);
            out[(size_t)t * out_stride + (size_t)head * hd + d] = from_f32<T>(acc * inv);
        }
        if (lane == 0) {
            const float total = L > 0.0f ? M + log2f(L) : INFINITY;
            lse[head * lse_ld + place] = rounded ? -total : total;
        }
    }
}

int shares_join(Shares sh, int join_tokens, int dtype, void* out, long long out_stride, float* lse, long long lse_ld, int rounded,
                const int* seq_start, const int* seq_pos0, int span, int keys, int window, int n_tokens, int n_seqs, int nh, int hd, cudaStream_t s) {
    if (join_tokens == 0) return 0;
    const dim3 grid(join_tokens, (nh + 7) / 8);
    cudaError_t e = dtype == HB_BF16 ? hb_launch(shares_join_kernel<bf16>, grid, dim3(256), 0, s, sh, (bf16*)out, out_stride, lse, lse_ld, rounded,
                                                 seq_start, seq_pos0, span, keys, window, n_tokens, n_seqs, nh, hd)
                                     : hb_launch(shares_join_kernel<float>, grid, dim3(256), 0, s, sh, (float*)out, out_stride, lse, lse_ld, rounded,
                                                 seq_start, seq_pos0, span, keys, window, n_tokens, n_seqs, nh, hd);
    if (e != cudaSuccess) return hb_fail("attention_mass: launch failed: %s", cudaGetErrorString(e));
    return hb_check_launch("attention_mass (join of the shares)");
}

// A block per (64 keys = a page, kv head, share of the work): the scores of these keys with the queries that see them, in tiles
// of 64 queries of one head.
template <typename T, int NC>
__global__ void __launch_bounds__(AM_THREADS)
mass_rows_kernel(const T* __restrict__ q, long long q_stride, const T* __restrict__ kc, const int* __restrict__ page_table, int pt_width,
                 const int* __restrict__ seq_start, const int* __restrict__ seq_pos0, const float* __restrict__ lse, MassOut mo, int n_tokens,
                 int n_seqs, int nh, int nkv, int hd, float scale_log2e, int window, int n_pages, int vec_q, int vec_kv, int* status) {
    extern __shared__ __align__(16) float am_smem[];
    pdl_trigger();
    pdl_wait();
    mass_fresh(page_table, seq_start, seq_pos0);
    q = pdl_fresh(q);
    kc = pdl_fresh(kc);
    lse = pdl_fresh(lse);
    const int ld = am_ld(hd);
    float* ks = am_smem;                                 // [64][ld]
    float* qs = ks + AM_KEYS * ld;                       // [64][ld]
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int g = blockIdx.y, G = nh / nkv, S = gridDim.z, z = blockIdx.z;
    int b, pi, place0;
    if (!mass_find_keys(seq_start, seq_pos0, n_seqs, blockIdx.x, AM_KEYS, b, pi, place0)) return;
    const int page = pi < pt_width ? page_table[(size_t)b * pt_width + pi] : -1;
    const bool held = page >= 0 && page < n_pages;
    const int t_begin = seq_start[b], n_new = seq_start[b + 1] - t_begin, pos0 = seq_pos0[b];
    // the new tokens [n0, n1) that see some key of the page, cut at multiples of 64 from the first
    int n0, n1;
    mass_queries(pi * HB_PAGE_TOKENS, HB_PAGE_TOKENS, pos0, n_new, window, n0, n1);
    const int blocks = (n1 - n0 + AM_ROWS - 1) / AM_ROWS, items = blocks * G;
    if (!held && items > 0) {
        if (tid == 0) hb_note(status, HB_STATUS_PAGE, 1 + b);
    }
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};             // of keys tx + 16 j, over rows ty + 16 i
    if (held && items > 0) {
        const size_t row0 = ((size_t)page * nkv + g) * HB_PAGE_TOKENS;
        AmTile<T, NC> tile;
        tile.load(kc + row0 * hd, hd, hd, min(HB_PAGE_TOKENS, pos0 + n_new - pi * HB_PAGE_TOKENS), vec_kv, tid);
        tile.store(ks, hd, ld, tid);
        const int it1 = (int)((long long)items * (z + 1) / S);
        auto load = [&](int it) {
            const int q0 = n0 + (it % blocks) * AM_ROWS;
            tile.load(q + (size_t)(t_begin + q0) * q_stride + (size_t)(g * G + it / blocks) * hd, q_stride, hd, min(AM_ROWS, n1 - q0), vec_q, tid);
        };
        int it = (int)((long long)items * z / S);
        if (it < it1) load(it);
        for (; it < it1; it++) {
            const int head = g * G + it / blocks, q0 = n0 + (it % blocks) * AM_ROWS;
            __syncthreads();
            tile.store(qs, hd, ld, tid);
            __syncthreads();
            if (it + 1 < it1) load(it + 1);
            float s[4][4];
            am_scores(s, qs, ks, ld, tx, ty);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int t = q0 + ty + 16 * i, p = pos0 + t, lo = hb_oldest_visible(p, window, 0);
                if (t >= n1) continue;
                const float total = lse[(size_t)head * n_tokens + t_begin + t];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int key = pi * HB_PAGE_TOKENS + tx + 16 * j;
                    if (key >= lo && key <= p) sum[j] += exp2f(fmaf(s[i][j], scale_log2e, -total));
                }
            }
        }
    }
    __syncthreads();
    float* part = am_smem;                               // [16][64], over the keys: the sums of the 16 rows of threads
#pragma unroll
    for (int j = 0; j < 4; j++) part[ty * AM_KEYS + tx + 16 * j] = sum[j];
    __syncthreads();
    if (tid < AM_KEYS) {
        float s = 0.0f;
        for (int i = 0; i < 16; i++) s += part[i * AM_KEYS + tid];
        mass_store(mo, s, b, g, pi * HB_PAGE_TOKENS + tid, page, nkv, n_pages, pos0, n_new, z, S, blockIdx.x * AM_KEYS + tid, gridDim.x * AM_KEYS);
    }
}

// The shares of a key's sum, added in their order.  One thread per (key of a tile, kv head); `tile` keys per tile of the
// kernel that wrote the shares.
__global__ void mass_join_kernel(const int* __restrict__ page_table, int pt_width, const int* __restrict__ seq_start,
                                 const int* __restrict__ seq_pos0, MassOut mo, int n_seqs, int nkv, int n_pages, int tile, int S) {
    pdl_trigger();
    pdl_wait();
    mass_fresh(page_table, seq_start, seq_pos0);
    const int g = blockIdx.y, tid = threadIdx.x;
    int b, kt, place0;
    if (!mass_find_keys(seq_start, seq_pos0, n_seqs, blockIdx.x, tile, b, kt, place0)) return;
    const int key = kt * tile + tid, pi = key / HB_PAGE_TOKENS;
    const int page = pi < pt_width ? page_table[(size_t)b * pt_width + pi] : -1;
    const size_t place = (size_t)blockIdx.x * tile + tid, places = (size_t)gridDim.x * tile;
    float s = 0.0f;
    for (int z = 0; z < S; z++) s += __ldcg(mo.parts + ((size_t)z * nkv + g) * places + place);
    mass_write(mo, s, g, key, page, nkv, n_pages, seq_pos0[b], seq_start[b + 1] - seq_start[b]);
}

int mass_join(const int* page_table, int pt_width, const int* seq_start, const int* seq_pos0, MassOut mo, int n_seqs, int nkv, int n_pages, int tile,
              int key_tiles, int splits, cudaStream_t s) {
    cudaError_t e = hb_launch(mass_join_kernel, dim3(key_tiles, nkv), dim3(tile), 0, s, page_table, pt_width, seq_start, seq_pos0, mo, n_seqs, nkv,
                              n_pages, tile, splits);
    if (e != cudaSuccess) return hb_fail("attention_mass: launch failed: %s", cudaGetErrorString(e));
    return hb_check_launch("attention_mass (join)");
}

template <typename F>
static int am_reserve(F* kernel, int bytes, bool (&done)[HB_MAX_DEVICES]) {
    bool& set = done[hb_device_slot()];
    if (set) return 0;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return hb_fail("attention_mass: cannot reserve %d bytes of shared memory: %s", bytes, cudaGetErrorString(e));
    set = true;
    return 0;
}

#define AM_SMEM_ROWS(hd) ((3 * 64 * am_ld(hd) + 64 * 68) * 4)
#define AM_SMEM_MASS(hd) (2 * 64 * am_ld(hd) * 4)

template <typename T, int NC>
static int launch_rows(const void* q, long long q_stride, const void* kc, const void* vc, const int* page_table, int pt_width, const int* seq_start,
                       const int* seq_pos0, void* out, long long out_stride, float* lse, Shares sh, int max_shares, int join_tokens, MassOut mo,
                       int splits, int n_tokens, int n_seqs, int q_blocks, int key_tiles, int nh, int nkv, int hd, float scale, int window,
                       int n_pages, int* status, cudaStream_t s) {
    static_assert(AM_SMEM_ROWS(256) <= 227 * 1024, "attention tiles do not fit shared memory");
    static bool done[HB_MAX_DEVICES] = {}, done_mass[HB_MAX_DEVICES] = {};
    if (am_reserve(attention_rows_kernel<T, NC>, AM_SMEM_ROWS(16 * NC), done)) return 1;
    if (am_reserve(mass_rows_kernel<T, NC>, AM_SMEM_MASS(16 * NC), done_mass)) return 1;
    const uintptr_t four = 4 * sizeof(T);                      // four elements at a time where rows and heads begin at a multiple of that
    const int vec_kv = hd % 4 == 0 && (((uintptr_t)kc | (uintptr_t)vc) & (four - 1)) == 0;
    const int vec_q = hd % 4 == 0 && q_stride % 4 == 0 && ((uintptr_t)q & (four - 1)) == 0;
    cudaError_t e = hb_launch(attention_rows_kernel<T, NC>, dim3(nh, q_blocks, max_shares), dim3(AM_THREADS), AM_SMEM_ROWS(hd), s, (const T*)q,
                              q_stride, (const T*)kc, (const T*)vc, page_table, pt_width, seq_start, seq_pos0, (T*)out, out_stride, lse, sh,
                              n_tokens, n_seqs, nh, nkv, hd, scale * MASS_LOG2E, window, n_pages, vec_q, vec_kv, status);
    if (e != cudaSuccess) return hb_fail("attention_mass: launch failed: %s", cudaGetErrorString(e));
    if (hb_check_launch("attention_mass (rows)")) return 1;
    if (max_shares > 1 && shares_join(sh, join_tokens, sizeof(T) == 4 ? HB_F32 : HB_BF16, out, out_stride, lse, n_tokens, 0, seq_start, seq_pos0,
                                      AM_ROWS,
                                      HB_PAGE_TOKENS, window, n_tokens, n_seqs, nh, hd, s))
        return 1;
    e = hb_launch(mass_rows_kernel<T, NC>, dim3(key_tiles, nkv, splits), dim3(AM_THREADS), AM_SMEM_MASS(hd), s, (const T*)q, q_stride, (const T*)kc,
                  page_table, pt_width, seq_start, seq_pos0, (const float*)lse, mo, n_tokens, n_seqs, nh, nkv, hd, scale * MASS_LOG2E, window,
                  n_pages, vec_q, vec_kv, status);
    if (e != cudaSuccess) return hb_fail("attention_mass: launch failed: %s", cudaGetErrorString(e));
    if (hb_check_launch("attention_mass (weights)")) return 1;
    return splits > 1 ? mass_join(page_table, pt_width, seq_start, seq_pos0, mo, n_seqs, nkv, n_pages, AM_KEYS, key_tiles, splits, s) : 0;
}

// Steps of many tokens (HbMassMany in api.h): blocks of 64 queries, tiles of 64 keys.
extern "C" int hb_attention_mass(const HbMassMany* a, int fields, float scale) {
    HB_REQUIRE(fields * sizeof(long long) == sizeof(*a), "attention_mass: %d fields given", fields);
    const int n_tokens = (int)a->n_tokens, n_seqs = (int)a->n_seqs, n_heads = (int)a->n_heads, n_kv_heads = (int)a->n_kv_heads, hd = (int)a->head_dim;
    const int splits = (int)a->splits, max_shares = (int)a->max_shares, n_pages = (int)a->n_pages, pt_width = (int)a->pt_width, dtype = (int)a->dtype;
    const int q_blocks = (int)a->q_blocks, key_tiles = (int)a->key_tiles, share_tiles = (int)a->share_tiles, join_tokens = (int)a->join_tokens;
    const int window = (int)a->window;
    if (n_seqs == 0 || n_tokens == 0) return 0;
    HB_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && hd > 0 && hd <= 256 && n_pages > 0 && pt_width > 0,
               "attention_mass: %d heads over %d kv heads of size %d are not built (sizes up to 256)", n_heads, n_kv_heads, hd);
    HB_REQUIRE(n_kv_heads <= 65535 && q_blocks <= 65535 && key_tiles > 0 && splits >= 1 && splits <= 65535 && (splits == 1 || a->parts != nullptr) &&
                   max_shares >= 1 && max_shares <= 32 && share_tiles >= 1 && (max_shares == 1 || a->chunk_parts != nullptr),
               "attention_mass: the step is too large for one launch");
    HB_REQUIRE(a->lse != nullptr && a->mass != nullptr, "attention_mass: missing buffers");
    HB_REQUIRE(dtype == HB_F32 || dtype == HB_BF16, "attention_mass: unsupported dtype %d", dtype);
    MassOut mo = {a->before, a->mass, a->parts};
    // (maximum, sum) pairs in front: 8-byte aligned whatever the head size; one share: no block is cut, whatever it sees
    const Shares sh = {a->chunk_parts == nullptr ? nullptr : a->chunk_parts + (size_t)max_shares * n_heads * n_tokens * 2, a->chunk_parts,
                       max_shares == 1 ? 0x3fffffff : share_tiles};
    cudaStream_t s = (cudaStream_t)a->stream;
#define HB_AM_LAUNCH(T, NC)                                                                                                                       \
    launch_rows<T, NC>(a->q, a->q_stride, a->k_cache, a->v_cache, a->page_table, pt_width, a->seq_start, a->seq_pos0, a->out, a->out_stride, a->lse, sh, \
                       max_shares, join_tokens, mo, splits, n_tokens, n_seqs, q_blocks, key_tiles, n_heads, n_kv_heads, hd, scale, window, n_pages,   \
                       a->status, s)
    if (dtype == HB_F32) return hd <= 64 ? HB_AM_LAUNCH(float, 4) : hd <= 128 ? HB_AM_LAUNCH(float, 8) : HB_AM_LAUNCH(float, 16);
    return hd <= 64 ? HB_AM_LAUNCH(bf16, 4) : hd <= 128 ? HB_AM_LAUNCH(bf16, 8) : HB_AM_LAUNCH(bf16, 16);
#undef HB_AM_LAUNCH
}

// -------------------------------------------------------------------------------------------- few tokens, every head size
// A block per (share of the pages, kv head, eight (token, head) pairs of a sequence's new tokens and the kv head's group).  Keys and values
// stream through shared memory in tiles of 32 rows, cp.async stages, as they are stored.  Scores: a warp per pair, a lane per
// key, so that the softmax is a warp's; values: a thread per two columns (and share of the tile's keys), all eight pairs at once.
// Rows in shared memory lie an odd number of 16-byte units apart: the lanes' 16-byte reads of 32 rows then fall into different banks.
// Bound by the FP32 pipe or by memory: 32 keys of head size 152 take about 900 clocks of instructions and 20 KB.  (Keys and values
// read where they are used, a page at a time, took 404 us for five sequences of 8000 to 14000 rows, 16 heads of size
// 152, instead of 113, with 16 shares each.)
#define AF_THREADS 256
#define AF_PAIRS 8
#define AF_KEYS 32

static __host__ __device__ constexpr int af_row_bytes(int hd, int es) {
    const int units = (hd * es + 15) / 16;
    return (units | 1) * 16;
}
static __host__ __device__ constexpr int af_smem(int hd, int es, int stages) {
    return stages * 2 * AF_KEYS * af_row_bytes(hd, es) + AF_PAIRS * ((hd + 7) & ~7) * 4;
}
// three stages where two blocks of them fit an SM, else two (32-bit, head size 176: a second block hides more than a third stage)
static __host__ __device__ constexpr int af_stages(int hd, int es) { return 2 * (af_smem(hd, es, 3) + 3 * 1024) <= 227 * 1024 ? 3 : 2; }

// eight (bfloat16) or four (float32) elements of a 16-byte unit
__device__ __forceinline__ void unpack16(const uint4& u, float (&x)[8], const bf16*) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack16(const uint4& u, float (&x)[4], const float*) {
    x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ float2 two_columns(const uint8_t* p, const float*) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 two_columns(const uint8_t* p, const bf16*) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

template <typename T, int AF_STAGES>
__global__ void __launch_bounds__(AF_THREADS, 2)
few_rows_kernel(const T* __restrict__ q, long long q_stride, const T* __restrict__ kc, const T* __restrict__ vc, const int* __restrict__ page_table,
                int pt_width, const int* __restrict__ seq_start, const int* __restrict__ seq_pos0, float* __restrict__ part_o,
                float* __restrict__ part_ml, float* __restrict__ scores, long long score_ld, int n_seqs, int nh, int nkv, int hd, int share_pages,
                float scale_log2e, int window, int n_pages, int vec, MassWhole whole, int seq0, int* status) {
    extern __shared__ __align__(16) uint8_t af_raw[];
    __shared__ float4 w8[AF_KEYS][AF_PAIRS / 4];         // a tile's weights
    __shared__ float corr[AF_PAIRS], stat[2][AF_PAIRS];
    constexpr int UNIT = 16 / sizeof(T);
    pdl_trigger();
    pdl_wait();
    mass_fresh(page_table, seq_start, seq_pos0);
    q = pdl_fresh(q);
    kc = pdl_fresh(kc);
    vc = pdl_fresh(vc);
    const int G = nh / nkv, S = gridDim.x, z = blockIdx.x, g = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row_bytes = af_row_bytes(hd, sizeof(T)), hd8 = (hd + 7) & ~7;
    uint8_t* tiles = af_raw;                             // [stages][keys, values][32][row_bytes]
    float* qs = reinterpret_cast<float*>(af_raw + AF_STAGES * 2 * AF_KEYS * row_bytes);        // [8][hd8]
    int b, blk, unused;
    if (!mass_find(n_seqs, blockIdx.z, [&](int i) { return ((seq_start[i + 1] - seq_start[i]) * G + AF_PAIRS - 1) / AF_PAIRS; },
                   [](int) { return 0; },
                   b, blk, unused))
        return;
    const int t0 = seq_start[b], n_new = seq_start[b + 1] - t0, pos0 = seq_pos0[b];
    const int pair0 = blk * AF_PAIRS, pairs = min(AF_PAIRS, n_new * G - pair0);          // pair i is head i % G of token i / G
    const int p_first = pos0 + pair0 / G, p_last = pos0 + (pair0 + pairs - 1) / G;
    const int* pt = page_table + (size_t)b * pt_width;
    const int width = (int)min((long long)pt_width, score_ld / HB_PAGE_TOKENS);          // no score is written behind its pair's
    const int oldest = hb_oldest_visible(p_first, window, 0);
    int page0, page1;
    mass_share(oldest / HB_PAGE_TOKENS, min(p_last / HB_PAGE_TOKENS + 1, width), z, S, share_pages, page0, page1);
    if (z == 0 && tid == 0 && p_last >= width * HB_PAGE_TOKENS) hb_note(status, HB_STATUS_PAGE, 1 + seq0 + b);
    auto at_of = [&](int r) -> size_t { return (size_t)(t0 + (pair0 + r) / G) * nh + g * G + (pair0 + r) % G; };
    if (page0 >= page1 && whole.out == nullptr) {        // a share without keys
        if (tid < pairs) {
            part_ml[(at_of(tid) * S + z) * 2] = -INFINITY;
            part_ml[(at_of(tid) * S + z) * 2 + 1] = 0.0f;
        }
        return;
    }
    // what no copy fills (the columns behind hd) is read times zero
    for (int i = tid; i < AF_STAGES * 2 * AF_KEYS * row_bytes / 16; i += AF_THREADS) reinterpret_cast<uint4*>(tiles)[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int i = tid; i < AF_PAIRS * hd8; i += AF_THREADS) {
        const int r = i / hd8, d = i - r * hd8;
        qs[i] = r < pairs && d < hd ? to_f32(q[(size_t)(t0 + (pair0 + r) / G) * q_stride + (size_t)(g * G + (pair0 + r) % G) * hd + d]) : 0.0f;
    }
    __syncthreads();
    const int n_tiles = (page1 - page0) * (HB_PAGE_TOKENS / AF_KEYS);
    bool bad = false;
    auto load_tile = [&](int it) {
        if (it < n_tiles) {
            const int key0 = page0 * HB_PAGE_TOKENS + it * AF_KEYS;
            int page = pt[key0 / HB_PAGE_TOKENS];
            const bool held = page >= 0 && page < n_pages;
            if (!held) {
                bad = true;
                page = 0;                                // never read outside the cache; its keys count as not there
            }
            const size_t row0 = ((size_t)page * nkv + g) * HB_PAGE_TOKENS + (key0 & (HB_PAGE_TOKENS - 1));
            uint8_t* dst = tiles + (size_t)(it % AF_STAGES) * 2 * AF_KEYS * row_bytes;
            if (vec) {
                const int units = hd / UNIT;             // whole, and aligned
                for (int i = tid; i < 2 * AF_KEYS * units; i += AF_THREADS) {
                    const int r = i / units, u = i - r * units, key = r & (AF_KEYS - 1);
                    const bool there = held && key0 + key >= oldest && key0 + key <= p_last;
                    const T* src = (r < AF_KEYS ? kc : vc) + (row0 + key) * hd + u * UNIT;
                    cp_async_16_or_zero((uint32_t)__cvta_generic_to_shared(dst + r * row_bytes + u * 16), src, there);
                }
            } else {
                for (int i = tid; i < 2 * AF_KEYS * hd; i += AF_THREADS) {
                    const int r = i / hd, d = i - r * hd, key = r & (AF_KEYS - 1);
                    const bool there = held && key0 + key >= oldest && key0 + key <= p_last;
                    reinterpret_cast<T*>(dst + r * row_bytes)[d] = there ? ((r < AF_KEYS ? kc : vc) + (row0 + key) * hd)[d] : from_f32<T>(0.0f);
                }
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < AF_STAGES - 1; i++) load_tile(i);
    const int pos = pos0 + (pair0 + min(warp, pairs - 1)) / G, lo = hb_oldest_visible(pos, window, 0);      // of this warp's pair
    float* my_scores = scores + at_of(min(warp, pairs - 1)) * score_ld;
    float m = -INFINITY, l = 0.0f;                        // in every lane
    const int columns = (hd + 1) / 2, slices = AF_THREADS / columns, slice = tid / columns, column = (tid - slice * columns) * 2;
    float2 acc[AF_PAIRS];
#pragma unroll
    for (int r = 0; r < AF_PAIRS; r++) acc[r] = make_float2(0.0f, 0.0f);
    for (int it = 0; it < n_tiles; it++) {
        cp_async_wait<AF_STAGES - 2>();
        __syncthreads();
        load_tile(it + AF_STAGES - 1);
        const uint8_t* kt = tiles + (size_t)(it % AF_STAGES) * 2 * AF_KEYS * row_bytes;
        const uint8_t* vt = kt + AF_KEYS * row_bytes;
        const int key0 = page0 * HB_PAGE_TOKENS + it * AF_KEYS, key = key0 + lane;
        if (warp < pairs) {
            const uint4* kr = reinterpret_cast<const uint4*>(kt + lane * row_bytes);
            const float4* qr = reinterpret_cast<const float4*>(qs + warp * hd8);
            float dot[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
            for (int u = 0; u < (hd + UNIT - 1) / UNIT; u++) {
                float x[UNIT];
                unpack16(kr[u], x, (const T*)nullptr);
#pragma unroll
                for (int c = 0; c < UNIT / 4; c++) {
                    const float4 y = qr[u * (UNIT / 4) + c];
                    dot[0] = fmaf(x[4 * c], y.x, dot[0]);
                    dot[1] = fmaf(x[4 * c + 1], y.y, dot[1]);
                    dot[2] = fmaf(x[4 * c + 2], y.z, dot[2]);
                    dot[3] = fmaf(x[4 * c + 3], y.w, dot[3]);
                }
            }
            // a page that is missing: its keys are not there
            const int page = pt[key0 / HB_PAGE_TOKENS];
            const bool seen = key >= lo && key <= pos && page >= 0 && page < n_pages;
            const float s = seen ? ((dot[0] + dot[1]) + (dot[2] + dot[3])) * scale_log2e : -INFINITY;
            my_scores[key] = s;
            const float m_new = fmaxf(m, warp_max(s)), m_safe = m_new == -INFINITY ? 0.0f : m_new;
            const float f = exp2f(m - m_safe), w = exp2f(s - m_safe);
            m = m_new;
            l = l * f + warp_sum(w);
            reinterpret_cast<float*>(&w8[lane][0])[warp] = w;
            if (lane == 0) corr[warp] = f;
        } else {
            reinterpret_cast<float*>(&w8[lane][0])[warp] = 0.0f;
            if (lane == 0) corr[warp] = 1.0f;
        }
        __syncthreads();
        if (slice < slices) {
#pragma unroll
            for (int r = 0; r < AF_PAIRS; r++) {
                acc[r].x *= corr[r];
                acc[r].y *= corr[r];
            }
#pragma unroll 4
            for (int e = slice; e < AF_KEYS; e += slices) {
                const float2 x = two_columns(vt + e * row_bytes + column * sizeof(T), (const T*)nullptr);
                const float4 wa = w8[e][0], wb = w8[e][1];
                const float w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
                for (int r = 0; r < AF_PAIRS; r++) {
                    acc[r].x = fmaf(w[r], x.x, acc[r].x);
                    acc[r].y = fmaf(w[r], x.y, acc[r].y);
                }
            }
        }
    }
    cp_async_wait<0>();
    if (bad && tid == 0) hb_note(status, HB_STATUS_PAGE, 1 + seq0 + b);
    // join the slices: one after another adds to the first's sums, in shared memory over the tiles
    float* so = reinterpret_cast<float*>(af_raw);         // [8][2 columns]
    for (int c = 0; c < slices; c++) {
        __syncthreads();
        if (slice == c) {
#pragma unroll
            for (int r = 0; r < AF_PAIRS; r++) {
                float2* o = reinterpret_cast<float2*>(so + r * 2 * columns + column);
                const float2 old = c > 0 ? *o : make_float2(0.0f, 0.0f);
                *o = make_float2(old.x + acc[r].x, old.y + acc[r].y);
            }
        }
    }
    if (lane == 0) {
        stat[0][warp] = m;
        stat[1][warp] = l;
    }
    __syncthreads();
    if (whole.out != nullptr) {
        for (int i = tid; i < pairs * hd; i += AF_THREADS) {
            const int r = i / hd, d = i - r * hd;
            const float L = stat[1][r];
            ((T*)whole.out)[(size_t)(t0 + r / G) * whole.out_stride + (size_t)(g * G + r % G) * hd + d] =
                from_f32<T>(so[r * 2 * columns + d] * (L > 0.0f ? 1.0f / L : 0.0f));
        }
        if (tid < pairs) corr[tid] = stat[1][tid] > 0.0f ? stat[0][tid] + log2f(stat[1][tid]) : INFINITY;      // now the pairs' log-sums
        __syncthreads();
        mass_whole(whole.mo, scores, score_ld, corr, n_new, G, g, t0, nh, nkv, pos0, window, pt, pt_width, n_pages);
        return;
    }
    for (int i = tid; i < pairs * hd; i += AF_THREADS) {
        const int r = i / hd, d = i - r * hd;
        const size_t base = at_of(r) * S + z;
        part_o[base * hd + d] = so[r * 2 * columns + d];
        if (d == 0) {
            part_ml[base * 2] = stat[0][r];
            part_ml[base * 2 + 1] = stat[1][r];
        }
    }
}

// maximum and sum of a (token, head) over its S shares; every lane of the warp gets them
__device__ __forceinline__ void join_stats(const float* __restrict__ part_ml, size_t base, int S, int lane, float& M, float& L) {
    M = -INFINITY;
    L = 0.0f;
    for (int z = lane; z < S; z += 32) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_ml) + base + z);
        const float m = fmaxf(M, ml.x);
        if (m != -INFINITY) L = L * exp2f(M - m) + ml.y * exp2f(ml.x - m);
        M = m;
    }
    const float top = warp_max(M);
    L = warp_sum(M != -INFINITY ? L * exp2f(M - top) : 0.0f);
    M = top;
}

// The second half of a step of few tokens.  grid: (tokens of a sequence + blocks of FF_KEYS keys, kv heads, sequences).  The first blocks
// join a token's partial outputs; a block of keys joins the log-sums of the sequence's tokens and heads from the shares' maxima
// and sums, then turns its keys' scores into weights, four keys a thread.  (With 256 keys to a block the log-sums' round trips took most of the time:
// 55 us for two sequences of 100000 and 65538 rows.)
#define FF_THREADS 256
#define FF_KEYS 1024

template <typename T>
__global__ void __launch_bounds__(FF_THREADS)
few_finish_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, const float* __restrict__ scores, long long score_ld,
                  const int* __restrict__ page_table, int pt_width, const int* __restrict__ seq_start, const int* __restrict__ seq_pos0,
                  T* __restrict__ out, long long out_stride, MassOut mo, int token_rows, int nh, int nkv, int hd, int S, int window, int n_pages,
                  int vec) {
    __shared__ float lse[MASS_FEW_PAIRS];
    pdl_trigger();
    pdl_wait();
    mass_fresh(page_table, seq_start, seq_pos0);
    part_o = pdl_fresh(part_o);
    part_ml = pdl_fresh(part_ml);
    scores = pdl_fresh(scores);
    const int g = blockIdx.y, b = blockIdx.z, G = nh / nkv, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int t0 = seq_start[b], n_new = seq_start[b + 1] - t0, pos0 = seq_pos0[b];
    if ((int)blockIdx.x < token_rows) {
        const int i = blockIdx.x;
        if (i >= n_new) return;
        const int t = t0 + i;
        for (int h = warp; h < G; h += FF_THREADS / 32) {
            const size_t base = ((size_t)t * nh + g * G + h) * S;
            float M, L;
            join_stats(part_ml, base, S, lane, M, L);
            const float inv = L > 0.0f ? 1.0f / L : 0.0f;
            // (four columns a lane, the loads of four shares in flight: asked for one share after another, 18 shares of two sequences of
            // 100000 and 65538 rows held the kernel up for 35 us instead of 12.5)
            for (int d0 = 0; d0 < hd; d0 += 128) {
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                auto shares = [&](int z0, auto count) {
                    constexpr int N = decltype(count)::value;
                    float mz[N], x[N][4];
#pragma unroll
                    for (int k = 0; k < N; k++) {
                        mz[k] = __ldcg(part_ml + (base + z0 + k) * 2);
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const int d = d0 + u * 32 + lane;
                            x[k][u] = d < hd ? __ldcg(part_o + (base + z0 + k) * hd + d) : 0.0f;
                        }
                    }
#pragma unroll
                    for (int k = 0; k < N; k++) {
                        const float w = mz[k] != -INFINITY ? exp2f(mz[k] - M) : 0.0f;
#pragma unroll
                        for (int u = 0; u < 4; u++)
                            if (w != 0.0f) acc[u] = fmaf(x[k][u], w, acc[u]);          // a share without keys has written no output
                    }
                };
                int z = 0;
                for (; z + 4 <= S; z += 4) shares(z, std::integral_constant<int, 4>());
                for (; z < S; z++) shares(z, std::integral_constant<int, 1>());
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int d = d0 + u * 32 + lane;
                    if (d < hd) out[(size_t)t * out_stride + (size_t)(g * G + h) * hd + d] = from_f32<T>(acc[u] * inv);
                }
            }
        }
        return;
    }
    if (n_new * G > MASS_FEW_PAIRS) return;                    // no step of few tokens: the host refuses it
    const int n = (int)min((long long)(pos0 + n_new), score_ld), key0 = ((int)blockIdx.x - token_rows) * FF_KEYS;
    if (key0 >= n) return;
    for (int i = warp; i < n_new * G; i += FF_THREADS / 32) {
        float M, L;
        join_stats(part_ml, ((size_t)(t0 + i / G) * nh + g * G + i % G) * S, S, lane, M, L);
        if (lane == 0) lse[i] = L > 0.0f ? M + log2f(L) : INFINITY;
    }
    __syncthreads();
    const int key = key0 + tid * 4, pi = key / HB_PAGE_TOKENS; // this thread's four keys, on one page
    if (key >= n) return;
    const int page = pi < pt_width ? page_table[(size_t)b * pt_width + pi] : -1;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < n_new; i++) {
        const int p = pos0 + i, lo = hb_oldest_visible(p, window, 0);
        if (key > p || key + 3 < lo) continue;
        const float* row = scores + ((size_t)(t0 + i) * nh + g * G) * score_ld + key;
#pragma unroll 4
        for (int h = 0; h < G; h++) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(row + h * score_ld));
            const float e = lse[i * G + h];
            s[0] += key >= lo ? exp2f(x.x - e) : 0.0f;
            s[1] += key + 1 >= lo && key + 1 <= p ? exp2f(x.y - e) : 0.0f;
            s[2] += key + 2 >= lo && key + 2 <= p ? exp2f(x.z - e) : 0.0f;
            s[3] += key + 3 >= lo && key + 3 <= p ? exp2f(x.w - e) : 0.0f;
        }
    }
    if (vec && key + 3 < pos0 && page >= 0 && page < n_pages) {
        const size_t at = ((size_t)page * nkv + g) * HB_PAGE_TOKENS + (key & (HB_PAGE_TOKENS - 1));
        const float4 old = mo.before != nullptr ? __ldcg(reinterpret_cast<const float4*>(mo.before + at)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        *reinterpret_cast<float4*>(mo.mass + at) = make_float4(old.x + s[0], old.y + s[1], old.z + s[2], old.w + s[3]);
    } else {
#pragma unroll
        for (int u = 0; u < 4; u++) mass_write(mo, s[u], g, key + u, page, nkv, n_pages, pos0, n_new);
    }
}

extern "C" int hb_attention_few_pairs(void) { return MASS_FEW_PAIRS; }

// Scratch floats of a step of few tokens: partial outputs, (maximum, sum) pairs, scores.  max_len: rows of the longest sequence.
extern "C" long long hb_attention_mass_few_floats(int n_tokens, int n_heads, int head_dim, int splits, int max_len) {
    return (long long)n_tokens * n_heads * ((long long)splits * (head_dim + 2) + mass_score_ld(max_len));
}

template <typename T>
static int launch_few(MassWhole whole, const void* q, long long q_stride, const void* kc, const void* vc, const int* page_table, int pt_width,
                      const int* seq_start, const int* seq_pos0, float* part_o, float* part_ml, float* scores, long long score_ld, int splits,
                      int share_pages, int blocks, int n_seqs, int nh, int nkv, int hd, float scale, int window, int n_pages, int seq0, int* status,
                      cudaStream_t s) {
    static_assert(af_smem(256, 4, 2) <= 227 * 1024, "tiles do not fit shared memory");
    static bool done[2][HB_MAX_DEVICES] = {};
    if (am_reserve(few_rows_kernel<T, 2>, af_smem(256, sizeof(T), 2), done[0]) || am_reserve(few_rows_kernel<T, 3>, 114 * 1024, done[1])) return 1;
    const int vec = hd % (16 / (int)sizeof(T)) == 0 && (((uintptr_t)kc | (uintptr_t)vc) & 15) == 0, stages = af_stages(hd, sizeof(T));
#define HB_AF_LAUNCH(ST)                                                                                                                           \
    hb_launch(few_rows_kernel<T, ST>, dim3(splits, nkv, blocks), dim3(AF_THREADS), af_smem(hd, sizeof(T), ST), s, (const T*)q, q_stride, (const T*)kc, \
              (const T*)vc, page_table, pt_width, seq_start, seq_pos0, part_o, part_ml, scores, score_ld, n_seqs, nh, nkv, hd, share_pages,            \
              scale * MASS_LOG2E, window, n_pages, vec, whole, seq0, status)
    cudaError_t e = stages == 3 ? HB_AF_LAUNCH(3) : HB_AF_LAUNCH(2);
#undef HB_AF_LAUNCH
    if (e != cudaSuccess) return hb_fail("attention_mass: launch failed: %s", cudaGetErrorString(e));
    return hb_check_launch("attention_mass (few tokens)");
}

template <typename T>
static int launch_finish(const float* part_o, const float* part_ml, const float* scores, long long score_ld, const int* page_table, int pt_width,
                         const int* seq_start, const int* seq_pos0, void* out, long long out_stride, MassOut mo, int max_len, int max_new, int n_seqs,
                         int nh, int nkv, int hd, int splits, int window, int n_pages, cudaStream_t s) {
    const int key_blocks = (max_len + FF_KEYS - 1) / FF_KEYS;
    const int vec = (((uintptr_t)mo.before | (uintptr_t)mo.mass) & 15) == 0;
    cudaError_t e = hb_launch(few_finish_kernel<T>, dim3(max_new + key_blocks, nkv, n_seqs), dim3(FF_THREADS), 0, s, part_o, part_ml, scores,
                              score_ld, page_table, pt_width, seq_start, seq_pos0, (T*)out, out_stride, mo, max_new, nh, nkv, hd, splits, window,
                              n_pages, vec);
    if (e != cudaSuccess) return hb_fail("attention_mass: launch failed: %s", cudaGetErrorString(e));
    return hb_check_launch("attention_mass (finish)");
}

// Pairs of a token and a head that a block of the kernel for every head size takes, and how many of its blocks an SM holds.
extern "C" int hb_attention_few_block_pairs(void) { return AF_PAIRS; }
extern "C" int hb_attention_few_blocks_per_sm(int head_dim, int dtype) {
    const int es = dtype == HB_F32 ? 4 : 2, bytes = af_smem(head_dim, es, af_stages(head_dim, es)) + 3 * 1024, n = 227 * 1024 / bytes;
    return n < 1 ? 1 : n > 2 ? 2 : n;                      // registers hold two
}

// Steps of few tokens (at most hb_attention_few_pairs() pairs of a sequence's tokens and a group's heads); HbMassFew in api.h.
extern "C" int hb_attention_mass_few(const HbMassFew* a, int fields, float scale) {
    HB_REQUIRE(fields * sizeof(long long) == sizeof(*a), "attention_mass: %d fields given", fields);
    const int n_tokens = (int)a->n_tokens, n_seqs = (int)a->n_seqs, n_heads = (int)a->n_heads, n_kv_heads = (int)a->n_kv_heads, hd = (int)a->head_dim;
    const int max_new = (int)a->max_new, max_len = (int)a->max_len, splits = (int)a->splits, window = (int)a->window, n_pages = (int)a->n_pages;
    const int pt_width = (int)a->pt_width, share_pages = (int)a->share_pages, blocks = (int)a->blocks, dtype = (int)a->dtype, seq0 = (int)a->first_seq;
    if (n_seqs == 0 || n_tokens == 0) return 0;
    const int* page_table = a->page_table + (size_t)seq0 * pt_width;
    const int *seq_start = a->seq_start + seq0, *seq_pos0 = a->seq_pos0 + seq0;
    HB_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && hd > 0 && hd <= 256 && n_pages > 0 && pt_width > 0,
               "attention_mass: %d heads over %d kv heads of size %d are not built (sizes up to 256)", n_heads, n_kv_heads, hd);
    HB_REQUIRE((long long)max_new * (n_heads / n_kv_heads) <= MASS_FEW_PAIRS, "attention_mass: %d tokens of %d heads are no step of few tokens",
               max_new, n_heads / n_kv_heads);
    HB_REQUIRE(n_tokens > 0 && seq0 >= 0 && a->first_token >= 0 && n_seqs <= 65535 && n_kv_heads <= 65535 && splits >= 1 && share_pages >= 1 &&
                   blocks >= 1 && blocks <= 65535 && max_len >= 1 &&
                   a->scratch != nullptr && a->mass != nullptr,
               "attention_mass: bad sizes");
    HB_REQUIRE(!a->whole || (splits == 1 && blocks == n_seqs), "attention_mass: a whole sequence to a block needs one share and one block each");
    HB_REQUIRE(dtype == HB_F32 || dtype == HB_BF16, "attention_mass: unsupported dtype %d", dtype);
    HB_REQUIRE(!a->tensor_cores || dtype == HB_BF16, "attention_mass: the tensor cores take bfloat16");
    HB_REQUIRE(((uintptr_t)a->scratch & 15) == 0, "attention_mass: scratch must be 16-byte aligned");
    const long long score_ld = mass_score_ld(max_len);
    // Scores, (maximum, sum) pairs and partial outputs of this call's (token, head) pairs.  The kernels number tokens from the step's
    // first, of which this call's are [first_token, first_token + n_tokens): each part's address is that of the step's first pair.
    const long long pairs = (long long)n_tokens * n_heads, in_front = a->first_token * n_heads;
    auto part = [&](long long begin, long long floats) { return (float*)((uintptr_t)a->scratch + 4 * (begin - in_front * floats)); };
    float *scores = part(0, score_ld), *part_ml = part(pairs * score_ld, 2LL * splits),
          *part_o = part(pairs * (score_ld + 2LL * splits), (long long)splits * hd);
    cudaStream_t s = (cudaStream_t)a->stream;
    MassOut mo = {a->before, a->mass, nullptr};
    const MassWhole whole = {a->whole ? a->out : nullptr, a->out_stride, mo};
#define HB_FEW_ARGS                                                                                                                              \
    whole, a->q, a->q_stride, a->k_cache, a->v_cache, page_table, pt_width, seq_start, seq_pos0, part_o, part_ml, scores, score_ld, splits, \
        share_pages, blocks
    int rc;
    if (a->tensor_cores)
        rc = attention_few_tc(HB_FEW_ARGS, max_new, n_seqs, n_heads, n_kv_heads, hd, scale, window, n_pages, seq0, a->status, s);
    else if (dtype == HB_F32)
        rc = launch_few<float>(HB_FEW_ARGS, n_seqs, n_heads, n_kv_heads, hd, scale, window, n_pages, seq0, a->status, s);
    else
        rc = launch_few<bf16>(HB_FEW_ARGS, n_seqs, n_heads, n_kv_heads, hd, scale, window, n_pages, seq0, a->status, s);
#undef HB_FEW_ARGS
    if (rc || a->whole) return rc;
    if (dtype == HB_F32)
        return launch_finish<float>(part_o, part_ml, scores, score_ld, page_table, pt_width, seq_start, seq_pos0, a->out, a->out_stride, mo, max_len,
                                    max_new, n_seqs, n_heads, n_kv_heads, hd, splits, window, n_pages, s);
    return launch_finish<bf16>(part_o, part_ml, scores, score_ld, page_table, pt_width, seq_start, seq_pos0, a->out, a->out_stride, mo, max_len, max_new,
                               n_seqs, n_heads, n_kv_heads, hd, splits, window, n_pages, s);
}
