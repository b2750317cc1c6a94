// Causal grouped attention over the paged cache that also adds up how much weight every cached row got: the kernels that take
// every head size up to 256, every group and both types, and the second half of steps of few tokens.
//
// For a token t of a sequence, a query head h of kv head g and a row j the token sees (lo..p, as in attention_general.cu):
//   s = scale q_th . k_jg,  lse_th = log sum_j exp(s),  w = exp(s - lse_th),  out_th = sum_j w v_jg,
//   mass_jg = (j appended by this step ? 0 : before_jg) + sum over the sequence's tokens t of the step and the heads h of g of w.
// A row's weight is known only once the token has seen all its keys, and then the scores are gone.  Two ways:
//   steps of few tokens   (memory-bound: keys and values are read once per token, a page at a time, by several blocks) the scores
//                         themselves are written beside the partial results, 4 bytes per (head, row) against the 2 head sizes of a
//                         key and a value; one more launch joins the partial results and turns the scores into weights.
//   steps of many tokens  (bound by arithmetic) the tokens' log-sums are kept and a second kernel, a block per tile of keys,
//                         computes its keys' scores with all queries once more: half as much arithmetic again instead of
//                         writing and reading a weight for every (token, head, row).  Every key's sum belongs to one thread from
//                         beginning to end, so the order of the additions is fixed.
// Softmax statistics, scores, sums and mass are float32; lse is in units of log 2.
#include "api.h"
#include "attention_mass.cuh"

// ------------------------------------------------------------------------------------------- many tokens, every head size
// Tiles of 64 queries (of one head) x 64 keys, 256 threads, 4 x 4 scores a thread (rows ty + 16 i, keys tx + 16 j), operands
// widened to float32 in shared memory, products on the FP32 pipe: the true 32-bit path has no other.  NC: value columns a thread
// holds (head size up to 16 NC).
#define AM_ROWS 64
#define AM_KEYS 64
#define AM_THREADS 256

// 64 rows of a tensor as float32 in shared memory, `ld` apart (a multiple of 4), in two halves so that the loads can be in flight while
// something else is computed: registers (up to 4 NC numbers a thread), then shared memory.  Rows from `rows` on and columns
// behind hd are zero.  vec: rows are aligned for four elements at a time.
template <typename T, int NC>
struct AmTile {
    float4 x[NC];
    __device__ __forceinline__ void load(const T* src, long long stride, int hd, int rows, bool vec, int tid) {
        const int per = (hd + 3) >> 2;
#pragma unroll
        for (int u = 0; u < NC; u++) {
            const int i = tid + u * AM_THREADS, r = i / per, d = (i - r * per) * 4;
            x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (r < rows) {
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
                      T* __restrict__ out, long long out_stride, float* __restrict__ lse, Shares sh, int n_tokens, int n_seqs, int nh, int nkv, int hd,
                      float scale_log2e, int window, int n_pages, int vec_q, int vec_kv, int* status) {
    extern __shared__ __align__(16) float am_smem[];
    pdl_trigger();
    pdl_wait();
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
    const int p0 = seq_pos0[b] + blk * AM_ROWS, p_last = p0 + rows - 1;
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
        tile.load(vc + row0 * hd, hd, hd, held, vec_kv, tid);
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
// block per token, a warp per head
template <typename T>
__global__ void __launch_bounds__(256)
shares_join_kernel(Shares sh, T* __restrict__ out, long long out_stride, float* __restrict__ lse, long long lse_ld, int rounded,
                   const int* __restrict__ seq_start, const int* __restrict__ seq_pos0, int span, int keys, int window, int n_tokens, int n_seqs, int nh,
                   int hd) {
    __shared__ float ws[8][32];
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, lane = threadIdx.x & 31;
    int b, i, place0;
    if (!mass_find_block(seq_start, n_seqs, t, 1, b, i, place0)) return;
    const int place = rounded ? place0 + i : t;
    const int n_new = seq_start[b + 1] - seq_start[b], row0 = (t - seq_start[b]) / span * span;
    int tile0;
    const int S = shares_of(sh, key_tiles_of(seq_pos0[b] + row0, seq_pos0[b] + min(row0 + span, n_new) - 1, window, keys, tile0));
    if (S == 1) return;
    float* mine = ws[threadIdx.x >> 5];
    for (int head = threadIdx.x >> 5; head < nh; head += 8) {
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
        __syncwarp();
    }
}

int shares_join(Shares sh, int dtype, void* out, long long out_stride, float* lse, long long lse_ld, int rounded, const int* seq_start,
                const int* seq_pos0, int span, int keys, int window, int n_tokens, int n_seqs, int nh, int hd, cudaStream_t s) {
    const dim3 grid(n_tokens);                             // a block per token: most tokens of a step with unequal sequences have one share
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
                       const int* seq_pos0, void* out, long long out_stride, float* lse, Shares sh, int max_shares, MassOut mo, int splits, int n_tokens,
                       int n_seqs, int q_blocks, int key_tiles, int nh, int nkv, int hd, float scale, int window, int n_pages, int* status, cudaStream_t s) {
    static_assert(AM_SMEM_ROWS(256) <= 227 * 1024, "attention tiles do not fit shared memory");
    static bool done[HB_MAX_DEVICES] = {}, done_mass[HB_MAX_DEVICES] = {};
    if (am_reserve(attention_rows_kernel<T, NC>, AM_SMEM_ROWS(16 * NC), done)) return 1;
    if (am_reserve(mass_rows_kernel<T, NC>, AM_SMEM_MASS(16 * NC), done_mass)) return 1;
    const uintptr_t four = 4 * sizeof(T);                      // four elements at a time where rows and heads begin at a multiple of that
    const int vec_kv = hd % 4 == 0 && (((uintptr_t)kc | (uintptr_t)vc) & (four - 1)) == 0;
    const int vec_q = hd % 4 == 0 && q_stride % 4 == 0 && ((uintptr_t)q & (four - 1)) == 0;
    cudaError_t e = hb_launch(attention_rows_kernel<T, NC>, dim3(nh, q_blocks, max_shares), dim3(AM_THREADS), AM_SMEM_ROWS(hd), s, (const T*)q, q_stride,
                              (const T*)kc, (const T*)vc, page_table, pt_width, seq_start, seq_pos0, (T*)out, out_stride, lse, sh, n_tokens, n_seqs, nh,
                              nkv, hd, scale * MASS_LOG2E, window, n_pages, vec_q, vec_kv, status);
    if (e != cudaSuccess) return hb_fail("attention_mass: launch failed: %s", cudaGetErrorString(e));
    if (hb_check_launch("attention_mass (rows)")) return 1;
    if (max_shares > 1 && shares_join(sh, sizeof(T) == 4 ? HB_F32 : HB_BF16, out, out_stride, lse, n_tokens, 0, seq_start, seq_pos0, AM_ROWS,
                                      HB_PAGE_TOKENS, window, n_tokens, n_seqs, nh, hd, s))
        return 1;
    e = hb_launch(mass_rows_kernel<T, NC>, dim3(key_tiles, nkv, splits), dim3(AM_THREADS), AM_SMEM_MASS(hd), s, (const T*)q, q_stride, (const T*)kc,
                  page_table, pt_width, seq_start, seq_pos0, (const float*)lse, mo, n_tokens, n_seqs, nh, nkv, hd, scale * MASS_LOG2E, window, n_pages,
                  vec_q, vec_kv, status);
    if (e != cudaSuccess) return hb_fail("attention_mass: launch failed: %s", cudaGetErrorString(e));
    if (hb_check_launch("attention_mass (weights)")) return 1;
    return splits > 1 ? mass_join(page_table, pt_width, seq_start, seq_pos0, mo, n_seqs, nkv, n_pages, AM_KEYS, key_tiles, splits, s) : 0;
}

// Steps of many tokens.  q_blocks: sum over sequences of ceil(new tokens / 64); key_tiles: sum of ceil(rows / 64); lse:
// n_heads * n_tokens floats; max_shares: the most blocks that a block of queries takes, share_tiles: the most pages of one of them;
// chunk_parts: max_shares * n_heads * n_tokens * (head_dim + 2) floats when max_shares > 1; parts: splits * n_kv_heads * key_tiles * 64
// floats when splits > 1.  before may be null or mass.
extern "C" int hb_attention_mass(const void* q, int dtype, long long q_stride, const void* k_cache, const void* v_cache, const int* page_table,
                                 int pt_width, const int* seq_start, const int* seq_pos0, void* out, long long out_stride, float* lse,
                                 const float* before, float* mass, float* parts, float* chunk_parts, int max_shares, int share_tiles, int splits,
                                 int n_tokens, int n_seqs, int q_blocks, int key_tiles, int n_heads, int n_kv_heads, int head_dim, float scale, int window,
                                 int n_pages, int* status, void* stream) {
    if (n_seqs == 0 || n_tokens == 0) return 0;
    HB_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && head_dim > 0 && head_dim <= 256 && n_pages > 0 && pt_width > 0,
               "attention_mass: %d heads over %d kv heads of size %d are not built (sizes up to 256)", n_heads, n_kv_heads, head_dim);
    HB_REQUIRE(n_kv_heads <= 65535 && q_blocks <= 65535 && key_tiles > 0 && splits >= 1 && splits <= 65535 && (splits == 1 || parts != nullptr) &&
                   max_shares >= 1 && max_shares <= 32 && share_tiles >= 1 && (max_shares == 1 || chunk_parts != nullptr),
               "attention_mass: the step is too large for one launch");
    HB_REQUIRE(lse != nullptr && mass != nullptr, "attention_mass: missing buffers");
    HB_REQUIRE(dtype == HB_F32 || dtype == HB_BF16, "attention_mass: unsupported dtype %d", dtype);
    MassOut mo = {before, mass, parts};
    // (maximum, sum) pairs in front: 8-byte aligned whatever the head size; one share: no block is cut, whatever it sees
    const Shares sh = {chunk_parts == nullptr ? nullptr : chunk_parts + (size_t)max_shares * n_heads * n_tokens * 2, chunk_parts,
                       max_shares == 1 ? 0x3fffffff : share_tiles};
    cudaStream_t s = (cudaStream_t)stream;
#define HB_AM_LAUNCH(T, NC)                                                                                                                     \
    launch_rows<T, NC>(q, q_stride, k_cache, v_cache, page_table, pt_width, seq_start, seq_pos0, out, out_stride, lse, sh, max_shares, mo, splits, \
                       n_tokens, n_seqs, q_blocks, key_tiles, n_heads, n_kv_heads, head_dim, scale, window, n_pages, status, s)
    if (dtype == HB_F32) return head_dim <= 64 ? HB_AM_LAUNCH(float, 4) : head_dim <= 128 ? HB_AM_LAUNCH(float, 8) : HB_AM_LAUNCH(float, 16);
    return head_dim <= 64 ? HB_AM_LAUNCH(bf16, 4) : head_dim <= 128 ? HB_AM_LAUNCH(bf16, 8) : HB_AM_LAUNCH(bf16, 16);
#undef HB_AM_LAUNCH
}

// -------------------------------------------------------------------------------------------- few tokens, every head size
// A block per (share of the token's pages, kv head and up to 8 of its query heads, token).  Scores: 4 threads per key, 16 bytes
// of the key's row each at a time; softmax: a warp per head; values: a thread per column (and share of the keys), 8 heads each.
#define AF_THREADS 256
#define AF_HEADS 8

template <typename T>
__global__ void __launch_bounds__(AF_THREADS)
few_rows_kernel(const T* __restrict__ q, long long q_stride, const T* __restrict__ kc, const T* __restrict__ vc, const int* __restrict__ page_table,
                int pt_width, const int* __restrict__ tok_seq, const int* __restrict__ positions, float* __restrict__ part_o,
                float* __restrict__ part_ml, float* __restrict__ scores, long long score_ld, int nh, int nkv, int hd, int head_blocks,
                int share_pages, float scale_log2e, int window, int n_pages, int* status) {
    extern __shared__ __align__(16) float am_smem[];
    __shared__ float sc[AF_HEADS][HB_PAGE_TOKENS + 1];   // a page's scores
    __shared__ float w8[HB_PAGE_TOKENS][AF_HEADS];       // and weights
    __shared__ float corr[AF_HEADS], stat[2][AF_HEADS];
    pdl_trigger();
    pdl_wait();
    q = pdl_fresh(q);
    kc = pdl_fresh(kc);
    vc = pdl_fresh(vc);
    const int G = nh / nkv, t = blockIdx.z, S = gridDim.x, z = blockIdx.x;
    const int g = blockIdx.y / head_blocks, h0 = (blockIdx.y % head_blocks) * AF_HEADS, H = min(AF_HEADS, G - h0);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = tok_seq[t], p = positions[t], lo = hb_oldest_visible(p, window, 0);
    const int* pt = page_table + (size_t)b * pt_width;
    const int width = (int)min((long long)pt_width, score_ld / HB_PAGE_TOKENS);      // no score is written behind its head's
    const int first = lo / HB_PAGE_TOKENS, last = min(p / HB_PAGE_TOKENS + 1, width);
    int p_begin, p_end;
    mass_share(first, last, z, S, share_pages, p_begin, p_end);
    if (z == 0 && tid == 0 && p >= width * HB_PAGE_TOKENS) hb_note(status, HB_STATUS_PAGE, 1 + b);
    const int hd4 = (hd + 3) & ~3;
    float* qs = am_smem;                                  // [8][hd4]
    float* so = qs + AF_HEADS * hd4;                      // [slices][8][hd]: at the end
    for (int i = tid; i < AF_HEADS * hd4; i += AF_THREADS) {
        const int h = i / hd4, d = i - h * hd4;
        qs[i] = (h < H && d < hd) ? to_f32(q[(size_t)t * q_stride + (size_t)(g * G + h0 + h) * hd + d]) : 0.0f;
    }
    float m = -INFINITY, l = 0.0f;                        // of head `warp`, in every lane
    const int slices = max(1, AF_THREADS / hd), d_own = tid % hd, slice = tid / hd;      // hd <= 256
    float acc[AF_HEADS];
#pragma unroll
    for (int h = 0; h < AF_HEADS; h++) acc[h] = 0.0f;
    const bool vec = hd % 4 == 0 && ((uintptr_t)kc & 15) == 0;
    for (int pi = p_begin; pi < p_end; pi++) {
        int page = pt[pi];
        if (page < 0 || page >= n_pages) {
            if (tid == 0) hb_note(status, HB_STATUS_PAGE, 1 + b);
            page = -1;
        }
        const size_t row0 = ((size_t)max(page, 0) * nkv + g) * HB_PAGE_TOKENS;
        __syncthreads();
        {
            const int e = tid >> 2, sub = tid & 3, key = pi * HB_PAGE_TOKENS + e;
            const bool seen = page >= 0 && key >= lo && key <= p;
            float dot[AF_HEADS];
#pragma unroll
            for (int h = 0; h < AF_HEADS; h++) dot[h] = 0.0f;
            if (seen) {
                const T* kr = kc + (row0 + e) * hd;
                for (int d = sub * 4; d < hd4; d += 16) {
                    float x[4];
                    if (vec) {
                        load4(kr + d, x);
                    } else {
#pragma unroll
                        for (int u = 0; u < 4; u++) x[u] = d + u < hd ? to_f32(kr[d + u]) : 0.0f;
                    }
#pragma unroll
                    for (int h = 0; h < AF_HEADS; h++) {
                        const float4 y = *reinterpret_cast<const float4*>(qs + h * hd4 + d);
                        dot[h] = fmaf(x[0], y.x, fmaf(x[1], y.y, fmaf(x[2], y.z, fmaf(x[3], y.w, dot[h]))));
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < AF_HEADS; h++) {
                dot[h] += __shfl_xor_sync(0xffffffffu, dot[h], 1);
                dot[h] += __shfl_xor_sync(0xffffffffu, dot[h], 2);
            }
            if (sub == 0) {
#pragma unroll
                for (int h = 0; h < AF_HEADS; h++) sc[h][e] = seen ? dot[h] * scale_log2e : -INFINITY;
            }
        }
        __syncthreads();
        {
            const float a = sc[warp][lane], c = sc[warp][lane + 32];
            const float m_new = fmaxf(m, warp_max(fmaxf(a, c))), m_safe = m_new == -INFINITY ? 0.0f : m_new;
            const float f = exp2f(m - m_safe), wa = exp2f(a - m_safe), wc = exp2f(c - m_safe);
            m = m_new;
            l = l * f + warp_sum(wa + wc);
            w8[lane][warp] = wa;
            w8[lane + 32][warp] = wc;
            if (lane == 0) corr[warp] = f;
            if (warp < H) {
                float* dst = scores + ((size_t)t * nh + g * G + h0 + warp) * score_ld + (size_t)pi * HB_PAGE_TOKENS;
                dst[lane] = a;
                dst[lane + 32] = c;
            }
        }
        __syncthreads();
        if (slice < slices) {
#pragma unroll
            for (int h = 0; h < AF_HEADS; h++) acc[h] *= corr[h];
            const int e_end = min(HB_PAGE_TOKENS, p - pi * HB_PAGE_TOKENS + 1);
            if (page >= 0) {
                for (int e = slice; e < e_end; e += slices) {
                    const float x = to_f32(vc[(row0 + e) * hd + d_own]);
                    const float4 wa = *reinterpret_cast<const float4*>(&w8[e][0]), wb = *reinterpret_cast<const float4*>(&w8[e][4]);
                    const float w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
                    if (pi * HB_PAGE_TOKENS + e < lo) continue;
#pragma unroll
                    for (int h = 0; h < AF_HEADS; h++) acc[h] = fmaf(w[h], x, acc[h]);
                }
            }
        }
    }
    __syncthreads();
    if (slice < slices) {
#pragma unroll
        for (int h = 0; h < AF_HEADS; h++) so[((size_t)slice * AF_HEADS + h) * hd + d_own] = acc[h];
    }
    if (lane == 0) {
        stat[0][warp] = m;
        stat[1][warp] = l;
    }
    __syncthreads();
    for (int i = tid; i < H * hd; i += AF_THREADS) {
        const int h = i / hd, d = i - h * hd;
        float s = 0.0f;
        for (int c = 0; c < slices; c++) s += so[((size_t)c * AF_HEADS + h) * hd + d];
        const size_t base = ((size_t)t * nh + g * G + h0 + h) * S + z;
        part_o[base * hd + d] = s;
        if (d == 0) {
            part_ml[base * 2] = stat[0][h];
            part_ml[base * 2 + 1] = stat[1][h];
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
                  const int* __restrict__ page_table, int pt_width, const int* __restrict__ seq_start, const int* __restrict__ seq_pos0, T* __restrict__ out,
                  long long out_stride, MassOut mo, int token_rows, int nh, int nkv, int hd, int S, int window, int n_pages, int vec) {
    __shared__ float lse[MASS_FEW_PAIRS];
    pdl_trigger();
    pdl_wait();
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
            for (int d0 = 0; d0 < hd; d0 += 128) {             // four columns a lane, all shares' loads in flight
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
                for (int z = 0; z < S; z++) {
                    const float mz = __ldcg(part_ml + (base + z) * 2);
                    const float w = mz != -INFINITY ? exp2f(mz - M) : 0.0f;
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const int d = d0 + u * 32 + lane;
                        const float x = d < hd ? __ldcg(part_o + (base + z) * hd + d) : 0.0f;
                        if (w != 0.0f) acc[u] = fmaf(x, w, acc[u]);          // a share without keys has written no output
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int d = d0 + u * 32 + lane;
                    if (d < hd) out[(size_t)t * out_stride + (size_t)(g * G + h) * hd + d] = from_f32<T>(acc[u] * inv);
                }
            }
        }
        return;
    }
    const int n = (int)min((long long)(pos0 + n_new), score_ld), key0 = ((int)blockIdx.x - token_rows) * FF_KEYS;
    if (key0 >= n) return;
    for (int i = warp; i < n_new * G; i += FF_THREADS / 32) {
        float M, L;
        join_stats(part_ml, ((size_t)(t0 + i / G) * nh + g * G + i % G) * S, S, lane, M, L);
        if (lane == 0) lse[i] = L > 0.0f ? M + log2f(L) : INFINITY;
    }
    __syncthreads();
    const int key = key0 + tid * 4;                            // this thread's four keys, on one page
    if (key >= n) return;
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
    const int pi = key / HB_PAGE_TOKENS;
    const int page = pi < pt_width ? page_table[(size_t)b * pt_width + pi] : -1;
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
static int launch_few(const void* q, long long q_stride, const void* kc, const void* vc, const int* page_table, int pt_width, const int* tok_seq,
                      const int* positions, float* part_o, float* part_ml, float* scores, long long score_ld, int splits, int share_pages, int n_tokens, int nh,
                      int nkv, int hd, float scale, int window, int n_pages, int* status, cudaStream_t s) {
    const int hd4 = (hd + 3) & ~3, slices = AF_THREADS / hd > 1 ? AF_THREADS / hd : 1, hb = (nh / nkv + AF_HEADS - 1) / AF_HEADS;
    const int smem = (AF_HEADS * hd4 + slices * AF_HEADS * hd) * 4;        // at most 16 KB
    HB_REQUIRE((long long)nkv * hb <= 65535, "attention_mass: too many heads for one launch");
    cudaError_t e = hb_launch(few_rows_kernel<T>, dim3(splits, nkv * hb, n_tokens), dim3(AF_THREADS), smem, s, (const T*)q, q_stride, (const T*)kc,
                              (const T*)vc, page_table, pt_width, tok_seq, positions, part_o, part_ml, scores, score_ld, nh, nkv, hd, hb, share_pages,
                              scale * MASS_LOG2E, window, n_pages, status);
    if (e != cudaSuccess) return hb_fail("attention_mass: launch failed: %s", cudaGetErrorString(e));
    return hb_check_launch("attention_mass (few tokens)");
}

template <typename T>
static int launch_finish(const float* part_o, const float* part_ml, const float* scores, long long score_ld, const int* page_table, int pt_width,
                         const int* seq_start, const int* seq_pos0, void* out, long long out_stride, MassOut mo, int max_len, int max_new, int n_seqs,
                         int nh, int nkv, int hd, int splits, int window, int n_pages, cudaStream_t s) {
    const int key_blocks = (max_len + FF_KEYS - 1) / FF_KEYS;
    const int vec = (((uintptr_t)mo.before | (uintptr_t)mo.mass) & 15) == 0;
    cudaError_t e = hb_launch(few_finish_kernel<T>, dim3(max_new + key_blocks, nkv, n_seqs), dim3(FF_THREADS), 0, s, part_o, part_ml, scores, score_ld,
                              page_table, pt_width, seq_start, seq_pos0, (T*)out, out_stride, mo, max_new, nh, nkv, hd, splits, window, n_pages, vec);
    if (e != cudaSuccess) return hb_fail("attention_mass: launch failed: %s", cudaGetErrorString(e));
    return hb_check_launch("attention_mass (finish)");
}

// Steps of few tokens (at most hb_attention_few_pairs() pairs of a sequence's tokens and a group's heads).  `scratch` holds
// hb_attention_mass_few_floats floats; token_blocks: 0, or for the tensor cores as attention_few_tc; a
// sequence's pages go into at most `splits` shares, of share_pages or more; max_len bounds the rows of every sequence, max_new their new tokens.
extern "C" int hb_attention_mass_few(const void* q, int dtype, long long q_stride, const void* k_cache, const void* v_cache, const int* page_table,
                                     int pt_width, const int* tok_seq, const int* positions, const int* seq_start, const int* seq_pos0, void* out,
                                     long long out_stride, float* scratch, const float* before, float* mass, int splits, int share_pages, int n_tokens,
                                     int n_seqs, int max_new, int max_len, int n_heads, int n_kv_heads, int head_dim, float scale, int window, int n_pages,
                                     int token_blocks, int* status, void* stream) {
    if (n_seqs == 0 || n_tokens == 0) return 0;
    HB_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && head_dim > 0 && head_dim <= 256 && n_pages > 0 && pt_width > 0,
               "attention_mass: %d heads over %d kv heads of size %d are not built (sizes up to 256)", n_heads, n_kv_heads, head_dim);
    HB_REQUIRE((long long)max_new * (n_heads / n_kv_heads) <= MASS_FEW_PAIRS, "attention_mass: %d tokens of %d heads are no step of few tokens",
               max_new, n_heads / n_kv_heads);
    HB_REQUIRE(n_tokens <= 65535 && n_seqs <= 65535 && n_kv_heads <= 65535 && splits >= 1 && max_len >= 1 && share_pages >= 1 && scratch != nullptr && mass != nullptr,
               "attention_mass: bad sizes");
    const size_t rows = (size_t)n_tokens * n_heads * splits;
    const long long score_ld = mass_score_ld(max_len);
    float *scores = scratch, *part_ml = scores + (size_t)n_tokens * n_heads * score_ld, *part_o = part_ml + rows * 2;
    HB_REQUIRE(((uintptr_t)scratch & 15) == 0, "attention_mass: scratch must be 16-byte aligned");
    cudaStream_t s = (cudaStream_t)stream;
    MassOut mo = {before, mass, nullptr};
    int rc;
    if (token_blocks > 0) {
        HB_REQUIRE(dtype == HB_BF16, "attention_mass: the tensor cores take bfloat16");
        rc = attention_few_tc(q, q_stride, k_cache, v_cache, page_table, pt_width, seq_start, seq_pos0, part_o, part_ml, scores, score_ld, splits, share_pages,
                              token_blocks, max_new, n_seqs, n_heads, n_kv_heads, head_dim, scale, window, n_pages, status, s);
    } else if (dtype == HB_F32)
        rc = launch_few<float>(q, q_stride, k_cache, v_cache, page_table, pt_width, tok_seq, positions, part_o, part_ml, scores, score_ld, splits, share_pages,
                               n_tokens, n_heads, n_kv_heads, head_dim, scale, window, n_pages, status, s);
    else if (dtype == HB_BF16)
        rc = launch_few<bf16>(q, q_stride, k_cache, v_cache, page_table, pt_width, tok_seq, positions, part_o, part_ml, scores, score_ld, splits, share_pages, n_tokens,
                              n_heads, n_kv_heads, head_dim, scale, window, n_pages, status, s);
    else
        return hb_fail("attention_mass: unsupported dtype %d", dtype);
    if (rc) return rc;
    if (dtype == HB_F32)
        return launch_finish<float>(part_o, part_ml, scores, score_ld, page_table, pt_width, seq_start, seq_pos0, out, out_stride, mo, max_len, max_new,
                                    n_seqs, n_heads, n_kv_heads, head_dim, splits, window, n_pages, s);
    return launch_finish<bf16>(part_o, part_ml, scores, score_ld, page_table, pt_width, seq_start, seq_pos0, out, out_stride, mo, max_len, max_new, n_seqs,
                               n_heads, n_kv_heads, head_dim, splits, window, n_pages, s);
}
