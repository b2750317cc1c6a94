// The first half of a step of few tokens with accumulated weights (attention_mass.cu) on the tensor cores, bfloat16, head sizes up to
// 128 in steps of 8: partial results over shares of the keys, and the scores themselves, for the kernel that joins the shares and turns the
// scores into weights; or, of short sequences, everything in one block (mass_whole).
//
// A CTA = a share of the pages x one kv head x a block of a sequence's new tokens: the rows of the mma.sync tiles (16 RT of them) are the
// (token, head) pairs of the block, so a page is read once for all of them.  Bound by memory: 2 head sizes of keys and values per row of
// the cache against 4 bytes of score per pair.  The pages stream through three cp.async stages; a warp takes a quarter of every page's
// keys for one tile of 16 rows, with its own running maximum and sum, joined through shared memory at the end: 28 us for 17 drafted
// tokens of four sequences.  (Two tiles of rows in one warp leave two warps to a quarter of the SM, latencies unhidden: a tenth slower.  With
// a CTA per token, as for single tokens, those tokens took 82 us in all instead of 46; their pages came from L2 17 times.)
#include "api.h"
#include "attention_mass.cuh"
#include "mma.cuh"

#define FT_STAGES 3

// FULL: the head size is HD; else it is hd < HD, and the columns behind it are zeros in the tiles and in the queries.
template <int HD, int RT, bool FULL>
__global__ void __launch_bounds__(128 * RT, 2)
few_tc_kernel(const bf16* __restrict__ q, long long q_stride, const bf16* __restrict__ kc, const bf16* __restrict__ vc,
              const int* __restrict__ page_table, int pt_width, const int* __restrict__ seq_start, const int* __restrict__ seq_pos0, float* part_o,
              float* part_ml, float* scores, long long score_ld, int tokens_per_block, int share_pages, int n_seqs, int nh, int nkv, int hd_given,
              float scale_log2e, int window, int n_pages, MassWhole whole, int seq0, int* status) {
    constexpr int ROW_BYTES = HD * 2, TILE_BYTES = HB_PAGE_TOKENS * ROW_BYTES, CHUNKS = ROW_BYTES / 16, KSTEPS = HD / 16, ROWS = 16 * RT,
    THREADS = 128 * RT;
    const int hd = FULL ? HD : hd_given, chunks = FULL ? CHUNKS : hd / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float lse[ROWS];                            // of a whole sequence's pairs
    pdl_trigger();
    pdl_wait();
    mass_fresh(page_table, seq_start, seq_pos0);
    q = pdl_fresh(q);
    const int z = blockIdx.x, g = blockIdx.y, S = gridDim.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = (tid >> 5) & 3, rt = tid >> 7;       // quarter of a page's keys, tile of rows
    const int G = nh / nkv;
    int b, blk, place0;
    if (!mass_find_block(seq_start, n_seqs, blockIdx.z, tokens_per_block, b, blk, place0)) return;
    const int t0 = seq_start[b] + blk * tokens_per_block, n_tok = min(tokens_per_block, seq_start[b + 1] - t0);
    const int p0 = seq_pos0[b] + blk * tokens_per_block, p_last = p0 + n_tok - 1;
    const int width = (int)min((long long)pt_width, score_ld / HB_PAGE_TOKENS);       // no score is written behind its head's
    const int oldest = hb_oldest_visible(p0, window, 0), first = oldest / HB_PAGE_TOKENS, last = min(p_last / HB_PAGE_TOKENS + 1, width);
    int page0, page1;
    mass_share(first, last, z, S, share_pages, page0, page1);
    const int* pt = page_table + (size_t)b * pt_width;
    if (z == 0 && tid == 0 && p_last >= width * HB_PAGE_TOKENS) hb_note(status, HB_STATUS_PAGE, 1 + seq0 + b);
    const int pairs = n_tok * G;                           // row r is head r % G of token r / G
    if (page0 >= page1 && whole.out == nullptr) {          // a share without keys
        for (int r = tid; r < pairs; r += THREADS) {
            float* ml = part_ml + (((size_t)(t0 + r / G) * nh + g * G + r % G) * S + z) * 2;
            ml[0] = -INFINITY;
            ml[1] = 0.0f;
        }
        return;
    }
    const uint32_t smem_base = (uint32_t)__cvta_generic_to_shared(smem);
    bool bad_page = false;
    auto load_page = [&](int stage, int pi) {
        if (pi < page1) {
            int page = pt[pi];
            if (page < 0 || page >= n_pages) {
                bad_page = true;
                page = 0;                                   // never read outside the cache
            }
            const uint8_t* ksrc = (const uint8_t*)(kc + ((size_t)page * nkv + g) * HB_PAGE_TOKENS * hd);
            const uint8_t* vsrc = (const uint8_t*)(vc + ((size_t)page * nkv + g) * HB_PAGE_TOKENS * hd);
            const uint32_t kdst = smem_base + stage * 2 * TILE_BYTES, vdst = kdst + TILE_BYTES;
#pragma unroll
            for (int i = tid; i < HB_PAGE_TOKENS * chunks; i += THREADS) {
                const int row = i / chunks, ch = i - row * chunks;
                const uint32_t off = swizzled<ROW_BYTES>(row, ch);
                cp_async_16(kdst + off, ksrc + (size_t)i * 16);
                // values behind the last key and in front of the oldest are whatever is there, and 0 * NaN is NaN
                const int key = pi * HB_PAGE_TOKENS + row;
                cp_async_16_or_zero(vdst + off, vsrc + (size_t)i * 16, key >= oldest && key <= p_last);
            }
        }
        cp_async_commit();
    };
    if (!FULL) {
        for (int i = tid; i < FT_STAGES * 2 * TILE_BYTES / 16; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
    }
#pragma unroll
    for (int s = 0; s < FT_STAGES - 1; s++) load_page(s, page0 + s);

    // this thread's rows: r = 16 rt + 8 h + lane / 4
    uint32_t qf[KSTEPS][4];
    int row_lo[2], row_end[2];                             // the row sees the keys [row_lo, row_end)
    float* row_scores[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int r = rt * 16 + h * 8 + (lane >> 2);
        const bool there = r < pairs;
        const int i = there ? r / G : 0, head = g * G + (there ? r - i * G : 0);
        row_lo[h] = hb_oldest_visible(p0 + i, window, 0);
        row_end[h] = there ? p0 + i + 1 : 0;
        row_scores[h] = scores + ((size_t)(t0 + i) * nh + head) * score_ld;
        const unsigned int* src = reinterpret_cast<const unsigned int*>(q + (size_t)(t0 + i) * q_stride + (size_t)head * hd + (lane & 3) * 2);
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ks++) {
            qf[ks][h] = there && (FULL || ks * 16 < hd) ? __ldcg(src + ks * 8) : 0u;
            qf[ks][h + 2] = there && (FULL || ks * 16 + 8 < hd) ? __ldcg(src + ks * 8 + 4) : 0u;
        }
    }
    float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < HD / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    for (int pi = page0; pi < page1; pi++) {
        const int it = pi - page0;
        cp_async_wait<FT_STAGES - 2>();
        __syncthreads();
        load_page((it + FT_STAGES - 1) % FT_STAGES, pi + FT_STAGES - 1);
        const uint32_t kt = smem_base + (it % FT_STAGES) * 2 * TILE_BYTES, vt = kt + TILE_BYTES;
        float s[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
        const int key_row = warp * 16 + ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ks++) {
            uint32_t kf[4];
            ldmatrix_x4(kf, kt + swizzled<ROW_BYTES>(key_row, 2 * ks + ((lane >> 3) & 1)));
            mma_bf16_16816(s[0], qf[ks], kf[0], kf[1]);
            mma_bf16_16816(s[1], qf[ks], kf[2], kf[3]);
        }
        const int key0 = pi * HB_PAGE_TOKENS + warp * 16 + (lane & 3) * 2;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float top = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < 2; nt++) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int key = key0 + nt * 8 + e;
                    const float v = key >= row_lo[h] && key < row_end[h] ? s[nt][2 * h + e] * scale_log2e : -INFINITY;
                    s[nt][2 * h + e] = v;
                    top = fmaxf(top, v);
                }
                if (row_end[h] > 0) *reinterpret_cast<float2*>(row_scores[h] + key0 + nt * 8) = make_float2(s[nt][2 * h], s[nt][2 * h + 1]);
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float m_new = fmaxf(m[h], top), m_safe = m_new == -INFINITY ? 0.0f : m_new;
            const float corr = exp2f(m[h] - m_safe);
            m[h] = m_new;
            float sum = 0.0f;
#pragma unroll
            for (int nt = 0; nt < 2; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float w = exp2f(s[nt][2 * h + e] - m_safe);
                    s[nt][2 * h + e] = w;
                    sum += w;
                }
            l[h] = l[h] * corr + sum;
            if (__any_sync(0xffffffffu, corr != 1.0f)) {   // a maximum grew: rarely, after the first pages
#pragma unroll
                for (int i = 0; i < HD / 8; i++) {
                    o[i][2 * h] *= corr;
                    o[i][2 * h + 1] *= corr;
                }
            }
        }
        const uint32_t pa[4] = {pack_bf16(s[0][0], s[0][1]), pack_bf16(s[0][2], s[0][3]), pack_bf16(s[1][0], s[1][1]), pack_bf16(s[1][2], s[1][3])};
        const int v_row = warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
        for (int dn = 0; dn < HD / 16; dn++) {
            uint32_t vf[4];
            ldmatrix_x4_trans(vf, vt + swizzled<ROW_BYTES>(v_row, 2 * dn + (lane >> 4)));
            mma_bf16_16816(o[2 * dn], pa, vf[0], vf[1]);
            mma_bf16_16816(o[2 * dn + 1], pa, vf[2], vf[3]);
        }
    }
    cp_async_wait<0>();
    __syncthreads();
    if (bad_page && tid == 0) hb_note(status, HB_STATUS_PAGE, 1 + seq0 + b);

    float* so = reinterpret_cast<float*>(smem);                        // [4 quarters][ROWS][HD]
    float* sm = so + 4 * ROWS * HD;                                    // [4][ROWS]
    float* sl = sm + 4 * ROWS;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int r = rt * 16 + h * 8 + (lane >> 2);
        float sum = l[h];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int i = 0; i < HD / 8; i++)
            *reinterpret_cast<float2*>(so + (size_t)(warp * ROWS + r) * HD + i * 8 + (lane & 3) * 2) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
        if ((lane & 3) == 0) {
            sm[warp * ROWS + r] = m[h];
            sl[warp * ROWS + r] = sum;
        }
    }
    __syncthreads();
    for (int idx = tid; idx < pairs * hd; idx += THREADS) {
        const int r = idx / hd, d = idx - r * hd, i = r / G;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; w++) M = fmaxf(M, sm[w * ROWS + r]);
        float acc = 0.0f, L = 0.0f;
        if (M != -INFINITY) {
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float e = exp2f(sm[w * ROWS + r] - M);
                acc += so[(size_t)(w * ROWS + r) * HD + d] * e;
                L += sl[w * ROWS + r] * e;
            }
        }
        if (whole.out != nullptr) {
            ((bf16*)whole.out)[(size_t)(t0 + i) * whole.out_stride + (size_t)(g * G + (r - i * G)) * hd + d] =
                __float2bfloat16_rn(acc * (L > 0.0f ? 1.0f / L : 0.0f));
            if (d == 0) lse[r] = L > 0.0f ? M + log2f(L) : INFINITY;
            continue;
        }
        const size_t base = ((size_t)(t0 + i) * nh + g * G + (r - i * G)) * S + z;
        part_o[base * hd + d] = acc;
        if (d == 0) {
            part_ml[base * 2] = M;
            part_ml[base * 2 + 1] = L;
        }
    }
    if (whole.out != nullptr) {
        __syncthreads();
        mass_whole(whole.mo, scores, score_ld, lse, n_tok, G, g, t0, nh, nkv, p0, window, pt, pt_width, n_pages);
    }
}

template <int HD, int RT, bool FULL>
static int launch_few_tc(MassWhole whole, const void* q, long long q_stride, const void* kc, const void* vc, const int* page_table, int pt_width,
                         const int* seq_start, const int* seq_pos0, float* part_o, float* part_ml, float* scores, long long score_ld, int splits,
                         int token_blocks, int tokens_per_block, int share_pages, int n_seqs, int nh, int nkv, int hd, float scale, int window,
                         int n_pages, int seq0, int* status, cudaStream_t s) {
    constexpr int PIPE = FT_STAGES * 2 * HB_PAGE_TOKENS * HD * 2, MERGE = (4 * 16 * RT * HD + 2 * 4 * 16 * RT) * 4,
    SMEM = PIPE > MERGE ? PIPE : MERGE;
    static bool done[HB_MAX_DEVICES] = {};
    bool& set = done[hb_device_slot()];
    if (!set) {
        cudaError_t e = cudaFuncSetAttribute(few_tc_kernel<HD, RT, FULL>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return hb_fail("attention_mass: cannot reserve %d bytes of shared memory: %s", SMEM, cudaGetErrorString(e));
        set = true;
    }
    cudaError_t e = hb_launch(few_tc_kernel<HD, RT, FULL>, dim3(splits, nkv, token_blocks), dim3(128 * RT), SMEM, s, (const bf16*)q, q_stride,
                              (const bf16*)kc, (const bf16*)vc, page_table, pt_width, seq_start, seq_pos0, part_o, part_ml, scores, score_ld,
                              tokens_per_block, share_pages, n_seqs, nh, nkv, hd, scale * MASS_LOG2E, window, n_pages, whole, seq0, status);
    if (e != cudaSuccess) return hb_fail("attention_mass: launch failed: %s", cudaGetErrorString(e));
    return hb_check_launch("attention_mass (few tokens, tensor cores)");
}

extern "C" int hb_attention_few_tc_tokens(int n_heads, int n_kv_heads, int head_dim, int max_new) {
    if (head_dim < 8 || head_dim > 128 || head_dim % 8 != 0 || n_kv_heads < 1 || n_heads % n_kv_heads != 0 || n_heads / n_kv_heads > 32 || max_new < 1) return 0;
    const int G = n_heads / n_kv_heads, rows = G * max_new <= 16 ? 16 : 32;
    return rows / G;
}

int attention_few_tc(MassWhole whole, const void* q, long long q_stride, const void* kc, const void* vc, const int* page_table, int pt_width,
                     const int* seq_start, const int* seq_pos0, float* part_o, float* part_ml, float* scores, long long score_ld, int splits,
                     int share_pages, int token_blocks, int max_new, int n_seqs, int nh, int nkv, int head_dim, float scale, int window, int n_pages,
                     int seq0, int* status, cudaStream_t s) {
    const int tokens = hb_attention_few_tc_tokens(nh, nkv, head_dim, max_new);
    HB_REQUIRE(tokens > 0, "attention_mass: head size %d with %d heads over %d kv heads is not built for the tensor cores (up to 128 in steps of 8, groups up to"
               " 32)",
               head_dim, nh, nkv);
    HB_REQUIRE(q_stride % 2 == 0 && ((uintptr_t)q & 3) == 0 && (((uintptr_t)kc | (uintptr_t)vc) & 15) == 0,
               "attention_mass: queries must be 4-byte and the cache 16-byte aligned");
    HB_REQUIRE(token_blocks <= 65535, "attention_mass: too many tokens for one launch");
    const bool two = nh / nkv * tokens > 16;
#define HB_FT_LAUNCH(HD, RT, FULL)                                                                                                                  \
    launch_few_tc<HD, RT, FULL>(whole, q, q_stride, kc, vc, page_table, pt_width, seq_start, seq_pos0, part_o, part_ml, scores, score_ld, splits, token_blocks, \
                                tokens, share_pages, n_seqs, nh, nkv, head_dim, scale, window, n_pages, seq0, status, s)
    if (head_dim == 128) return two ? HB_FT_LAUNCH(128, 2, true) : HB_FT_LAUNCH(128, 1, true);
    if (head_dim > 64) return two ? HB_FT_LAUNCH(128, 2, false) : HB_FT_LAUNCH(128, 1, false);
    if (head_dim == 64) return two ? HB_FT_LAUNCH(64, 2, true) : HB_FT_LAUNCH(64, 1, true);
    return two ? HB_FT_LAUNCH(64, 2, false) : HB_FT_LAUNCH(64, 1, false);
#undef HB_FT_LAUNCH
}
