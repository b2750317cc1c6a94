// The weights of steps of many tokens on the 5th-generation tensor cores (tcgen05 + TMEM + TMA), bfloat16, head sizes up to 128
// in steps of 8 (as attention_chunk_tc.cu): the second half of attention_mass.cu's arithmetic, behind the attention that leaves each
// row's log-sum.
//
// One CTA = 256 consecutive rows of a sequence's cache x one kv head x a share of the (head, 128 queries) tiles that see them.
// Keys are the M operand: a tile's 128 keys are the 128 lanes of tensor memory and the queries its columns, so that a key's sum over
// queries and heads stays in one thread's registers from beginning to end and is written once: no atomics, no shuffles.
//   warp 0      TMA producer: the two key tiles once, then query tiles with their log-sums (three stages)
//   warp 1      owns tensor memory; one thread issues S = K Q^T of the two key tiles (head size / 16 steps each) into two pairs of buffers
//   warps 2-17  weights: 8 warps per key tile, a thread has 64 queries of its key: w = 2^(s scale log2(e) - lse), added up
//               (the log-sums come negated)
// What bounds it: 16 exponentials a clock and SM (1024 clocks for 128 x 128 weights, against 512 for the product at head size
// 128), so a pair in eight is computed on the FMA pipe instead (none: 684, one: 654, three: 697 us for 2048 tokens behind 30001 rows of the
// 8B sizes when that was chosen, 636 now; the products alone take 418).  Two key tiles share a query tile because an SM takes about 32
// bytes a clock from L2: with one, loading a 32 KB query tile would last as long as its exponentials.
//
// Every wait is bounded; a wait that runs out sets *error_flag and the CTA drains and leaves.
#include "api.h"
#include "attention_mass.cuh"
#include "attention_tc.cuh"
#include "exp2_pair.cuh"

#define MT_KEYS 256
#define MT_THREADS 576
#define MT_STAGES 3
#define MT_WORKER_WARPS 16

// `bytes` from global into shared memory (both 16-byte aligned), counted on `bar`
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

template <int HD>
__global__ void __launch_bounds__(MT_THREADS, 1)
mass_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const int* __restrict__ page_table,
               int pt_width, const int* __restrict__ seq_start, const int* __restrict__ seq_pos0, const float* lse, long long lse_ld, MassOut mo,
               int n_seqs, int nh, int nkv, int hd, float scale_log2e, int window, int n_pages, int S, int* __restrict__ error_flag) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    // [K tiles 2][Q stages 3][log-sums of the stages][barriers]; a tile is 128 rows x HD
    constexpr int HALVES = HD / 64, TILE = HALVES * FA_HALF_BYTES;
    float* xlse = (float*)(smem + (2 + MT_STAGES) * TILE);     // [stages][128 queries]
    uint64_t* bars = (uint64_t*)(xlse + MT_STAGES * 128);
    uint32_t* tmem_slot = (uint32_t*)(bars + 16);
    float* xsum = (float*)(tmem_slot + 4);                     // [2 key tiles][128]
    const uint32_t smem_base = smem_u32(smem), q_smem = smem_base + 2 * TILE;
    const uint32_t k_full = smem_u32(bars), q_full0 = smem_u32(bars + 1), q_empty0 = smem_u32(bars + 4);
    const uint32_t s_full0 = smem_u32(bars + 7), s_empty0 = smem_u32(bars + 9);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Under a causal mask a sequence's first keys are seen by the most queries: with the tiles as the slowest index, the shares of its
    // heaviest ones start first and what ends last is light.  (Sequences start in the step's order.)
    const int z = blockIdx.x % S, g = blockIdx.x / S % nkv, G = nh / nkv, tile = blockIdx.x / (S * nkv);

    if (threadIdx.x == 0) {
        mbar_init(k_full, 1);
        for (int s = 0; s < MT_STAGES; s++) {
            mbar_init(q_full0 + 8 * s, 1);
            mbar_init(q_empty0 + 8 * s, 1 + MT_WORKER_WARPS);  // the products have read the queries, the workers the log-sums
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(s_full0 + 8 * s, 1);
            mbar_init(s_empty0 + 8 * s, MT_WORKER_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;                    // buffer s of key tile k at columns (2 s + k) * 128
    pdl_trigger();
    pdl_wait();
    mass_fresh(page_table, seq_start, seq_pos0);

    int b, kt, place0;
    const bool has_work = mass_find_keys(seq_start, seq_pos0, n_seqs, tile, MT_KEYS, b, kt, place0);
    const int t_begin = mass_uniform(has_work ? seq_start[b] : 0), n_new = mass_uniform(has_work ? seq_start[b + 1] - t_begin : 0),
              pos0 = mass_uniform(has_work ? seq_pos0[b] : 0);
    const int key0 = kt * MT_KEYS;
    int n0 = 0, n1 = 0;
    if (has_work) mass_queries(key0, MT_KEYS, pos0, n_new, window, n0, n1);
    n0 &= ~127;                                                // whole blocks of 128 new tokens, as the log-sums lie
    const int blocks = (n1 - n0 + 127) / 128;
    const int it0 = (int)((long long)blocks * G * z / S), n_it = (int)((long long)blocks * G * (z + 1) / S) - it0;

    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer
        if (lane == 0 && n_it > 0) {
            const int* pt = page_table + (size_t)b * pt_width;
            mbar_expect_tx(k_full, 2 * TILE);
            int pages[MT_KEYS / HB_PAGE_TOKENS];                    // asked for at once
#pragma unroll
            for (int pg = 0; pg < MT_KEYS / HB_PAGE_TOKENS; pg++) {
                const int pi = kt * (MT_KEYS / HB_PAGE_TOKENS) + pg;
                pages[pg] = pi < pt_width ? pt[pi] : -1;
            }
#pragma unroll
            for (int pg = 0; pg < MT_KEYS / HB_PAGE_TOKENS; pg++) {
                const int pi = kt * (MT_KEYS / HB_PAGE_TOKENS) + pg;
                int page = pages[pg];
                if (page < 0 || page >= n_pages) {
                    // a page that no token of the step sees (behind the end, or given back) may be missing
                    int a, e;
                    mass_queries(pi * HB_PAGE_TOKENS, HB_PAGE_TOKENS, pos0, n_new, window, a, e);
                    if (e > a) hb_note(error_flag, HB_STATUS_PAGE, 1 + b);
                    page = 0;                                       // never read outside the cache
                }
                const uint32_t dst = smem_base + (pg >> 1) * TILE + (pg & 1) * (FA_HALF_BYTES / 2);
                for (int half = 0; half < HALVES; half++)
                    tma_load_2d(dst + half * FA_HALF_BYTES, &map_k, k_full, half * 64, (page * nkv + g) * HB_PAGE_TOKENS);
            }
            const int lse0 = place0 + n0;                           // where the log-sums of token n0 lie
            int issued = 0;
            for (int it = 0; it < n_it; it++) {
                const int s = it % MT_STAGES;
                if (!mbar_wait(q_empty0 + 8 * s, ((it / MT_STAGES) & 1) ^ 1)) {
                    atomicExch(error_flag, 61);
                    break;
                }
                const int item = it0 + it, head = g * G + item / blocks, q0 = (item % blocks) * 128;
                mbar_expect_tx(q_full0 + 8 * s, TILE + 512);
                for (int half = 0; half < HALVES; half++)
                    tma_load_3d(q_smem + s * TILE + half * FA_HALF_BYTES, &map_q, q_full0 + 8 * s, half * 64, head, t_begin + n0 + q0);
                bulk_load(smem_u32(xlse + s * 128), lse + (size_t)head * lse_ld + lse0 + q0, 512, q_full0 + 8 * s);
                issued = it + 1;
            }
            for (int it = max(0, issued - MT_STAGES); it < issued; it++)
                if (!mbar_wait(q_full0 + 8 * (it % MT_STAGES), (it / MT_STAGES) & 1)) atomicExch(error_flag, 62);
            if (!mbar_wait(k_full, 0)) atomicExch(error_flag, 62);
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer: the warp waits, one lane issues
        constexpr uint32_t idesc = instr_desc_bf16_mn(128, 128);
        const uint64_t k_desc = smem_desc_sw128(smem_base), q_desc = smem_desc_sw128(q_smem);     // a step along a tile adds its bytes / 16
        bool alive = n_it > 0;
        if (alive && !__all_sync(0xffffffffu, mbar_wait(k_full, 0))) {
            atomicExch(error_flag, 63);
            alive = false;
        }
        for (int it = 0; it < n_it && alive; it++) {
            const int s = it % MT_STAGES, sb = it & 1;
            if (!__all_sync(0xffffffffu, mbar_wait(q_full0 + 8 * s, (it / MT_STAGES) & 1) && mbar_wait(s_empty0 + 8 * sb, ((it >> 1) & 1) ^ 1))) {
                atomicExch(error_flag, 64);
                break;
            }
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk++) {
                        if (kk * 16 >= hd) break;
                        const uint32_t off = (kk >> 2) * FA_HALF_BYTES + (kk & 3) * 32;
                        umma_bf16(tmem_base + (2 * sb + k) * 128, k_desc + ((k * TILE + off) >> 4), q_desc + ((s * TILE + off) >> 4), idesc,
                                  kk ? 1u : 0u);
                    }
                umma_commit(q_empty0 + 8 * s);
                umma_commit(s_full0 + 8 * sb);
            }
            __syncwarp();
        }
    } else {
        // ---------------------------------------------------------------- weights
        const int w = warp - 2, k = w >> 3;                    // key tile
        const int quarter = warp & 3, r = quarter * 32 + lane;  // key of the tile = lane of tensor memory (a warp reads its own quarter)
        const int hf = (w >> 2) & 1;                           // which 64 queries of a tile
        const int key = key0 + k * 128 + r;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const f32x2 scale2 = pair_of(scale_log2e, scale_log2e);
        f32x2 sum[4] = {0ull, 0ull, 0ull, 0ull};
        bool ok = true;
        for (int it = 0; it < n_it; it++) {
            const int sb = it & 1, s = it % MT_STAGES;
            // (the queries' barrier too: it says that the log-sums have arrived)
            if (!__all_sync(0xffffffffu, mbar_wait(s_full0 + 8 * sb, (it >> 1) & 1) && mbar_wait(q_full0 + 8 * s, (it / MT_STAGES) & 1))) {
                atomicExch(error_flag, 65);
                ok = false;
                break;
            }
            tc_fence_after();
            const int q0 = n0 + ((it0 + it) % blocks) * 128 + hf * 64;       // this thread's first query
            const int c_lo = key - pos0 - q0;                  // its queries [c_lo, c_hi] see the key
            int c_hi = n1 - 1 - q0;
            if (window > 0) c_hi = (int)min((long long)c_hi, (long long)key + window - 1 - pos0 - q0);
            const uint32_t tm_s = tmem_base + (2 * sb + k) * 128 + lane_base + hf * 64;
#pragma unroll
            for (int part = 0; part < 2; part++) {
                float sv[32];
                tmem_ld32(tm_s + part * 32, sv);
                if (part == 1) {
                    tc_fence_before();
                    if (lane == 0) mbar_arrive(s_empty0 + 8 * sb);           // all scores have been read (the load is the warp's)
                }
                const float4* ls = reinterpret_cast<const float4*>(xlse + s * 128 + hf * 64 + part * 32);
                const int lo = c_lo - part * 32, hi = c_hi - part * 32;
                if (lo <= 0 && hi >= 31) {
#pragma unroll
                    for (int c = 0; c < 32; c += 4) {
                        const float4 l4 = ls[c >> 2];
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const f32x2 x = pair_fma(pair_of(sv[c + 2 * u], sv[c + 2 * u + 1]), scale2, pair_of(u ? l4.z : l4.x, u ? l4.w : l4.y));
                            const int pair = (c >> 1) + u;     // 0..15
                            float a, d;
                            if ((pair & 7) == 4) {
                                exp2_pair<5>(x, a, d);
                            } else {
                                pair_parts(x, a, d);
                                a = exp2_approx(a);
                                d = exp2_approx(d);
                            }
                            sum[pair & 3] = pair_add(sum[pair & 3], pair_of(a, d));
                        }
                    }
                } else if (lo <= 31 && hi >= 0) {              // the causal diagonal, the window's edge, the last queries
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        const float a = c >= lo && c <= hi ? exp2_approx(fmaf(sv[c], scale_log2e, xlse[s * 128 + hf * 64 + part * 32 + c])) : 0.0f;
                        const float d = c + 1 >= lo && c + 1 <= hi ? exp2_approx(fmaf(sv[c + 1], scale_log2e,
                                                                                      xlse[s * 128 + hf * 64 + part * 32 + c + 1])) : 0.0f;
                        sum[(c >> 1) & 3] = pair_add(sum[(c >> 1) & 3], pair_of(a, d));
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(q_empty0 + 8 * s);      // and all log-sums
        }
        float a, d;
        pair_parts(pair_add(pair_add(sum[0], sum[1]), pair_add(sum[2], sum[3])), a, d);
        const float mine = a + d;
        if (hf == 1) xsum[k * 128 + r] = mine;
        asm volatile("bar.sync 2, 512;" ::: "memory");
        if (hf == 0 && has_work && ok) {
            const int pi = key / HB_PAGE_TOKENS;
            const int page = pi < pt_width ? page_table[(size_t)b * pt_width + pi] : -1;
            mass_store(mo, mine + xsum[k * 128 + r], b, g, key, page, nkv, n_pages, pos0, n_new, z, S, (size_t)tile * MT_KEYS + k * 128 + r,
                       (size_t)(gridDim.x / (S * nkv)) * MT_KEYS);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

template <int HD>
static int launch_mass_tc(const CUtensorMap& mq, const CUtensorMap& mk, const int* page_table, int pt_width, const int* seq_start,
                          const int* seq_pos0, const float* lse, long long lse_ld, MassOut mo, int splits, int n_seqs, int key_tiles, int nh,
                          int nkv, int hd, float scale, int window, int n_pages, int* error_flag, cudaStream_t s) {
    constexpr int SMEM = (2 + MT_STAGES) * (HD / 64) * FA_HALF_BYTES + (MT_STAGES * 128 + 256) * 4 + 16 * 8 + 16 + 1024;
    static_assert(SMEM <= 227 * 1024, "key and query tiles do not fit shared memory");
    static bool done[HB_MAX_DEVICES] = {};
    bool& set = done[hb_device_slot()];
    if (!set) {
        cudaError_t e = cudaFuncSetAttribute(mass_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return hb_fail("attention_mass_tc: cannot reserve %d bytes of shared memory: %s", SMEM, cudaGetErrorString(e));
        set = true;
    }
    cudaError_t e = hb_launch(mass_tc_kernel<HD>, dim3(key_tiles * nkv * splits), dim3(MT_THREADS), SMEM, s, mq, mk, page_table, pt_width, seq_start,
                              seq_pos0, lse, lse_ld, mo, n_seqs, nh, nkv, hd, scale * FA_LOG2E, window, n_pages, splits, error_flag);
    if (e != cudaSuccess) return hb_fail("attention_mass_tc: launch failed: %s", cudaGetErrorString(e));
    return hb_check_launch("attention_mass_tc");
}

extern "C" int hb_attention_mass_tc_keys(void) { return MT_KEYS; }

// Steps of many tokens (HbMassMany in api.h), bfloat16, sizes of hb_attention_mass_tc_supported, queries and output with 16-byte aligned
// rows: blocks of queries as attention_chunk_tc (attention_mass.cuh), tiles of 256 keys.
extern "C" int hb_attention_mass_tc(const HbMassMany* a, int fields, float scale) {
    HB_REQUIRE(fields * sizeof(long long) == sizeof(*a), "attention_mass: %d fields given", fields);
    const int n_tokens = (int)a->n_tokens, n_seqs = (int)a->n_seqs, n_heads = (int)a->n_heads, n_kv_heads = (int)a->n_kv_heads, hd = (int)a->head_dim;
    const int splits = (int)a->splits, n_pages = (int)a->n_pages, pt_width = (int)a->pt_width, key_tiles = (int)a->key_tiles, window = (int)a->window;
    if (n_seqs == 0 || n_tokens == 0) return 0;
    HB_REQUIRE(((uintptr_t)a->lse & 15) == 0 && a->lse_ld % 128 == 0, "attention_mass: the log-sums must be aligned");
    HB_REQUIRE(a->dtype == HB_BF16 && a->lse != nullptr && a->mass != nullptr && n_kv_heads > 0 && n_kv_heads <= 65535 && key_tiles > 0 && splits >= 1 &&
                   (long long)key_tiles * n_kv_heads * splits <= 0x7fffffffLL && (splits == 1 || a->parts != nullptr),
               "attention_mass: bad sizes");
    cudaStream_t s = (cudaStream_t)a->stream;
    if (attention_chunk_tc(a->q, a->q_stride, a->k_cache, a->v_cache, a->page_table, pt_width, a->seq_start, a->seq_pos0, a->out, a->out_stride, a->lse,
                           a->lse_ld, a->chunk_parts, (int)a->max_shares, (int)a->share_tiles, (int)a->join_tokens, n_tokens, n_seqs, (int)a->q_blocks,
                           n_heads, n_kv_heads, hd, scale, window, n_pages, a->status, s))
        return 1;
    CUtensorMap mq, mk;
    if (tc_make_map_heads(&mq, a->q, n_tokens, n_heads, hd, a->q_stride, 128)) return 1;
    if (tc_make_map(&mk, a->k_cache, (long long)n_pages * n_kv_heads * HB_PAGE_TOKENS, hd, hd, HB_PAGE_TOKENS)) return 1;
    MassOut mo = {a->before, a->mass, a->parts};
#define HB_MT_LAUNCH(HD)                                                                                                                   \
    launch_mass_tc<HD>(mq, mk, a->page_table, pt_width, a->seq_start, a->seq_pos0, a->lse, a->lse_ld, mo, splits, n_seqs, key_tiles, n_heads, \
                       n_kv_heads, hd, scale, window, n_pages, a->status, s)
    const int rc = hd > 64 ? HB_MT_LAUNCH(128) : HB_MT_LAUNCH(64);
#undef HB_MT_LAUNCH
    if (rc) return rc;
    return splits > 1 ? mass_join(a->page_table, pt_width, a->seq_start, a->seq_pos0, mo, n_seqs, n_kv_heads, n_pages, MT_KEYS, key_tiles, splits, s) : 0;
}
