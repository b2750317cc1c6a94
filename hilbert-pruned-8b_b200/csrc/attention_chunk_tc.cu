// Attention of a chunk of new tokens over the paged cache on the 5th-generation tensor cores (tcgen05 + TMEM + TMA), bfloat16, head
// sizes up to 128 in steps of 8, that leaves each row's log-sum, negated, for the weights' kernel (attention_mass_tc.cu): causal,
// grouped, with a window, sequences with unequal numbers of new tokens, the keys cut into shares where there are few rows.
//
// One CTA = two tiles of 128 query rows that read the same keys and values: two heads of a kv head with an even group, else two
// neighbouring blocks of one head's tokens.  A tile's rows are the 128 lanes of tensor memory.  What bounds it, per 128 x 128 scores at
// head size 128: 1024 clocks of the two products, 1024 clocks of exponentials (16 a clock and SM), and 64 KB of keys and values, which at the
// 32 bytes a clock that an SM takes from L2 would last 2048 clocks for one tile: hence two tiles, which halve that, and which take turns:
// while one tile's weights are made, the tensor cores work on the other.  Measured: 901 us for 2048 tokens behind 30001 rows, 32 heads over 8
// (1.16 PFLOP/s; with one tile to a CTA 1348 us); the products alone, with the same loads and hand-overs, took 832 of then 892: a tile's chain
// of products, softmax and hand-overs bounds it.
//   warps 0-3, 4-7  softmax of tile 0 and 1, a thread per row: 128 scores from tensor memory into registers, running maximum and sum in
//                   float32, weights as bfloat16, handed over in two halves.  No exchange between threads (two threads per row, which agree
//                   on the maximum through shared memory: 2.09 instead of 1.77 us for the two tiles at head size 128, 1.73 instead of 1.62 at
//                   64).  The output accumulator is rescaled only when a row's maximum grows by more than 2^8 (weights are taken against a
//                   maximum that may be stale by less).
//   warp 8          TMA producer: the query tiles once, then key and value tiles of 128 rows (two pages), two stages each
//   warp 9          owns tensor memory; one thread issues, per key tile and in this order: O0 += P0 V, S0 = Q0 K' (the next keys),
//                   O1 += P1 V, S1 = Q1 K'; with head size 64, whose weights do not lie over the scores, a tile's S before its O.
// Built for tiles of HD = 64 and 128 columns; a smaller head size hd has the rest of its tiles filled with zeros by the copies.
// Weights are rounded to bfloat16 for the product with the values (the sum they are divided by is taken before that).
//
// Every wait is bounded; a wait that runs out sets *error_flag and the CTA drains and leaves.
#include "api.h"
#include "attention_mass.cuh"
#include "attention_tc.cuh"
#include "exp2_pair.cuh"

#define CT_THREADS 320
#define CT_STAGES 2

// The weights 2^(s scale log2(e) - m) of 64 scores of a row, as bfloat16 over the scores, and their sum.  POLY: an eighth of the pairs on
// the FMA pipe (a masked score has to give exactly zero, which only the special-function unit does).
template <bool POLY>
__device__ __forceinline__ void chunk_weights(const float* sv, f32x2 scale2, f32x2 neg2, uint32_t tm_p, f32x2 (&sum)[2]) {
#pragma unroll
    for (int c = 0; c < 2; c++) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const f32x2 x = pair_fma(pair_of(sv[c * 32 + 2 * e], sv[c * 32 + 2 * e + 1]), scale2, neg2);
            float a, d;
            if (POLY && (e & 7) == 2) {
                exp2_pair<4>(x, a, d);
            } else {
                pair_parts(x, a, d);
                a = exp2_approx(a);
                d = exp2_approx(d);
            }
            sum[e & 1] = pair_add(sum[e & 1], pair_of(a, d));
            pk[e] = pack_bf16_pair(a, d);
        }
        tmem_st16u(tm_p + c * 16, pk);                         // P over S
    }
}

template <int HD>
__global__ void __launch_bounds__(CT_THREADS, 1)
chunk_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const int* __restrict__ page_table, int pt_width, const int* __restrict__ seq_start, const int* __restrict__ seq_pos0,
                bf16* __restrict__ out, long long out_stride, float* __restrict__ lse, long long lse_ld, Shares sh, int n_tokens, int n_seqs, int nh,
                int nkv, int hd, int head_pairs, float scale_log2e, int window, int n_pages, int* __restrict__ error_flag) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    // [Q tiles 2][K stages][V stages][barriers]; a tile is 128 rows x HD
    constexpr int HALVES = HD / 64, TILE = HALVES * FA_HALF_BYTES;
    uint64_t* bars = (uint64_t*)(smem + (2 + 2 * CT_STAGES) * TILE);
    uint32_t* tmem_slot = (uint32_t*)(bars + 22);
    const uint32_t smem_base = smem_u32(smem), k_smem = smem_base + 2 * TILE, v_smem = k_smem + CT_STAGES * TILE;
    const uint32_t q_full = smem_u32(bars), k_full0 = smem_u32(bars + 1), k_empty0 = smem_u32(bars + 3), v_full0 = smem_u32(bars + 5),
                   v_empty0 = smem_u32(bars + 7), s_full0 = smem_u32(bars + 9), p_full0 = smem_u32(bars + 11), pv_done0 = smem_u32(bars + 15),
                   s_free0 = smem_u32(bars + 17);              // p_full: [2 tiles][2 halves of the keys]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    mass_fresh(page_table, seq_start, seq_pos0);

    // The two tiles: heads head0 and head0 + 1 (head_pairs) of one block of tokens, or blocks 2 blk and 2 blk + 1 of head0.  Blocks
    // are taken from the back and heads are the fast index: a sequence's blocks that see the most keys start first.  Sequences start in
    // the opposite of the step's order, whatever they see (seven ragged sequences: 118 us with the longest last, 140 the other way round).
    const int z = blockIdx.z;
    const int head0 = head_pairs ? 2 * blockIdx.x : blockIdx.x, g = head0 / (nh / nkv);
    const int span = head_pairs ? FA_ROWS : 2 * FA_ROWS;
    int b, blk, place0;
    const bool has_work = mass_find_block(seq_start, n_seqs, gridDim.y - 1 - blockIdx.y, span, b, blk, place0);
    const int t_begin = mass_uniform(has_work ? seq_start[b] : 0), n_new = mass_uniform(has_work ? seq_start[b + 1] - t_begin : 1),
              pos0 = mass_uniform(has_work ? seq_pos0[b] : 0);
    const int row0 = blk * span;                               // the first of the CTA's new tokens
    const int first_pos = pos0 + row0, last_pos = pos0 + min(row0 + span, n_new) - 1;
    int jt0, n_it = key_tiles_of(first_pos, last_pos, window, FA_KEYS, jt0);
    const int S = shares_of(sh, n_it), lo_cta = hb_oldest_visible(first_pos, window, 0);
    if (!has_work || z >= S) return;
    {                                                          // this share's tiles of keys (none is empty: S <= n_it)
        const int a = (int)((long long)n_it * z / S), e = (int)((long long)n_it * (z + 1) / S);
        jt0 += a;
        n_it = e - a;
    }

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int s = 0; s < 2; s++) {
            mbar_init(k_full0 + 8 * s, 1);
            mbar_init(k_empty0 + 8 * s, 1);
            mbar_init(v_full0 + 8 * s, 1);
            mbar_init(v_empty0 + 8 * s, 1);
            mbar_init(s_full0 + 8 * s, 1);
            mbar_init(p_full0 + 16 * s, 4);
            mbar_init(p_full0 + 16 * s + 8, 4);
            mbar_init(pv_done0 + 8 * s, 1);
            mbar_init(s_free0 + 8 * s, 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 9) tmem_alloc(smem_u32(tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // S0, S1 at columns 0 and 128; head size 128: O0, O1 at 256 and 384, P over S; 64: O0, O1 at 256 and 320, P0, P1 at 384 and 448, so that
    // the next scores can be computed as soon as these have been read
    constexpr bool APART = HD == 64;
    const uint32_t tmem_base = *tmem_slot;
    pdl_trigger();

    if (warp == 8) {
        // ---------------------------------------------------------------- TMA producer
        if (lane == 0) {
            const int* pt = page_table + (size_t)b * pt_width;
            mbar_expect_tx(q_full, 2 * TILE);
            for (int i = 0; i < 2; i++)
                for (int half = 0; half < HALVES; half++)
                    tma_load_3d(smem_base + i * TILE + half * FA_HALF_BYTES, &map_q, q_full, half * 64, head0 + (head_pairs ? i : 0),
                                t_begin + row0 + (head_pairs ? 0 : i * FA_ROWS));
            // the pages of tile `it` of the keys and the values: both numbers asked for at once, a tile ahead
            int page[2], next_page[2];
            auto ask = [&](int it) {
#pragma unroll
                for (int pg = 0; pg < 2; pg++) {
                    const int pi = (jt0 + it) * 2 + pg;
                    next_page[pg] = it < n_it && pi < pt_width ? pt[pi] : -1;
                }
            };
            auto take = [&](int it) {
#pragma unroll
                for (int pg = 0; pg < 2; pg++) {
                    const int pi = (jt0 + it) * 2 + pg;
                    page[pg] = next_page[pg];
                    if (page[pg] < 0 || page[pg] >= n_pages) {
                        // a page behind the last row's key or in front of the oldest that the first row sees may be missing
                        if (page[pg] >= n_pages || (pi >= lo_cta / HB_PAGE_TOKENS && pi <= last_pos / HB_PAGE_TOKENS))
                            hb_note(error_flag, HB_STATUS_PAGE, 1 + b);
                        page[pg] = 0;                               // never read outside the cache
                    }
                }
            };
            auto load_tile = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar) {
                mbar_expect_tx(bar, TILE);
#pragma unroll
                for (int pg = 0; pg < 2; pg++)
                    for (int half = 0; half < HALVES; half++)
                        tma_load_2d(dst + half * FA_HALF_BYTES + pg * (FA_HALF_BYTES / 2), map, bar, half * 64, (page[pg] * nkv + g) * HB_PAGE_TOKENS);
            };
            ask(0);
            int k_issued = 0, v_issued = 0;
            for (int it = 0; it < n_it; it++) {
                const int s = it % CT_STAGES;
                take(it);
                ask(it + 1);
                if (!mbar_wait(k_empty0 + 8 * s, ((it / CT_STAGES) & 1) ^ 1)) {
                    atomicExch(error_flag, 51);
                    break;
                }
                load_tile(k_smem + s * TILE, &map_k, k_full0 + 8 * s);
                k_issued = it + 1;
                if (!mbar_wait(v_empty0 + 8 * s, ((it / CT_STAGES) & 1) ^ 1)) {
                    atomicExch(error_flag, 52);
                    break;
                }
                load_tile(v_smem + s * TILE, &map_v, v_full0 + 8 * s);
                v_issued = it + 1;
            }
            for (int it = max(0, k_issued - CT_STAGES); it < k_issued; it++)
                if (!mbar_wait(k_full0 + 8 * (it % CT_STAGES), (it / CT_STAGES) & 1)) atomicExch(error_flag, 53);
            for (int it = max(0, v_issued - CT_STAGES); it < v_issued; it++)
                if (!mbar_wait(v_full0 + 8 * (it % CT_STAGES), (it / CT_STAGES) & 1)) atomicExch(error_flag, 53);
            if (!mbar_wait(q_full, 0)) atomicExch(error_flag, 53);
        }
    } else if (warp == 9) {
        // ---------------------------------------------------------------- MMA issuer: the warp waits, one lane issues
        constexpr uint32_t idesc_qk = instr_desc_bf16_mn(128, FA_KEYS);
        constexpr uint32_t idesc_pv = instr_desc_bf16_mn(128, HD) | (1u << 16);               // B is MN-major
        // descriptors of the tiles' beginnings; a step along a tile adds its bytes / 16
        const uint64_t q_desc = smem_desc_sw128(smem_base), k_desc = smem_desc_sw128(k_smem), v_desc = smem_desc_mn_sw128(v_smem, FA_HALF_BYTES,
                                                                                                                          1024);
        auto scores = [&](int i, int it) {
            const int st = it % CT_STAGES;
#pragma unroll
            for (int kk = 0; kk < HD / 16; kk++) {
                if (kk * 16 >= hd) break;
                const uint32_t off = (kk >> 2) * FA_HALF_BYTES + (kk & 3) * 32;
                umma_bf16(tmem_base + i * 128, q_desc + ((i * TILE + off) >> 4), k_desc + ((st * TILE + off) >> 4), idesc_qk, kk ? 1u : 0u);
            }
            umma_commit(s_full0 + 8 * i);
            if (i == 1) umma_commit(k_empty0 + 8 * st);
        };
        bool alive = __all_sync(0xffffffffu, mbar_wait(q_full, 0) && mbar_wait(k_full0, 0));
        tc_fence_after();
        if (alive && elect_one()) {
            scores(0, 0);
            scores(1, 0);
        }
        __syncwarp();
        for (int it = 0; it < n_it && alive; it++) {
            const int sv = it % CT_STAGES;
            const bool more = it + 1 < n_it;
            const uint32_t next_k = k_full0 + 8 * ((it + 1) % CT_STAGES), next_parity = ((it + 1) / CT_STAGES) & 1;
#pragma unroll
            for (int i = 0; i < 2 && alive; i++) {
                if (APART && more) {                           // the next scores, once the softmax has these in registers
                    alive = __all_sync(0xffffffffu, mbar_wait(s_free0 + 8 * i, it & 1) && (i > 0 || mbar_wait(next_k, next_parity)));
                    if (!alive) break;
                    tc_fence_after();
                    if (elect_one()) scores(i, it + 1);
                    __syncwarp();
                }
#pragma unroll
                for (int half = 0; half < 2; half++) {         // the weights of a tile's first 64 keys, then the others
                    alive = alive && __all_sync(0xffffffffu, mbar_wait(p_full0 + 16 * i + 8 * half, it & 1) &&
                                                                 (i + half > 0 || mbar_wait(v_full0 + 8 * sv, (it / CT_STAGES) & 1)) &&
                                                                 (APART || i > 0 || half == 0 || !more || mbar_wait(next_k, next_parity)));
                    if (!alive) break;
                    tc_fence_after();
                    const int kbase = (jt0 + it) * FA_KEYS;
                    if (i + half == 0 && (kbase < lo_cta || kbase + FA_KEYS > pos0 + n_new)) {
                        // The tile that holds the sequence's end, or begins in front of the window: the values there are whatever a
                        // page held before, or of a page that was given back, and 0 * NaN is NaN.
                        const int from = lo_cta - kbase, to = pos0 + n_new - kbase;          // rows [from, to) stay; 128 bytes in each half
                        for (int u = lane; u < FA_KEYS * 8 * HALVES; u += 32) {
                            const int vr = u / (8 * HALVES), c = u % (8 * HALVES);
                            if (vr < from || vr >= to)
                                *reinterpret_cast<uint4*>(smem + (2 + CT_STAGES + sv) * TILE + (c >> 3) * FA_HALF_BYTES + vr * 128 + (c & 7) * 16) =
                                    make_uint4(0u, 0u, 0u, 0u);
                        }
                        fence_async_shared();                  // before the tensor core reads them
                        __syncwarp();
                    }
                    if (elect_one()) {
#pragma unroll
                        for (int kk = half * 4; kk < half * 4 + 4; kk++)
                            umma_bf16_ts(tmem_base + 256 + i * HD, tmem_base + (APART ? 384 + i * 64 : i * 128) + kk * 8,
                                         v_desc + ((sv * TILE + kk * 16 * 128) >> 4), idesc_pv, (it | kk) ? 1u : 0u);
                        if (half == 1) {
                            if (i == 1) umma_commit(v_empty0 + 8 * sv);
                            if (!APART && more) scores(i, it + 1);
                            if (APART || !more) umma_commit(pv_done0 + 8 * i);
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (!alive) atomicExch(error_flag, 55);
    } else {
        // ---------------------------------------------------------------- softmax and output: a thread per row
        const int i = warp >> 2, r = (warp & 3) * 32 + lane;   // tile, row = lane of tensor memory
        const int head = head0 + (head_pairs ? i : 0), row = row0 + (head_pairs ? 0 : i * FA_ROWS) + r;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tm_s = tmem_base + i * 128 + lane_base, tm_o = tmem_base + 256 + i * HD + lane_base;
        const uint32_t tm_p = APART ? tmem_base + 384 + i * 64 + lane_base : tm_s;
        const int qpos = pos0 + row, lo = hb_oldest_visible(qpos, window, 0);
        const bool valid = row < n_new;
        const f32x2 scale2 = pair_of(scale_log2e, scale_log2e);
        float m_run = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int it = 0; it < n_it; it++) {
            if (!__all_sync(0xffffffffu, mbar_wait(s_full0 + 8 * i, it & 1))) {
                atomicExch(error_flag, 56);
                ok = false;
                break;
            }
            tc_fence_after();
            float sv[128];
            tmem_ld64(tm_s, sv);
            tmem_ld64(tm_s + 64, sv + 64);
            if (APART) {
                tc_fence_before();
                if (lane == 0) mbar_arrive(s_free0 + 8 * i);   // the warp's scores are in registers (the load is the warp's)
            }
            // this row sees keys lo..qpos; as columns of the tile: [c_lo, c_hi]
            const int kbase = (jt0 + it) * FA_KEYS, c_lo = lo - kbase, c_hi = qpos - kbase;
            const bool edge = __any_sync(0xffffffffu, c_lo > 0 || c_hi < 127);      // the causal diagonal or the window's edge
            if (edge) {
#pragma unroll
                for (int e = 0; e < 128; e++)
                    if (e < c_lo || e > c_hi) sv[e] = -INFINITY;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 128; e += 8) {
#pragma unroll
                for (int u = 0; u < 4; u++) mx[u] = fmaxf(mx[u], fmaxf(sv[e + u], sv[e + 4 + u]));
            }
            const float m_tile = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale_log2e;
            if (APART && it > 0) {                             // the product before: it reads the weights and writes the accumulator
                if (!__all_sync(0xffffffffu, mbar_wait(pv_done0 + 8 * i, (it - 1) & 1))) {
                    atomicExch(error_flag, 59);
                    ok = false;
                    break;
                }
                tc_fence_after();
            }
            if (it == 0) {
                m_run = m_tile;
            } else {
                const bool grow = m_tile > m_run + FA_RESCALE_THRESHOLD;
                if (__any_sync(0xffffffffu, grow)) {
                    // nothing touches the accumulator now (P over S: S of this tile is complete, so is every product issued before it)
                    const float m_new = fmaxf(m_run, m_tile);
                    const float corr = m_new == -INFINITY ? 1.0f : exp2f(m_run - m_new);
                    m_run = m_new;
                    l *= corr;
#pragma unroll 1
                    for (int c = 0; c < HD / 16; c++) {
                        float v[16];
                        tmem_ld16(tm_o + c * 16, v);
                        uint32_t u[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) u[e] = __float_as_uint(v[e] * corr);
                        tmem_st16u(tm_o + c * 16, u);
                    }
                    tmem_wait_st();
                }
            }
            const float neg_m = m_run == -INFINITY ? 0.0f : -m_run;
            f32x2 sum[2] = {0ull, 0ull};
            const f32x2 neg2 = pair_of(neg_m, neg_m);
#pragma unroll
            for (int half = 0; half < 2; half++) {
                if (edge) chunk_weights<false>(sv + 64 * half, scale2, neg2, tm_p + half * 32, sum);
                else chunk_weights<true>(sv + 64 * half, scale2, neg2, tm_p + half * 32, sum);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full0 + 16 * i + 8 * half);       // one arrival a warp: arrivals of single threads queue up
            }
            float s0, s1;
            pair_parts(pair_add(sum[0], sum[1]), s0, s1);
            l += s0 + s1;
        }
        const size_t at = ((size_t)z * nh + head) * n_tokens + t_begin + row;
        if (ok && !__all_sync(0xffffffffu, mbar_wait(pv_done0 + 8 * i, APART ? (n_it - 1) & 1 : 0))) {
            atomicExch(error_flag, 58);
            ok = false;
        }
        if (ok) {
            tc_fence_after();
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            if (valid) {
                if (S > 1) *reinterpret_cast<float2*>(sh.ml + at * 2) = make_float2(m_run, l);
                else lse[head * lse_ld + place0 + row] = l > 0.0f ? -(m_run + log2f(l)) : -INFINITY;
            }
            bf16* dst = out + (size_t)(t_begin + row) * out_stride + (size_t)head * hd;
            float4* po = reinterpret_cast<float4*>(sh.o + at * hd);
#pragma unroll 1
            for (int c = 0; c * 32 < hd; c++) {
                float v[32];
                tmem_ld32(tm_o + c * 32, v);
                if (!valid) continue;
                if (S > 1) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        if (c * 32 + e < hd) po[c * 8 + (e >> 2)] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        if (c * 32 + e >= hd) break;
                        uint4 o4;
                        o4.x = pack_bf16_pair(v[e] * inv, v[e + 1] * inv);
                        o4.y = pack_bf16_pair(v[e + 2] * inv, v[e + 3] * inv);
                        o4.z = pack_bf16_pair(v[e + 4] * inv, v[e + 5] * inv);
                        o4.w = pack_bf16_pair(v[e + 6] * inv, v[e + 7] * inv);
                        *reinterpret_cast<uint4*>(dst + c * 32 + e) = o4;
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

template <int HD>
static int launch_chunk(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const int* page_table, int pt_width,
                        const int* seq_start, const int* seq_pos0, bf16* out, long long out_stride, float* lse, long long lse_ld, Shares sh,
                        int max_shares, int n_tokens, int n_seqs, int q_blocks, int nh, int nkv, int hd, int head_pairs, float scale, int window,
                        int n_pages, int* error_flag, cudaStream_t s) {
    constexpr int SMEM = (2 + 2 * CT_STAGES) * (HD / 64) * FA_HALF_BYTES + 22 * 8 + 16 + 1024;
    static_assert(SMEM <= 227 * 1024, "attention tiles do not fit shared memory");
    static bool done[HB_MAX_DEVICES] = {};
    bool& set = done[hb_device_slot()];
    if (!set) {
        cudaError_t e = cudaFuncSetAttribute(chunk_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return hb_fail("attention_mass: cannot reserve %d bytes of shared memory: %s", SMEM, cudaGetErrorString(e));
        set = true;
    }
    cudaError_t e = hb_launch(chunk_tc_kernel<HD>, dim3(head_pairs ? nh / 2 : nh, q_blocks, max_shares), dim3(CT_THREADS), SMEM, s, mq, mk, mv,
                              page_table,
                              pt_width, seq_start, seq_pos0, out, out_stride, lse, lse_ld, sh, n_tokens, n_seqs, nh, nkv, hd, head_pairs,
                              scale * FA_LOG2E, window, n_pages, error_flag);
    if (e != cudaSuccess) return hb_fail("attention_mass: launch failed: %s", cudaGetErrorString(e));
    return hb_check_launch("attention_mass (chunk)");
}

extern "C" int hb_attention_mass_tc_supported(int n_heads, int n_kv_heads, int head_dim) {
    return head_dim > 0 && head_dim <= 128 && head_dim % 8 == 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0;
}

int attention_chunk_tc(const void* q, long long q_stride, const void* k_cache, const void* v_cache, const int* page_table, int pt_width,
                       const int* seq_start, const int* seq_pos0, void* out, long long out_stride, float* lse, long long lse_ld, float* parts,
                       int max_shares, int share_tiles, int join_tokens, int n_tokens, int n_seqs, int q_blocks, int n_heads, int n_kv_heads,
                       int head_dim, float scale, int window, int n_pages, int* error_flag, cudaStream_t s) {
    HB_REQUIRE(hb_attention_mass_tc_supported(n_heads, n_kv_heads, head_dim),
               "attention_mass: %d heads over %d of size %d are not built for the tensor cores (sizes up to 128 in steps of 8)", n_heads, n_kv_heads, head_dim);
    HB_REQUIRE(q_blocks > 0 && q_blocks <= 65535 && error_flag != nullptr && max_shares >= 1 && max_shares <= 32 && share_tiles >= 1 &&
                   (max_shares == 1 || parts != nullptr),
               "attention_mass: the step is too large for one launch");
    HB_REQUIRE(q_stride % 8 == 0 && ((uintptr_t)q & 15) == 0, "attention_mass: queries must have 16-byte aligned rows");
    HB_REQUIRE(out_stride % 8 == 0 && ((uintptr_t)out & 15) == 0, "attention_mass: output must have 16-byte aligned rows");
    HB_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0, "attention_mass: cache must be 16-byte aligned");
    CUtensorMap mq, mk, mv;
    const long long cache_rows = (long long)n_pages * n_kv_heads * HB_PAGE_TOKENS;
    HB_REQUIRE(cache_rows <= 0x7fffffffLL, "attention_mass: the cache has too many rows for a tensor map");
    if (tc_make_map_heads(&mq, q, n_tokens, n_heads, head_dim, q_stride, FA_ROWS)) return 1;
    if (tc_make_map(&mk, k_cache, cache_rows, head_dim, head_dim, HB_PAGE_TOKENS)) return 1;
    if (tc_make_map(&mv, v_cache, cache_rows, head_dim, head_dim, HB_PAGE_TOKENS)) return 1;
    const int head_pairs = (n_heads / n_kv_heads) % 2 == 0;
    // one share: no block is cut, whatever it sees
    const Shares sh = {parts, parts == nullptr ? nullptr : parts + (size_t)max_shares * n_heads * n_tokens * head_dim,
                       max_shares == 1 ? 0x3fffffff : share_tiles};
    const int rc = head_dim > 64 ? launch_chunk<128>(mq, mk, mv, page_table, pt_width, seq_start, seq_pos0, (bf16*)out, out_stride, lse, lse_ld, sh,
                                                       max_shares, n_tokens, n_seqs, q_blocks, n_heads, n_kv_heads, head_dim, head_pairs, scale,
                                                       window, n_pages,
                                                       error_flag, s)
                                   : launch_chunk<64>(mq, mk, mv, page_table, pt_width, seq_start, seq_pos0, (bf16*)out, out_stride, lse, lse_ld, sh,
                                                      max_shares, n_tokens, n_seqs, q_blocks, n_heads, n_kv_heads, head_dim, head_pairs, scale,
                                                      window, n_pages, error_flag, s);
    if (rc || max_shares == 1) return rc;
    return shares_join(sh, join_tokens, HB_BF16, out, out_stride, lse, lse_ld, 1, seq_start, seq_pos0, head_pairs ? FA_ROWS : 2 * FA_ROWS, FA_KEYS,
                       window, n_tokens,
                       n_seqs, n_heads, head_dim, s);
}
