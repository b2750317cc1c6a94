// Eviction from the paged cache by accumulated attention weight: which rows of a sequence stay (evict_select), and their move
// to the front of its pages or into pages of their own (evict_rows).  Rows are chosen for every entry (layer), sequence and kv
// head alone: a kv head's attention reads its own rows only, and keys carry their rotation with them, so the rows of one page
// need not stand for the same tokens in every head.
#include <cooperative_groups.h>

#include "api.h"
#include "common.cuh"

namespace cg = cooperative_groups;

// ------------------------------------------------------------------------------------------------- which rows stay
// With n rows and budget c < n: the first `first`, the last `recent`, and of those between the c - first - recent with the
// largest mass (ties: the lower row).  A radix selection: the need-th largest value is found digit by digit (11, 11 and 10
// bits of the values' order-preserving integer form) from histograms in shared memory; the histogram of a later digit counts
// only the values whose digits so far are the chosen ones.  Then every warp counts what it keeps, one scan over the warps
// gives their places, and the rows are written in ascending order.
//
// What bounds it: the mass is read once (16 MB for 32 layers x 8 heads x 16384 rows: 2.6 us) and then lives in registers
// (ES_ITEMS values a thread); the rest is shared-memory atomics and barriers.  A warp owns a contiguous run of rows, so
// its loads are whole 128-byte lines and the ascending order needs one scan and no sort.  Rows longer than a block's registers
// are shared by a cluster of up to 8 blocks, which add their histograms through distributed shared memory; what does not fit
// 8 blocks' registers (above 262144 rows) is read again from L2 in every pass.
#define ES_ITEMS 32
#define ES_BINS 2048

// the value's place in the order of all values, 0 aside: that stands for a row that is not between the first and the last ones
__device__ __forceinline__ uint32_t es_key(float f) {
    const uint32_t u = __float_as_uint(f + 0.0f);         // -0 counts as 0
    const uint32_t k = u ^ (uint32_t)(((int32_t)u >> 31) | 0x80000000);
    return isnan(f) ? 1u : k;                             // below everything, -inf (0x007fffff) included
}

// bits [from, to) of 32
__device__ __forceinline__ uint32_t es_bits(int from, int to) {
    from = min(max(from, 0), 32);
    to = min(max(to, 0), 32);
    return from < to ? (0xffffffffu >> (32 - (to - from))) << from : 0u;
}

// sums over the warps in front of this one of two counts, and over all warps
template <int NW>
__device__ __forceinline__ void es_scan(int& a, int& b, int& all_a, int& all_b, int (*scratch)[NW], int warp, int lane) {
    if (lane == 0) {
        scratch[0][warp] = a;
        scratch[1][warp] = b;
    }
    __syncthreads();
    const int x = lane < NW ? scratch[0][lane] : 0, y = lane < NW ? scratch[1][lane] : 0;
    a = __reduce_add_sync(0xffffffffu, lane < warp ? x : 0);
    b = __reduce_add_sync(0xffffffffu, lane < warp ? y : 0);
    all_a = __reduce_add_sync(0xffffffffu, x);
    all_b = __reduce_add_sync(0xffffffffu, y);
}

template <int NT>
__global__ void __launch_bounds__(NT)
evict_select_kernel(const float* __restrict__ mass, const int* __restrict__ page_table, int pt_width, const int* __restrict__ lengths,
                    int* __restrict__ kept, int n_seqs, int nkv, int n_pages, int first, int recent, int budget, int* status) {
    constexpr int NW = NT / 32;
    __shared__ int hist[ES_BINS];
    __shared__ int sums[2][NW];
    __shared__ int totals[2];                             // this block's rows above the border, and at it
    __shared__ int chosen[3];                             // the digit, how many are wanted of what has it, and how many have it
    pdl_trigger();
    pdl_wait();
    mass = pdl_fresh(mass);
    page_table = pdl_fresh(page_table);
    lengths = pdl_fresh(lengths);
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int row = blockIdx.x / C;                       // (entry, sequence, kv head)
    const int g = row % nkv, b = (row / nkv) % n_seqs;
    const long long e = row / (nkv * n_seqs);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = min(max(lengths[b], 0), pt_width * HB_PAGE_TOKENS);
    if (tid == 0 && rank == 0 && n != lengths[b]) hb_note(status, HB_STATUS_PAGE, 1 + b);
    int* out = kept + (size_t)row * budget;
    if (n <= budget) {                                    // everything stays (the same for the whole cluster)
        for (int j = rank * NT + tid; j < budget; j += C * NT) out[j] = j < n ? j : -1;
        return;
    }
    const int* pt = page_table + (size_t)b * pt_width;
    const float* base = mass + ((size_t)e * n_pages * nkv + g) * HB_PAGE_TOKENS + lane;
    // rows [w_begin, w_begin + 32 * items) are this warp's, whole pages (an even number of 32 rows); row w_begin + 32 i + lane is
    // item i of this lane
    const int items = ((n + C * NT - 1) / (C * NT) + 1) & ~1;
    const int w_begin = (rank * NW + warp) * items * 32, r0 = w_begin + lane;
    const int mid_end = n - recent;
    const int need = budget - first - recent;
    auto item_of = [&](int r) { return (r - r0 + 31) >> 5; };             // the first item whose row is r or behind it

    // The warp's pages, 32 at a time, a lane each: all its values can then be asked for at once (with a look into the page table in
    // front of every two loads, 16384 rows in each of 256 lists took 6 us more than the 17.6 they take).  A missing page's rows have no mass.
    bool bad = false;
    const int first_page = w_begin / HB_PAGE_TOKENS;
    auto pages_from = [&](int at) -> int {                // this lane's page, the at + lane-th of the warp; -1: missing
        const int pi = first_page + at + lane;
        if (at + lane >= items / 2 || pi * HB_PAGE_TOKENS >= n) return 0;
        const int page = pt[pi];
        const bool held = page >= 0 && page < n_pages;
        bad |= !held;
        return held ? page : -1;
    };
    auto value = [&](int page, int half) -> float { return __ldcg(base + (size_t)max(page, 0) * nkv * HB_PAGE_TOKENS + half * 32); };
    uint32_t key[ES_ITEMS];
    const uint32_t middle = es_bits(item_of(first), min(items, item_of(mid_end)));
    {
        const int mine = pages_from(0);
        float x[ES_ITEMS];
#pragma unroll
        for (int i = 0; i < ES_ITEMS; i += 2) {
            x[i] = x[i + 1] = 0.0f;
            if (i < items) {
                const int page = __shfl_sync(0xffffffffu, mine, i / 2);
                x[i] = value(page, 0);
                x[i + 1] = value(page, 1);
            }
        }
        const uint32_t missing = __ballot_sync(0xffffffffu, mine < 0);
#pragma unroll
        for (int i = 0; i < ES_ITEMS; i++) key[i] = (middle >> i & 1u) ? es_key(x[i]) : 0u;
        if (missing != 0u) {                              // the host's fault: rare
#pragma unroll
            for (int i = 0; i < ES_ITEMS; i++)
                if ((missing >> (i / 2) & 1u) && key[i] != 0u) key[i] = 1u;
        }
    }
    // what the registers do not hold: the same key of item i >= ES_ITEMS, from memory
    auto far_key = [&](int i) -> uint32_t {
        const int r = r0 + i * 32;
        if (r < first || r >= mid_end) return 0u;
        const int page = pt[r / HB_PAGE_TOKENS];
        if (page < 0 || page >= n_pages) {
            bad = true;
            return 1u;
        }
        return es_key(value(page, i & 1));
    };

    uint32_t border = need > 0 ? 0u : 0xffffffffu;        // the need-th largest key; no key is as large as the other
    int want = need;                                      // of the keys that have the border's digits so far, how many stay
    if (need > 0) {
#pragma unroll
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
            const int bins = pass == 2 ? 1024 : 2048;
            for (int i = tid; i < ES_BINS; i += NT) hist[i] = 0;
            __syncthreads();
            auto count = [&](uint32_t k) {                // keys that agree with the border's digits so far
                if (k != 0u && (pass == 0 || ((k ^ border) >> (pass == 1 ? 21 : 10)) == 0u)) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
            };
#pragma unroll
            for (int i = 0; i < ES_ITEMS; i += 2)
                if (i < items) {
                    count(key[i]);
                    count(key[i + 1]);
                }
            for (int i = ES_ITEMS; i < items; i++) count(far_key(i));
            if (C > 1) cluster.sync();
            else __syncthreads();
            // bins from the top, PER per thread: thread t has bin bins - 1 - t * PER and the PER - 1 below it
            constexpr int PER = ES_BINS / NT;
            int mine[PER], sum = 0;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int bin = bins - 1 - (tid * PER + i);
                int c = 0;
                if (bin >= 0) {
                    if (C == 1) c = hist[bin];
                    else
                        for (int o = 0; o < C; o++) c += cluster.map_shared_rank(hist, o)[bin];
                }
                mine[i] = c;
                sum += c;
            }
            int inc = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += u;
            }
            int of_warp = __shfl_sync(0xffffffffu, inc, 31), none = 0, all, all_none;
            es_scan<NW>(of_warp, none, all, all_none, sums, warp, lane);
            int before = of_warp + inc - sum;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                if (before < want && before + mine[i] >= want) {
                    chosen[0] = bins - 1 - (tid * PER + i);
                    chosen[1] = want - before;
                    chosen[2] = mine[i];
                }
                before += mine[i];
            }
            if (C > 1) cluster.sync();                    // nobody still reads this block's histogram
            else __syncthreads();
            border |= (uint32_t)chosen[0] << shift;
            want = chosen[1];
            if (want == chosen[2]) {                      // all that have these digits stay: as good as a border just below them
                border -= 1u;
                want = 0;
                break;
            }
        }
    }
    // Rows that are not between stay, rows above the border stay, and the first `want` at it.  As bits of this lane's items.
    uint32_t stay = es_bits(0, min(items, item_of(n))) & ~middle, equal = 0u;
#pragma unroll
    for (int i = 0; i < ES_ITEMS; i++) {
        stay |= key[i] > border ? 1u << i : 0u;
        equal |= key[i] == border ? 1u << i : 0u;
    }
    int n_stay = __popc(stay), n_equal = __popc(equal);
    auto far_stays = [&](int i, uint32_t k) { return r0 + i * 32 < n && (k == 0u || k > border); };
    for (int i = ES_ITEMS; i < items; i++) {
        const uint32_t k = far_key(i);
        n_stay += far_stays(i, k) ? 1 : 0;
        n_equal += k == border ? 1 : 0;
    }
    n_stay = __reduce_add_sync(0xffffffffu, n_stay);
    n_equal = __reduce_add_sync(0xffffffffu, n_equal);
    const int equal_here = n_equal;
    int all_stay, all_equal;
    es_scan<NW>(n_stay, n_equal, all_stay, all_equal, sums, warp, lane);
    if (C > 1) {
        if (tid == 0) {
            totals[0] = all_stay;
            totals[1] = all_equal;
        }
        cluster.sync();
        for (int o = 0; o < rank; o++) {
            const int* t = cluster.map_shared_rank(totals, o);
            n_stay += t[0];
            n_equal += t[1];
        }
    }
    // n_stay, n_equal: how many stay, and how many lie at the border, in front of this warp's rows.  Does the limit for those at
    // the border fall inside this warp's rows?
    const uint32_t below = (1u << lane) - 1u;
    int at = n_stay + min(n_equal, want);
    if (n_equal >= want) {
        equal = 0u;
    } else if (n_equal + equal_here > want) {
        uint32_t in = 0u;
        int before = n_equal;
#pragma unroll
        for (int i = 0; i < ES_ITEMS; i++) {
            const uint32_t m = __ballot_sync(0xffffffffu, equal >> i & 1u);
            in |= (equal >> i & 1u) && before + __popc(m & below) < want ? 1u << i : 0u;
            before += __popc(m);
        }
        equal = in;
        n_equal = before;                                 // in front of item ES_ITEMS
    } else if (items > ES_ITEMS) {
        n_equal += (int)__reduce_add_sync(0xffffffffu, (uint32_t)__popc(equal));
    }
    stay |= equal;
#pragma unroll
    for (int i = 0; i < ES_ITEMS; i++) {
        if (i >= items) break;
        const uint32_t m = __ballot_sync(0xffffffffu, stay >> i & 1u);
        if (stay >> i & 1u) {
            const int j = at + __popc(m & below);
            if (j < budget) out[j] = r0 + i * 32;
        }
        at += __popc(m);
    }
    for (int i = ES_ITEMS; i < items; i++) {
        const uint32_t k = far_key(i);
        const bool up = far_stays(i, k), eq = k == border;
        const uint32_t me = __ballot_sync(0xffffffffu, eq);
        const bool in = up || (eq && n_equal + __popc(me & below) < want);
        const uint32_t m = __ballot_sync(0xffffffffu, in);
        if (in) {
            const int j = at + __popc(m & below);
            if (j < budget) out[j] = r0 + i * 32;
        }
        at += __popc(m);
        n_equal += __popc(me);
    }
    if (bad) hb_note(status, HB_STATUS_PAGE, 1 + b);
    if (C > 1) cluster.sync();                            // a block's totals stay readable until all have read them
}

template <int NT>
static int launch_select(int cluster, const float* mass, const int* page_table, int pt_width, const int* lengths, int* kept, int rows,
                         int n_seqs, int nkv, int n_pages, int first, int recent, int budget, int* status, cudaStream_t s) {
    cudaError_t e = hb_launch_clusters(evict_select_kernel<NT>, dim3(rows * cluster), dim3(NT), 0, s, (unsigned)cluster, mass, page_table,
                                       pt_width, lengths, kept, n_seqs, nkv, n_pages, first, recent, budget, status);
    if (e != cudaSuccess) return hb_fail("evict_select: launch failed: %s", cudaGetErrorString(e));
    return hb_check_launch("evict_select");
}

// mass: [entries][n_pages][n_kv_heads][64]; page_table: [n_seqs][pt_width]; lengths: rows of each sequence; kept:
// [entries][n_seqs][n_kv_heads][budget].  `threads` (512 or 1024) and `cluster` (1, 2, 4 or 8 blocks for one list of rows).
extern "C" int hb_evict_select(const float* mass, const int* page_table, int pt_width, const int* lengths, int* kept, int entries, int n_seqs,
                               int n_kv_heads, int n_pages, int first, int recent, int budget, int threads, int cluster, int* status,
                               void* stream) {
    if (entries == 0 || n_seqs == 0) return 0;
    HB_REQUIRE(entries > 0 && n_seqs > 0 && n_kv_heads > 0 && n_pages > 0 && pt_width > 0 && pt_width <= (1 << 24), "evict_select: bad sizes");
    HB_REQUIRE(first >= 0 && recent >= 0 && budget > 0 && (long long)first + recent <= budget,
               "evict_select: the first %d and the last %d rows do not fit a budget of %d", first, recent, budget);
    HB_REQUIRE((threads == 512 || threads == 1024) && (cluster == 1 || cluster == 2 || cluster == 4 || cluster == 8),
               "evict_select: blocks of %d threads in clusters of %d are not built", threads, cluster);
    const long long rows = (long long)entries * n_seqs * n_kv_heads;
    HB_REQUIRE(rows * cluster <= 0x7fffffffLL, "evict_select: too many lists of rows for one launch");
    cudaStream_t s = (cudaStream_t)stream;
    if (threads == 1024)
        return launch_select<1024>(cluster, mass, page_table, pt_width, lengths, kept, (int)rows, n_seqs, n_kv_heads, n_pages, first, recent,
                                   budget, status, s);
    return launch_select<512>(cluster, mass, page_table, pt_width, lengths, kept, (int)rows, n_seqs, n_kv_heads, n_pages, first, recent, budget,
                              status, s);
}

// --------------------------------------------------------------------------------------------------- rows move
// Row kept[j] of the keys, the values and the mass of (entry, sequence, kv head) becomes row j.  Memory-bound: every moved
// row is read once and written once.
//
// Into other pages: no order matters, a block takes ER_ROWS rows.  In place: kept is ascending, so kept[j] >= j, and a block
// walks a list's rows from the front, a chunk at a time: loads of a chunk, barrier, stores of the chunk.  The chunk behind
// it may be loaded before those stores: its sources lie at or behind its own rows, which lie behind the rows that are
// written.  Only rows of one list depend on one another, and every byte column of a row moves by itself, so a list is cut into
// `slices` of its rows' bytes for more blocks.
// Units of 32 bytes (the widest loads and stores of sm_100) where rows and addresses allow: with 16 the addresses' arithmetic kept the
// schedulers two thirds busy (104 instead of 96 us for 543 MB).
#define ER_THREADS 256

struct __align__(32) Unit32 {
    unsigned long long x[4];
};
template <typename U> __device__ __forceinline__ U er_load(const U* p) { return __ldcg(p); }
template <> __device__ __forceinline__ Unit32 er_load<Unit32>(const Unit32* p) {
    Unit32 u;
    asm volatile("ld.global.cg.v4.b64 {%0, %1, %2, %3}, [%4];" : "=l"(u.x[0]), "=l"(u.x[1]), "=l"(u.x[2]), "=l"(u.x[3]) : "l"(p) : "memory");
    return u;
}
template <typename U> __device__ __forceinline__ void er_store(U* p, const U& u) { *p = u; }
template <> __device__ __forceinline__ void er_store<Unit32>(Unit32* p, const Unit32& u) {
    asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(p), "l"(u.x[0]), "l"(u.x[1]), "l"(u.x[2]), "l"(u.x[3]) : "memory");
}

struct EvictRows {
    const int* kept;
    const int* from_table;
    const int* to_table;
    int from_width, to_width, n_seqs, nkv, n_pages, budget, in_place;
    int* status;
};

// one tensor [entries][pages][kv heads][64][row units], units [u0, u0 + un) of its rows, list `row`, kept rows [j0, j1)
template <typename U>
__device__ __forceinline__ void evict_move(const EvictRows& p, U* data, int row_units, int u0, int un, int row, int j0, int j1) {
    const int g = row % p.nkv, b = (row / p.nkv) % p.n_seqs;
    const size_t entry = (size_t)(row / (p.nkv * p.n_seqs)) * p.n_pages;
    const int* kept = p.kept + (size_t)row * p.budget;
    const int* from = p.from_table + (size_t)b * p.from_width;
    const int* to = p.to_table + (size_t)b * p.to_width;
    constexpr int ER_UNROLL = sizeof(U) == 32 ? 2 : 4;    // rows in flight: 64 bytes a thread, registers for four blocks to an SM
    const int per = ER_THREADS / un, sub = threadIdx.x % un, lead = threadIdx.x / un;     // rows per pass; un <= ER_THREADS
    const int chunk = per * ER_UNROLL;
    bool bad = false;
    auto address = [&](const int* table, int width, int r) -> U* {
        const int pi = r / HB_PAGE_TOKENS;
        const int page = pi < width ? table[pi] : -1;
        if (page < 0 || page >= p.n_pages) {
            bad = true;
            return nullptr;
        }
        return data + (((entry + page) * p.nkv + g) * HB_PAGE_TOKENS + (r & (HB_PAGE_TOKENS - 1))) * (size_t)row_units + u0 + sub;
    };
    U next[ER_UNROLL];
    bool have[ER_UNROLL];
    int src[ER_UNROLL];                                   // of the chunk behind the one that is loaded
    auto sources = [&](int c0) {
#pragma unroll
        for (int i = 0; i < ER_UNROLL; i++) {
            const int j = c0 + i * per + lead;
            src[i] = lead < per && j < j1 ? kept[j] : -1;
        }
    };
    auto load = [&](int c0) {
#pragma unroll
        for (int i = 0; i < ER_UNROLL; i++) {
            have[i] = false;
            if (src[i] >= 0 && !(p.in_place && src[i] == c0 + i * per + lead)) {
                const U* a = address(from, p.from_width, src[i]);
                if (a != nullptr) {
                    next[i] = er_load(a);
                    have[i] = true;
                }
            }
        }
        sources(c0 + chunk);
    };
    sources(j0);
    load(j0);
    for (int c0 = j0; c0 < j1; c0 += chunk) {
        U now[ER_UNROLL];
        bool write[ER_UNROLL];
#pragma unroll
        for (int i = 0; i < ER_UNROLL; i++) {
            now[i] = next[i];
            write[i] = have[i];
        }
        if (p.in_place) __syncthreads();                  // every load of this chunk came before every store of it
        load(c0 + chunk);
#pragma unroll
        for (int i = 0; i < ER_UNROLL; i++)
            if (write[i]) {
                U* a = address(to, p.to_width, c0 + i * per + lead);
                if (a != nullptr) er_store(a, now[i]);
            }
    }
    if (bad) hb_note(p.status, HB_STATUS_PAGE, 1 + b);
}

// grid: `blocks` of each list, list by list; a list's blocks are, for every range of rows, the slices of the keys, those of the values, the mass
template <typename U>
__global__ void __launch_bounds__(ER_THREADS)
evict_rows_kernel(EvictRows p, U* k, int k_units, int k_slices, U* v, int v_units, int v_slices, uint32_t* mass, int rows_per_block, int blocks) {
    // no pdl_trigger(): the decode attention kernels read pages of older tokens before their griddepcontrol.wait, and
    // with small kernels in between they could be resident while rows still move.  Without the trigger, nothing behind this
    // kernel starts before it has finished.
    pdl_wait();
    p.kept = pdl_fresh(p.kept);
    p.from_table = pdl_fresh(p.from_table);
    p.to_table = pdl_fresh(p.to_table);
    const int parts = k_slices + v_slices + (mass != nullptr ? 1 : 0);
    const int row = blockIdx.x / blocks, block = blockIdx.x % blocks, part = block % parts;
    const int j0 = (block / parts) * rows_per_block, j1 = min(j0 + rows_per_block, p.budget);
    if (p.kept[(size_t)row * p.budget + j0] < 0) return;      // behind the last kept row
    if (part < k_slices) {
        const int a = k_units * part / k_slices, z = k_units * (part + 1) / k_slices;
        evict_move<U>(p, k, k_units, a, z - a, row, j0, j1);
    } else if (part < k_slices + v_slices) {
        const int s = part - k_slices;
        const int a = v_units * s / v_slices, z = v_units * (s + 1) / v_slices;
        evict_move<U>(p, v, v_units, a, z - a, row, j0, j1);
    } else {
        evict_move<uint32_t>(p, mass, 1, 0, 1, row, j0, j1);
    }
}

// k, v: [entries][n_pages][n_kv_heads][64][row bytes]; mass (float32, may be null): [entries][n_pages][n_kv_heads][64]; kept:
// [entries][n_seqs][n_kv_heads][budget], ascending, -1 behind its end.  to_table == null: in place.
extern "C" int hb_evict_rows(const int* kept, void* k, int k_row_bytes, void* v, int v_row_bytes, float* mass, const int* from_table,
                             int from_width, const int* to_table, int to_width, int entries, int n_seqs, int n_kv_heads, int n_pages,
                             int budget, int sm_count, int* status, void* stream) {
    if (entries == 0 || n_seqs == 0) return 0;
    HB_REQUIRE(entries > 0 && n_seqs > 0 && n_kv_heads > 0 && n_pages > 0 && from_width > 0 && budget > 0 && sm_count > 0, "evict_rows: bad sizes");
    HB_REQUIRE(k_row_bytes > 0 && v_row_bytes > 0 && k_row_bytes % 2 == 0 && v_row_bytes % 2 == 0, "evict_rows: bad row sizes");
    const long long lists = (long long)entries * n_seqs * n_kv_heads;
    EvictRows p = {kept, from_table, to_table != nullptr ? to_table : from_table, from_width, to_table != nullptr ? to_width : from_width,
                   n_seqs, n_kv_heads, n_pages, budget, to_table == nullptr, status};
    HB_REQUIRE(p.in_place || budget <= (long long)p.to_width * HB_PAGE_TOKENS, "evict_rows: %d rows do not fit a page table of width %d", budget, p.to_width);
    const uintptr_t both = (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_row_bytes | (uintptr_t)v_row_bytes;
    const int unit = both % 32 == 0 ? 32 : both % 16 == 0 ? 16 : both % 4 == 0 ? 4 : 2;
    HB_REQUIRE(both % 2 == 0, "evict_rows: keys and values must be 2-byte aligned");
    const int ku = k_row_bytes / unit, vu = v_row_bytes / unit;
    int ks = (ku + ER_THREADS - 1) / ER_THREADS, vs = (vu + ER_THREADS - 1) / ER_THREADS;
    int rows_per_block;
    if (p.in_place) {
        // a list cannot be cut along its rows: slices of its bytes (64 at least, two 32-byte sectors) until the device is full
        while ((ks + vs) * lists < 2LL * sm_count && k_row_bytes / (2 * ks) >= 64 && v_row_bytes / (2 * vs) >= 64) ks *= 2, vs *= 2;
        rows_per_block = budget;
    } else {
        // about four blocks to a slot (an SM holds four): a block's first chunk waits for three loads in a row (kept, page, row), the
        // chunks behind it overlap with the one before
        const long long lists_parts = lists * (ks + vs), want = (16LL * sm_count + lists_parts - 1) / lists_parts;
        rows_per_block = (int)((budget + want - 1) / want);
        rows_per_block = rows_per_block < 64 ? 64 : rows_per_block;
    }
    const long long blocks = (long long)((budget + rows_per_block - 1) / rows_per_block) * (ks + vs + (mass != nullptr ? 1 : 0));
    HB_REQUIRE(blocks * lists <= 0x7fffffffLL, "evict_rows: %lld lists of %d rows are too many for one launch", lists, budget);
    dim3 grid((unsigned)(blocks * lists));
    cudaStream_t s = (cudaStream_t)stream;
#define HB_ER_LAUNCH(U) \
    hb_launch(evict_rows_kernel<U>, grid, dim3(ER_THREADS), 0, s, p, (U*)k, ku, ks, (U*)v, vu, vs, (uint32_t*)mass, rows_per_block, (int)blocks)
    cudaError_t e = unit == 32 ? HB_ER_LAUNCH(Unit32) : unit == 16 ? HB_ER_LAUNCH(uint4) : unit == 4 ? HB_ER_LAUNCH(uint32_t) : HB_ER_LAUNCH(unsigned short);
#undef HB_ER_LAUNCH
    if (e != cudaSuccess) return hb_fail("evict_rows: launch failed: %s", cudaGetErrorString(e));
    return hb_check_launch("evict_rows");
}
