// What the kernels of attention with accumulated weights share: where a block's queries or keys are, and how a key's sum of
// weights is written.
#pragma once
#include "common.cuh"

#define MASS_LOG2E 1.4426950408889634f
#define MASS_FEW_PAIRS 512           // (tokens of a sequence) x (heads of a group) that a step of few tokens may have

// before (null: nothing is added), mass: [n_pages][kv heads][64]; before may be mass.  parts: [shares][kv heads][places], where a
// place is a key's number over all tiles of keys of the step.
struct MassOut {
    const float* before;
    float* mass;
    float* parts;
};

// distance, in floats, of the scores of two heads
static __host__ __device__ inline long long mass_score_ld(int max_len) { return ((long long)max_len + 63) / 64 * 64; }

// A step's metadata may come from the kernel in front (lengths that a program works out on the device): read behind pdl_wait() only
__device__ __forceinline__ void mass_fresh(const int* __restrict__& page_table, const int* __restrict__& seq_start, const int* __restrict__& seq_pos0) {
    page_table = pdl_fresh(page_table);
    seq_start = pdl_fresh(seq_start);
    seq_pos0 = pdl_fresh(seq_pos0);
}

// A step's sequences are looked through 32 at a time, a lane each: which of them element number `at` of `count(b)` elements each belongs
// to, its number there, and the sum of `other(b)` over the sequences in front.  Called by whole warps; the same answer in every lane.
template <typename F, typename H>
__device__ __forceinline__ bool mass_find(int n_seqs, int at, F&& count, H&& other, int& b, int& inside, int& others) {
    const int lane = threadIdx.x & 31;
    int front = 0;
    others = 0;
    for (int b0 = 0; b0 < n_seqs; b0 += 32) {
        const bool there = b0 + lane < n_seqs;
        const int n = there ? count(b0 + lane) : 0, o = there ? other(b0 + lane) : 0;
        int sum = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += u;
        }
        const unsigned behind = __ballot_sync(0xffffffffu, at < front + sum);
        if (behind != 0u) {
            const int i = __ffs(behind) - 1;
            b = b0 + i;
            inside = at - front - (__shfl_sync(0xffffffffu, sum, i) - __shfl_sync(0xffffffffu, n, i));
            others += (int)__reduce_add_sync(0xffffffffu, (unsigned)(lane < i ? o : 0));
            return true;
        }
        front += __shfl_sync(0xffffffffu, sum, 31);
        others += (int)__reduce_add_sync(0xffffffffu, (unsigned)o);
    }
    b = inside = 0;
    return false;
}

// where the log-sums of a sequence's rows begin, in blocks of 128 rows (attention_chunk_tc below)
__host__ __device__ constexpr int mass_round128(int n) { return (n + 127) & ~127; }

// The sequence b and its block blk of `rows` new tokens that block number `at` of the step stands for; place0: mass_round128 of the
// new tokens of the sequences in front, added up.
__device__ __forceinline__ bool mass_find_block(const int* __restrict__ seq_start, int n_seqs, int at, int rows, int& b, int& blk, int& place0) {
    return mass_find(n_seqs, at, [&](int i) { return (seq_start[i + 1] - seq_start[i] + rows - 1) / rows; },
                     [&](int i) { return mass_round128(seq_start[i + 1] - seq_start[i]); }, b, blk, place0);
}

// The sequence b and its tile kt of `tile` rows of the cache (those behind this step) that tile number `at` stands for.
__device__ __forceinline__ bool mass_find_keys(const int* __restrict__ seq_start, const int* __restrict__ seq_pos0, int n_seqs, int at, int tile,
                                               int& b, int& kt, int& place0) {
    return mass_find(n_seqs, at, [&](int i) { return (seq_pos0[i] + seq_start[i + 1] - seq_start[i] + tile - 1) / tile; },
                     [&](int i) { return mass_round128(seq_start[i + 1] - seq_start[i]); }, b, kt, place0);
}

// The new tokens [n0, n1) of a sequence that see one of the keys [key0, key0 + keys): token i stands at pos0 + i.
__device__ __forceinline__ void mass_queries(int key0, int keys, int pos0, int n_new, int window, int& n0, int& n1) {
    n0 = max(0, key0 - pos0);
    n1 = n_new;
    if (window > 0) n1 = (int)min((long long)n_new, (long long)key0 + keys - 1 + window - pos0);
    if (n1 <= n0) n1 = n0 = 0;
}

__device__ __forceinline__ void mass_write(const MassOut& mo, float sum, int g, int key, int page, int nkv, int n_pages, int pos0, int n_new) {
    if (key >= pos0 + n_new || page < 0 || page >= n_pages) return;       // behind the end, or a page that was given back
    const size_t at = ((size_t)page * nkv + g) * HB_PAGE_TOKENS + (key & (HB_PAGE_TOKENS - 1));
    const float old = (key < pos0 && mo.before != nullptr) ? __ldcg(mo.before + at) : 0.0f;
    mo.mass[at] = old + sum;
}

// For blocks that have all of a sequence's new tokens and all of its keys (short sequences): they write the outputs and the weights
// themselves and no second kernel follows.  out null: a second kernel joins the shares.
struct MassWhole {
    void* out;
    long long out_stride;
    MassOut mo;
};

// The weights of a sequence's n keys from the scores that this block wrote, in the order of the second kernel's sums; lse: of pair r, which is
// head r % G of token r / G.
__device__ __forceinline__ void mass_whole(const MassOut& mo, const float* scores, long long score_ld, const float* lse, int n_new, int G, int g, int t0,
                                           int nh, int nkv, int pos0, int window, const int* __restrict__ pt, int pt_width, int n_pages) {
    const int n = (int)min((long long)(pos0 + n_new), score_ld);
    for (int key = threadIdx.x; key < n; key += blockDim.x) {
        float s = 0.0f;
        for (int i = 0; i < n_new; i++) {
            const int p = pos0 + i;
            if (key > p || key < hb_oldest_visible(p, window, 0)) continue;
            const float* row = scores + ((size_t)(t0 + i) * nh + g * G) * score_ld + key;
#pragma unroll 4
            for (int h = 0; h < G; h++) s += exp2f(row[h * score_ld] - lse[i * G + h]);
        }
        const int pi = key / HB_PAGE_TOKENS;
        mass_write(mo, s, g, key, pi < pt_width ? pt[pi] : -1, nkv, n_pages, pos0, n_new);
    }
}

// a key's sum, or with several shares (S) share z of it
__device__ __forceinline__ void mass_store(const MassOut& mo, float sum, int b, int g, int key, int page, int nkv, int n_pages, int pos0, int n_new,
                                           int z, int S, size_t place, size_t places) {
    if (S > 1) mo.parts[((size_t)z * nkv + g) * places + place] = sum;
    else mass_write(mo, sum, g, key, page, nkv, n_pages, pos0, n_new);
}

__device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ __forceinline__ void load4(const bf16* p, float (&x)[4]) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}

int mass_join(const int* page_table, int pt_width, const int* seq_start, const int* seq_pos0, MassOut mo, int n_seqs, int nkv, int n_pages, int tile,
              int key_tiles, int splits, cudaStream_t s);

// Share z of S of the pages [first, last): at most S equal shares of this sequence's pages, and no more than of `least` pages each.
__device__ __forceinline__ void mass_share(int first, int last, int z, int S, int least, int& page0, int& page1) {
    const int n = last - first, shares = max(1, min(S, (n + least - 1) / least)), per = max(1, (n + shares - 1) / shares);
    page0 = first + z * per;
    page1 = min(page0 + per, last);
}

// The keys of a block of queries, shared out: a block that sees n tiles of keys takes ceil(n / tiles) CTAs, and where those are several each
// leaves its unnormalised outputs and (maximum, sum) of its rows: o[(share * heads + head) * tokens + token][head size], ml likewise.
struct Shares {
    float* o;
    float* ml;
    int tiles;
};
__device__ __forceinline__ int shares_of(const Shares& sh, int n_tiles) { return max(1, (n_tiles + sh.tiles - 1) / sh.tiles); }
// how many tiles of `keys` keys a block of queries at positions first..last sees, and the first of them
__device__ __forceinline__ int key_tiles_of(int first, int last, int window, int keys, int& tile0) {
    tile0 = hb_oldest_visible(first, window, 0) / keys;
    return last / keys + 1 - tile0;
}

// A number that every lane of a warp has loaded alike, as one for the warp (the compiler then keeps it in a uniform register)
__device__ __forceinline__ int mass_uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// whether blocks of `span` tokens of a sequence of `rows` rows may see more tiles than go into one share (by the host's bound)
__device__ __forceinline__ bool shares_may_cut(const Shares& sh, int rows, int span, int window, int keys) {
    const int seen = window > 0 ? (int)min((long long)rows, (long long)window + span) : rows;
    return (seen + keys - 1) / keys + (window > 0 ? 1 : 0) > sh.tiles;
}

// joins the shares (attention_mass.cu): out and lse of the rows whose block has several; join_tokens: the new tokens of the sequences that
// shares_may_cut.  Blocks of `span` tokens, tiles of `keys`
// keys; lse[head * lse_ld + place], places in blocks of 128 per sequence and the log-sums negated (`rounded`), or the token's number
int shares_join(Shares sh, int join_tokens, int dtype, void* out, long long out_stride, float* lse, long long lse_ld, int rounded,
                const int* seq_start, const int* seq_pos0, int span, int keys, int window, int n_tokens, int n_seqs, int nh, int hd, cudaStream_t s);

// The first half of a step of many tokens on the tensor cores (attention_chunk_tc.cu): writes out and the rows'
// log-sums, negated, lse[head][place]: a sequence's places begin at a multiple of 128, behind those of the sequences in front.  q_blocks: sum
// over sequences of ceil(new tokens / span), span 128 with an even group of heads and 256 with an odd one; max_shares: the most CTAs
// that a block of queries takes, share_tiles: the most tiles of 128 keys of one of them; parts: max_shares * n_heads * n_tokens *
// (head_dim + 2) floats when max_shares > 1.
int attention_chunk_tc(const void* q, long long q_stride, const void* k_cache, const void* v_cache, const int* page_table, int pt_width,
                       const int* seq_start, const int* seq_pos0, void* out, long long out_stride, float* lse, long long lse_ld, float* parts,
                       int max_shares, int share_tiles, int join_tokens, int n_tokens, int n_seqs, int q_blocks, int n_heads, int n_kv_heads,
                       int head_dim, float scale, int window, int n_pages, int* error_flag, cudaStream_t s);

// The first half of a step of few tokens on the tensor cores (attention_few_tc.cu): token_blocks, the sum over sequences of ceil(new
// tokens / hb_attention_few_tc_tokens(...)); queries 4-byte, keys and values 16-byte aligned.
int attention_few_tc(MassWhole whole, const void* q, long long q_stride, const void* kc, const void* vc, const int* page_table, int pt_width,
                     const int* seq_start, const int* seq_pos0, float* part_o, float* part_ml, float* scores, long long score_ld, int splits,
                     int share_pages, int token_blocks, int max_new, int n_seqs, int nh, int nkv, int head_dim, float scale, int window, int n_pages,
                     int seq0, int* status, cudaStream_t s);
