// attention_tc.cuh -- the tensor-core attention kernel behind sptmm_attention_prompt (PREFIX false)
// and behind the shared prefix of sptmm_attention_decode (PREFIX true).
//
//     O = softmax(scale * Q K^T) V
//
// A CTA owns two tiles of query rows of one key head and walks over the keys in blocks of 128 with the
// running maximum m and sum l of the softmax, so scores never leave the SM.  A tile is 128 rows of
// (token, query head of the group): all heads that share the keys share their tiles, and a short
// sequence fills a tile with few tokens.  Per block and tile:
//     S = Q K^T                  tcgen05, operands from shared memory, S (128 x 128 fp32) in tensor memory
//     P = 2^(S scale - m)        one thread per row: m, l and the weights need no exchange between lanes
//     O += P V                   tcgen05, P (16 bit) from tensor memory where S was, O in tensor memory
// Warps: 0-3 the softmax of tile 0, 4-7 of tile 1, 8 the TMA loads (Q once, K and V blocks through a
// ring), 9 issues the products, 10 looks for values that are not finite (below), 11 keeps a caller's limit on the
// CTA's time, if there is one.  The products of one
// tile run while the other tile is in its softmax; tensor memory is full: S0 S1 O0 O1 are 512 columns
// at 128 channels.
// When a row's maximum grows, O and l would have to be scaled down; that is put off until it has grown by more
// than 2^8 (fp16: 2^6; see WeightRange), so after the first blocks it hardly ever happens.
// Masks: keys a row does not see get the score -inf before the maximum, blocks nobody sees are not
// visited, values behind the last visible key are overwritten with zeros in shared memory (a weight of
// zero times another sequence's NaN would be NaN).  Values that SOME rows of the CTA see (the causal
// diagonal) must stay; should one of them be NaN or infinite, warp 10 finds it and the CTA's rows are
// computed once more row by row (attend_row), where hidden keys are not touched at all.
//
// What bounds it (20 heads over 5, 128 channels, one sequence of 8192 tokens, causal: 344 GFLOP): 272 to 277 us
// = 1.25 PFLOP/s, 0.76 of the measured matmul rate; 321 us = 1.07 in runs of seconds, where the board's power
// cap holds the clock at 1.6 GHz.  A block takes 1.75 us: per tile about 1900 cycles of softmax (80 to load the
// scores, 380 for the maximum, 700 for each half of the exponentials, which the two warps of a scheduler share)
// and 1400 until the next scores (the second half of P V, Q K^T, and a few hundred cycles of barriers), while
// the tensor pipe is busy for 2460 of the 3300.  Weights are handed over in halves, so the product starts on the
// first while the second is computed (281 us whole).  Tried and slower: 64-key steps with two score buffers (332:
// Q K^T with 64 columns is bound by shared memory), one product warp per tile (347), the exponentials of the two
// warps of a scheduler taking turns (+1 %), an eighth to three eighths of the exponentials as a polynomial on
// the FMA pipe (+1 to +4 %), V and the next K on one barrier (283).  Up to 64 channels the exponentials are
// the limit (half the products per score); one tile per CTA and two CTAs per SM there: no gain.
// A CTA's beginning (2.5 us) and end (2.5 us) overlap with nothing: 9 % of the 8192-token prompt, most of a
// short one.
#pragma once
#include "tcgen05.cuh"

namespace sptmm {

struct TcParams {
    const void *Q, *K, *V;
    void *O;
    const int32_t *q_off, *k_off;            // prompt
    uint64_t ldq, ldk, ldv, ldo;
    uint32_t n_seqs, T, Tk, heads, kv_heads, group, head_dim, causal;
    uint32_t tokens;                         // tokens per tile, 128 / group
    uint32_t cluster;                        // CTAs that may share an item's keys
    uint32_t group_mul;                      // x * group_mul >> 16 = x / group for x < 256
    float scale;                             // scale * log2(e)
    // the shared prefix of a decode step: keys in pages, parts of the keys in different CTAs
    const int32_t *prefix_table;
    uint32_t prefix_len, n_pages, page_shift;
    uint32_t splits;                         // CTAs per item, each with an equal part of the keys
    float *part_o;                           // [token][head][split][head_dim], not divided by l
    float2 *part_ml;                         // [token][head][split]: (m in powers of two, l); l and O 2^up times as large (WeightRange)
    uint32_t *status;
    uint32_t wait_polls;                     // looks at its last product that a CTA may take; 0: no limit but that of every wait
};

constexpr uint32_t kTcThreads = 384;        // three warpgroups: two of softmax, one of loads, products and the value check
constexpr uint32_t kKeys = 128;              // keys per block

template <int DP> struct TcLayout {
    static constexpr uint32_t slabs = DP / 64, tile = 128 * DP * 2;
    static constexpr uint32_t stages = DP == 128 ? 5 : 8;
    static constexpr uint32_t smem = 2 * tile + stages * tile + 1024;      // 1024: room to align
    static constexpr uint32_t out = 256 * DP * 4;                          // the ring's memory at the end: O in fp32, then (m, l) of every row
    static_assert(out + 256 * 8 <= stages * tile, "the ring holds O and (m, l) at the end");
};

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of `addr` in the shared memory of CTA `rank` of the cluster
__device__ __forceinline__ uint32_t smem_of(uint32_t addr, uint32_t rank)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr)
{
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// One row by CUDA cores: a warp, four channels per lane, keys k0 .. k0 + n one after the other.
template <typename T>
__device__ void attend_row(const TcParams &p, uint32_t t, uint32_t h, uint32_t kh, uint32_t k0, uint32_t n)
{
    const uint32_t lane = threadIdx.x & 31, c = lane * 4, D = p.head_dim;
    float q[4] = {0, 0, 0, 0}, o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0;
    if (c < D) {
        const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const T *>(p.Q) + (uint64_t)t * p.ldq + (uint64_t)h * D + c);
        const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
        q[0] = a.x * p.scale; q[1] = a.y * p.scale; q[2] = b.x * p.scale; q[3] = b.y * p.scale;
    }
    for (uint32_t j = 0; j < n; j++) {
        float k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0};
        if (c < D) {
            const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const T *>(p.K) + (uint64_t)(k0 + j) * p.ldk + (uint64_t)kh * D + c);
            const uint2 z = *reinterpret_cast<const uint2 *>(static_cast<const T *>(p.V) + (uint64_t)(k0 + j) * p.ldv + (uint64_t)kh * D + c);
            float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
            k[0] = a.x; k[1] = a.y; k[2] = b.x; k[3] = b.y;
            a = unpack2<T>(z.x); b = unpack2<T>(z.y);
            v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
        }
        float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const float m1 = fmaxf(m, s), base = m1 == -INFINITY ? 0.0f : m1;
        const float w0 = ex2(m - base), w1 = ex2(s - base);
        m = m1;
        l = l * w0 + w1;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = o[i] * w0 + w1 * v[i];
    }
    if (c >= D) return;
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    *reinterpret_cast<uint2 *>(static_cast<T *>(p.O) + (uint64_t)t * p.ldo + (uint64_t)h * D + c) =
        make_uint2(pack2<T>(o[0] * r, o[1] * r), pack2<T>(o[2] * r, o[3] * r));
}

// What a CTA works on.  Query i of the sequence (0 .. n_q) is row q0 + i and sees keys 0 .. i + shift of
// the m keys from row k0, at most m.
struct TcItem {
    uint32_t q0, n_q, k0, m, first;          // `first`: the CTA's first query
    int32_t shift;                           // causal: m - n_q; else so large that every query sees all
    uint32_t block0, blocks;                 // blocks of 128 keys
    bool any;
    __device__ __forceinline__ uint32_t visible(uint32_t i) const
    {
        const int64_t v = (int64_t)i + shift + 1;
        return v < 0 ? 0u : (uint32_t)min(v, (int64_t)m);
    }
};

__device__ __forceinline__ void seq_range(const TcParams &p, uint32_t s, uint32_t &q0, uint32_t &n, uint32_t &k0, uint32_t &m)
{
    const int32_t a = min(max(p.q_off[s], 0), (int32_t)p.T), b = min(max(p.q_off[s + 1], a), (int32_t)p.T);
    const int32_t c = min(max(p.k_off[s], 0), (int32_t)p.Tk), d = min(max(p.k_off[s + 1], c), (int32_t)p.Tk);
    q0 = a; n = b - a; k0 = c; m = d - c;
}

// Items are pairs of tiles.  Up to kOrderedSeqs sequences they are taken in falling order of the keys they visit, so
// that the longest start first and the short ones fill the end.  An item's level is the number of its pair of tiles
// counted from the sequence's first key; rank `w` is looked up by counting the items at or above a level (a warp, a
// lane per sequence).
// For more sequences that would cost every CTA a few passes over all of them: 0.4 ms a call for 700 sequences of one
// token and 54 ms for 8192.  Then items are numbered by the offsets alone, sequence after sequence: those of s begin
// at q_off[s] / per + s, which leaves room for every partly filled pair and grows with s, so that a search in at most
// four steps finds s (0.18 and 1.9 ms).  Measured, ordered / by offset (20 heads over 5, lengths spread over their
// logarithm up to 1024): 16 sequences 31.7 / 32.5 us, 33 38 / 35, 64 96 / 85, 128 231 / 184; up to 4096 and in rising
// order, the longest last: 33 sequences 153 / 134, 64 476 / 424.
constexpr uint32_t kOrderedSeqs = 32;
// How many numbers the items of a call may take.
inline uint64_t item_numbers(uint64_t n_seqs, uint64_t T, uint64_t per)
{
    if (n_seqs > kOrderedSeqs) return T / per + n_seqs;
    return (T + (n_seqs < T ? n_seqs : T) * (per - 1)) / per;      // every sequence may end with a part of a pair
}

__device__ __forceinline__ bool find_item_by_offset(const TcParams &p, uint32_t w, uint32_t &seq, uint32_t &pair)
{
    const uint32_t lane = threadIdx.x & 31, per = 2 * p.tokens;
    auto begin = [&](uint32_t s) { return (uint32_t)min(max(p.q_off[s], 0), (int32_t)p.T) / per + s; };
    uint32_t lo = 0, span = p.n_seqs;        // begin(lo) <= w, and the last such sequence is one of lo .. lo + span
    if (begin(0) > w) return false;
    while (span > 1) {
        const uint32_t step = (span + 31) / 32, at = lane * step;
        const uint32_t last = 31 - __clz(__ballot_sync(0xffffffffu, at < span && begin(lo + at) <= w));      // lane 0 is always among them
        lo += last * step;
        span = min(step, span - last * step);
    }
    uint32_t q0, nq, k0, m;
    seq_range(p, lo, q0, nq, k0, m);
    const uint32_t n = (nq + per - 1) / per, i = w - begin(lo);
    seq = lo;
    pair = p.causal ? n - 1 - i : i;
    return i < n;
}

__device__ __forceinline__ bool find_item(const TcParams &p, uint32_t w, uint32_t &seq, uint32_t &pair)
{
    if (p.n_seqs > kOrderedSeqs) return find_item_by_offset(p, w, seq, pair);
    const uint32_t lane = threadIdx.x & 31, per = 2 * p.tokens;
    uint32_t q0, nq, k0, m, n = 0, low = 0;  // items and first level of sequence `lane`
    if (p.n_seqs == 1) {
        seq_range(p, 0, q0, nq, k0, m);
        n = (nq + per - 1) / per;
        seq = 0;
        pair = p.causal ? n - 1 - w : w;
        return w < n;
    }
    if (lane < p.n_seqs) {
        seq_range(p, lane, q0, nq, k0, m);
        n = (nq + per - 1) / per;
        low = p.causal ? (m > nq ? (m - nq) / per : 0u) : m / per;
    }
    auto at_or_above = [&](uint32_t x) -> uint32_t {
        if (!p.causal) return low >= x ? n : 0u;
        return x <= low ? n : (x - low >= n ? 0u : n - (x - low));
    };
    auto count = [&](uint32_t x) { return __reduce_add_sync(0xffffffffu, at_or_above(x)); };
    if (w >= count(0)) return false;
    uint32_t lo = 0, hi = __reduce_max_sync(0xffffffffu, n + low) + 1;          // count(lo) > w, count(hi) <= w
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (count(mid) > w) lo = mid; else hi = mid;
    }
    const uint32_t left = w - count(lo + 1), here = at_or_above(lo) - at_or_above(lo + 1);       // among the items of level lo, in order of sequences
    uint32_t sum = here;                     // inclusive prefix over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= (uint32_t)o) sum += y;
    }
    const int src = __ffs(__ballot_sync(0xffffffffu, left < sum)) - 1;
    seq = src;
    pair = __shfl_sync(0xffffffffu, p.causal ? lo - low : left - (sum - here), src);
    return true;
}

// SPLIT: clusters share the keys of an item.  A variant of its own, because what it keeps for the end costs the
// others registers in the softmax loop (8192 tokens: 323 us against 275).
template <typename T, int DP, bool PREFIX, bool SPLIT = false>
__global__ void __launch_bounds__(kTcThreads, 1)
k_attention_tc(const __grid_constant__ TcParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
               const __grid_constant__ CUtensorMap map_v)
{
    using L = TcLayout<DP>;
    constexpr bool kBf16 = sizeof(T) == 2 && !__is_same(T, __half);
    extern __shared__ unsigned char dyn[];
    __shared__ uint64_t bars[2 + 2 * L::stages + 2 + 4 + 2 + 1 + 1];
    __shared__ uint32_t tmem_base, abort_flag, bad_values, item_seq, item_pair, item_ok;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t bar0 = smem_addr(bars);
    const uint32_t b_q = bar0, b_full = bar0 + 16, b_empty = b_full + 8 * L::stages, b_s = b_empty + 8 * L::stages, b_p = b_s + 16,
                   b_o = b_p + 32, b_fix = b_o + 16, b_end = b_fix + 8;
    volatile uint32_t *abort_word = &abort_flag;
    if (!PREFIX) pdl_launch_dependents();
    if (warp == 8) {
        if (lane == 0) {
            mbar_init(b_q, 1); mbar_init(b_q + 8, 1);
            for (uint32_t i = 0; i < L::stages; i++) { mbar_init(b_full + 8 * i, 1); mbar_init(b_empty + 8 * i, 1); }
            for (uint32_t t = 0; t < 2; t++) { mbar_init(b_s + 8 * t, 1); mbar_init(b_p + 16 * t, 4); mbar_init(b_p + 16 * t + 8, 4); mbar_init(b_o + 8 * t, 1); }
            mbar_init(b_fix, 1); mbar_init(b_end, 1);
            abort_flag = 0; bad_values = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            tma_prefetch_map(&map_q); tma_prefetch_map(&map_k); tma_prefetch_map(&map_v);
        }
    } else if (warp == 9) {
        tmem_alloc(smem_addr(&tmem_base), 512);
    }
    pdl_wait_prior_grid();
    // The next kernel (k_decode) reads nothing this one writes: let it start as soon as what came before has
    // ended, that is from here on, and it need not wait for this one.
    if (PREFIX) pdl_launch_dependents();
    const uint32_t rank = SPLIT ? blockIdx.x % p.cluster : 0, unit = SPLIT ? blockIdx.x / p.cluster : blockIdx.x;
    uint32_t kh, split = 0;
    if constexpr (PREFIX) {
        split = unit % p.splits;
        kh = unit / p.splits % p.kv_heads;
    } else {
        kh = unit % p.kv_heads;
        if (warp == 0) {
            uint32_t s = 0, pr = 0;
            const bool ok = find_item(p, unit / p.kv_heads, s, pr);
            if (lane == 0) { item_ok = ok; item_seq = s; item_pair = pr; }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    TcItem it;
    bool spread;                             // the CTAs of the cluster share the item's keys
    if constexpr (PREFIX) {
        it.q0 = 0; it.n_q = p.T; it.k0 = 0; it.m = p.prefix_len; it.shift = (int32_t)p.prefix_len;
        it.first = unit / p.splits / p.kv_heads * 2 * p.tokens;
        it.any = true;
        spread = false;
        const uint32_t all = (p.prefix_len + kKeys - 1) / kKeys;
        it.block0 = (uint32_t)((uint64_t)all * split / p.splits);
        it.blocks = (uint32_t)((uint64_t)all * (split + 1) / p.splits) - it.block0;
    } else {
        it.any = item_ok;
        seq_range(p, it.any ? item_seq : 0, it.q0, it.n_q, it.k0, it.m);
        it.shift = p.causal ? (int32_t)it.m - (int32_t)it.n_q : 0x40000000;
        it.first = (it.any ? item_pair : 0) * 2 * p.tokens;
        const uint32_t all = it.any ? (it.visible(min(it.n_q, it.first + 2 * p.tokens) - 1) + kKeys - 1) / kKeys : 0;
        // two blocks each are the least that pays for the exchange at the end; else the first CTA alone
        spread = SPLIT && all >= 2 * p.cluster;
        it.any = it.any && (spread || rank == 0);
        it.block0 = spread ? all * rank / p.cluster : 0;
        it.blocks = spread ? all * (rank + 1) / p.cluster - it.block0 : it.any ? all : 0;
    }
    const uint32_t n_here = it.any ? min(it.n_q - it.first, 2 * p.tokens) : 0;      // queries of this CTA
    const uint32_t n_tiles = n_here > p.tokens ? 2 : 1;
    const uint32_t last_key = it.any ? it.visible(it.first + n_here - 1) : 0;       // keys nobody here sees start at this one
    const uint32_t q_smem = (smem_addr(dyn) + 1023) & ~1023u, ring = q_smem + 2 * L::tile;
    const uint32_t tmem = tmem_base;
    const uint32_t n = it.blocks;
    const uint32_t D = p.head_dim, slabs = (D + 63) / 64;
    uint32_t issued = 0;                     // ring loads on their way (the loading thread's)
    const bool cut = (it.block0 + n) * kKeys > last_key;                            // the last block holds keys nobody sees

    // registers: 3 x 168 at launch; a softmax thread holds 128 scores, the others next to nothing
    if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < 8) {
        // ---- softmax: thread = row --------------------------------------------------------------
        const uint32_t tile = warp >> 2, row = tid & 127, s_addr = tmem + tile * 128 + ((warp & 3) << 21), o_addr = tmem + 256 + tile * DP + ((warp & 3) << 21);
        const uint32_t tok = tile * p.tokens + row / p.group;      // row / group < tokens for rows in use
        const bool mine = row < p.tokens * p.group && tok < n_here;
        const uint32_t vis = mine ? it.visible(it.first + tok) : it.m;         // rows not in use are never stored: no mask for their sake
        float m = -INFINITY, l = 0.0f;       // m in units of the raw score
        const float sc = p.scale;
        bool ok = true;
        if (tile < n_tiles && n > 0) {
            for (uint32_t i = 0; i < n; i++) {
                const uint32_t j0 = (it.block0 + i) * kKeys;
                uint32_t pages_ok = 0xffu;
                if constexpr (PREFIX) {                                             // which pages of the block lie in the cache
                    const uint32_t per = kKeys >> p.page_shift, at = (j0 >> p.page_shift) + lane;
                    bool good = true;
                    if (lane < per && (at << p.page_shift) < p.prefix_len) good = (uint32_t)p.prefix_table[at] < p.n_pages;
                    pages_ok = __ballot_sync(0xffffffffu, good);
                }
                ok = ok && mbar_wait_warp(b_s + 8 * tile, i & 1, abort_word);
                if (!ok) break;
                tc_fence_after();
                uint32_t r[128];
#pragma unroll
                for (int c = 0; c < 4; c++) tmem_ld32(s_addr + 32 * c, r + 32 * c);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 4; c++) pin32(r + 32 * c);
                if (__any_sync(0xffffffffu, j0 + kKeys > vis)) {
                    const int32_t left = (int32_t)vis - (int32_t)j0;
#pragma unroll
                    for (int c = 0; c < 128; c++) if (c >= left) r[c] = 0xff800000u;
                }
                if constexpr (PREFIX) {
                    if ((pages_ok & 0xffu) != 0xffu)
#pragma unroll
                        for (int c = 0; c < 128; c++) if (!(pages_ok >> (c >> p.page_shift) & 1)) r[c] = 0xff800000u;
                }
                float mx[4];
#pragma unroll
                for (int c = 0; c < 4; c++) mx[c] = fmaxf(__uint_as_float(r[c]), __uint_as_float(r[c + 4]));
#pragma unroll
                for (int c = 8; c < 128; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; e++) mx[e] = max3(mx[e], __uint_as_float(r[c + e]), __uint_as_float(r[c + 4 + e]));
                const float mb = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                // a first finite maximum, or one too far above the one in use: scale O and l
                const bool grow = mine && mb > m && (m == -INFINITY || (mb - m) * sc > WeightRange<T>::lag);
                if (__any_sync(0xffffffffu, grow)) {
                    const float m1 = fmaxf(m, mb), w = m == -INFINITY ? (m1 == -INFINITY ? 1.0f : 0.0f) : ex2((m - m1) * sc);
                    m = m1;
                    l *= w;
                    if (i > 0) {
                        for (uint32_t c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(o_addr + c, o);
                            tmem_wait_ld();
                            pin32(o);
#pragma unroll
                            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * w);
                            tmem_st32(o_addr + c, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.0f : m * sc - WeightRange<T>::up;
                const uint64_t sc2 = f2_pack(sc, sc), nb2 = f2_pack(-base, -base);
                uint64_t sum[2] = {0, 0};
#pragma unroll
                for (int half = 0; half < 2; half++) {                               // the product starts on the first half
                    uint32_t w[32];
#pragma unroll
                    for (int c = 0; c < 64; c += 2) {
                        const float2 x = f2_unpack(f2_fma(f2_pack(__uint_as_float(r[64 * half + c]), __uint_as_float(r[64 * half + c + 1])), sc2, nb2));
                        const float a = ex2(x.x), b = ex2(x.y);
                        sum[(c >> 1) & 1] = f2_add(sum[(c >> 1) & 1], f2_pack(a, b));
                        w[c >> 1] = pack2<T>(a, b);
                    }
                    tmem_st32(s_addr + 32 * half, w);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(b_p + 16 * tile + 8 * half);
                }
                const float2 z = f2_unpack(f2_add(sum[0], sum[1]));
                l += z.x + z.y;
            }
            ok = ok && mbar_wait_warp(b_o + 8 * tile, 0, abort_word);
            if (SPLIT && spread) ok = ok && (n_tiles == 1 || mbar_wait_warp(b_o + 8 * (tile ^ 1), 0, abort_word));
            tc_fence_after();
        }
        // ---- out ----
        if (SPLIT && spread) {
            if (ok && tile < n_tiles && n > 0) {
                // every product is done: the ring's memory takes O (16-byte chunks swizzled by row) and (m, l)
                const uint32_t to = ring + (tile * 128 + row) * DP * 4;
                asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(ring + L::out + (tile * 128 + row) * 8), "f"(m == -INFINITY ? -INFINITY : m * sc), "f"(l) : "memory");
                for (uint32_t c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(o_addr + c, o);
                    tmem_wait_ld();
                    pin32(o);
#pragma unroll
                    for (uint32_t e = 0; e < 8; e++)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + (((c >> 2) + (e ^ (row & 7))) << 4)), "r"(o[4 * e]), "r"(o[4 * e + 1]),
                                     "r"(o[4 * e + 2]), "r"(o[4 * e + 3]) : "memory");
                }
            }
            // the CTAs of the cluster share the rows: first every row's weights, a thread per row, then the rows,
            // four of a warp at a time from four CTAs at a time (half a warp to a row up to 64 channels).  A part counts
            // with a factor of 0 too, so that an infinite value whose weight has underflowed stays seen, as within a part
            // (one that a row does not see at all is warp 10's business).
            cluster_sync();
            constexpr uint32_t kLanes = DP / 4, kRows = 32 / kLanes, kBatch = 4, kFrom = 4;
            const uint32_t ranks = p.cluster, used = p.tokens * p.group, here = n_here * p.group, weights = q_smem;      // weights: Q is done with; 8 factors and 1 / l per row
            auto place = [&](uint32_t x) { return x + (x >= used ? 128 - used : 0); };       // row x of those in use, counted over both tiles
            const uint32_t share = (here + ranks - 1) / ranks, x_lo = rank * share, x_hi = min(here, x_lo + share);
            if (x_lo + tid < x_hi) {
                float2 y[8];
                float M = -INFINITY, sum = 0.0f;
#pragma unroll
                for (uint32_t s = 0; s < 8; s++) {
                    y[s] = make_float2(-INFINITY, 0.0f);
                    if (s < ranks) y[s] = ld_cluster2(smem_of(ring + L::out + place(x_lo + tid) * 8, s));
                }
#pragma unroll
                for (uint32_t s = 0; s < 8; s++) M = fmaxf(M, y[s].x);
#pragma unroll
                for (uint32_t s = 0; s < 8; s++) {
                    const float f = y[s].x == -INFINITY ? (y[s].y == 0.0f ? 0.0f : 1.0f) : ex2(y[s].x - M);
                    sum += y[s].y * f;
                    y[s].x = f;
                }
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                for (uint32_t s = 0; s < 8; s++) asm volatile("st.shared.f32 [%0], %1;" ::"r"(weights + (tid * 8 + s) * 4), "f"(y[s].x == 0.0f ? 0.0f : y[s].x * inv) : "memory");
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const uint32_t c = lane % kLanes * 4;
            for (uint32_t x0 = x_lo + warp * kRows + lane / kLanes; x0 - lane / kLanes < x_hi && ok; x0 += kBatch * 8 * kRows) {
                float4 o[kBatch];
#pragma unroll
                for (uint32_t b = 0; b < kBatch; b++) o[b] = make_float4(0, 0, 0, 0);
                for (uint32_t s0 = 0; s0 < ranks; s0 += kFrom) {
                    float4 v[kFrom][kBatch];
#pragma unroll
                    for (uint32_t k = 0; k < kFrom; k++) {
                        const uint32_t from = smem_of(ring, min(s0 + k, ranks - 1));
#pragma unroll
                        for (uint32_t b = 0; b < kBatch; b++) {
                            const uint32_t R = place(min(x0 + b * 8 * kRows, here - 1));
                            if (s0 + k < ranks) v[k][b] = ld_cluster4(from + R * DP * 4 + (((c >> 2) ^ (R & 7)) << 4));
                        }
                    }
#pragma unroll
                    for (uint32_t k = 0; k < kFrom; k++)
                        if (s0 + k < ranks)
#pragma unroll
                            for (uint32_t b = 0; b < kBatch; b++) {
                                float f;
                                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(weights + (min(x0 + b * 8 * kRows, x_hi - 1) - x_lo) * 32 + (s0 + k) * 4) : "memory");
                                o[b].x += v[k][b].x * f; o[b].y += v[k][b].y * f; o[b].z += v[k][b].z * f; o[b].w += v[k][b].w * f;
                            }
                }
#pragma unroll
                for (uint32_t b = 0; b < kBatch; b++) {
                    const uint32_t x = x0 + b * 8 * kRows, i = x * p.group_mul >> 16, head = kh * p.group + x - i * p.group;
                    if (x < x_hi && c < D)
                        *reinterpret_cast<uint2 *>(static_cast<T *>(p.O) + (uint64_t)(it.q0 + it.first + i) * p.ldo + (uint64_t)head * D + c) =
                            make_uint2(pack2<T>(o[b].x, o[b].y), pack2<T>(o[b].z, o[b].w));
                }
            }
        } else if (PREFIX && ok && tile < n_tiles) {
            // fp32 parts, through the memory of the warp's own rows of Q (their products are done), 32 channels at a
            // time, so that stores are whole lines; a thread storing its own row touches 32 lines per instruction
            const uint32_t buf = q_smem + tile * L::tile + (warp & 3) * 32 * 128;
            auto at_of = [&](uint32_t R) {
                const uint32_t q = R * p.group_mul >> 16;
                return ((uint64_t)(it.first + tile * p.tokens + q) * p.heads + kh * p.group + R - q * p.group) * p.splits + split;
            };
            if (mine) p.part_ml[at_of(row)] = make_float2(m == -INFINITY ? -INFINITY : m * sc, l);
            for (uint32_t c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_ld32(o_addr + c, o);
                tmem_wait_ld();
                pin32(o);
#pragma unroll
                for (uint32_t e = 0; e < 8; e++)
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(buf + lane * 128 + ((e ^ (lane & 7)) << 4)), "r"(o[4 * e]), "r"(o[4 * e + 1]),
                                 "r"(o[4 * e + 2]), "r"(o[4 * e + 3]) : "memory");
                __syncwarp();
#pragma unroll
                for (uint32_t r0 = 0; r0 < 32; r0 += 4) {
                    const uint32_t r = r0 + lane / 8, e = lane & 7, R = (warp & 3) * 32 + r;
                    uint4 y;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w) : "r"(buf + r * 128 + ((e ^ (r & 7)) << 4)) : "memory");
                    if (R < p.tokens * p.group && tile * p.tokens + (R * p.group_mul >> 16) < n_here && c + e * 4 < D)
                        *reinterpret_cast<uint4 *>(p.part_o + at_of(R) * D + c + e * 4) = y;
                }
                __syncwarp();
            }
        } else if (!PREFIX && ok && tile < n_tiles) {
            // The warp's rows through the memory of its own rows of Q (their products are done), so that lanes
            // store neighbouring chunks of a row; a thread storing its own row touches 32 lines per instruction.
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;                           // no visible key, or none above -infinity: zeros
            const uint32_t buf = q_smem + tile * L::tile + (warp & 3) * 32 * 128;    // rows of 128 bytes, 64 channels to a slab
#pragma unroll
            for (uint32_t c = 0; c < DP; c += 32) {
                if (c >= D) break;
                uint32_t o[32] = {};
                if (n > 0) {
                    tmem_ld32(o_addr + c, o);
                    tmem_wait_ld();
                    pin32(o);
                }
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) {
                    uint32_t y[4];
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        y[x] = vis == 0 ? 0u : pack2<T>(__uint_as_float(o[8 * e + 2 * x]) * inv, __uint_as_float(o[8 * e + 2 * x + 1]) * inv);
                    const uint32_t chunk = (c % 64) / 8 + e;
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(buf + c / 64 * 16384 + lane * 128 + ((chunk ^ (lane & 7)) << 4)), "r"(y[0]), "r"(y[1]),
                                 "r"(y[2]), "r"(y[3]) : "memory");
                }
            }
            __syncwarp();
            constexpr uint32_t kChunks = DP / 8, kRows = 32 / kChunks;               // lanes per row, rows per pass
            const uint32_t chunk = lane % kChunks;
#pragma unroll 4
            for (uint32_t r0 = 0; r0 < 32; r0 += kRows) {
                const uint32_t r = r0 + lane / kChunks, R = (warp & 3) * 32 + r, q = R * p.group_mul >> 16, i = tile * p.tokens + q;
                uint4 y;
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                             : "r"(buf + chunk / 8 * 16384 + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)) : "memory");
                if (R < p.tokens * p.group && i < n_here && chunk * 8 < D)
                    *reinterpret_cast<uint4 *>(static_cast<T *>(p.O) + (uint64_t)(it.q0 + it.first + i) * p.ldo + (uint64_t)(kh * p.group + R - q * p.group) * D + chunk * 8) = y;
            }
        }
    } else if (warp == 8) {
        // ---- loads -------------------------------------------------------------------------------
        bool ok = true;
        const uint32_t group = p.group;
        auto load_q = [&](uint32_t t) {
            mbar_expect(b_q + 8 * t, slabs * p.tokens * group * 128);
            for (uint32_t s = 0; s < slabs; s++)
                tma_load_3d(q_smem + t * L::tile + s * 16384, &map_q, b_q + 8 * t, s * 64, kh * group, it.q0 + it.first + t * p.tokens);
        };
        if (lane == 0 && n > 0) load_q(0);                                          // then K, which tile 0 waits for, then the rest
        if constexpr (PREFIX) {
            // A block is up to eight pages of up to two slabs, a box each: lane s * 8 + g loads slab s of page g,
            // whose number it looked up a block ahead.
            const uint32_t size = 1u << p.page_shift, g = lane & 7, s = lane >> 3;
            auto page_of = [&](uint32_t i) -> int32_t {                             // outside the cache: a page that reads as zeros
                const uint32_t key = (it.block0 + i) * kKeys + g * size;
                if (i >= n || g * size >= kKeys || key >= p.prefix_len) return (int32_t)p.n_pages;
                const uint32_t page = (uint32_t)p.prefix_table[key >> p.page_shift];
                return page < p.n_pages ? (int32_t)page : (int32_t)p.n_pages;
            };
            int32_t page = page_of(0), next = page_of(1);
            for (uint32_t x = 0; x < 2 * n && ok; x++) {                            // K0 V0 K1 V1 ...
                const uint32_t st = x % L::stages, use = x / L::stages, i = x >> 1;
                if (use > 0 && !mbar_wait_warp(b_empty + 8 * st, (use - 1) & 1, abort_word)) { ok = false; break; }
                issued = x + 1;
                const uint32_t bar = b_full + 8 * st, keys = min(kKeys, p.prefix_len - (it.block0 + i) * kKeys), pages = (keys + size - 1) >> p.page_shift;
                if (lane == 0) mbar_expect(bar, slabs * pages * size * 128);
                __syncwarp();
                if (x == 1 && lane == 0 && n_tiles > 1) load_q(1);
                if (g < pages && s < slabs) tma_load_4d(ring + st * L::tile + s * 16384 + g * size * 128, x & 1 ? &map_v : &map_k, bar, s * 64, 0, kh, page);
                if (x & 1) { page = next; next = page_of(i + 2); }
            }
        } else if (lane == 0) {
            for (uint32_t x = 0; x < 2 * n && ok; x++) {                            // K0 V0 K1 V1 ...
                const uint32_t st = x % L::stages, use = x / L::stages, i = x >> 1;
                if (use > 0 && !mbar_wait(b_empty + 8 * st, (use - 1) & 1, abort_word)) { ok = false; break; }
                issued = x + 1;
                const uint32_t dst = ring + st * L::tile, bar = b_full + 8 * st, j0 = (it.block0 + i) * kKeys;
                if (x == 1 && n_tiles > 1) load_q(1);
                mbar_expect(bar, slabs * 16384);
                for (uint32_t s = 0; s < slabs; s++) tma_load_3d(dst + s * 16384, x & 1 ? &map_v : &map_k, bar, s * 64, kh, it.k0 + j0);
            }
        }
        ok = __shfl_sync(0xffffffffu, (uint32_t)ok, 0);
        // zeros over the values that nobody here sees
        if (ok && n > 0 && cut) {
            const uint32_t x = 2 * n - 1, st = x % L::stages;
            if (mbar_wait_warp(b_full + 8 * st, x / L::stages & 1, abort_word)) {
                const uint32_t from = last_key - (it.block0 + n - 1) * kKeys;
                for (uint32_t s = 0; s < slabs; s++)
                    for (uint32_t a = from * 128 + lane * 16; a < 16384; a += 512)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(ring + st * L::tile + s * 16384 + a), "r"(0u) : "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(b_fix);
            }
        }
    } else if (warp == 9) {
        // ---- products ----------------------------------------------------------------------------
        if (n > 0) {
            const uint32_t steps = (D + 15) / 16, last_step = steps - 1;
            const uint32_t desc_s = mma_desc(kBf16, 128, false), desc_o = mma_desc(kBf16, steps * 16, true);
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const bool leader = elect_one();
            bool ok = true;
            const uint32_t k_hi = smem_desc(0, 0, 1024) >> 32, v_hi = smem_desc(0, 16384, 1024) >> 32;
            auto slot_lo = [&](uint32_t addr, uint32_t lead) { return (uint32_t)smem_desc(addr, lead, 1024); };
            auto scores = [&](uint32_t t, uint32_t x) {                              // S_t = Q_t K^T, K in ring use x
                const uint32_t kb = slot_lo(ring + x % L::stages * L::tile, 0), qb = slot_lo(q_smem + t * L::tile, 0);
                if (leader) {
#pragma unroll
                    for (uint32_t k = 0; k < DP / 16; k++) {
                        const uint32_t off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
                        if (k <= last_step) mma_ss(tm + t * 128, qb + off, k_hi, kb + off, k_hi, desc_s, k > 0);
                    }
                    tc_commit(b_s + 8 * t);
                }
                __syncwarp();
            };
            auto full = [&](uint32_t x) { return mbar_wait_warp(b_full + 8 * (x % L::stages), x / L::stages & 1, abort_word); };
            // A wait costs one or two hundred cycles even when there is nothing to wait for, a commit as much: those for
            // loads stand behind products just issued, and nothing stands between the last product of a step and
            // the wait for the first weights of the next.
            auto values_in = [&](uint32_t i) { return full(2 * i + 1) && (i + 1 < n || !cut || mbar_wait_warp(b_fix, 0, abort_word)); };
            ok = full(0);
            for (uint32_t t = 0; t < n_tiles && ok; t++) {
                ok = mbar_wait_warp(b_q + 8 * t, 0, abort_word);
                if (ok) { tc_fence_after(); scores(t, 0); }
            }
            if (ok && leader) tc_commit(b_empty);
            ok = ok && values_in(0) && (n == 1 || full(2));
            for (uint32_t i = 0; i < n && ok; i++) {
                const bool last = i + 1 == n;
                const uint32_t vb = slot_lo(ring + (2 * i + 1) % L::stages * L::tile, 16384);
#pragma unroll
                for (uint32_t t = 0; t < 2; t++) {
                    if (t >= n_tiles || !ok) break;
#pragma unroll
                    for (uint32_t half = 0; half < 2; half++) {                      // O_t += P_t V, sixteen keys at a time
                        ok = ok && mbar_wait_warp(b_p + 16 * t + 8 * half, i & 1, abort_word);
                        if (!ok) break;
                        tc_fence_after();
                        if (leader) {
#pragma unroll
                            for (uint32_t k = 0; k < 4; k++)
                                mma_ts(tm + 256 + t * DP, tm + t * 128 + (4 * half + k) * 8, vb + (4 * half + k) * 128, v_hi, desc_o, i > 0 || half > 0 || k > 0);
                            if (t == 0 && half == 0 && i > 0) {                         // what the step before read
                                tc_commit(b_empty + 8 * ((2 * i - 1) % L::stages));
                                tc_commit(b_empty + 8 * (2 * i % L::stages));
                            }
                        }
                        __syncwarp();
                        if (t + 1 == n_tiles && half == 0 && !last) ok = values_in(i + 1) && (i + 2 == n || full(2 * i + 4));
                    }
                    if (!ok) break;
                    if (!last) scores(t, 2 * i + 2);
                    else if (leader) tc_commit(b_o + 8 * t);
                }
                __syncwarp();
            }
        }
    } else if (!PREFIX && warp == 10 && it.any && p.causal) {
        // ---- values that some rows here see and others do not: all finite? --------------------------
        const uint32_t from = it.visible(it.first);                                  // (every CTA of a cluster looks, and finds the same)
        uint32_t found = 0;
        const uint32_t per = D / 8;                                                  // 16-byte words per row
        for (uint32_t x = lane; x < (last_key - from) * per; x += 32) {
            const uint32_t j = from + x / per, c = x % per * 8;
            const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.V) + (uint64_t)(it.k0 + j) * p.ldv + (uint64_t)kh * D + c);
            constexpr uint32_t e = kBf16 ? 0x7f807f80u : 0x7c007c00u;                // exponent bits; all set in a half: not finite
            for (uint32_t y : {v.x, v.y, v.z, v.w}) {
                const uint32_t b = y & e;
                if ((b & 0xffffu) == (e & 0xffffu) || (b >> 16) == (e >> 16)) found = 1;
            }
        }
        if (__any_sync(0xffffffffu, found) && lane == 0) bad_values = 1;
    } else if (warp == 11 && p.wait_polls && n > 0) {
        // ---- the caller's limit: ends the waits of the others unless the last product is done by then -----------
        mbar_poll(b_o + 8 * (n_tiles - 1), 0, abort_word, p.wait_polls);             // (tested in the waits themselves it costs a long prompt 3 %)
    }
    __syncwarp();
    if (SPLIT && warp >= 8 && spread) cluster_sync();         // the one the softmax warps pass before they join
    __syncthreads();
    if (abort_flag) {
        // a wait ran out (never in a healthy run with the default limit): report, then let copies and products in flight end
        if (tid == 0) atomicOr(p.status, 1u);
        uint32_t never = 0;
        if (warp == 9 && n > 0) {
            __syncwarp();
            if (elect_one()) tc_commit(b_end);       // arrives when every product issued so far is done
            mbar_wait_warp(b_end, 0, &never);
        }
        if (tid == 8 * 32 && n > 0) {
            for (uint32_t t = 0; t < n_tiles; t++) mbar_wait(b_q + 8 * t, 0, &never);
            for (uint32_t x = issued > L::stages ? issued - L::stages : 0; x < issued; x++) mbar_wait(b_full + 8 * (x % L::stages), x / L::stages & 1, &never);
        }
        __syncwarp();
        __syncthreads();
    }
    if (SPLIT && spread) cluster_sync();     // nobody leaves while its memory is read
    if (!PREFIX && bad_values && !abort_flag && rank == 0 && it.any) {
        __syncthreads();                     // over the rows just written
        for (uint32_t x = warp; x < n_here * p.group; x += kTcThreads / 32) {
            const uint32_t i = it.first + x / p.group;
            attend_row<T>(p, it.q0 + i, kh * p.group + x % p.group, kh, it.k0, it.visible(i));
        }
    }
    if (warp == 9) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
}

}  // namespace sptmm
