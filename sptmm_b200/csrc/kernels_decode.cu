// kernels_decode.cu -- attention of one new token per sequence over a paged cache, behind an optional
// prefix that the batch shares.
//
// The reference has no attention (its only operator is the matmul, main.cu:993-1961).  HBM bound: a key
// and its value are read once and used for the query heads that share them.  Three kernels, launched
// with programmatic overlap:
//   k_attention_tc<.., true>   (only with a prefix and more than 32 rows) all rows of the batch against the
//                              prefix, each part of its keys in another CTA; see attention_tc.cuh
//   k_decode                   every sequence's own keys, and the prefix's for few rows
//   k_decode_join              the parts of a row -> one softmax: with parts (m_i, l_i, o_i) and M = max m_i,
//                              O = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i
// k_decode splits the work by keys, not by sequences: all (sequence, key head) units are laid end to end
// in blocks of 64 keys and every CTA takes an equal run of blocks, wherever sequences begin and end in
// it, so that one sequence of 128k tokens fills the GPU as well as 64 of different lengths do.  The
// lengths are read on the device.  Unit u's piece in CTA c is number u + c: along the walk either u or c
// grows, so numbers are unique and a unit's pieces are neighbours.
// Within a CTA each of four warps takes 16 keys of a block for itself: K and V go through its own ring
// of asynchronous copies (16-byte chunks, XOR-swizzled), scores and P V through m16n8k16 products with the
// (at most 16) query heads of the group as rows, and running maximum and sum stay in its registers; the
// warps meet only at the end of a unit.  Scores cost 8 KB of smem reads per 16 keys against 8 KB from HBM;
// the products are far from any limit, so tensor memory would buy nothing here.  A warp's requests run on into
// the CTA's next unit while one is joined: 24 KB per warp, 192 KB per SM on their way at any time.
// Measured (20 heads over 5, 128 channels): two sequences of 128k tokens (668 MB) 110 us, 6.1 TB/s, 0.93 of the
// copy rate; 64 sequences of 1 to 6991 tokens (191 MB) 39 us, 4.9 TB/s, of which 2.5 us pass before the first
// keys are requested (lengths, then pages) and 3 us between the last CTA's end and the joining kernel's; one of
// 300 tokens 6.7 us.  Draining the ring at the end of every unit and equal blocks whatever the units: 63 us
// for the 64, because a CTA met up to twenty one-block sequences.  A warp that joins a row's parts one after
// the other: 23 us for the rows of 128k tokens instead of 5.
#include "attention_tc.cuh"

namespace sptmm {

constexpr uint32_t kDecodeWarps = 4, kDecodeThreads = 32 * kDecodeWarps, kTileKeys = 16, kBlockKeys = kTileKeys * kDecodeWarps;
constexpr uint32_t kMaxDecodeCtas = 384;     // two per SM on up to 192 SMs
constexpr uint32_t kDecodeStages = 3;

struct DecodeParams {
    const void *Q;
    void *O;
    CacheView cache;
    const int32_t *lengths, *table;
    uint64_t ldq, ldo;
    uint32_t B, heads, group, max_pages, row_tiles;            // row_tiles: tiles of 16 query heads per key head
    uint32_t partial;                        // never store to O: the prefix's parts are still to be joined
    uint32_t beside;                         // the prefix's kernel runs before this one
    // A prefix read by this kernel: `prefix_tiles` tiles of up to 16 of the batch's rows per key head; 0: none
    const int32_t *prefix_table;
    uint32_t prefix_len, prefix_tiles;
    uint32_t piece_rows;                     // rows between pieces
    float scale;                             // scale * log2(e)
    uint2 *span;                             // [unit]: its first and last piece
    float2 *part_ml;                         // [piece][piece_rows]: (m in powers of two, l); l and O 2^up times as large (WeightRange)
    float *part_o;                           // [piece][piece_rows][head_dim]
    // the prefix's parts
    const float2 *prefix_ml;
    const float *prefix_o;
    uint32_t splits;
    // Beside the prefix's kernel only this many CTAs find an SM at once, the others when that kernel ends; `lead`:
    // blocks that the early ones have done by then.  0: all start together.
    uint32_t early, lead;
};

__device__ __forceinline__ uint32_t own_keys(const DecodeParams &p, uint32_t b)
{
    const uint64_t room = (uint64_t)p.max_pages << p.cache.page_shift;
    return (uint32_t)min(room, (uint64_t)max(p.lengths[b], 0));
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (__is_same(T, __half))
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes, or zeros where `bytes` is 0
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint32_t bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <int DP> struct DecodeLayout {
    static constexpr uint32_t row = DP * 2, tile = kTileKeys * row, stage = 2 * tile;      // K tile, V tile
    static constexpr uint32_t ring = kDecodeWarps * kDecodeStages * stage;
    static constexpr uint32_t smem = ring + kDecodeWarps * 8 * DP * 4;                      // and eight rows of every warp's sums
};

// A run of blocks of one unit that a CTA takes on.  b = kPrefix: a tile of the batch's rows over the prefix.
constexpr uint32_t kPrefix = 0xffffffffu;
struct Piece {
    uint32_t b, kh, rt, rows, unit, len, blk0, blk1, blocks;       // blocks: of the whole unit; blk0 .. blk1: this piece
};

// The CTA's way through its run [w, w1) of the units laid end to end: the prefix's, if it is read here, then the
// sequences' one after the other.  A unit counts kUnitCost blocks more than it has, the time its first loads and
// its end take, so that a CTA with many short units gets fewer blocks.
constexpr uint32_t kUnitCost = 2;
struct Walk {
    uint64_t w, w1, at;                      // at: where sequence b begins
    uint32_t b;                              // kPrefix, 0, 1, ...
    __device__ __forceinline__ bool next(const DecodeParams &p, Piece &x)
    {
        while (w < w1) {
            const bool pre = b == kPrefix;
            const uint32_t tiles = pre ? p.prefix_tiles : p.row_tiles, per_seq = p.cache.kv_heads * tiles;
            const uint32_t len = pre ? p.prefix_len : own_keys(p, b), nb = (len + kBlockKeys - 1) / kBlockKeys, cost = nb + kUnitCost;
            if (nb == 0 || w >= at + (uint64_t)cost * per_seq) { at += nb ? (uint64_t)cost * per_seq : 0; b++; continue; }
            const uint32_t sub = (uint32_t)((w - at) / cost), v0 = (uint32_t)(w - at - (uint64_t)sub * cost), v1 = (uint32_t)min((uint64_t)cost, v0 + (w1 - w));
            w += v1 - v0;
            x.blk0 = v0 > kUnitCost ? v0 - kUnitCost : 0; x.blk1 = v1 > kUnitCost ? v1 - kUnitCost : 0;
            if (x.blk0 == x.blk1) continue;  // only a part of the cost, none of the blocks
            x.b = b; x.kh = sub / tiles; x.rt = sub % tiles; x.len = len; x.blocks = nb;
            x.rows = min(16u, (pre ? p.B * p.group : p.group) - x.rt * 16);
            x.unit = (pre ? 0 : p.cache.kv_heads * p.prefix_tiles + b * per_seq) + sub;
            return true;
        }
        x.blk0 = x.blk1 = 0;
        return false;
    }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kDecodeThreads)
k_decode(const DecodeParams p)
{
    using L = DecodeLayout<DP>;
    constexpr uint32_t chunks = DP / 8;      // 16-byte chunks of a row
    extern __shared__ __align__(1024) unsigned char dyn[];
    __shared__ uint64_t warp_sum[kDecodeWarps];
    __shared__ uint32_t start_b;
    __shared__ uint64_t start_w;
    __shared__ float2 ml[kDecodeWarps][16];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
    const uint32_t D = p.cache.head_dim, per_seq = p.cache.kv_heads * p.row_tiles;
    pdl_launch_dependents();
    // Behind the prefix's kernel this one starts when all that came before has ended (that kernel lets it go only
    // then) and reads nothing of the prefix's: it runs beside it, and waits at its own end so that the joining
    // kernel, which waits for this one, finds both done.  What came before is in L2 by then, but no wait of this kernel's
    // says that an SM's first-level cache holds nothing older: the fence drops it.  (Lengths, pages and Q read past that
    // cache instead: 64 sequences of 1 to 6991 tokens 44.5 us for 39.6.)
    auto end = [&]() { if (p.beside) pdl_wait_prior_grid(); };
    if (p.beside) __threadfence();
    else pdl_wait_prior_grid();
    // ---- this CTA's run: thread t sums a contiguous range of sequences ---------------------------------
    auto cost_of = [&](uint32_t b) -> uint64_t {
        const uint32_t nb = (own_keys(p, b) + kBlockKeys - 1) / kBlockKeys;
        return nb ? (uint64_t)(nb + kUnitCost) * per_seq : 0;
    };
    const uint32_t each = (p.B + kDecodeThreads - 1) / kDecodeThreads, b_lo = min(p.B, tid * each), b_hi = min(p.B, b_lo + each);
    uint64_t mine = 0;
    for (uint32_t b = b_lo; b < b_hi; b++) mine += cost_of(b);
    uint64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= (uint32_t)o) upto += y;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    const uint64_t prefix_cost = p.prefix_tiles ? (uint64_t)((p.prefix_len + kBlockKeys - 1) / kBlockKeys + kUnitCost) * p.cache.kv_heads * p.prefix_tiles : 0;
    uint64_t total = prefix_cost, before = prefix_cost + upto - mine;
    for (uint32_t w = 0; w < kDecodeWarps; w++) {
        if (w < warp) before += warp_sum[w];
        total += warp_sum[w];
    }
    // Equal runs; behind a prefix the early CTAs take `lead` blocks more than the late ones, or everything.  No CTA
    // between two that work may stay empty, or a unit's pieces would not be neighbours.
    const uint64_t lead = (uint64_t)p.early * p.lead;
    const bool late = p.early && total >= lead + gridDim.x;
    const uint64_t even = late ? total - lead : total, active = late ? gridDim.x : min((uint64_t)(p.early ? p.early : gridDim.x), total);
    if (cta >= active) { end(); return; }
    auto start_of = [&](uint64_t c) { return even * c / active + (late ? min(c, (uint64_t)p.early) * p.lead : 0); };
    Walk walk;
    walk.w = start_of(cta); walk.w1 = start_of(cta + 1);
    if (tid == 0 && walk.w < prefix_cost) { start_b = kPrefix; start_w = 0; }
    if (before <= walk.w && walk.w < before + mine) {
        uint64_t at = before;
        uint32_t b = b_lo;
        for (;; b++) {
            const uint64_t c = cost_of(b);
            if (walk.w < at + c) break;
            at += c;
        }
        start_b = b; start_w = at;
    }
    __syncthreads();
    walk.b = start_b; walk.at = start_w;

    Piece cur, nxt, iss;                     // worked on, after it, being requested (one of the two)
    if (!walk.next(p, cur)) { end(); return; }
    const uint32_t ring = smem_addr(dyn) + warp * kDecodeStages * L::stage;
    float *sums = reinterpret_cast<float *>(dyn + L::ring);
    // tile i of a piece, for this warp: keys from ((blk0 + i) * warps + warp) * 16
    auto key_of = [&](const Piece &x, uint32_t i) { return ((x.blk0 + i) * kDecodeWarps + warp) * kTileKeys; };
    auto page_of = [&](const Piece &x, uint32_t i) -> uint32_t {
        const uint32_t key = key_of(x, i);
        if (i >= x.blk1 - x.blk0 || key >= x.len) return 0xffffffffu;
        return (uint32_t)(x.b == kPrefix ? p.prefix_table : p.table + (uint64_t)x.b * p.max_pages)[key >> p.cache.page_shift];
    };
    uint32_t ii = 0, page_lane = page_of(cur, lane), page_next = page_of(cur, 32 + lane);      // pages of tiles ii & ~31 .. + 32 of `iss`, one per lane; the 32 after
    iss = cur;
    walk.next(p, nxt);
    uint32_t nxt_page = page_of(nxt, lane);
    bool on_next = false;                    // iss is nxt
    uint32_t ahead = 0, slot_in = 0, slot_out = 0, valid_bits = 0;      // tiles requested and not used; bit s: the tile in ring slot s lies in the cache
    auto request = [&]() {                   // fills the ring's free slots, into the next piece if need be
        while (ahead < kDecodeStages) {
            if (ii == iss.blk1 - iss.blk0) {
                if (on_next || nxt.blk0 == nxt.blk1) return;
                iss = nxt; on_next = true; ii = 0;
                page_lane = nxt_page; page_next = page_of(iss, 32 + lane);
            }
            const uint32_t page = __shfl_sync(0xffffffffu, page_lane, ii & 31);
            const uint32_t key0 = key_of(iss, ii);
            const bool good = page < p.cache.n_pages;
            valid_bits = (valid_bits & ~(1u << slot_in)) | (uint32_t)good << slot_in;
            const uint64_t base = good ? p.cache.at(page, iss.kh, key0 & (p.cache.page_size() - 1)) : 0;
            const uint32_t dst = ring + slot_in * L::stage;
#pragma unroll
            for (uint32_t x = 0; x < kTileKeys * chunks / 32; x++) {
                const uint32_t r = (x * 32 + lane) / chunks, c = (x * 32 + lane) % chunks;
                const uint32_t bytes = good && key0 + r < iss.len && c * 8 < D ? 16 : 0;
                const uint64_t off = bytes ? base + r * D + c * 8 : 0;
                const uint32_t to = dst + r * L::row + ((c ^ (r & 7)) << 4);
                copy16(to, static_cast<const T *>(p.cache.k) + off, bytes);
                copy16(to + L::tile, static_cast<const T *>(p.cache.v) + off, bytes);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            slot_in = slot_in + 1 == kDecodeStages ? 0 : slot_in + 1;
            ahead++; ii++;
            if ((ii & 31) == 0) { page_lane = page_next; page_next = page_of(iss, ii + 32 + lane); }
        }
    };
    request();
    uint32_t qa[DP / 16][4];                 // query rows as A fragments: rows lane / 4 and + 8, channels 2 (lane % 4) and + 8 of every sixteen
    auto load_q = [&](const Piece &x) {
        const T *q[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t r = x.rt * 16 + lane / 4 + h * 8;                         // of the group, or of the batch's rows
            const uint32_t b = x.b == kPrefix ? r / p.group : x.b, g = x.b == kPrefix ? r % p.group : r;
            q[h] = lane / 4 + h * 8 < x.rows ? static_cast<const T *>(p.Q) + (uint64_t)b * p.ldq + (uint64_t)(x.kh * p.group + g) * D : nullptr;
        }
#pragma unroll
        for (int k = 0; k < DP / 16; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t c = k * 16 + (lane & 3) * 2 + (e >> 1) * 8;
                qa[k][e] = q[e & 1] && c < D ? *reinterpret_cast<const uint32_t *>(q[e & 1] + c) : 0u;
            }
    };
    load_q(cur);
    for (;;) {
        float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0, 0};
#pragma unroll
        for (int n = 0; n < DP / 8; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[n][e] = 0.0f;
        const uint32_t tiles = cur.blk1 - cur.blk0, len = cur.len;
        for (uint32_t i = 0; i < tiles; i++) {
            request();
            static_assert(kDecodeStages == 3, "the waits below count three slots");
            if (ahead == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
            else if (ahead == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
            else asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
            const uint32_t key0 = key_of(cur, i), kb = ring + slot_out * L::stage, vb = kb + L::tile;
            if (key0 < len && (valid_bits >> slot_out & 1)) {
                float s[2][4] = {};
#pragma unroll
                for (int k = 0; k < DP / 16; k++) {
                    const uint32_t r = (lane & 7) + (lane >> 4) * 8, c = k * 2 + (lane >> 3 & 1);
                    uint32_t f[4];
                    ldsm4(kb + r * L::row + ((c ^ (r & 7)) << 4), f);
                    mma16816<T>(s[0], qa[k], f[0], f[1]);
                    mma16816<T>(s[1], qa[k], f[2], f[3]);
                }
                const uint32_t col = key0 + (lane & 3) * 2;
                if (key0 + kTileKeys > len) {
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) if (col + n * 8 + (e & 1) >= len) s[n][e] = -INFINITY;
                }
                float mx[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    mx[h] = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2)) * p.scale;
                }
                // scale down only when a maximum has grown by more than the lag (or is the first)
                const bool grow = (mx[0] > m[0] && (m[0] == -INFINITY || mx[0] - m[0] > WeightRange<T>::lag)) || (mx[1] > m[1] && (m[1] == -INFINITY || mx[1] - m[1] > WeightRange<T>::lag));
                if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const float m1 = fmaxf(m[h], mx[h]), f = m[h] == -INFINITY ? (m1 == -INFINITY ? 1.0f : 0.0f) : ex2(m[h] - m1);
                        m[h] = m1; l[h] *= f;
#pragma unroll
                        for (int n = 0; n < DP / 8; n++) { o[n][2 * h] *= f; o[n][2 * h + 1] *= f; }
                    }
                }
                uint32_t pa[4];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float base = m[h] == -INFINITY ? 0.0f : m[h] - WeightRange<T>::up;
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const float x = ex2(fmaf(s[n][2 * h], p.scale, -base)), y = ex2(fmaf(s[n][2 * h + 1], p.scale, -base));
                        l[h] += x + y;
                        pa[n * 2 + h] = pack2<T>(x, y);
                    }
                }
#pragma unroll
                for (int n = 0; n < DP / 16; n++) {
                    const uint32_t r = (lane & 7) + (lane >> 3 & 1) * 8, c = n * 2 + (lane >> 4);
                    uint32_t f[4];
                    ldsm4_t(vb + r * L::row + ((c ^ (r & 7)) << 4), f);
                    mma16816<T>(o[2 * n], pa, f[0], f[1]);
                    mma16816<T>(o[2 * n + 1], pa, f[2], f[3]);
                }
            }
            __syncwarp();                    // the slot may be filled again
            ahead--;
            slot_out = slot_out + 1 == kDecodeStages ? 0 : slot_out + 1;
        }
        // ---- on to the next piece: its loads and queries travel while this one's parts are joined ----
        const Piece done = cur;
        const bool more = nxt.blk0 != nxt.blk1;
        if (more) {
            if (!on_next) { iss = nxt; ii = 0; page_lane = nxt_page; page_next = page_of(iss, 32 + lane); }
            on_next = false;
            cur = nxt;
            walk.next(p, nxt);
            nxt_page = page_of(nxt, lane);
            request();
            load_q(cur);
        }
        // ---- the warps' parts -> one, eight rows at a time -------------------------------------------
        const uint32_t head0 = done.kh * p.group + done.rt * 16, rows = done.rows, piece = done.unit + cta;
        const bool whole = done.blk0 == 0 && done.blk1 == done.blocks && !p.partial;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (h * 8 >= (int)rows) break;
            __syncthreads();                 // what was joined before has been read
            const uint32_t r = lane / 4;
            if ((lane & 3) == 0) ml[warp][r] = make_float2(m[h], l[h]);
            if (r + h * 8 < rows)
#pragma unroll
                for (int n = 0; n < DP / 8; n++)
                    *reinterpret_cast<float2 *>(sums + (warp * 8 + r) * DP + n * 8 + (lane & 3) * 2) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
            __syncthreads();
            const uint32_t here = min(8u, rows - h * 8);
            for (uint32_t x = tid; x < here * (D / 4); x += kDecodeThreads) {
                const uint32_t q = x / (D / 4), c = x % (D / 4) * 4, row = q + h * 8;
                float4 v = make_float4(0, 0, 0, 0);
                float M = -INFINITY, sum = 0;
#pragma unroll
                for (uint32_t y = 0; y < kDecodeWarps; y++) M = fmaxf(M, ml[y][q].x);
#pragma unroll
                for (uint32_t y = 0; y < kDecodeWarps; y++) {
                    const float2 part = ml[y][q];
                    const float f = part.x == -INFINITY ? (part.y == 0.0f ? 0.0f : 1.0f) : ex2(part.x - M);      // l of 0 without a key, else not a number
                    const float4 z = *reinterpret_cast<const float4 *>(sums + (y * 8 + q) * DP + c);
                    sum += part.y * f;
                    v.x += z.x * f; v.y += z.y * f; v.z += z.z * f; v.w += z.w * f;
                }
                if (whole) {
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    *reinterpret_cast<uint2 *>(static_cast<T *>(p.O) + (uint64_t)done.b * p.ldo + (uint64_t)(head0 + row) * D + c) =
                        make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
                } else {
                    *reinterpret_cast<float4 *>(p.part_o + ((uint64_t)piece * p.piece_rows + row) * D + c) = v;
                    if (c == 0) p.part_ml[(uint64_t)piece * p.piece_rows + row] = make_float2(M, sum);
                }
            }
        }
        if (tid == 0) {
            if (done.blk0 == 0) p.span[done.unit].x = whole ? 0xffffffffu : piece;
            if (done.blk1 == done.blocks) p.span[done.unit].y = piece;
        }
        if (!more) break;
    }
    end();
}

// A CTA per (sequence, query head): joins the prefix's and the pieces' parts, a fourth of them per warp, all
// loads of a warp on their way together.
template <typename T>
__global__ void __launch_bounds__(128) k_decode_join(const DecodeParams p)
{
    __shared__ float2 ml[4];
    __shared__ float4 sums[4][32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane * 4, D = p.cache.head_dim;
    const uint32_t b = blockIdx.x / p.heads, h = blockIdx.x % p.heads, kh = h / p.group, g = h % p.group;
    const uint32_t unit = p.cache.kv_heads * p.prefix_tiles + (b * p.cache.kv_heads + kh) * p.row_tiles + g / 16, r = g % 16;
    const uint32_t R = b * p.group + g;      // among the batch's rows, of the prefix read by k_decode
    const uint64_t row = blockIdx.x;
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    uint32_t first = 0, count = 0, pre_first = 0, pre_count = p.splits;
    const uint2 span = p.span[unit];         // not written where there are no keys: looked at below
    if (own_keys(p, b) > 0) {
        if (span.x == 0xffffffffu) return;   // the whole unit went straight to O
        first = span.x; count = span.y - span.x + 1;
    }
    if (p.prefix_tiles) {
        const uint2 pre = p.span[kh * p.prefix_tiles + R / 16];
        pre_first = pre.x; pre_count = pre.y - pre.x + 1;
    }
    const uint32_t parts = pre_count + count, each = (parts + 3) / 4, i0 = min(parts, warp * each), i1 = min(parts, i0 + each);
    float M = -INFINITY, l = 0;
    float4 o = make_float4(0, 0, 0, 0);
    for (uint32_t i = i0; i < i1; i += 8) {
        float2 y[8];
        float4 v[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) {
            y[k] = make_float2(-INFINITY, 0.0f); v[k] = make_float4(0, 0, 0, 0);
            if (i + k < i1) {
                const uint32_t part = i + k;
                const bool split = part < p.splits;              // written by the prefix's kernel; else a piece
                const uint64_t at = split ? row * p.splits + part
                                          : part < pre_count ? (uint64_t)(pre_first + part) * p.piece_rows + R % 16
                                                             : (uint64_t)(first + part - pre_count) * p.piece_rows + r;
                y[k] = split ? p.prefix_ml[at] : p.part_ml[at];
                if (c < D) v[k] = *reinterpret_cast<const float4 *>((split ? p.prefix_o : p.part_o) + at * D + c);
            }
        }
        float m1 = M;
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) m1 = fmaxf(m1, y[k].x);
        const float f0 = M == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : ex2(M - m1);
        M = m1; l *= f0; o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) {
            const float f = y[k].x == -INFINITY ? (y[k].y == 0.0f ? 0.0f : 1.0f) : ex2(y[k].x - M);
            l += y[k].y * f;
            o.x += v[k].x * f; o.y += v[k].y * f; o.z += v[k].z * f; o.w += v[k].w * f;      // a factor of 0 too: an infinite value stays seen
        }
    }
    if (lane == 0) ml[warp] = make_float2(M, l);
    sums[warp][lane] = o;
    __syncthreads();
    if (warp || c >= D) return;
    M = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
    l = 0; o = make_float4(0, 0, 0, 0);
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
        const float f = ml[k].x == -INFINITY ? (ml[k].y == 0.0f ? 0.0f : 1.0f) : ex2(ml[k].x - M);
        const float4 v = sums[k][lane];
        l += ml[k].y * f;
        o.x += v.x * f; o.y += v.y * f; o.z += v.z * f; o.w += v.w * f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *reinterpret_cast<uint2 *>(static_cast<T *>(p.O) + (uint64_t)b * p.ldo + (uint64_t)h * D + c) = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
}

// How the prefix's keys are divided: over half of the SMs, while the sequences' own keys, whose number only the
// device knows, stream on the other half (k_decode's early CTAs).  More parts shorten the prefix but every part
// of a row is written and read once more in fp32.  Measured with 40 / 74 / 90 CTAs: 64 sequences of up to 700
// own keys behind 8192 (20 heads over 5, 128 channels) 27.9 / 27.4 / 29.8 us (34 on all SMs, one kernel after the
// other), 128 of up to 100 behind 16384 71.8 / 48.9 / 42.3, 16 of up to 4000 behind 2048 23.3 / 26.1 / 25.6.
constexpr uint32_t kPrefixCtas = 74;
struct PrefixPlan { uint32_t pairs, splits; };
static PrefixPlan plan_prefix(uint32_t B, uint32_t kv_heads, uint32_t group, uint32_t prefix_len)
{
    PrefixPlan pl{};
    if (!prefix_len) return pl;
    const uint32_t tokens = 128 / group, blocks = (prefix_len + kKeys - 1) / kKeys;
    pl.pairs = (B + 2 * tokens - 1) / (2 * tokens);
    const uint64_t items = (uint64_t)pl.pairs * kv_heads;
    const uint32_t want = items >= kPrefixCtas ? 1u : (uint32_t)(kPrefixCtas / items);
    pl.splits = want < blocks ? want : blocks;
    return pl;
}

// Up to this many rows (sequences times query heads per key head) a prefix is read by k_decode itself, a tile of 16
// rows as if it were one more sequence: no kernel of its own, no tile of 128 rows to fill.  Measured, own kernel
// against read here: 4 rows over 8192 keys of five key heads 21.1 / 11.8 us, 16 rows 21.5 / 14.0, 32 rows over
// 16384 keys of eight 47.4 / 26.8; 40 rows 35.3 / 33.1; 64 rows 22.1 / 23.1, 128 rows 22.2 / 31.6.
constexpr uint64_t kPrefixRows = 32;
struct WorkspacePlan {
    uint64_t span, part_ml, part_o, prefix_ml, prefix_o, bytes, units;
    uint32_t row_tiles, prefix_tiles, piece_rows;
    PrefixPlan prefix;                       // splits 0: no kernel for the prefix
};
static WorkspacePlan plan_workspace(uint32_t B, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t prefix_len)
{
    WorkspacePlan w{};
    const uint32_t group = heads / kv_heads;
    w.row_tiles = (group + 15) / 16;
    if (prefix_len && (uint64_t)B * group <= kPrefixRows) w.prefix_tiles = (B * group + 15) / 16;
    else w.prefix = plan_prefix(B, kv_heads, group, prefix_len);
    w.piece_rows = w.prefix_tiles || group > 16 ? 16 : group;
    w.units = (uint64_t)B * kv_heads * w.row_tiles + (uint64_t)kv_heads * w.prefix_tiles;
    const uint64_t pieces = w.units + kMaxDecodeCtas, parts = (uint64_t)B * heads * w.prefix.splits;
    uint64_t cur = 0;
    auto take = [&](uint64_t bytes) { const uint64_t at = cur; cur += (bytes + 255) & ~255ull; return at; };
    w.span = take(w.units * sizeof(uint2));
    w.part_ml = take(pieces * w.piece_rows * sizeof(float2));
    w.part_o = take(pieces * w.piece_rows * head_dim * sizeof(float));
    w.prefix_ml = take(parts * sizeof(float2));
    w.prefix_o = take(parts * head_dim * sizeof(float));
    w.bytes = cur;
    return w;
}

// What suffices for every batch of up to B sequences.  The plan of one batch alone may need less than that of a smaller
// one: a prefix is divided into fewer parts per row as the pairs of tiles get more, and few rows come in pieces of 16.
// Between two such steps the size grows with B, so the largest is at the end of one or at B; from kPrefixCtas
// pairs on there is one part per row.
static uint64_t workspace_bytes_up_to(uint32_t B, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t prefix_len)
{
    uint64_t most = plan_workspace(B, heads, kv_heads, head_dim, prefix_len).bytes;
    if (!prefix_len) return most;
    auto look = [&](uint64_t b) {
        if (b >= B) return;
        const uint64_t bytes = plan_workspace((uint32_t)b, heads, kv_heads, head_dim, prefix_len).bytes;
        if (bytes > most) most = bytes;
    };
    const uint32_t group = heads / kv_heads;
    look(kPrefixRows / group);               // the last batch whose prefix k_decode reads
    for (uint64_t pairs = 1; pairs <= kPrefixCtas; pairs++) look(pairs * 2 * (128 / group));
    return most;
}

template <typename T, int DP>
static cudaError_t launch_decode(const DecodeParams &d, const TcParams &t, const PrefixPlan &pl, const CUtensorMap *maps, uint32_t ctas, void *stream, bool pdl)
{
    cudaError_t e;
    if (pl.splits) {
        e = cudaFuncSetAttribute(k_attention_tc<T, DP, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcLayout<DP>::smem);
        if (e != cudaSuccess) return e;
        e = launch(k_attention_tc<T, DP, true>, dim3(pl.pairs * t.kv_heads * pl.splits), dim3(kTcThreads), TcLayout<DP>::smem, stream, pdl, t, maps[0], maps[1], maps[2]);
        if (e != cudaSuccess) return e;
        pdl = true;
    }
    e = cudaFuncSetAttribute(k_decode<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeLayout<DP>::smem);
    if (e != cudaSuccess) return e;
    e = launch(k_decode<T, DP>, dim3(ctas), dim3(kDecodeThreads), DecodeLayout<DP>::smem, stream, pdl, d);
    if (e != cudaSuccess) return e;
    return launch(k_decode_join<T>, dim3(d.B * d.heads), dim3(128), 0, stream, true, d);
}

}  // namespace sptmm

using namespace sptmm;

extern "C" uint64_t sptmm_attention_decode_workspace(uint32_t B, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t prefix_len)
{
    const char *who = "attention_decode_workspace";
    if (check_heads(who, heads, kv_heads, head_dim, SPTMM_F16) != SPTMM_OK) return 0;
    if (B > 65536 || prefix_len > 0x7fffffffu - 128) { fail(SPTMM_ERR_INVALID, "%s: B=%u prefix_len=%u", who, B, prefix_len); return 0; }
    return workspace_bytes_up_to(B, heads, kv_heads, head_dim, prefix_len);
}

extern "C" int sptmm_attention_decode(const sptmm_decode_params *a, uint32_t flags, void *stream)
{
    const char *who = "attention_decode";
    if (!a || !a->cache) return fail(SPTMM_ERR_INVALID, "%s: null pointer", who);
    int rc = check_heads(who, a->heads, a->cache->kv_heads, a->cache->head_dim, a->cache->dtype);
    DecodeParams prm{};
    if (rc == SPTMM_OK) rc = check_cache(who, a->cache, prm.cache);
    if (rc != SPTMM_OK) return rc;
    if (flags & ~(uint32_t)SPTMM_LAUNCH_PDL) return fail(SPTMM_ERR_INVALID, "%s: flags %u", who, flags);
    if (!(a->scale >= 0.0f) || a->scale > 1e30f) return fail(SPTMM_ERR_INVALID, "%s: scale %g", who, (double)a->scale);
    prm.ldq = a->ldq; prm.ldo = a->ldo;
    const uint64_t q_width = (uint64_t)a->heads * a->cache->head_dim;
    rc = check_stride(who, "ldq", prm.ldq, q_width, 8);
    if (rc == SPTMM_OK) rc = check_stride(who, "ldo", prm.ldo, q_width, 8);
    if (rc != SPTMM_OK) return rc;
    if (a->B > 65536) return fail(SPTMM_ERR_UNSUPPORTED, "%s: B=%u (at most 65536)", who, a->B);
    if ((uint64_t)a->max_pages * a->cache->page_size > 0x7fffffffull || a->prefix_len > 0x7fffffffu - 128)
        return fail(SPTMM_ERR_INVALID, "%s: max_pages=%u of %u slots, prefix_len=%u", who, a->max_pages, a->cache->page_size, a->prefix_len);
    if (a->B == 0) return SPTMM_OK;
    if (!a->Q || !a->O || !a->lengths || (a->max_pages && !a->table) || (a->prefix_len && !a->prefix_table))
        return fail(SPTMM_ERR_INVALID, "%s: null pointer", who);
    if (!aligned16(a->Q) || !aligned16(a->O) || !aligned16(a->workspace)) return fail(SPTMM_ERR_INVALID, "%s: an address is not 16-byte aligned", who);
    if (!aligned4(a->lengths) || !aligned4(a->table) || !aligned4(a->prefix_table)) return fail(SPTMM_ERR_INVALID, "%s: an index array is not 4-byte aligned", who);
    const uint32_t kv_heads = a->cache->kv_heads, D = a->cache->head_dim, group = a->heads / kv_heads, dtype = a->cache->dtype;
    const WorkspacePlan w = plan_workspace(a->B, a->heads, kv_heads, D, a->prefix_len);
    if (!a->workspace || a->workspace_bytes < w.bytes)
        return fail(SPTMM_ERR_INVALID, "%s: workspace of %llu bytes, %llu needed", who, (unsigned long long)(a->workspace ? a->workspace_bytes : 0), (unsigned long long)w.bytes);
    if (w.units + kMaxDecodeCtas > 0x7fffffffull || (uint64_t)w.prefix.pairs * kv_heads * w.prefix.splits > 0x7fffffffull ||
        (uint64_t)a->B * a->heads > 0x7fffffffull)
        return fail(SPTMM_ERR_UNSUPPORTED, "%s: %u sequences of %u key heads in one call", who, a->B, kv_heads);
    char *ws = static_cast<char *>(a->workspace);
    prm.Q = a->Q; prm.O = a->O; prm.lengths = a->lengths; prm.table = a->table;
    prm.B = a->B; prm.heads = a->heads; prm.group = group; prm.max_pages = a->max_pages;
    prm.row_tiles = w.row_tiles; prm.piece_rows = w.piece_rows; prm.partial = a->prefix_len ? 1 : 0;
    prm.beside = w.prefix.splits ? 1 : 0; prm.prefix_table = a->prefix_table; prm.prefix_len = a->prefix_len; prm.prefix_tiles = w.prefix_tiles;
    prm.scale = (a->scale > 0.0f ? a->scale : 1.0f / sqrtf((float)D)) * 1.4426950408889634f;      // log2(e): the kernels work with exp2
    prm.span = reinterpret_cast<uint2 *>(ws + w.span);
    prm.part_ml = reinterpret_cast<float2 *>(ws + w.part_ml); prm.part_o = reinterpret_cast<float *>(ws + w.part_o);
    prm.prefix_ml = reinterpret_cast<float2 *>(ws + w.prefix_ml); prm.prefix_o = reinterpret_cast<float *>(ws + w.prefix_o);
    prm.splits = w.prefix.splits;
    TcParams t{};
    CUtensorMap maps[3];
    if (w.prefix.splits) {
        t.Q = a->Q; t.ldq = prm.ldq; t.T = a->B; t.heads = a->heads; t.kv_heads = kv_heads; t.group = group; t.head_dim = D;
        t.tokens = 128 / group; t.group_mul = 65535 / group + 1; t.scale = prm.scale;
        t.prefix_table = a->prefix_table; t.prefix_len = a->prefix_len; t.n_pages = prm.cache.n_pages; t.page_shift = prm.cache.page_shift;
        t.splits = w.prefix.splits; t.cluster = 1;
        t.part_o = reinterpret_cast<float *>(ws + w.prefix_o); t.part_ml = reinterpret_cast<float2 *>(ws + w.prefix_ml);
        rc = attention_status_word(&t.status);
        if (rc != SPTMM_OK) return rc;
        t.wait_polls = attention_wait_polls();
        const uint64_t dims_q[3] = {D, a->heads, a->B}, str_q[2] = {D * 2ull, prm.ldq * 2};
        const uint64_t dims_k[4] = {D, a->cache->page_size, kv_heads, a->cache->n_pages};
        const uint64_t str_k[3] = {D * 2ull, (uint64_t)a->cache->page_size * D * 2, prm.cache.page_stride * 2};
        const uint32_t box_q[3] = {64, group, t.tokens}, box_k[4] = {64, a->cache->page_size, 1, 1};
        rc = make_tensor_map(who, &maps[0], a->Q, dtype, 3, dims_q, str_q, box_q);
        if (rc == SPTMM_OK) rc = make_tensor_map(who, &maps[1], a->cache->k, dtype, 4, dims_k, str_k, box_k);
        if (rc == SPTMM_OK) rc = make_tensor_map(who, &maps[2], a->cache->v, dtype, 4, dims_k, str_k, box_k);
        if (rc != SPTMM_OK) return rc;
    }
    int dev = 0, sms = 0;
    SPTMM_CUDA_TRY(cudaGetDevice(&dev));
    SPTMM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    const uint32_t ctas = 2 * (uint32_t)sms < kMaxDecodeCtas ? 2 * (uint32_t)sms : kMaxDecodeCtas;
    if (w.prefix.splits) {
        const uint32_t busy = w.prefix.pairs * kv_heads * w.prefix.splits, per_split = (a->prefix_len + kKeys * w.prefix.splits - 1) / (kKeys * w.prefix.splits);
        if (busy < (uint32_t)sms) {
            prm.early = 2 * ((uint32_t)sms - busy) < ctas ? 2 * ((uint32_t)sms - busy) : ctas;
            // A part of the prefix takes about 5 us and 1.7 us per block of 128 keys, a late CTA another 4 us to its
            // first keys; an early CTA gets through 64 keys of 128 channels in 1 us or less.
            prm.lead = (8 + per_split * 12 / 5) * (D > 64 ? 1 : 2);
        }
    }
    const bool pdl = flags & SPTMM_LAUNCH_PDL, wide = D > 64;
    cudaError_t e;
    if (dtype == SPTMM_F16) e = wide ? launch_decode<__half, 128>(prm, t, w.prefix, maps, ctas, stream, pdl) : launch_decode<__half, 64>(prm, t, w.prefix, maps, ctas, stream, pdl);
    else e = wide ? launch_decode<__nv_bfloat16, 128>(prm, t, w.prefix, maps, ctas, stream, pdl) : launch_decode<__nv_bfloat16, 64>(prm, t, w.prefix, maps, ctas, stream, pdl);
    if (e != cudaSuccess) return fail(SPTMM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return SPTMM_OK;
}
