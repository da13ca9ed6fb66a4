// kernels_decode.cu -- attention of one new token per sequence over a paged cache, behind an optional
// prefix that the batch shares.
//
// The reference has no attention (its only operator is the matmul, main.cu:993-1961).
// Simplest form: a warp per (sequence, head), four channels per lane, keys one after the other.
#include "attention.cuh"

namespace sptmm {

struct DecodeParams {
    const void *Q;
    void *O;
    CacheView cache;
    const int32_t *lengths, *table, *prefix_table;
    uint64_t ldq, ldo;
    uint32_t B, heads, group, max_pages, prefix_len;
    float scale;
};

template <typename T>
__global__ void __launch_bounds__(256) k_decode_rows(const DecodeParams p)
{
    const uint32_t lane = threadIdx.x & 31, c = lane * 4, D = p.cache.head_dim;
    const uint64_t item = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    if (item >= (uint64_t)p.B * p.heads) return;
    const uint32_t b = (uint32_t)(item / p.heads), h = (uint32_t)(item % p.heads), kh = h / p.group;
    float q[4] = {0, 0, 0, 0}, o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0;
    if (c < D) {
        const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const T *>(p.Q) + (uint64_t)b * p.ldq + (uint64_t)h * D + c);
        const float2 a = unpack2<T>(w.x), d = unpack2<T>(w.y);
        q[0] = a.x * p.scale; q[1] = a.y * p.scale; q[2] = d.x * p.scale; q[3] = d.y * p.scale;
    }
    const uint64_t room = (uint64_t)p.max_pages << p.cache.page_shift;
    const uint32_t own = (uint32_t)min(room, (uint64_t)max(p.lengths[b], 0));
    for (uint32_t part = 0; part < 2; part++) {
        const int32_t *table = part ? p.table + (uint64_t)b * p.max_pages : p.prefix_table;
        const uint32_t n = part ? own : p.prefix_len;
        for (uint32_t j = 0; j < n; j++) {
            const uint32_t page = (uint32_t)table[j >> p.cache.page_shift];
            if (page >= p.cache.n_pages) continue;
            float k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0};
            if (c < D) {
                const uint64_t at = p.cache.at(page, kh, j & (p.cache.page_size() - 1)) + c;
                const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const T *>(p.cache.k) + at);
                const uint2 z = *reinterpret_cast<const uint2 *>(static_cast<const T *>(p.cache.v) + at);
                float2 a = unpack2<T>(w.x), d = unpack2<T>(w.y);
                k[0] = a.x; k[1] = a.y; k[2] = d.x; k[3] = d.y;
                a = unpack2<T>(z.x); d = unpack2<T>(z.y);
                v[0] = a.x; v[1] = a.y; v[2] = d.x; v[3] = d.y;
            }
            float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
            for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            const float m1 = fmaxf(m, s), w0 = m1 == -INFINITY ? 1.0f : exp2f(m - m1), w1 = m1 == -INFINITY ? 0.0f : exp2f(s - m1);
            m = m1;
            l = l * w0 + w1;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = o[i] * w0 + w1 * v[i];
        }
    }
    if (c >= D) return;
    const float r = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
    *reinterpret_cast<uint2 *>(static_cast<T *>(p.O) + (uint64_t)b * p.ldo + (uint64_t)h * D + c) =
        make_uint2(pack2<T>(o[0] * r, o[1] * r), pack2<T>(o[2] * r, o[3] * r));
}

}  // namespace sptmm

using namespace sptmm;

extern "C" uint64_t sptmm_attention_decode_workspace(uint32_t B, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t prefix_len)
{
    if (check_heads("attention_decode_workspace", heads, kv_heads, head_dim, SPTMM_F16) != SPTMM_OK) return 0;
    (void)prefix_len;
    return 16 * ((uint64_t)B + 1);
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
    const uint64_t need = sptmm_attention_decode_workspace(a->B, a->heads, a->cache->kv_heads, a->cache->head_dim, a->prefix_len);
    if (!a->workspace || a->workspace_bytes < need)
        return fail(SPTMM_ERR_INVALID, "%s: workspace of %llu bytes, %llu needed", who, (unsigned long long)(a->workspace ? a->workspace_bytes : 0), (unsigned long long)need);
    prm.Q = a->Q; prm.O = a->O; prm.lengths = a->lengths; prm.table = a->table; prm.prefix_table = a->prefix_table;
    prm.B = a->B; prm.heads = a->heads; prm.group = a->heads / a->cache->kv_heads; prm.max_pages = a->max_pages; prm.prefix_len = a->prefix_len;
    prm.scale = (a->scale > 0.0f ? a->scale : 1.0f / sqrtf((float)a->cache->head_dim)) * 1.4426950408889634f;      // log2(e): the kernel works with exp2
    const dim3 grid((uint32_t)(((uint64_t)a->B * a->heads + 7) / 8));
    const cudaError_t e = a->cache->dtype == SPTMM_F16 ? launch(k_decode_rows<__half>, grid, dim3(256), 0, stream, flags & SPTMM_LAUNCH_PDL, prm)
                                                       : launch(k_decode_rows<__nv_bfloat16>, grid, dim3(256), 0, stream, flags & SPTMM_LAUNCH_PDL, prm);
    if (e != cudaSuccess) return fail(SPTMM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return SPTMM_OK;
}
