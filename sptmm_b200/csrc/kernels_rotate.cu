// kernels_rotate.cu -- norms of query and key heads, position rotation and the stores into packed
// rows and cache slots, in one pass over the fused qkv rows.
//
// The reference has no attention (its only operator is the matmul, main.cu:993-1961).  Per token and
// head x of D channels:
//     x *= w * rsqrt(mean(x^2) + eps)                          (query and key heads, where asked for)
//     (a, b) -> (a cos t - b sin t, a sin t + b cos t)         t = position * inv_freq[pair]
// and one rounding to 16 bits.  HBM bound: every input element is read once and every output element
// written once.  A CTA takes one token, because its heads share the cosines; a group of LPH lanes
// takes a head, each lane four neighbouring channels (16-byte loads of fp32, 8-byte of 16-bit rows),
// so the mean is a butterfly over the group and a pair's partner lies in the same lane (interleaved
// pairs) or one shuffle away (pairs half the rotated range apart).  The loads of four heads per group
// are in flight while the angles are formed: position * inv_freq / 2 pi in 64 bits, reduced to a
// fraction of a turn, then sincospif in 32 -- at position 131071 a product in 32 bits would already be
// off by 2^-8 radians.
#include "attention.cuh"

namespace sptmm {

struct RotateParams {
    const void *X;
    const float *q_norm, *k_norm;
    const int32_t *positions, *slots;
    void *Q, *K, *V;
    CacheView cache;
    uint64_t ldx, ldq, ldk, ldv;
    uint32_t heads, kv_heads, head_dim, rot_dim, interleaved, has_cache;
    uint32_t heads_per_cta;                  // heads (q, k and v counted alike) along grid.y
    float eps;
    double inv_freq[kMaxHeadDim / 2];
};

template <typename T> struct In4;            // four neighbouring elements as loaded
template <> struct In4<float> { using raw = uint4; };
template <> struct In4<__half> { using raw = uint2; };
template <> struct In4<__nv_bfloat16> { using raw = uint2; };

template <typename T> __device__ __forceinline__ void to_float(const typename In4<T>::raw &r, float (&x)[4])
{
    const float2 a = unpack2<T>(r.x), b = unpack2<T>(r.y);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}
template <> __device__ __forceinline__ void to_float<float>(const uint4 &r, float (&x)[4])
{
    x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
}

constexpr int kRotateThreads = 256, kRotateBatch = 4;

// LPH lanes of four channels each hold a head: 16 up to 64 channels, 32 beyond.
template <typename TI, typename TO, int LPH>
__global__ void __launch_bounds__(kRotateThreads) k_rotate(const __grid_constant__ RotateParams p)
{
    __shared__ float2 turn[kMaxHeadDim / 2];                 // (cos, sin) of the token's angles
    constexpr int GROUPS = kRotateThreads / LPH;
    const uint32_t t = blockIdx.x, tid = threadIdx.x, c = tid % LPH, group = tid / LPH;
    const uint32_t D = p.head_dim, rot = p.rot_dim, n_heads = p.heads + 2 * p.kv_heads;
    const uint32_t first = blockIdx.y * p.heads_per_cta, last = min(n_heads, first + p.heads_per_cta);
    const bool active = c * 4 < D;
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const TI *row = static_cast<const TI *>(p.X) + (uint64_t)t * p.ldx;
    for (uint32_t h0 = first; h0 < last; h0 += GROUPS * kRotateBatch) {
        typename In4<TI>::raw raw[kRotateBatch];
#pragma unroll
        for (int u = 0; u < kRotateBatch; u++) {
            const uint32_t h = h0 + u * GROUPS + group;
            raw[u] = typename In4<TI>::raw{};
            if (h < last && active) raw[u] = __ldcs(reinterpret_cast<const typename In4<TI>::raw *>(row + (uint64_t)h * D + c * 4));
        }
        if (h0 == first) {
            if (tid < rot / 2) {
                double turns = (double)p.positions[t] * p.inv_freq[tid] * 0.15915494309189533577;      // 1 / (2 pi)
                turns -= rint(turns);
                float s, co;
                sincospif(2.0f * (float)turns, &s, &co);
                turn[tid] = make_float2(co, s);
            }
            __syncthreads();
        }
        const int32_t slot = p.has_cache ? p.slots[t] : -1;
        const bool cached = slot >= 0 && ((uint32_t)slot >> p.cache.page_shift) < p.cache.n_pages;
#pragma unroll
        for (int u = 0; u < kRotateBatch; u++) {
            const uint32_t h = h0 + u * GROUPS + group;
            float x[4];
            to_float<TI>(raw[u], x);
            if (h < p.heads + p.kv_heads) {                  // a query or key head; the same for all lanes of the group
                const float *w = h < p.heads ? p.q_norm : p.k_norm;
                if (w) {
                    float ss = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
#pragma unroll
                    for (int o = LPH / 2; o; o >>= 1) ss += __shfl_xor_sync(LPH == 32 ? 0xffffffffu : 0xffffu << (tid & 16), ss, o);
                    const float r = rsqrtf(ss / (float)D + p.eps);
                    const float4 g = active ? *reinterpret_cast<const float4 *>(w + c * 4) : make_float4(0, 0, 0, 0);
                    x[0] *= r * g.x; x[1] *= r * g.y; x[2] *= r * g.z; x[3] *= r * g.w;
                }
                if (rot) {
                    if (p.interleaved) {
                        if (c * 4 < rot) {
                            const float2 a = turn[c * 2], b = turn[c * 2 + 1];
                            const float x0 = x[0], x2 = x[2];
                            x[0] = x0 * a.x - x[1] * a.y; x[1] = x0 * a.y + x[1] * a.x;
                            x[2] = x2 * b.x - x[3] * b.y; x[3] = x2 * b.y + x[3] * b.x;
                        }
                    } else {
                        const uint32_t half = rot / 8;       // lanes per half of the rotated range
                        const uint32_t other = c < half ? c + half : c < 2 * half ? c - half : c;
                        float y[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) y[i] = __shfl_sync(LPH == 32 ? 0xffffffffu : 0xffffu << (tid & 16), x[i], other, LPH);
                        if (c < 2 * half) {
                            const uint32_t pair = (c < half ? c : c - half) * 4;
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const float2 a = turn[pair + i];
                                x[i] = c < half ? x[i] * a.x - y[i] * a.y : y[i] * a.y + x[i] * a.x;
                            }
                        }
                    }
                }
            }
            if (h >= last || !active) continue;
            const uint2 w = make_uint2(pack2<TO>(x[0], x[1]), pack2<TO>(x[2], x[3]));
            if (h < p.heads) {
                *reinterpret_cast<uint2 *>(static_cast<TO *>(p.Q) + (uint64_t)t * p.ldq + (uint64_t)h * D + c * 4) = w;
            } else {
                const bool is_v = h >= p.heads + p.kv_heads;
                const uint32_t kh = h - p.heads - (is_v ? p.kv_heads : 0);
                if (p.K) {
                    TO *o = static_cast<TO *>(is_v ? p.V : p.K) + (uint64_t)t * (is_v ? p.ldv : p.ldk);
                    *reinterpret_cast<uint2 *>(o + (uint64_t)kh * D + c * 4) = w;
                }
                if (cached) {
                    TO *o = static_cast<TO *>(is_v ? p.cache.v : p.cache.k);
                    o += p.cache.at((uint32_t)slot >> p.cache.page_shift, kh, (uint32_t)slot & (p.cache.page_size() - 1));
                    *reinterpret_cast<uint2 *>(o + c * 4) = w;
                }
            }
        }
    }
}

template <typename TI, typename TO>
static cudaError_t launch_rotate(const RotateParams &prm, dim3 grid, void *stream, bool pdl)
{
    if (prm.head_dim <= 64) return launch(k_rotate<TI, TO, 16>, grid, dim3(kRotateThreads), 0, stream, pdl, prm);
    return launch(k_rotate<TI, TO, 32>, grid, dim3(kRotateThreads), 0, stream, pdl, prm);
}

template <typename TI>
static cudaError_t launch_rotate_to(const RotateParams &prm, uint32_t dtype, dim3 grid, void *stream, bool pdl)
{
    return dtype == SPTMM_F16 ? launch_rotate<TI, __half>(prm, grid, stream, pdl) : launch_rotate<TI, __nv_bfloat16>(prm, grid, stream, pdl);
}

}  // namespace sptmm

using namespace sptmm;

extern "C" int sptmm_rotate_heads(const sptmm_rotate_params *a, uint32_t flags, void *stream)
{
    const char *who = "rotate_heads";
    if (!a) return fail(SPTMM_ERR_INVALID, "%s: null pointer", who);
    int rc = check_heads(who, a->heads, a->kv_heads, a->head_dim, a->dtype);
    if (rc != SPTMM_OK) return rc;
    if (a->in_dtype != SPTMM_F16 && a->in_dtype != SPTMM_F32 && a->in_dtype != SPTMM_BF16)
        return fail(SPTMM_ERR_INVALID, "%s: input dtype %u is neither fp32, fp16 nor bf16", who, a->in_dtype);
    if (flags & ~(uint32_t)SPTMM_LAUNCH_PDL) return fail(SPTMM_ERR_INVALID, "%s: flags %u", who, flags);
    if (a->rot_dim > a->head_dim || a->rot_dim % 8) return fail(SPTMM_ERR_INVALID, "%s: rot_dim %u of %u channels (a multiple of 8)", who, a->rot_dim, a->head_dim);
    if (a->rot_dim && !a->inv_freq) return fail(SPTMM_ERR_INVALID, "%s: rotation without inv_freq", who);
    if (!(a->eps >= 0.0f)) return fail(SPTMM_ERR_INVALID, "%s: eps %g", who, (double)a->eps);
    if (!a->K != !a->V) return fail(SPTMM_ERR_INVALID, "%s: K and V come together", who);
    if (!a->K && !a->cache) return fail(SPTMM_ERR_INVALID, "%s: neither packed rows nor a cache for the keys and values", who);
    if (!a->cache != !a->slots && a->T) return fail(SPTMM_ERR_INVALID, "%s: a cache comes with slots", who);
    RotateParams prm{};
    if (a->cache) {
        if (a->cache->kv_heads != a->kv_heads || a->cache->head_dim != a->head_dim || a->cache->dtype != a->dtype)
            return fail(SPTMM_ERR_INVALID, "%s: the cache holds %u heads of %u channels of dtype %u", who, a->cache->kv_heads, a->cache->head_dim, a->cache->dtype);
        rc = check_cache(who, a->cache, prm.cache);
        if (rc != SPTMM_OK) return rc;
    }
    const uint64_t kv_width = (uint64_t)a->kv_heads * a->head_dim, q_width = (uint64_t)a->heads * a->head_dim;
    prm.ldx = a->ldqkv; prm.ldq = a->ldq; prm.ldk = a->ldk; prm.ldv = a->ldv;
    rc = check_stride(who, "ldqkv", prm.ldx, q_width + 2 * kv_width, a->in_dtype == SPTMM_F32 ? 4 : 8);
    if (rc == SPTMM_OK) rc = check_stride(who, "ldq", prm.ldq, q_width, 8);
    if (rc == SPTMM_OK) rc = check_stride(who, "ldk", prm.ldk, kv_width, 8);
    if (rc == SPTMM_OK) rc = check_stride(who, "ldv", prm.ldv, kv_width, 8);
    if (rc != SPTMM_OK) return rc;
    if (a->T > 0x7fffffffu) return fail(SPTMM_ERR_INVALID, "%s: T=%u", who, a->T);
    if (a->T == 0) return SPTMM_OK;
    if (!a->QKV || !a->Q || (a->rot_dim && !a->positions)) return fail(SPTMM_ERR_INVALID, "%s: null pointer", who);
    for (const void *x : {a->QKV, (const void *)a->Q, (const void *)a->K, (const void *)a->V, (const void *)a->q_norm, (const void *)a->k_norm})
        if (!aligned16(x)) return fail(SPTMM_ERR_INVALID, "%s: an address is not 16-byte aligned", who);
    prm.X = a->QKV; prm.q_norm = a->q_norm; prm.k_norm = a->k_norm; prm.positions = a->positions; prm.slots = a->slots;
    prm.Q = a->Q; prm.K = a->K; prm.V = a->V;
    prm.heads = a->heads; prm.kv_heads = a->kv_heads; prm.head_dim = a->head_dim; prm.rot_dim = a->rot_dim;
    prm.interleaved = a->interleaved ? 1 : 0; prm.has_cache = a->cache ? 1 : 0; prm.eps = a->eps;
    for (uint32_t i = 0; i < a->rot_dim / 2; i++) prm.inv_freq[i] = a->inv_freq[i];
    prm.heads_per_cta = a->heads + 2 * a->kv_heads;
    const dim3 grid(a->T);
    const bool pdl = flags & SPTMM_LAUNCH_PDL;
    cudaError_t e;
    if (a->in_dtype == SPTMM_F32) e = launch_rotate_to<float>(prm, a->dtype, grid, stream, pdl);
    else if (a->in_dtype == SPTMM_F16) e = launch_rotate_to<__half>(prm, a->dtype, grid, stream, pdl);
    else e = launch_rotate_to<__nv_bfloat16>(prm, a->dtype, grid, stream, pdl);
    if (e != cudaSuccess) return fail(SPTMM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return SPTMM_OK;
}
