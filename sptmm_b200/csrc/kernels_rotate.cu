// kernels_rotate.cu -- norms of query and key heads, position rotation and the stores into packed
// rows and cache slots, in one pass over the fused qkv rows.
//
// The reference has no attention (its only operator is the matmul, main.cu:993-1961).  Per token and
// head x of D channels:
//     x *= w * rsqrt(mean(x^2) + eps)                          (query and key heads, where asked for)
//     (a, b) -> (a cos t - b sin t, a sin t + b cos t)         t = position * inv_freq[pair]
// and one rounding to 16 bits.  HBM bound: every input element is read once and every output element
// written once.  A CTA takes one token, because its heads share the cosines.  A group of 16 lanes (8 up to
// 64 channels) takes a head, eight channels to a lane and chosen so that a channel and its partner meet in
// one lane whichever way pairs are formed: only the mean needs shuffles, and a lane's four cosines serve
// all of its heads.  All loads of a token are in flight while the angles are formed:
// position * inv_freq / 2 pi in 64 bits, reduced to a fraction of a turn, then sincospif in 32 -- at
// position 131071 a product in 32 bits would already be off by 2^-8 radians.
// Measured on 8192 tokens of 20 + 5 + 5 heads of 128 channels, fp32 -> bf16 (210 MB): 36 to 37 us, 5.7 TB/s, 0.87
// of the copy rate, with five CTAs per SM (48 registers); four or six: 38.6, 36.6; eight (32 registers):
// 47.9.  Four channels per lane with partners shuffled: 57.  CTAs that walk over tokens and fetch the next
// one's heads ahead: 64, for the registers that takes.  One to sixteen tokens: 2.9 us, a launch.
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

constexpr int kRotateThreads = 256, kRotateBatch = 2;

// LPH lanes of eight channels each hold a head: 8 up to 64 channels, 16 beyond.  grid.x: tokens, grid.y: batches
// of GROUPS * 2 of a token's heads.
template <typename TI, typename TO, int LPH>
__global__ void __launch_bounds__(kRotateThreads, 5) k_rotate(const __grid_constant__ RotateParams p)
{
    using Raw = typename In4<TI>::raw;
    __shared__ alignas(16) float2 turn[kMaxHeadDim / 2];     // (cos, sin) of the token's angles, read two at a time
    constexpr uint32_t GROUPS = kRotateThreads / LPH;
    const uint32_t tid = threadIdx.x, lane = tid % LPH, group = tid / LPH, mask = ((1u << LPH) - 1) << (tid & 31 & ~(LPH - 1));
    const uint32_t D = p.head_dim, rot = p.rot_dim, qk_heads = p.heads + p.kv_heads, n_heads = qk_heads + p.kv_heads;
    const uint32_t t = blockIdx.x, first = blockIdx.y * GROUPS * kRotateBatch;
    // This lane's channels: a .. a + 4 and b .. b + 4, the partners of one another where pairs lie rot / 2 apart
    const bool active = lane * 8 < D, apart = !p.interleaved && lane * 8 < rot;
    const uint32_t a = apart ? lane * 4 : lane * 8, b = apart ? rot / 2 + lane * 4 : lane * 8 + 4;
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int32_t pos = tid < rot / 2 ? p.positions[t] : 0;
    const int32_t slot = p.has_cache ? p.slots[t] : -1;
    const bool cached = slot >= 0 && ((uint32_t)slot >> p.cache.page_shift) < p.cache.n_pages;
    const TI *row = static_cast<const TI *>(p.X) + (uint64_t)t * p.ldx;
    Raw raw[kRotateBatch][2];
#pragma unroll
    for (uint32_t u = 0; u < kRotateBatch; u++) {
        const uint32_t h = first + u * GROUPS + group;
        raw[u][0] = raw[u][1] = Raw{};
        if (h < n_heads && active) {
            raw[u][0] = __ldcs(reinterpret_cast<const Raw *>(row + (uint64_t)h * D + a));
            raw[u][1] = __ldcs(reinterpret_cast<const Raw *>(row + (uint64_t)h * D + b));
        }
    }
    if (tid < rot / 2) {
        double turns = (double)pos * p.inv_freq[tid] * 0.15915494309189533577;                 // 1 / (2 pi)
        turns -= rint(turns);
        float s, co;
        sincospif(2.0f * (float)turns, &s, &co);
        turn[tid] = make_float2(co, s);
    }
    __syncthreads();
    // the four pairs of this lane, the same for every head
    float4 cs[2] = {};
    if (lane * 8 < rot) {
        cs[0] = *reinterpret_cast<const float4 *>(&turn[lane * 4]);
        cs[1] = *reinterpret_cast<const float4 *>(&turn[lane * 4 + 2]);
    }
#pragma unroll
    for (uint32_t u = 0; u < kRotateBatch; u++) {
        const uint32_t h = first + u * GROUPS + group;
        float x[4], y[4];
        to_float<TI>(raw[u][0], x);
        to_float<TI>(raw[u][1], y);
        if (h < qk_heads) {                              // a query or key head; the same for all lanes of the group
            if (h < p.heads ? p.q_norm != nullptr : p.k_norm != nullptr) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; i++) ss += x[i] * x[i] + y[i] * y[i];
#pragma unroll
                for (int o = LPH / 2; o; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
                const float r = rsqrtf(ss / (float)D + p.eps);
                const float *w = h < p.heads ? p.q_norm : p.k_norm;
                if (active) {
                    const float4 g = *reinterpret_cast<const float4 *>(w + a), k = *reinterpret_cast<const float4 *>(w + b);
                    x[0] *= r * g.x; x[1] *= r * g.y; x[2] *= r * g.z; x[3] *= r * g.w;
                    y[0] *= r * k.x; y[1] *= r * k.y; y[2] *= r * k.z; y[3] *= r * k.w;
                }
            }
            const float co[4] = {cs[0].x, cs[0].z, cs[1].x, cs[1].z}, si[4] = {cs[0].y, cs[0].w, cs[1].y, cs[1].w};
            if (lane * 8 >= rot) {
                // not rotated
            } else if (p.interleaved) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float x0 = x[2 * i], y0 = y[2 * i];
                    x[2 * i] = x0 * co[i] - x[2 * i + 1] * si[i]; x[2 * i + 1] = x0 * si[i] + x[2 * i + 1] * co[i];
                    y[2 * i] = y0 * co[2 + i] - y[2 * i + 1] * si[2 + i]; y[2 * i + 1] = y0 * si[2 + i] + y[2 * i + 1] * co[2 + i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x0 = x[i];
                    x[i] = x0 * co[i] - y[i] * si[i]; y[i] = x0 * si[i] + y[i] * co[i];
                }
            }
        }
        if (h < n_heads && active) {
            const uint2 w0 = make_uint2(pack2<TO>(x[0], x[1]), pack2<TO>(x[2], x[3])), w1 = make_uint2(pack2<TO>(y[0], y[1]), pack2<TO>(y[2], y[3]));
            auto store = [&](TO *o) { *reinterpret_cast<uint2 *>(o + a) = w0; *reinterpret_cast<uint2 *>(o + b) = w1; };
            if (h < p.heads) {
                store(static_cast<TO *>(p.Q) + (uint64_t)t * p.ldq + (uint64_t)h * D);
            } else {
                const bool is_v = h >= qk_heads;
                const uint32_t kh = h - (is_v ? qk_heads : p.heads);
                if (p.K) store(static_cast<TO *>(is_v ? p.V : p.K) + (uint64_t)t * (is_v ? p.ldv : p.ldk) + (uint64_t)kh * D);
                if (cached)
                    store(static_cast<TO *>(is_v ? p.cache.v : p.cache.k) +
                          p.cache.at((uint32_t)slot >> p.cache.page_shift, kh, (uint32_t)slot & (p.cache.page_size() - 1)));
            }
        }
    }
}

template <typename TI, typename TO, int LPH>
static cudaError_t launch_rotate(const RotateParams &prm, uint32_t T, void *stream, bool pdl)
{
    constexpr uint32_t heads = kRotateThreads / LPH * kRotateBatch;
    return launch(k_rotate<TI, TO, LPH>, dim3(T, (prm.heads + 2 * prm.kv_heads + heads - 1) / heads), dim3(kRotateThreads), 0, stream, pdl, prm);
}

template <typename TI, typename TO>
static cudaError_t launch_rotate(const RotateParams &prm, uint32_t T, void *stream, bool pdl)
{
    return prm.head_dim <= 64 ? launch_rotate<TI, TO, 8>(prm, T, stream, pdl) : launch_rotate<TI, TO, 16>(prm, T, stream, pdl);
}

template <typename TI>
static cudaError_t launch_rotate_to(const RotateParams &prm, uint32_t dtype, uint32_t T, void *stream, bool pdl)
{
    return dtype == SPTMM_F16 ? launch_rotate<TI, __half>(prm, T, stream, pdl) : launch_rotate<TI, __nv_bfloat16>(prm, T, stream, pdl);
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
    if (!aligned4(a->positions) || !aligned4(a->slots)) return fail(SPTMM_ERR_INVALID, "%s: an index array is not 4-byte aligned", who);
    prm.X = a->QKV; prm.q_norm = a->q_norm; prm.k_norm = a->k_norm; prm.positions = a->positions; prm.slots = a->slots;
    prm.Q = a->Q; prm.K = a->K; prm.V = a->V;
    prm.heads = a->heads; prm.kv_heads = a->kv_heads; prm.head_dim = a->head_dim; prm.rot_dim = a->rot_dim;
    prm.interleaved = a->interleaved ? 1 : 0; prm.has_cache = a->cache ? 1 : 0; prm.eps = a->eps;
    for (uint32_t i = 0; i < a->rot_dim / 2; i++) prm.inv_freq[i] = a->inv_freq[i];
    const bool pdl = flags & SPTMM_LAUNCH_PDL;
    cudaError_t e;
    if (a->in_dtype == SPTMM_F32) e = launch_rotate_to<float>(prm, a->dtype, a->T, stream, pdl);
    else if (a->in_dtype == SPTMM_F16) e = launch_rotate_to<__half>(prm, a->dtype, a->T, stream, pdl);
    else e = launch_rotate_to<__nv_bfloat16>(prm, a->dtype, a->T, stream, pdl);
    if (e != cudaSuccess) return fail(SPTMM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return SPTMM_OK;
}
