// attention.cuh -- what the attention kernels share: 16-bit element types, the paged cache's
// addresses, argument checks and the launch with the programmatic-dependent-launch attribute.
#pragma once
#include <cuda_bf16.h>

#include "device_common.cuh"

namespace sptmm {

constexpr uint32_t kMaxHeadDim = 128;
constexpr uint32_t kMaxGroup = 128;             // query heads per key head

// two fp32 values -> one 32-bit word of two 16-bit values (round to nearest even), lo in the low half
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w)
{
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// How softmax weights are held in 16 bits.  A weight is 2^(x - m + up), x the score and m the running maximum in
// powers of two: `up` cancels between O and the normaliser.  m follows the true maximum only when that has grown
// by more than `lag`, because O and the sum have to be scaled down then.
// bf16 rounds weights of any size alike.  fp16 has full precision down to 2^-14 only and nothing below 2^-25, while
// the normaliser sums unrounded weights: with the largest weight at 1, thousands of keys 2^-20 below it -- all that
// counts where the largest one's value is small, an attention sink -- came out up to 10 % off.  So its weights are
// raised as far as 65504 allows: up + lag = 15.  A weight 2^-23 of the largest still has full precision, and the
// error of a smaller one is at most 2^-34 of the largest.  Less lag means scaling down more often: a mixed batch of
// prompts, 31k tokens of 20 heads over 5, takes 1515 us with a lag of 8 (and nothing raised: the same), 1519 with 6,
// 1527 with 5, 1551 with 4.
template <typename T> struct WeightRange { static constexpr float lag = 8.0f, up = 0.0f; };
template <> struct WeightRange<__half> { static constexpr float lag = 6.0f, up = 9.0f; };

// Device-side view of a cache (host struct sptmm_kv_cache with the default stride filled in).
struct CacheView {
    void *k, *v;
    uint64_t page_stride;
    uint32_t n_pages, page_shift, kv_heads, head_dim;
    __device__ __forceinline__ uint32_t page_size() const { return 1u << page_shift; }
    // element index of (page, head, slot, 0): 64 bits, a long cache passes 2^32 elements
    __device__ __forceinline__ uint64_t at(uint32_t page, uint32_t head, uint32_t slot) const
    {
        return (uint64_t)page * page_stride + (uint64_t)((((uint64_t)head << page_shift) + slot) * head_dim);
    }
};

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
inline bool aligned4(const void *p) { return ((uintptr_t)p & 3) == 0; }       // index arrays

inline int check_heads(const char *who, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t dtype)
{
    if (dtype != SPTMM_F16 && dtype != SPTMM_BF16) return fail(SPTMM_ERR_INVALID, "%s: dtype %u is neither fp16 nor bf16", who, dtype);
    if (heads == 0 || kv_heads == 0 || heads % kv_heads || heads > 65535)
        return fail(SPTMM_ERR_INVALID, "%s: %u query heads over %u key heads", who, heads, kv_heads);
    if (heads / kv_heads > kMaxGroup) return fail(SPTMM_ERR_UNSUPPORTED, "%s: %u query heads per key head (at most %u)", who, heads / kv_heads, kMaxGroup);
    if (head_dim == 0 || head_dim % 8) return fail(SPTMM_ERR_INVALID, "%s: head_dim %u is not a multiple of 8", who, head_dim);
    if (head_dim > kMaxHeadDim) return fail(SPTMM_ERR_UNSUPPORTED, "%s: head_dim %u (at most %u)", who, head_dim, kMaxHeadDim);
    return SPTMM_OK;
}

// `ld` elements between rows of `width` elements: 0 = back to back
inline int check_stride(const char *who, const char *name, uint64_t &ld, uint64_t width, uint32_t multiple)
{
    if (ld == 0) ld = width;
    if (ld < width || ld % multiple || ld > (1ull << 32))
        return fail(SPTMM_ERR_INVALID, "%s: %s=%llu for rows of %llu elements (a multiple of %u, not less than the row)", who, name,
                    (unsigned long long)ld, (unsigned long long)width, multiple);
    return SPTMM_OK;
}

inline int check_cache(const char *who, const sptmm_kv_cache *c, CacheView &v)
{
    if (!c->k || !c->v || !aligned16(c->k) || !aligned16(c->v)) return fail(SPTMM_ERR_INVALID, "%s: cache address null or not 16-byte aligned", who);
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return fail(SPTMM_ERR_INVALID, "%s: page_size %u (16, 32, 64 or 128)", who, c->page_size);
    if (c->n_pages == 0 || c->reserved) return fail(SPTMM_ERR_INVALID, "%s: cache of %u pages, reserved %u", who, c->n_pages, c->reserved);
    const uint64_t least = (uint64_t)c->kv_heads * c->page_size * c->head_dim;
    const uint64_t stride = c->page_stride ? c->page_stride : least;
    if (stride < least || stride % 8 || stride > (1ull << 36))
        return fail(SPTMM_ERR_INVALID, "%s: page_stride %llu for pages of %llu elements", who, (unsigned long long)stride, (unsigned long long)least);
    if ((uint64_t)c->n_pages * c->page_size > 0x7fffffffull) return fail(SPTMM_ERR_INVALID, "%s: %u pages of %u slots pass 31 bits", who, c->n_pages, c->page_size);
    v.k = c->k; v.v = c->v; v.page_stride = stride; v.n_pages = c->n_pages; v.kv_heads = c->kv_heads; v.head_dim = c->head_dim;
    v.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    return SPTMM_OK;
}

// One launch, with the programmatic-dependent-launch attribute when `pdl`, in clusters when `cluster` > 1.
template <typename... P, typename... A>
inline cudaError_t launch_clusters(uint32_t cluster, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, void *stream, bool pdl, A &&...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    uint32_t n = 0;
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster; attr[n].val.clusterDim.y = 1; attr[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr; cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}
template <typename... P, typename... A>
inline cudaError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, void *stream, bool pdl, A &&...args)
{
    return launch_clusters(1, kernel, grid, block, smem, stream, pdl, static_cast<A &&>(args)...);
}

}  // namespace sptmm
