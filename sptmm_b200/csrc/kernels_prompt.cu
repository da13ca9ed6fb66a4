// kernels_prompt.cu -- attention over packed prompts.
//
// The reference has no attention (its only operator is the matmul, main.cu:993-1961).
// Simplest form: a warp per (query row, head), four channels per lane, keys one after the other with
// the running maximum and sum of the softmax in fp32.
#include "attention.cuh"

namespace sptmm {

struct PromptParams {
    const void *Q, *K, *V;
    void *O;
    const int32_t *q_off, *k_off;
    uint64_t ldq, ldk, ldv, ldo;
    uint32_t n_seqs, T, Tk, heads, group, head_dim, causal;
    float scale;
};

template <typename T>
__global__ void __launch_bounds__(256) k_prompt_rows(const PromptParams p)
{
    const uint32_t lane = threadIdx.x & 31, c = lane * 4, D = p.head_dim;
    const uint64_t item = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    if (item >= (uint64_t)p.T * p.heads) return;
    const uint32_t t = (uint32_t)(item / p.heads), h = (uint32_t)(item % p.heads), kh = h / p.group;
    uint32_t lo = 0, hi = p.n_seqs;                          // the last sequence that starts at or before t
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (p.q_off[mid] <= (int32_t)t) lo = mid; else hi = mid;
    }
    const int32_t q0 = max(p.q_off[lo], 0), q1 = min(p.q_off[lo + 1], (int32_t)p.T);        // offsets past the rows are cut
    if ((int32_t)t < q0 || (int32_t)t >= q1) return;
    const int32_t k0 = max(p.k_off[lo], 0), k1 = max(k0, min(p.k_off[lo + 1], (int32_t)p.Tk));
    int64_t n = k1 - k0;
    if (p.causal) n = min(n, max((int64_t)0, (int64_t)(t - q0) + n - (q1 - q0) + 1));
    float q[4] = {0, 0, 0, 0}, o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0;
    if (c < D) {
        const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const T *>(p.Q) + (uint64_t)t * p.ldq + (uint64_t)h * D + c);
        const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
        q[0] = a.x * p.scale; q[1] = a.y * p.scale; q[2] = b.x * p.scale; q[3] = b.y * p.scale;
    }
    for (int64_t j = 0; j < n; j++) {
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
        const float m1 = fmaxf(m, s), w0 = m1 == -INFINITY ? 1.0f : exp2f(m - m1), w1 = m1 == -INFINITY ? 0.0f : exp2f(s - m1);
        m = m1;
        l = l * w0 + w1;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = o[i] * w0 + w1 * v[i];
    }
    if (c >= D) return;
    const float r = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
    *reinterpret_cast<uint2 *>(static_cast<T *>(p.O) + (uint64_t)t * p.ldo + (uint64_t)h * D + c) =
        make_uint2(pack2<T>(o[0] * r, o[1] * r), pack2<T>(o[2] * r, o[3] * r));
}

}  // namespace sptmm

using namespace sptmm;

extern "C" int sptmm_attention_prompt(const sptmm_prompt_params *a, uint32_t flags, void *stream)
{
    const char *who = "attention_prompt";
    if (!a) return fail(SPTMM_ERR_INVALID, "%s: null pointer", who);
    int rc = check_heads(who, a->heads, a->kv_heads, a->head_dim, a->dtype);
    if (rc != SPTMM_OK) return rc;
    if (flags & ~(uint32_t)SPTMM_LAUNCH_PDL) return fail(SPTMM_ERR_INVALID, "%s: flags %u", who, flags);
    if (!(a->scale >= 0.0f) || a->scale > 1e30f) return fail(SPTMM_ERR_INVALID, "%s: scale %g", who, (double)a->scale);
    PromptParams prm{};
    prm.ldq = a->ldq; prm.ldk = a->ldk; prm.ldv = a->ldv; prm.ldo = a->ldo;
    const uint64_t q_width = (uint64_t)a->heads * a->head_dim, kv_width = (uint64_t)a->kv_heads * a->head_dim;
    rc = check_stride(who, "ldq", prm.ldq, q_width, 8);
    if (rc == SPTMM_OK) rc = check_stride(who, "ldk", prm.ldk, kv_width, 8);
    if (rc == SPTMM_OK) rc = check_stride(who, "ldv", prm.ldv, kv_width, 8);
    if (rc == SPTMM_OK) rc = check_stride(who, "ldo", prm.ldo, q_width, 8);
    if (rc != SPTMM_OK) return rc;
    if (a->T > 0x3fffffffu || a->Tk > 0x3fffffffu) return fail(SPTMM_ERR_INVALID, "%s: T=%u Tk=%u", who, a->T, a->Tk);
    if (a->n_seqs > 65536) return fail(SPTMM_ERR_UNSUPPORTED, "%s: %u sequences (at most 65536)", who, a->n_seqs);
    if (a->T == 0 || a->n_seqs == 0) return SPTMM_OK;
    if (!a->Q || !a->O || !a->q_offsets || !a->k_offsets || (a->Tk && (!a->K || !a->V))) return fail(SPTMM_ERR_INVALID, "%s: null pointer", who);
    for (const void *x : {a->Q, a->K, a->V, (const void *)a->O})
        if (!aligned16(x)) return fail(SPTMM_ERR_INVALID, "%s: an address is not 16-byte aligned", who);
    prm.Q = a->Q; prm.K = a->K; prm.V = a->V; prm.O = a->O; prm.q_off = a->q_offsets; prm.k_off = a->k_offsets;
    prm.n_seqs = a->n_seqs; prm.T = a->T; prm.Tk = a->Tk; prm.heads = a->heads; prm.group = a->heads / a->kv_heads;
    prm.head_dim = a->head_dim; prm.causal = a->causal ? 1 : 0;
    prm.scale = (a->scale > 0.0f ? a->scale : 1.0f / sqrtf((float)a->head_dim)) * 1.4426950408889634f;     // log2(e): the kernel works with exp2
    const uint64_t warps = (uint64_t)a->T * a->heads;
    if (warps > 0x7fffffffull * 8) return fail(SPTMM_ERR_UNSUPPORTED, "%s: %u rows of %u heads in one call", who, a->T, a->heads);
    const dim3 grid((uint32_t)((warps + 7) / 8));
    const cudaError_t e = a->dtype == SPTMM_F16 ? launch(k_prompt_rows<__half>, grid, dim3(256), 0, stream, flags & SPTMM_LAUNCH_PDL, prm)
                                                : launch(k_prompt_rows<__nv_bfloat16>, grid, dim3(256), 0, stream, flags & SPTMM_LAUNCH_PDL, prm);
    if (e != cudaSuccess) return fail(SPTMM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return SPTMM_OK;
}
