// kernels_prompt.cu -- attention over packed prompts.
//
// The reference has no attention (its only operator is the matmul, main.cu:993-1961).
// The kernel is k_attention_tc (attention_tc.cuh); here are its host side, the tensor maps and the word
// an expired wait is reported in.
#include <atomic>

#include "attention_tc.cuh"

namespace sptmm {

__device__ uint32_t g_attention_status;

int attention_status_word(uint32_t **dev_word)
{
    SPTMM_CUDA_TRY(cudaGetSymbolAddress(reinterpret_cast<void **>(dev_word), g_attention_status));
    return SPTMM_OK;
}

static std::atomic<uint32_t> g_wait_polls{0};        // 0: the default

uint32_t attention_wait_polls() { return g_wait_polls.load(); }

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                 const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int make_tensor_map(const char *who, CUtensorMap *map, const void *base, uint32_t dtype, uint32_t rank, const uint64_t *dims,
                    const uint64_t *strides, const uint32_t *box)
{
    static std::atomic<void *> entry{nullptr};       // the driver's function; the same whoever looks it up first
    void *fn = entry.load();
    if (!fn) {
        cudaDriverEntryPointQueryResult found;
        SPTMM_CUDA_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found));
        if (found != cudaDriverEntryPointSuccess || !fn) return fail(SPTMM_ERR_CUDA, "%s: the driver has no tensor maps", who);
        entry.store(fn);
    }
    cuuint64_t d[4], st[3];
    cuuint32_t b[4], one[4];
    for (uint32_t i = 0; i < rank; i++) { d[i] = dims[i]; b[i] = box[i]; one[i] = 1; if (i) st[i - 1] = strides[i - 1]; }
    const CUresult rc = reinterpret_cast<EncodeTiled>(fn)(map, dtype == SPTMM_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                                          rank, const_cast<void *>(base), d, st, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return fail(SPTMM_ERR_CUDA, "%s: tensor map refused (%d)", who, (int)rc);
    return SPTMM_OK;
}

template <typename T, int DP, bool SPLIT>
static cudaError_t launch_prompt(const TcParams &prm, uint32_t grid, const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, void *stream, bool pdl)
{
    const cudaError_t e = cudaFuncSetAttribute(k_attention_tc<T, DP, false, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcLayout<DP>::smem);
    if (e != cudaSuccess) return e;
    return launch_clusters(prm.cluster, k_attention_tc<T, DP, false, SPLIT>, dim3(grid), dim3(kTcThreads), TcLayout<DP>::smem, stream, pdl, prm, q, k, v);
}

template <typename T>
static cudaError_t launch_prompt(const TcParams &prm, uint32_t grid, const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, void *stream, bool pdl)
{
    if (prm.head_dim > 64) return prm.cluster > 1 ? launch_prompt<T, 128, true>(prm, grid, q, k, v, stream, pdl) : launch_prompt<T, 128, false>(prm, grid, q, k, v, stream, pdl);
    return prm.cluster > 1 ? launch_prompt<T, 64, true>(prm, grid, q, k, v, stream, pdl) : launch_prompt<T, 64, false>(prm, grid, q, k, v, stream, pdl);
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
    TcParams prm{};
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
    if (!aligned4(a->q_offsets) || !aligned4(a->k_offsets)) return fail(SPTMM_ERR_INVALID, "%s: an index array is not 4-byte aligned", who);
    prm.Q = a->Q; prm.K = a->K; prm.V = a->V; prm.O = a->O; prm.q_off = a->q_offsets; prm.k_off = a->k_offsets;
    prm.n_seqs = a->n_seqs; prm.T = a->T; prm.Tk = a->Tk; prm.heads = a->heads; prm.kv_heads = a->kv_heads; prm.group = a->heads / a->kv_heads;
    prm.head_dim = a->head_dim; prm.causal = a->causal ? 1 : 0;
    prm.tokens = 128 / prm.group; prm.group_mul = 65535 / prm.group + 1;
    prm.scale = (a->scale > 0.0f ? a->scale : 1.0f / sqrtf((float)a->head_dim)) * 1.4426950408889634f;     // log2(e): the kernel works with exp2
    const uint64_t items = item_numbers(a->n_seqs, a->T, 2 * prm.tokens);
    if (items * a->kv_heads > 0x7fffffffull / 8) return fail(SPTMM_ERR_UNSUPPORTED, "%s: %u rows of %u key heads in one call", who, a->T, a->kv_heads);
    // Few items leave SMs idle: then up to eight CTAs, as many as there is an SM for, share an item's keys
    // (if it has two blocks of keys for each; see the kernel).  512 queries over 8192 keys, 40 items: 126 us by
    // 40 CTAs, 51 to 66 us, from process to process, by as many clusters of three.
    int dev = 0, sms = 0;
    SPTMM_CUDA_TRY(cudaGetDevice(&dev));
    SPTMM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    const uint64_t room = (uint64_t)sms / (items * a->kv_heads);
    prm.cluster = room > 8 ? 8 : room < 1 ? 1 : (uint32_t)room;
    rc = attention_status_word(&prm.status);
    if (rc != SPTMM_OK) return rc;
    prm.wait_polls = attention_wait_polls();
    const uint64_t D = a->head_dim, es = 2;
    const uint64_t dims_q[3] = {D, a->heads, a->T}, str_q[2] = {D * es, prm.ldq * es};
    const uint64_t dims_k[3] = {D, a->kv_heads, a->Tk ? a->Tk : 1}, str_k[2] = {D * es, prm.ldk * es}, str_v[2] = {D * es, prm.ldv * es};
    const uint32_t box_q[3] = {64, prm.group, prm.tokens}, box_k[3] = {64, 1, kKeys};
    CUtensorMap mq, mk, mv;
    rc = make_tensor_map(who, &mq, a->Q, a->dtype, 3, dims_q, str_q, box_q);
    if (rc == SPTMM_OK) rc = make_tensor_map(who, &mk, a->Tk ? a->K : a->Q, a->dtype, 3, dims_k, str_k, box_k);     // no keys: never read
    if (rc == SPTMM_OK) rc = make_tensor_map(who, &mv, a->Tk ? a->V : a->Q, a->dtype, 3, dims_k, str_v, box_k);
    if (rc != SPTMM_OK) return rc;
    const uint32_t grid = (uint32_t)(items * a->kv_heads) * prm.cluster;
    const bool pdl = flags & SPTMM_LAUNCH_PDL;
    const cudaError_t e = a->dtype == SPTMM_F16 ? launch_prompt<__half>(prm, grid, mq, mk, mv, stream, pdl) : launch_prompt<__nv_bfloat16>(prm, grid, mq, mk, mv, stream, pdl);
    if (e != cudaSuccess) return fail(SPTMM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return SPTMM_OK;
}

extern "C" int sptmm_attention_set_wait_limit(uint32_t polls)
{
    g_wait_polls.store(polls);
    return SPTMM_OK;
}

extern "C" int sptmm_attention_status(uint32_t *status)
{
    if (!status) return fail(SPTMM_ERR_INVALID, "attention_status: null pointer");
    SPTMM_CUDA_TRY(cudaDeviceSynchronize());
    SPTMM_CUDA_TRY(cudaMemcpyFromSymbol(status, g_attention_status, sizeof(uint32_t)));
    if (*status) {
        const uint32_t zero = 0;
        SPTMM_CUDA_TRY(cudaMemcpyToSymbol(g_attention_status, &zero, sizeof zero));
    }
    return SPTMM_OK;
}
