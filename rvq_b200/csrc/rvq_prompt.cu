// Attention of whole prompts (rvq_prompt_attention, include/rvq_b200.h).

#include <string.h>

#include "rvq_common.cuh"

namespace rvq {

int take_step_timeout();                     // the step attention's flag (rvq_cache4_attn.cu)

namespace prompt {

__device__ int g_attention_timeout;          // sticky: a bounded wait gave up

// One warp per (token, query head): the keys one after the other, running
// maximum and sum of the softmax.  Lane l holds elements l, l + 32, ...
__global__ void __launch_bounds__(128) prompt_simple_kernel(rvq_prompt_attn_args a) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (unit >= a.tokens * a.n_heads) return;
    const int64_t tok = unit / a.n_heads;
    const int h = (int)(unit - tok * a.n_heads), g = h / (a.n_heads / a.n_kv);
    int64_t q0 = 0, q1 = a.tokens, k0 = 0, k1 = a.keys;
    if (a.cu_q != nullptr) {
        int lo = 0, hi = a.n_seq;                 // the last sequence that starts at or before tok
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (a.cu_q[mid] <= tok) lo = mid;
            else hi = mid;
        }
        q0 = max(0, a.cu_q[lo]), q1 = min(a.tokens, (int64_t)a.cu_q[lo + 1]);
        const int32_t* cu_k = a.cu_k != nullptr ? a.cu_k : a.cu_q;
        k0 = max((int64_t)0, (int64_t)cu_k[lo]), k1 = min(a.keys, (int64_t)cu_k[lo + 1]);
        if (tok < q0 || tok >= q1) return;
    }
    const int64_t lk = max((int64_t)0, k1 - k0);
    const int64_t n = a.causal ? min(lk, tok - q0 + 1 + lk - (q1 - q0)) : lk;
    const int hd = a.head_dim;
    float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < 4; ++j) {
        const int d = lane + 32 * j;
        qv[j] = d < hd ? load_as_f32(a.q, tok * a.q_stride[0] + h * a.q_stride[1] + d, a.kind) : 0.f;
    }
    float m = -INFINITY, sum = 0.f;
    for (int64_t i = 0; i < n; ++i) {
        const int64_t kr = (k0 + i) * a.k_stride[0] + g * a.k_stride[1];
        const int64_t vr = (k0 + i) * a.v_stride[0] + g * a.v_stride[1];
        float s = 0.f;
        for (int j = 0; j < 4; ++j)
            if (lane + 32 * j < hd) s = fmaf(qv[j], load_as_f32(a.k, kr + lane + 32 * j, a.kind), s);
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= a.scaling;
        const float mn = fmaxf(m, s);
        const float old = mn == -INFINITY ? 1.f : expf(m - mn), p = mn == -INFINITY ? expf(s) : expf(s - mn);
        sum = sum * old + p;
        for (int j = 0; j < 4; ++j)
            if (lane + 32 * j < hd) acc[j] = acc[j] * old + p * load_as_f32(a.v, vr + lane + 32 * j, a.kind);
        m = mn;
    }
    for (int j = 0; j < 4; ++j) {
        const int d = lane + 32 * j;
        if (d < hd)
            store_from_f32(a.out, tok * a.out_stride[0] + h * a.out_stride[1] + d, a.kind, sum != 0.f ? acc[j] / sum : 0.f);
    }
    if (a.lse != nullptr && lane == 0) a.lse[(int64_t)h * a.tokens + tok] = m + logf(sum);
}

int check(const rvq_prompt_attn_args* a) {
    if (a == nullptr || a->tokens < 0 || a->keys < 0 || a->n_seq < 1) return RVQ_ERR_INVALID;
    if (a->n_kv < 1 || a->n_heads < a->n_kv || a->n_heads % a->n_kv != 0) return RVQ_ERR_INVALID;
    if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8 || a->n_heads / a->n_kv > 64) return RVQ_ERR_UNSUPPORTED;
    if (a->kind != RVQ_BF16 && a->kind != RVQ_F16) return RVQ_ERR_UNSUPPORTED;
    if (a->tokens >= (1ll << 31) || a->keys >= (1ll << 31)) return RVQ_ERR_TOO_LARGE;
    if (a->tokens > 0 && (a->q == nullptr || a->out == nullptr)) return RVQ_ERR_INVALID;
    if (a->keys > 0 && (a->k == nullptr || a->v == nullptr)) return RVQ_ERR_INVALID;
    if (a->cu_q == nullptr && (a->n_seq != 1 || a->cu_k != nullptr)) return RVQ_ERR_INVALID;
    if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out) & 15) return RVQ_ERR_INVALID;
    for (int i = 0; i < 2; ++i) {
        const int64_t s[4] = {a->q_stride[i], a->k_stride[i], a->v_stride[i], a->out_stride[i]};
        for (int j = 0; j < 4; ++j)
            if (s[j] < 8 || s[j] % 8 || s[j] >= (1ll << 39)) return RVQ_ERR_INVALID;
    }
    return RVQ_OK;
}

}  // namespace prompt
}  // namespace rvq

using namespace rvq;
using namespace rvq::prompt;

extern "C" size_t rvq_prompt_attention_workspace_size(const rvq_prompt_attn_args* a) {
    return 0;
}

extern "C" int rvq_prompt_attention(const rvq_prompt_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check(a);
    if (rc != RVQ_OK || a->tokens == 0) return rc;
    const int64_t blocks = (a->tokens * a->n_heads + 3) / 4;
    if (blocks >= (1ll << 31)) return RVQ_ERR_TOO_LARGE;
    const cudaError_t e = launch_pdl(prompt_simple_kernel, dim3((unsigned)blocks), dim3(128), 0, (cudaStream_t)stream, *a);
    if (e != cudaSuccess) last_cuda_error_slot() = (int)e;
    return e == cudaSuccess ? RVQ_OK : RVQ_ERR_CUDA;
}

extern "C" int rvq_take_attention_timeout(void) {
    int v = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, g_attention_timeout, sizeof(int));
    const int zero = 0;
    if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_attention_timeout, &zero, sizeof(int));
    if (e != cudaSuccess) {
        last_cuda_error_slot() = (int)e;
        return -RVQ_ERR_CUDA;
    }
    const int step = take_step_timeout();
    return step < 0 ? step : v | step;
}
