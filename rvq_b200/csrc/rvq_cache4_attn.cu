// Step attention over the 4-bit cache (rvq_cache4_attention, include/rvq_b200.h).

#include <string.h>

#include "rvq_cache4.cuh"
#include "rvq_stepops.cuh"

namespace rvq {
namespace cache4 {

using namespace stepops;

constexpr int kAttnThreads = 256;
constexpr int kAttnWarps = kAttnThreads / 32;
constexpr int kMaxRep = 64;

// Extremes of a group held by 8 adjacent lanes x 4 values; NaN if it holds one.
__device__ __forceinline__ void extremes(const float (&v)[4], float* lo, float* hi) {
    float l = v[0], h = v[0];
    bool bad = v[0] != v[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) l = fminf(l, v[i]), h = fmaxf(h, v[i]), bad |= v[i] != v[i];
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        l = fminf(l, __shfl_xor_sync(0xffffffffu, l, o));
        h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, o));
        bad |= __shfl_xor_sync(0xffffffffu, (int)bad, o) != 0;
    }
    *lo = bad ? NAN : l;
    *hi = bad ? NAN : h;
}

// Byte of value d's code within the codes of a row, by the record's order.
template <int HD>
__device__ __forceinline__ int code_byte(int d) {
    return (d % 32 / 8 * (HD / kGroup) + d / 32) * 4 + d % 8 / 2;
}

template <int HD>
__device__ __forceinline__ float held(const uint8_t* rec, int which, int d) {
    const uint32_t c = rec[which * (HD / 2) + code_byte<HD>(d)] >> (4 * (d & 1)) & 15;
    const uint32_t p = reinterpret_cast<const uint32_t*>(rec + HD + which * (HD / 8))[d / 32];
    return value_of(c, zero_of(p), step_of(p));
}

// One CTA per (kv head, sequence); warp per query head, the keys one by one.
template <int HD>
__global__ void __launch_bounds__(kAttnThreads) cache4_attn_simple_kernel(rvq_cache4_attn_args a) {
    constexpr int J = HD / 32, REC = record_bytes(HD);
    __shared__ float norm[4][HD];
    __shared__ float raw[HD], qs[kAttnWarps][HD];
    __shared__ float top[kMaxRep], total[kMaxRep];
    pdl_launch_dependents();
    pdl_wait();
    const int g = blockIdx.x, b = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nkv = a.cache.n_kv, rep = a.n_heads / nkv;
    const int64_t rows = a.rows[b];
    if (rows < 0) return;
    const bool append = a.k.ptr != nullptr;
    const int64_t n = rows + (append ? 1 : 0);
    const int64_t pos = a.pos != nullptr ? a.pos[b] : 0;
    const int64_t q_at = ((int64_t)b * a.n_heads + g * rep) * HD, kv_at = ((int64_t)b * nkv + g) * HD;
    const int out_kind = a.q.kind == RVQ_F16 ? RVQ_F16 : RVQ_BF16;
    if (n < 1 || n > a.cache.max_len || pos < 0 || (a.pos != nullptr && pos >= a.table_len)) {
        for (int i = tid; i < rep * HD; i += kAttnThreads) store_from_f32(a.out, q_at + i, out_kind, 0.f);
        return;
    }
    for (int i = tid; i < HD; i += kAttnThreads) {
        norm[0][i] = a.q_norm != nullptr ? bf16_at(a.q_norm, i) : 0.f;
        norm[1][i] = a.q_norm != nullptr ? bf16_at(a.k_norm, i) : 0.f;
        norm[2][i] = a.cos != nullptr ? bf16_at(a.cos, pos * HD + i) : 1.f;
        norm[3][i] = a.cos != nullptr ? bf16_at(a.sin, pos * HD + i) : 0.f;
    }
    uint8_t* base = reinterpret_cast<uint8_t*>(a.cache.data) + ((int64_t)b * nkv + g) * a.cache.max_len * REC;
    __syncthreads();
    auto prepare = [&](const float* x, const float* w, float* o) {       // norm and rotation of one head by one warp
        float v[J];
        float ss = 0.f;
        for (int j = 0; j < J; ++j) v[j] = x[lane + 32 * j], ss = fmaf(v[j], v[j], ss);
        if (a.q_norm != nullptr) {
            const float inv = rsqrtf(warp_sum(ss) / (float)HD + a.eps);
            for (int j = 0; j < J; ++j) v[j] = bf16r(w[lane + 32 * j] * bf16r(v[j] * inv));
        }
        for (int j = 0; j < J; ++j) {
            const int d = lane + 32 * j;
            const float rot = j < J / 2 ? -v[j + J / 2] : v[j - J / 2];
            o[d] = a.cos != nullptr ? bf16r(bf16r(v[j] * norm[2][d]) + bf16r(rot * norm[3][d])) : v[j];
        }
    };
    if (append) {
        uint8_t* rec = base + rows * REC;
        for (int which = 0; which < 2; ++which) {
            for (int i = tid; i < HD; i += kAttnThreads) raw[i] = vec_value(which ? a.v : a.k, kv_at + i);
            __syncthreads();
            if (warp == 0 && which == 0) prepare(raw, norm[1], raw);
            __syncthreads();
            if (warp == 0) {                              // the whole warp: extremes shuffles
                float v[4], lo, hi;
                for (int i = 0; i < 4; ++i) v[i] = raw[(4 * tid + i) % HD];
                extremes(v, &lo, &hi);
                const uint32_t p = params_of(lo, hi);
                for (int i = 0; i < 4 && tid < HD / 4; i += 2)
                    rec[which * (HD / 2) + code_byte<HD>(4 * tid + i)] =
                        (uint8_t)(code_of(v[i], zero_of(p), step_of(p)) | code_of(v[i + 1], zero_of(p), step_of(p)) << 4);
                if (tid % 8 == 0 && tid < HD / 4) reinterpret_cast<uint32_t*>(rec + HD + which * (HD / 8))[tid / 8] = p;
            }
            __syncthreads();
        }
    }
    for (int r = warp; r < rep; r += kAttnWarps) {
        for (int d = lane; d < HD; d += 32) qs[warp][d] = vec_value(a.q, q_at + r * HD + d);
        __syncwarp();
        prepare(qs[warp], norm[0], qs[warp]);
        __syncwarp();
        float m = -INFINITY, sum = 0.f, acc[J];
        for (int j = 0; j < J; ++j) acc[j] = 0.f;
        float* sc = a.weights != nullptr ? a.scores + ((int64_t)b * a.n_heads + g * rep + r) * a.cache.max_len : nullptr;
        for (int64_t i = 0; i < n; ++i) {
            float s = 0.f;
            for (int j = 0; j < J; ++j)
                s = fmaf(qs[warp][lane + 32 * j], held<HD>(base + i * REC, 0, lane + 32 * j), s);
            s = warp_sum(s) * a.scaling;
            if (sc != nullptr && lane == 0) sc[i] = s;
            const float mn = fmaxf(m, s);
            const float old = mn == -INFINITY ? 1.f : expf(m - mn), p = mn == -INFINITY ? expf(s) : expf(s - mn);
            sum = sum * old + p;
            for (int j = 0; j < J; ++j) acc[j] = acc[j] * old + p * held<HD>(base + i * REC, 1, lane + 32 * j);
            m = mn;
        }
        for (int j = 0; j < J; ++j) store_from_f32(a.out, q_at + r * HD + lane + 32 * j, out_kind, sum != 0.f ? acc[j] / sum : 0.f);
        if (lane == 0) top[r] = m, total[r] = sum;
        __syncwarp();
    }
    if (a.weights == nullptr) return;
    __syncthreads();
    float* w = a.weights + ((int64_t)b * nkv + g) * a.cache.max_len;
    const float* sc = a.scores + ((int64_t)b * a.n_heads + g * rep) * a.cache.max_len;
    for (int64_t i = tid; i < n; i += kAttnThreads) {
        float t = append && i == rows ? 0.f : w[i];
        for (int r = 0; r < rep; ++r) if (total[r] != 0.f) t += expf(sc[(int64_t)r * a.cache.max_len + i] - top[r]) / total[r];
        w[i] = t;
    }
}

bool vec_fits(const rvq_vec& v, int64_t n) {
    if (v.ptr == nullptr || v.n != n || v.ntiles < 1) return false;
    return v.kind == RVQ_F32 || ((v.kind == RVQ_BF16 || v.kind == RVQ_F16) && v.ntiles == 1);
}

int check(const rvq_cache4_attn_args* a) {
    if (a == nullptr) return RVQ_ERR_INVALID;
    const rvq_cache4& c = a->cache;
    if (c.data == nullptr || c.n_seq < 1 || c.n_kv < 1 || c.max_len < 1 || ((uintptr_t)c.data & 15)) return RVQ_ERR_INVALID;
    if (c.head_dim != 64 && c.head_dim != 128) return RVQ_ERR_UNSUPPORTED;
    if (a->n_heads < c.n_kv || a->n_heads % c.n_kv) return RVQ_ERR_INVALID;
    if (a->n_heads / c.n_kv > kMaxRep) return RVQ_ERR_UNSUPPORTED;
    if (a->rows == nullptr || a->out == nullptr || ((uintptr_t)a->out & 15)) return RVQ_ERR_INVALID;
    if (!vec_fits(a->q, (int64_t)c.n_seq * a->n_heads * c.head_dim)) return RVQ_ERR_INVALID;
    if ((a->k.ptr == nullptr) != (a->v.ptr == nullptr)) return RVQ_ERR_INVALID;
    if (a->k.ptr != nullptr) {
        const int64_t n = (int64_t)c.n_seq * c.n_kv * c.head_dim;
        if (!vec_fits(a->k, n) || !vec_fits(a->v, n) || a->k.kind != a->q.kind || a->v.kind != a->q.kind)
            return RVQ_ERR_INVALID;
    }
    if ((a->q_norm == nullptr) != (a->k_norm == nullptr)) return RVQ_ERR_INVALID;
    if ((a->cos == nullptr) != (a->sin == nullptr) || (a->cos == nullptr) != (a->pos == nullptr)) return RVQ_ERR_INVALID;
    if (a->cos != nullptr && a->table_len < 1) return RVQ_ERR_INVALID;
    if (a->q.kind == RVQ_F16 && (a->q_norm != nullptr || a->cos != nullptr)) return RVQ_ERR_UNSUPPORTED;
    if (a->weights != nullptr && a->scores == nullptr) return RVQ_ERR_INVALID;
    if (c.n_seq > 65535 || c.n_kv > 65535) return RVQ_ERR_TOO_LARGE;
    return RVQ_OK;
}

}  // namespace cache4
}  // namespace rvq

using namespace rvq;
using namespace rvq::cache4;

extern "C" int rvq_cache4_attention(const rvq_cache4_attn_args* a, void* stream) {
    const int rc = check(a);
    if (rc != RVQ_OK) return rc;
    auto* kernel = a->cache.head_dim == 128 ? cache4_attn_simple_kernel<128> : cache4_attn_simple_kernel<64>;
    const cudaError_t e = launch_pdl(kernel, dim3(a->cache.n_kv, a->cache.n_seq), dim3(kAttnThreads), 0,
                                     (cudaStream_t)stream, *a);
    if (e != cudaSuccess) last_cuda_error_slot() = (int)e;
    return e == cudaSuccess ? RVQ_OK : RVQ_ERR_CUDA;
}
