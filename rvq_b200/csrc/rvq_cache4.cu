// The 4-bit key / value cache: rows in and out (rvq_cache4_write, _read) and
// eviction (rvq_cache4_evict).  The step attention over it is in rvq_cache4_attn.cu.

#include <string.h>

#include "rvq_cache4.cuh"

namespace rvq {
namespace cache4 {

constexpr int kRowsThreads = 256;

__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Record of packed token `tok` and its kv head, or NULL where the token is in
// no sequence; *row_ok: the row lies in the cache.
__device__ __forceinline__ uint8_t* record_of(const rvq_cache4_rows_args& a, int64_t tok, int g, int rec, bool* row_ok) {
    int b = 0;
    int64_t i = tok;
    if (a.cu != nullptr) {
        int hi = a.cache.n_seq;                   // the last sequence that starts at or before tok
        while (hi - b > 1) {
            const int mid = (b + hi) / 2;
            if (__ldg(a.cu + mid) <= tok) b = mid;
            else hi = mid;
        }
        i = tok - __ldg(a.cu + b);
        if (i < 0 || tok >= __ldg(a.cu + b + 1)) return nullptr;
    }
    const int64_t row = (a.start != nullptr ? __ldg(a.start + b) : 0) + i;
    *row_ok = row >= 0 && row < a.cache.max_len;
    return reinterpret_cast<uint8_t*>(a.cache.data) +
           (((int64_t)b * a.cache.n_kv + g) * a.cache.max_len + (*row_ok ? row : 0)) * rec;
}

// HD / 4 adjacent threads per (token, kv head): half of them K, half V; four
// adjacent ones hold a group, 8 values (one 16-byte load or store) each, which
// are one code word.  A warp's code words fill whole 32-byte sectors.
template <int HD, bool kWrite>
__global__ void __launch_bounds__(kRowsThreads) cache4_rows_kernel(rvq_cache4_rows_args a) {
    constexpr int T = HD / 4, G = HD / kGroup;
    pdl_launch_dependents();
    pdl_wait();
    const int64_t idx = (int64_t)blockIdx.x * kRowsThreads + threadIdx.x;
    const int64_t unit = idx / T;
    const bool live = unit < a.tokens * a.cache.n_kv;
    const int in = (int)(idx % T), which = in / (T / 2), grp = in % (T / 2) / 4, w = in & 3;
    const int64_t tok = live ? unit / a.cache.n_kv : 0;
    const int g = live ? (int)(unit - tok * a.cache.n_kv) : 0;
    bool row_ok = false;
    uint8_t* rec = live ? record_of(a, tok, g, record_bytes(HD), &row_ok) : nullptr;
    const int64_t* st = which ? a.v_stride : a.k_stride;
    uint4* x = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(which ? a.v : a.k) + tok * st[0] + g * st[1] +
                                        grp * kGroup + 8 * w);
    uint32_t* codes = reinterpret_cast<uint32_t*>(rec + which * (HD / 2)) + w * G + grp;
    uint32_t* params = reinterpret_cast<uint32_t*>(rec + HD + which * (HD / 8)) + grp;
    if constexpr (kWrite) {
        const uint4 raw = rec != nullptr ? *x : make_uint4(0, 0, 0, 0);
        const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint16_t u = (uint16_t)(r[i / 2] >> (16 * (i & 1)));
            v[i] = a.kind == RVQ_F16 ? __half2float(__ushort_as_half(u)) : __bfloat162float(__ushort_as_bfloat16(u));
        }
        float lo = v[0], hi = v[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) lo = min_nan(lo, v[i]), hi = max_nan(hi, v[i]);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const uint32_t p = params_of(lo, hi);
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) word |= code_of(v[i], zero_of(p), step_of(p)) << (4 * i);
        if (rec != nullptr && row_ok) {
            *codes = word;
            if (w == 0) *params = p;
        }
    } else if (rec != nullptr) {
        const uint32_t word = row_ok ? *codes : 0, p = row_ok ? *params : 0;
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = pack2(value_of(word >> (8 * i) & 15, zero_of(p), step_of(p)),
                         value_of(word >> (8 * i + 4) & 15, zero_of(p), step_of(p)), a.kind);
        *x = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// ---------------------------------------------------------------------------
// Eviction.  select: a CTA per (sequence, kv head) finds the (keep - recent)-th
// largest weight of the older rows bit by bit, then walks the rows in order and
// writes the kept ones' indices and weights.  move: the records follow.  Rows
// only move down, so a chunk that is loaded whole before it is stored never
// overwrites a row that is still to be read: the same walk serves in place.
// ---------------------------------------------------------------------------
constexpr int kEvictThreads = 1024;

// Weights ordered as unsigned integers: -0 as 0, NaN above everything.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ int64_t live_rows(const rvq_cache4_evict_args& a, int b) {
    const int64_t n = a.rows[b];
    return n > a.cache.max_len ? a.cache.max_len : n;
}

__global__ void __launch_bounds__(kEvictThreads) evict_select_kernel(rvq_cache4_evict_args a) {
    __shared__ int red[kEvictThreads / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x / a.cache.n_kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t n = live_rows(a, b);
    const float* w = a.weights + (int64_t)blockIdx.x * a.cache.max_len;
    float* wo = a.out_weights + (int64_t)blockIdx.x * a.out.max_len;
    int32_t* kept = a.kept + (int64_t)blockIdx.x * a.keep;
    if (a.new_rows != nullptr && blockIdx.x % a.cache.n_kv == 0 && tid == 0)
        a.new_rows[b] = n < a.keep ? n : a.keep;
    const int64_t old = n > a.keep ? n - a.recent : 0;      // rows [0, old) compete for want places
    const int want = a.keep - a.recent;
    uint32_t bar = 0;
    int ties = 0;
    if (n > a.keep && want > 0) {
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t cand = bar | 1u << bit;
            int c = 0;
            for (int64_t i = tid; i < old; i += kEvictThreads) c += order_key(w[i]) >= cand;
            for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
            __syncthreads();
            if (lane == 0) red[warp] = c;
            __syncthreads();
            int t = 0;
            for (int i = 0; i < kEvictThreads / 32; ++i) t += red[i];
            if (t >= want) bar = cand;
        }
        int c = 0;
        for (int64_t i = tid; i < old; i += kEvictThreads) c += order_key(w[i]) > bar;
        for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
        __syncthreads();
        if (lane == 0) red[warp] = c;
        __syncthreads();
        ties = want;
        for (int i = 0; i < kEvictThreads / 32; ++i) ties -= red[i];
    }
    int64_t at = 0;                                         // rows written so far
    int tied = 0;                                           // equal rows seen so far
    for (int64_t base = 0; base < n; base += kEvictThreads) {
        const int64_t i = base + tid;
        const float v = i < n ? w[i] : 0.f;
        const uint32_t key = order_key(v);
        const bool older = i < old;
        const bool tie = older && want > 0 && key == bar;
        const uint32_t tb = __ballot_sync(0xffffffffu, tie);
        __syncthreads();
        if (lane == 0) red[warp] = __popc(tb);
        __syncthreads();
        int rank = tied + __popc(tb & ((1u << lane) - 1));
        for (int k = 0; k < kEvictThreads / 32; ++k) {
            if (k < warp) rank += red[k];
            tied += red[k];
        }
        const bool keep = i < n && (!older || (want > 0 && (key > bar || (tie && rank < ties))));
        const uint32_t kb = __ballot_sync(0xffffffffu, keep);
        __syncthreads();                                    // the chunk's weights are read, and red
        if (lane == 0) red[warp] = __popc(kb);
        __syncthreads();
        int64_t pos = at + __popc(kb & ((1u << lane) - 1));
        for (int k = 0; k < kEvictThreads / 32; ++k) {
            if (k < warp) pos += red[k];
            at += red[k];
        }
        if (keep) {
            kept[pos] = (int32_t)i;
            wo[pos] = v;
        }
    }
    for (int64_t i = (at > 0 ? at : 0) + tid; i < a.keep; i += kEvictThreads) kept[i] = -1;
}

constexpr int kMoveThreads = 512;

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(rvq_cache4_evict_args a, int vecs) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t n = live_rows(a, blockIdx.x / a.cache.n_kv);
    const bool in_place = a.out.data == a.cache.data;
    if (n <= 0 || (in_place && n <= a.keep)) return;
    const int count = (int)(n < a.keep ? n : a.keep);
    const uint4* src = reinterpret_cast<const uint4*>(a.cache.data) + (int64_t)blockIdx.x * a.cache.max_len * vecs;
    uint4* dst = reinterpret_cast<uint4*>(a.out.data) + (int64_t)blockIdx.x * a.out.max_len * vecs;
    const int32_t* kept = a.kept + (int64_t)blockIdx.x * a.keep;
    constexpr int U = 4;
    const int64_t total = (int64_t)count * vecs;
    for (int64_t base = 0; base < total; base += kMoveThreads * U) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = base + u * kMoveThreads + threadIdx.x;
            if (i < total) v[u] = src[(int64_t)kept[i / vecs] * vecs + i % vecs];
        }
        if (in_place) __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = base + u * kMoveThreads + threadIdx.x;
            if (i < total) dst[i] = v[u];
        }
    }
}

int check_cache(const rvq_cache4& c) {
    if (c.data == nullptr || c.n_seq < 1 || c.n_kv < 1 || c.max_len < 1 || ((uintptr_t)c.data & 15)) return RVQ_ERR_INVALID;
    return c.head_dim == 64 || c.head_dim == 128 ? RVQ_OK : RVQ_ERR_UNSUPPORTED;
}

int check_rows(const rvq_cache4_rows_args* a) {
    if (a == nullptr || a->tokens < 0) return RVQ_ERR_INVALID;
    const int rc = check_cache(a->cache);
    if (rc != RVQ_OK) return rc;
    if (a->kind != RVQ_BF16 && a->kind != RVQ_F16) return RVQ_ERR_UNSUPPORTED;
    if (a->tokens > 0 && (a->k == nullptr || a->v == nullptr)) return RVQ_ERR_INVALID;
    if (((uintptr_t)a->k | (uintptr_t)a->v) & 15) return RVQ_ERR_INVALID;
    if (a->cu == nullptr && a->cache.n_seq != 1) return RVQ_ERR_INVALID;
    if (a->tokens >= (1ll << 31)) return RVQ_ERR_TOO_LARGE;
    for (int i = 0; i < 2; ++i) {
        const int64_t s[2] = {a->k_stride[i], a->v_stride[i]};
        for (int j = 0; j < 2; ++j)
            if (s[j] < 8 || s[j] % 8 || s[j] >= (1ll << 39)) return RVQ_ERR_INVALID;
    }
    return RVQ_OK;
}

template <bool kWrite>
int run_rows(const rvq_cache4_rows_args* a, void* stream) {
    const int rc = check_rows(a);
    if (rc != RVQ_OK || a->tokens == 0) return rc;
    const int64_t blocks = (a->tokens * a->cache.n_kv * (a->cache.head_dim / 4) + kRowsThreads - 1) / kRowsThreads;
    if (blocks >= (1ll << 31)) return RVQ_ERR_TOO_LARGE;
    auto* kernel = a->cache.head_dim == 128 ? cache4_rows_kernel<128, kWrite> : cache4_rows_kernel<64, kWrite>;
    return status(launch_pdl(kernel, dim3((unsigned)blocks), dim3(kRowsThreads), 0, (cudaStream_t)stream, *a));
}

// Whether two byte ranges share a byte.
bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

int64_t cache_bytes(const rvq_cache4& c) {
    return (int64_t)c.n_seq * c.n_kv * c.max_len * record_bytes(c.head_dim);
}

}  // namespace cache4
}  // namespace rvq

using namespace rvq;
using namespace rvq::cache4;

extern "C" int rvq_cache4_record_bytes(int head_dim) {
    return head_dim == 64 || head_dim == 128 ? record_bytes(head_dim) : 0;
}

extern "C" int rvq_cache4_write(const rvq_cache4_rows_args* a, void* stream) { return run_rows<true>(a, stream); }

extern "C" int rvq_cache4_read(const rvq_cache4_rows_args* a, void* stream) { return run_rows<false>(a, stream); }

extern "C" int rvq_cache4_evict(const rvq_cache4_evict_args* a, void* stream) {
    if (a == nullptr) return RVQ_ERR_INVALID;
    int rc = check_cache(a->cache);
    if (rc == RVQ_OK) rc = check_cache(a->out);
    if (rc != RVQ_OK) return rc;
    const rvq_cache4 &c = a->cache, &o = a->out;
    if (a->weights == nullptr || a->out_weights == nullptr || a->rows == nullptr || a->kept == nullptr)
        return RVQ_ERR_INVALID;
    if (o.n_seq != c.n_seq || o.n_kv != c.n_kv || o.head_dim != c.head_dim || o.max_len < a->keep) return RVQ_ERR_INVALID;
    if (a->keep < 1 || a->keep > c.max_len || a->recent < 0 || a->recent > a->keep) return RVQ_ERR_INVALID;
    const int64_t heads = (int64_t)c.n_seq * c.n_kv;
    if (heads >= (1ll << 31)) return RVQ_ERR_TOO_LARGE;
    if (o.data == c.data ? o.max_len != c.max_len : overlap(c.data, cache_bytes(c), o.data, cache_bytes(o)))
        return RVQ_ERR_INVALID;
    if (a->out_weights == a->weights ? o.max_len != c.max_len
                                     : overlap(a->weights, heads * c.max_len * 4, a->out_weights, heads * o.max_len * 4))
        return RVQ_ERR_INVALID;
    if (a->new_rows != nullptr && overlap(a->rows, 8ll * c.n_seq, a->new_rows, 8ll * c.n_seq)) return RVQ_ERR_INVALID;
    rc = status(launch_pdl(evict_select_kernel, dim3((unsigned)heads), dim3(kEvictThreads), 0, (cudaStream_t)stream, *a));
    if (rc != RVQ_OK) return rc;
    return status(launch_pdl(evict_move_kernel, dim3((unsigned)heads), dim3(kMoveThreads), 0, (cudaStream_t)stream, *a,
                             record_bytes(c.head_dim) / 16));
}
