// The 4-bit key / value cache: rows in and out (rvq_cache4_write, _read) and
// eviction (rvq_cache4_evict).  The step attention over it is in rvq_cache4_attn.cu.

#include <string.h>

#include "rvq_cache4.cuh"

namespace rvq {
namespace cache4 {

constexpr int kRowsThreads = 256;

// Two 16-bit minima or maxima; a NaN stays.
template <int kKind, bool kMax>
__device__ __forceinline__ uint32_t extreme2(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (kKind == RVQ_F16) {
        if constexpr (kMax) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    } else {
        if constexpr (kMax) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    }
    return d;
}

template <int kKind>
__device__ __forceinline__ float half_value(uint32_t w, int i) {
    const uint16_t h = (uint16_t)(w >> (16 * (i & 1)));
    return kKind == RVQ_F16 ? __half2float(__ushort_as_half(h)) : __bfloat162float(__ushort_as_bfloat16(h));
}

// The extreme of the group that four adjacent lanes hold, 8 values each.
template <int kKind, bool kMax>
__device__ __forceinline__ float group_extreme(const uint32_t (&r)[4]) {
    uint32_t m = extreme2<kKind, kMax>(extreme2<kKind, kMax>(r[0], r[1]), extreme2<kKind, kMax>(r[2], r[3]));
    m = extreme2<kKind, kMax>(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = extreme2<kKind, kMax>(m, __shfl_xor_sync(0xffffffffu, m, 2));
    return half_value<kKind>(extreme2<kKind, kMax>(m, m >> 16), 0);
}

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Record of packed token `tok` and kv head g, or NULL where the token is in no sequence; *row_ok: the row lies in the cache.
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

// HD / 4 adjacent threads per token of the block's kv head: half of them K, half V; four adjacent ones hold a group, 8
// values (one 16-byte load or store) each, which are one code word.  A block's tokens are neighbouring records, so code
// words and parameters fill whole sectors.  (Two or four tokens a thread: 4,096 tokens as fast, 700 at half the speed.)  Bound by
// the issue of instructions (write: issue 87 %, ALU pipe 60 %, DRAM 32 %; read: 78, 54 and 38 %): 8 heads of 128, 65,536 tokens
// written in 125 us (2.8 TB/s moved) and read in 92 us (3.8 TB/s), 1.9 and 1.4 us for every further 1,000 tokens; 4,096 tokens, in L2, 8.9
// and 6.4 us; 9 sequences of up to 700 tokens, 2 heads of 64: 3.5 and 2.6 us, a launch.

template <int HD, bool kWrite, int kKind>
__global__ void __launch_bounds__(kRowsThreads) cache4_rows_kernel(rvq_cache4_rows_args a) {
    constexpr int T = HD / 4, G = HD / kGroup, B = kRowsThreads / T;
    pdl_launch_dependents();
    pdl_wait();
    const int in = threadIdx.x % T, which = in / (T / 2), grp = in % (T / 2) / 4, w = in & 3;
    const int g = blockIdx.y;
    const int64_t* st = which ? a.v_stride : a.k_stride;
    uint16_t* base = reinterpret_cast<uint16_t*>(which ? a.v : a.k) + g * st[1] + grp * kGroup + 8 * w;
    const int64_t tok = (int64_t)blockIdx.x * B + threadIdx.x / T;
    uint4* x = reinterpret_cast<uint4*>(base + tok * st[0]);
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (kWrite && tok < a.tokens) raw = *x;                  // on its way while the row is looked up
    bool row_ok = false;
    uint8_t* rec = tok < a.tokens ? record_of(a, tok, g, record_bytes(HD), &row_ok) : nullptr;
    uint32_t* codes = reinterpret_cast<uint32_t*>(rec + which * (HD / 2)) + w * G + grp;
    uint32_t* params = reinterpret_cast<uint32_t*>(rec + HD + which * (HD / 8)) + grp;
    if constexpr (kWrite) {
        const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
        const uint32_t p = params_of(group_extreme<kKind, false>(r), group_extreme<kKind, true>(r));
        const float zero = zero_of(p), step = step_of(p), inv = rcp_approx(step);
        uint32_t word = 0, again = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            bool near;
            word |= code_near<kKind == RVQ_F16>(half_value<kKind>(r[i / 2], i), zero, step, inv, &near) << (4 * i);
            again |= (uint32_t)near << i;
        }
        while (again) {                                      // few: these divide
            const int i = __ffs(again) - 1;
            again &= again - 1;
            const float v = half_value<kKind>(i < 4 ? i < 2 ? r[0] : r[1] : i < 6 ? r[2] : r[3], i);
            word = (word & ~(15u << (4 * i))) | code_of(v, zero, step) << (4 * i);
        }
        if (rec != nullptr && row_ok) {
            *codes = word;
            if (w == 0) *params = p;
        }
    } else if (rec != nullptr) {
        const uint32_t word = row_ok ? *codes : 0, p = row_ok ? *params : 0;
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = pack2(value_of(word >> (8 * i) & 15, zero_of(p), step_of(p)), value_of(word >> (8 * i + 4) & 15, zero_of(p), step_of(p)),
                         kKind);
        *x = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// ---------------------------------------------------------------------------
// Eviction.  select: a CTA per (sequence, kv head) finds the (keep - recent)-th
// largest weight of the older rows, 11, 11 and 10 bits of it a pass by a histogram
// in shared memory (and no further than it takes to tell the wanted rows from the
// others), then writes the kept rows' indices in order (each warp a contiguous
// part of the rows, whose counts are added up first) and gathers the weights.
// Up to 8,192 rows stay in registers over the passes.
// move: the records follow.  Rows only move down, so rows that are loaded before
// any row behind them is stored over serve in place too.
//
// 36 x 8 heads, up to 8,500 rows to 4,096: select 26 us (latency of its passes: a CTA
// a head), move 64 us, 378 MB at 5.9 TB/s; together 91 us.  1 x 8 heads, 1,100 rows to
// 1,024: 11 us, two launches and the passes' barriers.
// ---------------------------------------------------------------------------
constexpr int kEvictThreads = 1024;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kAhead = 8;                    // rows that a thread loads before it looks at them

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
    __shared__ int hist[2048];
    __shared__ int above[kEvictWarps], equal[kEvictWarps];
    __shared__ uint32_t sh_bar;
    __shared__ int sh_want, sh_count;
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x / a.cache.n_kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t live = live_rows(a, b);
    const int n = (int)(live < 0 ? 0 : live);
    const float* w = a.weights + (int64_t)blockIdx.x * a.cache.max_len;
    float* wo = a.out_weights + (int64_t)blockIdx.x * a.out.max_len;
    int32_t* kept = a.kept + (int64_t)blockIdx.x * a.keep;
    if (a.new_rows != nullptr && blockIdx.x % a.cache.n_kv == 0 && tid == 0) a.new_rows[b] = live < a.keep ? live : a.keep;
    if (n <= a.keep) {                                      // every row stays
        for (int i = tid; i < a.keep; i += kEvictThreads) {
            kept[i] = i < n ? i : -1;
            if (i < n && wo != w) wo[i] = w[i];
        }
        return;
    }
    const int old = n - a.recent;                           // rows [0, old) compete for want places
    uint32_t bar = 0, mask = 0;                             // the bits of the want-th largest key found so far
    int want = a.keep - a.recent;                           // among the keys with those bits
    const bool select = want > 0;
    if (select) {
        const bool resident = old <= kEvictThreads * kAhead;
        float x[kAhead];
        auto fill = [&](int base) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) x[u] = base + u * kEvictThreads + tid < old ? w[base + u * kEvictThreads + tid] : 0.f;
        };
        if (resident) fill(0);
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
            const uint32_t digit = pass == 2 ? 1023u : 2047u;
            hist[tid] = hist[tid + 1024] = 0;
            __syncthreads();
            for (int base = 0; base < old; base += kEvictThreads * kAhead) {
                if (!resident) fill(base);
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const uint32_t key = order_key(x[u]);
                    if (base + u * kEvictThreads + tid < old && (key & mask) == bar) atomicAdd(&hist[key >> shift & digit], 1);
                }
            }
            __syncthreads();
            // the bin where the count from the top reaches want; thread t: bins 2047 - 2 t and 2046 - 2 t
            const int c0 = hist[2047 - 2 * tid], c1 = hist[2046 - 2 * tid];
            int upto = c0 + c1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            if (lane == 31) above[warp] = upto;
            __syncthreads();
            int before = lane < warp ? above[lane] : 0;     // summed over the lanes: the warps before this one
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
            before += upto - c0 - c1;
            if (before < want && want <= before + c0 + c1) {
                const bool second = want > before + c0;
                sh_bar = bar | (uint32_t)(2047 - 2 * tid - second) << shift;
                sh_want = want - before - (second ? c0 : 0);
                sh_count = second ? c1 : c0;
            }
            __syncthreads();
            bar = sh_bar;
            want = sh_want;
            mask |= digit << shift;
            if (want == sh_count) {                         // every key with these bits is wanted: all above bar - 1
                --bar;
                want = 0;
                break;
            }
        }
    }
    // rows above bar, and the first `want` of those at it; each warp its part of the rows
    const int part = (n + kEvictThreads - 1) / kEvictThreads * 32;
    const int r0 = min(n, warp * part), r1 = min(n, r0 + part);
    int na = 0, ne = 0;
    for (int base = r0; base < r1; base += 32 * kAhead) {
        float x[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) x[u] = base + 32 * u + lane < r1 ? w[base + 32 * u + lane] : 0.f;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = base + 32 * u + lane;
            const uint32_t key = order_key(x[u]);
            na += __popc(__ballot_sync(0xffffffffu, i < r1 && (i >= old || (select && key > bar))));
            ne += __popc(__ballot_sync(0xffffffffu, i < r1 && i < old && select && key == bar));
        }
    }
    if (lane == 0) above[warp] = na, equal[warp] = ne;
    __syncthreads();
    int pos = 0, tied = 0;                                  // rows kept, and rows at bar, before this warp's
    for (int k = 0; k < warp; ++k) {
        pos += above[k];
        tied += equal[k];
    }
    pos += min(tied, want);
    for (int base = r0; base < r1; base += 32 * kAhead) {
        float x[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) x[u] = base + 32 * u + lane < r1 ? w[base + 32 * u + lane] : 0.f;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = base + 32 * u + lane;
            const uint32_t key = order_key(x[u]);
            const bool tie = i < r1 && i < old && select && key == bar;
            const uint32_t tb = __ballot_sync(0xffffffffu, tie);
            const uint32_t below = (1u << lane) - 1;
            const bool keep = i < r1 && (i >= old || (select && key > bar) || (tie && tied + __popc(tb & below) < want));
            const uint32_t kb = __ballot_sync(0xffffffffu, keep);
            if (keep) kept[pos + __popc(kb & below)] = i;
            pos += __popc(kb);
            tied += __popc(tb);
        }
    }
    __syncthreads();                                        // kept is complete, and the old weights are read
    constexpr int U = kAhead;
    for (int base = 0; base < a.keep; base += kEvictThreads * U) {
        float v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = base + u * kEvictThreads + tid;
            if (i < a.keep) v[u] = w[kept[i]];
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = base + u * kEvictThreads + tid;
            if (i < a.keep) wo[i] = v[u];
        }
    }
}

constexpr int kMoveThreads = 256;
constexpr int kMoveLoads = 4;

// blockIdx.y: apart, a part of the rows; in place, a fifth of every record (its rows depend on one another, its columns do
// not): 32 or 16 bytes wide, whole sectors of a head_dim 128 record.
template <int VECS>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(rvq_cache4_evict_args a) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t live = live_rows(a, blockIdx.x / a.cache.n_kv);
    const bool in_place = a.out.data == a.cache.data;
    if (live <= 0 || (in_place && live <= a.keep)) return;
    const int count = (int)(live < a.keep ? live : a.keep);
    const uint4* src = reinterpret_cast<const uint4*>(a.cache.data) + (int64_t)blockIdx.x * a.cache.max_len * VECS;
    uint4* dst = reinterpret_cast<uint4*>(a.out.data) + (int64_t)blockIdx.x * a.out.max_len * VECS;
    const int32_t* kept = a.kept + (int64_t)blockIdx.x * a.keep;
    constexpr int U = kMoveLoads, W = VECS / 5;
    if (!in_place) {
        const int64_t total = (int64_t)count * VECS;
        for (int64_t base = (int64_t)blockIdx.y * kMoveThreads * U; base < total; base += (int64_t)gridDim.y * kMoveThreads * U) {
            uint4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t i = base + u * kMoveThreads + threadIdx.x;
                const int row = (int)(i / VECS);
                if (i < total) v[u] = src[(int64_t)__ldg(kept + row) * VECS + (i - (int64_t)row * VECS)];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t i = base + u * kMoveThreads + threadIdx.x;
                if (i < total) dst[i] = v[u];
            }
        }
        return;
    }
    const int rows = kMoveThreads / W, col = blockIdx.y * W + threadIdx.x % W, r = threadIdx.x / W;
    for (int base = 0; base < count; base += rows * U) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (base + u * rows + r < count) v[u] = src[(int64_t)__ldg(kept + base + u * rows + r) * VECS + col];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (base + u * rows + r < count) dst[(int64_t)(base + u * rows + r) * VECS + col] = v[u];
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
    if (a->tokens > (1ll << 30)) return RVQ_ERR_TOO_LARGE;
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
    const int per_block = kRowsThreads / (a->cache.head_dim / 4);
    const int64_t blocks = (a->tokens + per_block - 1) / per_block;
    if (a->cache.n_kv > 65535) return RVQ_ERR_TOO_LARGE;
    auto* kernel = a->cache.head_dim == 128
                       ? a->kind == RVQ_F16 ? cache4_rows_kernel<128, kWrite, RVQ_F16> : cache4_rows_kernel<128, kWrite, RVQ_BF16>
                       : a->kind == RVQ_F16 ? cache4_rows_kernel<64, kWrite, RVQ_F16> : cache4_rows_kernel<64, kWrite, RVQ_BF16>;
    return status(launch_pdl(kernel, dim3((unsigned)blocks, a->cache.n_kv), dim3(kRowsThreads), 0, (cudaStream_t)stream, *a));
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
    if (heads >= (1ll << 31) || c.max_len > (1 << 30) || o.max_len > (1 << 30)) return RVQ_ERR_TOO_LARGE;
    if (o.data == c.data ? o.max_len != c.max_len : overlap(c.data, cache_bytes(c), o.data, cache_bytes(o)))
        return RVQ_ERR_INVALID;
    if (a->out_weights == a->weights ? o.max_len != c.max_len
                                     : overlap(a->weights, heads * c.max_len * 4, a->out_weights, heads * o.max_len * 4))
        return RVQ_ERR_INVALID;
    if (a->new_rows != nullptr && overlap(a->rows, 8ll * c.n_seq, a->new_rows, 8ll * c.n_seq)) return RVQ_ERR_INVALID;
    rc = status(launch_pdl(evict_select_kernel, dim3((unsigned)heads), dim3(kEvictThreads), 0, (cudaStream_t)stream, *a));
    if (rc != RVQ_OK) return rc;
    // apart: blocks of 4 loads a thread; in place: the five columns
    const int vecs = record_bytes(c.head_dim) / 16;
    const int64_t chunks = ((int64_t)a->keep * vecs + kMoveThreads * kMoveLoads - 1) / (kMoveThreads * kMoveLoads);
    const unsigned parts = o.data == c.data ? 5 : (unsigned)(chunks < 256 ? chunks : 256);
    auto* move = c.head_dim == 128 ? evict_move_kernel<10> : evict_move_kernel<5>;
    return status(launch_pdl(move, dim3((unsigned)heads, parts), dim3(kMoveThreads), 0, (cudaStream_t)stream, *a));
}
