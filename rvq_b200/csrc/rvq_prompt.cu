// Attention of whole prompts (rvq_prompt_attention, include/rvq_b200.h).

#include <cuda.h>
#include <cudaTypedefs.h>
#include <string.h>

#include <mutex>

#include "rvq_common.cuh"
#include "rvq_sm100.cuh"

namespace rvq {
namespace prompt {

using namespace sm100;

__device__ int g_attention_timeout;          // sticky: a bounded wait gave up

// ---------------------------------------------------------------------------
// A CTA takes 2 tiles of 128 operand rows of one kv head and walks the keys in
// tiles of 128.  A row is (token, query head of the kv head): a tile holds
// 128 / rep tokens with all their rep heads, so grouped heads share every K and
// V tile and short sequences fill the rows.  Roles by warp: 0-7 and 8-15 the
// softmax of the two tiles (two threads a row, 64 columns each), 16 the TMA
// loads, 17 (one thread) the MMAs.
//
//   S = Q K^T       tcgen05.mma, both operands in shared memory, S in TMEM
//   P = 2^(c S - m) fp32; rounded to the operand type and written over S in TMEM
//   O += P V        tcgen05.mma, P from TMEM, V as it lies in shared memory
//
// While one tile's softmax runs, the tensor cores work for the other one.  A CTA
// takes such pairs of tiles one after the other (by a ticket from the second on,
// the longest of a causal sequence first); the next one's loads and its first S
// run beside this one's last softmax and output.
//
// The maximum that is subtracted only follows the true one when that has grown by
// 2^8: O is then rescaled by the row's own threads, which is rare after the first
// tiles; p stays below 2^8, and its rounding to the operand type, half a step
// relative, is the same at any size (the sums take p unrounded).
// Keys that a tile brings along but a row does not see (behind the sequence, later
// than the query) get p = 0; values behind the sequence are zeroed in shared
// memory, and a row that came out non-finite is looked at again (repair), so
// that no hidden NaN or infinity reaches it through 0 * NaN.
//
// Bound by the chain S -> softmax -> P -> PV -> S of a tile: of 3,570 clocks a step of
// both tiles the tensor cores work 2,048 (timestamps of one CTA: softmax 1,880, of
// which the exponentials 1,300; PV and S 1,030; waits 300); no unit is full (4,096 tokens:
// tensor pipe 52 %, exponentials 52 %, issue 42 %).  8,192 tokens, 32/8 heads of 128,
// short runs: causal 462 us, 1,190 TFLOP/s (71 % of the measured matrix peak), not causal
// 877 us, 1,254; back to back until the power cap holds the clock 513 and 978 us.  Tried:
// a thread a row with its 128 columns (1,094 not causal, before the MMA warp became one
// thread); a quarter or half of the
// exponentials as a polynomial on the FMA pipe (no faster: registers spill).
// ---------------------------------------------------------------------------
constexpr int kRows = 128;                   // operand rows of a tile (MMA M)
constexpr int kKeys = 128;                   // keys of a tile
constexpr int kMaxSplits = 64;               // parts of the keys
constexpr int kSoftmaxWarps = 16;            // 8 a tile
constexpr int kThreads = 32 * (kSoftmaxWarps + 2);
constexpr int kHalf = kRows * 128;           // bytes of 64 columns of a tile
constexpr int kWaitPolls = 1 << 22;
constexpr float kGrow = 8.f;                 // the maximum may be passed by 2^kGrow

struct Params {
    CUtensorMap q, k, v;
    rvq_prompt_attn_args a;
    int32_t rep;
    int32_t tile_tokens;                     // 128 / rep
    int32_t pairs;                           // upper bound of the pairs of tiles of all sequences
    int32_t splits;                          // parts of the keys, each with CTAs of its own
    int32_t sms;
    int32_t wide;                            // 32 bytes of an output row (of a part's, where there are parts) start at 32-byte steps
    int32_t units;                           // pairs x kv heads x parts: what the CTAs take one after the other
    uint32_t* tickets;                       // units beyond the first one of every CTA given out, CTAs done; NULL: there are none
    float* part_o;                           // splits > 1: [splits][tokens][n_heads][head_dim], not yet divided by the sum
    float2* part_ml;                         // [splits][tokens][n_heads]: maximum (times c) and sum
};

// A CTA's part of the call.
struct Work {
    int64_t q0, k0;                          // first query and key of the sequence
    int32_t lq, lk;                          // their number
    int32_t tok0;                            // first token of tile 0 in the sequence
    int32_t j0;                              // first tile of keys
    int32_t n[2];                            // tiles of keys that the two tiles of queries take from there on (0, 0: nothing to do)
    int32_t live;                            // 1; 0: the pair is in no sequence; -1: no unit is left
    int32_t kv, split;
    int32_t clean;                           // the last tile of keys reaches into another sequence
};

template <int HD>
struct Smem {
    static constexpr int kTileBytes = HD / 64 * kHalf;
    uint8_t q[2][kTileBytes];
    uint8_t k[2][kTileBytes];
    uint8_t v[2][kTileBytes];
    uint64_t q_full, drain, v_clean, s_full[2], p_full[2], o_full[2];
    uint64_t first_full, first_empty;        // K of a unit's tile 0
    uint64_t kv_full[2], kv_empty[2];        // steps, counted over all units: V of tile j and K of tile j + 1
    uint64_t work_full[2], work_empty[2];
    float top[2][2][kRows];                  // a row's maximum (at the end: sum) over either half of the columns
    Work work[2];
    int32_t fail[8];                         // of two warps of the same rows one has given up
    uint32_t tmem;
    int32_t dead;                            // a bounded wait gave up
    int32_t busy;                            // warps that do what may take long
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];\n" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}

// N-major operand (rows of 64 N-elements, one row per k) with 128-byte swizzle:
// 8-row atoms of 1024 bytes along k (stride offset), `next` bytes from one block
// of 64 columns to the next (leading offset).
__device__ __forceinline__ uint64_t sw128_desc_mn(uint32_t saddr, uint32_t next) {
    return (sw128_desc(saddr) & ~(0x3fffull << 16)) | (uint64_t)(next >> 4) << 16;
}

__device__ __forceinline__ void store16x2(void* to, const uint32_t (&y)[8]) {
    uint4* t = reinterpret_cast<uint4*>(to);
    t[0] = make_uint4(y[0], y[1], y[2], y[3]);
    t[1] = make_uint4(y[4], y[5], y[6], y[7]);
}

// A whole sector by one thread.  Rows lie apart, so a warp's store is 32 lines' work whatever its width, and half a sector at
// a time is a good part of a unit's end: 64 tokens 10.7 us with halves, 9.4 so; 2,048 tokens 47.1 and 45.0, 12 packed prompts 237
// and 221, 77 queries after 9,000 keys 34.8 and 32.5.
__device__ __forceinline__ void store32(void* to, const uint32_t (&y)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(to), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]),
                 "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7])
                 : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 8 consecutive 32-bit columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}

// Bounded wait of a thread; once one wait of the CTA has given up, the others end at once.  The bound does not count while a warp
// sums rows again (repair) or walks over empty sequences (find_work), which wait for nothing but may take long.
template <int HD>
__device__ __forceinline__ bool wait1(Smem<HD>& S, uint32_t bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    for (int i = 0; i < kWaitPolls; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63) == 63) {
            if (*(volatile int32_t*)&S.dead) return false;
            if (*(volatile int32_t*)&S.busy) i = 0;
        }
    }
    atomicExch(&g_attention_timeout, 1);
    *(volatile int32_t*)&S.dead = 1;
    return false;
}

// The same of a whole warp.
template <int HD>
__device__ __forceinline__ bool wait(Smem<HD>& S, uint64_t& bar, uint32_t parity) {
    const bool ok = wait1(S, smem_addr(&bar), parity);
    return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// x b + c and y b + c in one instruction, each rounded as by itself
__device__ __forceinline__ void fma2(float& x, float& y, float b, float c) {
    asm("{\n .reg .b64 X, B, C;\n mov.b64 X, {%0, %1};\n mov.b64 B, {%2, %2};\n mov.b64 C, {%3, %3};\n"
        " fma.rn.f32x2 X, X, B, C;\n mov.b64 {%0, %1}, X;\n}\n"
        : "+f"(x), "+f"(y)
        : "f"(b), "f"(c));
}

// Half of a row's scores of a tile (64 columns of a thread's TMEM lane): its columns from `seen` on are hidden.
template <bool kMasked>
__device__ __forceinline__ float row_max(float (&s)[2][32], int seen) {
    if constexpr (kMasked) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 32; ++e)
                if (32 * x + e >= seen) s[x][e] = -INFINITY;
    }
    float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < 32; e += 4)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            t[2 * x] = max3(t[2 * x], s[x][e], s[x][e + 1]);
            t[2 * x + 1] = max3(t[2 * x + 1], s[x][e + 2], s[x][e + 3]);
        }
    return fmaxf(max3(t[0], t[1], t[2]), t[3]);
}

// p = 2^(c s - sub) in the operand type, over scores in TMEM at ts; returns their sum.
template <bool kMasked, bool kHalfType>
__device__ __forceinline__ float row_exp(float (&s)[2][32], int seen, float c, float sub, uint32_t ts) {
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        uint4 q[4];
        uint32_t* w = reinterpret_cast<uint32_t*>(q);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
            float& p0 = s[x][e];
            float& p1 = s[x][e + 1];
            fma2(p0, p1, c, -sub);
            p0 = exp2_approx(p0);
            p1 = exp2_approx(p1);
            if constexpr (kMasked) {                         // c may be 0
                if (32 * x + e >= seen) p0 = 0.f;
                if (32 * x + e + 1 >= seen) p1 = 0.f;
            }
            part[2 * x] += p0;
            part[2 * x + 1] += p1;
            w[e / 2] = pack2(p0, p1, kHalfType ? RVQ_F16 : RVQ_BF16);
        }
        tmem_st16(ts + 16 * x, q);
    }
    return (part[0] + part[1]) + (part[2] + part[3]);
}

// Where find_work left off: sequences done with (from the last one on), and their pairs.
struct Cursor {
    int32_t base;
    int64_t before;
};

// Pair number `want` and part `split` of its keys, by one warp.  Pairs are counted from the last one of the last sequence
// down; a CTA's numbers only rise, so over all its units it goes over the sequences once.  *busy counts while that goes on.
__device__ __forceinline__ Work find_work(const Params& p, int32_t* busy, int want, int split, Cursor& at) {
    const rvq_prompt_attn_args& a = p.a;
    const int lane = threadIdx.x & 31, T = p.tile_tokens;
    const int32_t* cu_k = a.cu_k != nullptr ? a.cu_k : a.cu_q;
    Work w = {};
    bool far = false;
    for (; at.base < a.n_seq; at.base += 32) {
        const int b = a.n_seq - 1 - at.base - lane;
        int64_t q0 = 0, q1 = 0, k0 = 0, k1 = 0;
        if (b >= 0) {
            q1 = a.tokens, k1 = a.keys;
            if (a.cu_q != nullptr) {
                q0 = max(0, __ldg(a.cu_q + b)), q1 = min(q1, (int64_t)__ldg(a.cu_q + b + 1));
                k0 = max(0, __ldg(cu_k + b)), k1 = min(k1, (int64_t)__ldg(cu_k + b + 1));
            }
        }
        const int64_t mine = q1 > q0 ? (q1 - q0 + 2 * T - 1) / (2 * T) : 0, before = at.before;
        int64_t upto = mine;                                 // inclusive prefix sum over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const int64_t total = __shfl_sync(0xffffffffu, upto, 31);
        if (want >= before + total) {
            at.before += total;
            if (!far && lane == 0) atomicAdd(busy, 1);       // a walk over many empty sequences may take long
            far = true;
            continue;
        }
        const int l = __ffs(__ballot_sync(0xffffffffu, want < before + upto)) - 1;
        if (far && lane == 0) atomicSub(busy, 1);
        w.live = 1;
        w.q0 = __shfl_sync(0xffffffffu, q0, l);
        w.k0 = __shfl_sync(0xffffffffu, k0, l);
        w.lq = (int)(__shfl_sync(0xffffffffu, q1, l) - w.q0);
        w.lk = (int)max((int64_t)0, __shfl_sync(0xffffffffu, k1, l) - w.k0);
        w.tok0 = (int)(before + __shfl_sync(0xffffffffu, upto, l) - 1 - want) * 2 * T;
#pragma unroll
        for (int i = 0; i < 2; ++i) {                        // what tile i's last token sees
            const int last = min(w.lq, w.tok0 + (i + 1) * T) - 1;
            const int see = last < w.tok0 + i * T ? 0 : a.causal ? min(w.lk, max(0, last + 1 + w.lk - w.lq)) : w.lk;
            w.n[i] = (see + kKeys - 1) / kKeys;
        }
        const int64_t most = max(w.n[0], w.n[1]);
        w.j0 = (int)(most * split / p.splits);
        const int j1 = (int)(most * (split + 1) / p.splits);
#pragma unroll
        for (int i = 0; i < 2; ++i) w.n[i] = max(0, min(w.n[i], j1) - w.j0);
        const int total_tiles = max(w.n[0], w.n[1]);
        w.clean = w.lk % kKeys != 0 && total_tiles > 0 && (w.j0 + total_tiles) * kKeys > w.lk && w.k0 + w.lk < a.keys;
        return w;
    }
    if (far && lane == 0) atomicSub(busy, 1);
    return w;
}

// Element i of a pair of 16-bit numbers.
template <bool kHalfType>
__device__ __forceinline__ float half_at(uint32_t w, int i) {
    if constexpr (kHalfType) return __half2float(__ushort_as_half((uint16_t)(w >> (16 * i))));
    else return __uint_as_float(i ? w & 0xffff0000u : w << 16);
}

// A warp's half of the columns of an output row of a query whose hidden values (keys [n, hidden_end) of the last tiles) may have
// leaked in: where one of them is not finite and no seen value in the last tile is NaN, the column is summed again over the keys
// [begin, n) that the query sees; into out (times inv), or into part.  A NaN stays: once all such columns are, that is it.  Takes
// 8 keys at a time, HD / 8 lanes a key for the scores: 16 take registers from the kernel around it (12 packed prompts 215 -> 218
// us).  Slow, and that is for rows beside values that are not finite only: 2,048 causal tokens of 32/8 heads of 128 whose last
// value is NaN throughout, 39 ms; 16,384 tokens 340 ms.
template <int HD, bool kHalfType>
__device__ __forceinline__ void repair(const rvq_prompt_attn_args& a, int64_t tok, int h, int64_t k0, int64_t begin, int64_t n,
                                    int64_t hidden_end, float c, float m, float inv, float* part) {
    constexpr int J = HD / 64, L = HD / 8, P = 32 / L, U = 8 / P;
    const int lane = threadIdx.x & 31, g = h / (a.n_heads / a.n_kv), hd = a.head_dim;
    const int d0 = (threadIdx.x >> 7 & 1) * (HD / 2) + lane;             // this lane's columns: d0, d0 + 32
    const int64_t v0 = k0 * a.v_stride[0] + g * a.v_stride[1] + d0;
    bool leak[J];
    bool any = false;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        leak[j] = false;
        if (d0 + 32 * j >= hd) continue;
        for (int64_t i = n; i < hidden_end; ++i) {
            const float v = load_as_f32(a.v, v0 + i * a.v_stride[0] + 32 * j, a.kind);
            leak[j] |= !(fabsf(v) <= 3.4e38f);
        }
        for (int64_t i = max(begin, hidden_end - kKeys); leak[j] && i < n; ++i) {
            const float v = load_as_f32(a.v, v0 + i * a.v_stride[0] + 32 * j, a.kind);
            leak[j] = v == v;
        }
        any |= leak[j];
    }
    if (!__any_sync(0xffffffffu, any)) return;
    const int chunk = lane % L * 8;                                      // 8 values of q and of a key
    const bool live = chunk < hd;
    const uint16_t* k = reinterpret_cast<const uint16_t*>(a.k) + k0 * a.k_stride[0] + g * a.k_stride[1] + (live ? chunk : 0);
    const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + tok * a.q_stride[0] + h * a.q_stride[1] + (live ? chunk : 0);
    const uint4 qw = *reinterpret_cast<const uint4*>(qp);
    float acc[J];
#pragma unroll
    for (int j = 0; j < J; ++j) acc[j] = 0.f;
    for (int64_t base = begin; base < n; base += U * P) {
        float p[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint4 kw = *reinterpret_cast<const uint4*>(k + min(base + u * P + lane / L, n - 1) * a.k_stride[0]);
            const uint32_t kk[4] = {kw.x, kw.y, kw.z, kw.w}, qq[4] = {qw.x, qw.y, qw.z, qw.w};
            float x = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) x = fmaf(half_at<kHalfType>(qq[e / 2], e & 1), half_at<kHalfType>(kk[e / 2], e & 1), x);
            p[u] = live ? x : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) p[u] += __shfl_xor_sync(0xffffffffu, p[u], o);
            p[u] = exp2_approx(fmaf(p[u], c, -m));
        }
#pragma unroll
        for (int l = 0; l < U * P; ++l) {
            const float w = __shfl_sync(0xffffffffu, p[l / P], l % P * L);
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (leak[j] && base + l < n)
                    acc[j] = fmaf(w, load_as_f32(a.v, v0 + (base + l) * a.v_stride[0] + 32 * j, a.kind), acc[j]);
        }
        bool open = false;
#pragma unroll
        for (int j = 0; j < J; ++j) open |= leak[j] && acc[j] == acc[j];
        if (!__any_sync(0xffffffffu, open)) break;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int d = d0 + 32 * j;
        if (leak[j] && part != nullptr) part[d] = acc[j];
        else if (leak[j]) store_from_f32(a.out, tok * a.out_stride[0] + h * a.out_stride[1] + d, a.kind, acc[j] * inv);
    }
}

// The rows of the lanes in `again`, one after the other; tok, seen_end, m and inv: of the lane's row, head: of its kv head's.
template <int HD, bool kHalfType>
__device__ __noinline__ void repair_rows(const Params& p, Smem<HD>& S, const Work& w, uint32_t again, int head, int tok, int seen_end,
                                         float m, float inv) {
    const rvq_prompt_attn_args& a = p.a;
    const int lane = threadIdx.x & 31, i = threadIdx.x >> 8;             // tile of queries
    const float c = a.scaling * 1.4426950408889634f;
    const int begin = w.j0 * kKeys, hidden_end = min(w.lk, (w.j0 + w.n[i]) * kKeys);
    if (lane == 0) atomicAdd(&S.busy, 1);
    while (again) {
        const int l = __ffs(again) - 1;
        again &= again - 1;
        __syncwarp();
        const int64_t row = w.q0 + __shfl_sync(0xffffffffu, tok, l);
        const int h = w.kv * p.rep + __shfl_sync(0xffffffffu, head, l);
        repair<HD, kHalfType>(a, row, h, w.k0, begin, __shfl_sync(0xffffffffu, seen_end, l), hidden_end, c,
                              __shfl_sync(0xffffffffu, m, l), __shfl_sync(0xffffffffu, inv, l),
                              p.splits == 1 ? nullptr : p.part_o + (((int64_t)w.split * a.tokens + row) * a.n_heads + h) * a.head_dim);
    }
    if (lane == 0) atomicSub(&S.busy, 1);
}

template <int HD, bool kHalfType>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const __grid_constant__ Params p) {
    extern __shared__ uint8_t smem_raw[];
    Smem<HD>& S = *reinterpret_cast<Smem<HD>*>(smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023));
    const rvq_prompt_attn_args& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int T = p.tile_tokens;
    pdl_launch_dependents();
    if (warp == kSoftmaxWarps && lane == 0) {
        mbar_init(smem_addr(&S.q_full), 1);
        mbar_init(smem_addr(&S.v_clean), 1);
        mbar_init(smem_addr(&S.drain), 1);
        mbar_init(smem_addr(&S.first_full), 1);
        mbar_init(smem_addr(&S.first_empty), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_addr(&S.kv_full[i]), 1);
            mbar_init(smem_addr(&S.kv_empty[i]), 1);
            mbar_init(smem_addr(&S.s_full[i]), 1);
            mbar_init(smem_addr(&S.p_full[i]), kSoftmaxWarps / 2);
            mbar_init(smem_addr(&S.o_full[i]), 1);
            mbar_init(smem_addr(&S.work_full[i]), 1);
            mbar_init(smem_addr(&S.work_empty[i]), kSoftmaxWarps + 1);
        }
        S.dead = S.busy = 0;
        for (int i = 0; i < 8; ++i) S.fail[i] = 0;
        mbar_init_fence();
        fence_async_shared();
    }
    if (warp == kSoftmaxWarps + 1) tmem_alloc(smem_addr(&S.tmem), 512);
    // Work of a unit, by the loading warp, and its loads that need no other buffers than free ones
    Cursor cursor = {};
    auto find = [&](int unit) {
        Work w = {};
        w.live = -1;
        if (unit < p.units) {
            const int split = unit % p.splits, rest = unit / p.splits;
            // the last pairs of a causal sequence see the most keys: they start first
            w = find_work(p, &S.busy, rest / a.n_kv, split, cursor);
            w.kv = rest % a.n_kv, w.split = split;
        }
        return w;
    };
    auto load = [&](const CUtensorMap& map, int head, uint8_t* dst, int64_t row, uint64_t& bar) {     // 128 keys, or a tile's tokens
        for (int h = 0; h < HD / 64; ++h)
            tma_load_3d(smem_addr(dst + h * kHalf), &map, 64 * h, head, (int)row, smem_addr(&bar));
    };
    auto load_step = [&](const Work& w, int step, int j, int total) {      // V of tile j and K of tile j + 1
        uint64_t& bar = S.kv_full[step & 1];
        mbar_expect_tx(smem_addr(&bar), (j + 1 < total ? 2 : 1) * Smem<HD>::kTileBytes);
        load(p.v, w.kv, S.v[step & 1], w.k0 + (int64_t)(w.j0 + j) * kKeys, bar);
        if (j + 1 < total) load(p.k, w.kv, S.k[(step + 1) & 1], w.k0 + (int64_t)(w.j0 + j + 1) * kKeys, bar);
    };
    auto load_first = [&](const Work& w, int step, int total) {
        const int tiles = w.tok0 + T < w.lq ? 2 : 1;
        mbar_expect_tx(smem_addr(&S.q_full), tiles * (HD / 64) * (uint32_t)(T * p.rep * 128));
        for (int i = 0; i < tiles; ++i) load(p.q, w.kv * p.rep, S.q[i], w.q0 + w.tok0 + i * T, S.q_full);
        mbar_expect_tx(smem_addr(&S.first_full), Smem<HD>::kTileBytes);
        load(p.k, w.kv, S.k[step & 1], w.k0 + (int64_t)w.j0 * kKeys, S.first_full);
        load_step(w, step, 0, total);
    };
    pdl_wait();
    Work first = {};
    if (warp == kSoftmaxWarps) {                             // the first unit's loads, while the other warps get ready
        __syncwarp();
        first = find(blockIdx.x);
        const int total = max(first.n[0], first.n[1]);
        if (lane == 0) {
            S.work[0] = first;
            mbar_arrive(smem_addr(&S.work_full[0]));
            if (total > 0) load_first(first, 0, total);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = S.tmem;
    if (warp == kSoftmaxWarps) {
        int steps = 0, loaded = 0, used = 0;                 // steps of the units before, steps loaded, units with tiles
        int cleaned = -1;                                    // the last step whose values were cleaned
        Work w = first;
        bool ok = true;
        for (int it = 0; ok; ++it) {
            const int slot = it & 1;
            if (it >= 2) ok = wait(S, S.work_empty[slot], (it / 2 - 1) & 1);
            if (!ok) break;
            if (it > 0 && lane == 0) {
                S.work[slot] = w;
                mbar_arrive(smem_addr(&S.work_full[slot]));
            }
            if (w.live < 0) break;
            const int total = max(w.n[0], w.n[1]);
            int next = p.units;
            if (total > 0) {
                if (it > 0) {
                    // Q and the K buffers are free with the last S of the unit before: with its last step but one, or with its first
                    // S where it has one tile; the V buffer with the step before the last
                    if (steps >= 2) ok = wait(S, S.kv_empty[steps & 1], (steps / 2 - 1) & 1);
                    if (ok && used > 0) ok = wait(S, S.first_empty, (used - 1) & 1);
                    if (!ok) break;
                    if (lane == 0) load_first(w, steps, total);
                }
                loaded = steps + 1;
                for (int j = 1; j < total && ok; ++j) {
                    const int step = steps + j;
                    if (step >= 2) ok = wait(S, S.kv_empty[step & 1], (step / 2 - 1) & 1);
                    if (ok && j == 1) ok = wait(S, S.first_empty, used & 1);           // K of tile 2 replaces that of tile 0
                    if (!ok) break;
                    if (lane == 0) load_step(w, step, j, total);
                    loaded = step + 1;
                }
                steps += total;
                ++used;
            }
            // the next unit only now that this one is loaded: who has long units takes fewer of them
            if (ok && lane == 0 && p.tickets != nullptr) next = (int)(gridDim.x + atomicAdd(p.tickets, 1u));
            if (total > 0) {
                if (ok && w.clean) {
                    const int last = steps - 1;
                    // one clean tile at a time: the one before may be this one's neighbour, not yet used
                    if (cleaned >= 0 && last < cleaned + 2) ok = wait(S, S.kv_empty[cleaned & 1], (cleaned / 2) & 1);
                    if (ok) ok = wait(S, S.kv_full[last & 1], (last / 2) & 1);
                    if (!ok) break;
                    cleaned = last;
                    const int r0 = w.lk - (w.j0 + total - 1) * kKeys;        // rows r0 .. 127 belong to others (a swizzled row stays a row)
                    for (int h = 0; h < HD / 64; ++h)
                        for (int i = r0 * 8 + lane; i < kRows * 8; i += 32)
                            reinterpret_cast<uint4*>(S.v[last & 1] + h * kHalf)[i] = make_uint4(0, 0, 0, 0);
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_addr(&S.v_clean));
                }
            }
            if (ok) w = find(__shfl_sync(0xffffffffu, next, 0));
        }
        if (lane == 0 && p.tickets != nullptr) {             // the last CTA leaves the tickets as they were
            __threadfence();
            if (atomicAdd(p.tickets + 1, 1u) == gridDim.x - 1) p.tickets[0] = p.tickets[1] = 0;
        }
        if (!ok) {                                           // copies in flight end before this CTA's shared memory is given up
            for (int j = max(0, loaded - 2); j < loaded; ++j)
                mbar_wait(smem_addr(&S.kv_full[j & 1]), (j / 2) & 1, kWaitPolls, &g_attention_timeout);
            if (loaded > 0) {
                const int u = (used > 0 && loaded == steps ? used - 1 : used) & 1;
                mbar_wait(smem_addr(&S.first_full), u, kWaitPolls, &g_attention_timeout);
                mbar_wait(smem_addr(&S.q_full), u, kWaitPolls, &g_attention_timeout);
            }
        }
    } else if (warp == kSoftmaxWarps + 1) {
        // One thread from here to the end: what it does between two products, the tensor cores wait for.
        constexpr uint32_t kTypes = kHalfType ? 0u : (1u << 7) | (1u << 10);
        constexpr uint32_t kS = (1u << 4) | kTypes | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
        constexpr uint32_t kO = (1u << 4) | kTypes | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
        if (lane == 0) {
            // c is |scaling|: a negative one negates Q on its way (so that the largest score stays the largest)
            const uint32_t types_s = kS | (a.scaling < 0.f ? 1u << 13 : 0u);
            const uint64_t dq = sw128_desc(smem_addr(S.q[0])), dk = sw128_desc(smem_addr(S.k[0]));
            const uint64_t dv = sw128_desc_mn(smem_addr(S.v[0]), kHalf);
            constexpr uint32_t kTile = Smem<HD>::kTileBytes >> 4;          // descriptors count 16 bytes
            auto scores = [&](int i, int at) {               // S_i = Q_i K^T, K in buffer `at`
                const uint64_t q = dq + i * kTile, k = dk + at * kTile;
#pragma unroll
                for (int x = 0; x < HD / 16; ++x)
                    mma_bf16(tmem + i * kKeys, q + (x / 4) * (kHalf >> 4) + (x % 4) * 2, k + (x / 4) * (kHalf >> 4) + (x % 4) * 2,
                             types_s, x > 0);
                mma_commit(smem_addr(&S.s_full[i]));
            };
            int steps = 0, used = 0, cleaned = 0;
            uint32_t pp = 0;                                 // parities of the tiles' next P
            bool ok = true;
            for (int it = 0; ok; ++it) {
                ok = wait1(S, smem_addr(&S.work_full[it & 1]), (it / 2) & 1);
                if (!ok) break;
                const Work& w = S.work[it & 1];
                if (w.live < 0) break;
                const int n[2] = {w.n[0], w.n[1]}, total = max(n[0], n[1]);
                const bool clean = w.clean;
                if (total > 0) {
                    ok = wait1(S, smem_addr(&S.q_full), used & 1) && wait1(S, smem_addr(&S.first_full), used & 1);
                    if (ok) {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if (n[i] > 0) scores(i, steps & 1);
                        mma_commit(smem_addr(&S.first_empty));
                    }
                    for (int j = 0; ok && j < total; ++j, ++steps) {
                        ok = wait1(S, smem_addr(&S.kv_full[steps & 1]), (steps / 2) & 1);
                        if (ok && clean && j == total - 1) ok = wait1(S, smem_addr(&S.v_clean), cleaned++ & 1);
                        const uint64_t v = dv + (steps & 1) * kTile;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            if (!ok || j >= n[i]) continue;
                            ok = wait1(S, smem_addr(&S.p_full[i]), pp >> i & 1);
                            if (!ok) continue;
                            pp ^= 1u << i;
                            tc_fence_after();
#pragma unroll
                            for (int k = 0; k < kKeys / 16; ++k)
                                mma_bf16_ts(tmem + 2 * kKeys + i * HD, tmem + i * kKeys + 8 * k, v + k * (2048 >> 4), kO, j > 0 || k > 0);
                            if (j + 1 < n[i]) scores(i, (steps + 1) & 1);
                            else mma_commit(smem_addr(&S.o_full[i]));
                        }
                        if (ok) mma_commit(smem_addr(&S.kv_empty[steps & 1]));
                    }
                    ++used;
                }
                if (ok) mbar_arrive(smem_addr(&S.work_empty[it & 1]));
            }
            if (!ok) {                                       // products in flight end before TMEM is given up
                mma_commit(smem_addr(&S.drain));
                mbar_wait(smem_addr(&S.drain), 0, kWaitPolls, &g_attention_timeout);
            }
        }
        __syncwarp();
    } else {
        // two threads a row, 64 columns of S and half of O's each
        const int i = warp >> 3, half = warp >> 2 & 1, row = tid & 127;
        const int pair_bar = 1 + i * 4 + (warp & 3);         // named barrier of the two warps of these rows
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + i * kKeys, to = tmem + lanes + 2 * kKeys + i * HD + half * (HD / 2);
        const float c = fabsf(a.scaling) * 1.4426950408889634f;
        // fp16 has few small numbers: p up to 2^15 instead of 2^kGrow, and so 2^-32 of the row's largest one instead of 2^-25
        // for the rounding of the smallest
        constexpr float kShift = kHalfType ? 15.f - kGrow : 0.f;
        const int in = row / p.rep, head = row - in * p.rep;
        uint32_t sp = 0, op = 0;                             // parities of the next S and O
        bool ok = true;
        for (int it = 0;; ++it) {
            ok = ok && wait(S, S.work_full[it & 1], (it / 2) & 1);
            if (!ok && lane == 0) *(volatile int32_t*)&S.fail[pair_bar - 1] = 1;
            named_sync(pair_bar, 64);                        // both warps go on, or neither
            if (*(volatile int32_t*)&S.fail[pair_bar - 1]) break;
            const Work& w = S.work[it & 1];
            if (w.live < 0) break;
            const int n = w.n[i], j0 = w.j0;
            int limit;                                       // keys that the row sees
            {
                const int tok = w.tok0 + i * T + in;         // in the sequence
                limit = !w.live || in >= T || tok >= w.lq ? 0 : a.causal ? min(w.lk, max(0, tok + 1 + w.lk - w.lq)) : w.lk;
            }
            float m = -INFINITY, sum = 0.f;                  // m: of the scores times c
            for (int j = 0; j < n; ++j, sp ^= 1) {
                ok = ok && wait(S, S.s_full[i], sp);
                if (!ok) {                                   // the partner may still come to its barriers
                    named_sync(pair_bar, 64);
                    continue;
                }
                tc_fence_after();
                uint32_t r[2][32];
                tmem_ld32(ts + half * 64, r[0]);
                tmem_ld32(ts + half * 64 + 32, r[1]);
                tmem_ld_wait();
                float (&s)[2][32] = reinterpret_cast<float (&)[2][32]>(r);
                const int seen = limit - (j0 + j) * kKeys - half * 64;             // of this half's columns the row sees these
                const bool masked = __any_sync(0xffffffffu, seen < kKeys / 2);
                float raw = masked ? row_max<true>(s, seen) : row_max<false>(s, seen);
                // both halves are in registers when the barrier opens: P may overwrite either
                S.top[i][half][row] = raw;
                tc_fence_before();
                named_sync(pair_bar, 64);
                tc_fence_after();
                raw = fmaxf(raw, S.top[i][half ^ 1][row]);
                const float top = raw == -INFINITY ? -INFINITY : raw * c;
                const bool grow = j == 0 ? top > m : top > m + kGrow;
                if (j == 0) {
                    m = top;
                } else if (__any_sync(0xffffffffu, grow)) {
                    // S is full: the products before it, which summed into O, are complete
                    const float f = grow ? exp2_approx(m - top) : 1.f;
                    if (grow) m = top;
                    sum *= f;
#pragma unroll 1
                    for (int x = 0; x < HD / 16; ++x) {      // few columns at a time: the scores stay in registers
                        uint32_t o[8];
                        tmem_ld8(to + 8 * x, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st8(to + 8 * x, make_uint4(o[0], o[1], o[2], o[3]), make_uint4(o[4], o[5], o[6], o[7]));
                    }
                    tmem_st_wait();
                }
                const float sub = (m == -INFINITY ? 0.f : m) - kShift;
                sum += masked ? row_exp<true, kHalfType>(s, seen, c, sub, ts + half * 32) : row_exp<false, kHalfType>(s, seen, c, sub, ts + half * 32);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&S.p_full[i]));
            }
            if (ok && n > 0) ok = wait(S, S.o_full[i], op);
            op ^= n > 0;
            // read from shared memory again: kept over the steps, they cost the inner loop registers (16,384 tokens 2,061 -> 2,038 us)
            const volatile Work& u = S.work[it & 1];
            const int64_t q0 = u.q0;
            const int h = u.kv * p.rep + head, split = u.split, lk = u.lk, tok = u.tok0 + i * T + in;
            const bool valid = u.live && in < T && tok < u.lq;
            tc_fence_after();
            named_sync(pair_bar, 64);                        // the partner has read this half's last maximum
            S.top[i][half][row] = sum;
            named_sync(pair_bar, 64);
            sum = S.top[i][0][row] + S.top[i][1][row];
            m -= kShift;                                     // p and its sum are relative to that
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const bool whole = p.splits == 1, none = limit == 0 || (whole && inv == 0.f);
            const int64_t at = (q0 + tok) * a.out_stride[0] + h * a.out_stride[1];
            uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + at + half * (HD / 2);
            const int64_t slot = ((int64_t)split * a.tokens + q0 + tok) * a.n_heads + h;
            float* part = whole ? nullptr : p.part_o + slot * a.head_dim;
            bool bad = false;
#pragma unroll 1
            for (int x = 0; x < HD / 32; ++x) {              // 16 columns
                uint32_t o[16];
                if (ok && n > 0) {
                    tmem_ld8(to + 16 * x, *reinterpret_cast<uint32_t (*)[8]>(o));
                    tmem_ld8(to + 16 * x + 8, *reinterpret_cast<uint32_t (*)[8]>(o + 8));
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = 0;
                }
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    v[e] = __uint_as_float(o[e]);
                    bad |= !(fabsf(v[e]) <= 3.4e38f);
                    v[e] = none ? 0.f : whole ? v[e] * inv : v[e];
                }
                const int d = half * (HD / 2) + 16 * x;
                if (valid && whole) {
                    constexpr int kOut = kHalfType ? RVQ_F16 : RVQ_BF16;
                    uint32_t y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = pack2(v[2 * e], v[2 * e + 1], kOut);
                    if (p.wide) {
                        if (d < a.head_dim) store32(out + 16 * x, y);
                    } else {
                        if (d < a.head_dim) *reinterpret_cast<uint4*>(out + 16 * x) = make_uint4(y[0], y[1], y[2], y[3]);
                        if (d + 8 < a.head_dim) *reinterpret_cast<uint4*>(out + 16 * x + 8) = make_uint4(y[4], y[5], y[6], y[7]);
                    }
                } else if (valid) {
#pragma unroll
                    for (int e = 0; e < 16; e += 8) {
                        uint32_t y[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) y[i] = __float_as_uint(v[e + i]);
                        if (d + e < a.head_dim) {
                            if (p.wide) store32(part + d + e, y);
                            else store16x2(part + d + e, y);
                        }
                    }
                }
            }
            if (valid && half == 0 && whole && a.lse != nullptr)
                a.lse[(int64_t)h * a.tokens + q0 + tok] = none ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
            if (valid && half == 0 && !whole) p.part_ml[slot] = make_float2(m, limit == 0 ? 0.f : sum);
            // values between this row's last key and the end of its last tile may have leaked in (a row without weights has zeros,
            // one whose sum is infinite or NaN is not finite by itself)
            const int begin = j0 * kKeys, hidden_end = min(lk, (j0 + n) * kKeys), seen_end = min(limit, hidden_end);
            const uint32_t again = __ballot_sync(0xffffffffu, ok && valid && bad && seen_end > begin && seen_end < hidden_end && inv > 0.f);
            if (again) repair_rows<HD, kHalfType>(p, S, w, again, head, tok, seen_end, m, inv);
            tc_fence_before();                               // O is read: the next unit's products may come
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(smem_addr(&S.work_empty[it & 1]));
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kSoftmaxWarps + 1) tmem_dealloc(tmem, 512);
}

// The parts of every row joined, in order: a warp a (token, head).  Rows in no sequence have none.
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Params p) {
    const rvq_prompt_attn_args& a = p.a;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (unit >= a.tokens * a.n_heads) return;
    const int64_t tok = unit / a.n_heads;
    const int h = (int)(unit - tok * a.n_heads);
    if (a.cu_q != nullptr) {
        int lo = 0, hi = a.n_seq;                            // the last sequence that starts at or before tok
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (__ldg(a.cu_q + mid) <= tok) lo = mid;
            else hi = mid;
        }
        if (tok < __ldg(a.cu_q + lo) || tok >= __ldg(a.cu_q + lo + 1)) return;
    }
    // maxima and sums: a part a lane, then the outputs with their factors
    const int64_t step = a.tokens * a.n_heads;
    constexpr int U = kMaxSplits / 32;
    float2 ml[U];
    float m = -INFINITY, total = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f}, f[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        ml[u] = 32 * u + lane < p.splits ? __ldcg(p.part_ml + (32 * u + lane) * step + unit) : make_float2(-INFINITY, 0.f);
        m = fmaxf(m, ml[u].x);
    }
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
#pragma unroll
    for (int u = 0; u < U; ++u) {
        f[u] = ml[u].y == 0.f ? 0.f : ml[u].x == m ? 1.f : exp2_approx(ml[u].x - m);      // 0: nothing seen in this part
        total = fmaf(f[u], ml[u].y, total);
    }
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) total += __shfl_xor_sync(0xffffffffu, total, i);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll 4
        for (int s = 32 * u; s < min(p.splits, 32 * u + 32); ++s) {
            const float g = __shfl_sync(0xffffffffu, f[u], s - 32 * u);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v = lane + 32 * j < a.head_dim ? __ldcg(p.part_o + (s * step + unit) * a.head_dim + lane + 32 * j) : 0.f;
                o[j] = g == 0.f ? o[j] : fmaf(g, v, o[j]);
            }
        }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (lane + 32 * j < a.head_dim)
            store_from_f32(a.out, tok * a.out_stride[0] + h * a.out_stride[1] + lane + 32 * j, a.kind, inv == 0.f ? 0.f : o[j] * inv);
    if (lane == 0 && a.lse != nullptr)
        a.lse[(int64_t)h * a.tokens + tok] = total == 0.f ? -INFINITY : (m + log2f(total)) * 0.6931471805599453f;
}

int check(const rvq_prompt_attn_args* a) {
    if (a == nullptr || a->tokens < 0 || a->keys < 0 || a->n_seq < 1) return RVQ_ERR_INVALID;
    if (a->n_kv < 1 || a->n_heads < a->n_kv || a->n_heads % a->n_kv != 0) return RVQ_ERR_INVALID;
    if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8 || a->n_heads / a->n_kv > 64) return RVQ_ERR_UNSUPPORTED;
    if (a->kind != RVQ_BF16 && a->kind != RVQ_F16) return RVQ_ERR_UNSUPPORTED;
    if (a->tokens > (1ll << 30) || a->keys > (1ll << 30)) return RVQ_ERR_TOO_LARGE;
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

std::mutex g_mu;
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

int prepare() {
    std::lock_guard<std::mutex> lock(g_mu);
    if (g_encode != nullptr) return RVQ_OK;
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
    if (e != cudaSuccess || q != cudaDriverEntryPointSuccess) {
        last_cuda_error_slot() = (int)e;
        return RVQ_ERR_UNAVAILABLE;
    }
    g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    return RVQ_OK;
}

// [rows][heads][head_dim] by boxes of 64 columns, `heads` heads and `rows` rows.
bool encode(CUtensorMap* map, const void* ptr, const rvq_prompt_attn_args& a, int64_t n_rows, int64_t n_heads,
            const int64_t* stride, int box_heads, int box_rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)a.head_dim, (cuuint64_t)n_heads, (cuuint64_t)n_rows};
    const cuuint64_t strides[2] = {(cuuint64_t)stride[1] * 2, (cuuint64_t)stride[0] * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
    const cuuint32_t estr[3] = {1, 1, 1};
    return g_encode(map, a.kind == RVQ_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                    const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int status(cudaError_t e) {
    if (e != cudaSuccess) last_cuda_error_slot() = (int)e;
    return e == cudaSuccess ? RVQ_OK : RVQ_ERR_CUDA;
}

template <int HD, bool kHalfType>
int run(const Params& p, cudaStream_t s) {
    auto* kernel = prompt_kernel<HD, kHalfType>;
    const int smem = (int)sizeof(Smem<HD>) + 1024;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess)
        e = launch_pdl(kernel, dim3((unsigned)(p.tickets != nullptr ? p.sms : p.units)), dim3(kThreads), (size_t)smem, s, p);
    if (e == cudaSuccess && p.splits > 1)
        e = launch_pdl(join_kernel, dim3((unsigned)((p.a.tokens * p.a.n_heads + 3) / 4)), dim3(128), 0, s, p);
    return status(e);
}

// Sizes of the launch: the pairs of tiles (each sequence has at most one that is not full) and the parts of the keys.  With
// fewer CTAs than half the SMs and keys enough, the keys are split so that every SM has a CTA, into parts of at
// least 4 tiles (the mean sequence's) each.  32/8 heads of 128, whole and as split: 64 queries (8 CTAs) after 1,024 keys 23.9 and
// 21.3 us, after 8,192 keys 126 and 28; 512 queries (64 CTAs) after 1,024 keys 31.0 and 30.1, after 8,192 keys 133 and 81.  At 8
// tiles the two are even (512 queries after 512 keys 24.1 and 25.9), below them whole is faster (256 after 512: 18.6, halved 20.0).
// Parts shorter than 4 tiles would pay where CTAs are very few (64 queries after 2,048 keys 21.9, with 6 parts 19.0; 16 queries
// 18.4 and with 9 parts 13.8).
int plan(const rvq_prompt_attn_args& a, Params* p) {
    p->rep = a.n_heads / a.n_kv;
    p->tile_tokens = kRows / p->rep;
    const int64_t per = 2 * p->tile_tokens;
    const int64_t pairs = a.n_seq == 1 ? (a.tokens + per - 1) / per : a.tokens / per + a.n_seq;
    if (pairs * a.n_kv >= (1ll << 31)) return RVQ_ERR_TOO_LARGE;
    p->pairs = (int32_t)pairs;
    p->splits = 1;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return status(e);
    const int64_t units = pairs * a.n_kv, tiles = (a.keys / a.n_seq + kKeys - 1) / kKeys;
    if (units * 2 <= sms && tiles >= 8) {
        const int64_t most = sms / units, parts = tiles / 4;
        const int64_t s = most < parts ? most : parts;
        p->splits = (int32_t)(s < kMaxSplits ? s : kMaxSplits);
    }
    p->sms = sms;
    p->units = (int32_t)(units * p->splits);
    return RVQ_OK;
}

size_t part_bytes(const rvq_prompt_attn_args& a, const Params& p) {
    if (p.units > p.sms) return 2 * sizeof(uint32_t);        // tickets
    return p.splits == 1 ? 0 : (size_t)p.splits * a.tokens * a.n_heads * (a.head_dim + 2) * 4;
}

}  // namespace prompt
}  // namespace rvq

using namespace rvq;
using namespace rvq::prompt;

extern "C" size_t rvq_prompt_attention_workspace_size(const rvq_prompt_attn_args* a) {
    Params p;
    if (check(a) != RVQ_OK || a->tokens == 0 || plan(*a, &p) != RVQ_OK) return 0;
    return part_bytes(*a, p);
}

extern "C" int rvq_prompt_attention(const rvq_prompt_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check(a);
    if (rc != RVQ_OK || a->tokens == 0) return rc;
    rc = prepare();
    if (rc != RVQ_OK) return rc;
    Params p;
    memset(&p, 0, sizeof(p));
    p.a = *a;
    rc = plan(*a, &p);
    if (rc != RVQ_OK) return rc;
    if (part_bytes(*a, p) > 0) {
        if (workspace == nullptr || workspace_bytes < part_bytes(*a, p) || ((uintptr_t)workspace & 15)) return RVQ_ERR_INVALID;
        if (p.units > p.sms) p.tickets = reinterpret_cast<uint32_t*>(workspace);
        p.part_o = reinterpret_cast<float*>(workspace);
        p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)p.splits * a->tokens * a->n_heads * a->head_dim);
    }
    // without keys nothing is loaded: any valid map will do
    const bool none = a->keys == 0;
    if (!encode(&p.q, a->q, *a, a->tokens, a->n_heads, a->q_stride, p.rep, p.tile_tokens) ||
        !encode(&p.k, none ? a->q : a->k, *a, none ? 1 : a->keys, none ? 1 : a->n_kv, a->k_stride, 1, kKeys) ||
        !encode(&p.v, none ? a->q : a->v, *a, none ? 1 : a->keys, none ? 1 : a->n_kv, a->v_stride, 1, kKeys))
        return RVQ_ERR_INVALID;
    p.wide = p.splits > 1 ? ((uintptr_t)workspace & 31) == 0
                          : ((uintptr_t)a->out & 31) == 0 && ((a->out_stride[0] | a->out_stride[1] | a->head_dim) & 15) == 0;
    cudaStream_t s = (cudaStream_t)stream;
    if (a->kind == RVQ_F16) return a->head_dim > 64 ? run<128, true>(p, s) : run<64, true>(p, s);
    return a->head_dim > 64 ? run<128, false>(p, s) : run<64, false>(p, s);
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
    return v;
}
