// Step attention over the 4-bit cache (rvq_cache4_attention, include/rvq_b200.h).

#include <string.h>

#include <cooperative_groups.h>

#include "rvq_cache4.cuh"
#include "rvq_sm100.cuh"
#include "rvq_stepops.cuh"

namespace cg = cooperative_groups;

namespace rvq {
namespace cache4 {

using namespace stepops;
using namespace sm100;

__device__ int g_step_timeout;               // sticky: a bounded wait gave up

// ---------------------------------------------------------------------------
// A cluster of C CTAs per (kv head, group of at most 8 query heads, sequence)
// splits the live rows into contiguous ranges of 32-row tiles; in a CTA the
// warps take the range's tiles in turn, each through a ring of its own that
// bulk copies fill (a tile's records are contiguous).  Both products run on
// mma.m16n8k16 with the heads as rows:
//
//   scores   q . k = sum over groups of  step (q . c) + zero (q . 1)
//   output   sum_j p_j v_j = sum_j (p_j step_j) c_j + sum_j p_j zero_j
//
// so an operand is a 4-bit code, never a rounded value.  A code becomes a bf16
// number by placing it in the mantissa of 1.0: 1 + c / 16, exact, one shift and
// one lop3 for two codes; the 1 is taken out again by starting the score
// accumulator at -(q . 1) and by subtracting 16 p step in the zeros' sum.
// p step is split into a bf16 part in rows 0..7 and the bf16 remainder in rows
// 8..15 of the same operand (16 bits of it, at no further MMA); an fp16 q the
// same way.  Softmax: one pass, running maximum and sum per warp, partial
// results joined warp by warp and CTA by CTA in fixed order through shared
// and distributed shared memory, so results do not depend on scheduling.
// ---------------------------------------------------------------------------
constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 32;                    // rows of a ring stage
constexpr int kStages = 3;
constexpr int kHeads = 8;                    // query heads of a pass
constexpr int kMaxRep = 64;
constexpr long long kWaitPolls = 1ll << 22;  // a try_wait sleeps in hardware: seconds

template <int HD>
struct Smem {
    static constexpr int REC = record_bytes(HD), G = HD / kGroup;
    alignas(128) uint8_t ring[kWarps][kStages][kTile * REC];
    alignas(16) uint8_t fresh[kTile * REC];  // the appended record, the other rows zero
    float q[kHeads][HD];
    float qsum[kHeads][G];
    float kv[2][HD];                         // the new key and value
    float norm[4][HD];
    float wm[kWarps][kHeads], wl[kWarps][kHeads];
    float m[kHeads], l[kHeads];              // this CTA's maximum and sum
    float fm[kHeads], fr[kHeads];            // the final maximum and 1 / sum
    alignas(8) uint64_t bar[kWarps][kStages];
};

// 1 + c / 16 for the codes in bits 4 i .. 4 i + 3 and 4 i + 16 .. of a word
template <int I>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
    const uint32_t x = I == 0 ? w << 3 : w >> (4 * I - 3 > 0 ? 4 * I - 3 : 0);
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(x), "r"(0x00780078u), "r"(0x3f803f80u));   // (x & m) | o
    return r;
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// hi + lo = x to 16 bits
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t* hi, uint32_t* lo) {
    *hi = pack_bf16(x, y);
    *lo = pack_bf16(x - __uint_as_float(*hi << 16), y - __uint_as_float(*hi & 0xffff0000u));
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// What a warp carries over its tiles.  Lane 4 g + t: head g's maximum, the parts of its sums over this lane's rows,
// and output values of head g (bf16 parts, then remainders).
template <int HD>
struct State {
    static constexpr int G = HD / kGroup;
    float m, l;
    float zero[G];                           // sum of p (zero - 16 step)
    float o[G][4][4];
};

// One tile of `valid` rows (the records behind them hold zeros if valid < kTile).
template <int HD, bool kSplitQ>
__device__ __forceinline__ void tile_step(const uint8_t* rec, int valid, const uint32_t (&qa)[HD / 16][kSplitQ ? 4 : 2],
                                          const float (&qs)[HD / kGroup], float scale16, State<HD>& st, float* scores) {
    constexpr int G = HD / kGroup, REC = record_bytes(HD);
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll 1
    for (int half = 0; half < kTile / 16; ++half) {
        if (half * 16 >= valid) break;
        const uint8_t* base = rec + half * 16 * REC;
        // columns n of a score tile hold row (n with its two low bits swapped): a quarter warp's 16-byte loads of two
        // rows then fall into different banks, and this lane's columns 2 t and 2 t + 1 are rows ra and ra + 2
        const int rn = (g & 4) | (g & 1) << 1 | (g >> 1 & 1);
        const int ra = (t >> 1) * 4 + (t & 1);
        float s[4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const uint8_t* r0 = base + (8 * n + ra) * REC + HD;
            uint32_t kc[G], pa[G], pb[G];
            if constexpr (HD == 128) {
                *reinterpret_cast<uint4*>(kc) = *reinterpret_cast<const uint4*>(base + (8 * n + rn) * REC + 16 * t);
                *reinterpret_cast<uint4*>(pa) = *reinterpret_cast<const uint4*>(r0);
                *reinterpret_cast<uint4*>(pb) = *reinterpret_cast<const uint4*>(r0 + 2 * REC);
            } else {
                *reinterpret_cast<uint2*>(kc) = *reinterpret_cast<const uint2*>(base + (8 * n + rn) * REC + 8 * t);
                *reinterpret_cast<uint2*>(pa) = *reinterpret_cast<const uint2*>(r0);
                *reinterpret_cast<uint2*>(pb) = *reinterpret_cast<const uint2*>(r0 + 2 * REC);
            }
            float sa = 0.f, sb = 0.f;
#pragma unroll
            for (int i = 0; i < G; ++i) {
                float c[4] = {-qs[i], -qs[i], 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t a[4] = {qa[2 * i + k][0], 0u, qa[2 * i + k][1], 0u};
                    if constexpr (kSplitQ) a[1] = qa[2 * i + k][2], a[3] = qa[2 * i + k][3];
                    mma16816(c, a, k ? code_pair<2>(kc[i]) : code_pair<0>(kc[i]), k ? code_pair<3>(kc[i]) : code_pair<1>(kc[i]));
                }
                if constexpr (kSplitQ) c[0] += c[2], c[1] += c[3];
                // in units of 16: step (q . c) / 16 + zero (q . 1) / 16
                sa = fmaf(step_of(pa[i]), c[0], fmaf(zero_of(pa[i]), qs[i] * 0.0625f, sa));
                sb = fmaf(step_of(pb[i]), c[1], fmaf(zero_of(pb[i]), qs[i] * 0.0625f, sb));
            }
            s[2 * n] = sa * scale16;
            s[2 * n + 1] = sb * scale16;
        }
        if (half * 16 + 16 > valid) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (half * 16 + 8 * (i >> 1) + ra + 2 * (i & 1) >= valid) s[i] = -INFINITY;
        }
        if (scores != nullptr) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = half * 16 + 8 * (i >> 1) + ra + 2 * (i & 1);
                if (row < valid) scores[row] = s[i];
            }
        }
        float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const bool grows = top > st.m;
        if (__any_sync(0xffffffffu, grows)) {
            const float m = fmaxf(st.m, top);
            const float f = st.m == m ? 1.f : exp2_approx(st.m - m);
            st.m = m;
            st.l *= f;
#pragma unroll
            for (int i = 0; i < G; ++i) {
                st.zero[i] *= f;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) st.o[i][j][c] *= f;
            }
        }
        // nothing but -infinities so far: p = exp(-infinity) = 0, not exp(-infinity + infinity)
        const float sub = st.m == -INFINITY ? 0.f : st.m;
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[i] = exp2_approx(s[i] - sub);
            st.l += p[i];
        }
        uint32_t vc[4][G], vp[4][G];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint8_t* r = base + (8 * (i >> 1) + ra + 2 * (i & 1)) * REC;
            if constexpr (HD == 128) {
                *reinterpret_cast<uint4*>(vc[i]) = *reinterpret_cast<const uint4*>(r + HD / 2 + 16 * (g >> 1));
                *reinterpret_cast<uint4*>(vp[i]) = *reinterpret_cast<const uint4*>(r + HD + HD / 8);
            } else {
                *reinterpret_cast<uint2*>(vc[i]) = *reinterpret_cast<const uint2*>(r + HD / 2 + 8 * (g >> 1));
                *reinterpret_cast<uint2*>(vp[i]) = *reinterpret_cast<const uint2*>(r + HD + HD / 8);
            }
        }
        const uint32_t half_sel = g & 1 ? 0x7632u : 0x5410u;      // this lane's 4 values are half a code word
#pragma unroll
        for (int i = 0; i < G; ++i) {
            float ps[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float step = step_of(vp[k][i]);
                ps[k] = p[k] * step;
                st.zero[i] = fmaf(p[k], fmaf(-16.f, step, zero_of(vp[k][i])), st.zero[i]);
            }
            uint32_t a[4];
            split_bf16(ps[0], ps[1], &a[0], &a[1]);
            split_bf16(ps[2], ps[3], &a[2], &a[3]);
            const uint32_t w0 = __byte_perm(vc[0][i], vc[1][i], half_sel);
            const uint32_t w1 = __byte_perm(vc[2][i], vc[3][i], half_sel);
            mma16816(st.o[i][0], a, code_pair<0>(w0), code_pair<0>(w1));
            mma16816(st.o[i][1], a, code_pair<1>(w0), code_pair<1>(w1));
            mma16816(st.o[i][2], a, code_pair<2>(w0), code_pair<2>(w1));
            mma16816(st.o[i][3], a, code_pair<3>(w0), code_pair<3>(w1));
        }
    }
}

// Norm and rotation of one head held by one warp in shared memory, rounding as step attention does.
template <int HD>
__device__ __forceinline__ void norm_rope(float* x, const float* w, const rvq_cache4_attn_args& a, const float* cv,
                                          const float* sv) {
    constexpr int J = HD / 32;
    const int lane = threadIdx.x & 31;
    float v[J];
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) v[j] = x[lane + 32 * j], ss = fmaf(v[j], v[j], ss);
    if (a.q_norm != nullptr) {
        const float inv = rsqrtf(warp_sum(ss) / (float)HD + a.eps);
#pragma unroll
        for (int j = 0; j < J; ++j) v[j] = bf16r(w[lane + 32 * j] * bf16r(v[j] * inv));
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int d = lane + 32 * j;
        const float rot = j < J / 2 ? -v[j + J / 2] : v[j - J / 2];
        x[d] = a.cos != nullptr ? bf16r(bf16r(v[j] * cv[d]) + bf16r(rot * sv[d])) : v[j];
    }
    __syncwarp();
}

// The record of the new token (S.kv) by one warp; lane l holds values (HD / 32) l ...
template <int HD>
__device__ __forceinline__ void encode(const float* x, uint8_t* codes, uint32_t* params) {
    constexpr int E = HD / 32, LG = 32 / E;                  // values of a lane, lanes of a group
    const int lane = threadIdx.x & 31;
    float v[E], lo = INFINITY, hi = -INFINITY;
    int bad = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] = x[E * lane + e];
        lo = fminf(lo, v[e]);
        hi = fmaxf(hi, v[e]);
        bad |= v[e] != v[e];
    }
#pragma unroll
    for (int o = 1; o < LG; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad |= __shfl_xor_sync(0xffffffffu, bad, o);
    }
    const uint32_t p = bad ? params_of(NAN, NAN) : params_of(lo, hi);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        const int d = E * lane + e;
        codes[(d % 32 / 8 * (HD / kGroup) + d / 32) * 4 + d % 8 / 2] =
            (uint8_t)(code_of(v[e], zero_of(p), step_of(p)) | code_of(v[e + 1], zero_of(p), step_of(p)) << 4);
    }
    if (lane % LG == 0) params[lane / LG] = p;
}

template <int HD, bool kSplitQ>
__global__ void __launch_bounds__(kThreads, 1) cache4_attn_kernel(rvq_cache4_attn_args a, int passes) {
    constexpr int G = HD / kGroup, REC = record_bytes(HD);
    extern __shared__ __align__(128) uint8_t smem_raw[];
    Smem<HD>& S = *reinterpret_cast<Smem<HD>*>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int nkv = a.cache.n_kv, rep = a.n_heads / nkv;
    const int kv = blockIdx.y % nkv, b = blockIdx.z;
    pdl_launch_dependents();
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(smem_addr(&S.bar[warp][i]), 1);
        mbar_init_fence();
        fence_async_shared();
    }
    pdl_wait();
    const int64_t rows = a.rows[b];
    if (rows < 0) return;                                    // the same in every CTA of the cluster
    const bool append = a.k.ptr != nullptr;
    const int64_t pos = a.pos != nullptr ? a.pos[b] : 0;
    const int64_t kv_at = ((int64_t)b * nkv + kv) * HD;
    const int out_kind = a.q.kind == RVQ_F16 ? RVQ_F16 : RVQ_BF16;
    // heads [h0, h1) of the kv head: all of them in `passes` passes of this CTA, or one group of them per CTA
    const int groups = (rep + kHeads - 1) / kHeads, per = (rep + groups - 1) / groups;
    const int first = passes == groups ? 0 : blockIdx.y / nkv;
    if (rows + append < 1 || rows + append > a.cache.max_len || pos < 0 || (a.pos != nullptr && pos >= a.table_len)) {
        if (rank == 0) {
            const int h0 = first * per, h1 = min(rep, (first + passes) * per);
            const int64_t at = ((int64_t)b * a.n_heads + kv * rep) * HD;
            for (int i = h0 * HD + tid; i < h1 * HD; i += kThreads) store_from_f32(a.out, at + i, out_kind, 0.f);
        }
        return;
    }
    uint8_t* cache = reinterpret_cast<uint8_t*>(a.cache.data) + ((int64_t)b * nkv + kv) * a.cache.max_len * REC;
    const int tiles = (int)((rows + kTile - 1) / kTile);
    const int t0 = (int)((int64_t)tiles * rank / C), t1 = (int)((int64_t)tiles * (rank + 1) / C);
    const bool owner = append && rank == 0;                  // this CTA attends to the new row

    int issued = 0, used = 0;                                // ring stages filled and read by this warp
    bool dead = false;                                       // a copy did not arrive: the result is invalid, flagged
    auto issue = [&](int tile) {                             // lane 0
        const int valid = (int)min((int64_t)kTile, rows - (int64_t)tile * kTile);
        const uint32_t bar = smem_addr(&S.bar[warp][issued % kStages]);
        mbar_expect_tx(bar, (uint32_t)(valid * REC));
        bulk_load(smem_addr(S.ring[warp][issued % kStages]), cache + (int64_t)tile * kTile * REC, (uint32_t)(valid * REC), bar);
        ++issued;
    };

    for (int pass = 0; pass < passes; ++pass) {
        const int h0 = (first + pass) * per, heads = min(per, rep - h0);
        const int64_t q_at = ((int64_t)b * a.n_heads + kv * rep + h0) * HD;
        int next = t0 + warp;                                // this warp's next tile to fetch
        if (lane == 0)
            for (; !dead && issued - used < kStages && next < t1; next += kWarps) issue(next);
        next = __shfl_sync(0xffffffffu, next, 0);

        // the heads' q, and the new record
        if (pass == 0 && (a.q_norm != nullptr || a.cos != nullptr)) {
            for (int i = tid; i < HD; i += kThreads) {
                S.norm[0][i] = a.q_norm != nullptr ? bf16_at(a.q_norm, i) : 0.f;
                S.norm[1][i] = a.q_norm != nullptr ? bf16_at(a.k_norm, i) : 0.f;
                S.norm[2][i] = a.cos != nullptr ? bf16_at(a.cos, pos * HD + i) : 0.f;
                S.norm[3][i] = a.cos != nullptr ? bf16_at(a.sin, pos * HD + i) : 0.f;
            }
        }
        for (int i = tid; i < kHeads * HD; i += kThreads)
            (&S.q[0][0])[i] = i < heads * HD ? vec_value_deep(a.q, q_at + i) : 0.f;
        if (owner && pass == 0) {
            for (int i = tid; i < 2 * HD; i += kThreads) (&S.kv[0][0])[i] = vec_value_deep(i < HD ? a.k : a.v, kv_at + i % HD);
            for (int i = tid; i < kTile * REC / 4; i += kThreads) reinterpret_cast<uint32_t*>(S.fresh)[i] = 0;
        }
        __syncthreads();
        if (a.q_norm != nullptr || a.cos != nullptr) {
            norm_rope<HD>(S.q[warp], S.norm[0], a, S.norm[2], S.norm[3]);
            if (owner && pass == 0 && warp == 0) norm_rope<HD>(S.kv[0], S.norm[1], a, S.norm[2], S.norm[3]);
        }
        {
            float v[G];
#pragma unroll
            for (int i = 0; i < G; ++i) {
                v[i] = warp_sum(S.q[warp][kGroup * i + lane]);
                if (lane == 0) S.qsum[warp][i] = v[i];
            }
        }
        if (owner && pass == 0 && warp < 2) {
            encode<HD>(S.kv[warp], S.fresh + warp * (HD / 2), reinterpret_cast<uint32_t*>(S.fresh + HD + warp * (HD / 8)));
        }
        __syncthreads();
        if (owner && pass == 0 && first == 0 && tid < REC / 16)
            reinterpret_cast<uint4*>(cache + rows * REC)[tid] = reinterpret_cast<const uint4*>(S.fresh)[tid];

        // operand rows 0..7: q (its bf16 part), rows 8..15: the remainder; column pairs in the code words' order
        uint32_t qa[HD / 16][kSplitQ ? 4 : 2];
        float qs[G];
#pragma unroll
        for (int i = 0; i < G; ++i) qs[i] = S.qsum[g][i];
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            const float* q = &S.q[g][i / 2 * kGroup + 8 * t + 2 * (i & 1)];
            if constexpr (kSplitQ) {
                split_bf16(q[0], q[4], &qa[i][0], &qa[i][2]);
                split_bf16(q[1], q[5], &qa[i][1], &qa[i][3]);
            } else {
                qa[i][0] = pack_bf16(q[0], q[4]);
                qa[i][1] = pack_bf16(q[1], q[5]);
            }
        }
        State<HD> st;
        st.m = -INFINITY, st.l = 0.f;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            st.zero[i] = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) st.o[i][j][c] = 0.f;
        }
        const float scale16 = a.scaling * 16.f * 1.4426950408889634f;      // scores in powers of two
        float* sc = a.weights != nullptr && g < heads
                        ? a.scores + ((int64_t)b * a.n_heads + kv * rep + h0 + g) * a.cache.max_len : nullptr;
        if (owner && warp == kWarps - 1) tile_step<HD, kSplitQ>(S.fresh, 1, qa, qs, scale16, st, sc ? sc + rows : sc);
        for (int tile = t0 + warp; tile < t1 && !dead; tile += kWarps) {
            const int slot = used % kStages;
            const bool here = mbar_wait(smem_addr(&S.bar[warp][slot]), used / kStages & 1, kWaitPolls, &g_step_timeout);
            if (__any_sync(0xffffffffu, !here)) {
                dead = true;
                break;
            }
            const int valid = (int)min((int64_t)kTile, rows - (int64_t)tile * kTile);
            uint8_t* rec = S.ring[warp][slot];
            if (valid < kTile) {                             // only the last tile: no copy follows into this stage in this pass
                for (int i = valid * REC / 16 + lane; i < kTile * REC / 16; i += 32)
                    reinterpret_cast<uint4*>(rec)[i] = make_uint4(0, 0, 0, 0);
                fence_async_shared();
                __syncwarp();
            }
            tile_step<HD, kSplitQ>(rec, valid, qa, qs, scale16, st, sc ? sc + (int64_t)tile * kTile : sc);
            __syncwarp();                                    // every lane has read the stage
            ++used;
            if (next < t1) {
                if (lane == 0) issue(next);
                next += kWarps;
            }
        }
        if (dead && lane == 0)                               // once more for the copies in flight, before their stages are reused
            for (; used < issued; ++used)
                mbar_wait(smem_addr(&S.bar[warp][used % kStages]), used / kStages & 1, kWaitPolls, &g_step_timeout);
        __syncwarp();
        // lanes 4 g .. 4 g + 3 hold parts of head g's sums
        float l = st.l;
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
#pragma unroll
        for (int i = 0; i < G; ++i) {
            st.zero[i] += __shfl_xor_sync(0xffffffffu, st.zero[i], 1);
            st.zero[i] += __shfl_xor_sync(0xffffffffu, st.zero[i], 2);
        }
        __syncthreads();                                     // the rings are read: they take the warps' outputs
        float* wo = reinterpret_cast<float*>(S.ring);        // [kWarps][kHeads][HD], then the CTA's [kHeads][HD]
        float* co = wo + kWarps * kHeads * HD;
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float* d = wo + (warp * kHeads + g) * HD + kGroup * i + 8 * t + j;
                d[0] = fmaf(16.f, st.o[i][j][0] + st.o[i][j][2], st.zero[i]);
                d[4] = fmaf(16.f, st.o[i][j][1] + st.o[i][j][3], st.zero[i]);
            }
        if (t == 0) S.wm[warp][g] = st.m, S.wl[warp][g] = l;
        __syncthreads();
        {
            // warp w joins head w over the warps
            float m = S.wm[0][warp];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) m = fmaxf(m, S.wm[w][warp]);
            float f[kWarps], total = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                f[w] = S.wm[w][warp] == m ? 1.f : exp2_approx(S.wm[w][warp] - m);
                total = fmaf(f[w], S.wl[w][warp], total);
            }
#pragma unroll
            for (int d = lane; d < HD; d += 32) {
                float o = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) o = fmaf(f[w], wo[(w * kHeads + warp) * HD + d], o);
                co[warp * HD + d] = o;
            }
            if (lane == 0) S.m[warp] = m, S.l[warp] = total;
        }
        cluster.sync();
        if (tid < heads) {
            float m = -INFINITY, total = 0.f;
            for (int c = 0; c < C; ++c) m = fmaxf(m, cluster.map_shared_rank(S.m, c)[tid]);
            for (int c = 0; c < C; ++c) {
                const float mc = cluster.map_shared_rank(S.m, c)[tid];
                total = fmaf(mc == m ? 1.f : exp2_approx(mc - m), cluster.map_shared_rank(S.l, c)[tid], total);
            }
            S.fm[tid] = m;
            S.fr[tid] = total == 0.f ? 0.f : 1.f / total;    // no score above -infinity: zeros
        }
        __syncthreads();
        const int n = heads * HD, chunk = (n + C - 1) / C;
        for (int i = rank * chunk + tid; i < min(n, (rank + 1) * chunk); i += kThreads) {
            const int h = i / HD;
            float o = 0.f;
            for (int c = 0; c < C; ++c) {
                const float mc = cluster.map_shared_rank(S.m, c)[h];
                o = fmaf(mc == S.fm[h] ? 1.f : exp2_approx(mc - S.fm[h]), cluster.map_shared_rank(co, c)[i], o);
            }
            store_from_f32(a.out, q_at + i, out_kind, S.fr[h] == 0.f ? 0.f : o * S.fr[h]);
        }
        if (a.weights != nullptr) {                          // this CTA's rows, heads in order
            float* w = a.weights + ((int64_t)b * nkv + kv) * a.cache.max_len;
            const float* s0 = a.scores + ((int64_t)b * a.n_heads + kv * rep + h0) * a.cache.max_len;
            auto add = [&](int64_t row, float v) {
                for (int h = 0; h < heads; ++h)
                    if (S.fr[h] != 0.f) v += exp2_approx(s0[(int64_t)h * a.cache.max_len + row] - S.fm[h]) * S.fr[h];
                w[row] = v;
            };
            const int64_t r1 = min(rows, (int64_t)t1 * kTile);
            for (int64_t row = (int64_t)t0 * kTile + tid; row < r1; row += kThreads) add(row, w[row]);
            if (owner && tid == 0) add(rows, pass == 0 ? 0.f : w[rows]);
        }
        fence_async_shared();                                // copies may fill the rings again
        cluster.sync();                                      // once the others have read this CTA's parts
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
    if (c.n_seq > 65535 || a->n_heads > 65535) return RVQ_ERR_TOO_LARGE;
    return RVQ_OK;
}

template <int HD, bool kSplitQ>
int run(const rvq_cache4_attn_args& a, cudaStream_t s) {
    auto* kernel = cache4_attn_kernel<HD, kSplitQ>;
    const int smem = (int)sizeof(Smem<HD>);
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return status(e);
    const int rep = a.n_heads / a.cache.n_kv, groups = (rep + kHeads - 1) / kHeads;
    const int passes = a.weights != nullptr ? groups : 1;
    const int64_t units = (int64_t)a.cache.n_seq * a.cache.n_kv * (groups / passes);
    int c = 1;
    while (c < 16 && units * c * 2 <= sms && (int64_t)c * kWarps * kTile < a.cache.max_len) c *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c, a.cache.n_kv * (groups / passes), a.cache.n_seq);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = c;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return status(cudaLaunchKernelEx(&cfg, kernel, a, passes));
}

}  // namespace cache4

// 1 if the sticky flag was set (it is cleared), 0 if not, a negative status on an error.
int take_step_timeout() {
    int v = 0;
    const int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, cache4::g_step_timeout, sizeof(int));
    if (e == cudaSuccess) e = cudaMemcpyToSymbol(cache4::g_step_timeout, &zero, sizeof(int));
    return e == cudaSuccess ? v : -cache4::status(e);
}

}  // namespace rvq

using namespace rvq;
using namespace rvq::cache4;

extern "C" int rvq_cache4_attention(const rvq_cache4_attn_args* a, void* stream) {
    const int rc = check(a);
    if (rc != RVQ_OK) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    const bool split = a->q.kind == RVQ_F16;
    if (a->cache.head_dim == 128) return split ? run<128, true>(*a, s) : run<128, false>(*a, s);
    return split ? run<64, true>(*a, s) : run<64, false>(*a, s);
}
