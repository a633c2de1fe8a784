// Step attention over the 4-bit cache (rvq_cache4_attention, include/rvq_b200.h).

#include <string.h>

#include "rvq_cache4.cuh"
#include "rvq_sm100.cuh"
#include "rvq_stepops.cuh"

namespace rvq {
namespace cache4 {

using namespace stepops;
using sm100::smem_addr;

// ---------------------------------------------------------------------------
// The live rows of a (kv head, group of at most 8 query heads, sequence) are
// split into contiguous ranges of 16-row tiles, a CTA each; in a CTA the warps
// take the range's tiles in turn, each through a ring of its own (cp.async).
// Both products run on mma.m16n8k16:
//
//   scores   q . k = sum over groups of  step (q . c) + zero (q . 1)
//   output   sum_j p_j v_j = sum_j (p_j step_j) c_j + sum_j p_j zero_j
//
// so an operand is a 4-bit code (exact), never a rounded value; the sums with
// the zeros are one more MMA each, on the parameter words as they lie there.
// p step is split into two bf16 parts (16 bits), q . 1 into three (24 bits).  Softmax: one pass, running maximum and sum per warp;
// partial results are joined in fixed order, warp by warp in the CTA and range
// by range in a second launch, so results do not depend on scheduling.
//
// No unit is full: of about 540 instructions a tile 250 are masks, shifts and conversions on
// the ALU pipe (55 % of its peak), issue 60 %, tensor pipe 25 %; a warp that could go on waits for its turn
// (1.3 clocks an instruction), the ALU (1.1) and results (0.9 fixed, 0.5 loads).  HBM is far away: 64 sequences of
// 4,096 rows, 64/8 heads of 128, 113 us, 2.96 TB/s of records (45 % of measured copy
// bandwidth).  One sequence of 40,000 rows with weights:
// 27.6 us; of 300 rows: 7.5 us, a chain of latencies (row count, copies, three tiles,
// the join of the warps).  Measured against this form: clusters of CTAs joining over
// distributed shared memory left SMs idle (40,000 rows: 54 us); bulk copies with
// mbarriers cost more instructions than cp.async (64 x 4,096: 154 against 134 us);
// the heads as the M of both MMAs left half the operand rows zero (118 against 129).
// ---------------------------------------------------------------------------
constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 16;                    // rows of a ring stage
constexpr int kStages = 4;
constexpr int kHeads = kWarps;               // query heads of a pass (a warp each where heads are worked on)
constexpr int kMaxRep = 64;
constexpr float kGrow = 8.f;

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
    float m[kHeads], r[kHeads];              // of the heads joined: maximum and reciprocal sum
};

// c / 64 for the codes c in bits 4 I .. and 4 I + 16 .. (I = 0 or 1) of a word, as a bf16 pair.  A code in a bf16
// number's lowest bits is the (sub)normal number c 2^-133 (c 2^-129 in bits 4 to 7: the step from the mantissa into the
// exponent is linear there), which one multiplication makes c / 64: exact, and on the FMA pipe, of which there is more.
template <int I>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w & (I ? 0x00f000f0u : 0x000f000fu)), "r"(I ? 0x7d007d00u : 0x7f007f00u));
    return r;
}

// The same as fp16 numbers, c / 512 (a code in the lowest 10 bits is a subnormal number): against an fp16 q.
template <int I>
__device__ __forceinline__ uint32_t code_pair_half(uint32_t w) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w & (I ? 0x00f000f0u : 0x000f000fu)), "r"(I ? 0x68006800u : 0x78007800u));
    return r;
}

// Numbers of a parameter word: the shift as a multiplication (`shift` holds 65536 where the compiler cannot see it), which
// runs on the FMA pipe; the masks and shifts of this kernel's integer pipe are what bounds it.
__device__ __forceinline__ float zero_by(uint32_t p, uint32_t shift) {
    uint32_t r;
    asm("mul.lo.u32 %0, %1, %2;" : "=r"(r) : "r"(p), "r"(shift));
    return __uint_as_float(r);
}

// D += A B, and D = A B
template <bool kHalf = false>
__device__ __forceinline__ void mma_add(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    if constexpr (kHalf)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool kHalf = false>
__device__ __forceinline__ void mma_set(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    if constexpr (kHalf)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};\n"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};\n"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// hi + lo = x to 16 bits
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t* hi, uint32_t* lo, uint32_t shift) {
    *hi = pack_bf16(x, y);
    *lo = pack_bf16(x - zero_by(*hi, shift), y - step_of(*hi));
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16 bytes to shared memory, or 16 zero bytes.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

// What a warp carries over its tiles.  Lane 4 g + t has heads 2 t and 2 t + 1 everywhere: their maxima and the parts of
// their sums from rows g and g + 8; the sums of p times halfword g of the parameters (zero of group g / 2 for even g) in
// zero[0] and [1]; and of the output, transposed, value 4 g + i of group G in o[G][i / 2][2 (i & 1) + (0, 1)].
template <int HD>
struct State {
    static constexpr int G = HD / kGroup;
    float m[2], l[2];
    float zero[4];
    float o[G][2][4];
};

// The 8 x 8 matrix of 16-bit values of which lane 4 g + t holds row g, columns 2 t and 2 t + 1, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <int G>
__device__ __forceinline__ void load_words(uint32_t (&w)[G], uint32_t addr) {
    if constexpr (G == 4)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
    else
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
}

// A tile of 16 rows, `valid` of them live (the records behind those hold zeros).  The rows are the M of the scores'
// MMA and the K of the output's, the heads the N of both; between the two the probabilities, heads along the lanes'
// registers, are transposed to rows along them.
template <int HD, bool kHalfQ>
__device__ __forceinline__ void tile_step(uint32_t base, int valid, const uint32_t (&qa)[HD / 16][2],
                                          const uint32_t (&qz)[3], float scale, uint32_t shift, State<HD>& st,
                                          bool keep, float* const (&scores)[2]) {
    constexpr int G = HD / kGroup, REC = record_bytes(HD);
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // row g of an MMA is row (g with its two low bits swapped) of the tile: a quarter warp's 16-byte loads of two rows then
    // fall into different banks; rows 2 t and 2 t + 1 are so ra and ra + 2
    const int rn = (g & 4) | (g & 1) << 1 | (g >> 1 & 1);
    const int ra = (t >> 1) * 4 + (t & 1);
    const uint32_t r0 = base + rn * REC, r1 = r0 + 8 * REC;
    float s[4];                                              // rows rn (heads 2 t, 2 t + 1) and rn + 8
    {
        uint32_t k0[G], k1[G], p0[G], p1[G], z0, z1;
        load_words<G>(k0, r0 + 4 * G * t);
        load_words<G>(k1, r1 + 4 * G * t);
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(z0) : "r"(r0 + HD + 4 * (t & (G - 1))));
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(z1) : "r"(r1 + HD + 4 * (t & (G - 1))));
        load_words<G>(p0, r0 + HD);
        load_words<G>(p1, r1 + HD);
        float z[4], c[G][4];                                 // zero . (q . 1) and q . c of every group, over 64 (512 for fp16)
        auto c0 = [](uint32_t w) { return kHalfQ ? code_pair_half<0>(w) : code_pair<0>(w); };
        auto c1 = [](uint32_t w) { return kHalfQ ? code_pair_half<1>(w) : code_pair<1>(w); };
        mma_set(z, z0, z1, z0, z1, qz[0], qz[1]);
#pragma unroll
        for (int i = 0; i < G; ++i) mma_set<kHalfQ>(c[i], c0(k0[i]), c0(k1[i]), c1(k0[i]), c1(k1[i]), qa[2 * i][0], qa[2 * i][1]);
        mma_add(z, z0, z1, z0, z1, qz[2], 0u);
#pragma unroll
        for (int i = 0; i < G; ++i) {
            k0[i] >>= 8, k1[i] >>= 8;
            mma_add<kHalfQ>(c[i], c0(k0[i]), c0(k1[i]), c1(k0[i]), c1(k1[i]), qa[2 * i + 1][0], qa[2 * i + 1][1]);
        }
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const float x = step_of(p0[i]), y = step_of(p1[i]);
            z[0] = fmaf(x, c[i][0], z[0]), z[1] = fmaf(x, c[i][1], z[1]);
            z[2] = fmaf(y, c[i][2], z[2]), z[3] = fmaf(y, c[i][3], z[3]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = z[i] * scale;
    }
    if (valid < 16) {
        if (rn >= valid) s[0] = s[1] = -INFINITY;
        if (rn + 8 >= valid) s[2] = s[3] = -INFINITY;
    }
    if (keep) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (scores[i & 1] != nullptr && rn + 8 * (i >> 1) < valid) scores[i & 1][rn + 8 * (i >> 1)] = s[i];
    }
    // the maximum that is subtracted follows the true one only when that has grown by 2^8 (p stays below 2^8): of 16
    // rows and 8 heads some has a new maximum in most tiles
    float top0 = fmaxf(s[0], s[2]), top1 = fmaxf(s[1], s[3]);
    if (__any_sync(0xffffffffu, top0 > st.m[0] + kGrow || top1 > st.m[1] + kGrow)) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, o));
            top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, o));
        }
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float m = fmaxf(st.m[i], i ? top1 : top0);
            f[i] = st.m[i] == m ? 1.f : exp2_approx(st.m[i] - m);
            st.m[i] = m;
            st.l[i] *= f[i];
            st.zero[i] *= f[i];
        }
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) st.o[i][j][c] *= f[c & 1];
    }
    // nothing but -infinities so far: p = exp(-infinity) = 0, not exp(-infinity + infinity)
    const float sub0 = st.m[0] == -INFINITY ? 0.f : st.m[0], sub1 = st.m[1] == -INFINITY ? 0.f : st.m[1];
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = exp2_approx(s[i] - (i & 1 ? sub1 : sub0));
    st.l[0] += p[0] + p[2];
    st.l[1] += p[1] + p[3];
    uint32_t vc[4][G], p0[G], p1[G], h[4], zs[4];
    load_words<G>(p0, r0 + HD + HD / 8);
    load_words<G>(p1, r1 + HD + HD / 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t r = base + (8 * (i >> 1) + ra + 2 * (i & 1)) * REC + HD / 2;
        load_words<G>(vc[i], r + 4 * G * (g >> 1));
        asm volatile("ld.shared.u16 %0, [%1];" : "=r"(zs[i]) : "r"(r + HD / 2 + HD / 8 + 2 * (g & (2 * G - 1))));
    }
    // two parts of (x, y) in rows rn and of (u, v) in rows rn + 8, transposed: {part 0, part 1} of rows ra and ra + 2, then + 8
    auto operand = [&](float x, float y, float u, float v) {
        split_bf16(x, y, &h[0], &h[1], shift);
        split_bf16(u, v, &h[2], &h[3], shift);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = transpose8(h[i]);
    };
    operand(p[0], p[1], p[2], p[3]);
    const uint32_t za = __byte_perm(zs[0], zs[1], 0x5410u), zb = __byte_perm(zs[2], zs[3], 0x5410u);
    mma_add(st.zero, za, 0u, zb, 0u, h[0], h[2]);
    mma_add(st.zero, za, 0u, zb, 0u, h[1], h[3]);
    const uint32_t half_sel = g & 1 ? 0x7632u : 0x5410u;     // this lane's 4 values are half a code word
#pragma unroll
    for (int i = 0; i < G; ++i) {
        const float x = step_of(p0[i]), y = step_of(p1[i]);
        operand(p[0] * x, p[1] * x, p[2] * y, p[3] * y);
        const uint32_t w0 = __byte_perm(vc[0][i], vc[1][i], half_sel), w1 = __byte_perm(vc[2][i], vc[3][i], half_sel);
        const uint32_t v0 = code_pair<0>(w0), v1 = code_pair<1>(w0), v2 = code_pair<0>(w1), v3 = code_pair<1>(w1);
        const uint32_t x0 = code_pair<0>(w0 >> 8), x1 = code_pair<1>(w0 >> 8);
        const uint32_t x2 = code_pair<0>(w1 >> 8), x3 = code_pair<1>(w1 >> 8);
        mma_add(st.o[i][0], v0, v1, v2, v3, h[0], h[2]);
        mma_add(st.o[i][1], x0, x1, x2, x3, h[0], h[2]);
        mma_add(st.o[i][0], v0, v1, v2, v3, h[1], h[3]);
        mma_add(st.o[i][1], x0, x1, x2, x3, h[1], h[3]);
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

// Workspace: the ranges' partial results, then the scores (with weights only), in powers of two.
struct Work {
    float2* ml;                              // [splits][n_seq][n_heads]: maximum and sum
    float* o;                                // [splits][n_seq][n_heads][head_dim]
    float* scores;                           // [n_seq][n_heads][max_len]
    int32_t splits;
};

// Whether a sequence has something to attend to: 1; zeros in its output: 0; left alone: -1.
__device__ __forceinline__ int state_of(const rvq_cache4_attn_args& a, int64_t rows, int64_t pos) {
    if (rows < 0) return -1;
    const bool append = a.k.ptr != nullptr;
    return rows + append >= 1 && rows + append <= a.cache.max_len && pos >= 0 && (a.pos == nullptr || pos < a.table_len);
}

constexpr int kRowLoads = 4;                 // rows of a thread in add_weights
constexpr int kJoinRows = kRowLoads * kThreads;

// Whether a CTA, which has all rows and all heads of its kv head, adds the weights itself, in one go: 64 x 8 heads of 500 rows
// 31.5 -> 28.5 us.  Longer caches leave it to the second launch: of 4,096 rows 154 us, here 165.
__host__ __device__ __forceinline__ bool weights_here(const rvq_cache4_attn_args& a, int splits) {
    return splits == 1 && a.n_heads / a.cache.n_kv <= kHeads && a.cache.max_len <= kJoinRows;
}

// The weights of rows [first, first + kRowLoads * kThreads) below n: those from before (`was`; the appended row's: none)
// and the heads', in order; m and r: the heads' maxima and reciprocal sums (0: nothing seen).
__device__ __forceinline__ void old_weights(float (&was)[kRowLoads], const float* w, int64_t first, int64_t n, int64_t appended) {
#pragma unroll
    for (int u = 0; u < kRowLoads; ++u) {
        const int64_t row = first + u * kThreads + threadIdx.x;
        was[u] = row < n && row != appended ? __ldcg(w + row) : 0.f;
    }
}
__device__ __forceinline__ void add_weights(float (&was)[kRowLoads], float* w, const float* scores, int64_t max_len, int64_t first,
                                            int64_t n, int heads, const float* m, const float* r) {
#pragma unroll 4
    for (int h = 0; h < heads; ++h) {
#pragma unroll
        for (int u = 0; u < kRowLoads; ++u) {
            const int64_t row = first + u * kThreads + threadIdx.x;
            const float s = row < n ? __ldcg(scores + h * max_len + row) : 0.f;
            if (r[h] != 0.f) was[u] += exp2_approx(s - m[h]) * r[h];
        }
    }
#pragma unroll
    for (int u = 0; u < kRowLoads; ++u) {
        const int64_t row = first + u * kThreads + threadIdx.x;
        if (row < n) w[row] = was[u];
    }
}

template <int HD, bool kHalfQ>
__global__ void __launch_bounds__(kThreads, 2) cache4_attn_kernel(rvq_cache4_attn_args a, Work work) {
    constexpr int G = HD / kGroup, REC = record_bytes(HD);
    extern __shared__ __align__(128) uint8_t smem_raw[];
    Smem<HD>& S = *reinterpret_cast<Smem<HD>*>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int nkv = a.cache.n_kv, rep = a.n_heads / nkv;
    const int split = blockIdx.x, kv = blockIdx.y % nkv, group = blockIdx.y / nkv, b = blockIdx.z;
    pdl_wait();
    pdl_launch_dependents();                                 // after the wait: the join may read what this kernel does not write
    const int64_t rows = a.rows[b], pos = a.pos != nullptr ? a.pos[b] : 0;
    const bool append = a.k.ptr != nullptr;
    const int groups = (rep + kHeads - 1) / kHeads, per = (rep + groups - 1) / groups;
    const int h0 = group * per, heads = min(per, rep - h0);
    const int64_t head0 = (int64_t)b * a.n_heads + kv * rep + h0, q_at = head0 * HD;      // of all sequences' heads
    float qv[kHeads * HD / kThreads];                        // on their way while rows is
#pragma unroll
    for (int i = 0; i < kHeads * HD / kThreads; ++i)
        qv[i] = tid + i * kThreads < heads * HD ? vec_value_deep(a.q, q_at + tid + i * kThreads) : 0.f;
    const int state = state_of(a, rows, pos);
    if (state < 0) return;
    const int out_kind = a.q.kind == RVQ_F16 ? RVQ_F16 : RVQ_BF16;
    if (state == 0) {
        if (split == 0)
            for (int i = tid; i < heads * HD; i += kThreads) store_from_f32(a.out, q_at + i, out_kind, 0.f);
        return;
    }
    const int live = (int)rows, tiles = (live + kTile - 1) / kTile;
    const int t0 = (int)((int64_t)tiles * split / work.splits), t1 = (int)((int64_t)tiles * (split + 1) / work.splits);
    const bool owner = append && split == 0;                 // this CTA attends to the new row
    float2* ml = work.ml + ((int64_t)split * a.cache.n_seq * a.n_heads + head0);
    if (t0 == t1 && !owner) {                                // fewer tiles than ranges
        if (tid < heads) ml[tid] = make_float2(-INFINITY, 0.f);
        return;
    }
    uint8_t* cache = reinterpret_cast<uint8_t*>(a.cache.data) + ((int64_t)b * nkv + kv) * a.cache.max_len * REC;
    uint32_t shift;
    asm volatile("mov.u32 %0, 65536;" : "=r"(shift));
    // this lane's 16-byte pieces of tile number `tile`, into a stage of the warp's ring; a group for every stage, so that
    // the number of groups behind a tile is known
    const uint32_t ring = smem_addr(S.ring[warp][0]) + 16 * lane;
    auto fetch = [&](int tile, int stage) {
        if (tile < t1) {
            const uint8_t* src = cache + (int64_t)tile * (kTile * REC) + 16 * lane;
            const uint32_t dst = ring + stage * (kTile * REC);
            const int bytes = min(kTile, live - tile * kTile) * REC - 16 * lane;      // of live rows, from this lane's first piece on
            const bool full = (tile + 1) * kTile <= live;
#pragma unroll
            for (int i = 0; i < (kTile * REC + 511) / 512; ++i)
                if ((i + 1) * 512 <= kTile * REC || lane < kTile * REC % 512 / 16) {
                    if (full) copy16(dst + 512 * i, src + 512 * i, true);
                    else copy16(dst + 512 * i, bytes > 512 * i ? src + 512 * i : cache, bytes > 512 * i);
                }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    for (int i = 0; i < kStages - 1; ++i) fetch(t0 + warp + i * kWarps, i);

    // the heads' q, and the new record
    const bool rotate = a.q_norm != nullptr || a.cos != nullptr;
    if (rotate) {
        for (int i = tid; i < HD; i += kThreads) {
            S.norm[0][i] = a.q_norm != nullptr ? bf16_at(a.q_norm, i) : 0.f;
            S.norm[1][i] = a.q_norm != nullptr ? bf16_at(a.k_norm, i) : 0.f;
            S.norm[2][i] = a.cos != nullptr ? bf16_at(a.cos, pos * HD + i) : 0.f;
            S.norm[3][i] = a.cos != nullptr ? bf16_at(a.sin, pos * HD + i) : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < kHeads * HD / kThreads; ++i) (&S.q[0][0])[tid + i * kThreads] = qv[i];
    if (owner) {
        const int64_t kv_at = ((int64_t)b * nkv + kv) * HD;
        for (int i = tid; i < 2 * HD; i += kThreads) (&S.kv[0][0])[i] = vec_value_deep(i < HD ? a.k : a.v, kv_at + i % HD);
        for (int i = tid; i < kTile * REC / 4; i += kThreads) reinterpret_cast<uint32_t*>(S.fresh)[i] = 0;
    }
    __syncthreads();
    if (rotate) {
        norm_rope<HD>(S.q[warp], S.norm[0], a, S.norm[2], S.norm[3]);
        if (owner && warp == 0) norm_rope<HD>(S.kv[0], S.norm[1], a, S.norm[2], S.norm[3]);
    }
#pragma unroll
    for (int i = 0; i < G; ++i) {
        const float x = warp_sum(S.q[warp][kGroup * i + lane]);
        if (lane == 0) S.qsum[warp][i] = x;
    }
    if (owner && warp < 2)                                   // the warp that rotated the key, and another
        encode<HD>(S.kv[warp], S.fresh + warp * (HD / 2), reinterpret_cast<uint32_t*>(S.fresh + HD + warp * (HD / 8)));
    __syncthreads();
    if (owner && group == 0 && tid < REC / 16)
        reinterpret_cast<uint4*>(cache + rows * REC)[tid] = reinterpret_cast<const uint4*>(S.fresh)[tid];

    // column g of the operand: q of head g, in pairs in the code words' order; and (q . 1) of group t against the pairs
    // (zero, step), in three bf16 parts: 24 bits
    constexpr float kUnit = kHalfQ ? 512.f : 64.f;
    uint32_t qa[HD / 16][2], qz[3] = {0u, 0u, 0u};
    if (t < G) {
        const float x = S.qsum[g][t] * (1.f / kUnit);
        const float hi = bf16r(x), lo = bf16r(x - hi);
        qz[0] = pack_bf16(hi, 0.f), qz[1] = pack_bf16(lo, 0.f), qz[2] = pack_bf16(x - hi - lo, 0.f);
    }
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
        const float* q = &S.q[g][i / 2 * kGroup + 8 * t + 2 * (i & 1)];
        qa[i][0] = pack2(q[0], q[4], kHalfQ ? RVQ_F16 : RVQ_BF16);
        qa[i][1] = pack2(q[1], q[5], kHalfQ ? RVQ_F16 : RVQ_BF16);
    }
    State<HD> st;
    st.m[0] = st.m[1] = -INFINITY, st.l[0] = st.l[1] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) st.zero[i] = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) st.o[i][j][c] = 0.f;
    const float scale = a.scaling * kUnit * 1.4426950408889634f;       // scores in powers of two
    float* sc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        sc[i] = a.weights != nullptr && 2 * t + i < heads ? work.scores + (head0 + 2 * t + i) * a.cache.max_len : nullptr;
    // the warp whose turn it would be after the last tile takes the appended record, first
    bool extra = owner && warp == (t1 - t0) % kWarps;
    for (int tile = t0 + warp, stage = 0; tile < t1 || extra;) {
        uint32_t rec = smem_addr(S.fresh);
        int row = live, valid = 1;
        if (!extra) {
            asm volatile("cp.async.wait_group %0;\n" ::"n"(kStages - 2) : "memory");
            __syncwarp();                                    // every lane's pieces are here, and the stage before this one is read
            fetch(tile + (kStages - 1) * kWarps, stage == 0 ? kStages - 1 : stage - 1);
            rec = smem_addr(S.ring[warp][stage]);
            row = tile * kTile;
            valid = min(kTile, live - row);
            tile += kWarps;
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }
        extra = false;
        float* const at[2] = {sc[0] ? sc[0] + row : nullptr, sc[1] ? sc[1] + row : nullptr};
        tile_step<HD, kHalfQ>(rec, valid, qa, qz, scale, shift, st, a.weights != nullptr, at);
    }
    // the lanes with the same t hold parts of heads 2 t and 2 t + 1
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
        st.l[0] += __shfl_xor_sync(0xffffffffu, st.l[0], o);
        st.l[1] += __shfl_xor_sync(0xffffffffu, st.l[1], o);
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    __syncthreads();                                         // the rings are read: they take the warps' outputs
    float* wo = reinterpret_cast<float*>(S.ring);            // [kWarps][kHeads][HD]
#pragma unroll
    for (int i = 0; i < G; ++i) {
        // the sums with the group's zeros
        const float z0 = __shfl_sync(0xffffffffu, st.zero[0], 8 * i + t), z1 = __shfl_sync(0xffffffffu, st.zero[1], 8 * i + t);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float* d = wo + (warp * kHeads + 2 * t) * HD + kGroup * i + 4 * g + j;
            d[0] = fmaf(64.f, st.o[i][j >> 1][2 * (j & 1)], z0);
            d[HD] = fmaf(64.f, st.o[i][j >> 1][2 * (j & 1) + 1], z1);
        }
    }
    if (g < 2) S.wm[warp][2 * t + g] = g ? st.m[1] : st.m[0], S.wl[warp][2 * t + g] = g ? st.l[1] : st.l[0];
    __syncthreads();
    // warp w joins head w over the warps
    if (warp < heads) {
        float m = S.wm[0][warp];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) m = fmaxf(m, S.wm[w][warp]);
        float total = 0.f, o[HD / 32];
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) o[d] = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = S.wm[w][warp] == m ? 1.f : exp2_approx(S.wm[w][warp] - m);
            total = fmaf(f, S.wl[w][warp], total);
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) o[d] = fmaf(f, wo[(w * kHeads + warp) * HD + 32 * d + lane], o[d]);
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;  // no score above -infinity: zeros
        if (lane == 0) ml[warp] = make_float2(m, total), S.m[warp] = m, S.r[warp] = inv;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) {
            if (work.splits == 1)
                store_from_f32(a.out, q_at + warp * HD + 32 * d + lane, out_kind, inv == 0.f ? 0.f : o[d] * inv);
            else
                work.o[((int64_t)split * a.cache.n_seq * a.n_heads + head0 + warp) * HD + 32 * d + lane] = o[d];
        }
    }
    if (a.weights != nullptr && weights_here(a, work.splits)) {
        __syncthreads();
        float* w = a.weights + ((int64_t)b * nkv + kv) * a.cache.max_len;
        const int64_t n = live + (a.k.ptr != nullptr);
        float was[kRowLoads];
        old_weights(was, w, 0, n, a.k.ptr != nullptr ? live : -1);
        add_weights(was, w, work.scores + head0 * a.cache.max_len, a.cache.max_len, 0, n, heads, S.m, S.r);
    }
}

// The ranges joined.  Blocks x < out_blocks: 256 output values of the kv head's query heads each; the others: the weights of
// kJoinRows rows each, heads in order.
constexpr int kJoinThreads = kThreads;
constexpr int kMaxSplits = 320;              // plan keeps below it
constexpr int kEarly = 16;

// Maximum and sum of a head over the ranges, by one warp; with f, the ranges' factors (0 for an empty one).
__device__ __forceinline__ float2 join_head(const float2* ml, int64_t step, int splits, float* f) {
    constexpr int U = kMaxSplits / 32;
    const int lane = threadIdx.x & 31;
    float2 x[U];
    float m = -INFINITY, total = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int s = 32 * u + lane;
        x[u] = s < splits ? __ldcg(ml + s * step) : make_float2(-INFINITY, 0.f);
        m = fmaxf(m, x[u].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const float g = x[u].y == 0.f ? 0.f : x[u].x == m ? 1.f : exp2_approx(x[u].x - m);
        total = fmaf(g, x[u].y, total);
        if (f != nullptr && 32 * u + lane < splits) f[32 * u + lane] = g;
    }
    return make_float2(m, warp_sum(total));
}

__global__ void __launch_bounds__(kJoinThreads) cache4_join_kernel(rvq_cache4_attn_args a, Work work, int out_blocks) {
    constexpr int kBlockHeads = kJoinThreads / 64;           // heads that 256 output values may touch
    __shared__ float fm[kMaxRep], fr[kMaxRep], f[kBlockHeads][kMaxSplits];
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nkv = a.cache.n_kv, rep = a.n_heads / nkv, hd = a.cache.head_dim;
    const int kv = blockIdx.y, b = blockIdx.z;
    // the rows and the weights are not the first kernel's, and what came before is complete (it waited for that): these loads
    // run before its end
    const int64_t rows = __ldcg(a.rows + b), pos = a.pos != nullptr ? __ldcg(a.pos + b) : 0;
    const int64_t head0 = (int64_t)b * a.n_heads + kv * rep, all = (int64_t)a.cache.n_seq * a.n_heads;
    const bool append = a.k.ptr != nullptr;
    const int64_t n = rows + append, first = (int64_t)((int)blockIdx.x - out_blocks) * kJoinRows;
    const bool output = first < 0, used = state_of(a, rows, pos) == 1 && (output || first < n);
    float* w = a.weights + ((int64_t)b * nkv + kv) * a.cache.max_len;
    float was[kRowLoads];
    if (used && !output) old_weights(was, w, first, n, append ? rows : -1);
    pdl_wait();
    if (!used) return;
    // the first ranges' outputs come with their maxima and sums
    const int at = blockIdx.x * kJoinThreads + tid;
    const bool mine = output && at < rep * hd;
    const float* o = work.o + head0 * hd + at;
    float early[kEarly];
#pragma unroll
    for (int s = 0; s < kEarly; ++s) early[s] = mine && s < work.splits ? __ldcg(o + s * all * hd) : 0.f;
    const int h0 = output ? blockIdx.x * (kJoinThreads / hd) : 0, h1 = output ? min(rep, h0 + kJoinThreads / hd) : rep;
    for (int h = h0 + warp; h < h1; h += kJoinThreads / 32) {
        const float2 x = join_head(work.ml + head0 + h, all, work.splits, output ? f[h - h0] : nullptr);
        if (lane == 0) fm[h] = x.x, fr[h] = x.y == 0.f ? 0.f : 1.f / x.y;
    }
    __syncthreads();
    if (!output) {
        add_weights(was, w, work.scores + head0 * a.cache.max_len, a.cache.max_len, first, n, rep, fm, fr);
        return;
    }
    if (!mine) return;
    const int h = at / hd;
    const float* g = f[h - h0];
    float sum = 0.f;                                         // of an empty range: whatever is there
#pragma unroll
    for (int s = 0; s < kEarly; ++s) sum = s >= work.splits || g[s] == 0.f ? sum : fmaf(g[s], early[s], sum);
#pragma unroll 8
    for (int s = kEarly; s < work.splits; ++s) {
        const float v = __ldcg(o + s * all * hd);
        sum = g[s] == 0.f ? sum : fmaf(g[s], v, sum);
    }
    store_from_f32(a.out, head0 * hd + at, a.q.kind == RVQ_F16 ? RVQ_F16 : RVQ_BF16, fr[h] == 0.f ? 0.f : sum * fr[h]);
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
    if (a->rows == nullptr || a->out == nullptr) return RVQ_ERR_INVALID;
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
    if (c.n_seq > 65535 || a->n_heads > 65535 || c.max_len > (1 << 30)) return RVQ_ERR_TOO_LARGE;
    return RVQ_OK;
}

// Ranges of the rows: as many CTAs as the SMs hold (two each), and two ranges where that is between one and two (160 heads
// of 4,096 rows: 45 us whole, 40 us halved; of mixed lengths 38 and 26), but none shorter than a tile for every warp of a
// full cache.  Above that a range is a whole sequence: halves cost 64 x 8 heads of 4,096 rows 113 -> 120 us.
// A short cache is one range, which needs no second launch: 8 heads, 300 rows 9.1 -> 7.5 us, 600 rows 9.7 -> 9.5, 750 rows
// 9.3 -> 10.4; with weights 300 rows 9.5 -> 9.0, 500 rows 10.1 -> 10.9.  The limits go by one sequence.  Many have more to lose by a
// second launch, and at the limits' far side one range would still pay: 8 sequences x 8 heads of 512 rows 12.3 -> 9.9 us, but of 768
// rows (two launches) 13.0 against 11.6 in one; 32 sequences of 1,024 rows 29.7 against 20.0.  The rule goes by the cache's length, as
// the host does not know the rows: 300 rows in a cache of 8,192 take 13.4 us.
int plan(const rvq_cache4_attn_args& a, int* splits) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return status(e);
    const int rep = a.n_heads / a.cache.n_kv, groups = (rep + kHeads - 1) / kHeads;
    const int64_t units = (int64_t)a.cache.n_seq * a.cache.n_kv * groups;
    const int64_t most = units > sms && units < 2 * sms ? 2 : 2 * sms / units, parts = (a.cache.max_len + kWarps * kTile - 1) / (kWarps * kTile);
    const bool alone = parts <= (a.weights == nullptr ? 5 : groups == 1 ? 3 : 0);
    const int64_t s = alone ? 1 : most < parts ? most : parts;
    *splits = s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : (int)s;
    return RVQ_OK;
}

// Bytes of the workspace's parts: maxima and sums, outputs, scores.
void sizes(const rvq_cache4_attn_args& a, int splits, size_t (&n)[3]) {
    const size_t heads = (size_t)a.cache.n_seq * a.n_heads;
    n[0] = (heads * splits * sizeof(float2) + 15) / 16 * 16;
    n[1] = splits > 1 ? heads * splits * a.cache.head_dim * sizeof(float) : 0;
    n[2] = a.weights != nullptr ? heads * a.cache.max_len * sizeof(float) : 0;
}

template <int HD, bool kHalfQ>
int run(const rvq_cache4_attn_args& a, const Work& work, cudaStream_t s) {
    auto* kernel = cache4_attn_kernel<HD, kHalfQ>;
    const int smem = (int)sizeof(Smem<HD>), rep = a.n_heads / a.cache.n_kv, groups = (rep + kHeads - 1) / kHeads;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess)
        e = launch_pdl(kernel, dim3(work.splits, a.cache.n_kv * groups, a.cache.n_seq), dim3(kThreads), (size_t)smem, s, a, work);
    const int out_blocks = work.splits > 1 ? (rep * HD + kJoinThreads - 1) / kJoinThreads : 0;
    const int row_blocks = a.weights != nullptr && !weights_here(a, work.splits) ? (a.cache.max_len + kJoinRows - 1) / kJoinRows : 0;
    if (e == cudaSuccess && out_blocks + row_blocks > 0)
        e = launch_pdl(cache4_join_kernel, dim3(out_blocks + row_blocks, a.cache.n_kv, a.cache.n_seq), dim3(kJoinThreads), 0, s, a,
                       work, out_blocks);
    return status(e);
}

}  // namespace cache4
}  // namespace rvq

using namespace rvq;
using namespace rvq::cache4;

extern "C" size_t rvq_cache4_attention_workspace_size(const rvq_cache4_attn_args* a) {
    int splits = 1;
    if (check(a) != RVQ_OK || plan(*a, &splits) != RVQ_OK) return 0;
    size_t n[3];
    sizes(*a, splits, n);
    return n[0] + n[1] + n[2];
}

extern "C" int rvq_cache4_attention(const rvq_cache4_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check(a);
    if (rc != RVQ_OK) return rc;
    Work work;
    rc = plan(*a, &work.splits);
    if (rc != RVQ_OK) return rc;
    size_t n[3];
    sizes(*a, work.splits, n);
    if (workspace == nullptr || workspace_bytes < n[0] + n[1] + n[2] || ((uintptr_t)workspace & 15)) return RVQ_ERR_INVALID;
    uint8_t* p = reinterpret_cast<uint8_t*>(workspace);
    work.ml = reinterpret_cast<float2*>(p);
    work.o = reinterpret_cast<float*>(p + n[0]);
    work.scores = reinterpret_cast<float*>(p + n[0] + n[1]);
    cudaStream_t s = (cudaStream_t)stream;
    const bool split = a->q.kind == RVQ_F16;
    if (a->cache.head_dim == 128) return split ? run<128, true>(*a, work, s) : run<128, false>(*a, work, s);
    return split ? run<64, true>(*a, work, s) : run<64, false>(*a, work, s);
}
