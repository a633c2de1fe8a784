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
using sm100::smem_addr;

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
    float m[kHeads], l[kHeads];              // this CTA's maximum and sum
    float fm[kHeads], fr[kHeads];            // the final maximum and 1 / sum
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

// Numbers of a parameter word: the shift as a multiplication (`shift` holds 65536 where the compiler cannot see it), which
// runs on the FMA pipe; the masks and shifts of this kernel's integer pipe are what bounds it.
__device__ __forceinline__ float zero_by(uint32_t p, uint32_t shift) {
    uint32_t r;
    asm("mul.lo.u32 %0, %1, %2;" : "=r"(r) : "r"(p), "r"(shift));
    return __uint_as_float(r);
}

// D += A B, and D = A B
__device__ __forceinline__ void mma_add(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_set(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};\n"
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

// What a warp carries over its tiles.  Lane 4 g + t: head g's maximum and this lane's part of its sum; of the sums of
// p zero and p step, those of group t for head g (and the parts from p's remainder); and of the output, transposed: heads
// 2 t and 2 t + 1, value 4 g + i of group G in o[G][i / 2][2 (i & 1) + (0, 1)].
template <int HD>
struct State {
    static constexpr int G = HD / kGroup;
    float m, l;
    float zero[4];
    float o[G][2][4];
};

template <int G>
__device__ __forceinline__ void load_words(uint32_t (&w)[G], uint32_t addr) {
    if constexpr (G == 4)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
    else
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
}

// A tile of 16 rows, `valid` of them live (the records behind those hold zeros).
template <int HD, bool kSplitQ>
__device__ __forceinline__ void tile_step(uint32_t base, int valid, const uint32_t (&qa)[HD / 16][kSplitQ ? 4 : 2],
                                          const uint32_t (&qz)[3], float scale64, uint32_t shift, State<HD>& st,
                                          float* scores) {
    constexpr int G = HD / kGroup, REC = record_bytes(HD), kLo = kSplitQ ? 2 : 0;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // columns n of a score tile hold row (n with its two low bits swapped): a quarter warp's 16-byte loads of two
    // rows then fall into different banks, and this lane's columns 2 t and 2 t + 1 are rows ra and ra + 2
    const int rn = (g & 4) | (g & 1) << 1 | (g >> 1 & 1);
    const int ra = (t >> 1) * 4 + (t & 1);
    float s[4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const uint32_t rk = base + (8 * n + rn) * REC, r0 = base + (8 * n + ra) * REC + HD;
        uint32_t kc[G], pa[G], pb[G], pz;
        load_words<G>(kc, rk + 4 * G * t);
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(pz) : "r"(rk + HD + 4 * (t & (G - 1))));
        load_words<G>(pa, r0);
        load_words<G>(pb, r0 + 2 * REC);
        float z[4], c[G][4];                                 // zero . (q . 1) / 64; q . c / 64 of every group
        mma_set(z, qz[0], qz[2], qz[1], 0u, pz, pz);
#pragma unroll
        for (int i = 0; i < G; ++i)
            mma_set(c[i], qa[2 * i][0], kSplitQ ? qa[2 * i][kLo] : 0u, qa[2 * i][1], kSplitQ ? qa[2 * i][kLo + 1] : 0u,
                    code_pair<0>(kc[i]), code_pair<1>(kc[i]));
#pragma unroll
        for (int i = 0; i < G; ++i)
            mma_add(c[i], qa[2 * i + 1][0], kSplitQ ? qa[2 * i + 1][kLo] : 0u, qa[2 * i + 1][1],
                    kSplitQ ? qa[2 * i + 1][kLo + 1] : 0u, code_pair<0>(kc[i] >> 8), code_pair<1>(kc[i] >> 8));
        float sa = z[0] + z[2], sb = z[1] + z[3];
#pragma unroll
        for (int i = 0; i < G; ++i) {
            if constexpr (kSplitQ) c[i][0] += c[i][2], c[i][1] += c[i][3];
            sa = fmaf(step_of(pa[i]), c[i][0], sa);
            sb = fmaf(step_of(pb[i]), c[i][1], sb);
        }
        s[2 * n] = sa * scale64;
        s[2 * n + 1] = sb * scale64;
    }
    if (valid < 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (8 * (i >> 1) + ra + 2 * (i & 1) >= valid) s[i] = -INFINITY;
    }
    if (scores != nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 8 * (i >> 1) + ra + 2 * (i & 1);
            if (row < valid) scores[row] = s[i];
        }
    }
    float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    // the maximum that is subtracted follows the true one only when that has grown by 2^8 (p stays below 2^8): of 32
    // rows and heads some has a new maximum in most tiles, and following it at once costs a fifth of the loop
    if (__any_sync(0xffffffffu, top > st.m + kGrow)) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float m = fmaxf(st.m, top);
        const float f = st.m == m ? 1.f : exp2_approx(st.m - m);
        st.m = m;
        st.l *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) st.zero[i] *= f;
        const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                st.o[i][j][0] *= f0, st.o[i][j][2] *= f0;
                st.o[i][j][1] *= f1, st.o[i][j][3] *= f1;
            }
    }
    // nothing but -infinities so far: p = exp(-infinity) = 0, not exp(-infinity + infinity)
    const float sub = st.m == -INFINITY ? 0.f : st.m;
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = exp2_approx(s[i] - sub);
    st.l += (p[0] + p[1]) + (p[2] + p[3]);
    uint32_t vc[4][G], vp[4][G], h[4], zs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t r = base + (8 * (i >> 1) + ra + 2 * (i & 1)) * REC + HD / 2;
        load_words<G>(vc[i], r + 4 * G * (g >> 1));
        load_words<G>(vp[i], r + HD / 2 + HD / 8);
        asm volatile("ld.shared.u16 %0, [%1];" : "=r"(zs[i]) : "r"(r + HD / 2 + HD / 8 + 2 * (g & (2 * G - 1))));
    }
    // sums of p zero (columns 2 group) and p step (2 group + 1)
    split_bf16(p[0], p[1], &h[0], &h[1], shift);
    split_bf16(p[2], p[3], &h[2], &h[3], shift);
    mma_add(st.zero, h[0], h[1], h[2], h[3], __byte_perm(zs[0], zs[1], 0x5410u), __byte_perm(zs[2], zs[3], 0x5410u));
    const uint32_t half_sel = g & 1 ? 0x7632u : 0x5410u;     // this lane's 4 values are half a code word
#pragma unroll
    for (int i = 0; i < G; ++i) {
        split_bf16(p[0] * step_of(vp[0][i]), p[1] * step_of(vp[1][i]), &h[0], &h[1], shift);
        split_bf16(p[2] * step_of(vp[2][i]), p[3] * step_of(vp[3][i]), &h[2], &h[3], shift);
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

template <int HD, bool kSplitQ>
__global__ void __launch_bounds__(kThreads, 2) cache4_attn_kernel(rvq_cache4_attn_args a, int passes) {
    constexpr int G = HD / kGroup, REC = record_bytes(HD);
    extern __shared__ __align__(128) uint8_t smem_raw[];
    Smem<HD>& S = *reinterpret_cast<Smem<HD>*>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int nkv = a.cache.n_kv, rep = a.n_heads / nkv;
    const int kv = blockIdx.y % nkv, b = blockIdx.z;
    pdl_launch_dependents();
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

    uint32_t shift;
    asm volatile("mov.u32 %0, 65536;" : "=r"(shift));
    const int live = (int)rows;
    // this lane's 16-byte pieces of tile number `tile`, into a stage of the warp's ring; a group for every stage, so that
    // the number of groups behind a tile is known
    const uint32_t ring = smem_addr(S.ring[warp][0]) + 16 * lane;
    auto fetch = [&](int tile, int stage) {
        if (tile < t1) {
            const uint8_t* src = cache + (int64_t)tile * (kTile * REC) + 16 * lane;
            const int bytes = (live - tile * kTile) * REC - 16 * lane;
#pragma unroll
            for (int i = 0; i < (kTile * REC + 511) / 512; ++i)
                if ((i + 1) * 512 <= kTile * REC || lane < kTile * REC % 512 / 16)
                    copy16(ring + stage * (kTile * REC) + 512 * i, bytes > 512 * i ? src + 512 * i : cache, bytes > 512 * i);
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };

    for (int pass = 0; pass < passes; ++pass) {
        const int h0 = (first + pass) * per, heads = min(per, rep - h0);
        const int64_t q_at = ((int64_t)b * a.n_heads + kv * rep + h0) * HD;
        for (int i = 0; i < kStages - 1; ++i) fetch(t0 + warp + i * kWarps, i);

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
        if (owner && pass == 0 && warp < 2)                  // the warp that rotated the key, and another
            encode<HD>(S.kv[warp], S.fresh + warp * (HD / 2), reinterpret_cast<uint32_t*>(S.fresh + HD + warp * (HD / 8)));
        __syncthreads();
        if (owner && pass == 0 && first == 0 && tid < REC / 16)
            reinterpret_cast<uint4*>(cache + rows * REC)[tid] = reinterpret_cast<const uint4*>(S.fresh)[tid];

        // operand rows 0..7: q (its bf16 part), rows 8..15: the remainder; column pairs in the code words' order
        uint32_t qa[HD / 16][kSplitQ ? 4 : 2];
        // (q . 1) / 64 of group t against the pairs (zero, step), in three bf16 parts: 24 bits
        uint32_t qz[3] = {0u, 0u, 0u};
        if (t < G) {
            const float x = S.qsum[g][t] * 0.015625f;
            const float hi = bf16r(x), lo = bf16r(x - hi);
            qz[0] = pack_bf16(hi, 0.f), qz[1] = pack_bf16(lo, 0.f), qz[2] = pack_bf16(x - hi - lo, 0.f);
        }
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            const float* q = &S.q[g][i / 2 * kGroup + 8 * t + 2 * (i & 1)];
            if constexpr (kSplitQ) {
                split_bf16(q[0], q[4], &qa[i][0], &qa[i][2], 65536u);
                split_bf16(q[1], q[5], &qa[i][1], &qa[i][3], 65536u);
            } else {
                qa[i][0] = pack_bf16(q[0], q[4]);
                qa[i][1] = pack_bf16(q[1], q[5]);
            }
        }
        State<HD> st;
        st.m = -INFINITY, st.l = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) st.zero[i] = 0.f;
#pragma unroll
        for (int i = 0; i < G; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) st.o[i][j][c] = 0.f;
        }
        const float scale64 = a.scaling * 64.f * 1.4426950408889634f;      // scores in powers of two
        float* sc = a.weights != nullptr && g < heads
                        ? a.scores + ((int64_t)b * a.n_heads + kv * rep + h0 + g) * a.cache.max_len : nullptr;
        // the last warp begins with the appended record
        bool extra = owner && warp == kWarps - 1;
        for (int tile = t0 + warp, stage = 0; tile < t1 || extra;) {
            uint32_t rec = smem_addr(S.fresh);
            int row = live, valid = 1;
            if (!extra) {
                asm volatile("cp.async.wait_group %0;\n" ::"n"(kStages - 2) : "memory");
                __syncwarp();                                // every lane's pieces are here, and the stage before this one is read
                fetch(tile + (kStages - 1) * kWarps, stage == 0 ? kStages - 1 : stage - 1);
                rec = smem_addr(S.ring[warp][stage]);
                row = tile * kTile;
                valid = min(kTile, live - row);
                tile += kWarps;
                stage = stage + 1 == kStages ? 0 : stage + 1;
            }
            extra = false;
            tile_step<HD, kSplitQ>(rec, valid, qa, qz, scale64, shift, st, sc ? sc + row : sc);
        }
        // lanes 4 g .. 4 g + 3 hold parts of head g's sums
        float l = st.l;
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const float zero = st.zero[0] + st.zero[2];          // head g, group t
        __syncthreads();                                     // the rings are read: they take the warps' outputs
        float* wo = reinterpret_cast<float*>(S.ring);        // [kWarps][kHeads][HD], then the CTA's [kHeads][HD]
        float* co = wo + kWarps * kHeads * HD;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            // the zeros' sums of heads 2 t and 2 t + 1
            const float z0 = __shfl_sync(0xffffffffu, zero, 8 * t + i), z1 = __shfl_sync(0xffffffffu, zero, 8 * t + 4 + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float* d = wo + (warp * kHeads + 2 * t) * HD + kGroup * i + 4 * g + j;
                d[0] = fmaf(64.f, st.o[i][j >> 1][2 * (j & 1)], z0);
                d[HD] = fmaf(64.f, st.o[i][j >> 1][2 * (j & 1) + 1], z1);
            }
        }
        if (t == 0) S.wm[warp][g] = st.m, S.wl[warp][g] = l;
        __syncthreads();
        {
            // warp w joins head w over the warps
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
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) co[warp * HD + 32 * d + lane] = o[d];
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
        cluster.sync();                                      // the others have read this CTA's parts: the rings may be filled again
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
    while (c < 16 && units * c * 2 <= 2 * sms && (int64_t)c * kWarps * kTile < a.cache.max_len) c *= 2;
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
