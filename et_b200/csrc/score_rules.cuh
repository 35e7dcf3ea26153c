// Attention with rules on its scores: what its kernels share. A score is kept in the log2 domain (everything times log2 e), so that
// a weight is one 2^x. Capped: c tanh(s / c) = c - 2 c / (1 + 2^(2 log2(e) s / c)), one exponential and a reciprocal; of a large
// score the power is infinite or 0 and the result +-c. (Absolute error some 1e-7 c: the error of a weight relative to it.)
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include "vec_math.cuh"

namespace et {

constexpr float kRulesLog2e = 1.4426950408889634f;
constexpr int kNoLimit = 1 << 30;   // a window without a limit; positions are below it

struct RuleParams {
    half* out;
    const half *q, *k, *v;
    long long out_pitch, q_pitch, k_pitch, v_pitch;
    int nhead, group, head_dim;            // group: query heads to a K/V head
    const int *cu_seqlens, *k_start, *k_lens;
    int batch, q_tokens, k_rows, max_q_len, max_k_len;
    float scale_log2;                      // score -> log2 domain
    float cap_in, cap_out;                 // 2 log2(e) scale / cap and cap log2(e); cap_out 0: not capped
    float to_y, cap_near;                  // capped: score -> score / cap, and the largest score for which cap_near2 is taken
    bool cap_wide;                         // a cap above kWideCap
    const float* slopes;
    const half* table;                     // [nhead][2 reach + 1]
    int reach, window_left, window_right;  // windows: kNoLimit without one
    const int *prefix_lens, *q_docs, *k_docs;
};

__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// c tanh(y) = c y P(y^2), y = s / c, of two scores whose size is at most kCapNear caps: P the polynomial of degree 4 with the smallest relative error for tanh(y) / y up to
// there (by the exchange of extremes; 2.8e-8 with its coefficients as they stand here, beside some 2e-7 that fp32 products and sums lose): no exponential, no reciprocal.
// to_out: score -> log2 domain.
constexpr float kCapNear = 0.5f;
__device__ __forceinline__ void cap_near2(float& a, float& b, float to_y, float to_out) {
    const float2 s = make_float2(a, b), y = mul2(s, make_float2(to_y, to_y)), t = mul2(y, y);
    auto both = [](float x) { return make_float2(x, x); };
    float2 p = fma2(both(0.017135007306933403f), t, both(-0.05298607423901558f));
    p = fma2(p, t, both(0.13324779272079468f));
    p = fma2(p, t, both(-0.3333306908607483f));
    p = fma2(p, t, both(1.f));
    const float2 out = mul2(mul2(s, make_float2(to_out, to_out)), p);
    a = out.x;
    b = out.y;
}
// Caps above kWideCap: c - 2 c / (1 + 2^x) would be off by more than a fraction of a weight's half step in fp16 (4.9e-4): 1e-4 there, everything at 1e7. Each score
// by the polynomial where it is within half a cap; beyond, that error is one of the score's own size. (A kernel of its own, as
// the choice for each score costs more than one for all: single tokens, 64 x 8192 keys, 97 us with both in one kernel, 94 so.)
constexpr float kWideCap = 512.f;
__device__ __forceinline__ void cap_wide2(float& a, float& b, const RuleParams& p) {
    float x = a, y = b;
    cap_near2(x, y, p.to_y, p.scale_log2);
    a = fabsf(a) <= p.cap_near ? x : fmaf(rcp_fast(1.f + ex2_fast(a * p.cap_in)), -2.f * p.cap_out, p.cap_out);
    b = fabsf(b) <= p.cap_near ? y : fmaf(rcp_fast(1.f + ex2_fast(b * p.cap_in)), -2.f * p.cap_out, p.cap_out);
}

// Where a sequence's queries and keys are.
struct RuleSeq {
    int q0, qlen;
    int k0, klen;      // rows of K and V; keys that may be seen
    int qpos0;         // position of the first query among the keys
    int prefix;
};

__device__ __forceinline__ RuleSeq rule_seq(const RuleParams& p, int b) {
    RuleSeq s;
    if (p.cu_seqlens) {
        s.q0 = p.cu_seqlens[b];
        s.qlen = p.cu_seqlens[b + 1] - s.q0;
    } else {
        s.q0 = b * p.max_q_len;
        s.qlen = p.max_q_len;
    }
    s.qlen = max(0, min(s.qlen, min(p.max_q_len, p.q_tokens - s.q0)));
    if (s.q0 < 0) s.qlen = 0;
    if (p.k_start) {
        s.k0 = p.k_start[b];
        s.klen = max(0, min(p.k_lens[b], kNoLimit));
        s.qpos0 = s.klen - s.qlen;
    } else {
        s.k0 = s.q0;
        s.klen = p.k_lens ? max(0, min(p.k_lens[b], s.qlen)) : s.qlen;
        s.qpos0 = 0;
    }
    s.klen = s.k0 < 0 ? 0 : max(0, min(min(s.klen, p.max_k_len), p.k_rows - s.k0));
    s.prefix = p.prefix_lens ? p.prefix_lens[b] : 0;
    return s;
}

// One query of one head by one warp, for any head width up to 256 and any alignment: a key to a lane for the scores, features to the lanes for
// the sum of V. Scores and sums in fp32. What is not seen is not read into any sum.
static __device__ __noinline__ void rules_row(const RuleParams& p, const RuleSeq& s, int i, int h) {
    const int lane = threadIdx.x & 31, hd = p.head_dim;
    const half* const q = p.q + (s.q0 + i) * p.q_pitch + (size_t)h * hd;
    const half* const k = p.k + s.k0 * p.k_pitch + (size_t)(h / p.group) * hd;
    const half* const v = p.v + s.k0 * p.v_pitch + (size_t)(h / p.group) * hd;
    const int qpos = s.qpos0 + i;
    const int lo = p.window_left == kNoLimit ? 0 : qpos - p.window_left, hi = p.window_right == kNoLimit ? kNoLimit : qpos + p.window_right;
    const int doc = p.q_docs ? p.q_docs[s.q0 + i] : 0;
    const float slope = p.slopes ? p.slopes[h] * kRulesLog2e : 0.f;
    const half* const table = p.table ? p.table + (size_t)h * (2 * p.reach + 1) + p.reach : nullptr;
    const bool vec = hd % 8 == 0 && ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k)) & 15) == 0 && (p.q_pitch | p.k_pitch) % 8 == 0;
    float top = -INFINITY, sum = 0.f, o[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c] = 0.f;
    const int end = doc < 0 ? 0 : min(s.klen, max(hi == kNoLimit ? hi : hi + 1, s.prefix));
    const int begin = s.prefix > 0 ? 0 : max(lo, 0) & ~31;
    for (int j0 = begin; j0 < end; j0 += 32) {
        const int j = j0 + lane;
        const bool seen = j < end && ((j >= lo && j <= hi) || j < s.prefix) && (!p.k_docs || p.k_docs[s.k0 + j] == doc);
        const unsigned any = __ballot_sync(0xffffffffu, seen);
        if (!any) continue;
        float score = -INFINITY;
        if (seen) {
            const half* const kr = k + j * p.k_pitch;
            float dot = 0.f;
            if (vec) {
                for (int d = 0; d < hd; d += 8) {
                    const uint4 a = *reinterpret_cast<const uint4*>(q + d), b = *reinterpret_cast<const uint4*>(kr + d);
                    const half2 *ah = reinterpret_cast<const half2*>(&a), *bh = reinterpret_cast<const half2*>(&b);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 x = __half22float2(ah[e]), y = __half22float2(bh[e]);
                        dot = fmaf(x.y, y.y, fmaf(x.x, y.x, dot));
                    }
                }
            } else {
                for (int d = 0; d < hd; ++d) dot = fmaf(__half2float(q[d]), __half2float(kr[d]), dot);
            }
            if (p.cap_wide) {
                float none = 0.f;
                cap_wide2(dot, none, p);
                score = dot;
            } else {
                score = p.cap_out > 0.f ? p.cap_out - 2.f * p.cap_out / (1.f + exp2f(dot * p.cap_in)) : dot * p.scale_log2;
            }
            const int away = j - qpos;
            if (p.slopes) score -= slope * fabsf((float)away);
            if (table) score = fmaf(__half2float(table[max(-p.reach, min(p.reach, away))]), kRulesLog2e, score);
        }
        // (a score that is not a number makes the row not a number: the maximum leaves it out, the weight below does not)
        float m = score;
#pragma unroll
        for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
        m = fmaxf(m, top);
        const float shift = m == -INFINITY ? 0.f : m;
        const float w = seen ? exp2f(score - shift) : 0.f, keep = top == -INFINITY ? 0.f : exp2f(top - shift);
        top = m;
        sum = sum * keep + w;   // each lane its own keys'
        if (__any_sync(0xffffffffu, w != w)) {   // so is the whole row, whatever follows
#pragma unroll
            for (int c = 0; c < 8; ++c) o[c] = NAN;
            sum = 1.f;
            break;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) o[c] *= keep;
        for (unsigned left = any; left; left &= left - 1) {
            const int from = __ffs(left) - 1;
            const float weight = __shfl_sync(0xffffffffu, w, from);
            const half* const vr = v + (j0 + from) * p.v_pitch;
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (c * 32 + lane < hd) o[c] = fmaf(weight, __half2float(vr[c * 32 + lane]), o[c]);
        }
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    half* const out = p.out + (s.q0 + i) * p.out_pitch + (size_t)h * hd;
#pragma unroll
    for (int c = 0; c < 8; ++c)
        if (c * 32 + lane < hd) out[c * 32 + lane] = __float2half_rn(sum == 0.f ? 0.f : o[c] / sum);
}

}  // namespace et
