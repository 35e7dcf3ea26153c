// Attention with rules on its scores for single tokens over keys kept from before (and for the few queries of short calls): bound by reading K and V once.
//
// The query heads that share a K/V head (and the queries of a sequence, if there are a few) are the rows of one m16n8k16 tile, so that keys and values are read
// once for all of them. A cluster of CTAs shares the keys of a sequence and K/V head: its warps take blocks of 16 keys in turn, each through a ring
// of its own in shared memory, filled by TMA (a warp waits for nobody else), with a running maximum and sum of its own. At the end the
// warps' sums are joined in shared memory and the CTAs' through distributed shared memory, in a fixed order: one launch, no workspace, the same bits every time.
// With copies of 16 bytes a lane, their addresses and a mask for every score a block took 1170 instructions, and 64 requests of up to 8192 keys (16 heads of 128
// over 4) 299 us.
//
// Scores, maxima and sums are fp32; the weights go to the second product as fp16 (half a step of 2^-11 of a weight), relative to a reference that moves when
// the maximum has grown by more than 2^8. V behind the last key is cleared in shared memory. A row whose result is not finite
// is computed again from the keys that it sees (rules_row), as not a number times the weight 0 is not a number.
#include <cooperative_groups.h>
#include "attention.h"
#include "attention_rules.h"
#include "common.h"
#include "ptx.cuh"
#include "tmap.h"

namespace cg = cooperative_groups;

namespace et {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kKeys = 16;                 // of a block
constexpr int kRows = 16;                 // of a tile
constexpr int kMaxCluster = 16;
constexpr float kRescaleStep = 8.f;       // log2 units

template <int kHD>
struct Cfg {
    static constexpr int kPanels = kHD / 64;                     // of 64 features: rows of 128 bytes, granule c of row r at c ^ (r & 7), as TMA swizzles them
    static constexpr int kPanel = kKeys * 128;
    static constexpr int kTile = kPanels * kPanel;               // a block of K or of V
    static constexpr int kStages = kHD == 64 ? 6 : 3;
    static constexpr int kRing = kStages * 2 * kTile;            // of a warp
    static constexpr int kSumAt = kWarps * kRing;                // this CTA's rows: [kRows][kHD] floats, then maxima and sums
    static constexpr int kBarAt = kSumAt + kRows * kHD * 4 + 2 * kRows * 4;
    static constexpr int kBytes = kBarAt + kWarps * kStages * 8 + 1024;
    static_assert(kWarps * (kRows * kHD + 2 * kRows) * 4 <= kSumAt, "the warps' sums fit where their rings were");
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// kHD: 64 or 128, the head's width rounded up. kTall: more than eight rows; otherwise the lower half of the tile is empty and left out of everything but the products.
// kWide: a cap above kWideCap.
template <int kHD, bool kTall, bool kWide>
__global__ void __launch_bounds__(kThreads) attention_rules_token_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                                                                         const __grid_constant__ RuleParams p, int row_tiles, bool longest_first, int* err) {
    using C = Cfg<kHD>;
    constexpr int kX = kTall ? 2 : 1;     // rows of a lane: g and g + 8
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t smem_at = smem_u32(smem);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    cg::cluster_group cluster = cg::this_cluster();
    const int csize = cluster.num_blocks(), crank = cluster.block_rank();
    const int hd = p.head_dim, steps = hd >> 4;
    int unit = blockIdx.x / csize;        // sequence, K/V head, tile of rows
    const int tile = unit % row_tiles;
    unit /= row_tiles;
    const int n_kv = p.nhead / p.group, kv_head = unit % n_kv;
    int b = unit / n_kv;
    const uint32_t ring = smem_at + warp * C::kRing, bars = smem_at + C::kBarAt + warp * C::kStages * 8;
    if (lane == 0) {
        for (int i = 0; i < C::kStages; ++i) mbar_init(reinterpret_cast<uint64_t*>(smem + C::kBarAt) + warp * C::kStages + i, 1);
        fence_mbar_init();
    }
    __syncwarp();
    pdl_launch_dependents();
    pdl_wait();
    if (longest_first) {   // the b-th sequence in order of length: the one that has b longer (or as long and earlier) ones
        __shared__ int lens[kThreads], found;
        const int i = threadIdx.x, len = i < p.batch ? p.k_lens[i] : 0;
        lens[i] = len;
        __syncthreads();
        int before = 0;
        for (int j = 0; j < p.batch; ++j) before += lens[j] > len || (lens[j] == len && j < i) ? 1 : 0;
        if (i < p.batch && before == b) found = i;
        __syncthreads();
        b = found;
    }
    const RuleSeq s = rule_seq(p, b);
    const int rows = min(s.qlen * p.group - tile * kRows, kRows);
    if (rows <= 0) return;                // the same for the whole cluster
    // blocks of keys that some row sees: of the prefix, then of the window
    const int qa = s.qpos0 + tile * kRows / p.group, qb = s.qpos0 + (tile * kRows + rows - 1) / p.group;
    const int pre = max(0, min(s.prefix, s.klen));
    const int n_prefix = (pre + kKeys - 1) / kKeys;
    const int lo = p.window_left == kNoLimit ? 0 : max(qa - p.window_left, 0), hi = p.window_right == kNoLimit ? s.klen - 1 : min(qb + p.window_right, s.klen - 1);
    const int first = max(lo / kKeys, n_prefix);
    const int n_blocks = n_prefix + (hi >= lo ? max(hi / kKeys - first + 1, 0) : 0);
    auto key_of = [&](int i) { return (i < n_prefix ? i : first + i - n_prefix) * kKeys; };
    const int stride = csize * kWarps, mine = crank * kWarps + warp;
    auto fetch = [&](int i, int stage) {
        if (lane == 0 && i < n_blocks) {
            const int row = s.k0 + key_of(i);
            const uint32_t to = ring + stage * 2 * C::kTile, bar = bars + stage * 8;
            mbar_expect_tx_at(bar, 2 * C::kTile);
#pragma unroll
            for (int c = 0; c < C::kPanels; ++c) tma_load_3d_at(to + c * C::kPanel, &tmK, c * 64, kv_head, row, bar);
#pragma unroll
            for (int c = 0; c < C::kPanels; ++c) tma_load_3d_at(to + C::kTile + c * C::kPanel, &tmV, c * 64, kv_head, row, bar);
        }
    };
#pragma unroll
    for (int n = 0; n < C::kStages - 1; ++n) fetch(mine + n * stride, n);
    // the lane's rows: query, head, position
    int qi[kX], head[kX], qpos[kX], doc[kX];
    float slope[kX];
    const half* table[kX];
    bool real[kX];
#pragma unroll
    for (int x = 0; x < kX; ++x) {
        real[x] = g + 8 * x < rows;
        const int r = tile * kRows + (real[x] ? g + 8 * x : 0);
        qi[x] = r / p.group;
        head[x] = kv_head * p.group + r % p.group;
        qpos[x] = s.qpos0 + qi[x];
        doc[x] = p.q_docs ? p.q_docs[s.q0 + qi[x]] : 0;
        slope[x] = p.slopes ? -p.slopes[head[x]] * kRulesLog2e : 0.f;
        table[x] = p.table + (size_t)head[x] * (2 * p.reach + 1) + p.reach;
    }
    uint32_t qf[kHD / 16][2 * kX];
#pragma unroll
    for (int k = 0; k < kHD / 16; ++k)
#pragma unroll
        for (int x = 0; x < kX; ++x) {
            const half* const q = p.q + (s.q0 + qi[x]) * p.q_pitch + head[x] * hd + k * 16 + 2 * t;
            qf[k][2 * x] = k < steps && real[x] ? *reinterpret_cast<const uint32_t*>(q) : 0u;
            qf[k][2 * x + 1] = k < steps && real[x] ? *reinterpret_cast<const uint32_t*>(q + 8) : 0u;
        }
    float o[kHD / 8][4];
#pragma unroll
    for (int n = 0; n < kHD / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    float top[kX], sum[kX];
#pragma unroll
    for (int x = 0; x < kX; ++x) {
        top[x] = -INFINITY;
        sum[x] = 0.f;
    }
    int stage = 0, fill = C::kStages - 1;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = mine; i < n_blocks; i += stride) {
        fetch(i + (C::kStages - 1) * stride, fill);   // (the stage was left at the end of the turn before)
        ok = mbar_wait_at(bars + stage * 8, phase);
        if (!ok) break;
        const uint32_t at = ring + stage * 2 * C::kTile, vat = at + C::kTile;
        const int key0 = key_of(i), left = s.klen - key0;
        if (left < kKeys) {
            for (int e = lane; e < (kKeys - left) * 8 * C::kPanels; e += 32) {
                const int r = left + e / (8 * C::kPanels), c = e % (8 * C::kPanels);
                sts128(vat + (c >> 3) * C::kPanel + r * 128 + (c & 7) * 16, make_uint4(0u, 0u, 0u, 0u));
            }
            __syncwarp();
        }
        // ---- scores of the rows and 16 keys: the lane has keys 2t, 2t + 1, 2t + 8, 2t + 9 of its rows
        float sc[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
        const int kr = (lane >> 4) * 8 + (lane & 7), kc = (lane >> 3) & 1;
#pragma unroll
        for (int k = 0; k < kHD / 16; ++k) {
            if (k >= steps) break;
            uint32_t kf[4];
            ldsm4(kf, at + (k >> 2) * C::kPanel + kr * 128 + ((((k & 3) * 2 + kc) ^ (kr & 7)) << 4));
            const uint32_t a1 = kTall ? qf[k][2 * kX - 2] : 0u, a3 = kTall ? qf[k][2 * kX - 1] : 0u;
            mma_16816(sc[0], qf[k][0], a1, qf[k][1], a3, kf[0], kf[1]);
            mma_16816(sc[1], qf[k][0], a1, qf[k][1], a3, kf[2], kf[3]);
        }
        float v[kX][4];       // of a row: keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
        for (int x = 0; x < kX; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[x][e] = sc[e >> 1][2 * x + (e & 1)];
        if (kWide) {
#pragma unroll
            for (int x = 0; x < kX; ++x) {
                cap_wide2(v[x][0], v[x][1], p);
                cap_wide2(v[x][2], v[x][3], p);
            }
        } else if (p.cap_out > 0.f) {
#pragma unroll
            for (int x = 0; x < kX; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[x][e] = fmaf(rcp_fast(1.f + ex2_fast(v[x][e] * p.cap_in)), -2.f * p.cap_out, p.cap_out);
        } else {
#pragma unroll
            for (int x = 0; x < kX; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[x][e] *= p.scale_log2;
        }
        if (p.slopes) {
#pragma unroll
            for (int x = 0; x < kX; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[x][e] = fmaf(slope[x], fabsf((float)(key0 + (e >> 1) * 8 + 2 * t + (e & 1) - qpos[x])), v[x][e]);
        }
        if (p.table) {
#pragma unroll
            for (int x = 0; x < kX; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[x][e] = fmaf(__half2float(table[x][max(-p.reach, min(p.reach, key0 + (e >> 1) * 8 + 2 * t + (e & 1) - qpos[x]))]), kRulesLog2e, v[x][e]);
        }
        // masks, where not every row sees every key of the block
        const bool inside = (p.window_left == kNoLimit || key0 >= qb - p.window_left) && (p.window_right == kNoLimit || key0 + kKeys - 1 <= qa + p.window_right);
        if (p.k_docs || left < kKeys || !(inside || key0 + kKeys <= pre)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = key0 + (e >> 1) * 8 + 2 * t + (e & 1);
                const int d = p.k_docs && j < s.klen ? p.k_docs[s.k0 + j] : 0;
#pragma unroll
                for (int x = 0; x < kX; ++x) {
                    const bool in_window = (p.window_left == kNoLimit || j >= qpos[x] - p.window_left) && (p.window_right == kNoLimit || j <= qpos[x] + p.window_right);
                    if (!(j < s.klen && (in_window || j < s.prefix) && doc[x] >= 0 && (!p.k_docs || d == doc[x]))) v[x][e] = -INFINITY;
                }
            }
        }
        float most[kX];
        bool grow = false;
#pragma unroll
        for (int x = 0; x < kX; ++x) {
            most[x] = fmaxf(fmaxf(v[x][0], v[x][1]), fmaxf(v[x][2], v[x][3]));
            most[x] = fmaxf(most[x], __shfl_xor_sync(0xffffffffu, most[x], 1));
            most[x] = fmaxf(most[x], __shfl_xor_sync(0xffffffffu, most[x], 2));
            grow = grow || most[x] > top[x] + kRescaleStep;   // also true for the first finite score of a row
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int x = 0; x < kX; ++x) {
                if (most[x] > top[x] + kRescaleStep) {
                    const float keep = top[x] == -INFINITY ? 0.f : ex2_fast(top[x] - most[x]);
                    top[x] = most[x];
                    sum[x] *= keep;
#pragma unroll
                    for (int n = 0; n < kHD / 8; ++n) {
                        o[n][2 * x] *= keep;
                        o[n][2 * x + 1] *= keep;
                    }
                }
            }
        }
        uint32_t w[2 * kX];   // weights: keys 2t, 2t + 1, then 2t + 8, 2t + 9 of a row
#pragma unroll
        for (int x = 0; x < kX; ++x) {
            const float shift = top[x] == -INFINITY ? 0.f : top[x];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[x][e] = ex2_fast(v[x][e] - shift);
                sum[x] += v[x][e];
            }
            w[2 * x] = pack2(v[x][0], v[x][1]);
            w[2 * x + 1] = pack2(v[x][2], v[x][3]);
        }
        const uint32_t w1 = kTall ? w[2 * kX - 2] : 0u, w3 = kTall ? w[2 * kX - 1] : 0u;
        const int vr = ((lane >> 3) & 1) * 8 + (lane & 7), vc = lane >> 4;
#pragma unroll
        for (int n = 0; n < kHD / 16; ++n) {
            if (n >= steps) break;
            uint32_t vf[4];
            ldsm4_trans(vf, vat + (n >> 2) * C::kPanel + vr * 128 + ((((n & 3) * 2 + vc) ^ (vr & 7)) << 4));
            mma_16816(o[2 * n], w[0], w1, w[1], w3, vf[0], vf[1]);
            mma_16816(o[2 * n + 1], w[0], w1, w[1], w3, vf[2], vf[3]);
        }
        __syncwarp();   // the stage has been read
        if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1u;
        }
        fill = fill + 1 == C::kStages ? 0 : fill + 1;
    }
    if (!ok) {   // (the copies that are still on their way land before the CTA leaves; bounded)
        if (lane == 0) atomicExch(err, 24);
        for (int n = 0; n < C::kStages; ++n) mbar_wait_at(bars + n * 8, n < stage ? phase ^ 1u : phase);
    }
    // ---- the warps' rows are joined, then the CTAs'
#pragma unroll
    for (int x = 0; x < kX; ++x) {
        sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 1);
        sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 2);
    }
    __syncthreads();
    float* const warp_o = reinterpret_cast<float*>(smem);                      // [kWarps][kRows][kHD]
    float* const warp_ms = warp_o + kWarps * kRows * kHD;                      // [kWarps][2][kRows]
    float* const cta_o = reinterpret_cast<float*>(smem + C::kSumAt);           // [kRows][kHD]
    float* const cta_ms = cta_o + kRows * kHD;                                 // [2][kRows]
#pragma unroll
    for (int n = 0; n < kHD / 8; ++n)
#pragma unroll
        for (int x = 0; x < kX; ++x)
            if (n < 2 * steps && real[x])
                *reinterpret_cast<float2*>(warp_o + (warp * kRows + g + 8 * x) * kHD + n * 8 + 2 * t) = make_float2(o[n][2 * x], o[n][2 * x + 1]);
    if (t == 0) {
#pragma unroll
        for (int x = 0; x < kX; ++x) {
            // (scores that are not numbers leave no maximum: any finite one makes the part count below)
            warp_ms[warp * 2 * kRows + g + 8 * x] = sum[x] == sum[x] ? top[x] : 0.f;
            warp_ms[warp * 2 * kRows + kRows + g + 8 * x] = sum[x];
        }
    }
    __syncthreads();
    // A part that has a maximum has seen something, and its share counts even times 0: what is not finite in it makes the row not finite, and the row is
    // computed again. (The sums of a part without one are 0 times what is masked.)
    auto saw = [](float m) { return m != -INFINITY; };
    for (int e = threadIdx.x; e < rows * hd; e += kThreads) {
        const int r = e / hd, c = e % hd;
        float m = -INFINITY, l = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, warp_ms[w * 2 * kRows + r]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float part = warp_ms[w * 2 * kRows + r];
            if (saw(part)) {
                const float f = ex2_fast(part - m);
                v = fmaf(f, warp_o[(w * kRows + r) * kHD + c], v);
                l = fmaf(f, warp_ms[w * 2 * kRows + kRows + r], l);
            }
        }
        cta_o[r * kHD + c] = v;
        if (c == 0) {
            cta_ms[r] = m;
            cta_ms[kRows + r] = l;
        }
    }
    cluster.sync();
    // a row to a CTA, a feature to a thread
    static_assert(kThreads >= kHD, "a thread for each feature");
    for (int r = crank; r < rows; r += csize) {
        const int c = threadIdx.x;
        float part_m[kMaxCluster], m = -INFINITY, l = 0.f, v = 0.f;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) part_m[k] = k < csize ? cluster.map_shared_rank(cta_ms, k)[r] : -INFINITY;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) m = fmaxf(m, part_m[k]);
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            if (saw(part_m[k]) && c < hd) {
                const float f = ex2_fast(part_m[k] - m);
                v = fmaf(f, cluster.map_shared_rank(cta_o, k)[r * kHD + c], v);
                l = fmaf(f, cluster.map_shared_rank(cta_ms, k)[kRows + r], l);
            }
        }
        const int row = tile * kRows + r, i = row / p.group, h = kv_head * p.group + row % p.group;
        const half z = __float2half_rn(l == 0.f && v == 0.f ? 0.f : v / l);
        const bool odd = c < hd && !(__habs(z) <= __float2half_rn(65504.f));
        if (__syncthreads_or(odd)) {
            if (warp == 0) rules_row(p, s, i, h);
        } else if (c < hd) {
            p.out[(s.q0 + i) * p.out_pitch + h * hd + c] = z;
        }
    }
    cluster.sync();   // nobody leaves while its rows are read
}

template <int kHD, bool kTall, bool kWide>
cudaError_t launch(const CUtensorMap& tk, const CUtensorMap& tv, const RuleParams& p, int row_tiles, long long units, int csize, int* err, cudaStream_t st) {
    const auto kernel = attention_rules_token_kernel<kHD, kTall, kWide>;
    static PerDeviceOnce once;
    cudaError_t e = once.run([&] {
        cudaError_t x = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<kHD>::kBytes);
        if (x == cudaSuccess) x = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        return x;
    });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * csize));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg<kHD>::kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)csize;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    // What outlasts a wave of CTAs is taken longest first, so that short sequences are left for the end.
    const bool longest_first = p.batch <= kThreads && units * csize > 2 * sm_count();
    return cudaLaunchKernelEx(&cfg, kernel, tk, tv, p, row_tiles, longest_first, err);
}

template <int kHD, bool kTall>
cudaError_t launch_with(const CUtensorMap& tk, const CUtensorMap& tv, const RuleParams& p, int row_tiles, long long units, int csize, int* err, cudaStream_t st) {
    return (p.cap_wide ? launch<kHD, kTall, true> : launch<kHD, kTall, false>)(tk, tv, p, row_tiles, units, csize, err, st);
}

}  // namespace

bool attention_rules_token_takes(const RuleParams& p) {
    const long long units = (long long)p.batch * (p.nhead / p.group) * ((p.max_q_len * (long long)p.group + kRows - 1) / kRows);
    return p.k_start && p.max_q_len <= 4 && p.head_dim % 16 == 0 && p.head_dim <= 128 && ((p.q_pitch | p.k_pitch | p.v_pitch) & 7) == 0 && aligned16(p.q) && aligned16(p.k) && aligned16(p.v) &&
           units * kMaxCluster <= 0x7fffffff && p.k_rows > 0 && p.max_k_len > 0;
}

int attention_rules_token_launch(const RuleParams& p, cudaStream_t st) {
    const int row_tiles = (p.max_q_len * p.group + kRows - 1) / kRows;
    const long long units = (long long)p.batch * (p.nhead / p.group) * row_tiles;
    int* err = nullptr;
    const int rc = attn_err_address(&err);
    if (rc) return rc;
    CUtensorMap tk, tv;
    if (!make_tmap_heads_f16(&tk, p.k, p.k_rows, p.nhead / p.group, p.head_dim, p.k_pitch, kKeys) ||
        !make_tmap_heads_f16(&tv, p.v, p.k_rows, p.nhead / p.group, p.head_dim, p.v_pitch, kKeys))
        return fail(ET_ERR_CUDA, "et_attention_rules: cuTensorMapEncodeTiled failed");
    // CTAs that share a sequence's keys: as many as give each warp a block, up to four CTAs to an SM; more than eight to a cluster (which not every
    // place on the chip can hold at once) only where the SMs would not all have one.
    int csize = 1;
    while (csize < kMaxCluster && (long long)csize * kWarps * kKeys < p.max_k_len && units * csize * 2 <= (csize < 8 ? 4 : 1) * sm_count()) csize *= 2;
    const bool tall = p.max_q_len * p.group > 8;
    const auto run = p.head_dim <= 64 ? (tall ? launch_with<64, true> : launch_with<64, false>) : (tall ? launch_with<128, true> : launch_with<128, false>);
    return cuda_status(run(tk, tv, p, row_tiles, units, csize, err, st), "et_attention_rules launch");
}

}  // namespace et
