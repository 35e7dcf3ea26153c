// Attention with rules on its scores for single tokens over keys kept from before (and for the few queries of short calls): bound by reading K and V once.
//
// The query heads that share a K/V head (and the queries of a sequence, if there are a few) are the rows of one m16n8k16 tile, so that keys and values are read
// once for all of them. A cluster of CTAs shares the keys of a sequence and K/V head: its warps take blocks of 16 keys in turn, each through a ring
// of its own in shared memory, filled by asynchronous copies (a warp waits for nobody else), with a running maximum and sum of its own. At the end the
// warps' sums are joined in shared memory and the CTAs' through distributed shared memory, in a fixed order: one launch, no workspace, the same bits every time.
//
// Scores, maxima and sums are fp32; the weights go to the second product as fp16 (half a step of 2^-11 of a weight). A row whose result is not finite
// is computed again from the keys that it sees (rules_row), as not a number times the weight 0 is not a number.
#include <cooperative_groups.h>
#include "attention_rules.h"
#include "common.h"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace et {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kKeys = 16;                 // of a block
constexpr int kRows = 16;                 // of a tile
constexpr int kMaxCluster = 16;

template <int kHD>
struct Cfg {
    static constexpr int kPitch = kHD * 2;                       // bytes of a row of K or V in shared memory
    static constexpr int kStage = 2 * kKeys * kPitch;            // a block of K and of V
    static constexpr int kStages = kHD == 64 ? 6 : 3;
    static constexpr int kRing = kStages * kStage;               // of a warp
    static constexpr int kSumAt = kWarps * kRing;                // this CTA's rows: [kRows][kHD] floats, then maxima and sums
    static constexpr int kBytes = kSumAt + kRows * kHD * 4 + 2 * kRows * 4;
    static_assert(kWarps * (kRows * kHD + 2 * kRows) * 4 <= kSumAt, "the warps' sums fit where their rings were");
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {   // zeros where there is nothing
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
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

// kHD: 64 or 128, the head's width rounded up.
template <int kHD>
__global__ void __launch_bounds__(kThreads) attention_rules_token_kernel(const __grid_constant__ RuleParams p, int row_tiles) {
    using C = Cfg<kHD>;
    constexpr int kChunks = kHD / 8;      // 16-byte granules of a padded row
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    cg::cluster_group cluster = cg::this_cluster();
    const int csize = cluster.num_blocks(), crank = cluster.block_rank();
    const int hd = p.head_dim, steps = hd >> 4;
    int unit = blockIdx.x / csize;        // sequence, K/V head, tile of rows
    const int tile = unit % row_tiles;
    unit /= row_tiles;
    const int n_kv = p.nhead / p.group, kv_head = unit % n_kv, b = unit / n_kv;
    pdl_launch_dependents();
    pdl_wait();
    const RuleSeq s = rule_seq(p, b);
    const int rows = min(s.qlen * p.group - tile * kRows, kRows);
    if (rows <= 0) return;                // the same for the whole cluster
    // the lane's two rows: query, head, position
    int qi[2], head[2], qpos[2], doc[2];
    float slope[2];
    bool real[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        real[i] = g + 8 * i < rows;
        const int r = tile * kRows + (real[i] ? g + 8 * i : 0);
        qi[i] = r / p.group;
        head[i] = kv_head * p.group + r % p.group;
        qpos[i] = s.qpos0 + qi[i];
        doc[i] = p.q_docs ? p.q_docs[s.q0 + qi[i]] : 0;
        slope[i] = p.slopes ? p.slopes[head[i]] * kRulesLog2e : 0.f;
    }
    uint32_t qf[kHD / 16][4];
#pragma unroll
    for (int k = 0; k < kHD / 16; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const half* const q = p.q + (s.q0 + qi[i & 1]) * p.q_pitch + head[i & 1] * hd + k * 16 + (i >> 1) * 8 + 2 * t;
            qf[k][i] = k < steps && real[i & 1] ? *reinterpret_cast<const uint32_t*>(q) : 0u;
        }
    // blocks of keys that some row sees: of the prefix, then of the window
    const int qa = s.qpos0 + tile * kRows / p.group, qb = s.qpos0 + (tile * kRows + rows - 1) / p.group;
    const int pre = max(0, min(s.prefix, s.klen));
    const int n_prefix = (pre + kKeys - 1) / kKeys;
    const int lo = p.window_left == kNoLimit ? 0 : max(qa - p.window_left, 0), hi = p.window_right == kNoLimit ? s.klen - 1 : min(qb + p.window_right, s.klen - 1);
    const int first = max(lo / kKeys, n_prefix);
    const int n_blocks = n_prefix + (hi >= lo ? max(hi / kKeys - first + 1, 0) : 0);
    auto key_of = [&](int i) { return (i < n_prefix ? i : first + i - n_prefix) * kKeys; };

    const uint32_t ring = smem_u32(smem) + warp * C::kRing;
    const half* const kbase = p.k + s.k0 * p.k_pitch + kv_head * hd;
    const half* const vbase = p.v + s.k0 * p.v_pitch + kv_head * hd;
    const int stride = csize * kWarps;
    auto fetch = [&](int i, int stage) {      // granule c of row r lies at c ^ (r & 7): eight rows' granules fall into different banks
        if (i < n_blocks) {
            const int key0 = key_of(i);
            const uint32_t at = ring + stage * C::kStage;
#pragma unroll
            for (int n = 0; n < kKeys * kChunks / 32; ++n) {
                const int e = n * 32 + lane, r = e / kChunks, c = e % kChunks;
                const bool in = key0 + r < s.klen && c * 8 < hd;
                const uint32_t to = at + r * C::kPitch + ((c ^ (r & 7)) << 4);
                const long long row = in ? key0 + r : 0;
                const int col = in ? c * 8 : 0;
                copy16(to, kbase + row * p.k_pitch + col, in);
                copy16(to + kKeys * C::kPitch, vbase + row * p.v_pitch + col, in);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float o[kHD / 8][4];
#pragma unroll
    for (int n = 0; n < kHD / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    const int mine = crank * kWarps + warp;
#pragma unroll
    for (int n = 0; n < C::kStages - 1; ++n) fetch(mine + n * stride, n);
    int stage = 0, fill = C::kStages - 1;
    for (int i = mine; i < n_blocks; i += stride) {
        fetch(i + (C::kStages - 1) * stride, fill);
        asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
        __syncwarp();
        const uint32_t at = ring + stage * C::kStage;
        const int key0 = key_of(i);
        // ---- scores of 16 rows and 16 keys: the lane has keys 2t, 2t + 1, 2t + 8, 2t + 9 of its rows
        float sc[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
#pragma unroll
        for (int k = 0; k < kHD / 16; ++k) {
            if (k >= steps) break;
            uint32_t kf[4];
            const int r = (lane >> 4) * 8 + (lane & 7), c = k * 2 + ((lane >> 3) & 1);
            ldsm4(kf, at + r * C::kPitch + ((c ^ (r & 7)) << 4));
            mma_16816(sc[0], qf[k][0], qf[k][1], qf[k][2], qf[k][3], kf[0], kf[1]);
            mma_16816(sc[1], qf[k][0], qf[k][1], qf[k][2], qf[k][3], kf[2], kf[3]);
        }
        float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = key0 + n * 8 + 2 * t + (e & 1), x = e >> 1;
                const bool in_window = (p.window_left == kNoLimit || j >= qpos[x] - p.window_left) && (p.window_right == kNoLimit || j <= qpos[x] + p.window_right);
                bool seen = real[x] && j < s.klen && (in_window || j < s.prefix);
                if (p.k_docs) seen = seen && doc[x] >= 0 && p.k_docs[s.k0 + j] == doc[x];
                float v = sc[n][e];
                v = p.cap_out > 0.f ? p.cap_out - 2.f * p.cap_out / (1.f + ex2_fast(v * p.cap_in)) : v * p.scale_log2;
                if (p.slopes) v = fmaf(-slope[x], fabsf((float)(j - qpos[x])), v);
                if (p.table) v = fmaf(__half2float(p.table[(size_t)head[x] * (2 * p.reach + 1) + p.reach + max(-p.reach, min(p.reach, j - qpos[x]))]), kRulesLog2e, v);
                v = seen ? v : -INFINITY;
                sc[n][e] = v;
                most[x] = fmaxf(most[x], v);
            }
        float shift[2], keep[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            most[x] = fmaxf(most[x], __shfl_xor_sync(0xffffffffu, most[x], 1));
            most[x] = fmaxf(most[x], __shfl_xor_sync(0xffffffffu, most[x], 2));
            const float m = fmaxf(top[x], most[x]);
            shift[x] = m == -INFINITY ? 0.f : m;
            keep[x] = top[x] == -INFINITY ? 0.f : ex2_fast(top[x] - shift[x]);
            top[x] = m;
        }
        if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
            for (int n = 0; n < kHD / 8; ++n) {
                o[n][0] *= keep[0];
                o[n][1] *= keep[0];
                o[n][2] *= keep[1];
                o[n][3] *= keep[1];
            }
            sum[0] *= keep[0];
            sum[1] *= keep[1];
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sc[n][e] = ex2_fast(sc[n][e] - shift[e >> 1]);
                sum[e >> 1] += sc[n][e];
            }
        const uint32_t p0 = pack2(sc[0][0], sc[0][1]), p1 = pack2(sc[0][2], sc[0][3]), p2 = pack2(sc[1][0], sc[1][1]), p3 = pack2(sc[1][2], sc[1][3]);
        const uint32_t vat = at + kKeys * C::kPitch;
#pragma unroll
        for (int n = 0; n < kHD / 16; ++n) {
            if (n >= steps) break;
            uint32_t vf[4];
            const int r = ((lane >> 3) & 1) * 8 + (lane & 7), c = n * 2 + (lane >> 4);
            ldsm4_trans(vf, vat + r * C::kPitch + ((c ^ (r & 7)) << 4));
            mma_16816(o[2 * n], p0, p1, p2, p3, vf[0], vf[1]);
            mma_16816(o[2 * n + 1], p0, p1, p2, p3, vf[2], vf[3]);
        }
        __syncwarp();   // the stage has been read
        stage = stage + 1 == C::kStages ? 0 : stage + 1;
        fill = fill + 1 == C::kStages ? 0 : fill + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // ---- the warps' rows are joined, then the CTAs'
#pragma unroll
    for (int x = 0; x < 2; ++x) {
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
        for (int x = 0; x < 2; ++x)
            if (n < 2 * steps && real[x])
                *reinterpret_cast<float2*>(warp_o + (warp * kRows + g + 8 * x) * kHD + n * 8 + 2 * t) = make_float2(o[n][2 * x], o[n][2 * x + 1]);
    if (t == 0) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            warp_ms[warp * 2 * kRows + g + 8 * x] = top[x];
            warp_ms[warp * 2 * kRows + kRows + g + 8 * x] = sum[x];
        }
    }
    __syncthreads();
    auto factor = [](float m, float all) { return m == -INFINITY ? 0.f : ex2_fast(m - all); };   // of sums relative to m, to make them relative to `all`
    for (int e = threadIdx.x; e < rows * hd; e += kThreads) {
        const int r = e / hd, c = e % hd;
        float m = -INFINITY, l = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, warp_ms[w * 2 * kRows + r]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = factor(warp_ms[w * 2 * kRows + r], m);
            if (f != 0.f) {
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
            const float f = factor(part_m[k], m);
            if (f != 0.f && c < hd) {
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

template <int kHD>
cudaError_t launch(const RuleParams& p, int row_tiles, long long units, int csize, cudaStream_t st) {
    const auto kernel = attention_rules_token_kernel<kHD>;
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
    return cudaLaunchKernelEx(&cfg, kernel, p, row_tiles);
}

}  // namespace

bool attention_rules_token_takes(const RuleParams& p) {
    const long long units = (long long)p.batch * (p.nhead / p.group) * ((p.max_q_len * (long long)p.group + kRows - 1) / kRows);
    return p.k_start && p.max_q_len <= 4 && p.head_dim % 16 == 0 && p.head_dim <= 128 && ((p.q_pitch | p.k_pitch | p.v_pitch) & 7) == 0 && aligned16(p.q) && aligned16(p.k) && aligned16(p.v) &&
           units * kMaxCluster <= 0x7fffffff;
}

cudaError_t attention_rules_token_launch(const RuleParams& p, cudaStream_t st) {
    const int row_tiles = (p.max_q_len * p.group + kRows - 1) / kRows;
    const long long units = (long long)p.batch * (p.nhead / p.group) * row_tiles;
    // CTAs that share a sequence's keys: as many as give each warp two blocks, up to some six CTAs to an SM; more than eight (which not every
    // place on the chip can hold at once) only where the SMs would not all have one.
    int csize = 1;
    while (csize < kMaxCluster && (long long)csize * kWarps * kKeys * 2 < p.max_k_len && units * csize * 2 <= (csize < 8 ? 6 : 2) * sm_count()) csize *= 2;
    return p.head_dim <= 64 ? launch<64>(p, row_tiles, units, csize, st) : launch<128>(p, row_tiles, units, csize, st);
}

}  // namespace et
