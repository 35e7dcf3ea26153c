// Attention of drafted tokens (a tree of up to 64, or single tokens) over keys and values kept in int8 pages: softmax(scale q . k) v over the keys kept before and, of the drafted
// tokens' own, those whose bit is set. Bound by reading the codes once where there are few rows.
//
// The queries and query heads of a K/V head are rows, 16 to a tile of mma.sync m16n8k16. Codes become halves exactly (three operations for four), the key's scale multiplies the
// score, the value's scale the weight. Which features a step of the first product takes, and which the columns of the second are, is free: a lane has 16 neighbouring codes of a key
// of K, and for V of four keys the codes of kHD / 8 neighbouring features, so both come by wide loads, each lane's into a place of shared memory that only it reads
// (cp.async, no barrier). A cluster of CTAs shares a sequence's keys, its warps take blocks of 16 in turn with a reference, sum and O of their own, joined in shared
// and then distributed shared memory in a fixed order: no workspace, one launch, the same bits every time.
//
// Scores, references and sums are fp32; the weights times the values' scales go to the second product as fp16 (half a step of 2^-11 of a weight).
#include <cooperative_groups.h>
#include "attention_tree.cuh"
#include "attention_tree.h"
#include "common.h"
#include "ptx.cuh"

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
    static constexpr int kFeat = kHD / 8;                        // features of V that a lane has
    static constexpr int kKLoads = 2 * (kHD / 64);               // of 16 bytes: two keys
    static constexpr int kVLoads = 4 * (kHD >= 128 ? kHD / 128 : 1);   // four keys, of 16 bytes (of 8 in heads of 64)
    static constexpr int kVBytes = kHD >= 128 ? 16 : 8;
    static constexpr int kStages = kHD == 64 ? 5 : kHD == 128 ? 4 : 3;
    // of a warp's stage: [load][lane]
    static constexpr int kVAt = kKLoads * 512, kScaleAt = kVAt + kVLoads * 32 * kVBytes, kStage = kScaleAt + 4 * 32 * 8;
    static constexpr int kRing = kStages * kStage;
    static constexpr int kJoin = kWarps * (kRows * kHD + 2 * kRows) * 4;
    static constexpr int kSumAt = kWarps * kRing > kJoin ? kWarps * kRing : kJoin;   // this CTA's rows: [kRows][kHD] floats, then references and sums
    static constexpr int kBytes = kSumAt + (kRows * kHD + 2 * kRows) * 4;
};

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// `size` bytes, of which `real` are read and the others are zeros.
template <int kSize>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from, int real) {
    if constexpr (kSize == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(real) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
// An infinite feature of a query makes its row not a number, as it does in 0 times infinity and in infinity - infinity.
__device__ __forceinline__ uint32_t no_infinity(uint32_t two) {
    const uint32_t lo = (two & 0x7fffu) == 0x7c00u ? 0x7fffu : two & 0xffffu, hi = (two & 0x7fff0000u) == 0x7c000000u ? 0x7fff0000u : two & 0xffff0000u;
    return lo | hi;
}

// kHD: 64, 128 or 256, the head's width rounded up. kTall: more than eight rows; otherwise the lower half of the tile is empty and left out of everything but the products.
template <int kHD, bool kTall>
__global__ void __launch_bounds__(kThreads) attention_tree_kernel(const __grid_constant__ TreeParams p, int row_tiles, bool longest_first) {
    using C = Cfg<kHD>;
    constexpr int kX = kTall ? 2 : 1;     // rows of a lane: g and g + 8
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    cg::cluster_group cluster = cg::this_cluster();
    const int csize = cluster.num_blocks(), crank = cluster.block_rank();
    const int hd = p.head_dim;
    int unit = blockIdx.x / csize;        // sequence, K/V head, tile of rows
    const int tile = unit % row_tiles;
    unit /= row_tiles;
    const int n_kv = p.nhead / p.group, kv_head = unit % n_kv;
    int b = unit / n_kv;
    pdl_wait();
    pdl_launch_dependents();
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
    const TreeSeq s = tree_seq(p, b);
    const int rows = min(s.qlen * p.group - tile * kRows, kRows);
    if (rows <= 0) return;                // the same for the whole cluster
    const int n_blocks = (s.klen + kKeys - 1) / kKeys;
    const int stride = csize * kWarps, mine = crank * kWarps + warp;
    const int* const table = p.table + (long long)b * p.table_width;
    const uint32_t ring = smem_u32(smem) + warp * C::kRing;
    auto page_of = [&](int i) {
        const int id = i < n_blocks ? __ldg(table + i * kKeys / p.page) : -1;
        return id < p.pages ? id : -1;
    };
    // Block i, which lies in page id: the lane's codes and scales.
    auto fetch = [&](int i, int id, int stage) {
        if (i < n_blocks) {
            const uint32_t to = ring + stage * C::kStage + lane * 16;
            const bool good = id >= 0;
            const long long row_k = ((long long)max(id, 0) * 2 * n_kv + kv_head) * p.page + (i * kKeys) % p.page, row_v = row_k + (long long)n_kv * p.page;
            const int8_t* const k = p.codes + row_k * hd;
            const int8_t* const v = p.codes + row_v * hd;
#pragma unroll
            for (int n = 0; n < C::kKLoads; ++n) {
                const int f = (n >> 1) * 64 + t * 16;
                copy_async<16>(to + n * 512, f < hd ? k + ((n & 1) * 8 + g) * hd + f : k, good && f < hd ? 16 : 0);
            }
#pragma unroll
            for (int n = 0; n < C::kVLoads; ++n) {
                const int key = 2 * t + (n & 1) + ((n >> 1) & 1) * 8, f = g * C::kFeat + (n >> 2) * 16;
                copy_async<C::kVBytes>(ring + stage * C::kStage + C::kVAt + (n * 32 + lane) * C::kVBytes, f < hd ? v + key * hd + f : v, good && f < hd ? C::kVBytes : 0);
            }
#pragma unroll
            for (int n = 0; n < 4; ++n)
                copy_async<8>(ring + stage * C::kStage + C::kScaleAt + (n * 32 + lane) * 8, p.scales + (n < 2 ? row_k : row_v) + (n & 1) * 8 + 2 * t, good ? 8 : 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int id_next = -1, ids[C::kStages];    // of the blocks on their way
#pragma unroll
    for (int n = 0; n < C::kStages - 1; ++n) ids[n] = page_of(mine + n * stride);
    id_next = page_of(mine + (C::kStages - 1) * stride);
#pragma unroll
    for (int n = 0; n < C::kStages - 1; ++n) fetch(mine + n * stride, ids[n], n);
    // the lane's rows
    unsigned long long bits[kX];
    bool real[kX];
    uint32_t qf[kHD / 16][2 * kX];
#pragma unroll
    for (int x = 0; x < kX; ++x) {
        real[x] = g + 8 * x < rows;
        const int r = tile * kRows + (real[x] ? g + 8 * x : 0), i = r / p.group, head = kv_head * p.group + r % p.group;
        bits[x] = tree_bits(p, s, i);
        const half* const q = p.q + (s.q0 + i) * p.q_pitch + (long long)head * hd;
#pragma unroll
        for (int n = 0; n < kHD / 64; ++n) {   // 16 features of the lane in each 64, four to a step
            const int f = n * 64 + t * 16;
            uint4 a = make_uint4(0u, 0u, 0u, 0u), c = a;
            if (f < hd && real[x]) {
                a = *reinterpret_cast<const uint4*>(q + f);
                c = *reinterpret_cast<const uint4*>(q + f + 8);
            }
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                qf[n * 4 + k][2 * x] = no_infinity(w[2 * k]);
                qf[n * 4 + k][2 * x + 1] = no_infinity(w[2 * k + 1]);
            }
        }
    }
    float o[C::kFeat][4];
#pragma unroll
    for (int n = 0; n < C::kFeat; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    float top[kX], sum[kX];
#pragma unroll
    for (int x = 0; x < kX; ++x) {
        top[x] = -INFINITY;
        sum[x] = 0.f;
    }
    int stage = 0, fill = C::kStages - 1;
    for (int i = mine; i < n_blocks; i += stride) {
        fetch(i + (C::kStages - 1) * stride, id_next, fill);   // (the lane has read that stage a turn ago)
        id_next = page_of(i + C::kStages * stride);
        asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
        const uint32_t at = ring + stage * C::kStage;
        const int key0 = i * kKeys;
        // ---- scores: the lane has keys 2t, 2t + 1, 2t + 8, 2t + 9 of its rows
        float sc[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
#pragma unroll
        for (int n = 0; n < kHD / 64; ++n) {
            const uint4 k0 = lds128(at + (2 * n * 32 + lane) * 16), k1 = lds128(at + ((2 * n + 1) * 32 + lane) * 16);
            const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t u0 = codes_biased(w0[k]), u1 = codes_biased(w1[k]);
                const uint32_t(&a)[2 * kX] = qf[n * 4 + k];
                const uint32_t a1 = kTall ? a[2 * kX - 2] : 0u, a3 = kTall ? a[2 * kX - 1] : 0u;
                mma_16816(sc[0], a[0], a1, a[1], a3, codes_to_half2<0>(u0), codes_to_half2<1>(u0));
                mma_16816(sc[1], a[0], a1, a[1], a3, codes_to_half2<0>(u1), codes_to_half2<1>(u1));
            }
        }
        float ks[4], vs[4], lv[4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const uint2 a = lds64(at + C::kScaleAt + (n * 32 + lane) * 8), c = lds64(at + C::kScaleAt + ((n + 2) * 32 + lane) * 8);
            ks[2 * n] = __uint_as_float(a.x) * p.scale_log2;
            ks[2 * n + 1] = __uint_as_float(a.y) * p.scale_log2;
            vs[2 * n] = __uint_as_float(c.x);
            vs[2 * n + 1] = __uint_as_float(c.y);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) lv[e] = log2_of_scale(vs[e]);
        float v[kX][4], scale[kX][4];
#pragma unroll
        for (int x = 0; x < kX; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[x][e] = sc[e >> 1][2 * x + (e & 1)] * ks[e];
                scale[x][e] = vs[e];
            }
        // masks, where not every row sees every key of the block
        const bool no_page = __ldg(table + key0 / p.page) < 0 || __ldg(table + key0 / p.page) >= p.pages;
        if (key0 + kKeys > s.kept || key0 + kKeys > s.klen || no_page) {
#pragma unroll
            for (int x = 0; x < kX; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (no_page || !tree_sees(s, bits[x], key0 + (e >> 1) * 8 + 2 * t + (e & 1))) {   // (what is not seen may have any scale)
                        v[x][e] = -INFINITY;
                        scale[x][e] = 0.f;
                    }
        }
        float most[kX];
        bool grow = false;
#pragma unroll
        for (int x = 0; x < kX; ++x) {
            most[x] = fmaxf(fmaxf(v[x][0] + lv[0], v[x][1] + lv[1]), fmaxf(v[x][2] + lv[2], v[x][3] + lv[3]));
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
                    for (int n = 0; n < C::kFeat; ++n) {
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
                v[x][e] *= scale[x][e];
            }
            w[2 * x] = pack2(v[x][0], v[x][1]);
            w[2 * x + 1] = pack2(v[x][2], v[x][3]);
        }
        const uint32_t w1 = kTall ? w[2 * kX - 2] : 0u, w3 = kTall ? w[2 * kX - 1] : 0u;
        // ---- O: step j of the lane's features is a tile of eight columns, column n the feature n kFeat + j
#pragma unroll
        for (int c = 0; c < C::kFeat / 4; ++c) {   // four features
            uint32_t u[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] = codes_biased(lds32(at + C::kVAt + (((c >> 2) * 4 + k) * 32 + lane) * C::kVBytes + (c & 3) * 4));
            const uint32_t lo0 = __byte_perm(u[0], u[1], 0x5140), hi0 = __byte_perm(u[0], u[1], 0x7362), lo1 = __byte_perm(u[2], u[3], 0x5140), hi1 = __byte_perm(u[2], u[3], 0x7362);
            mma_16816(o[4 * c], w[0], w1, w[1], w3, codes_to_half2<0>(lo0), codes_to_half2<0>(lo1));
            mma_16816(o[4 * c + 1], w[0], w1, w[1], w3, codes_to_half2<1>(lo0), codes_to_half2<1>(lo1));
            mma_16816(o[4 * c + 2], w[0], w1, w[1], w3, codes_to_half2<0>(hi0), codes_to_half2<0>(hi1));
            mma_16816(o[4 * c + 3], w[0], w1, w[1], w3, codes_to_half2<1>(hi0), codes_to_half2<1>(hi1));
        }
        stage = stage + 1 == C::kStages ? 0 : stage + 1;
        fill = fill + 1 == C::kStages ? 0 : fill + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // ---- the warps' rows are joined, then the CTAs'
#pragma unroll
    for (int x = 0; x < kX; ++x) {
        sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 1);
        sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 2);
    }
    __syncthreads();
    float* const warp_o = reinterpret_cast<float*>(smem);                      // [kWarps][kRows][kHD], features in the order of the columns
    float* const warp_ms = warp_o + kWarps * kRows * kHD;                      // [kWarps][2][kRows]
    float* const cta_o = reinterpret_cast<float*>(smem + C::kSumAt);           // [kRows][kHD]
    float* const cta_ms = cta_o + kRows * kHD;                                 // [2][kRows]
#pragma unroll
    for (int n = 0; n < C::kFeat; ++n)
#pragma unroll
        for (int x = 0; x < kX; ++x)
            if (real[x]) *reinterpret_cast<float2*>(warp_o + (warp * kRows + g + 8 * x) * kHD + n * 8 + 2 * t) = make_float2(o[n][2 * x], o[n][2 * x + 1]);
    if (t == 0) {
#pragma unroll
        for (int x = 0; x < kX; ++x) {
            // (scores that are not numbers leave no reference: any finite one makes the part count below)
            warp_ms[warp * 2 * kRows + g + 8 * x] = sum[x] == sum[x] ? top[x] : 0.f;
            warp_ms[warp * 2 * kRows + kRows + g + 8 * x] = sum[x];
        }
    }
    __syncthreads();
    auto saw = [](float m) { return m != -INFINITY; };   // (a part that has seen nothing has no reference)
    for (int e = threadIdx.x; e < rows * kHD; e += kThreads) {
        const int r = e / kHD, c = e % kHD;
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
    for (int r = crank; r < rows; r += csize) {
        float part_m[kMaxCluster], m = -INFINITY;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) part_m[k] = k < csize ? cluster.map_shared_rank(cta_ms, k)[r] : -INFINITY;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) m = fmaxf(m, part_m[k]);
        for (int f = threadIdx.x; f < hd; f += kThreads) {
            const int c = f % C::kFeat * 8 + f / C::kFeat;
            float l = 0.f, v = 0.f;
#pragma unroll
            for (int k = 0; k < kMaxCluster; ++k) {
                if (saw(part_m[k])) {
                    const float x = ex2_fast(part_m[k] - m);
                    v = fmaf(x, cluster.map_shared_rank(cta_o, k)[r * kHD + c], v);
                    l = fmaf(x, cluster.map_shared_rank(cta_ms, k)[kRows + r], l);
                }
            }
            const int row = tile * kRows + r, i = row / p.group, h = kv_head * p.group + row % p.group;
            p.out[(s.q0 + i) * p.out_pitch + (long long)h * hd + f] = __float2half_rn(l == 0.f ? 0.f : v / l);
        }
    }
    cluster.sync();   // nobody leaves while its rows are read
}

template <int kHD, bool kTall>
cudaError_t launch(const TreeParams& p, int row_tiles, long long units, int csize, cudaStream_t st) {
    const auto kernel = attention_tree_kernel<kHD, kTall>;
    static PerDeviceOnce once;
    const cudaError_t e = once.run([&] {
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
    return cudaLaunchKernelEx(&cfg, kernel, p, row_tiles, longest_first);
}

}  // namespace
}  // namespace et

extern "C" int et_attention_tree(const et_attention_tree_args* a) {
    using namespace et;
    ET_REQUIRE(a, "et_attention_tree: null pointer");
    ET_REQUIRE(a->batch >= 0 && a->q_tokens >= 0 && a->max_q_len >= 0 && a->max_k_len >= 0 && a->pages >= 0 && a->table_width >= 0, "et_attention_tree: negative size");
    ET_REQUIRE(a->nhead_kv > 0 && a->nhead > 0 && a->nhead % a->nhead_kv == 0, "et_attention_tree: nhead must be a multiple of nhead_kv");
    ET_REQUIRE(a->head_dim >= 16 && a->head_dim <= 256 && a->head_dim % 16 == 0, "et_attention_tree: head_dim must be a multiple of 16 up to 256");
    ET_REQUIRE(a->page >= 16 && a->page % 16 == 0, "et_attention_tree: the rows of a page must be a multiple of 16");
    ET_REQUIRE(a->max_q_len <= 64, "et_attention_tree: at most 64 drafted tokens to a sequence");
    ET_REQUIRE(a->scale >= 0.f && a->scale < INFINITY, "et_attention_tree: scale must be a finite number, 0 for 1 / sqrt(head_dim)");
    ET_REQUIRE((long long)a->nhead * a->head_dim <= 0x7fffffff && (long long)a->nhead / a->nhead_kv * a->max_q_len <= 0x7fffff && (long long)a->batch * a->max_q_len <= 0x7fffffff &&
                   a->max_k_len <= 0x7fffffff - 64,
               "et_attention_tree: too large");
    if (a->batch == 0 || a->q_tokens == 0 || a->max_q_len == 0) return ET_OK;
    ET_REQUIRE(a->out && a->q && a->k_lens, "et_attention_tree: null pointer");
    ET_REQUIRE(a->max_k_len == 0 || (a->codes && a->scales && a->table), "et_attention_tree: null pointer");
    const long long width = (long long)a->nhead * a->head_dim;
    const long long q_pitch = a->q_tokens == 1 ? width : a->q_pitch, out_pitch = a->q_tokens == 1 ? width : a->out_pitch;
    ET_REQUIRE(q_pitch >= width && out_pitch >= width, "et_attention_tree: pitch below the width of the heads");
    ET_REQUIRE(aligned16(a->q) && aligned16(a->out) && aligned16(a->codes) && aligned16(a->scales) && ((q_pitch | out_pitch) & 7) == 0, "et_attention_tree: rows must start on 16 bytes");
    ET_REQUIRE(a->out != a->q, "et_attention_tree: out may not be q");
    TreeParams p;
    p.out = static_cast<half*>(a->out); p.q = static_cast<const half*>(a->q);
    p.codes = static_cast<const int8_t*>(a->codes); p.scales = a->scales;
    p.table = a->table; p.k_lens = a->k_lens; p.cu_seqlens = a->cu_seqlens; p.tree = reinterpret_cast<const long long*>(a->tree);
    p.out_pitch = out_pitch; p.q_pitch = q_pitch;
    p.nhead = a->nhead; p.group = a->nhead / a->nhead_kv; p.head_dim = a->head_dim;
    p.batch = a->batch; p.q_tokens = a->q_tokens; p.max_q_len = a->max_q_len; p.max_k_len = a->max_k_len;
    p.pages = a->pages; p.page = a->page; p.table_width = a->table_width;
    p.scale_log2 = (a->scale == 0.f ? 1.f / sqrtf((float)a->head_dim) : a->scale) * 1.4426950408889634f;
    return (attention_tree_tc_takes(p) ? attention_tree_tc_launch : attention_tree_launch)(p, static_cast<cudaStream_t>(a->stream));
}

namespace et {

int attention_tree_launch(const TreeParams& p, cudaStream_t st) {
    const int row_tiles = (p.max_q_len * p.group + kRows - 1) / kRows;
    const long long units = (long long)p.batch * (p.nhead / p.group) * row_tiles;
    if (units * kMaxCluster > 0x7fffffff) return fail(ET_ERR_INVALID, "et_attention_tree: too large");
    // CTAs that share a sequence's keys: as many as give each warp a block, up to four CTAs to an SM; more than eight to a cluster (which not every
    // place on the chip can hold at once) only where the SMs would not all have one.
    int csize = 1;
    while (csize < kMaxCluster && (long long)csize * kWarps * kKeys < p.max_k_len && units * csize * 2 <= (csize < 8 ? 4 : 1) * sm_count()) csize *= 2;
    const bool tall = p.max_q_len * p.group > 8;
    const auto run = p.head_dim <= 64    ? (tall ? launch<64, true> : launch<64, false>)
                     : p.head_dim <= 128 ? (tall ? launch<128, true> : launch<128, false>)
                                         : (tall ? launch<256, true> : launch<256, false>);
    return cuda_status(run(p, row_tiles, units, csize, st), "et_attention_tree launch");
}

}  // namespace et
