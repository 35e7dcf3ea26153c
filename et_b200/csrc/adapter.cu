// Low-rank adapters of many requests beside a shared projection: out_t = base_t + scale_a B_a (A_a x_t), a the adapter of token t's sequence.
//
// A bank holds the adapters of one projection in the order in which the tensor cores take them, so that a warp loads its fragments of
// A and B with 16 bytes a lane, side by side, and needs no shared memory for them: they come from L1 and L2, where a bank stays.
// One launch does both products. 16 or 32 tokens of one sequence are kWk warps' work: each takes a share of the K range for A x, the
// shares are added in shared memory, and each takes a share of the output columns for B (A x), which go straight into base's granules.
// Where there are few tokens a cluster of CTAs takes the place of one: its CTAs split K and the columns once more and add the
// shares through distributed shared memory.
//
// Sums are fp32. A x is rounded to fp16 between the products, as the second one needs it, each row scaled by a power of two so that its
// largest value lies in [1, 2): it can not overflow, and the rounding (2^-11 of a term of the delta) is that of the result's own type.
// Both products' fragments are permuted so that a lane has eight neighbouring elements of X, of base and of the result: the sum over k
// does not depend on the order of k, and which column a lane of the second product computes is free.
//
// What bounds it: HBM. X is read once, base read and out written once; two operations a byte and rank, far below what mma.sync delivers.
#include <cooperative_groups.h>
#include <new>
#include <vector>
#include "common.h"

namespace cg = cooperative_groups;

namespace et {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kMaxRank = 128;
constexpr int kMaxCluster = 8;

struct Slot {
    int rank;      // 0: nothing to add
    float scale;
};

struct AdapterParams {
    half* out;
    const half* base;
    const half* x;
    const int* cu_seqlens;
    const int* ids;
    const Slot* slots;
    const half *a, *b;                  // packed, all slots
    long long out_pitch, base_pitch, x_pitch, a_stride, b_stride;   // of a slot, in elements
    int batch, tokens, n_slots, in_feat, out_feat;
    bool copy;                          // out is not base: what has no adapter is copied
};

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The tile of kTile tokens that CTA or cluster `tile` has: sequence, first token, tokens (whole warp). Without cu_seqlens a sequence is one token.
template <int kTile>
__device__ __forceinline__ int find_tile(const AdapterParams& p, int tile, int& seq, int& t0) {
    const int lane = threadIdx.x & 31;
    if (!p.cu_seqlens) {
        seq = t0 = tile;
        return tile < p.batch ? 1 : 0;
    }
    for (int base = 0; base < p.batch; base += 32) {
        const int i = base + lane;
        const int first = i < p.batch ? p.cu_seqlens[i] : 0;
        const int len = i < p.batch ? max(p.cu_seqlens[i + 1] - first, 0) : 0;
        const int n = (len + kTile - 1) / kTile;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, tile < incl);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int at = (tile - __shfl_sync(0xffffffffu, incl - n, src)) * kTile;
            seq = base + src;
            t0 = __shfl_sync(0xffffffffu, first, src) + at;
            const int end = min(__shfl_sync(0xffffffffu, first + len, src), p.tokens);   // (never beyond the rows that there are)
            return t0 < 0 ? 0 : max(min(end - t0, kTile), 0);
        }
        tile -= __shfl_sync(0xffffffffu, incl, 31);
    }
    return 0;
}

// kRt: 16-wide steps of the bank's largest rank; kMt: 16-token tiles of a warp; kWk: warps that share them.
template <int kRt, int kMt, int kWk, bool kCluster>
__global__ void __launch_bounds__(kThreads) adapter_kernel(const __grid_constant__ AdapterParams p) {
    constexpr int kWm = kWarps / kWk, kTile = kWm * kMt * 16;
    constexpr int kFrags = kMt * kRt * 2;                  // accumulator fragments of a warp
    extern __shared__ float4 parts[];                      // [kWarps][kFrags][32]: shares of A x, as accumulator fragments; then their sums
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wm = warp / kWk, wk = warp % kWk;
    const int g = lane >> 2, t = lane & 3;
    unsigned crank = 0, csize = 1;
    if constexpr (kCluster) {
        crank = cg::this_cluster().block_rank();
        csize = cg::this_cluster().num_blocks();
    }
    pdl_launch_dependents();
    pdl_wait();
    int seq = 0, t0 = 0;
    const int rows_in_tile = find_tile<kTile>(p, blockIdx.x / csize, seq, t0);
    if (rows_in_tile <= 0) return;   // the same for the whole cluster
    const int id = p.ids[seq];
    Slot slot = {0, 0.f};
    if (id >= 0 && id < p.n_slots) slot = p.slots[id];
    const int part = crank * kWk + wk, n_parts = csize * kWk;   // this warp's share of K and of the columns
    const int col_groups = (p.out_feat + 31) / 32;
    int row[kMt][2];        // the lane's rows, -1 beyond the tile
#pragma unroll
    for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = (wm * kMt + m) * 16 + h * 8 + g;
            row[m][h] = r < rows_in_tile ? t0 + r : -1;
        }
    if (slot.rank == 0) {
        if (!p.copy) return;
        for (int c = part; c < col_groups; c += n_parts) {
            const int col = c * 32 + t * 8;
            if (col >= p.out_feat) continue;
#pragma unroll
            for (int m = 0; m < kMt; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (row[m][h] >= 0)
                        *reinterpret_cast<uint4*>(p.out + row[m][h] * p.out_pitch + col) = *reinterpret_cast<const uint4*>(p.base + row[m][h] * p.base_pitch + col);
        }
        return;
    }
    // ---- A x: chunks of 32 features; a lane has eight neighbouring ones of its two rows, the operands of two steps of 16
    float acc[kMt][kRt * 2][4];
#pragma unroll
    for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int j = 0; j < kRt * 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
    const int chunks = (p.in_feat + 31) / 32;
    const uint4* const a = reinterpret_cast<const uint4*>(p.a + id * p.a_stride);
    constexpr int kUnroll = kMt == 1 ? 4 : 2;
    for (int c0 = part; c0 < chunks; c0 += n_parts * kUnroll) {
        uint4 xv[kUnroll][kMt][2];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int k = (c0 + u * n_parts) * 32 + t * 8;
#pragma unroll
            for (int m = 0; m < kMt; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    xv[u][m][h] = make_uint4(0u, 0u, 0u, 0u);
                    if (k < p.in_feat && row[m][h] >= 0) xv[u][m][h] = *reinterpret_cast<const uint4*>(p.x + row[m][h] * p.x_pitch + k);
                }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int c = c0 + u * n_parts;
            if (c >= chunks) break;
#pragma unroll
            for (int j = 0; j < kRt * 2; ++j) {
                const uint4 w = __ldg(a + ((size_t)c * (kRt * 2) + j) * 32 + lane);
#pragma unroll
                for (int m = 0; m < kMt; ++m) {
                    mma_16816(acc[m][j], xv[u][m][0].x, xv[u][m][1].x, xv[u][m][0].y, xv[u][m][1].y, w.x, w.y);
                    mma_16816(acc[m][j], xv[u][m][0].z, xv[u][m][1].z, xv[u][m][0].w, xv[u][m][1].w, w.z, w.w);
                }
            }
        }
    }
    // ---- the shares are added, in the order of the warps, then of the CTAs: each thread adds a few places of all of them, so that what another CTA
    // holds crosses to this one once
    float4* const sums = parts + kWarps * kFrags * 32;     // [kWm][kFrags][32]: of this CTA's warps
    float4* const all = sums + kWm * kFrags * 32;          // of all CTAs
#pragma unroll
    for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int j = 0; j < kRt * 2; ++j)
            parts[(warp * kFrags + m * kRt * 2 + j) * 32 + lane] = make_float4(acc[m][j][0], acc[m][j][1], acc[m][j][2], acc[m][j][3]);
    __syncthreads();
    for (int e = threadIdx.x; e < kWm * kFrags * 32; e += kThreads) {
        const int group = e / (kFrags * 32), at = e % (kFrags * 32);
        float4 s = parts[group * kWk * kFrags * 32 + at];
#pragma unroll
        for (int w = 1; w < kWk; ++w) {
            const float4 v = parts[(group * kWk + w) * kFrags * 32 + at];
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        sums[e] = s;
    }
    if constexpr (kCluster) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        for (int e = threadIdx.x; e < kWm * kFrags * 32; e += kThreads) {
            float4 v[kMaxCluster];
#pragma unroll
            for (int c = 0; c < kMaxCluster; ++c)
                if (c < (int)csize) v[c] = cluster.map_shared_rank(sums, c)[e];
            float4 s = v[0];
#pragma unroll
            for (int c = 1; c < kMaxCluster; ++c)
                if (c < (int)csize) { s.x += v[c].x; s.y += v[c].y; s.z += v[c].z; s.w += v[c].w; }
            all[e] = s;
        }
        cluster.sync();   // nobody leaves while its shares are read
    } else {
        __syncthreads();
    }
#pragma unroll
    for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int j = 0; j < kRt * 2; ++j) {
            const float4 v = (kCluster ? all : sums)[(wm * kFrags + m * kRt * 2 + j) * 32 + lane];
            acc[m][j][0] = v.x; acc[m][j][1] = v.y; acc[m][j][2] = v.z; acc[m][j][3] = v.w;
        }
    // ---- to fp16, each row by a power of two of its own; ranks that only pad a step are zeros even where x is not finite
#pragma unroll
    for (int j = 0; j < kRt * 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (j * 8 + 2 * t + i >= slot.rank) {
#pragma unroll
                for (int m = 0; m < kMt; ++m) acc[m][j][i] = acc[m][j][i + 2] = 0.f;
            }
    uint32_t h[kMt][kRt][4];
    float factor[kMt][2];
#pragma unroll
    for (int m = 0; m < kMt; ++m) {
        float top[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kRt * 2; ++j) {
            top[0] = fmaxf(top[0], fmaxf(fabsf(acc[m][j][0]), fabsf(acc[m][j][1])));
            top[1] = fmaxf(top[1], fmaxf(fabsf(acc[m][j][2]), fabsf(acc[m][j][3])));
        }
        float down[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
            const int e = __float_as_int(top[i]) >> 23;   // infinity stays one; below 2^-100 it makes no difference to the result
            const int ex = e == 255 ? 127 : max(27, min(e, 227));
            down[i] = __int_as_float((254 - ex) << 23);
            factor[m][i] = slot.scale * __int_as_float(ex << 23);
        }
#pragma unroll
        for (int q = 0; q < kRt; ++q) {
            h[m][q][0] = pack_h2(acc[m][2 * q][0] * down[0], acc[m][2 * q][1] * down[0]);
            h[m][q][1] = pack_h2(acc[m][2 * q][2] * down[1], acc[m][2 * q][3] * down[1]);
            h[m][q][2] = pack_h2(acc[m][2 * q + 1][0] * down[0], acc[m][2 * q + 1][1] * down[0]);
            h[m][q][3] = pack_h2(acc[m][2 * q + 1][2] * down[1], acc[m][2 * q + 1][3] * down[1]);
        }
    }
    // ---- base + B (A x): groups of 32 columns, of which a lane has eight neighbouring ones in each of its rows
    const uint4* const b = reinterpret_cast<const uint4*>(p.b + id * p.b_stride);
#pragma unroll 2
    for (int c = part; c < col_groups; c += n_parts) {
        const int col = c * 32 + t * 8;
        const bool in = col < p.out_feat;
        uint4 old[kMt][2];
#pragma unroll
        for (int m = 0; m < kMt; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (in && row[m][i] >= 0) old[m][i] = *reinterpret_cast<const uint4*>(p.base + row[m][i] * p.base_pitch + col);
        float d[kMt][4][4];
#pragma unroll
        for (int m = 0; m < kMt; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) d[m][j][i] = 0.f;
#pragma unroll
        for (int q = 0; q < kRt; ++q) {
            const uint4* const w = b + (((size_t)c * kRt + q) * 32 + lane) * 2;
            const uint4 w0 = __ldg(w), w1 = __ldg(w + 1);
#pragma unroll
            for (int m = 0; m < kMt; ++m) {
                mma_16816(d[m][0], h[m][q][0], h[m][q][1], h[m][q][2], h[m][q][3], w0.x, w0.y);
                mma_16816(d[m][1], h[m][q][0], h[m][q][1], h[m][q][2], h[m][q][3], w0.z, w0.w);
                mma_16816(d[m][2], h[m][q][0], h[m][q][1], h[m][q][2], h[m][q][3], w1.x, w1.y);
                mma_16816(d[m][3], h[m][q][0], h[m][q][1], h[m][q][2], h[m][q][3], w1.z, w1.w);
            }
        }
#pragma unroll
        for (int m = 0; m < kMt; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (!in || row[m][i] < 0) continue;
                half2* const o = reinterpret_cast<half2*>(&old[m][i]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 v = __half22float2(o[j]);
                    o[j] = __floats2half2_rn(fmaf(factor[m][i], d[m][j][2 * i], v.x), fmaf(factor[m][i], d[m][j][2 * i + 1], v.y));
                }
                *reinterpret_cast<uint4*>(p.out + row[m][i] * p.out_pitch + col) = old[m][i];
            }
    }
}

template <int kRt, int kMt, int kWk, bool kCluster>
cudaError_t launch(const AdapterParams& p, int tiles, int csize, cudaStream_t st) {
    const size_t smem = (size_t)(kWarps + kWarps / kWk * (kCluster ? 2 : 1)) * kMt * kRt * 2 * 32 * sizeof(float4);
    const auto kernel = adapter_kernel<kRt, kMt, kWk, kCluster>;
    static PerDeviceOnce once;
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * csize));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)csize;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = kCluster ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int kRt>
cudaError_t launch_for(const AdapterParams& p, cudaStream_t st) {
    constexpr int kBigMt = kRt <= 4 ? 2 : 1;     // a rank of 128 has no registers for two tiles' sums
    constexpr int kBigTile = kBigMt * 16;
    const bool big = kBigMt > 1 && p.cu_seqlens && p.tokens > 16 * p.batch;
    if (big) return launch<kRt, kBigMt, 8, false>(p, p.tokens / kBigTile + p.batch, 1, st);
    const int tiles = p.cu_seqlens ? p.tokens / 16 + p.batch : p.batch;
    int csize = 1;
    while (csize < kMaxCluster && tiles * csize * 2 <= sm_count() * 2) csize *= 2;
    return csize == 1 ? launch<kRt, 1, 8, false>(p, tiles, 1, st) : launch<kRt, 1, 8, true>(p, tiles, csize, st);
}

}  // namespace
}  // namespace et

struct et_adapter_bank {
    int in_feat, out_feat, max_rank, n_slots, rank_tiles, device;
    long long a_stride, b_stride;
    half *a = nullptr, *b = nullptr;
    et::Slot* slots = nullptr;
};

extern "C" int et_adapter_bank_create(et_adapter_bank** out, int in_feat, int out_feat, int max_rank, int n_slots) {
    using namespace et;
    ET_REQUIRE(out, "et_adapter_bank_create: null output");
    *out = nullptr;
    ET_REQUIRE(in_feat > 0 && out_feat > 0 && in_feat % 16 == 0 && out_feat % 16 == 0, "et_adapter_bank_create: in_feat and out_feat must be positive multiples of 16");
    ET_REQUIRE(max_rank >= 1 && max_rank <= kMaxRank, "et_adapter_bank_create: max_rank must be 1 to 128");
    ET_REQUIRE(n_slots >= 1, "et_adapter_bank_create: at least one slot");
    auto* bank = new (std::nothrow) et_adapter_bank;
    if (!bank) return fail(ET_ERR_CUDA, "et_adapter_bank_create: out of host memory");
    bank->in_feat = in_feat; bank->out_feat = out_feat; bank->max_rank = max_rank; bank->n_slots = n_slots;
    bank->rank_tiles = max_rank <= 16 ? 1 : max_rank <= 32 ? 2 : max_rank <= 64 ? 4 : 8;   // 16-wide steps: what the kernels are made for
    bank->a_stride = (long long)((in_feat + 31) / 32) * bank->rank_tiles * 2 * 256;
    bank->b_stride = (long long)((out_feat + 31) / 32) * bank->rank_tiles * 512;
    cudaError_t e = cudaGetDevice(&bank->device);
    if (e == cudaSuccess) e = cudaMalloc(&bank->a, (size_t)bank->a_stride * n_slots * sizeof(half));
    if (e == cudaSuccess) e = cudaMalloc(&bank->b, (size_t)bank->b_stride * n_slots * sizeof(half));
    if (e == cudaSuccess) e = cudaMalloc(&bank->slots, (size_t)n_slots * sizeof(Slot));
    if (e == cudaSuccess) e = cudaMemset(bank->slots, 0, (size_t)n_slots * sizeof(Slot));
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e != cudaSuccess) {
        et_adapter_bank_destroy(bank);
        return cuda_status(e, "et_adapter_bank_create");
    }
    *out = bank;
    return ET_OK;
}

extern "C" int et_adapter_bank_destroy(et_adapter_bank* bank) {
    if (!bank) return ET_OK;
    cudaFree(bank->a);
    cudaFree(bank->b);
    cudaFree(bank->slots);
    delete bank;
    return ET_OK;
}

extern "C" int et_adapter_bank_set(et_adapter_bank* bank, int slot, int rank, const void* a_host, const void* b_host, float scale) {
    using namespace et;
    ET_REQUIRE(bank, "et_adapter_bank_set: null bank");
    ET_REQUIRE(slot >= 0 && slot < bank->n_slots, "et_adapter_bank_set: no such slot");
    ET_REQUIRE(rank >= 0 && rank <= bank->max_rank, "et_adapter_bank_set: rank above the bank's largest");
    ET_REQUIRE(rank == 0 || (a_host && b_host), "et_adapter_bank_set: null pointer");
    int dev = -1;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_status(e, "et_adapter_bank_set");
    ET_REQUIRE(dev == bank->device, "et_adapter_bank_set: the bank belongs to another device");
    std::vector<half> pa, pb;
    try {
        pa.assign((size_t)bank->a_stride, __float2half(0.f));
        pb.assign((size_t)bank->b_stride, __float2half(0.f));
    } catch (...) {
        return fail(ET_ERR_CUDA, "et_adapter_bank_set: out of host memory");
    }
    const half* const A = static_cast<const half*>(a_host);   // [rank x in_feat]
    const half* const B = static_cast<const half*>(b_host);   // [out_feat x rank]
    // A: [chunk of 32 features][8 ranks][lane = rank * 4 + t][features 8t .. 8t + 7 of the chunk]
    for (int r = 0; r < rank; ++r)
        for (int k = 0; k < bank->in_feat; ++k) {
            const size_t tile = (size_t)(k / 32) * (bank->rank_tiles * 2) + r / 8;
            pa[(tile * 32 + (r % 8) * 4 + (k % 32) / 8) * 8 + k % 8] = A[(size_t)r * bank->in_feat + k];
        }
    // B: [group of 32 columns][16 ranks][lane][tile 0 .. 3][ranks 2t, 2t + 1, 2t + 8, 2t + 9]; column c of the group is column
    // 2 (c / 8) + c % 2 of tile (c / 2) % 4, which is the lane's number / 4
    for (int n = 0; n < bank->out_feat; ++n)
        for (int r = 0; r < rank; ++r) {
            const int c = n % 32, q = r % 16;
            const int lane = (2 * (c / 8) + c % 2) * 4 + (q % 8) / 2;
            const size_t tile = (size_t)(n / 32) * bank->rank_tiles + r / 16;
            pb[(tile * 32 + lane) * 16 + (c / 2) % 4 * 4 + q / 8 * 2 + q % 2] = B[(size_t)n * rank + r];
        }
    const Slot entry = {rank, scale};
    e = cudaDeviceSynchronize();   // launches that read the slot as it was have finished
    if (e == cudaSuccess) e = cudaMemcpy(bank->a + slot * bank->a_stride, pa.data(), pa.size() * sizeof(half), cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaMemcpy(bank->b + slot * bank->b_stride, pb.data(), pb.size() * sizeof(half), cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaMemcpy(bank->slots + slot, &entry, sizeof(entry), cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    return cuda_status(e, "et_adapter_bank_set");
}

extern "C" int et_adapter_add(const et_adapter_bank* bank, void* out, const void* base, const void* x, int out_pitch, int base_pitch, int x_pitch,
                              const int* cu_seqlens, const int* adapter_ids, int batch, int tokens, void* stream) {
    using namespace et;
    ET_REQUIRE(bank, "et_adapter_add: null bank");
    ET_REQUIRE(batch >= 0 && tokens >= 0, "et_adapter_add: negative size");
    if (batch == 0 || tokens == 0) return ET_OK;
    ET_REQUIRE(out && base && x && adapter_ids, "et_adapter_add: null pointer");
    ET_REQUIRE(cu_seqlens || batch <= tokens, "et_adapter_add: without cu_seqlens every sequence is one token");
    ET_REQUIRE(out_pitch >= bank->out_feat && base_pitch >= bank->out_feat && x_pitch >= bank->in_feat, "et_adapter_add: pitch below the width");
    ET_REQUIRE(out_pitch % 8 == 0 && base_pitch % 8 == 0 && x_pitch % 8 == 0 && aligned16(out) && aligned16(base) && aligned16(x),
               "et_adapter_add: rows must start on 16 bytes");
    ET_REQUIRE(out != base || out_pitch == base_pitch, "et_adapter_add: in place the pitches must be equal");
    int dev = -1;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_status(e, "et_adapter_add");
    ET_REQUIRE(dev == bank->device, "et_adapter_add: the bank belongs to another device");
    AdapterParams p;
    p.out = static_cast<half*>(out); p.base = static_cast<const half*>(base); p.x = static_cast<const half*>(x);
    p.cu_seqlens = cu_seqlens; p.ids = adapter_ids; p.slots = bank->slots; p.a = bank->a; p.b = bank->b;
    p.out_pitch = out_pitch; p.base_pitch = base_pitch; p.x_pitch = x_pitch; p.a_stride = bank->a_stride; p.b_stride = bank->b_stride;
    p.batch = batch; p.tokens = tokens; p.n_slots = bank->n_slots; p.in_feat = bank->in_feat; p.out_feat = bank->out_feat;
    p.copy = out != base;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int rt = bank->rank_tiles;
    const cudaError_t r = rt <= 1 ? launch_for<1>(p, st) : rt <= 2 ? launch_for<2>(p, st) : rt <= 4 ? launch_for<4>(p, st) : launch_for<8>(p, st);
    return cuda_status(r, "et_adapter_add launch");
}
