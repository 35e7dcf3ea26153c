// Low-rank adapters of many requests beside a shared projection: out_t = base_t + scale_a B_a (A_a x_t), a the adapter of token t's sequence.
//
// A bank holds the adapters of one projection in the order in which the tensor cores take them, so that a warp loads its fragments of
// A and B with 16 bytes a lane, side by side, and needs no shared memory for them: they come from L1 and L2, where a bank stays.
// One launch does both products. 16 or 32 tokens of one sequence are a CTA's work: its eight warps each take a share of the K range for A x, the
// shares are added in shared memory, and each takes a share of the output columns for B (A x). Where there are many tokens base and out move by TMA, 64
// columns at a time through a ring of each warp; where there are few, CTAs share a tile's columns, each with all of A x.
//
// Sums are fp32. A x is rounded to fp16 between the products, as the second one needs it, each row scaled by a power of two so that its
// largest value lies in [1, 2): it can not overflow, and the rounding (2^-11 of a term of the delta) is that of the result's own type.
// Both products' fragments are permuted so that a lane has eight neighbouring elements of X, of base and of the result: the sum over k
// does not depend on the order of k, and which column a lane of the second product computes is free.
//
// What bounds it: X is read once, base read and out written once; two operations a byte and rank, far below what mma.sync delivers. 32 prompts of 18 thousand
// tokens, 1024 -> 4096, rank 32: 88 us, 61 at copy bandwidth (a plain copy of base in tiles of 32 rows takes 55); the rest is the weights, which every
// tile of 32 tokens reads again (195 MB beside 340, from L2: rings of two stages, which leave them more of L1, gain 6 us over three), and the start of a
// tile. 64 single tokens 4.0 us. Tried: clusters of 2, 4, 8 CTAs that share a tile's K range and columns through distributed shared memory (103, 131, 235 us;
// single tokens 5.0, 5.3, 7.3), tiles of 64 tokens (103), CTAs that share the columns where there are many tokens (91).
#include <cstring>
#include <new>
#include <vector>
#include "attention.h"
#include "common.h"
#include "ptx.cuh"
#include "tmap.h"

namespace et {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kMaxRank = 128;

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
    int n_split;                        // CTAs that share a tile's columns, each with all of A x
    int* err;                           // of bounded waits
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

// 16 rows and 32 columns of B (A x): the lane's columns 8t .. 8t + 7 of rows g (elements 0 and 1 of each fragment) and g + 8 (2 and 3).
template <int kRt>
__device__ __forceinline__ void product(float (&d)[4][4], const uint32_t (&h)[kRt][4], const uint4 (&w)[kRt][2]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[j][i] = 0.f;
#pragma unroll
    for (int q = 0; q < kRt; ++q) {
        mma_16816(d[0], h[q][0], h[q][1], h[q][2], h[q][3], w[q][0].x, w[q][0].y);
        mma_16816(d[1], h[q][0], h[q][1], h[q][2], h[q][3], w[q][0].z, w[q][0].w);
        mma_16816(d[2], h[q][0], h[q][1], h[q][2], h[q][3], w[q][1].x, w[q][1].y);
        mma_16816(d[3], h[q][0], h[q][1], h[q][2], h[q][3], w[q][1].z, w[q][1].w);
    }
}
// Adds it to eight elements of base; i: which of the two rows.
__device__ __forceinline__ void add_to(uint4& old, const float (&d)[4][4], int i, float factor) {
    half2* const o = reinterpret_cast<half2*>(&old);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 v = __half22float2(o[j]);
        o[j] = __floats2half2_rn(fmaf(factor, d[j][2 * i], v.x), fmaf(factor, d[j][2 * i + 1], v.y));
    }
}

// Where base passes through, by warps.
template <int kMt>
struct Ring {
    static constexpr int kStage = kMt * 16 * 128;          // 64 columns of a tile's rows, 128-byte swizzle
    static constexpr int kStages = 2;
    static constexpr int kBarAt = kWarps * kStages * kStage;
    static constexpr int kBytes = kBarAt + kWarps * kStages * 8 + 1024;
};

// The tile of kTile tokens with number `tile`: sequence, first token, tokens (whole warp). Without cu_seqlens a sequence is one token.
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

// kRt: 16-wide steps of the bank's largest rank; kMt: 16-token tiles of a CTA. kTma: base and out move by TMA, 64 columns of a
// tile at a time, through a ring of each warp; only a tile that ends inside a sequence's last rows is written row by row.
template <int kRt, int kMt, bool kTma>
__global__ void __launch_bounds__(kThreads, kTma && kRt <= 4 ? 2 : 1) adapter_kernel(const __grid_constant__ AdapterParams p, const __grid_constant__ CUtensorMap tm_base,
                                                           const __grid_constant__ CUtensorMap tm_out) {
    constexpr int kTile = kMt * 16;
    constexpr int kFrags = kMt * kRt * 2;                  // accumulator fragments of a warp
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = kTma ? (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023) : smem_raw;
    float4* const parts = reinterpret_cast<float4*>(smem);   // [kWarps][kFrags][32]: shares of A x, as accumulator fragments; then their sums
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    pdl_launch_dependents();
    pdl_wait();
    int seq = 0, t0 = 0;
    const int rows_in_tile = find_tile<kTile>(p, blockIdx.x / p.n_split, seq, t0);
    if (rows_in_tile <= 0) return;
    const int id = p.ids[seq];
    Slot slot = {0, 0.f};
    if (id >= 0 && id < p.n_slots) slot = p.slots[id];
    const int all_groups = (p.out_feat + 31) / 32, split = blockIdx.x % p.n_split;
    const int first_group = split * all_groups / p.n_split, col_groups = (split + 1) * all_groups / p.n_split;
    int row[kMt][2];        // the lane's rows, -1 beyond the tile
#pragma unroll
    for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = m * 16 + h * 8 + g;
            row[m][h] = r < rows_in_tile ? t0 + r : -1;
        }
    if (slot.rank == 0) {
        if (!p.copy) return;
        for (int c = first_group + warp; c < col_groups; c += kWarps) {
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
    constexpr int kUnroll = kMt == 1 ? 4 : kMt == 2 ? 2 : 1;
    for (int c0 = warp; c0 < chunks; c0 += kWarps * kUnroll) {
        uint4 xv[kUnroll][kMt][2];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int k = (c0 + u * kWarps) * 32 + t * 8;
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
            const int c = c0 + u * kWarps;
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
    const uint4* const b = reinterpret_cast<const uint4*>(p.b + id * p.b_stride);
    uint4 old_next[kMt][2], w_next[kRt][2];
    auto request = [&](int c) {
        if (c >= col_groups) return;
        const int col = c * 32 + t * 8;
#pragma unroll
        for (int m = 0; m < kMt; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (col < p.out_feat && row[m][i] >= 0) old_next[m][i] = *reinterpret_cast<const uint4*>(p.base + row[m][i] * p.base_pitch + col);
#pragma unroll
        for (int q = 0; q < kRt; ++q) {
            const uint4* const w = b + (((size_t)c * kRt + q) * 32 + lane) * 2;
            w_next[q][0] = __ldg(w);
            w_next[q][1] = __ldg(w + 1);
        }
    };
    if constexpr (!kTma) request(first_group + warp);   // before the shares are exchanged
    // ---- the shares are added, in the order of the warps: each thread adds a few places of all of them
    float4* const sums = parts + kWarps * kFrags * 32;     // [kFrags][32]
#pragma unroll
    for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int j = 0; j < kRt * 2; ++j)
            parts[(warp * kFrags + m * kRt * 2 + j) * 32 + lane] = make_float4(acc[m][j][0], acc[m][j][1], acc[m][j][2], acc[m][j][3]);
    __syncthreads();
    for (int e = threadIdx.x; e < kFrags * 32; e += kThreads) {
        float4 s = parts[e];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            const float4 v = parts[w * kFrags * 32 + e];
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        sums[e] = s;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int j = 0; j < kRt * 2; ++j) {
            const float4 v = sums[(m * kRt * 2 + j) * 32 + lane];
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
    if constexpr (kTma) {
        // ---- base + B (A x): units of 64 columns. A unit's base lands in a stage, is added to there and leaves from there.
        using R = Ring<kMt>;
        const uint32_t ring = smem_u32(smem) + warp * R::kStages * R::kStage, bars = smem_u32(smem) + R::kBarAt + warp * R::kStages * 8;
        if (lane == 0) {
            for (int i = 0; i < R::kStages; ++i) mbar_init(reinterpret_cast<uint64_t*>(smem + R::kBarAt) + warp * R::kStages + i, 1);
            fence_mbar_init();
            fence_proxy_async_smem();
        }
        __syncthreads();   // everyone has read the sums, which lie where the rings are
        const int first_unit = split * ((p.out_feat + 63) / 64) / p.n_split, units = (split + 1) * ((p.out_feat + 63) / 64) / p.n_split;
        const bool whole = rows_in_tile == kTile;
        auto fetch = [&](int u, int stage) {
            if (lane == 0 && u < units) {
                mbar_expect_tx_at(bars + stage * 8, R::kStage);
                tma_load_2d_at(ring + stage * R::kStage, &tm_base, u * 64, t0, bars + stage * 8);
            }
        };
#pragma unroll
        for (int i = 0; i < R::kStages - 1; ++i) fetch(first_unit + warp + i * kWarps, i);
        auto weights = [&](uint4 (&w)[kRt][2], int c) {
            if (c >= all_groups) return;
#pragma unroll
            for (int q = 0; q < kRt; ++q) {
                const uint4* const from = b + (((size_t)c * kRt + q) * 32 + lane) * 2;
                w[q][0] = __ldg(from);
                w[q][1] = __ldg(from + 1);
            }
        };
        uint4 w[2][kRt][2];
        weights(w[0], (first_unit + warp) * 2);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int u = first_unit + warp; u < units; u += kWarps) {
            weights(w[1], u * 2 + 1);
            ok = mbar_wait_at(bars + stage * 8, phase);
            if (!ok) break;
            const uint32_t at = ring + stage * R::kStage;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (u * 2 + x >= all_groups) break;
                const int col = u * 64 + x * 32 + t * 8;
#pragma unroll
                for (int m = 0; m < kMt; ++m) {
                    float d[4][4];
                    product(d, h[m], w[x]);
                    if (x == 0 && m == kMt - 1) weights(w[0], (u + kWarps) * 2);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = m * 16 + i * 8 + g;
                        const uint32_t place = at + r * 128 + (((x * 4 + t) ^ (r & 7)) << 4);
                        uint4 old = lds128(place);
                        add_to(old, d, i, factor[m][i]);
                        if (whole) sts128(place, old);
                        else if (col < p.out_feat && row[m][i] >= 0) *reinterpret_cast<uint4*>(p.out + row[m][i] * p.out_pitch + col) = old;
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (whole) tma_store_2d_at(&tm_out, at, u * 64, t0);
                tma_store_commit();
                tma_store_wait_read_but_one();   // the unit before this one has left its stage
            }
            fetch(u + (R::kStages - 1) * kWarps, stage == 0 ? R::kStages - 1 : stage - 1);
            if (++stage == R::kStages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (lane == 0) tma_store_wait();
        if (!ok) {   // (copies on their way land before the CTA leaves; bounded)
            if (lane == 0) atomicExch(p.err, 51);
            for (int i = 0; i < R::kStages; ++i) mbar_wait_at(bars + i * 8, i < stage ? phase ^ 1u : phase);
        }
    } else
    // ---- base + B (A x): groups of 32 columns, of which a lane has eight neighbouring ones in each of its rows
    for (int c = first_group + warp; c < col_groups; c += kWarps) {
        const int col = c * 32 + t * 8;
        uint4 old[kMt][2], w[kRt][2];
#pragma unroll
        for (int q = 0; q < kRt; ++q) {
            w[q][0] = w_next[q][0];
            w[q][1] = w_next[q][1];
        }
#pragma unroll
        for (int m = 0; m < kMt; ++m) {
            old[m][0] = old_next[m][0];
            old[m][1] = old_next[m][1];
        }
        request(c + kWarps);
#pragma unroll
        for (int m = 0; m < kMt; ++m) {
            float d[4][4];
            product(d, h[m], w);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (col >= p.out_feat || row[m][i] < 0) continue;
                add_to(old[m][i], d, i, factor[m][i]);
                *reinterpret_cast<uint4*>(p.out + row[m][i] * p.out_pitch + col) = old[m][i];
            }
        }
    }
}

template <int kRt, int kMt, bool kTma>
cudaError_t launch(const AdapterParams& p, const CUtensorMap& tm_base, const CUtensorMap& tm_out, long long tiles, cudaStream_t st) {
    constexpr size_t sums = (size_t)(kWarps + 1) * kMt * kRt * 2 * 32 * sizeof(float4);
    constexpr size_t smem = kTma && Ring<kMt>::kBytes > sums + 1024 ? Ring<kMt>::kBytes : sums + (kTma ? 1024 : 0);
    const auto kernel = adapter_kernel<kRt, kMt, kTma>;
    static PerDeviceOnce once;
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); });
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3((unsigned)(tiles * p.n_split)), dim3(kThreads), smem, st, p, tm_base, tm_out);
}

template <int kRt>
int launch_for(AdapterParams p, cudaStream_t st) {
    constexpr int kBigMt = kRt <= 4 ? 2 : 1;     // a rank of 128 has no registers for two tiles' sums
    CUtensorMap tm_base = {}, tm_out = {};
    // Tiles of 32 tokens where they give every SM two CTAs; with fewer tokens, or sequences that would not fill a tile, tiles of 16, whose columns are
    // shared by CTAs as long as each warp has three groups of them. (1100 tokens of nine sequences, 768 -> 2304, rank 8: 11.0 us in the former form, 7.5 in the latter;
    // single tokens of 64 sequences, 1024 -> 1024: 4.0 us, with two CTAs to a tile 4.2.)
    const long long big_tiles = p.tokens / (kBigMt * 16) + p.batch;
    if (p.cu_seqlens && p.tokens > 16 * p.batch && big_tiles > 2 * sm_count()) {
        p.n_split = 1;
        if (!make_tmap_2d_f16(&tm_base, p.base, p.tokens, p.out_feat, p.base_pitch, kBigMt * 16, 64, 128) ||
            !make_tmap_2d_f16(&tm_out, p.out, p.tokens, p.out_feat, p.out_pitch, kBigMt * 16, 64, 128))
            return fail(ET_ERR_CUDA, "et_adapter_add: cuTensorMapEncodeTiled failed");
        return cuda_status(launch<kRt, kBigMt, true>(p, tm_base, tm_out, big_tiles, st), "et_adapter_add launch");
    }
    const long long tiles = p.cu_seqlens ? p.tokens / 16 + p.batch : p.batch;
    p.n_split = (int)max(1LL, min(2LL * sm_count() / tiles, (long long)((p.out_feat + 31) / 32 / (3 * kWarps))));
    return cuda_status(launch<kRt, 1, false>(p, tm_base, tm_out, tiles, st), "et_adapter_add launch");
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
        for (int k = 0; k < bank->in_feat; k += 8) {
            const size_t tile = (size_t)(k / 32) * (bank->rank_tiles * 2) + r / 8;
            std::memcpy(&pa[(tile * 32 + (r % 8) * 4 + (k % 32) / 8) * 8], A + (size_t)r * bank->in_feat + k, 16);
        }
    // B: [group of 32 columns][16 ranks][lane][tile 0 .. 3][ranks 2t, 2t + 1, 2t + 8, 2t + 9]; column c of the group is column
    // 2 (c / 8) + c % 2 of tile (c / 2) % 4, which is the lane's number / 4
    for (int n = 0; n < bank->out_feat; ++n) {
        const int c = n % 32;
        half* const column = &pb[((size_t)(n / 32) * bank->rank_tiles * 32 + (2 * (c / 8) + c % 2) * 4) * 16 + (c / 2) % 4 * 4];
        for (int r = 0; r < rank; ++r) column[(size_t)(r / 16) * 512 + (r % 8) / 2 * 16 + r % 16 / 8 * 2 + r % 2] = B[(size_t)n * rank + r];
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
    const int rc = attn_err_address(&p.err);
    if (rc) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int rt = bank->rank_tiles;
    return rt <= 1 ? launch_for<1>(p, st) : rt <= 2 ? launch_for<2>(p, st) : rt <= 4 ? launch_for<4>(p, st) : launch_for<8>(p, st);
}
