// Low-rank adapters of many requests beside a shared projection: out_t = base_t + scale_a B_a (A_a x_t), a the adapter of token t's sequence. The bank, the entry
// points, and the kernel for few tokens (adapter_tc.cu has that for many).
//
// A bank holds the adapters of one projection in the order in which the tensor cores take them: for this kernel so that a warp loads its fragments of
// A and B with 16 bytes a lane, side by side, and needs no shared memory for them (they come from L1 and L2, where a bank stays), and as shared memory
// wants them for the other.
// One launch does both products. 16 tokens of one sequence are a CTA's work: its eight warps each take a share of the K range for A x, the
// shares are added in shared memory, and each takes a share of the output columns for B (A x). CTAs share a tile's columns where there are few tiles, each with all of A x.
//
// Sums are fp32. A x is rounded to fp16 between the products, as the second one needs it, each row scaled by a power of two so that its
// largest value lies in [1, 2): it can not overflow, and the rounding (2^-11 of a term of the delta) is that of the result's own type.
// Both products' fragments are permuted so that a lane has eight neighbouring elements of X, of base and of the result: the sum over k
// does not depend on the order of k, and which column a lane of the second product computes is free.
//
// What bounds it: latency, the chain id -> A x -> exchange -> B. 64 single tokens, 1024 -> 1024, rank 16: 4.0 us; nine sequences of 1.1 thousand tokens, 768 -> 2304, rank 8:
// 6.8 us. Tried: clusters of 2, 4, 8 CTAs that share a tile's K range and columns through distributed shared memory (single tokens 5.0, 5.3, 7.3 us).
#include <cstring>
#include <new>
#include <vector>
#include "adapter.h"
#include "attention.h"
#include "common.h"
#include "ptx.cuh"
#include "tmap.h"

namespace et {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kTile = 16, kMaxRank = 128;

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

// kRt: 16-wide steps of the bank's largest rank.
template <int kRt>
__global__ void __launch_bounds__(kThreads, 1) adapter_kernel(const __grid_constant__ AdapterParams p) {
    constexpr int kFrags = kRt * 2;                        // accumulator fragments of a warp
    extern __shared__ float4 parts[];                      // [kWarps][kFrags][32]: shares of A x, as accumulator fragments; then their sums [kFrags][32]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    pdl_launch_dependents();
    pdl_wait();
    int seq = 0, t0 = 0;
    const int rows_in_tile = find_tile(p, blockIdx.x / p.n_split, kTile, seq, t0);
    if (rows_in_tile <= 0) return;
    const int id = p.ids[seq];
    AdapterSlot slot = {0, 0.f};
    if (id >= 0 && id < p.n_slots) slot = p.slots[id];
    const int all_groups = (p.out_feat + 31) / 32, split = blockIdx.x % p.n_split;
    const int first_group = split * all_groups / p.n_split, col_groups = (split + 1) * all_groups / p.n_split;
    const int row[2] = {g < rows_in_tile ? t0 + g : -1, g + 8 < rows_in_tile ? t0 + g + 8 : -1};   // the lane's rows, -1 beyond the tile
    if (slot.rank == 0) {
        if (!p.copy) return;
        for (int c = first_group + warp; c < col_groups; c += kWarps) {
            const int col = c * 32 + t * 8;
            if (col >= p.out_feat) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (row[i] >= 0) *reinterpret_cast<uint4*>(p.out + row[i] * p.out_pitch + col) = *reinterpret_cast<const uint4*>(p.base + row[i] * p.base_pitch + col);
        }
        return;
    }
    // ---- A x: chunks of 32 features; a lane has eight neighbouring ones of its two rows, the operands of two steps of 16
    float acc[kFrags][4];
#pragma unroll
    for (int j = 0; j < kFrags; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
    const int chunks = (p.in_feat + 31) / 32;
    const uint4* const a = reinterpret_cast<const uint4*>(p.a + id * p.stride);
    constexpr int kUnroll = 4;
    for (int c0 = warp; c0 < chunks; c0 += kWarps * kUnroll) {
        uint4 xv[kUnroll][2];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int k = (c0 + u * kWarps) * 32 + t * 8;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                xv[u][i] = make_uint4(0u, 0u, 0u, 0u);
                if (k < p.in_feat && row[i] >= 0) xv[u][i] = *reinterpret_cast<const uint4*>(p.x + row[i] * p.x_pitch + k);
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int c = c0 + u * kWarps;
            if (c >= chunks) break;
#pragma unroll
            for (int j = 0; j < kFrags; ++j) {
                const uint4 w = __ldg(a + ((size_t)c * kFrags + j) * 32 + lane);
                mma_16816(acc[j], xv[u][0].x, xv[u][1].x, xv[u][0].y, xv[u][1].y, w.x, w.y);
                mma_16816(acc[j], xv[u][0].z, xv[u][1].z, xv[u][0].w, xv[u][1].w, w.z, w.w);
            }
        }
    }
    const uint4* const b = reinterpret_cast<const uint4*>(p.b + id * p.stride);
    uint4 old_next[2], w_next[kRt][2];
    auto request = [&](int c) {
        if (c >= col_groups) return;
        const int col = c * 32 + t * 8;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (col < p.out_feat && row[i] >= 0) old_next[i] = *reinterpret_cast<const uint4*>(p.base + row[i] * p.base_pitch + col);
#pragma unroll
        for (int q = 0; q < kRt; ++q) {
            const uint4* const w = b + (((size_t)c * kRt + q) * 32 + lane) * 2;
            w_next[q][0] = __ldg(w);
            w_next[q][1] = __ldg(w + 1);
        }
    };
    request(first_group + warp);   // before the shares are exchanged
    // ---- the shares are added, in the order of the warps: each thread adds a few places of all of them
    float4* const sums = parts + kWarps * kFrags * 32;
#pragma unroll
    for (int j = 0; j < kFrags; ++j) parts[(warp * kFrags + j) * 32 + lane] = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
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
    for (int j = 0; j < kFrags; ++j) {
        const float4 v = sums[j * 32 + lane];
        acc[j][0] = v.x; acc[j][1] = v.y; acc[j][2] = v.z; acc[j][3] = v.w;
    }
    // ---- to fp16, each row by a power of two of its own; ranks that only pad a step are zeros even where x is not finite
    float top[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kFrags; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (j * 8 + 2 * t + i >= slot.rank) acc[j][i] = acc[j][i + 2] = 0.f;
            top[0] = fmaxf(top[0], fabsf(acc[j][i]));
            top[1] = fmaxf(top[1], fabsf(acc[j][i + 2]));
        }
    float down[2], factor[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        const int ex = row_exponent(top[i]);
        down[i] = __int_as_float((254 - ex) << 23);
        factor[i] = slot.scale * __int_as_float(ex << 23);
    }
    uint32_t h[kRt][4];
#pragma unroll
    for (int q = 0; q < kRt; ++q) {
        h[q][0] = pack_h2(acc[2 * q][0] * down[0], acc[2 * q][1] * down[0]);
        h[q][1] = pack_h2(acc[2 * q][2] * down[1], acc[2 * q][3] * down[1]);
        h[q][2] = pack_h2(acc[2 * q + 1][0] * down[0], acc[2 * q + 1][1] * down[0]);
        h[q][3] = pack_h2(acc[2 * q + 1][2] * down[1], acc[2 * q + 1][3] * down[1]);
    }
    // ---- base + B (A x): groups of 32 columns, of which a lane has eight neighbouring ones in each of its rows
    for (int c = first_group + warp; c < col_groups; c += kWarps) {
        const int col = c * 32 + t * 8;
        uint4 old[2], w[kRt][2];
#pragma unroll
        for (int q = 0; q < kRt; ++q) {
            w[q][0] = w_next[q][0];
            w[q][1] = w_next[q][1];
        }
        old[0] = old_next[0];
        old[1] = old_next[1];
        request(c + kWarps);
        float d[4][4];
        product(d, h, w);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (col >= p.out_feat || row[i] < 0) continue;
            add_to(old[i], d, i, factor[i]);
            *reinterpret_cast<uint4*>(p.out + row[i] * p.out_pitch + col) = old[i];
        }
    }
}

template <int kRt>
int launch(AdapterParams p, cudaStream_t st) {
    constexpr size_t smem = (size_t)(kWarps + 1) * kRt * 2 * 32 * sizeof(float4);
    const auto kernel = adapter_kernel<kRt>;
    static PerDeviceOnce once;
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); });
    if (e != cudaSuccess) return cuda_status(e, "et_adapter_add");
    // A tile's columns are shared by as many CTAs as all find a place at once (by their registers three, two or one to an SM), each with 18 groups of columns at least.
    // (Nine sequences of 1.1 thousand tokens, 768 -> 2304, rank 8, in two, three, four CTAs to a tile 8.4, 7.3, 6.8 us, in more than there are places for 9.5; 64 single tokens, 1024 -> 4096,
    // rank 128, in one round 11.2, in two 16.2; 64 single tokens, 1024 -> 1024, rank 16, in one CTA to a tile 4.0, in two 4.2.)
    constexpr int kPlaces = kRt == 1 ? 3 : kRt == 8 ? 1 : 2;
    const long long tiles = p.cu_seqlens ? (long long)p.tokens / kTile + p.batch : p.batch;
    p.n_split = (int)max(1LL, min((long long)kPlaces * sm_count() / tiles, (long long)((p.out_feat + 31) / 32 / 18)));
    return cuda_status(launch_pdl(kernel, dim3((unsigned)(tiles * p.n_split)), dim3(kThreads), smem, st, p), "et_adapter_add launch");
}

}  // namespace
}  // namespace et

struct et_adapter_bank {
    int in_feat, out_feat, max_rank, n_slots, rank_tiles, device;
    long long b_at, a_tc_at, b_tc_at, stride;   // of a slot, in elements: where its parts begin (A at 0; for many tokens A and B), all of it
    half* weights = nullptr;
    et::AdapterSlot* slots = nullptr;
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
    bank->b_at = (long long)((in_feat + 31) / 32) * bank->rank_tiles * 2 * 256;
    bank->a_tc_at = bank->b_at + (long long)((out_feat + 31) / 32) * bank->rank_tiles * 512;
    bank->b_tc_at = bank->a_tc_at + adapter_tc_a_stride(in_feat, bank->rank_tiles * 16);
    bank->stride = bank->b_tc_at + adapter_tc_b_stride(out_feat, bank->rank_tiles * 16);
    cudaError_t e = cudaGetDevice(&bank->device);
    if (e == cudaSuccess) e = cudaMalloc(&bank->weights, (size_t)bank->stride * n_slots * sizeof(half));
    if (e == cudaSuccess) e = cudaMalloc(&bank->slots, (size_t)n_slots * sizeof(AdapterSlot));
    if (e == cudaSuccess) e = cudaMemset(bank->slots, 0, (size_t)n_slots * sizeof(AdapterSlot));
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
    cudaFree(bank->weights);
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
    std::vector<half> packed;
    try {
        packed.assign((size_t)bank->stride, __float2half(0.f));
    } catch (...) {
        return fail(ET_ERR_CUDA, "et_adapter_bank_set: out of host memory");
    }
    half *const pa = packed.data(), *const pb = pa + bank->b_at;
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
    adapter_tc_pack(pa + bank->a_tc_at, pa + bank->b_tc_at, A, B, rank, bank->in_feat, bank->out_feat, bank->rank_tiles * 16);
    const AdapterSlot entry = {rank, scale};
    e = cudaDeviceSynchronize();   // launches that read the slot as it was have finished
    if (e == cudaSuccess && rank > 0) e = cudaMemcpy(bank->weights + slot * bank->stride, pa, packed.size() * sizeof(half), cudaMemcpyHostToDevice);
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
    p.cu_seqlens = cu_seqlens; p.ids = adapter_ids; p.slots = bank->slots; p.a = bank->weights; p.b = bank->weights + bank->b_at;
    p.out_pitch = out_pitch; p.base_pitch = base_pitch; p.x_pitch = x_pitch; p.stride = bank->stride;
    p.batch = batch; p.tokens = tokens; p.n_slots = bank->n_slots; p.in_feat = bank->in_feat; p.out_feat = bank->out_feat;
    p.copy = out != base;
    const int rc = attn_err_address(&p.err);
    if (rc) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int rt = bank->rank_tiles;
    // The tensor cores' kernel where there is enough to do: it takes some 10 us however little that is, but reads the weights for 64 to 128 tokens where the other
    // reads them for 16. (8 sequences of 6205 tokens, 1024 -> 4096, rank 32: 25 us, 41 in the other; 16 of 2055: 20 and 14; 768 -> 768, rank 16, 32 of 8509: 12.4 and 12.2. Of short sequences
    // its tiles are mostly empty: 1000 sequences of 24 tokens, 1024 -> 1024, rank 16: 84 and 49, 200 of 50, 768 -> 2304: 34 and 30, 128 of 64, 1024 -> 1024: 16 and 17.)
    if (cu_seqlens && tokens >= 56LL * batch && (tokens >= 8192 || (long long)tokens * (bank->in_feat + 2LL * bank->out_feat) >= 30'000'000)) {
        p.a = bank->weights + bank->a_tc_at;
        p.b = bank->weights + bank->b_tc_at;
        return adapter_tc_launch(p, rt * 16, st);
    }
    return rt <= 1 ? launch<1>(p, st) : rt <= 2 ? launch<2>(p, st) : rt <= 4 ? launch<4>(p, st) : launch<8>(p, st);
}

extern "C" int et_adapter_add_by(const et_adapter_add_args* a) {
    ET_REQUIRE(a, "et_adapter_add_by: null pointer");
    return et_adapter_add(a->bank, a->out, a->base, a->x, a->out_pitch, a->base_pitch, a->x_pitch, a->cu_seqlens, a->adapter_ids, a->batch, a->tokens, a->stream);
}
