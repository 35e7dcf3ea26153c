// Low-rank adapters: what the two kernels share.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace et {

struct AdapterSlot {
    int rank;      // 0: nothing to add
    float scale;
};

struct AdapterParams {
    half* out;
    const half* base;
    const half* x;
    const int* cu_seqlens;
    const int* ids;
    const AdapterSlot* slots;
    const half *a, *b;                  // packed, of the first slot: for the kernel that is launched
    long long out_pitch, base_pitch, x_pitch, stride;   // stride: from slot to slot, in elements
    int batch, tokens, n_slots, in_feat, out_feat;
    int n_split;                        // CTAs that share a tile's columns, each with all of A x
    int* err;                           // of bounded waits
    bool copy;                          // out is not base: what has no adapter is copied
};

// The tile of `size` tokens with number `tile`: sequence, first token, tokens (whole warp). Without cu_seqlens a sequence is one token.
__device__ __forceinline__ int find_tile(const AdapterParams& p, int tile, int size, int& seq, int& t0) {
    const int lane = threadIdx.x & 31;
    if (!p.cu_seqlens) {
        seq = t0 = tile;
        return tile < p.batch ? 1 : 0;
    }
    for (int base = 0; base < p.batch; base += 128) {   // four sequences to a lane
        int first[5], n[4];
#pragma unroll
        for (int j = 0; j < 5; ++j) first[j] = p.cu_seqlens[min(base + lane * 4 + j, p.batch)];   // (behind the last one all are empty)
#pragma unroll
        for (int j = 0; j < 4; ++j) n[j] = (max(first[j + 1] - first[j], 0) + size - 1) / size;
        const int sum = n[0] + n[1] + n[2] + n[3];
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, tile < incl);
        if (hit) {
            const int src = __ffs(hit) - 1;
            int left = tile - (incl - sum), at = 0;   // (of the lane that has it)
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (at == j && left >= n[j]) {
                    left -= n[j];
                    ++at;
                }
            const int from = at == 0 ? first[0] : at == 1 ? first[1] : at == 2 ? first[2] : first[3], to = at == 0 ? first[1] : at == 1 ? first[2] : at == 2 ? first[3] : first[4];
            seq = base + src * 4 + __shfl_sync(0xffffffffu, at, src);
            t0 = __shfl_sync(0xffffffffu, from + left * size, src);
            const int end = min(__shfl_sync(0xffffffffu, to, src), p.tokens);   // (never beyond the rows that there are)
            return t0 < 0 ? 0 : max(min(end - t0, size), 0);
        }
        tile -= __shfl_sync(0xffffffffu, incl, 31);
    }
    return 0;
}

// The power of two (its exponent's bits) that brings a row of A x with that largest value into [1, 2): infinity stays one; below 2^-100 it makes no difference
// to the result.
__device__ __forceinline__ int row_exponent(float top) {
    const int e = __float_as_int(top) >> 23;
    return e == 255 ? 127 : max(27, min(e, 227));
}

// tcgen05 kernel for many tokens (adapter_tc.cu): rank_step 16, 32, 64 or 128, the rank that the bank's slots are laid out for.
int adapter_tc_launch(AdapterParams p, int rank_step, cudaStream_t st);
// Elements of A and B in the layouts that it takes, and the layouts: A [chunk of 64 features][rank_step][64] with 128-byte swizzle, B [unit of 64 columns]
// [8 columns][8 ranks] as core matrices of 8 columns x 16 bytes.
long long adapter_tc_a_stride(int in_feat, int rank_step);
long long adapter_tc_b_stride(int out_feat, int rank_step);
void adapter_tc_pack(half* pa, half* pb, const half* A, const half* B, int rank, int in_feat, int out_feat, int rank_step);

}  // namespace et
