// Low-rank adapters of many requests, many tokens: out_t = base_t + scale_a B_a (A_a x_t), both products by tcgen05.
//
// Up to 128 tokens of one sequence are a tile, a CTA's work. A x accumulates in tensor memory over chunks of 64 features (M 128, N the rank), is brought to fp16
// there, each row scaled by a power of two so that its largest value lies in [1, 2), and is the A operand of the second product from where it lies: 64 columns
// at a time (N 64, K the rank) into two places, so that one is multiplied while the other is added to base. Rows that the tile has not are multiplied too, with
// whatever lies there: rows do not mix, and those are not written.
// One ring of shared memory carries everything: a stage is the tile's rows of 128 bytes, of x and then of base, and the weights that go with them (64 features of A, 64
// columns of B: as many bytes), which lie in global memory as shared memory wants them and come by one bulk copy. The loads of base run ahead while A x is
// still taken. Four warps add, a row to a thread: base is read from its stage and the result written there, from where a warp of its own sends it off by TMA, in one piece, or in
// pieces of eight rows where a sequence ends (what is left of eight is written by its threads).
//
// What bounds it: x and base are read and the result is written once; the weights come from L2 once for a tile (of 72 rows, rank 32, 1024 -> 4096: 327 KB beside 1.3 MB). 32 prompts
// of 21 thousand tokens, 1024 -> 4096, rank 32: 76 us, 61 at copy bandwidth, 5.2 TB/s (ncu: DRAM 306 MB for 333 MB of operands, L2 702 MB, the tensor pipe 10 %); the rest is the start, while only
// x is read, and the end. 18966 tokens with rank 128: 79 us; 4096 -> 1024 with rank 64: 50 us. Before, mma.sync with fragments from L1 and L2, tiles of 32 tokens (16 with
// rank 128) and base through rings of the warps: 88, 183, 99 us. Tried: every warp sending its own 32 rows off 71 us where this takes 70 (66 and 53 with ranks of 32
// and 64 in whole tiles against 65 and 50), eight adding warps that take turns 78; a ring of ten stages with one CTA to an SM gains nothing (67 against 65).
#include <cstring>
#include "adapter.h"
#include "attention.h"
#include "common.h"
#include "ptx.cuh"
#include "tmap.h"

namespace et {
namespace {

constexpr int kAddWarps = 4, kLoadWarp = 4, kMmaWarp = 5, kStoreWarp = 6, kThreads = 7 * 32;
constexpr int kRowBytes = 128;                       // of a row in a stage
constexpr int kMaxTile = 128, kMaxStages = 12;
constexpr uint32_t kTmemCols = 256;
constexpr int kSmemForCta = 112 * 1024;              // two CTAs to an SM

struct Barriers {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t written[kMaxStages];   // units of 64 columns in turn: the tile's rows are in the stage (or written)
    uint64_t low_full, low_ready;   // A x is summed; is there in fp16
    uint64_t sum_full[2], sum_empty[2];
    uint32_t tmem_base;
};

// A ring of stages as one role walks it.
struct RingAt {
    int stage = 0;
    uint32_t wraps = 0;
    __device__ __forceinline__ void next(int stages) {
        if (++stage == stages) {
            stage = 0;
            ++wraps;
        }
    }
};

template <int kR>
__global__ void __launch_bounds__(kThreads, 2) adapter_tc_kernel(const __grid_constant__ AdapterParams p, const int tile_rows, const int stages, const __grid_constant__ CUtensorMap tm_x,
                                                                 const __grid_constant__ CUtensorMap tm_base, const __grid_constant__ CUtensorMap tm_out,
                                                                 const __grid_constant__ CUtensorMap tm_out8) {
    constexpr int kWeights = kR * 128;                 // 64 features of A, or 64 columns of B
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ Barriers barriers;
    Barriers* const sh = &barriers;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (warp == kLoadWarp) {
        if (lane == 0) {
            for (int i = 0; i < stages; ++i) {
                mbar_init(&sh->full[i], 1);
                mbar_init(&sh->empty[i], 1);
                mbar_init(&sh->written[i], kAddWarps);
            }
            mbar_init(&sh->low_full, 1);
            mbar_init(&sh->low_ready, kAddWarps);
            for (int i = 0; i < 2; ++i) {
                mbar_init(&sh->sum_full[i], 1);
                mbar_init(&sh->sum_empty[i], kAddWarps);
            }
            fence_mbar_init();
            prefetch_tmap(&tm_x);
            prefetch_tmap(&tm_base);
            prefetch_tmap(&tm_out);
            prefetch_tmap(&tm_out8);
        }
    } else if (warp == kMmaWarp) {
        tmem_alloc(&sh->tmem_base, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base, sum_at = tmem + 128;   // A x, then in fp16, in columns 0 .. kR - 1; two places of 64 columns from 128 on
    pdl_launch_dependents();
    pdl_wait();

    int seq = 0, t0 = 0;
    const int rows = find_tile(p, blockIdx.x / p.n_split, tile_rows, seq, t0);
    const int id = rows > 0 ? p.ids[seq] : -1;
    AdapterSlot slot = {0, 0.f};
    if (id >= 0 && id < p.n_slots) slot = p.slots[id];
    const int all_units = (p.out_feat + 63) / 64, split = blockIdx.x % p.n_split;
    const int first_unit = (int)((long long)split * all_units / p.n_split), units = (int)((long long)(split + 1) * all_units / p.n_split) - first_unit;
    const int chunks = (p.in_feat + 63) / 64;
    const int weights_at = tile_rows * kRowBytes, stage_bytes = weights_at + kWeights;
    const bool whole = rows == tile_rows;              // leaves in one piece, else in pieces of eight rows

    if (rows > 0 && slot.rank == 0) {   // base passes on
        if (p.copy) {
            const int granules = min(p.out_feat - first_unit * 64, units * 64) / 8;
            for (int i = threadIdx.x; i < rows * granules; i += kThreads) {
                const int r = i / granules, col = first_unit * 64 + (i - r * granules) * 8;
                *reinterpret_cast<uint4*>(p.out + (t0 + r) * p.out_pitch + col) = *reinterpret_cast<const uint4*>(p.base + (t0 + r) * p.base_pitch + col);
            }
        }
    } else if (rows > 0 && warp == kLoadWarp) {
        if (lane == 0) {
            const half* const a = p.a + id * p.stride;
            const half* const b = p.b + id * p.stride + (long long)first_unit * (kWeights / 2);
            const int n = chunks + units;
            bool ok = true;
            RingAt at;
            int issued = 0;
            for (; issued < n; ++issued, at.next(stages)) {
                const int i = issued, s = at.stage;
                if (at.wraps > 0 && !mbar_wait(&sh->empty[s], (at.wraps - 1) & 1)) {
                    ok = false;
                    break;
                }
                uint8_t* const to = smem + s * stage_bytes;
                mbar_expect_tx(&sh->full[s], stage_bytes);
                const bool is_x = i < chunks;
                if (is_x) tma_load_2d(to, &tm_x, i * 64, t0, &sh->full[s]);
                else tma_load_2d(to, &tm_base, (first_unit + i - chunks) * 64, t0, &sh->full[s]);
                bulk_load(to + weights_at, is_x ? a + (long long)i * (kWeights / 2) : b + (long long)(i - chunks) * (kWeights / 2), kWeights, &sh->full[s]);
            }
            for (int i = max(issued - stages, 0); i < issued; ++i) ok &= mbar_wait(&sh->full[i % stages], (i / stages) & 1);   // nothing lands after the CTA has left
            if (!ok) atomicExch(p.err, 51);
        }
        __syncwarp();
    } else if (rows > 0 && warp == kMmaWarp) {
        if (lane == 0) {
            constexpr uint32_t idesc_low = make_idesc_f16(128, kR), idesc_sum = make_idesc_f16(128, 64);
            const uint64_t x_desc = make_smem_desc(smem_u32(smem), 16, 1024, 2), a_desc = make_smem_desc(smem_u32(smem) + weights_at, 16, 1024, 2);
            const uint64_t b_desc = make_smem_desc(smem_u32(smem) + weights_at, 128, kR / 8 * 128, 0);
            bool ok = true;
            RingAt at;
            for (int i = 0; i < chunks; ++i, at.next(stages)) {
                ok = mbar_wait(&sh->full[at.stage], at.wraps & 1);
                if (!ok) break;
                tc_fence_after();
                const uint64_t off = at.stage * (stage_bytes >> 4);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) umma_f16(tmem, x_desc + off + ks * 2, a_desc + off + ks * 2, idesc_low, i > 0 || ks > 0);
                umma_commit(&sh->empty[at.stage]);
            }
            umma_commit(&sh->low_full);
            ok = ok && mbar_wait(&sh->low_ready, 0);
            tc_fence_after();
            const int steps = (slot.rank + 15) / 16;
            for (int u = 0; u < units && ok; ++u, at.next(stages)) {
                ok = mbar_wait(&sh->full[at.stage], at.wraps & 1) && (u < 2 || mbar_wait(&sh->sum_empty[u & 1], ((u >> 1) - 1) & 1));
                if (!ok) break;
                tc_fence_after();
                const uint64_t off = at.stage * (stage_bytes >> 4);
                for (int ks = 0; ks < steps; ++ks) umma_f16_ts(sum_at + (u & 1) * 64, tmem + ks * 8, b_desc + off + ks * 16, idesc_sum, ks > 0);
                umma_commit(&sh->sum_full[u & 1]);
            }
            if (!ok) atomicExch(p.err, 51);
        }
        __syncwarp();
    } else if (rows > 0 && warp == kStoreWarp) {
        if (lane == 0) {
            bool ok = true;
            RingAt at, unit;
            for (int i = 0; i < chunks; ++i) at.next(stages);
            int before = -1;
            for (int u = 0; u < units; ++u, at.next(stages), unit.next(stages)) {
                ok = mbar_wait(&sh->written[unit.stage], unit.wraps & 1);
                if (!ok) break;
                uint8_t* const from = smem + at.stage * stage_bytes;
                if (whole) {
                    tma_store_2d(&tm_out, from, (first_unit + u) * 64, t0);
                } else {
                    for (int r = 0; r + 8 <= rows; r += 8) tma_store_2d(&tm_out8, from + r * kRowBytes, (first_unit + u) * 64, t0 + r);
                }
                tma_store_commit();
                tma_store_wait_read_but_one();   // the unit before this one has left its stage
                if (before >= 0) mbar_arrive(&sh->empty[before]);
                before = at.stage;
            }
            tma_store_wait();
            if (!ok) atomicExch(p.err, 51);
        }
        __syncwarp();
    } else if (rows > 0) {
        // ---- a row to a thread
        const int row = warp * 32 + lane;
        const uint32_t mine = (uint32_t)warp << 21;   // the warp's lanes of tensor memory
        bool ok = mbar_wait(&sh->low_full, 0);
        float factor = 0.f;
        if (ok) {
            tc_fence_after();
            float top = 0.f;
#pragma unroll
            for (int c = 0; c < kR; c += 16) {
                uint32_t v[16];
                tmem_ld16(tmem + mine + c, v);
                tmem_ld_wait(v);
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (c + j < slot.rank) top = fmaxf(top, fabsf(__uint_as_float(v[j])));
            }
            const int ex = row_exponent(top);
            const float down = __int_as_float((254 - ex) << 23);
            factor = slot.scale * __int_as_float(ex << 23);
#pragma unroll
            for (int c = 0; c < kR; c += 16) {   // (16 columns in 8: what is overwritten has been read; ranks that only pad a step are zeros even where x is not finite)
                uint32_t v[16], h[8];
                tmem_ld16(tmem + mine + c, v);
                tmem_ld_wait(v);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float lo = c + 2 * j < slot.rank ? __uint_as_float(v[2 * j]) * down : 0.f, hi = c + 2 * j + 1 < slot.rank ? __uint_as_float(v[2 * j + 1]) * down : 0.f;
                    const half2 w = __floats2half2_rn(lo, hi);
                    h[j] = *reinterpret_cast<const uint32_t*>(&w);
                }
                tmem_store8(tmem + mine + c / 2, h);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->low_ready);
        }
        const bool in = row < rows, by_tma = row < (whole ? rows : rows & ~7);
        RingAt at, unit;
        for (int i = 0; i < chunks; ++i) at.next(stages);
        for (int u = 0; u < units && ok; ++u, at.next(stages), unit.next(stages)) {
            ok = mbar_wait(&sh->full[at.stage], at.wraps & 1);
            if (!ok) break;
            const int col0 = (first_unit + u) * 64;
            const uint32_t line = smem_u32(smem) + at.stage * stage_bytes + row * kRowBytes;
            uint4 v[8];
            if (in) {   // before the products are there
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = lds128(line + ((c ^ (row & 7)) << 4));
            }
            ok = mbar_wait(&sh->sum_full[u & 1], (u >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t d[32];
                tmem_ld32(sum_at + mine + (u & 1) * 64 + h * 32, d);
                tmem_ld_wait(d);
                if (h) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh->sum_empty[u & 1]);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    half2* const o = reinterpret_cast<half2*>(&v[h * 4 + c]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 b = __half22float2(o[j]);
                        o[j] = __floats2half2_rn(fmaf(factor, __uint_as_float(d[c * 8 + 2 * j]), b.x), fmaf(factor, __uint_as_float(d[c * 8 + 2 * j + 1]), b.y));
                    }
                }
            }
            if (by_tma) {
#pragma unroll
                for (int c = 0; c < 8; ++c) sts128(line + ((c ^ (row & 7)) << 4), v[c]);
            } else if (in) {
                half* const to = p.out + (t0 + row) * p.out_pitch + col0;
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (col0 + c * 8 < p.out_feat) *reinterpret_cast<uint4*>(to + c * 8) = v[c];
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->written[unit.stage]);
        }
        if (!ok && lane == 0) atomicExch(p.err, 51);
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
}

// Bytes of the ring: the first product reads 128 rows from where a stage's rows begin, however many they are.
int ring_bytes(int tile_rows, int weights, int stages) {
    const int stage = tile_rows * kRowBytes + weights;
    return (stages - 1) * stage + max(stage, kMaxTile * kRowBytes);
}

template <int kR>
cudaError_t launch(const AdapterParams& p, int tile_rows, const CUtensorMap& tm_x, const CUtensorMap& tm_base, const CUtensorMap& tm_out, const CUtensorMap& tm_out8, cudaStream_t st) {
    constexpr int kMaxSmem = kSmemForCta - 1024 - (int)sizeof(Barriers);
    int stages = kMaxStages;
    while (ring_bytes(tile_rows, kR * 128, stages) + 1024 > kMaxSmem) --stages;   // (3 at least: 128 rows, rank 128)
    const auto kernel = adapter_tc_kernel<kR>;
    static PerDeviceOnce once;
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem); });
    if (e != cudaSuccess) return e;
    const long long tiles = (long long)p.tokens / tile_rows + p.batch;
    return launch_pdl(kernel, dim3((unsigned)(tiles * p.n_split)), dim3(kThreads), (size_t)ring_bytes(tile_rows, kR * 128, stages) + 1024, st, p, tile_rows, stages, tm_x, tm_base, tm_out, tm_out8);
}

}  // namespace

int adapter_tc_launch(AdapterParams p, int rank_step, cudaStream_t st) {
    // As few waves as tiles of 128 rows make, and in them tiles of equal height: so many rows that the last wave is full too, instead of a few tiles that all
    // wait for. A single wave that leaves SMs empty shares the tiles' columns, two to four CTAs to a tile. (18966 tokens of 32 sequences, 1024 -> 4096, tiles of 64 (312: a second
    // wave), 72, 96, 128 rows: rank 32 90, 70, 67, 69 us, rank 128 119, 79, 97, 100.) About half a tile for each sequence is not full.
    const long long slots = 2LL * sm_count(), tiles = max((long long)p.batch, p.tokens / kMaxTile + p.batch / 2 + 1LL), waves = (tiles + slots - 1) / slots;
    p.n_split = (int)max(1LL, min(min(slots / tiles, 4LL), (p.out_feat + 63LL) / 64));
    const long long height = p.tokens / max(1LL, waves * slots / p.n_split - p.batch / 2) + 1;
    const int tile_rows = (int)max(32LL, min((height + 7) / 8 * 8, (long long)kMaxTile));
    CUtensorMap tm_x, tm_base, tm_out, tm_out8;
    if (!make_tmap_2d_f16(&tm_x, p.x, p.tokens, p.in_feat, p.x_pitch, tile_rows, 64, 128) || !make_tmap_2d_f16(&tm_base, p.base, p.tokens, p.out_feat, p.base_pitch, tile_rows, 64, 128) ||
        !make_tmap_2d_f16(&tm_out, p.out, p.tokens, p.out_feat, p.out_pitch, tile_rows, 64, 128) ||
        !make_tmap_2d_f16(&tm_out8, p.out, p.tokens, p.out_feat, p.out_pitch, 8, 64, 128))
        return fail(ET_ERR_CUDA, "et_adapter_add: cuTensorMapEncodeTiled failed");
    const cudaError_t e = rank_step <= 16   ? launch<16>(p, tile_rows, tm_x, tm_base, tm_out, tm_out8, st)
                          : rank_step <= 32 ? launch<32>(p, tile_rows, tm_x, tm_base, tm_out, tm_out8, st)
                          : rank_step <= 64 ? launch<64>(p, tile_rows, tm_x, tm_base, tm_out, tm_out8, st)
                                            : launch<128>(p, tile_rows, tm_x, tm_base, tm_out, tm_out8, st);
    return cuda_status(e, "et_adapter_add launch");
}

long long adapter_tc_a_stride(int in_feat, int rank_step) { return (long long)((in_feat + 63) / 64) * rank_step * 64; }
long long adapter_tc_b_stride(int out_feat, int rank_step) { return (long long)((out_feat + 63) / 64) * rank_step * 64; }

void adapter_tc_pack(half* pa, half* pb, const half* A, const half* B, int rank, int in_feat, int out_feat, int rank_step) {
    for (int r = 0; r < rank; ++r)   // in_feat is a multiple of 16
        for (int k = 0; k < in_feat; k += 8)
            std::memcpy(pa + ((size_t)(k / 64) * rank_step + r) * 64 + ((k % 64 / 8) ^ (r & 7)) * 8, A + (size_t)r * in_feat + k, 16);
    for (int n = 0; n < out_feat; ++n) {
        half* const column = pb + (size_t)(n / 64) * rank_step * 64 + (size_t)(n % 64 / 8) * (rank_step * 8) + n % 8 * 8;
        for (int r = 0; r < rank; ++r) column[r / 8 * 64 + r % 8] = B[(size_t)n * rank + r];
    }
}

}  // namespace et
