// Linear with operands in e4m3: Y[T x N] = sum over blocks of 128 k of sx[block][t] sw[n / 128][block] (X . W^T over the block) + bias, optional tanh-GELU, fp16 out.
//
// The scales change every 128 k, so a block's products can not go on accumulating where the last block's are: each block is summed by tcgen05 (kind::f8f6f4, both operands from
// 128-byte-swizzled shared memory, four UMMAs of 32 k) into a place of tensor memory of its own, and the epilogue's warps add it, times its scale, to sums in
// registers while the next block is multiplied into another place. Two kernels:
//
// fp8_pair_kernel, many tokens: persistent pairs of CTAs (cta_group::2), 256 tokens x kBN features to a tile. A thread has a token's row of kBN / 2 columns. 16384 x 4096 -> 4096:
// 255 us (2.2e15 operations a second), with GELU 273 (calls one after another for a quarter of a second 318: power). Of the ~900 clocks a block of 256 x 256 takes (UMMAs: 512) copies alone would take ~800 (the way from L2), sums and hand-overs
// alone ~850. Tried, against 244 and with GELU 254 us (a cooler card, a GELU by tanh.approx, waits without votes): one warp that issues all UMMAs 244 / 253 us, four of them 248 / 256, sixteen warps that sum 255 / 266, eight with one
// load from tensor memory at a time 260 / 275, waits by one lane of a warp 267, scales read behind the wait 269. A vote of the warp behind each wait, instead of at every try of it, takes 10 us more, at the end of the block 15, lanes that go on without
// one and without a branch (which the compiler schedules worse) 20 to 40.
//
// fp8_few_kernel, few tokens: operands exchanged, 128 features are the tile's rows and kTokens tokens its columns, so that the weight, which is what has to
// be read, fills the tile; K split over a cluster. Each CTA sends the others their columns' parts (asynchronous stores that count towards a barrier of the receiver) and
// adds what it gets in the order of the ranks.
//
// The weight does not depend on the preceding kernel: its first copies are requested before griddepcontrol.wait, behind which all other roles begin. Every wait is bounded; a role that gives up records a code and all
// threads reach the common exit.
#include <algorithm>
#include <cstring>
#include <new>
#include <vector>
#include "common.h"
#include "ptx.cuh"
#include "tmap.h"
#include "vec_math.cuh"

namespace et {
namespace {

constexpr int kBlock = 128;                       // k (and features of the weight) that share a scale; bytes of a panel's rows
constexpr int kSmemMax = 232448;

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address of the same shared-memory object in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t in_cta(uint32_t at, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at), "r"(rank));
    return a;
}
// Arrives at a barrier of another CTA of the cluster. Relaxed: what was read from tensor memory is in registers by then, and nothing in shared or global memory
// is handed over. (A release waits for the thread's loads of the next scales: a block of 128 k took 2120 clocks instead of 600.)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// A copy into this CTA's shared memory that reports to a barrier of either CTA of the pair (cluster address).
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void* tmap, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives on the barrier at this address in both CTAs of the pair once every UMMA issued so far has completed.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// Instruction descriptor of kind::f8f6f4 with e4m3 A and B, both K-major, and fp32 D: the fields lie as those of kind::f16, and e4m3 is type 0 as f16 is there.
__host__ __device__ constexpr uint32_t make_idesc_e4m3(int M, int N) { return make_idesc_f16(M, N); }

// 8 columns of the thread's lane.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}

// tanh-GELU of two values in fp32: x / 2 (1 + tanh(u)) = x / (1 + exp(-2u)), in which nothing cancels: right to 2^-16 of the result wherever fp16 has one. (tanh.approx instead leaves 2^-11 of
// x / 2, a fifth of the result at x = -3 and nothing of it at -4.) The reciprocal is taken without the special-function unit, which the exponentials fill (with it 2048 tokens, 1024 -> 4096 took 18.1 us where
// this takes 16.8, no GELU 14.1): a first guess r from the exponent and, linearly, the mantissa, off by h = 1 - d r of at most 0.051, and r (1 + h) (1 + h^2), off by h^4.
__device__ __forceinline__ float2 gelu2(float a, float b) {
    constexpr float k1 = 2.f * 1.4426950408889634f * 0.7978845608028654f, k3 = k1 * 0.044715f;
    // (-x; left of -9.9 the result is below 2^-119, and the exponent would pass fp32's)
    float2 x;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(x.x) : "f"(-a), "f"(9.9f));
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(x.y) : "f"(-b), "f"(9.9f));
    const float2 t = mul2(x, fma2(mul2(x, x), make_float2(k3, k3), make_float2(k1, k1)));
    const float2 one = make_float2(1.f, 1.f), d = add2(make_float2(ex2_fast(t.x), ex2_fast(t.y)), one);
    const float2 r = make_float2(__uint_as_float(0xfef31000u - __float_as_uint(d.x)), __uint_as_float(0xfef31000u - __float_as_uint(d.y)));   // (-r)
    const float2 h = fma2(d, r, one), y = mul2(x, r), z = fma2(y, h, y);
    return fma2(z, mul2(h, h), z);
}
// Two results, in fp16.
template <bool kGelu>
__device__ __forceinline__ half2 finish(float a, float b) {
    if constexpr (kGelu) {
        const float2 y = gelu2(a, b);
        return __floats2half2_rn(y.x, y.y);
    }
    return __floats2half2_rn(a, b);
}

struct Fp8Params {
    half* Y;
    const half* bias;                             // padded with zeros to whole tiles
    const float *x_scales, *w_scales;             // [blocks][T], [blocks of N][blocks]
    long long y_pitch;
    int T, N, k_blocks, tiles_n, tiles, stages;
    int* err;
};

// ------------------------------------------------------------------------------------------ many tokens
// Warps: 0 copies X, 1 copies W, 2 and 3 issue UMMAs, 4 to 11 sum.
constexpr int kXCopy = 0, kFirstMma = 2, kFirstEpi = 4, kEpiWarps = 8;
// Registers of a thread: launched with 168, the roles' warpgroup gives some to the sums' two. (With 168 for all the scales on their way were spilled, that is waited for.)
constexpr int kRoleRegs = 40, kSumRegs = 232;
static_assert(kRoleRegs + 2 * kSumRegs <= 3 * 168, "the block's registers at launch");
constexpr int kPairThreads = 32 * (kFirstEpi + kEpiWarps);
constexpr int kXPanel = 128 * kBlock;             // of a CTA's tokens
constexpr int kUnitCols = 32, kUnitBytes = 32 * kUnitCols * 2;
constexpr int kMaxStages = 8;

template <int kBN>
struct PairCfg {
    static constexpr int kWPanel = kBN / 2 * kBlock, kStage = kXPanel + kWPanel;
    static constexpr int kCols = kBN / 2;                        // of a thread
    // Tensor memory: tiles of 256 take all of it with two places, each in two halves that are multiplied, added and freed by themselves: a half's round (256 clocks of
    // UMMAs, some 500 of hand-overs, the additions) fits into the 1024 clocks that it may take. Tiles of 128 have four places.
    static constexpr int kHalves = kBN == 256 ? 2 : 1;
    static constexpr int kSlots = 512 / kBN * kHalves, kSlotCols = kBN / kHalves;
    static_assert(kSlots == 4, "two to each warp that issues");
    static constexpr int kOut = kEpiWarps * (kCols / kUnitCols) * kUnitBytes;   // a tile's results, on their way out while the next tile is summed
    static constexpr int kStages = kBN == 256 ? 5 : 8;
    static_assert(kHalves == 2 || kStages % 2 == 0, "a stage always falls to the same warp that issues");   // (a parity wait needs a waiter that has seen the phase before)
    static constexpr int kBytes = kStages * kStage + kOut + 1024;
};

struct PairShared {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t acc_full[4], acc_empty[4];
    uint32_t tmem_base;
};

template <int kBN, bool kGelu>
__global__ void __launch_bounds__(kPairThreads, 1) fp8_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmY,
                                                                   const __grid_constant__ Fp8Params p) {
    using C = PairCfg<kBN>;
    constexpr int S = C::kStages, kStage = C::kStage, kCols = C::kCols;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ PairShared shared;
    PairShared* const sh = &shared;
    const uint32_t ring = smem_u32(smem), epi = ring + S * kStage;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_rank();
    const int pair = (int)blockIdx.x >> 1, G = (int)gridDim.x >> 1;
    const int my_tiles = (p.tiles - pair + G - 1) / G;
    if (tid == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(&sh->full[i], 1); mbar_init(&sh->empty[i], C::kHalves); }
        for (int i = 0; i < C::kSlots; ++i) { mbar_init(&sh->acc_full[i], 1); mbar_init(&sh->acc_empty[i], 2 * kEpiWarps / C::kHalves); }
        fence_mbar_init();
        prefetch_tmap(&tmX);
        prefetch_tmap(&tmW);
    }
    if (warp == kFirstMma) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh->tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();   // the other CTA's barriers exist
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;
    const int total = my_tiles * p.k_blocks;
    if (warp < kFirstEpi) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRoleRegs));
        if (warp < kFirstMma) {
            // ---- copies; both CTAs' report to the first one's barriers
            const bool is_x = warp == kXCopy;
            if (is_x) pdl_wait();
            if (lane == 0) {
                bool ok = true;
                int s = 0, kb = 0, tile = pair;
                uint32_t ph = 1;
                for (int c = 0; c < total; ++c) {
                    if (!is_x && c == S) pdl_wait();   // (the weight's first copies go ahead; what follows waits for products of X)
                    ok = mbar_wait_at(smem_u32(&sh->empty[s]), ph);
                    if (!ok) break;
                    const uint32_t bar = in_cta(smem_u32(&sh->full[s]), 0);
                    if (is_x) {
                        tma_load_2d_pair(ring + s * kStage, &tmX, kb * kBlock, (tile / p.tiles_n) * 256 + (int)rank * 128, bar);
                    } else {
                        if (rank == 0) mbar_expect_tx(&sh->full[s], 2 * kStage);
                        tma_load_2d_pair(ring + s * kStage + kXPanel, &tmW, kb * kBlock, (tile % p.tiles_n) * kBN + (int)rank * (kBN / 2), bar);
                    }
                    if (++kb == p.k_blocks) { kb = 0; tile += G; }
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
                // (On the normal way out every copy has been consumed. A wait that gives up has lasted far longer than any copy.)
                if (!ok) atomicExch(p.err, 61);
            }
            __syncwarp();
        } else if (rank == 0) {
            // ---- UMMAs of the pair, by two warps: either has a half of each block, or (tiles of 128) every other block
            if (elect_one()) {
                constexpr uint32_t idesc = make_idesc_e4m3(256, C::kSlotCols);
                constexpr int kStep = 3 - C::kHalves;
                const int m = warp - kFirstMma;
                // (half h: rows h * 64 .. of the weight's panel in either CTA, columns of the first CTA's and then of the second's)
                const uint64_t x0 = make_smem_desc(ring, 16, 1024, 2), w0 = make_smem_desc(ring + kXPanel + (C::kHalves == 2 ? m * (kBN / 4 * kBlock) : 0), 16, 1024, 2);
                const uint32_t full = smem_u32(&sh->full[0]), empty = smem_u32(&sh->empty[0]), acc_full = smem_u32(&sh->acc_full[0]), acc_empty = smem_u32(&sh->acc_empty[0]);
                bool ok = true;
                int s = C::kHalves == 2 ? 0 : m, slot = m;
                uint32_t ph = 0, slot_ph = 1;
                pdl_wait();   // (X's copies do: a wait for them may not begin while the preceding kernel runs, whose length has no limit)
                for (int c = s; c < total; c += kStep) {
                    ok = mbar_wait_at(acc_empty + slot * 8, slot_ph) && mbar_wait_at(full + s * 8, ph);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t at = (uint64_t)(s * kStage) >> 4;   // descriptors count 16-byte units
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) umma_f8_pair(tmem + slot * C::kSlotCols, x0 + at + ks * 2, w0 + at + ks * 2, idesc, ks > 0);
                    umma_commit_pair(acc_full + slot * 8);
                    umma_commit_pair(empty + s * 8);
                    slot += 2;
                    if (slot >= 4) { slot -= 4; slot_ph ^= 1u; }
                    s += kStep;
                    if (s >= S) { s -= S; ph ^= 1u; }
                }
                if (!ok) atomicExch(p.err, 62);
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
        // ---- sums of this CTA's 128 tokens: a row to a thread, two warps share its columns
        const int w = warp - kFirstEpi, q = warp & 3, h = w >> 2;
        const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + (C::kHalves == 2 ? 0 : h * kCols);
        const uint32_t buf_at = epi + w * (kCols / kUnitCols) * kUnitBytes;
        const uint32_t to = buf_at + lane * 64, swizzle = (lane >> 1) & 3;   // row `lane`: four 16-byte chunks under the 64-byte swizzle
        const uint32_t empty_bar = in_cta(smem_u32(&sh->acc_empty[0]), 0), acc_full = smem_u32(&sh->acc_full[0]);
        const int n_blocks = (p.N + kBlock - 1) / kBlock;
        bool ok = true;
        pdl_wait();
        auto row_scales = [&](int tile) { return p.x_scales + min((tile / p.tiles_n) * 256 + (int)rank * 128 + q * 32 + lane, p.T - 1); };
        // The token's scales are requested two blocks ahead: of even blocks, of odd ones.
        float even = __ldcg(row_scales(pair)), odd = p.k_blocks > 1 ? __ldcg(row_scales(pair) + p.T) : 0.f;
        int slot = C::kHalves == 2 ? h : 0;
        uint32_t slot_ph = 0;
        for (int tl = 0; tl < my_tiles && ok; ++tl) {
            const int tile = pair + tl * G;
            const int m0 = (tile / p.tiles_n) * 256 + (int)rank * 128 + q * 32, n0 = (tile % p.tiles_n) * kBN;
            // Columns of the thread, 32 at a time: of half h of a tile of 256 the features h 64 .. and 128 + h 64 .. (64 each), else h 64 ...
            auto column = [&](int u) { return n0 + h * 64 + (u < 2 ? u * kUnitCols : 128 + (u - 2) * kUnitCols); };
            const float* const sx = row_scales(tile);
            // the scales of the weight for the first and for the last 64 columns
            const float* const sw0 = p.w_scales + (long long)(n0 / kBlock) * p.k_blocks;
            const float* const sw1 = p.w_scales + (long long)min(n0 / kBlock + 1, n_blocks - 1) * p.k_blocks;
            float next0 = __ldg(sw0), next1 = C::kHalves == 2 ? __ldg(sw1) : 0.f;
            float acc[kCols];   // from the bias on (padded with zeros to a multiple of 256)
#pragma unroll
            for (int i = 0; i < kCols; i += 8) {
                const uint4 bv = __ldg(reinterpret_cast<const uint4*>(p.bias + column(i / kUnitCols) + i % kUnitCols));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = __half22float2(reinterpret_cast<const half2*>(&bv)[j]);
                    acc[i + 2 * j] = f.x;
                    acc[i + 2 * j + 1] = f.y;
                }
            }
            auto add_block = [&](int kb, float& token) {
                const float scale0 = token * next0, scale1 = token * next1;
                if (kb + 2 < p.k_blocks) token = __ldcg(sx + (long long)(kb + 2) * p.T);
                if (kb + 1 < p.k_blocks) {
                    next0 = __ldg(sw0 + kb + 1);
                    if (C::kHalves == 2) next1 = __ldg(sw1 + kb + 1);
                }
                if (!mbar_wait_warp_at(acc_full + slot * 8, slot_ph)) return false;
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < kCols; i += 32) {
                    uint32_t lo[16], hi[16];
                    tmem_ld16(from + slot * C::kSlotCols + i, lo);
                    tmem_ld16(from + slot * C::kSlotCols + i + 16, hi);
                    tmem_ld_wait(lo, hi);
                    if (i + 32 == kCols) {   // the slot may be overwritten
                        tc_fence_before();
                        __syncwarp();
                        if (elect_one()) mbar_arrive_cluster(empty_bar + slot * 8);
                    }
                    const float f = C::kHalves == 2 && i >= 64 ? scale1 : scale0;
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float2 d = j < 16 ? make_float2(__uint_as_float(lo[j]), __uint_as_float(lo[j + 1])) : make_float2(__uint_as_float(hi[j - 16]), __uint_as_float(hi[j - 15]));
                        const float2 r = fma2(d, make_float2(f, f), make_float2(acc[i + j], acc[i + j + 1]));
                        acc[i + j] = r.x;
                        acc[i + j + 1] = r.y;
                    }
                }
                slot += C::kHalves;
                if (slot >= C::kSlots) {
                    slot -= C::kSlots;
                    slot_ph ^= 1u;
                }
                return true;
            };
            for (int kb = 0; kb < p.k_blocks && ok; kb += 2) {
                ok = add_block(kb, even);
                if (ok && kb + 1 < p.k_blocks) ok = add_block(kb + 1, odd);
            }
            if (tl + 1 < my_tiles) {
                even = __ldcg(row_scales(tile + G));
                if (p.k_blocks > 1) odd = __ldcg(row_scales(tile + G) + p.T);
            }
            if (!ok) break;
            if (tl + 1 == my_tiles) pdl_launch_dependents();
            tma_store_wait_read();   // the stores of the tile before have read the buffers
            __syncwarp();
#pragma unroll
            for (int u = 0; u < kCols / kUnitCols; ++u) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint4 ov;
                    half2* const o = reinterpret_cast<half2*>(&ov);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = finish<kGelu>(acc[u * kUnitCols + j * 8 + 2 * i], acc[u * kUnitCols + j * 8 + 2 * i + 1]);
                    sts128(to + u * kUnitBytes + ((j ^ swizzle) << 4), ov);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (m0 < p.T && elect_one()) {
#pragma unroll
                for (int u = 0; u < kCols / kUnitCols; ++u)
                    if (column(u) < p.N) tma_store_2d(&tmY, smem + (buf_at - ring) + u * kUnitBytes, column(u), m0);
                tma_store_commit();
            }
            __syncwarp();
        }
        if (!ok && lane == 0) atomicExch(p.err, 63);
        tma_store_wait_read();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();   // nobody still reads this CTA's shared memory or signals its barriers
    tc_fence_after();
    if (warp == kFirstMma) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ------------------------------------------------------------------------------------------ few tokens
constexpr int kFewEpi = 8, kWWarp = 8, kXWarp = 9, kFewMma = 10, kFewThreads = 11 * 32;
constexpr int kMaxPlaces = 8;
constexpr int kScaleBlocks = 16;                  // blocks whose scales are fetched at once
constexpr int kWTile = 128 * kBlock;              // 128 features of the weight

struct FewShared {
    uint64_t full[kMaxPlaces], empty[kMaxPlaces];
    uint64_t acc_full[kMaxPlaces], acc_empty[kMaxPlaces];
    uint64_t received;
    uint32_t tmem_base;
    __align__(16) float scales[kScaleBlocks * 128];   // of the tokens and of the weight, multiplied: [block][token]
};

// Four words to the address `addr` of CTA `rank` of the cluster, which count towards the bytes that its barrier at `bar` waits for.
__device__ __forceinline__ void st_async_cluster(uint32_t addr, uint32_t bar, uint32_t rank, const float* v) {
    asm volatile("{\n.reg .b32 a, b;\nmapa.shared::cluster.u32 a, %0, %2;\nmapa.shared::cluster.u32 b, %1, %2;\n"
                 "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [a], {%3,%4,%5,%6}, [b];\n}" ::"r"(addr), "r"(bar), "r"(rank), "r"(__float_as_uint(v[0])),
                 "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3]))
                 : "memory");
}
__device__ __forceinline__ void few_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kFewEpi) : "memory"); }
// A bounded wait like mbar_wait_warp, for what other CTAs of the cluster have written.
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity) {
#pragma unroll 1
    for (uint32_t i = 0; i < kMbarSpinLimit; ++i) {
        uint32_t ok;
        asm volatile("{\n.reg .pred P;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P, [%1], %2;\nselp.u32 %0, 1, 0, P;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (__all_sync(0xffffffffu, ok)) return true;
    }
    return false;
}

// Places of tensor memory, of kTokens columns each.
__host__ __device__ constexpr int few_places(int tokens) { return tokens <= 64 ? 4 : 2; }
// A CTA that waits for the others of its cluster may not have to wait for tensor memory that another cluster's CTA holds, which may wait for this one's. So each
// takes no smaller a part of an SM's shared memory (227 KB) than of its tensor memory (512 columns): those that find a place find both.
constexpr int kSmemPerColumn = 454;

template <int kTokens, bool kGelu>
__global__ void __launch_bounds__(kFewThreads, 1) fp8_few_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ Fp8Params p,
                                                                 int log_split) {
    constexpr int kXTile = kTokens * kBlock, kStage = kWTile + kXTile;
    constexpr int kPlaces = few_places(kTokens);
    constexpr int kAlloc = kPlaces * kTokens;
    constexpr int kCols = kTokens / 2;                        // of a warp
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ FewShared shared;
    FewShared* const sh = &shared;
    const int S = p.stages, split = 1 << log_split, own_cols = kTokens >> log_split, log_own = 31 - __clz(own_cols);
    const uint32_t ring = smem_u32(smem);
    float4* const recv = reinterpret_cast<float4*>(smem + S * kStage);   // of each share, this CTA's columns: [share][four columns][row]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)cluster_rank(), tile = (int)blockIdx.x / split;
    const int n0 = (tile % p.tiles_n) * 128, t0 = (tile / p.tiles_n) * kTokens;
    const int kb0 = (int)((long long)rank * p.k_blocks / split), kn = (int)((long long)(rank + 1) * p.k_blocks / split) - kb0;
    if (warp == kWWarp) {
        if (lane == 0) {
            for (int i = 0; i < S; ++i) { mbar_init(&sh->full[i], 2); mbar_init(&sh->empty[i], 1); }
            for (int i = 0; i < kPlaces; ++i) { mbar_init(&sh->acc_full[i], 1); mbar_init(&sh->acc_empty[i], kFewEpi); }
            mbar_init(&sh->received, 1);
            fence_mbar_init();
            mbar_expect_tx(&sh->received, (uint32_t)((split - 1) * own_cols * 128 * 4));
        }
    } else if (warp == kFewMma) {
        tmem_alloc(&sh->tmem_base, kAlloc);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this CTA runs and its barriers exist: its memory may be written to
    const uint32_t tmem = sh->tmem_base;
    bool ok = true;
    float acc[kCols];
#pragma unroll
    for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
    if (warp == kWWarp || warp == kXWarp) {
        const bool is_x = warp == kXWarp;
        if (is_x) pdl_wait();
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 1;
            int i = 0;
            for (; i < kn; ++i) {
                if (!is_x && i == S) pdl_wait();   // (the weight's first copies go ahead; what follows waits for products of X)
                ok = i < S || mbar_wait(&sh->empty[s], ph);
                if (!ok) break;
                mbar_expect_tx(&sh->full[s], is_x ? kXTile : kWTile);
                if (is_x) tma_load_2d(smem + s * kStage + kWTile, &tmX, (kb0 + i) * kBlock, t0, &sh->full[s]);
                else tma_load_2d(smem + s * kStage, &tmW, (kb0 + i) * kBlock, n0, &sh->full[s]);
                if (++s == S) { s = 0; ph ^= 1u; }
            }
            if (!ok) {   // copies in flight land before the CTA leaves (bounded)
                atomicExch(p.err, 64);
                for (int j = max(i - S, 0); j < i; ++j) mbar_wait(&sh->full[j % S], (j / S) & 1);
            }
        }
        __syncwarp();
    } else if (warp == kFewMma) {
        if (elect_one()) {
            constexpr uint32_t idesc = make_idesc_e4m3(128, kTokens);
            const uint64_t w0 = make_smem_desc(ring, 16, 1024, 2), x0 = make_smem_desc(ring + kWTile, 16, 1024, 2);
            int s = 0;
            uint32_t ph = 0;
            pdl_wait();   // (X's copies do: a wait for them may not begin while the preceding kernel runs, whose length has no limit)
            for (int i = 0; i < kn; ++i) {
                const int place = i % kPlaces;
                ok = (i < kPlaces || mbar_wait(&sh->acc_empty[place], (uint32_t)(i / kPlaces - 1) & 1u)) && mbar_wait(&sh->full[s], ph);
                if (!ok) break;
                tc_fence_after();
                const uint64_t at = (uint64_t)(s * kStage) >> 4;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) umma_f8(tmem + place * kTokens, w0 + at + ks * 2, x0 + at + ks * 2, idesc, ks > 0);
                umma_commit(&sh->empty[s]);
                umma_commit(&sh->acc_full[place]);
                if (++s == S) { s = 0; ph ^= 1u; }
            }
            if (!ok) atomicExch(p.err, 65);
        }
        __syncwarp();
    } else {
        // ---- a feature to a thread, two warps share the tokens
        const int q = warp & 3, h = warp >> 2;
        const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + h * kCols;
        const float* const sw = p.w_scales + (long long)(n0 / kBlock) * p.k_blocks + kb0;
        pdl_wait();
        for (int i = 0; i < kn; ++i) {
            const int place = i % kPlaces;
            const float* const mine = sh->scales + (i % kScaleBlocks) * kTokens + h * kCols;
            if (i % kScaleBlocks == 0) {
                if (i > 0) few_barrier();   // (the scales before have been read)
                const int n = min(kScaleBlocks, kn - i) * kTokens;
#pragma unroll 4
                for (int e = tid; e < n; e += 32 * kFewEpi) {
                    const int kb = i + e / kTokens, t = t0 + e % kTokens;
                    sh->scales[e] = t < p.T ? __ldcg(p.x_scales + (long long)(kb0 + kb) * p.T + t) * __ldg(sw + kb) : 0.f;
                }
                few_barrier();
            }
            // (A warp that gives up stays in the loop without waiting again: few_barrier counts every warp.)
            ok = ok && mbar_wait_warp_at(smem_u32(&sh->acc_full[place]), (uint32_t)(i / kPlaces) & 1u);
            if (!ok) continue;
            tc_fence_after();
            constexpr int kStep = kCols < 16 ? kCols : 16;
#pragma unroll
            for (int c = 0; c < kCols; c += kStep) {
                uint32_t d[kStep];
                if constexpr (kStep == 8) tmem_ld8(from + place * kTokens + c, d);
                else tmem_ld16(from + place * kTokens + c, d);
                tmem_ld_wait(d);
#pragma unroll
                for (int j = 0; j < kStep; j += 4) {
                    const float4 f = *reinterpret_cast<const float4*>(mine + c + j);
                    acc[c + j] = fmaf(__uint_as_float(d[j]), f.x, acc[c + j]);
                    acc[c + j + 1] = fmaf(__uint_as_float(d[j + 1]), f.y, acc[c + j + 1]);
                    acc[c + j + 2] = fmaf(__uint_as_float(d[j + 2]), f.z, acc[c + j + 2]);
                    acc[c + j + 3] = fmaf(__uint_as_float(d[j + 3]), f.w, acc[c + j + 3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->acc_empty[place]);
        }
        if (!ok && lane == 0) atomicExch(p.err, 66);
    }
    __syncwarp();
    pdl_launch_dependents();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // every CTA of the cluster runs
    bool got = true;
    if (warp < kFewEpi) {
        const int row = (warp & 3) * 32 + lane, h = warp >> 2;
#pragma unroll
        for (int c = 0; c < kCols; c += 4) {
            const int col = h * kCols + c, dst = col >> log_own;
            float4* const to = recv + (rank * (own_cols / 4) + ((col & (own_cols - 1)) >> 2)) * 128 + row;
            if (dst == rank) *to = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);   // (the same for the whole warp)
            else st_async_cluster(smem_u32(to), smem_u32(&sh->received), dst, acc + c);
        }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this warp has sent everything
    if (warp < kFewEpi) {
        few_barrier();
        if (split > 1) got = mbar_wait_cluster(smem_u32(&sh->received), 0);
        if (!got && lane == 0) atomicExch(p.err, 67);
        const int row = tid & 127, n = n0 + row;
        const float bias = __half2float(p.bias[n]);
        half* y = p.Y + (long long)(t0 + rank * own_cols) * p.y_pitch + n;
        for (int g = tid >> 7; g < own_cols / 4; g += kFewEpi / 4) {
            const int t = t0 + rank * own_cols + g * 4;
            if (t >= p.T) break;
            const float4* const from = recv + g * 128 + row;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < split; ++k) {   // in the order of the shares
                const float4 x = from[k * (own_cols / 4) * 128];
                v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
            }
            if (n < p.N) {
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    const half2 o = finish<kGelu>(v[j] + bias, v[j + 1] + bias);
                    if (t + j < p.T) y[(g * 4 + j) * p.y_pitch] = __low2half(o);
                    if (t + j + 1 < p.T) y[(g * 4 + j + 1) * p.y_pitch] = __high2half(o);
                }
            }
        }
    }
    __syncwarp();
    // Normally all have sent when this CTA has received. One that gave up stays until nothing is on its way to it.
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (!got) mbar_wait_cluster(smem_u32(&sh->received), 0);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kFewMma) tmem_dealloc(tmem, kAlloc);
}

bool make_tmap_bytes(CUtensorMap* out, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, uint32_t box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {pitch};
    cuuint32_t box[2] = {kBlock, box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace et

struct et_fp8_weight {
    int device = 0, K = 0, N = 0;
    uint8_t* codes = nullptr;     // [N x K]
    float* scales = nullptr;      // [blocks of N][blocks of K]
    half* bias = nullptr;         // padded with zeros to a multiple of 256
    int* err = nullptr;
    CUtensorMap map64, map128;    // 64 and 128 rows to a copy
};

namespace et {
namespace {

struct Fp8Plan {
    int bn;        // > 0: pairs with tiles of bn features
    int tokens;    // few tokens: columns of a tile, and CTAs that share a tile's K
    int log_split;
};

// Clocks of a launch, fitted to 790 launches of 1 to 1700 tokens, seven shapes and every plan: the plan taken takes 0.8 % longer than the fastest in the mean, 18 % at most. A few-token
// CTA's block costs its hand-overs or its copies (26 clocks a KB), a tile at its end 65 clocks a token (exchange and stores).
// (64 x 4096 -> 4096, tiles of 64, four CTAs to a tile's K 6.7 us, of 16 10.9, pairs 14.2; 512 tokens pairs 15.4, tiles of 128 17.9.)
Fp8Plan fp8_plan(int T, int N, int k_blocks) {
    Fp8Plan best = {0, 0, 0};
    double least = 1e30;
    auto take = [&](const Fp8Plan& plan, double cost) {
        if (cost < least) {
            least = cost;
            best = plan;
        }
    };
    auto waves = [](long long n, long long at_once) { return (double)((n + at_once - 1) / at_once); };
    for (int bn : {128, 256}) {
        const double w = waves((T + 255LL) / 256 * ((N + bn - 1) / bn), sm_count() / 2);
        take({bn, 0, 0}, 4100.0 + w * (k_blocks * (bn == 128 ? 670.0 : 790.0) + 12.4 * bn));
    }
    if (T > 4096) return best;
    for (int tokens : {16, 32, 64, 128})
        for (int log_split = 0; log_split < 4 && (1 << log_split) <= k_blocks && (tokens >> log_split) >= 4; ++log_split) {
            // CTAs of clusters that run at once: clusters do not straddle the groups of 16 to 20 SMs
            const int at_once = log_split == 3 ? 14 * 8 : log_split == 2 ? 33 * 4 : sm_count();
            const double w = waves((N + 127LL) / 128 * ((T + tokens - 1) / tokens) << log_split, at_once);
            const int blocks = (k_blocks + (1 << log_split) - 1) >> log_split;
            take({0, tokens, log_split}, 2950.0 + w * (blocks * std::max(577.0, 0.0257 * (kWTile + tokens * kBlock)) + 65.0 * tokens) + (w - 1) * 500.0);
        }
    return best;
}

template <int kBN, bool kGelu>
cudaError_t launch_pair(const CUtensorMap& tx, const CUtensorMap& tw, const CUtensorMap& ty, Fp8Params p, cudaStream_t st) {
    const auto kernel = fp8_pair_kernel<kBN, kGelu>;
    static PerDeviceOnce once;
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg<kBN>::kBytes); });
    if (e != cudaSuccess) return e;
    p.tiles_n = (p.N + kBN - 1) / kBN;
    p.tiles = (p.T + 255) / 256 * p.tiles_n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * std::min(p.tiles, sm_count() / 2)));
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = PairCfg<kBN>::kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, tx, tw, ty, p);
}

template <int kTokens, bool kGelu>
cudaError_t launch_few(const CUtensorMap& tx, const CUtensorMap& tw, Fp8Params p, int log_split, cudaStream_t st) {
    const int split = 1 << log_split;
    constexpr int kStage = kWTile + kTokens * kBlock;
    const auto kernel = fp8_few_kernel<kTokens, kGelu>;
    static PerDeviceOnce once;
    const int max_smem = kSmemMax - ((int)sizeof(FewShared) + 1023) / 1024 * 1024;
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, max_smem); });
    if (e != cudaSuccess) return e;
    p.tiles_n = (p.N + 127) / 128;
    p.tiles = (p.T + kTokens - 1) / kTokens * p.tiles_n;
    const int recv = kTokens * 128 * 4;   // of all shares, the CTA's columns
    p.stages = std::min({kMaxPlaces, (max_smem - 1024 - recv) / kStage, (p.k_blocks + split - 1) / split});
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.tiles * split));
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = (size_t)std::max(p.stages * kStage + recv + 1024, few_places(kTokens) * kTokens * kSmemPerColumn);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, tx, tw, p, log_split);
}

template <bool kGelu>
int fp8_run(const et_fp8_weight* w, const Fp8Params& p, const Fp8Plan& plan, const void* x, long long x_pitch, cudaStream_t st) {
    CUtensorMap tx, ty;
    const int x_rows = plan.bn ? 128 : plan.tokens;
    if (!make_tmap_bytes(&tx, x, (uint64_t)p.T, (uint64_t)w->K, (uint64_t)x_pitch, (uint32_t)x_rows)) return fail(ET_ERR_CUDA, "et_fp8_linear: cuTensorMapEncodeTiled failed");
    cudaError_t e;
    if (plan.bn) {
        if (!make_tmap_2d_f16(&ty, p.Y, (uint64_t)p.T, (uint64_t)p.N, (uint64_t)p.y_pitch, 32, kUnitCols, 64)) return fail(ET_ERR_CUDA, "et_fp8_linear: cuTensorMapEncodeTiled failed");
        e = plan.bn == 256 ? launch_pair<256, kGelu>(tx, w->map128, ty, p, st) : launch_pair<128, kGelu>(tx, w->map64, ty, p, st);
    } else {
        e = plan.tokens == 16   ? launch_few<16, kGelu>(tx, w->map128, p, plan.log_split, st)
            : plan.tokens == 32 ? launch_few<32, kGelu>(tx, w->map128, p, plan.log_split, st)
            : plan.tokens == 64 ? launch_few<64, kGelu>(tx, w->map128, p, plan.log_split, st)
                                : launch_few<128, kGelu>(tx, w->map128, p, plan.log_split, st);
    }
    return cuda_status(e, "et_fp8_linear launch");
}

}  // namespace
}  // namespace et

extern "C" int et_fp8_weight_destroy(et_fp8_weight* w) {
    if (!w) return ET_OK;
    cudaFree(w->codes);
    cudaFree(w->scales);
    cudaFree(w->bias);
    cudaFree(w->err);
    delete w;
    return ET_OK;
}

extern "C" int et_fp8_weight_create(et_fp8_weight** out, int in_feat, int out_feat, const void* codes_host, const float* scales_host, const void* bias_host) {
    using namespace et;
    ET_REQUIRE(out, "et_fp8_weight_create: null output");
    *out = nullptr;
    ET_REQUIRE(in_feat > 0 && out_feat > 0 && in_feat % 16 == 0 && out_feat % 16 == 0, "et_fp8_weight_create: in_feat and out_feat must be positive multiples of 16");
    ET_REQUIRE(codes_host && scales_host, "et_fp8_weight_create: null pointer");
    auto* w = new (std::nothrow) et_fp8_weight;
    if (!w) return fail(ET_ERR_CUDA, "et_fp8_weight_create: out of host memory");
    w->K = in_feat;
    w->N = out_feat;
    const size_t bytes = (size_t)in_feat * out_feat, n_scales = (size_t)((in_feat + kBlock - 1) / kBlock) * ((out_feat + kBlock - 1) / kBlock), n_bias = ((size_t)out_feat + 255) / 256 * 256;
    cudaError_t e = cudaGetDevice(&w->device);
    if (e == cudaSuccess) e = cudaMalloc(&w->codes, bytes);
    if (e == cudaSuccess) e = cudaMalloc(&w->scales, n_scales * sizeof(float));
    if (e == cudaSuccess) e = cudaMalloc(&w->bias, n_bias * sizeof(half));
    if (e == cudaSuccess) e = cudaMalloc(&w->err, sizeof(int));
    if (e == cudaSuccess) e = cudaMemset(w->bias, 0, n_bias * sizeof(half));
    if (e == cudaSuccess) e = cudaMemset(w->err, 0, sizeof(int));
    if (e == cudaSuccess) e = cudaMemcpy(w->codes, codes_host, bytes, cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaMemcpy(w->scales, scales_host, n_scales * sizeof(float), cudaMemcpyHostToDevice);
    if (e == cudaSuccess && bias_host) e = cudaMemcpy(w->bias, bias_host, (size_t)out_feat * sizeof(half), cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e != cudaSuccess) {
        et_fp8_weight_destroy(w);
        return cuda_status(e, "et_fp8_weight_create");
    }
    if (!make_tmap_bytes(&w->map64, w->codes, (uint64_t)out_feat, (uint64_t)in_feat, (uint64_t)in_feat, 64) ||
        !make_tmap_bytes(&w->map128, w->codes, (uint64_t)out_feat, (uint64_t)in_feat, (uint64_t)in_feat, 128)) {
        et_fp8_weight_destroy(w);
        return fail(ET_ERR_CUDA, "et_fp8_weight_create: cuTensorMapEncodeTiled failed");
    }
    *out = w;
    return ET_OK;
}

extern "C" int et_fp8_weight_check(const et_fp8_weight* w, int* code) {
    using namespace et;
    ET_REQUIRE(w && code, "et_fp8_weight_check: null pointer");
    *code = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpy(code, w->err, sizeof(int), cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && *code) e = cudaMemset(w->err, 0, sizeof(int));
    if (e != cudaSuccess) return cuda_status(e, "et_fp8_weight_check");
    if (*code) {
        set_error("8-bit linear: device wait %d gave up", *code);
        return ET_ERR_DEVICE_TIMEOUT;
    }
    return ET_OK;
}

namespace et {
namespace {
// forced: a plan, or null for the one that the model says.
int fp8_linear(const et_fp8_linear_args* a, const Fp8Plan* forced) {
    ET_REQUIRE(a && a->weight, "et_fp8_linear: null weight");
    const et_fp8_weight* const w = a->weight;
    ET_REQUIRE(a->tokens >= 0 && a->tokens <= 0x7ff00000, "et_fp8_linear: negative size, or more tokens than 32 bits number");
    if (a->tokens == 0) return ET_OK;
    ET_REQUIRE(a->y && a->x && a->x_scales, "et_fp8_linear: null pointer");
    const long long y_pitch = a->tokens == 1 ? (w->N + 7) / 8 * 8 : a->y_pitch, x_pitch = a->tokens == 1 ? w->K : a->x_pitch;
    ET_REQUIRE(y_pitch >= w->N && x_pitch >= w->K, "et_fp8_linear: pitch below the width");
    ET_REQUIRE(aligned16(a->x) && aligned16(a->y) && x_pitch % 16 == 0 && y_pitch % 8 == 0, "et_fp8_linear: rows must start on 16 bytes");
    int dev = -1;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_status(e, "et_fp8_linear");
    ET_REQUIRE(dev == w->device, "et_fp8_linear: the weight belongs to another device");
    Fp8Params p = {};
    p.Y = static_cast<half*>(a->y); p.bias = w->bias; p.x_scales = a->x_scales; p.w_scales = w->scales;
    p.y_pitch = y_pitch; p.T = a->tokens; p.N = w->N; p.k_blocks = (w->K + kBlock - 1) / kBlock; p.err = w->err;
    const Fp8Plan plan = forced ? *forced : fp8_plan(a->tokens, w->N, p.k_blocks);
    return (a->gelu ? fp8_run<true> : fp8_run<false>)(w, p, plan, a->x, x_pitch, static_cast<cudaStream_t>(a->stream));
}
}  // namespace
}  // namespace et

extern "C" int et_fp8_linear(const et_fp8_linear_args* a) { return et::fp8_linear(a, nullptr); }
// Not part of the public header: one of the plans, pairs with tiles of bn features, or (bn 0) tiles of so many tokens whose K 2^log_split CTAs share, for tests that reach each of them.
extern "C" int et_debug_fp8_linear(const et_fp8_linear_args* a, int bn, int tokens, int log_split) {
    const et::Fp8Plan plan = {bn, tokens, log_split};
    const bool pairs = (bn == 128 || bn == 256) && tokens == 0 && log_split == 0;
    const bool few = bn == 0 && (tokens == 16 || tokens == 32 || tokens == 64 || tokens == 128) && log_split >= 0 && log_split < 4 && (tokens >> log_split) >= 4;
    if (!a || !a->weight || !(pairs || (few && (1 << log_split) <= (a->weight->K + et::kBlock - 1) / et::kBlock))) return et::fail(ET_ERR_INVALID, "et_debug_fp8_linear: no such plan");
    return et::fp8_linear(a, &plan);
}
