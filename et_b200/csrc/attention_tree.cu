// Attention of drafted tokens (a tree of up to 64, or single tokens) over keys and values kept in int8 pages: softmax(scale q . k) v over the keys kept before and, of the drafted
// tokens' own, those whose bit is set. Bound by reading the codes once where there are few rows.
//
// The queries and query heads of a K/V head are rows, eight to a tile of mma.sync m16n8k16: 16 keys x 8 rows of scores, then 16 features x 8 rows of O, so that no part of a tile is empty (with the
// rows as the tile's 16, which four query heads fill to a quarter, twice the products). Codes become halves exactly (three operations for four), the key's scale multiplies the
// score, the value's scale the weight. A block of 16 keys of a head lies in one page: K and V of it come by one TMA copy (16 x 128 bytes each, swizzled; heads of 256 by two),
// a block or two ahead, into a ring that each warp has for itself. (Each lane's pieces by cp.async, 60 instructions of all lanes to a block, took 69 us where this took 58, below; heads of up to 64,
// whose copies are half as large, are 6 to 9 % faster that way and have it.)
// Which features a step of the first product takes, and which the rows of the second are, is free: a lane has 16 neighbouring codes of a key of K, and for V of four keys the codes of 16 (8)
// neighbouring features, by wide loads without bank conflicts. A cluster of CTAs shares a sequence's keys, its warps take blocks of 16 in turn with a reference, sum and O of their own,
// joined in shared and then distributed shared memory in a fixed order: no workspace, one launch, the same bits every time.
//
// 64 sequences of up to 8192 keys, single tokens of 16 heads of 128 over 4: 57 us; codes read once 42. (16 rows of heads of 128 and of 256 spill 12 and 52 bytes.)
//
// Scores, references and sums are fp32; the weights times the values' scales go to the second product as fp16: up to 2^-11 of a weight, at random, so that a result is off by up to 1.4 times what its
// own rounding to fp16 makes. Weights as two halves each, which leaves that rounding alone, need twice the products: single tokens 57 -> 60 us, 16 rows 7 % more.
#include <algorithm>
#include <cooperative_groups.h>
#include "attention.h"
#include "attention_tree.cuh"
#include "attention_tree.h"
#include "common.h"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace et {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kKeys = 16;                 // of a block
constexpr int kMaxCluster = 16;

template <int kHD, int kX>
struct Cfg {
    static constexpr int kRows = 8 * kX;                         // of a CTA
    static constexpr int kFeat = kHD / 8;                        // features of V that a lane has
    static constexpr bool kTma = kHD > 64;
    static constexpr int kPanels = kTma ? kHD / 128 : 1;         // of 128 bytes of a key in shared memory, swizzled
    static constexpr int kSide = kKeys * (kTma ? 128 : 64);      // of K or V in a panel
    static constexpr int kStages = kTma ? 3 : 5;
    static constexpr int kStage = 2 * kPanels * kSide;           // of a warp: [panel][K, V][key], or [copy][lane]: two of 16 bytes of K, four of 8 of V
    static constexpr int kRing = kStages * kStage, kScaleAt = kWarps * kRing;           // then [warp][stage]: the scales of 16 keys of K and of V
    static constexpr int kCopies = kScaleAt + kWarps * kStages * 128;
    static constexpr int kLine = kHD + 4;                        // of a row of O in shared memory, in floats: lanes write to different banks
    static constexpr int kJoin = kWarps * (kRows * kLine + 2 * kRows) * 4;
    static constexpr int kSumAt = kCopies > kJoin ? kCopies : kJoin;   // this CTA's rows: [kRows][kLine] floats, then references and sums
    static constexpr int kBytes = kSumAt + (kRows * kLine + 2 * kRows) * 4 + (kTma ? 1024 : 0);
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
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
// An 8 x 8 matrix of halves, two neighbours of row lane / 4 in each lane, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// An infinite feature of a query makes its row not a number, as it does in 0 times infinity and in infinity - infinity.
__device__ __forceinline__ uint32_t no_infinity(uint32_t two) {
    const uint32_t lo = (two & 0x7fffu) == 0x7c00u ? 0x7fffu : two & 0xffffu, hi = (two & 0x7fff0000u) == 0x7c000000u ? 0x7fff0000u : two & 0xffff0000u;
    return lo | hi;
}

// kHD: 64, 128 or 256, the head's width rounded up. kX: tiles of eight rows.
template <int kHD, int kX>
__global__ void __launch_bounds__(kThreads, kHD == 256 ? 1 : kX == 2 ? 3 : 4) attention_tree_kernel(const __grid_constant__ CUtensorMap codes, const __grid_constant__ TreeParams p, int row_tiles, bool longest_first,
                                                                                                      int* err) {
    using C = Cfg<kHD, kX>;
    constexpr int kRows = C::kRows;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = C::kTma ? (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023) : smem_raw;
    __shared__ uint64_t bars[kWarps][C::kStages];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    cg::cluster_group cluster = cg::this_cluster();
    const int csize = cluster.num_blocks(), crank = cluster.block_rank();
    const int hd = p.head_dim;
    int unit = blockIdx.x / csize;        // sequence, K/V head, tile of rows
    const int tile = unit % row_tiles;
    unit /= row_tiles;
    const int n_kv = p.nhead / p.group, kv_head = unit % n_kv;
    int b = unit / n_kv;
    if (C::kTma && lane == 0) {
        for (int i = 0; i < C::kStages; ++i) mbar_init(&bars[warp][i], 1);
        fence_mbar_init();
        prefetch_tmap(&codes);
    }
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();
    const int len = longest_first ? nth_longest<kThreads>(p, b) : p.k_lens[b];
    const TreeSeq s = tree_seq(p, b, len);
    const int rows = min(s.qlen * p.group - tile * kRows, kRows);
    if (rows <= 0) return;                // the same for the whole cluster
    const int n_blocks = (s.klen + kKeys - 1) / kKeys;
    const int stride = csize * kWarps, mine = crank * kWarps + warp;
    const int* const table = p.table + (long long)b * p.table_width;
    const uint32_t ring = smem_u32(smem) + warp * C::kRing, scales_ring = smem_u32(smem) + C::kScaleAt + warp * C::kStages * 128, bar0 = smem_u32(&bars[warp][0]);
    // Where a block's 16 keys are, which lie in one page: its number is requested a block before it is needed. Blocks are looked up in turn (no division).
    int page_id = -1, page_off = 0, next_n = mine * kKeys / p.page, next_off = mine * kKeys - next_n * p.page, next_i = mine;
    const int step_n = stride * kKeys / p.page, step_off = stride * kKeys - step_n * p.page;
    auto look_up = [&]() {
        page_id = -1;
        if (next_i < n_blocks) {
            page_id = __ldg(table + next_n);
            page_off = next_off;
            next_i += stride;
            next_n += step_n;
            next_off += step_off;
            if (next_off >= p.page) {
                next_off -= p.page;
                ++next_n;
            }
        }
    };
    const long long v_rows = (long long)n_kv * p.page;   // from a key's K to its V
    const float* const scales_at = p.scales + (long long)kv_head * p.page + (lane >> 4) * v_rows + (lane & 15);
    // What the lane reads of a block in heads of up to 64 (nothing behind the head's last feature), from the head's first row in a page on: of K key g and 16 features, of V key 2t and 8.
    const long long page_codes = 2 * v_rows * hd;
    const int8_t* const codes_k = p.codes + (long long)kv_head * p.page * hd + g * hd + t * 16;
    const int8_t* const codes_v = p.codes + (long long)kv_head * p.page * hd + v_rows * hd + 2 * t * hd + g * 8;
    // The block that has been looked up: its codes and scales. Whether its page is there.
    auto fetch = [&](int i, int stage) {
        const bool there = i < n_blocks && page_id >= 0 && page_id < p.pages;
        if (there) {
            const uint32_t to = ring + stage * C::kStage;
            copy_async<4>(scales_ring + stage * 128 + lane * 4, scales_at + (page_id * 2 * v_rows + page_off));
            if constexpr (C::kTma) {
                if (elect_one()) {
                    const uint32_t bar = bar0 + stage * 8;
                    mbar_expect_tx_at(bar, C::kStage);
#pragma unroll
                    for (int n = 0; n < C::kPanels; ++n) load_keys(to + n * 2 * C::kSide, &codes, n * 128, page_off, kv_head, 2 * page_id, bar);
                }
                __syncwarp();
            } else {
                const long long from = page_id * page_codes + (long long)page_off * hd;
                if (t * 16 < hd) {
#pragma unroll
                    for (int n = 0; n < 2; ++n) copy_async<16>(to + n * 512 + lane * 16, codes_k + from + n * 8 * hd);
                }
                if (g * 8 < hd) {
#pragma unroll
                    for (int n = 0; n < 4; ++n) copy_async<8>(to + C::kSide + n * 256 + lane * 8, codes_v + from + ((n & 1) + (n >> 1) * 8) * hd);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return there;
    };
    uint32_t there_bits = 0;              // of the blocks on their way, by stage
    look_up();
#pragma unroll
    for (int n = 0; n < C::kStages - 1; ++n) {
        if (fetch(mine + n * stride, n)) there_bits |= 1u << n;
        look_up();
    }
    // the lane's rows: in scores 8x + 2t and 8x + 2t + 1, as an operand 8x + g
    unsigned long long bits[kX][2];
    uint32_t qf[kX][kHD / 16][2];
#pragma unroll
    for (int x = 0; x < kX; ++x) {
#pragma unroll
        for (int e = 0; e < 2; ++e) bits[x][e] = tree_bits(p, s, (tile * kRows + min(8 * x + 2 * t + e, rows - 1)) / p.group);
        const bool real = 8 * x + g < rows;
        const int r = tile * kRows + (real ? 8 * x + g : 0);
        const half* const q = p.q + (s.q0 + r / p.group) * p.q_pitch + (long long)(kv_head * p.group + r % p.group) * hd;
#pragma unroll
        for (int n = 0; n < kHD / 64; ++n) {   // 16 features of the lane in each 64, four to a step
            const int f = kHD == 64 ? t * 16 : n / 2 * 128 + t * 32 + n % 2 * 16;   // (of a panel: such that neighbouring lanes' pieces of K lie in different banks)
            uint4 a = make_uint4(0u, 0u, 0u, 0u), c = a;
            if (f < hd && real) {
                a = *reinterpret_cast<const uint4*>(q + f);
                c = *reinterpret_cast<const uint4*>(q + f + 8);
            }
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                qf[x][n * 4 + k][0] = no_infinity(w[2 * k]);
                qf[x][n * 4 + k][1] = no_infinity(w[2 * k + 1]);
            }
        }
    }
    float o[kX][C::kFeat / 2][4];         // features 2i and 2i + 1 of the lane's, rows 2t and 2t + 1
    float top[kX][2], sum[kX][2];
#pragma unroll
    for (int x = 0; x < kX; ++x) {
#pragma unroll
        for (int n = 0; n < C::kFeat / 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[x][n][i] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            top[x][e] = -INFINITY;
            sum[x][e] = 0.f;
        }
    }
    bool ok = true;
    uint32_t phases = 0;                  // of the stages' barriers
    int stage = 0, fill = C::kStages - 1;
    for (int i = mine; i < n_blocks; i += stride) {
        const bool next_there = fetch(i + (C::kStages - 1) * stride, fill);   // (the stage was left at the end of the turn before)
        there_bits = (there_bits & ~(1u << fill)) | (next_there ? 1u : 0u) << fill;
        look_up();
        fill = fill + 1 == C::kStages ? 0 : fill + 1;
        const int turn = stage;
        stage = stage + 1 == C::kStages ? 0 : stage + 1;
        if (!((there_bits >> turn) & 1u)) continue;   // keys in a page that there is not: nobody sees them
        asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
        if constexpr (C::kTma) {
            ok = mbar_wait_at(bar0 + turn * 8, (phases >> turn) & 1u);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            phases ^= 1u << turn;
        }
        __syncwarp();                     // (the scales come by all lanes)
        const uint32_t at = ring + turn * C::kStage, scales = scales_ring + turn * 128;
        const int key0 = i * kKeys;
        // ---- scores: the lane has keys g and g + 8 of its rows
        float v[kX][4], v2[kX][4];        // key g: rows 2t, 2t + 1; key g + 8 (every other step, so that a product does not wait for the one before)
#pragma unroll
        for (int x = 0; x < kX; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[x][e] = v2[x][e] = 0.f;
#pragma unroll
        for (int n = 0; n < kHD / 64; ++n) {
            // keys g and g + 8, whose rows' chunks lie in the same order
            const uint32_t k_at = C::kTma ? at + n / 2 * 2 * C::kSide + g * 128 + (((2 * t + n % 2) ^ g) << 4) : at + lane * 16;
            const uint4 k0 = lds128(k_at), k1 = lds128(k_at + C::kSide / 2);
            const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t u0 = codes_biased(w0[k]), u1 = codes_biased(w1[k]);
                const uint32_t a0 = codes_to_half2<0>(u0), a1 = codes_to_half2<0>(u1), a2 = codes_to_half2<1>(u0), a3 = codes_to_half2<1>(u1);
#pragma unroll
                for (int x = 0; x < kX; ++x) mma_16816(k & 1 ? v2[x] : v[x], a0, a1, a2, a3, qf[x][n * 4 + k][0], qf[x][n * 4 + k][1]);
            }
        }
        float ks[2], vs[2], lv[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            ks[e] = __uint_as_float(lds32(scales + (g + 8 * e) * 4)) * p.scale_log2;
            vs[e] = __uint_as_float(lds32(scales + 64 + (g + 8 * e) * 4));
            lv[e] = log2_of_scale(vs[e]);
        }
        float scale[kX][4];
#pragma unroll
        for (int x = 0; x < kX; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[x][e] = (v[x][e] + v2[x][e]) * ks[e >> 1];
                scale[x][e] = vs[e >> 1];
            }
        // masks, where not every row sees every key of the block
        if (key0 + kKeys > s.kept || key0 + kKeys > s.klen) {
#pragma unroll
            for (int x = 0; x < kX; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!tree_sees(s, bits[x][e & 1], key0 + g + (e >> 1) * 8)) {   // (what is not seen may have any scale)
                        v[x][e] = -INFINITY;
                        scale[x][e] = 0.f;
                    }
        }
        bool grow = false;
        float most[kX][2];
#pragma unroll
        for (int x = 0; x < kX; ++x)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                most[x][e] = fmaxf(v[x][e] + lv[0], v[x][e + 2] + lv[1]);
                grow = grow || most[x][e] > top[x][e] + kRescaleStep;   // also true for the first finite score of a row
            }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int x = 0; x < kX; ++x)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) most[x][e] = fmaxf(most[x][e], __shfl_xor_sync(0xffffffffu, most[x][e], d));
                    if (most[x][e] > top[x][e] + kRescaleStep) {
                        const float keep = top[x][e] == -INFINITY ? 0.f : ex2_fast(top[x][e] - most[x][e]);
                        top[x][e] = most[x][e];
                        sum[x][e] *= keep;
#pragma unroll
                        for (int n = 0; n < C::kFeat / 2; ++n) {
                            o[x][n][e] *= keep;
                            o[x][n][e + 2] *= keep;
                        }
                    }
                }
        }
        uint32_t w[kX][2];                // weights as an operand: of row g keys 2t, 2t + 1, then 2t + 8, 2t + 9
#pragma unroll
        for (int x = 0; x < kX; ++x) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float m = top[x][e & 1];
                v[x][e] = ex2_fast(v[x][e] - (m == -INFINITY ? 0.f : m - kLift));
                sum[x][e & 1] += v[x][e];
                v[x][e] *= scale[x][e];
            }
            w[x][0] = transposed(pack2(v[x][0], v[x][1]));
            w[x][1] = transposed(pack2(v[x][2], v[x][3]));
        }
        // ---- O: rows m and m + 8 of the product's tile are features 2i and 2i + 1 of lane m's
#pragma unroll
        for (int h = 0; h < C::kPanels; ++h) {
            uint32_t u[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (C::kTma) {
                    const int key = 2 * t + (k & 1) + (k >> 1) * 8;
                    const uint32_t from = at + h * 2 * C::kSide + C::kSide + key * 128 + ((g ^ (key & 7)) << 4);
                    const uint4 q = lds128(from);
                    u[k][0] = codes_biased(q.x);
                    u[k][1] = codes_biased(q.y);
                    u[k][2] = codes_biased(q.z);
                    u[k][3] = codes_biased(q.w);
                } else {
                    const uint2 q = lds64(at + C::kSide + k * 256 + lane * 8);
                    u[k][0] = codes_biased(q.x);
                    u[k][1] = codes_biased(q.y);
                }
            }
#pragma unroll
            for (int c = 0; c < (kHD == 64 ? 2 : 4); ++c) {   // four features
                const uint32_t lo0 = __byte_perm(u[0][c], u[1][c], 0x5140), hi0 = __byte_perm(u[0][c], u[1][c], 0x7362);
                const uint32_t lo1 = __byte_perm(u[2][c], u[3][c], 0x5140), hi1 = __byte_perm(u[2][c], u[3][c], 0x7362);
                const int n = h * 8 + 2 * c;
#pragma unroll
                for (int x = 0; x < kX; ++x) {
                    mma_16816(o[x][n], codes_to_half2<0>(lo0), codes_to_half2<1>(lo0), codes_to_half2<0>(lo1), codes_to_half2<1>(lo1), w[x][0], w[x][1]);
                    mma_16816(o[x][n + 1], codes_to_half2<0>(hi0), codes_to_half2<1>(hi0), codes_to_half2<0>(hi1), codes_to_half2<1>(hi1), w[x][0], w[x][1]);
                }
            }
        }
        __syncwarp();                     // the stage has been read
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (C::kTma && !ok) {   // (what was requested lands before the CTA leaves, bounded)
        if (lane == 0) {
            atomicExch(err, 28);
            for (int n = 0; n < C::kStages; ++n)
                if ((there_bits >> n) & 1u) mbar_wait_at(bar0 + n * 8, (phases >> n) & 1u);
        }
        __syncwarp();
    }
    // ---- the warps' rows are joined, then the CTAs'
#pragma unroll
    for (int x = 0; x < kX; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int d = 4; d < 32; d *= 2) sum[x][e] += __shfl_xor_sync(0xffffffffu, sum[x][e], d);
    __syncthreads();
    float* const warp_o = reinterpret_cast<float*>(smem);                      // [kWarps][kRows][kLine], feature n of lane m's in column (n / 2) 16 + (n % 2) 8 + m
    float* const warp_ms = warp_o + kWarps * kRows * C::kLine;                 // [kWarps][2][kRows]
    float* const cta_o = reinterpret_cast<float*>(smem + C::kSumAt);           // [kRows][kLine]
    float* const cta_ms = cta_o + kRows * C::kLine;                            // [2][kRows]
#pragma unroll
    for (int x = 0; x < kX; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 8 * x + 2 * t + e;
            float* const line = warp_o + (warp * kRows + r) * C::kLine + g;
#pragma unroll
            for (int n = 0; n < C::kFeat / 2; ++n) {
                line[n * 16] = o[x][n][e];
                line[n * 16 + 8] = o[x][n][e + 2];
            }
            if (g == 0) {
                // (scores that are not numbers leave no reference: any finite one makes the part count below)
                warp_ms[warp * 2 * kRows + r] = sum[x][e] == sum[x][e] ? top[x][e] : 0.f;
                warp_ms[warp * 2 * kRows + kRows + r] = sum[x][e];
            }
        }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * kHD; e += kThreads) {
        const int r = e / kHD, c = e % kHD;
        float m = -INFINITY, l = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, warp_ms[w * 2 * kRows + r]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float part = warp_ms[w * 2 * kRows + r];
            if (tree_saw(part)) {
                const float f = ex2_fast(part - m);
                v = fmaf(f, warp_o[(w * kRows + r) * C::kLine + c], v);
                l = fmaf(f, warp_ms[w * 2 * kRows + kRows + r], l);
            }
        }
        cta_o[r * C::kLine + c] = v;
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
            const int n = kHD == 64 ? f % 8 : f / 128 * 16 + f % 16, c = n / 2 * 16 + n % 2 * 8 + (kHD == 64 ? f / 8 : f % 128 / 16);
            float l = 0.f, v = 0.f;
#pragma unroll
            for (int k = 0; k < kMaxCluster; ++k) {
                if (tree_saw(part_m[k])) {
                    const float x = ex2_fast(part_m[k] - m);
                    v = fmaf(x, cluster.map_shared_rank(cta_o, k)[r * C::kLine + c], v);
                    l = fmaf(x, cluster.map_shared_rank(cta_ms, k)[kRows + r], l);
                }
            }
            const int row = tile * kRows + r, i = row / p.group, h = kv_head * p.group + row % p.group;
            p.out[(s.q0 + i) * p.out_pitch + (long long)h * hd + f] = __float2half_rn(l == 0.f ? 0.f : v / l);
        }
    }
    cluster.sync();   // nobody leaves while its rows are read
}

template <int kHD, int kX>
cudaError_t launch(const TreeParams& p, int row_tiles, long long units, int csize, int* err, cudaStream_t st) {
    CUtensorMap codes = {};
    if (Cfg<kHD, kX>::kTma && p.pages > 0 && p.codes && !make_tmap_codes(&codes, p, true)) return cudaErrorInvalidValue;
    const auto kernel = attention_tree_kernel<kHD, kX>;
    static PerDeviceOnce once;
    const cudaError_t e = once.run([&] {
        cudaError_t x = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<kHD, kX>::kBytes);
        if (x == cudaSuccess) x = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        return x;
    });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * csize));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg<kHD, kX>::kBytes;
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
    return cudaLaunchKernelEx(&cfg, kernel, codes, p, row_tiles, longest_first, err);
}

}  // namespace
}  // namespace et

namespace et {
namespace {
// kernel: 0 few rows, 1 many rows, below 0 the one that the model says, with its cluster.
int tree_run(const et_attention_tree_args* a, int kernel, int csize) {
    ET_REQUIRE(a, "et_attention_tree: null pointer");
    ET_REQUIRE(a->batch >= 0 && a->q_tokens >= 0 && a->max_q_len >= 0 && a->max_k_len >= 0 && a->pages >= 0 && a->table_width >= 0, "et_attention_tree: negative size");
    ET_REQUIRE(a->nhead_kv > 0 && a->nhead > 0 && a->nhead % a->nhead_kv == 0, "et_attention_tree: nhead must be a multiple of nhead_kv");
    ET_REQUIRE(a->head_dim >= 16 && a->head_dim <= 256 && a->head_dim % 16 == 0, "et_attention_tree: head_dim must be a multiple of 16 up to 256");
    ET_REQUIRE(a->page >= 16 && a->page % 16 == 0, "et_attention_tree: the rows of a page must be a multiple of 16");
    ET_REQUIRE(a->max_q_len <= 64, "et_attention_tree: at most 64 drafted tokens to a sequence");
    ET_REQUIRE(a->scale >= 0.f && a->scale < INFINITY, "et_attention_tree: scale must be a finite number, 0 for 1 / sqrt(head_dim)");
    ET_REQUIRE((long long)a->nhead * a->head_dim <= 0x7fffffff && (long long)a->nhead / a->nhead_kv * a->max_q_len <= 0x7fffff && (long long)a->batch * a->max_q_len <= 0x7fffffff &&
                   a->max_k_len <= 0x7ff00000,
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
    const cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    if (kernel == 0) return attention_tree_launch(p, csize, st);
    if (kernel == 1) return attention_tree_tc_launch(p, csize, st);
    const TreePlan few = attention_tree_plan(p), many = attention_tree_tc_plan(p);
    return many.us < few.us ? attention_tree_tc_launch(p, many.csize, st) : attention_tree_launch(p, few.csize, st);
}
}  // namespace
}  // namespace et

extern "C" int et_attention_tree(const et_attention_tree_args* a) { return et::tree_run(a, -1, 1); }
// Not part of the public header: one of the kernels with a cluster of 1 to 16, for tests that reach each of them.
extern "C" int et_debug_attention_tree(const et_attention_tree_args* a, int kernel, int log_csize) {
    if (!a || kernel < 0 || kernel > 1 || log_csize < 0 || log_csize > 4 || (kernel == 1 && a->head_dim > 128)) return et::fail(ET_ERR_INVALID, "et_debug_attention_tree: no such kernel");
    return et::tree_run(a, kernel, 1 << log_csize);
}

namespace et {

TreePlan attention_tree_plan(const TreeParams& p) {
    const int rows = p.max_q_len * p.group, tiles = rows > 8 ? 2 : 1;
    const long long units = (long long)p.batch * (p.nhead / p.group) * ((rows + 8 * tiles - 1) / (8 * tiles));
    const int turns = std::max(1, (p.max_k_len + kKeys * kWarps - 1) / (kKeys * kWarps));
    const double sm = sm_count();
    static const TreeCosts costs[2][2] = {{{0.40, 1.04, 5.5, 2.4, 4.0, {1.0, 1.1, 1.1}, 0.0}, {0.49, 1.09, 7.6, 3.7, 3.0, {1.0, 1.1, 1.1}, 0.0}},
                                          {{0.67, 1.77, 5.5, 3.6, 4.0, {1.1, 1.1, 0.51}, 0.0}, {0.87, 1.89, 8.0, 6.8, 3.0, {1.1, 1.1, 1.1}, 0.0}}};
    TreeCosts c = costs[p.head_dim > 64][tiles - 1];
    if (p.head_dim > 128) c = {2 * c.alone, 2 * c.shared, c.start, c.start_shared, tiles == 2 ? 1.0 : 2.0, {1.0, 1.0, 0.44}, 0.0};   // (not fitted: twice a head of 128)
    c.places *= sm;
    return tree_plan(units, turns, sm_count(), c);
}

int attention_tree_launch(const TreeParams& p, int csize, cudaStream_t st) {
    const int all_rows = p.max_q_len * p.group, tiles = all_rows > 8 ? 2 : 1, row_tiles = (all_rows + 8 * tiles - 1) / (8 * tiles);
    const long long units = (long long)p.batch * (p.nhead / p.group) * row_tiles;
    if (units * kMaxCluster > 0x7fffffff) return fail(ET_ERR_INVALID, "et_attention_tree: too large");
    int* err = nullptr;
    const int rc = attn_err_address(&err);
    if (rc) return rc;
    const auto run = p.head_dim <= 64    ? (tiles == 2 ? launch<64, 2> : launch<64, 1>)
                     : p.head_dim <= 128 ? (tiles == 2 ? launch<128, 2> : launch<128, 1>)
                                         : (tiles == 2 ? launch<256, 2> : launch<256, 1>);
    return cuda_status(run(p, row_tiles, units, csize, err, st), "et_attention_tree launch");
}

}  // namespace et
