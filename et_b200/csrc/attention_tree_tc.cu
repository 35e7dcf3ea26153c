// Attention of drafted tokens over a cache of int8 codes, many rows: a CTA has up to 128 of the rows (queries x query heads) of a K/V head, so that both products go to tcgen05 and a
// code is converted once for all of them.
//
// Blocks of 64 keys. Four warps have 16 keys of a block each, which lie in one page: they fetch the codes (one TMA copy; heads of up to 64, whose copies are half as large, by cp.async) into a place of
// their own, a block or more ahead, and write them as halves where the tensor cores read them (rows of 64 features, 128-byte swizzle; V as it lies, features are its N). Q lies in tensor memory as the first product's A operand, the scores beside it, and the weights where the
// scores were, as the second product's A operand. A thread has a row: scale of the key, mask, weight times the value's scale, a running reference that moves when
// it has to (then O is rescaled in tensor memory). Two CTAs share an SM: while one waits for its products the other takes exponentials. A cluster shares a sequence's keys; its CTAs' rows are joined
// through distributed shared memory in a fixed order.
//
// 16 sequences of up to 12000 keys and 48 drafted tokens, 32 heads of 128 over 8: 149 us (146 without the warps' votes on their waits; with codes by cp.async 4 more, with the scores' UMMAs in a loop that is not unrolled 5 more besides); codes read once 36. No unit is full
// (shared-memory pipe 40 %, ALU 29 %, issue slots 38 %, tensor pipe 22 %): a CTA's block is a chain, scores -> 64 scales, maxima and exponentials -> weights -> both products, some 3200 clocks
// with two CTAs to an SM. (Of 128 registers a thread 12 bytes are spilled.) Tried, against 146: scores in halves of 32 keys, one multiplied while the other is weighed, by a warp of its own that issues UMMAs 165 (20 of them to a block instead of 12, some 45
// clocks of the issuing thread each); two places for scores, Q in shared memory (as tensor memory is full then), such a warp, registers handed over 174 (with Q in tensor memory and one place 163),
// with codes fetched into registers 168 to 178 (operands from shared memory take all of its bandwidth at N 64); codes fetched into registers in this form 189; clusters of two and eight 165 and 182. Weights
// as two halves each, for results as exact as fp16 has them, take 174 us (attention_tree.cu says what one half costs them).
#include <cooperative_groups.h>
#include <type_traits>
#include "attention.h"
#include "attention_tree.cuh"
#include "attention_tree.h"
#include "common.h"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace et {
namespace {

constexpr int kKeys = 64;                 // of a block
constexpr int kRows = 128;                // of a CTA
constexpr int kSoftmaxWarps = 4, kConvertWarps = 4, kThreads = 8 * 32;   // (two CTAs to an SM with 128 registers a thread)
constexpr int kMaxCluster = 16;
constexpr int kScaleStages = 4, kScaleBytes = kKeys * (4 + 4 + 2);
constexpr uint32_t kTmemCols = 256;

template <int kHD>
struct Cfg {
    static constexpr int kPanel = kKeys * 128, kTile = kHD / 64 * kPanel;       // halves of a block of K or V
    static constexpr int kChunks = kKeys * kHD / 16 / 128;                      // 16 codes each, of a thread, of K and of V
    static constexpr bool kTma = kHD > 64;
    static constexpr int kPiece = 2 * 16 * kHD;                                 // codes of 16 keys, of K and of V
    static constexpr int kRawStages = kHD == 64 ? 4 : 2;
    static constexpr uint32_t kQCol = 0, kSCol = kHD / 2, kOCol = kSCol + kKeys;
    static_assert(kOCol + kHD <= kTmemCols, "");
    static constexpr int kKAt = 0, kVAt = 2 * kTile, kRawAt = 4 * kTile;
    static constexpr int kScaleAt = kRawAt + kRawStages * kConvertWarps * (kPiece + 128);                 // [stage]: of 64 keys score factors, values' scales, their logarithms as fp16
    static constexpr int kPartAt = kScaleAt + kScaleStages * kScaleBytes;     // [reference, sum][128]
    // Half of an SM's shared memory for half of its tensor memory: a CTA that finds one finds the other, and none waits for columns that another cluster holds.
    static constexpr int kBytes = 113664;
    static_assert(kPartAt + 2 * kRows * 4 + 1024 <= kBytes && kTmemCols == 256, "");
    static_assert(kRows * kHD * 4 <= 4 * kTile, "O in 32 bits fits where the blocks were");
};

struct Shared {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t raw_full[kConvertWarps][4];
    uint64_t scales_full[kScaleStages], q_ready, s_full, p_ready, o_done;
    uint32_t good[kScaleStages];          // a byte for each 16 keys of a block: 1 if their page is there
    uint32_t tmem_base;
};

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t no_infinity(uint32_t two) {
    const uint32_t lo = (two & 0x7fffu) == 0x7c00u ? 0x7fffu : two & 0xffffu, hi = (two & 0x7fff0000u) == 0x7c000000u ? 0x7fff0000u : two & 0xffff0000u;
    return lo | hi;
}
// Two halves added to two fp32 values.
__device__ __forceinline__ void add_halves(uint32_t h, float a, float b, float& x, float& y) {
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\nadd.rn.f32.f16 %0, l, %3;\nadd.rn.f32.f16 %1, h, %4;\n}" : "=f"(x), "=f"(y) : "r"(h), "f"(a), "f"(b));
}
__device__ __forceinline__ float4 lds_f4(uint32_t a) {
    const uint4 v = lds128(a);
    return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}

template <int kHD>
__global__ void __launch_bounds__(kThreads, 2) attention_tree_tc_kernel(const __grid_constant__ CUtensorMap codes, const __grid_constant__ TreeParams p, int row_tiles, bool longest_first, int* err) {
    using C = Cfg<kHD>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ Shared shared;
    Shared* const sh = &shared;
    const uint32_t at = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    cg::cluster_group cluster = cg::this_cluster();
    const int csize = cluster.num_blocks(), crank = cluster.block_rank();
    int unit = blockIdx.x / csize;        // sequence, K/V head, tile of rows
    const int tile = unit % row_tiles;
    unit /= row_tiles;
    const int n_kv = p.nhead / p.group, kv_head = unit % n_kv;
    int b = unit / n_kv;
    pdl_wait();
    const int len = longest_first ? nth_longest<kThreads>(p, b) : p.k_lens[b];
    const TreeSeq s = tree_seq(p, b, len);
    const int rows = min(s.qlen * p.group - tile * kRows, kRows), hd = p.head_dim;
    if (rows <= 0) return;                // the same for the whole cluster
    const int row_warps = (rows + 31) / 32;   // the other softmax warps have no row: their lanes of tensor memory hold anything, which no row sees
    const int n_blocks = (s.klen + kKeys - 1) / kKeys, mine = n_blocks > crank ? (n_blocks - crank + csize - 1) / csize : 0;   // blocks crank, crank + csize, ..
    if (warp == kSoftmaxWarps) {
        if (lane == 0) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(&sh->k_full[i], kConvertWarps);
                mbar_init(&sh->v_full[i], kConvertWarps);
                mbar_init(&sh->k_empty[i], 1);
                mbar_init(&sh->v_empty[i], 1);
            }
            for (int i = 0; i < kScaleStages; ++i) mbar_init(&sh->scales_full[i], kConvertWarps);
            if (C::kTma)
                for (int i = 0; i < kConvertWarps * C::kRawStages; ++i) mbar_init(&sh->raw_full[i / C::kRawStages][i % C::kRawStages], 1);
            mbar_init(&sh->q_ready, row_warps);
            mbar_init(&sh->s_full, 1);
            mbar_init(&sh->p_ready, row_warps);
            mbar_init(&sh->o_done, 1);
            fence_mbar_init();
            if (C::kTma) prefetch_tmap(&codes);
        }
        __syncwarp();
        tmem_alloc(&sh->tmem_base, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;
    pdl_launch_dependents();
    bool ok = true;
    float top = -INFINITY, sum = 0.f;
    if (warp >= kSoftmaxWarps) {
        // ---- codes to halves: a warp has 16 keys of a block, which lie in one page
        const int w = warp - kSoftmaxWarps;
        constexpr int kPerKey = kHD / 16, kPass = 32 / kPerKey;       // lanes, of 16 codes each, to a key; keys at once
        const int key_c = lane / kPerKey, f = (lane % kPerKey) * 16, key_s = w * 16 + (lane & 15), side_s = lane >> 4;   // (whose scale it brings)
        const int* const table = p.table + (long long)b * p.table_width;
        const uint32_t raw = at + C::kRawAt + w * C::kRawStages * C::kPiece, raw_scales = at + C::kRawAt + kConvertWarps * C::kRawStages * C::kPiece + w * C::kRawStages * 128;
        const long long v_rows = (long long)n_kv * p.page, page_rows = 2 * v_rows;   // from a key's K to its V; of a page
        // what the lane reads of a block, from the head's first row in a page on (codes in heads of up to 64)
        const int8_t* const codes_at = p.codes + (long long)kv_head * p.page * hd + key_c * hd + f;
        const float* const scales_at = p.scales + (long long)kv_head * p.page + side_s * v_rows + (lane & 15);
        // The page's number is requested a block before it is needed, places in turn (no division).
        int piece_key = crank * kKeys + w * 16, piece_n = piece_key / p.page, next_off = piece_key - piece_n * p.page, piece_id = -1, piece_off = 0;
        const int step = csize * kKeys, step_n = step / p.page, step_off = step - step_n * p.page;
        auto look_up = [&]() {                                        // the next block
            piece_id = -1;
            if (piece_key < s.klen) {
                piece_id = __ldg(table + piece_n);
                piece_off = next_off;
                piece_key += step;
                piece_n += step_n;
                next_off += step_off;
                if (next_off >= p.page) {
                    next_off -= p.page;
                    ++piece_n;
                }
            }
        };
        uint32_t there_bits = 0, phases = 0;                          // of the places: their page is there; phases of their barriers
        auto fetch = [&](int j) {                                     // block j, whose page has been looked up
            const bool there = j < mine && piece_id >= 0 && piece_id < p.pages;
            const int place = j % C::kRawStages;
            there_bits = (there_bits & ~(1u << place)) | (there ? 1u : 0u) << place;
            if (there) {
                const uint32_t to = raw + place * C::kPiece;
                copy_async<4>(raw_scales + place * 128 + lane * 4, scales_at + (piece_id * page_rows + piece_off));
                if constexpr (C::kTma) {
                    if (elect_one()) {
                        const uint32_t bar = smem_u32(&sh->raw_full[w][place]);
                        mbar_expect_tx_at(bar, C::kPiece);
                        load_keys(to, &codes, 0, piece_off, kv_head, 2 * piece_id, bar);
                    }
                    __syncwarp();
                } else if (f < hd) {
                    const int8_t* const k = codes_at + (piece_id * page_rows + piece_off) * hd;
#pragma unroll
                    for (int n = 0; n < C::kChunks; ++n) {
                        copy_async<16>(to + n * 512 + lane * 16, k + n * kPass * hd);
                        copy_async<16>(to + C::kPiece / 2 + n * 512 + lane * 16, k + (v_rows + n * kPass) * hd);
                    }
                }
            }
            look_up();
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        // 16 codes of the thread as halves at 16 bytes 2 f / 16 and the next of the key's row. (Every second thread of eight that write at once takes the second 16 bytes first:
        // rows of two panels lie on the same banks.)
        auto convert = [&](uint32_t from, uint32_t tile_at, int key) {
            const uint4 w = lds128(from);
            const uint32_t u[4] = {codes_biased(w.x), codes_biased(w.y), codes_biased(w.z), codes_biased(w.w)};
            uint4 h[2];
            h[0] = make_uint4(codes_to_half2<0>(u[0]), codes_to_half2<1>(u[0]), codes_to_half2<0>(u[1]), codes_to_half2<1>(u[1]));
            h[1] = make_uint4(codes_to_half2<0>(u[2]), codes_to_half2<1>(u[2]), codes_to_half2<0>(u[3]), codes_to_half2<1>(u[3]));
            const uint32_t line = tile_at + (f >> 6) * C::kPanel + key * 128;
            const int chunk = (f & 63) >> 3, swap = kHD == 128 ? f >> 6 : 0;
            sts128(line + (((chunk + swap) ^ (key & 7)) << 4), swap ? h[1] : h[0]);
            sts128(line + (((chunk + 1 - swap) ^ (key & 7)) << 4), swap ? h[0] : h[1]);
        };
        look_up();
        for (int n = 0; n < C::kRawStages - 1; ++n) fetch(n);
        for (int j = 0; j < mine; ++j) {
            fetch(j + C::kRawStages - 1);   // (the warp has read that place a turn ago)
            const int st = j & 1, key0 = (crank + j * csize) * kKeys, place = j % C::kRawStages;
            const uint32_t ph = ((uint32_t)(j >> 1) & 1u) ^ 1u, from = raw + place * C::kPiece + lane * 16;
            const bool there = (there_bits >> place) & 1u;            // (where not, any codes are converted, which no row sees)
            asm volatile("cp.async.wait_group %0;" ::"n"(C::kRawStages - 1) : "memory");
            if (C::kTma && there) {
                ok = mbar_wait_warp(&sh->raw_full[w][place], (phases >> place) & 1u);
                if (!ok) break;
                phases ^= 1u << place;
                there_bits &= ~(1u << place);
            }
            ok = mbar_wait_warp(&sh->k_empty[st], ph);
            if (!ok) break;
#pragma unroll
            for (int n = 0; n < C::kChunks; ++n) convert(from + n * 512, at + C::kKAt + st * C::kTile, w * 16 + key_c + n * kPass);
            // Scales go to the places of block j - 4, whose scores are done with: those of block j - 2 have been multiplied, behind the weights of block j - 3.
            const float scale = __uint_as_float(lds32(raw_scales + place * 128 + lane * 4));
            const bool real = there && key0 + key_s < s.klen;   // (behind the last key anything may lie)
            uint8_t* const to = smem + C::kScaleAt + (j % kScaleStages) * kScaleBytes;
            if (side_s == 0) {
                reinterpret_cast<float*>(to)[key_s] = real ? scale * p.scale_log2 : 0.f;
            } else {
                reinterpret_cast<float*>(to)[kKeys + key_s] = real ? scale : 0.f;
                reinterpret_cast<half*>(to + 8 * kKeys)[key_s] = __float2half_rn(log2_of_scale(real ? scale : 0.f));   // (for the reference alone)
            }
            if (lane == 0) reinterpret_cast<uint8_t*>(&sh->good[j % kScaleStages])[w] = there ? 1 : 0;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh->scales_full[j % kScaleStages]);
                mbar_arrive(&sh->k_full[st]);
            }
            ok = mbar_wait_warp(&sh->v_empty[st], ph);
            if (!ok) break;
#pragma unroll
            for (int n = 0; n < C::kChunks; ++n) convert(from + C::kPiece / 2 + n * 512, at + C::kVAt + st * C::kTile, w * 16 + key_c + n * kPass);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->v_full[st]);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (!ok && lane == 0) {
            atomicExch(err, 26);
            for (int n = 0; C::kTma && n < C::kRawStages; ++n)   // what was requested lands before the CTA leaves (bounded)
                if ((there_bits >> n) & 1u) mbar_wait(&sh->raw_full[w][n], (phases >> n) & 1u);
        }
    } else if (warp < row_warps) {
        // ---- a row to a thread
        const uint32_t mine_at = tmem + ((uint32_t)warp << 21);       // the warp's lanes of tensor memory
        const bool real = tid < rows;
        const int r = tile * kRows + (real ? tid : 0), i = r / p.group;
        const unsigned long long bits = tree_bits(p, s, i);
        if (mine > 0) {
            const half* const q = p.q + (s.q0 + i) * p.q_pitch + (long long)(kv_head * p.group + r % p.group) * hd;
#pragma unroll
            for (int n = 0; n < kHD / 32; ++n) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int f = n * 32 + e * 8;
                    const uint4 v = real && f < hd ? *reinterpret_cast<const uint4*>(q + f) : make_uint4(0u, 0u, 0u, 0u);
                    w[4 * e] = no_infinity(v.x);
                    w[4 * e + 1] = no_infinity(v.y);
                    w[4 * e + 2] = no_infinity(v.z);
                    w[4 * e + 3] = no_infinity(v.w);
                }
                tmem_store16(mine_at + C::kQCol + n * 16, w);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->q_ready);
        }
        // The first warp issues the UMMAs too: everybody waits for them anyway.
        const uint32_t idesc_qk = make_idesc_f16(128, kKeys), idesc_pv = make_idesc_f16(128, hd, false, true);
        const uint64_t k_desc = make_smem_desc(at + C::kKAt, 16, 1024, 2), v_desc = make_smem_desc(at + C::kVAt, C::kPanel, 1024, 2);
        auto scores_of = [&](int j) {   // (where the weights of the block before lie, which are read by then: UMMAs of a thread run in order)
            if (!mbar_wait(&sh->k_full[j & 1], (uint32_t)(j >> 1) & 1u)) return false;
            tc_fence_after();
            const uint64_t kd = k_desc + (j & 1) * (C::kTile >> 4);
#pragma unroll
            for (int ks = 0; ks < kHD / 16; ++ks)
                if (ks * 16 < hd) umma_f16_ts(tmem + C::kSCol, tmem + C::kQCol + ks * 8, kd + ((ks >> 2) * C::kPanel + (ks & 3) * 32) / 16, idesc_qk, ks > 0);
            umma_commit(&sh->k_empty[j & 1]);
            umma_commit(&sh->s_full);
            return true;
        };
        if (warp == 0 && mine > 0) {
            if (elect_one()) ok = mbar_wait(&sh->q_ready, 0) && scores_of(0);
            __syncwarp();
        }
        for (int j = 0; j < mine; ++j) {
            const int key0 = (crank + j * csize) * kKeys;
            // (Not for k_full: the place may be full of block j + 2 before this warp looks, and the phases of two blocks look alike. The scales of block j + 4 wait for this one's weights.)
            ok = mbar_wait_warp(&sh->scales_full[j % kScaleStages], (uint32_t)(j / kScaleStages) & 1u) && mbar_wait_warp(&sh->s_full, (uint32_t)j & 1u);
            if (!ok) break;
            tc_fence_after();
            uint32_t raw[2][32];
            tmem_ld32(mine_at + C::kSCol, raw[0]);
            tmem_ld32(mine_at + C::kSCol + 32, raw[1]);
            tmem_ld_wait(raw[0], raw[1]);
            const uint32_t scales = at + C::kScaleAt + (j % kScaleStages) * kScaleBytes;
            // what the row sees of the block
            const uint32_t good = sh->good[j % kScaleStages];
            const bool masked = key0 + kKeys > s.kept || key0 + kKeys > s.klen || good != 0x01010101u;   // the same for the whole CTA
            unsigned long long seen = ~0ull;
            if (masked) {
                const int d = key0 - s.kept;   // place of the first key among the drafted tokens
                seen = d >= 64 ? 0ull : d >= 0 ? bits >> d : d > -64 ? (bits << -d) | ((1ull << -d) - 1ull) : ~0ull;
                const int left = s.klen - key0;
                if (left < 64) seen &= (1ull << left) - 1ull;
                if (good != 0x01010101u)
                    for (int n = 0; n < 4; ++n)
                        if (!((good >> (8 * n)) & 1u)) seen &= ~(0xffffull << (n * 16));
            }
            float most = -INFINITY;
            auto two = [](const uint32_t* x) { return make_float2(__uint_as_float(x[0]), __uint_as_float(x[1])); };
            // (with and without masks by themselves: a branch at every four keys kept the others' loads behind it, 2200 clocks for 700)
            auto largest = [&](auto with_masks) {
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < kKeys; e += 8) {
                    const uint4 lv8 = lds128(scales + 8 * kKeys + e * 2);
                    const uint32_t lv[4] = {lv8.x, lv8.y, lv8.z, lv8.w};
#pragma unroll
                    for (int k = 0; k < 8; k += 4) {
                        const float4 ks = lds_f4(scales + (e + k) * 4);
                        uint32_t* const x = &raw[e >> 5][(e & 31) + k];
                        const float2 a = mul2(two(x), make_float2(ks.x, ks.y)), c = mul2(two(x + 2), make_float2(ks.z, ks.w));
                        float v[4] = {a.x, a.y, c.x, c.y}, t[4];
                        if constexpr (with_masks) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (!((seen >> (e + k + i)) & 1ull)) v[i] = -INFINITY;
                        }
                        add_halves(lv[k / 2], v[0], v[1], t[0], t[1]);
                        add_halves(lv[k / 2 + 1], v[2], v[3], t[2], t[3]);
                        m4[k / 2] = max3(m4[k / 2], t[0], t[1]);
                        m4[k / 2 + 1] = max3(m4[k / 2 + 1], t[2], t[3]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[i] = __float_as_uint(v[i]);
                    }
                }
                return fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]);
            };
            most = masked ? largest(std::true_type()) : largest(std::false_type());
            const bool grow = most > top + kRescaleStep;   // also true for the first finite score of a row
            if (__any_sync(0xffffffffu, grow)) {
                const float keep = grow ? (top == -INFINITY ? 0.f : ex2_fast(top - most)) : 1.f;
                if (grow) top = most;
                sum *= keep;
                if (j > 0) {   // (these scores were multiplied behind the weights of the block before: O is at rest)
                    for (int n = 0; n < hd; n += 16) {
                        uint32_t o[16];
                        tmem_ld16(mine_at + C::kOCol + n, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                        tmem_store16(mine_at + C::kOCol + n, o);
                    }
                }
            }
            const float shift = top == -INFINITY ? 0.f : kLift - top;
            auto weights = [&](auto with_masks) {
                float2 sums = make_float2(0.f, 0.f);
                const float2 shift2 = make_float2(shift, shift);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 vs = lds_f4(scales + (kKeys + h * 32 + e) * 4);
                        float2 a = add2(two(&raw[h][e]), shift2), c = add2(two(&raw[h][e] + 2), shift2);
                        a.x = ex2_fast(a.x);
                        a.y = ex2_fast(a.y);
                        c.x = ex2_fast(c.x);
                        c.y = ex2_fast(c.y);
                        float2 x = mul2(a, make_float2(vs.x, vs.y)), y = mul2(c, make_float2(vs.z, vs.w));
                        if constexpr (with_masks) {   // (what is not seen may have any scale)
                            const uint32_t m = (uint32_t)(seen >> (h * 32 + e));
                            if (!(m & 1u)) x.x = 0.f;
                            if (!(m & 2u)) x.y = 0.f;
                            if (!(m & 4u)) y.x = 0.f;
                            if (!(m & 8u)) y.y = 0.f;
                        }
                        sums = add2(sums, add2(a, c));
                        w[e / 2] = pack2(x.x, x.y);
                        w[e / 2 + 1] = pack2(y.x, y.y);
                    }
                    tmem_store16(mine_at + C::kSCol + h * 16, w);
                }
                sum += sums.x + sums.y;
            };
            if (masked) weights(std::true_type());
            else weights(std::false_type());
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->p_ready);
            if (warp == 0) {
                if (elect_one()) {
                    ok = mbar_wait(&sh->p_ready, (uint32_t)j & 1u) && mbar_wait(&sh->v_full[j & 1], (uint32_t)(j >> 1) & 1u);
                    if (ok) {
                        tc_fence_after();
                        const uint64_t vd = v_desc + (j & 1) * (C::kTile >> 4);
#pragma unroll
                        for (int ks = 0; ks < kKeys / 16; ++ks) umma_f16_ts(tmem + C::kOCol, tmem + C::kSCol + ks * 8, vd + ks * (2048 / 16), idesc_pv, j > 0 || ks > 0);
                        umma_commit(&sh->v_empty[j & 1]);
                        if (j + 1 == mine) umma_commit(&sh->o_done);
                        else ok = scores_of(j + 1);
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
            }
        }
        // O goes to shared memory where the blocks were: [row][features], 16 bytes c of a row at c ^ row, so that rows lie on different banks
        if (ok && mine > 0) ok = mbar_wait_warp(&sh->o_done, 0);
        if (!ok && lane == 0) atomicExch(err, 27);
    }
    __syncwarp();
    __syncthreads();   // (whoever gave up: the converting warps write no more)
    if (warp < kSoftmaxWarps) {
        tc_fence_after();
        float* const part = reinterpret_cast<float*>(smem + C::kPartAt);
        // (scores that are not numbers leave no reference: any finite one makes the part count below)
        part[tid] = sum == sum ? top : 0.f;
        part[kRows + tid] = sum;
        if (mine > 0) {
            const uint32_t from = tmem + ((uint32_t)warp << 21) + C::kOCol;
#pragma unroll
            for (int n = 0; n < kHD; n += 16) {
                uint32_t o[16];
                tmem_ld16(from + n, o);
                tmem_ld_wait(o);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    sts128(at + tid * kHD * 4 + (((n / 4 + k) ^ (tid & (kHD / 4 - 1))) << 4), make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]));
            }
        }
    }
    tc_fence_before();
    cluster.sync();
    tc_fence_after();
    if (warp == kSoftmaxWarps) tmem_dealloc(tmem, kTmemCols);
    // ---- the CTAs' rows are joined: a row to kHD / 4 lanes
    constexpr int kLanes = kHD / 4, kGroups = kThreads / kLanes;
    for (int r = crank + csize * (tid / kLanes); r < rows; r += csize * kGroups) {
        const int chunk = tid % kLanes;
        float part_m[kMaxCluster], m = -INFINITY, l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) part_m[k] = k < csize ? reinterpret_cast<const float*>(cluster.map_shared_rank(smem, k) + C::kPartAt)[r] : -INFINITY;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) m = fmaxf(m, part_m[k]);
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            if (tree_saw(part_m[k])) {   // (a part that has seen nothing has no reference)
                const uint8_t* const other = cluster.map_shared_rank(smem, k);
                const float f = ex2_fast(part_m[k] - m);
                const float4 o = *reinterpret_cast<const float4*>(other + r * kHD * 4 + ((chunk ^ (r & (kHD / 4 - 1))) << 4));
                l = fmaf(f, reinterpret_cast<const float*>(other + C::kPartAt)[kRows + r], l);
                v.x = fmaf(f, o.x, v.x);
                v.y = fmaf(f, o.y, v.y);
                v.z = fmaf(f, o.z, v.z);
                v.w = fmaf(f, o.w, v.w);
            }
        }
        if (chunk * 4 < hd) {
            const float inv = 1.f / l;
            const bool none = l == 0.f;
            const int row = tile * kRows + r, i = row / p.group, h = kv_head * p.group + row % p.group;
            const uint2 z = none ? make_uint2(0u, 0u) : make_uint2(pack2(v.x * inv, v.y * inv), pack2(v.z * inv, v.w * inv));
            *reinterpret_cast<uint2*>(p.out + (s.q0 + i) * p.out_pitch + (long long)h * hd + chunk * 4) = z;
        }
    }
    cluster.sync();   // nobody leaves while its rows are read
}

template <int kHD>
cudaError_t launch(const TreeParams& p, int row_tiles, long long units, int csize, int* err, cudaStream_t st) {
    CUtensorMap codes = {};
    if (Cfg<kHD>::kTma && p.pages > 0 && p.codes && !make_tmap_codes(&codes, p, false)) return cudaErrorInvalidValue;
    const auto kernel = attention_tree_tc_kernel<kHD>;
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
    const bool longest_first = p.batch <= kThreads && units * csize > 2 * sm_count();
    return cudaLaunchKernelEx(&cfg, kernel, codes, p, row_tiles, longest_first, err);
}

}  // namespace

TreePlan attention_tree_tc_plan(const TreeParams& p) {
    if (p.head_dim > 128 || p.max_k_len < 1) return {1e30, 1};
    const int rows = p.max_q_len * p.group;
    const long long units = (long long)p.batch * (p.nhead / p.group) * ((rows + kRows - 1) / kRows);
    const double part = (rows < kRows ? rows : kRows) / (double)kRows, places = 2.0 * sm_count();
    const TreeCosts narrow = {1.03, 1.37, 7.1, 3.1, places, {1.0, 1.0, 0.78}, 0.22 * part}, wide = {1.10, 1.67, 7.7, 4.6, places, {1.1, 1.1, 0.59}, 0.445 * part};
    return tree_plan(units, (p.max_k_len + kKeys - 1) / kKeys, sm_count(), p.head_dim > 64 ? wide : narrow);
}

int attention_tree_tc_launch(const TreeParams& p, int csize, cudaStream_t st) {
    const int row_tiles = (p.max_q_len * p.group + kRows - 1) / kRows;
    const long long units = (long long)p.batch * (p.nhead / p.group) * row_tiles;
    if (units * kMaxCluster > 0x7fffffff) return fail(ET_ERR_INVALID, "et_attention_tree: too large");
    int* err = nullptr;
    const int rc = attn_err_address(&err);
    if (rc) return rc;
    return cuda_status((p.head_dim <= 64 ? launch<64> : launch<128>)(p, row_tiles, units, csize, err, st), "et_attention_tree launch");
}

}  // namespace et
