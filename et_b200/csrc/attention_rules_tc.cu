// Attention with rules on its scores, on the 5th-generation tensor cores (tcgen05 + TMEM + TMA): whole sequences, heads of a multiple of 16 up to 128.
//
// A work item is 128 queries of one head of one sequence; a block is 64 keys of it. Blocks that no query of the item sees are left out: the
// window and the prefix give two ranges of blocks, documents are looked up in a summary (lowest and highest document of every block) that a small kernel
// makes first. Blocks that all queries see take no mask.
//   S = Q K^T        SS UMMAs 128x64x16, fp32 in 64 TMEM columns; two places, so that the next block's scores are made during this one's softmax
//   softmax          four warps, a thread to a query row with its 64 scores in registers: capped, biased, masked, their maximum, exponentials
//   O += P V         TS UMMAs 128 x head x 16: A = P (fp16) in the place of the scores it came from, B = V as loaded
//   epilogue         O / row sum -> fp16 -> global
// Two CTAs share an SM (256 TMEM columns each), so that one's waits and maxima run under the other's exponentials. Heads of 64 have two places for
// O: an item's rows are written during the next one.
//
// Not a number times the weight 0 is not a number: V rows behind the last key are cleared in shared memory before P V, and a row whose result is not
// finite is computed again from the keys that it sees (rules_row), behind the CTA's last item. So is one whose result, a mean of values near fp16's largest, has left the range by the
// rounding of its weights.
//
// Every mbarrier wait is bounded; a wait that gives up sets the error word that et_attention_check reads and the CTA leaves through the common exit.
#include "attention.h"
#include "attention_rules.h"
#include "common.h"
#include "ptx.cuh"
#include "tmap.h"
#include "vec_math.cuh"

namespace et {

namespace {

constexpr int kBQ = 128, kBK = 64;
constexpr int kSoftmaxWarps = 4;
constexpr int kLoadWarp = 4, kMmaWarp = 5, kHelpWarp = 6, kHelpWarps = 2;
constexpr int kThreads = 256;
constexpr int kCtasPerSm = 2;
constexpr int kTmemCols = 256;
constexpr float kRescaleStep = 8.f;       // log2 units by which a row's maximum must grow before O is rescaled
constexpr int kItemRing = 4, kBlockRing = 8;
constexpr int kMaxSorted = 128;           // sequences of a ragged batch that a CTA keeps in order of length
constexpr int kLenClasses = 9;
constexpr int kShiftPitch = 800;          // bytes of one of four copies of a block's biases (fp32, log2 domain), each shifted by one more: 196 values and some against conflicts
constexpr int kShiftBytes = 4 * kShiftPitch;

enum Bias { kNoBias = 0, kSlopes = 1, kTable = 2 };
enum Cap { kNoCap = 0, kCapped = 1, kWide = 2 };   // kWide: above kWideCap
enum BlockFlags { kPartial = 1, kFirst = 2, kLast = 4, kEnd = 8, kMixed = 16 };   // kPartial: by place, kMixed: by document

struct TcRules {
    RuleParams r;
    const int2* summary;      // documents: document_summary_kernel's, [batch][summary_blocks]; null without documents
    int summary_blocks;
    bool take_over;           // CTAs ask for items that have not started
    bool sorted;              // a ragged batch of at most kMaxSorted sequences, the longest first
    bool heavy_first;         // equal lengths: late queries, which see more, first
    int* err;
};

struct Item {
    RuleSeq seq;
    int b, qi0, head;
    int state;                // -1: no more items, 0: no query sees a key, 1: blocks follow
};
struct alignas(16) Block {
    int j, left, flags, item; // number of the block, keys from its first one on, what it is, slot of its item
};

template <int kHD>
struct Cfg {
    static constexpr int kPanels = kHD / 64;                // of 64 features: rows of 128 bytes
    static constexpr int kQPanel = kBQ * 128, kKPanel = kBK * 128;
    static constexpr int kQTile = kPanels * kQPanel, kKTile = kPanels * kKPanel;
    static constexpr int kQStages = kHD == 64 ? 2 : 1;
    static constexpr int kStages = kHD == 64 ? 4 : 2;       // of K and V each
    static constexpr int kOPlaces = kHD == 64 ? 2 : 1;
    static constexpr uint32_t kSCol = 0, kOCol = 2 * kBK;   // S, 64 columns twice; O
    static constexpr int kKAt = kQStages * kQTile, kVAt = kKAt + kStages * kKTile, kHelpAt = kVAt + kStages * kKTile;
};

// Rows of an item that a softmax warp computes again once it has no more items: nobody may wait for that (some 14 us a key for 32 rows).
struct Again {
    int b, qi0, head;
    unsigned rows;
};
// A CTA takes no more items while one of these lists has no room for those that may be on their way when the loading warp looks: one in each slot, its own
// and the next. (What is not taken starts as a CTA of its own.)
constexpr int kMaxAgain = 16;
static_assert(kMaxAgain >= kItemRing + 3, "a CTA's first items have room");
struct TcShared {
    uint4 clc;
    uint64_t clc_full;
    uint64_t q_full[2], q_empty[2], k_full[4], k_empty[4], v_full[4], v_empty[4];
    uint64_t s_full[2], p_full[2], pv_done[2];   // by place of the scores
    uint64_t m_full[2], m_empty[2];       // what the helping warps bring of a block: documents of its keys, its biases
    uint64_t item_full[kItemRing], item_empty[kItemRing];
    uint64_t block_full[kBlockRing];
    Item item[kItemRing];
    Block block[kBlockRing];
    alignas(16) int docs[2][kBK];         // read four at a time
    uint32_t tmem_base;
    int n_again[kSoftmaxWarps], no_more;
    alignas(16) Again again[kSoftmaxWarps][kMaxAgain];
};
struct SeqTable {
    RuleSeq seq[kMaxSorted];
    int b[kMaxSorted];
    int before[kMaxSorted + 1];
    int class_at[kLenClasses + 1];
};

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// c - 2 c / (1 + 2^(x cap_in)) of four scores, with one reciprocal for the four: of the product of the denominators, which are at most 2^25 + 1 (from there
// on the result is c).
__device__ __forceinline__ void cap4(float& a, float& b, float& c, float& d, float cap_in, float cap_out) {
    const float2 in2 = make_float2(cap_in, cap_in), one2 = make_float2(1.f, 1.f);
    float2 x = mul2(make_float2(a, b), in2), y = mul2(make_float2(c, d), in2);
    x.x = ex2_fast(min_nan(x.x, 25.f));
    x.y = ex2_fast(min_nan(x.y, 25.f));
    y.x = ex2_fast(min_nan(y.x, 25.f));
    y.y = ex2_fast(min_nan(y.y, 25.f));
    x = add2(x, one2);
    y = add2(y, one2);
    const float2 xy = mul2(x, y);
    const float r = rcp_fast(xy.x * xy.y);
    const float2 inv = make_float2(r * xy.y, r * xy.x);   // 1 / (x y), each
    const float2 out2 = make_float2(cap_out, cap_out), n2 = make_float2(-2.f * cap_out, -2.f * cap_out);
    const float2 ab = fma2(mul2(inv, y), n2, out2), cd = fma2(mul2(inv, x), n2, out2);
    a = ab.x; b = ab.y; c = cd.x; d = cd.y;
}
// Bits i >= from of a word (from: any whole number).
__device__ __forceinline__ uint32_t bits_from(int from) { return from <= 0 ? ~0u : from >= 32 ? 0u : ~0u << from; }

__device__ __forceinline__ void clc_ask(uint4* answer, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool clc_answer(const uint4* answer, int& x) {
    uint32_t ok, cx;
    asm volatile(
        "{\n.reg .b128 h;\n.reg .pred p;\nld.shared.b128 h, [%2];\n"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\nselp.u32 %0, 1, 0, p;\nmov.u32 %1, 0;\n"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n}"
        : "=r"(ok), "=r"(cx)
        : "r"(smem_u32(answer))
        : "memory");
    x = (int)cx;
    return ok != 0;
}

// A ragged batch in order of its sequences' key blocks, the most first (whole warp), so that what is left when CTAs run out of items are short
// ones, and an item is found without reading memory.
__device__ __forceinline__ void sort_sequences(const RuleParams& p, SeqTable* t, int lane) {
    if (lane <= kLenClasses) t->class_at[lane] = 0;
    RuleSeq mine[kMaxSorted / 32];   // read at once, kept for both passes
#pragma unroll
    for (int n = 0; n < kMaxSorted / 32; ++n) {
        mine[n] = RuleSeq{};
        if (n * 32 + lane < p.batch) mine[n] = rule_seq(p, n * 32 + lane);
    }
    __syncwarp();
    const unsigned below = (1u << lane) - 1u;
    for (int pass = 0; pass < 2; ++pass) {   // count, place
#pragma unroll
        for (int n = 0; n < kMaxSorted / 32; ++n) {
            if (n * 32 >= p.batch) break;
            const int i = n * 32 + lane;
            const bool in = i < p.batch;
            const int c = in ? 8 - min((mine[n].klen + 127) / 128, 8) : kLenClasses;   // by 128 keys
            const unsigned same = __match_any_sync(0xffffffffu, c);
            const int at = t->class_at[c];
            __syncwarp();
            if ((same & below) == 0) t->class_at[c] = at + __popc(same);
            __syncwarp();
            if (pass == 1 && in) {
                const int pos = at + __popc(same & below);
                t->seq[pos] = mine[n];
                t->b[pos] = i;
            }
        }
        __syncwarp();
        if (pass == 0) {   // counts -> where each class starts
            const int n = lane < kLenClasses ? t->class_at[lane] : 0;
            int incl = n;
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            __syncwarp();
            if (lane < kLenClasses) t->class_at[lane] = incl - n;
            __syncwarp();
        }
    }
    int before = 0;
    for (int base = 0; base < p.batch; base += 32) {
        const int i = base + lane;
        int incl = i < p.batch ? (t->seq[i].qlen + kBQ - 1) / kBQ : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (i < p.batch) t->before[i + 1] = before + incl;
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) t->before[0] = 0;
    __syncwarp();
}

// The rows of a list, computed again (whole warp).
static __device__ __noinline__ void rows_again(const RuleParams& r, const Again* list, int n) {
    for (int i = 0; i < n; ++i) {
        const Again a = list[i];
        const RuleSeq s = rule_seq(r, a.b);
        for (unsigned left = a.rows; left; left &= left - 1) rules_row(r, s, a.qi0 + __ffs(left) - 1, a.head);
    }
}

// Which queries block `blk` is (whole warp); false: it lies beyond the batch (the grid of a ragged batch has slack).
__device__ __forceinline__ bool find_item(const TcRules& p, const SeqTable* t, int blk, int lane, Item& it) {
    const RuleParams& r = p.r;
    if (p.sorted) {
        for (int base = 0; base < r.batch; base += 32) {
            const unsigned hit = __ballot_sync(0xffffffffu, base + lane < r.batch && blk < t->before[min(base + lane, kMaxSorted - 1) + 1]);
            if (!hit) continue;
            const int pos = base + __ffs(hit) - 1;
            it.seq = t->seq[pos];
            it.b = t->b[pos];
            it.qi0 = (t->before[pos + 1] - 1 - blk) * kBQ;   // late queries first
            return true;
        }
        return false;
    } else if (r.cu_seqlens) {
        for (int base = 0; base < r.batch; base += 32) {
            const int i = base + lane;
            RuleSeq s = {};
            if (i < r.batch) s = rule_seq(r, i);
            const int n = (s.qlen + kBQ - 1) / kBQ;
            int incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, blk < incl);
            if (hit) {
                const int src = __ffs(hit) - 1;
                it.b = base + src;
                it.qi0 = (__shfl_sync(0xffffffffu, incl, src) - 1 - blk) * kBQ;
                it.seq.q0 = __shfl_sync(0xffffffffu, s.q0, src);
                it.seq.qlen = __shfl_sync(0xffffffffu, s.qlen, src);
                it.seq.k0 = __shfl_sync(0xffffffffu, s.k0, src);
                it.seq.klen = __shfl_sync(0xffffffffu, s.klen, src);
                it.seq.qpos0 = __shfl_sync(0xffffffffu, s.qpos0, src);
                it.seq.prefix = __shfl_sync(0xffffffffu, s.prefix, src);
                return true;
            }
            blk -= __shfl_sync(0xffffffffu, incl, 31);
        }
        return false;
    } else {
        const int nb = (r.max_q_len + kBQ - 1) / kBQ;
        if (blk >= nb * r.batch) return false;
        it.b = p.heavy_first ? blk % r.batch : blk / nb;
        it.qi0 = (p.heavy_first ? nb - 1 - blk / r.batch : blk % nb) * kBQ;
        it.seq = rule_seq(r, it.b);
        return true;
    }
}

// The blocks of keys that an item's queries see (whole warp): the prefix's blocks, then the window's; of documents those whose range meets the queries'. With slopes
// from the queries on to the end, then from the queries back to the beginning: so the largest scores tend to come first, while in order every block before the
// queries raises the maximum and O is rescaled. (4 x 4096 tokens, 16 heads of 64: 599 us in order, 507 so.)
struct Blocks {
    const int2* summary;
    int n_prefix, first, n;        // blocks of the prefix, the window's first block behind them, all of them
    int turn;                      // how many lie before the queries and come last, in reverse
    int at;                        // the next one to look at; documents: behind the 32 looked at
    unsigned seen, whole;          // documents: of the 32 looked at, those to come, and those of one document with all queries
    int d_lo, d_hi;                // lowest and highest of the queries
    bool d_odd;                    // some query is of none

    __device__ __forceinline__ int number(int i) const {
        i = i < n - turn ? i + turn : n - 1 - i;
        return i < n_prefix ? i : first + i - n_prefix;
    }
    __device__ __forceinline__ void start(const TcRules& p, const Item& it, int lane) {
        const RuleParams& r = p.r;
        const RuleSeq& s = it.seq;
        const int qa = s.qpos0 + it.qi0, qb = s.qpos0 + min(it.qi0 + kBQ, s.qlen) - 1;
        const int pre = max(0, min(s.prefix, s.klen));
        n_prefix = (pre + kBK - 1) / kBK;
        const int lo = r.window_left == kNoLimit ? 0 : max(qa - r.window_left, 0);
        const int hi = r.window_right == kNoLimit ? s.klen - 1 : min(qb + r.window_right, s.klen - 1);
        first = max(lo / kBK, n_prefix);
        n = n_prefix + (hi >= lo ? max(hi / kBK - first + 1, 0) : 0);
        turn = 0;
        if (r.slopes) {
            const int j = max(qa, 0) / kBK;   // the first query's block
            turn = min(j < n_prefix ? j : n_prefix + max(j - first, 0), n);
        }
        at = 0;
        if (p.summary) {
            int lowest = 0x7fffffff, highest = -1;
            bool none = false;
#pragma unroll
            for (int i = 0; i < kBQ / 32; ++i) {
                const int q = it.qi0 + i * 32 + lane;
                if (q < s.qlen) {
                    const int d = r.q_docs[s.q0 + q];
                    if (d >= 0) lowest = min(lowest, d);
                    highest = max(highest, d);
                    none = none || d < 0;
                }
            }
            d_lo = __reduce_min_sync(0xffffffffu, lowest);
            d_hi = __reduce_max_sync(0xffffffffu, highest);
            d_odd = __any_sync(0xffffffffu, none);
            summary = p.summary + (size_t)it.b * p.summary_blocks;
            seen = whole = 0;
        }
    }
    // Number of the next block, -1: no more; what: kPartial, kMixed
    __device__ __forceinline__ int next(const TcRules& p, const Item& it, int lane, int& what) {
        int i;
        what = 0;
        if (p.summary) {
            while (!seen) {
                if (at >= n) return -1;
                const int mine = at + lane;
                bool meets = false, same = false;
                if (mine < n) {
                    const int2 d = summary[number(mine)];
                    meets = d.y >= d_lo && (d.x & 0x7fffffff) <= d_hi;   // (without a document on one side never)
                    same = d.x == d.y && d_lo == d_hi && d.x == d_lo && !d_odd;
                }
                seen = __ballot_sync(0xffffffffu, meets);
                whole = __ballot_sync(0xffffffffu, same);
                at += 32;
            }
            const int bit = __ffs(seen) - 1;
            i = at - 32 + bit;
            if (!((whole >> bit) & 1u)) what = kMixed;
            seen &= seen - 1;
        } else {
            if (at >= n) return -1;
            i = at++;
        }
        const int j = number(i);
        const RuleParams& r = p.r;
        const RuleSeq& s = it.seq;
        const int qa = s.qpos0 + it.qi0, qb = s.qpos0 + min(it.qi0 + kBQ, s.qlen) - 1;
        const int ka = j * kBK, kb = ka + kBK - 1;
        const bool inside = (r.window_left == kNoLimit || ka >= qb - r.window_left) && (r.window_right == kNoLimit || kb <= qa + r.window_right);
        if (!(kb < s.klen && (inside || kb < s.prefix))) what |= kPartial;
        return j;
    }
};

template <int kHD, int kBias, int kCap>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) attention_rules_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                                                                                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TcRules p) {
    using C = Cfg<kHD>;
    const bool docs = p.summary != nullptr, help = kBias == kTable || docs;
    constexpr bool kChanged = kCap != kNoCap || kBias != kNoBias;   // scores are in the log2 domain before the maximum is taken
    const RuleParams& r = p.r;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* const sBias = smem + C::kHelpAt;
    TcShared* const sh = reinterpret_cast<TcShared*>(smem + C::kHelpAt + (kBias == kTable ? 2 * kShiftBytes : 0));
    SeqTable* const table = reinterpret_cast<SeqTable*>(sh + 1);   // p.sorted
    const uint32_t smem_at = smem_u32(smem), sh_at = smem_u32(sh);
    // Barriers by their 32-bit addresses: through a pointer that was rounded up a wait costs several times as much.
    auto bar = [&](size_t member, uint32_t i = 0) { return sh_at + (uint32_t)member + i * 8; };
#define ET_BAR(name, ...) bar(offsetof(TcShared, name), ##__VA_ARGS__)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int hd = r.head_dim, osteps = hd >> 4;

    if (warp == kLoadWarp) {
        if (lane == 0) {
            for (int i = 0; i < kSoftmaxWarps; ++i) sh->n_again[i] = 0;
            sh->no_more = 0;
            mbar_init(&sh->clc_full, 1);
            for (int i = 0; i < 2; ++i) {
                mbar_init(&sh->q_full[i], 1); mbar_init(&sh->q_empty[i], 1);
                mbar_init(&sh->s_full[i], 1);
                mbar_init(&sh->p_full[i], kSoftmaxWarps);
                mbar_init(&sh->pv_done[i], 1);
                mbar_init(&sh->m_full[i], 32 * kHelpWarps);
                mbar_init(&sh->m_empty[i], kSoftmaxWarps);
            }
            for (int i = 0; i < C::kStages; ++i) {
                mbar_init(&sh->k_full[i], 1); mbar_init(&sh->k_empty[i], 1);
                mbar_init(&sh->v_full[i], 1); mbar_init(&sh->v_empty[i], 1);
            }
            for (int i = 0; i < kItemRing; ++i) {
                mbar_init(&sh->item_full[i], 1);
                mbar_init(&sh->item_empty[i], kSoftmaxWarps);
            }
            for (int i = 0; i < kBlockRing; ++i) mbar_init(&sh->block_full[i], 1);
            fence_mbar_init();
            prefetch_tmap(&tmQ);
            prefetch_tmap(&tmK);
            prefetch_tmap(&tmV);
        }
    } else if (warp == kMmaWarp) {
        tmem_alloc(&sh->tmem_base, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();   // (behind the allocation: columns that a dependent CTA takes first it keeps until this kernel has ended)
    const uint32_t tmem = sh->tmem_base;

    if (warp == kLoadWarp) {
        // ---- items, their blocks and the loads (all lanes stay together; lane 0 issues)
        pdl_wait();
        if (p.sorted) sort_sequences(r, table, lane);
        int id = blockIdx.x;
        int ni = 0, nq = 0, nk = 0, nv = 0, g = 0;   // items handed out, tiles requested, blocks announced
        uint32_t clc_phase = 0;
        bool ok = true;
        auto load = [&](int at, int panel, int stages, const CUtensorMap* tm, int head, int row, size_t full, size_t empty, int& count) {
            const int st = count % stages;
            if (!mbar_wait_at(bar(empty, st), ((uint32_t)(count / stages) & 1u) ^ 1u)) return false;
            if (lane == 0) {
                mbar_expect_tx_at(bar(full, st), C::kPanels * panel);
#pragma unroll
                for (int c = 0; c < C::kPanels; ++c) tma_load_3d_at(smem_at + at + (st * C::kPanels + c) * panel, tm, c * 64, head, row, bar(full, st));
            }
            ++count;
            return true;
        };
        auto load_q = [&](int head, int row) { return load(0, C::kQPanel, C::kQStages, &tmQ, head, row, offsetof(TcShared, q_full), offsetof(TcShared, q_empty), nq); };
        auto load_k = [&](int head, int row) { return load(C::kKAt, C::kKPanel, C::kStages, &tmK, head, row, offsetof(TcShared, k_full), offsetof(TcShared, k_empty), nk); };
        auto load_v = [&](int head, int row) { return load(C::kVAt, C::kKPanel, C::kStages, &tmV, head, row, offsetof(TcShared, v_full), offsetof(TcShared, v_empty), nv); };
        // A block's entry may be overwritten kBlockRing blocks later: V of the block before that has then been requested, in a place that P V has
        // left kStages blocks before, and before P V of a block everyone has passed it.
        static_assert(C::kStages + 1 <= kBlockRing, "entries stay until everyone has read them");
        auto announce = [&](int j, int left, int flags, int slot) {
            if (lane == 0) {
                Block& b = sh->block[g % kBlockRing];
                b.j = j; b.left = left; b.flags = flags; b.item = slot;
                mbar_arrive_at(ET_BAR(block_full, g % kBlockRing));
            }
            __syncwarp();
            ++g;
        };
        for (;;) {
            const bool take_over = p.take_over && !__any_sync(0xffffffffu, *const_cast<volatile int*>(&sh->no_more));
            if (lane == 0 && take_over) {
                mbar_expect_tx(&sh->clc_full, 16);
                clc_ask(&sh->clc, &sh->clc_full);
            }
            Item it = {};
            it.head = id % r.nhead;
            if (find_item(p, table, id / r.nhead, lane, it)) {
                Blocks blocks;
                blocks.start(p, it, lane);
                int what = 0, what_next = 0;
                int j = blocks.next(p, it, lane, what);
                it.state = j >= 0 ? 1 : 0;
                const int slot = ni % kItemRing;
                if ((ok = mbar_wait_at(ET_BAR(item_empty, slot), ((uint32_t)(ni / kItemRing) & 1u) ^ 1u))) {
                    if (lane == 0) {
                        sh->item[slot] = it;
                        mbar_arrive_at(ET_BAR(item_full, slot));
                    }
                    __syncwarp();
                    ++ni;
                    const int kv_head = it.head / r.group;
                    if (j >= 0) ok = load_q(it.head, it.seq.q0 + it.qi0) && load_k(kv_head, it.seq.k0 + j * kBK);
                    int flags = kFirst;
                    while (ok && j >= 0) {   // K of the next block ahead of V of this one
                        const int jn = blocks.next(p, it, lane, what_next);
                        announce(j, it.seq.klen - j * kBK, flags | what | (jn < 0 ? kLast : 0), slot);
                        if (jn >= 0) ok = load_k(kv_head, it.seq.k0 + jn * kBK);
                        if (ok) ok = load_v(kv_head, it.seq.k0 + j * kBK);
                        j = jn;
                        what = what_next;
                        flags = 0;
                    }
                }
            }
            if (!take_over) break;
            // the answer is awaited even on the way out: nothing may be in flight towards shared memory when the CTA leaves
            const bool answered = mbar_wait(&sh->clc_full, clc_phase);
            clc_phase ^= 1u;
            ok = ok && answered;
            if (!ok) break;
            const bool more = clc_answer(&sh->clc, id);
            fence_proxy_async_smem();   // the answer has been read before the next one may be written
            __syncwarp();
            if (!more) break;
        }
        if (ok) {
            const int slot = ni % kItemRing;
            ok = mbar_wait_at(ET_BAR(item_empty, slot), ((uint32_t)(ni / kItemRing) & 1u) ^ 1u);
            if (ok) {
                if (lane == 0) {
                    sh->item[slot].state = -1;
                    mbar_arrive_at(ET_BAR(item_full, slot));
                }
                announce(0, 0, kEnd, slot);
            }
        }
        if (!ok) {
            if (lane == 0) atomicExch(p.err, 21);
            // copies still in flight land before the CTA leaves (bounded)
            for (int i = max(nq - C::kQStages, 0); i < nq; ++i) mbar_wait_at(ET_BAR(q_full, i % C::kQStages), (uint32_t)(i / C::kQStages) & 1u);
            for (int i = max(nk - C::kStages, 0); i < nk; ++i) mbar_wait_at(ET_BAR(k_full, i % C::kStages), (uint32_t)(i / C::kStages) & 1u);
            for (int i = max(nv - C::kStages, 0); i < nv; ++i) mbar_wait_at(ET_BAR(v_full, i % C::kStages), (uint32_t)(i / C::kStages) & 1u);
        }
        __syncwarp();
    } else if (warp == kMmaWarp) {
        // ---- UMMAs: one elected lane does everything, by 32-bit addresses. Blocks are numbered through across items. (As a converged warp that elects a lane for
        // each batch, with descriptors made in the loop, this role took 1900 clocks a block and bounded the kernel: heads of 64, 4 x 4096 tokens 451 us.)
        if (elect_one()) {
            const int steps = hd >> 4;
            const uint32_t idesc_qk = make_idesc_f16(128, kBK), idesc_pv = make_idesc_f16(128, hd, false, true);
            const uint64_t q_desc = make_smem_desc(smem_at, 16, 1024, 2), k_desc = make_smem_desc(smem_at + C::kKAt, 16, 1024, 2);
            const uint64_t v_desc = make_smem_desc(smem_at + C::kVAt, C::kKPanel, 1024, 2);
            int qs = C::kQStages - 1, q_phase = 1;    // of the current item's Q
            int place = 0;                            // of the current item's O
            uint32_t g = 0;
            int left = 0, flags = 0, next_left = 0, next_flags = 0;   // of the block in work, and of the one behind it
            auto entry = [&](uint32_t n) {
                if (!mbar_wait_at(ET_BAR(block_full, n % kBlockRing), (n / kBlockRing) & 1u)) return false;
                next_left = sh->block[n % kBlockRing].left;
                next_flags = sh->block[n % kBlockRing].flags;
                return true;
            };
            // S = Q K_n^T of the block whose entry has been read last; its place holds P of block n - 2 until P V of that is over
            auto qk = [&](uint32_t n) {
                if (next_flags & kFirst) {
                    qs = qs + 1 == C::kQStages ? 0 : qs + 1;
                    if (qs == 0) q_phase ^= 1;
                    if (!mbar_wait_at(ET_BAR(q_full, qs), q_phase)) return false;
                }
                const uint32_t ks0 = n % C::kStages;
                if (!mbar_wait_at(ET_BAR(k_full, ks0), (n / C::kStages) & 1u)) return false;
                if (n >= 2 && !mbar_wait_at(ET_BAR(pv_done, n & 1), ((n - 2) >> 1) & 1u)) return false;
                tc_fence_after();
                const uint64_t a = q_desc + qs * (C::kQTile >> 4), b = k_desc + ks0 * (C::kKTile >> 4);
                const uint32_t to = tmem + C::kSCol + (n & 1) * kBK;
#pragma unroll
                for (int ks = 0; ks < kHD / 16; ++ks)
                    if (ks < steps)
                        umma_f16(to, a + ((ks >> 2) * C::kQPanel + (ks & 3) * 32) / 16, b + ((ks >> 2) * C::kKPanel + (ks & 3) * 32) / 16, idesc_qk, ks > 0);
                umma_commit_at(ET_BAR(s_full, n & 1));
                umma_commit_at(ET_BAR(k_empty, ks0));
                if (next_flags & kLast) umma_commit_at(ET_BAR(q_empty, qs));
                return true;
            };
            bool ok = entry(0) && ((next_flags & kEnd) || qk(0));
            while (ok && !(next_flags & kEnd)) {
                left = next_left;
                flags = next_flags;
                if (C::kOPlaces > 1 && (flags & kFirst)) place ^= 1;
                // The next block's scores ahead of this one's P V; of the next item only where its Q has a place of its own (else it has just been requested) and where it is
                // known already: behind an item's last block may come so many without a key that the loading warp waits for this P V, which lets go of the item's slot.
                const bool ahead = !(flags & kLast) || (C::kQStages > 1 && mbar_test(ET_BAR(block_full, (g + 1) % kBlockRing), ((g + 1) / kBlockRing) & 1u));
                if (ahead && !(ok = entry(g + 1) && ((next_flags & kEnd) || qk(g + 1)))) break;
                // O += P V of block g
                const uint32_t vs = g % C::kStages;
                const int keys = min(left, kBK);
                ok = mbar_wait_at(ET_BAR(v_full, vs), (g / C::kStages) & 1u) && mbar_wait_at(ET_BAR(p_full, g & 1), (g >> 1) & 1u);
                if (!ok) break;
                tc_fence_after();
                const uint64_t b = v_desc + vs * (C::kKTile >> 4);
                const uint32_t a = tmem + C::kSCol + (g & 1) * kBK, to = tmem + C::kOCol + place * 64;
#pragma unroll
                for (int ks = 0; ks < kBK / 16; ++ks)   // P of keys 16ks .. 16ks + 15: 8 packed columns; V: panels of 64 features
                    if (ks * 16 < keys) umma_f16_ts(to, a + ks * 8, b + ks * (2048 / 16), idesc_pv, (!(flags & kFirst) || ks > 0) ? 1u : 0u);
                umma_commit_at(ET_BAR(pv_done, g & 1));
                umma_commit_at(ET_BAR(v_empty, vs));
                if (!ahead) ok = entry(g + 1) && ((next_flags & kEnd) || qk(g + 1));
                ++g;
            }
            if (!ok) atomicExch(p.err, 21);
        }
        __syncwarp();
    } else if (warp >= kHelpWarp) {
        // ---- what a block needs beside K and V: the documents of its keys, its biases by distance
        if (help) {
            pdl_wait();
            const int t = tid - 32 * kHelpWarp;
            bool ok = true;
            for (uint32_t g = 0;; ++g) {
                ok = mbar_wait_at(ET_BAR(block_full, g % kBlockRing), (g / kBlockRing) & 1u);
                if (!ok) break;
                const Block b = sh->block[g % kBlockRing];
                if (b.flags & kEnd) break;
                const int m = g & 1;
                ok = mbar_wait_at(ET_BAR(m_empty, m), ((g >> 1) & 1u) ^ 1u);
                if (!ok) break;
                const Item& it = sh->item[b.item];
                if (b.flags & kMixed) sh->docs[m][t] = t < b.left ? max(r.k_docs[it.seq.k0 + b.j * kBK + t], -1) : -1;
                if constexpr (kBias == kTable) {
                    // value n of copy s: the bias of a key n + s - 127 behind the first key's distance to the first query
                    const half* const row = r.table + (size_t)it.head * (2 * r.reach + 1) + r.reach;
                    const int corner = b.j * kBK - (it.seq.qpos0 + it.qi0) - 127;
                    float* const to = reinterpret_cast<float*>(sBias + m * kShiftBytes);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int n = t + 64 * i;
                        if (n >= kShiftPitch / 4) break;
                        const float v = __half2float(row[max(-r.reach, min(r.reach, corner + n))]) * kRulesLog2e;
#pragma unroll
                        for (int s = 0; s < 4; ++s)
                            if (n >= s) to[s * (kShiftPitch / 4) + n - s] = v;
                    }
                }
                mbar_arrive_at(ET_BAR(m_full, m));
            }
            if (!ok && lane == 0) atomicExch(p.err, 23);
        }
        __syncwarp();
    } else {
        // ---- softmax: one thread per query row (TMEM lane)
        pdl_wait();
        const int row = warp * 32 + lane;
        const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
        const bool wide = (r.out_pitch & 15) == 0 && (reinterpret_cast<uintptr_t>(r.out) & 31) == 0;
        uint32_t g = 0;
        int place = 0;          // of the current item's O
        bool ok = true;
        int done_slot = -1;     // item whose P V is on its way and whose rows are still to be written
        float done_sum = 0.f;   // its row sum
        auto arrive = [&](uint32_t at) {
            __syncwarp();
            if (lane == 0) mbar_arrive_at(at);
        };
        // O / row sum -> fp16 -> global, of the item whose last block is n - 1.
        auto finish = [&](uint32_t n, int from) {
            if (!mbar_wait_at(ET_BAR(pv_done, (n - 1) & 1), ((n - 1) >> 1) & 1u)) return false;
            tc_fence_after();
            const Item& it = sh->item[done_slot];
            const float inv = done_sum > 0.f ? 1.f / done_sum : done_sum == 0.f ? 0.f : done_sum;   // (not a number stays so)
            const int qi = it.qi0 + row;
            const bool in = qi < it.seq.qlen;
            half* const orow = r.out + (it.seq.q0 + qi) * r.out_pitch + it.head * hd;
            half2 top = __float2half2_rn(0.f);   // largest result; infinity or not a number if one of them is
            auto sixteen = [&](const uint32_t (&o)[32], int at, int c) {   // columns 16c .. 16c + 15 of the head, o[at] on
                if (c >= osteps) return;
                uint32_t ow[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    ow[i] = pack2(__uint_as_float(o[at + 2 * i]) * inv, __uint_as_float(o[at + 2 * i + 1]) * inv);
                    top = __hmax2_nan(top, __habs2(*reinterpret_cast<const half2*>(&ow[i])));
                }
                if (in) {
                    half* const z = orow + c * 16;
                    if (wide) {
                        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(z), "r"(ow[0]), "r"(ow[1]), "r"(ow[2]), "r"(ow[3]), "r"(ow[4]),
                                     "r"(ow[5]), "r"(ow[6]), "r"(ow[7])
                                     : "memory");
                    } else {
                        *reinterpret_cast<uint4*>(z) = make_uint4(ow[0], ow[1], ow[2], ow[3]);
                        *reinterpret_cast<uint4*>(z + 8) = make_uint4(ow[4], ow[5], ow[6], ow[7]);
                    }
                }
            };
#pragma unroll 1
            for (int c = 0; c < osteps; c += 4) {   // (columns beyond the head are there, whatever they hold)
                uint32_t o[2][32];
                tmem_ld32(tmem + lane_base + C::kOCol + from * 64 + c * 16, o[0]);
                tmem_ld32(tmem + lane_base + C::kOCol + from * 64 + c * 16 + 32, o[1]);
                tmem_ld_wait(o[0], o[1]);
                sixteen(o[0], 0, c);
                sixteen(o[0], 16, c + 1);
                sixteen(o[1], 0, c + 2);
                sixteen(o[1], 16, c + 3);
            }
            const float largest = fmaxf(__low2float(top), __high2float(top)), sum = __low2float(top) + __high2float(top);
            const unsigned again = __ballot_sync(0xffffffffu, in && !(largest <= 65504.f && sum == sum));
            if (again && lane == 0) {
                const int n = sh->n_again[warp]++;
                sh->again[warp][n] = Again{it.b, it.qi0 + warp * 32, it.head, again};
                if (n >= kMaxAgain - kItemRing - 3) sh->no_more = 1;
            }
            arrive(ET_BAR(item_empty, done_slot));
            done_slot = -1;
            return true;
        };
        for (int ni = 0; ok; ++ni) {
            const int slot = ni % kItemRing;
            ok = mbar_wait_at(ET_BAR(item_full, slot), (uint32_t)(ni / kItemRing) & 1u);
            if (!ok) break;
            const Item& it = sh->item[slot];
            const int state = it.state;
            // The rows of the item before are written within this one's first block where O has a second place. (The ring could run out of slots if an item
            // waited behind empty ones.)
            if (done_slot >= 0 && (C::kOPlaces == 1 || state <= 0)) {
                ok = finish(g, place);
                if (!ok) break;
            }
            if (state < 0) break;
            if (state == 0) {   // no query sees a key: zeros
                const int qi = it.qi0 + row;
                if (qi < it.seq.qlen) {
                    uint4* const z = reinterpret_cast<uint4*>(r.out + (it.seq.q0 + qi) * r.out_pitch + it.head * hd);
                    for (int i = 0; i < hd / 8; ++i) z[i] = make_uint4(0u, 0u, 0u, 0u);
                }
                arrive(ET_BAR(item_empty, slot));
                continue;
            }
            if (C::kOPlaces > 1) place ^= 1;
            const uint32_t o_addr = tmem + lane_base + C::kOCol + place * 64;
            const int qpos = it.seq.qpos0 + it.qi0 + row;
            const int prefix = it.seq.prefix;
            int my_doc = 0;
            if (docs) my_doc = it.qi0 + row < it.seq.qlen ? r.q_docs[it.seq.q0 + it.qi0 + row] : -1;
            if (my_doc < 0) my_doc = -2;   // (keys behind the last one, and those of no document, count as -1)
            float slope = 0.f;
            if constexpr (kBias == kSlopes) slope = r.slopes[it.head] * -kRulesLog2e;
            float m_run = -INFINITY;
            float2 l2 = make_float2(0.f, 0.f);
            bool last = false;
            for (; !last; ++g) {
                const uint32_t s_addr = tmem + lane_base + C::kSCol + (g & 1) * kBK;
                ok = mbar_wait_at(ET_BAR(s_full, g & 1), (g >> 1) & 1u);
                if (!ok) break;
                tc_fence_after();
                const uint4 b = lds128(sh_at + (uint32_t)offsetof(TcShared, block) + (g % kBlockRing) * (uint32_t)sizeof(Block));
                const int k0 = (int)b.x * kBK, left = (int)b.y, flags = (int)b.z;
                const bool first = flags & kFirst;
                last = flags & kLast;
                const int m = g & 1;
                float v[2][32];
                tmem_ld32(s_addr, reinterpret_cast<uint32_t(&)[32]>(v[0]));
                tmem_ld32(s_addr + 32, reinterpret_cast<uint32_t(&)[32]>(v[1]));
                tmem_ld_wait(v[0], v[1]);
                if constexpr (kCap != kNoCap) {
                    if (left < kBK) {   // four scores share a reciprocal: what lies behind the last key must not be not a number
#pragma unroll
                        for (int i = 0; i < 64; ++i) v[i >> 5][i & 31] = i < left ? v[i >> 5][i & 31] : 0.f;
                    }
                    // A warp takes the polynomial for a block all of whose scores are within half a cap: a tenth faster where scores are small, but a fifteenth slower where they are
                    // not, for the vote. (4 x 4096 tokens, cap 50, 16 heads of 64, scores of a deviation of 1: 691 us, 754 by cap4 alone; of 8, where no block is that small, 849
                    // and 794. Heads of 128: 747 and 843, 876 and 827.)
                    bool near = false;
                    if constexpr (kBias == kNoBias || kCap == kWide) {   // (where there is a bias the registers are short)
                        float size[2] = {0.f, 0.f};
#pragma unroll
                        for (int i = 0; i < 64; i += 2) size[(i >> 1) & 1] = max3(size[(i >> 1) & 1], fabsf(v[i >> 5][i & 31]), fabsf(v[i >> 5][(i & 31) + 1]));
                        near = __all_sync(0xffffffffu, fmaxf(size[0], size[1]) <= r.cap_near);
                    }
                    if (near) {
#pragma unroll
                        for (int i = 0; i < 64; i += 2) cap_near2(v[i >> 5][i & 31], v[i >> 5][(i & 31) + 1], r.to_y, r.scale_log2);
                    } else if constexpr (kCap == kWide) {
#pragma unroll
                        for (int i = 0; i < 64; i += 2) cap_wide2(v[i >> 5][i & 31], v[i >> 5][(i & 31) + 1], r);
                    } else {
#pragma unroll
                        for (int i = 0; i < 64; i += 4) cap4(v[i >> 5][i & 31], v[i >> 5][(i & 31) + 1], v[i >> 5][(i & 31) + 2], v[i >> 5][(i & 31) + 3], r.cap_in, r.cap_out);
                    }
                }
                const float sc = kCap ? 1.f : r.scale_log2;
                const float2 scale2 = make_float2(sc, sc);
                if constexpr (kBias == kSlopes) {
                    // On one side of the queries the bias is linear in the key; in the blocks around them it is not.
                    const float near = (float)(k0 - qpos);
                    const bool behind = k0 >= qpos, before = k0 + kBK - 1 <= qpos;
                    if (__all_sync(0xffffffffu, behind) || __all_sync(0xffffffffu, before)) {
                        const float s1 = behind ? slope : -slope;
                        const float2 step2 = make_float2(16.f * s1, 16.f * s1);
                        float2 bias[8];   // (chains of sums: as constants in registers the distances cost two moves each)
#pragma unroll
                        for (int i = 0; i < 8; ++i) bias[i] = make_float2((near + 2 * i) * s1, (near + 2 * i + 1) * s1);
#pragma unroll
                        for (int i = 0; i < 64; i += 2) {
                            float2& y = bias[(i >> 1) & 7];
                            float* const w = &v[i >> 5][i & 31];
                            const float2 x = kCap ? add2(make_float2(w[0], w[1]), y) : fma2(make_float2(w[0], w[1]), scale2, y);
                            w[0] = x.x;
                            w[1] = x.y;
                            if (i < 48) y = add2(y, step2);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 64; ++i) v[i >> 5][i & 31] = fmaf(fabsf(near + (float)i), slope, kCap ? v[i >> 5][i & 31] : v[i >> 5][i & 31] * sc);
                    }
                }
                if (help) {
                    ok = mbar_wait_at(ET_BAR(m_full, m), (g >> 1) & 1u);
                    if (!ok) break;
                }
                if constexpr (kBias == kTable) {
                    // the row's first value is number 127 - row: four at a time from the copy in which they start on 16 bytes
                    const int start = 127 - row;
                    const uint32_t biases = smem_u32(sBias) + m * kShiftBytes + (start & 3) * kShiftPitch + (start & ~3) * 4;
#pragma unroll
                    for (int i = 0; i < 64; i += 4) {
                        const uint4 four = lds128(biases + i * 4);
                        float* const x = &v[i >> 5][i & 31];
                        const float2 lo = make_float2(__uint_as_float(four.x), __uint_as_float(four.y)), hi = make_float2(__uint_as_float(four.z), __uint_as_float(four.w));
                        float2 a = make_float2(x[0], x[1]), bb = make_float2(x[2], x[3]);
                        a = kCap ? add2(a, lo) : fma2(a, scale2, lo);
                        bb = kCap ? add2(bb, hi) : fma2(bb, scale2, hi);
                        x[0] = a.x; x[1] = a.y; x[2] = bb.x; x[3] = bb.y;
                    }
                }
                if (flags & kMixed) {
                    const uint32_t ids = sh_at + (uint32_t)offsetof(TcShared, docs) + m * (kBK * 4);
#pragma unroll
                    for (int i = 0; i < 64; i += 4) {
                        const uint4 four = lds128(ids + i * 4);
                        float* const x = &v[i >> 5][i & 31];
                        x[0] = (int)four.x == my_doc ? x[0] : -INFINITY;
                        x[1] = (int)four.y == my_doc ? x[1] : -INFINITY;
                        x[2] = (int)four.z == my_doc ? x[2] : -INFINITY;
                        x[3] = (int)four.w == my_doc ? x[3] : -INFINITY;
                    }
                }
                if (help) arrive(ET_BAR(m_empty, m));
                if (flags & kPartial) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int at = k0 + h * 32;
                        uint32_t w = r.window_left == kNoLimit ? ~0u : bits_from(qpos - r.window_left - at);
                        if (r.window_right != kNoLimit) w &= ~bits_from(qpos + r.window_right + 1 - at);
                        w |= ~bits_from(prefix - at);
                        w &= ~bits_from(left - h * 32);
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[h][i] = (w >> i) & 1u ? v[h][i] : -INFINITY;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; ++i) mx[i & 3] = max3(mx[i & 3], v[i >> 4][2 * (i & 15)], v[i >> 4][2 * (i & 15) + 1]);
                const float to_log2 = kChanged ? 1.f : r.scale_log2;
                const float bmax = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * to_log2;   // the scale is positive
                // The reference point moves only when the row maximum has grown by more than 2^8; the final division by the row sum makes the
                // result independent of it.
                const bool grow = bmax > m_run + kRescaleStep;   // also true for the first finite score of a row
                if (__any_sync(0xffffffffu, grow)) {
                    float alpha = 1.f;
                    if (grow) {
                        alpha = m_run == -INFINITY ? 0.f : ex2_fast(m_run - bmax);
                        m_run = bmax;
                        l2.x *= alpha;
                        l2.y *= alpha;
                    }
                    if (!first) {   // O holds what the blocks before this one gave
                        ok = mbar_wait_at(ET_BAR(pv_done, (g - 1) & 1), ((g - 1) >> 1) & 1u);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < osteps; ++c) {
                            uint32_t o[16];
                            tmem_ld16(o_addr + c * 16, o);
                            tmem_ld_wait(o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_store16(o_addr + c * 16, o);
                        }
                    }
                }
                const float nshift = (m_run == -INFINITY) ? 0.f : -m_run;
                const float2 to_log22 = make_float2(to_log2, to_log2), shift2 = make_float2(nshift, nshift);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float2 e = make_float2(v[h][2 * i], v[h][2 * i + 1]);
                        e = kChanged ? add2(e, shift2) : fma2(e, to_log22, shift2);
                        e.x = ex2_fast(e.x);
                        e.y = ex2_fast(e.y);
                        l2 = add2(l2, e);
                        pk[i] = pack2(e.x, e.y);
                    }
                    tmem_store16(s_addr + h * 16, pk);   // where this block's first scores were: they have all been read
                }
                // V's rows behind the last key, up to the end of a 16-key step, may hold anything: they are cleared
                if (left < kBK && (left & 15)) {
                    const int vs = g % C::kStages, end = (left + 15) & ~15;
                    ok = mbar_wait_at(ET_BAR(v_full, vs), (g / C::kStages) & 1u);
                    if (!ok) break;
                    for (int i = row; i < (end - left) * 8 * C::kPanels; i += kBQ) {
                        const int key = left + i / (8 * C::kPanels), c = i % (8 * C::kPanels);
                        sts128(smem_at + C::kVAt + (vs * C::kPanels + (c >> 3)) * C::kKPanel + key * 128 + (c & 7) * 16, make_uint4(0u, 0u, 0u, 0u));
                    }
                    fence_proxy_async_smem();
                }
                tmem_st_wait();
                tc_fence_before();
                arrive(ET_BAR(p_full, g & 1));
                if (C::kOPlaces > 1 && first && done_slot >= 0) {
                    ok = finish(g, place ^ 1);
                    if (!ok) break;
                }
            }
            if (!ok) break;
            done_slot = slot;
            done_sum = l2.x + l2.y;
        }
        if (!ok && lane == 0) atomicExch(p.err, 22);
        __syncwarp();
        const int n_again = sh->n_again[warp];
        if (n_again) rows_again(r, sh->again[warp], n_again);
    }
#undef ET_BAR
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
}

// Lowest and highest document of every block of keys of every sequence (the lowest with its sign set where some key is of none): a warp to a block.
__global__ void __launch_bounds__(128) document_summary_kernel(const __grid_constant__ RuleParams p, int2* __restrict__ summary, int blocks) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, j = blockIdx.x * 4 + (threadIdx.x >> 5);
    for (int b = blockIdx.y; b < p.batch; b += gridDim.y) {
        const RuleSeq s = rule_seq(p, b);
        if (j * kBK >= s.klen) continue;
        int lo = 0x7fffffff, hi = -1;
        bool none = false;
#pragma unroll
        for (int i = 0; i < kBK / 32; ++i) {
            const int k = j * kBK + i * 32 + lane;
            if (k < s.klen) {
                const int d = p.k_docs[s.k0 + k];
                if (d >= 0) lo = min(lo, d);
                hi = max(hi, d);
                none = none || d < 0;
            }
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (__any_sync(0xffffffffu, none)) lo |= 0x80000000;   // never equal to the highest
        if (lane == 0) summary[(size_t)b * blocks + j] = make_int2(lo, hi);
    }
}

template <int kHD, int kBias, int kCap>
cudaError_t launch(int grid, cudaStream_t st, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const TcRules& p) {
    const auto kernel = attention_rules_tc_kernel<kHD, kBias, kCap>;
    static_assert(Cfg<kHD>::kHelpAt + 2 * kShiftBytes + sizeof(TcShared) + sizeof(SeqTable) + 2048 <= 233472 / kCtasPerSm, "two CTAs to an SM");
    static PerDeviceOnce once;
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448); });
    if (e != cudaSuccess) return e;
    const size_t smem = Cfg<kHD>::kHelpAt + (kBias == kTable ? 2 * kShiftBytes : 0) + sizeof(TcShared) + (p.sorted ? sizeof(SeqTable) : 0) + 1024;
    return launch_pdl(kernel, dim3(grid), dim3(kThreads), smem, st, tq, tk, tv, p);
}
template <int kHD, int kBias>
cudaError_t launch_with(int grid, cudaStream_t st, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const TcRules& p) {
    const auto run = p.r.cap_wide ? launch<kHD, kBias, kWide> : p.r.cap_out > 0.f ? launch<kHD, kBias, kCapped> : launch<kHD, kBias, kNoCap>;
    return run(grid, st, tq, tk, tv, p);
}
template <int kHD>
cudaError_t launch_for(int grid, cudaStream_t st, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const TcRules& p) {
    const auto run = p.r.slopes ? launch_with<kHD, kSlopes> : p.r.table ? launch_with<kHD, kTable> : launch_with<kHD, kNoBias>;
    return run(grid, st, tq, tk, tv, p);
}

}  // namespace

bool attention_rules_tc_takes(const RuleParams& p) {
    return p.head_dim % 16 == 0 && p.head_dim <= 128 && ((p.q_pitch | p.k_pitch | p.v_pitch | p.out_pitch) & 7) == 0 && aligned16(p.q) && aligned16(p.k) &&
           aligned16(p.v) && aligned16(p.out) && p.k_rows > 0 && p.max_k_len > 0 &&
           ((long long)p.q_tokens / kBQ + p.batch) * p.nhead <= 0x7fffffff;
}

int attention_rules_tc_launch(const RuleParams& r, void* scratch, cudaStream_t st) {
    TcRules p;
    p.r = r;
    int rc = attn_err_address(&p.err);
    if (rc) return rc;
    CUtensorMap tq, tk, tv;
    if (!make_tmap_heads_f16(&tq, r.q, r.q_tokens, r.nhead, r.head_dim, r.q_pitch, kBQ) ||
        !make_tmap_heads_f16(&tk, r.k, r.k_rows, r.nhead / r.group, r.head_dim, r.k_pitch, kBK) ||
        !make_tmap_heads_f16(&tv, r.v, r.k_rows, r.nhead / r.group, r.head_dim, r.v_pitch, kBK))
        return fail(ET_ERR_CUDA, "et_attention_rules: cuTensorMapEncodeTiled failed");
    p.summary = static_cast<const int2*>(scratch);
    p.summary_blocks = (r.max_k_len + kBK - 1) / kBK;
    if (scratch) {
        const cudaError_t e = launch_pdl(document_summary_kernel, dim3((p.summary_blocks + 3) / 4, min(r.batch, 0xffff)), dim3(128), 0, st, r, static_cast<int2*>(scratch), p.summary_blocks);
        if (e != cudaSuccess) return cuda_status(e, "et_attention_rules: summary of the documents");
    }
    const int blocks = r.cu_seqlens ? r.q_tokens / kBQ + r.batch : r.batch * ((r.max_q_len + kBQ - 1) / kBQ);
    // CTAs that all fit are left to the hardware: one that starts early would take an item for which a place is still free. (Of a ragged batch only the
    // tokens are known here: at least this many blocks.)
    const long long items = r.cu_seqlens ? (r.q_tokens + kBQ - 1) / kBQ : blocks;
    p.take_over = items * r.nhead > (long long)kCtasPerSm * sm_count();
    p.sorted = p.take_over && r.cu_seqlens && r.batch <= kMaxSorted;
    p.heavy_first = r.window_right != kNoLimit;
    const cudaError_t e = r.head_dim <= 64 ? launch_for<64>(blocks * r.nhead, st, tq, tk, tv, p) : launch_for<128>(blocks * r.nhead, st, tq, tk, tv, p);
    return cuda_status(e, "et_attention_rules launch");
}

}  // namespace et
