// Host-side launchers of the kernels for drafted tokens over a cache in int8.
#pragma once
#include <cuda_runtime.h>
#include "attention_tree.cuh"
#include "tmap.h"

namespace et {

// How CTAs share a sequence's keys, and what a launch takes in microseconds by a model fitted to 6200 launches (1 to 128 sequences of 200 to 16000 keys, all alike or ragged, 1 to 256 rows of
// a K/V head, heads of 64, 96 and 128, every cluster): the kernel and the cluster taken so cost 4 % over the fastest in the mean, 23 % at the 95th percentile (with rules of thumb, tcgen05
// from 32 rows on and clusters that fill the SMs, 26 and 100 %).
struct TreePlan {
    double us;
    int csize;
};
TreePlan attention_tree_plan(const TreeParams& p);
int attention_tree_launch(const TreeParams& p, int csize, cudaStream_t st);
// tcgen05 kernel for many rows (attention_tree_tc.cu), heads of up to 128.
TreePlan attention_tree_tc_plan(const TreeParams& p);
int attention_tree_tc_launch(const TreeParams& p, int csize, cudaStream_t st);

// What the model says of one kernel: a turn (a CTA's blocks of keys that its warps take at once) takes `alone` or, where all places are taken, `shared`, and `rows` for what it has of them; a CTA
// starts and ends in `start`, and up to `start_shared` more. places: CTAs that run at once, and the part of them that clusters of 4, 8, 16 find.
struct TreeCosts {
    double alone, shared, start, start_shared, places, part[3], rows;
};
// units: clusters; turns: of a sequence that one CTA has alone.
inline TreePlan tree_plan(long long units, int turns, int sms, const TreeCosts& c) {
    TreePlan best = {1e30, 1};
    for (int log = 0; log <= 4; ++log) {
        const int csize = 1 << log;
        if (log > 0 && (csize >= 2 * turns || (log == 4 && units * csize > sms))) break;   // (clusters of 16 find few places)
        const double n = (turns + csize - 1) / csize, load = units * csize / (c.places * (log < 2 ? 1.0 : c.part[log - 2]));
        auto least = [](double a, double b) { return a < b ? a : b; };
        auto most = [](double a, double b) { return a > b ? a : b; };
        const double start = c.start + c.start_shared * least(load, 1.0), waves = load > 1.0 ? 0.5 * (double)(long long)(load + 0.999999) + 0.5 * load : 1.0;
        // sequences all as long as the longest, and ragged ones, half as long in the mean, the longest first
        const double alike = waves * (n * (most(c.alone, c.shared * least(load, 1.0)) + c.rows) + start);
        const double ragged = most(n * (most(c.alone, c.shared * least(0.92 * load, 1.0)) + c.rows) + start, load * (0.55 * n * (c.shared + c.rows) + start));
        const double us = 0.25 * alike + 0.75 * ragged;
        if (us < 1.02 * best.us) best = {us, csize};   // (as good: the larger cluster, for ragged ones)
    }
    return best;
}

// The cache as [page and side][head][row][feature]; a copy brings 128 features of 16 keys, of K and then of V.
inline bool make_tmap_codes(CUtensorMap* out, const TreeParams& p, bool swizzled) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const uint64_t hd = (uint64_t)p.head_dim, heads = (uint64_t)(p.nhead / p.group);
    cuuint64_t dims[4] = {hd, (cuuint64_t)p.page, heads, 2 * (cuuint64_t)p.pages};
    cuuint64_t strides[3] = {hd, hd * p.page, hd * p.page * heads};
    cuuint32_t box[4] = {128, 16, 1, 2};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<int8_t*>(p.codes), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace et
