// Host-side launchers of the kernels for drafted tokens over a cache in int8.
#pragma once
#include <cuda_runtime.h>
#include "attention_tree.cuh"

namespace et {

// How CTAs share a sequence's keys, and what a launch takes in microseconds by a model fitted to 6500 launches (1 to 64 sequences of 200 to 16000 keys, 1 to 256 rows of a K/V head, heads
// of 64, 96 and 128, every cluster): the kernel and the cluster taken so cost 4.5 % over the fastest in the mean (with rules of thumb, tcgen05 from 32 rows on and clusters that fill the SMs, it
// was 26 %).
struct TreePlan {
    double us;
    int csize;
};
TreePlan attention_tree_plan(const TreeParams& p);
int attention_tree_launch(const TreeParams& p, int csize, cudaStream_t st);
// tcgen05 kernel for many rows (attention_tree_tc.cu), heads of up to 128.
TreePlan attention_tree_tc_plan(const TreeParams& p);
int attention_tree_tc_launch(const TreeParams& p, int csize, cudaStream_t st);

// units: clusters; blocks: of a sequence's keys, those of a CTA's share taking `alone` each, or `shared` where all places are taken; start: of a CTA; places: CTAs that run at once, by log2 of the
// cluster's size.
inline TreePlan tree_plan(long long units, int blocks, int per_turn, int max_log, int sms, double alone, double shared, double start, double fixed, double per_doubling, const double (&places)[5]) {
    TreePlan best = {1e30, 1};
    for (int log = 0; log <= max_log; ++log) {
        const int csize = 1 << log;
        if (log > 0 && (csize * per_turn >= 2 * blocks || (log == 4 && units * csize > sms))) break;   // (clusters of 16 find few places)
        const double turns = (blocks + csize * per_turn - 1) / (csize * per_turn), load = units * csize / places[log];
        double us = turns * alone + start;
        if (load > 1.0) {
            const double whole = (double)(long long)(load + 0.999999), many = 0.5 * (whole + load) * (turns * shared + start);
            if (many > us) us = many;
        }
        us += fixed + per_doubling * log;
        if (us < best.us) best = {us, csize};
    }
    return best;
}

}  // namespace et
