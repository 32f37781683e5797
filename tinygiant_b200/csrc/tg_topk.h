// tg_topk.h — the order in which experts are chosen.
#pragma once
#include <cmath>

#ifdef __CUDACC__
#define TG_HD __host__ __device__ __forceinline__
#else
#define TG_HD inline
#endif

namespace tg {

// How many elements beat element i: those with a larger logit, or an equal one and a larger
// id.  NaN counts as -inf.  That is a total order, so the ranks of E elements are 0 .. E - 1,
// whatever the logits.
TG_HD int topk_rank(const float* logits, int E, int i) {
    const float li = logits[i] == logits[i] ? logits[i] : -INFINITY;
    int rank = 0;
    for (int j = 0; j < E; j++) {
        const float lj = logits[j] == logits[j] ? logits[j] : -INFINITY;
        rank += (lj > li) || (lj == li && j > i);
    }
    return rank;
}

}  // namespace tg
