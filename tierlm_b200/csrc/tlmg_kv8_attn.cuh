// tlmg_kv8_attn.cuh - arguments of the 8-bit cache's attention kernels.
#pragma once
#include "tlmg_kv8.cuh"

namespace tlmg {

struct Kv8Attn {
    Kv8View c;
    tlmg_kv8_batch b;
    int H, G;
    const void *q;
    int64_t q_stride;
    void *out;
    float *lse;
    float *weights;
    int64_t w_stride;
    float scale, softcap, inv_cap;
    const float *slopes;
    const int32_t *prefix, *doc;
    int doc_stride, causal, window;
    // spans: partial outputs, maxima (log2 units) and sums [row][n_split], scores [row][s_stride]
    int n_split, tiles;
    float *po, *pm, *pl, *scores, *lse2;
    int64_t s_stride;
};

}  // namespace tlmg
