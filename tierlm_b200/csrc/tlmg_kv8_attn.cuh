// tlmg_kv8_attn.cuh - arguments of the 8-bit cache's attention kernels.
#pragma once
#include <algorithm>
#include <new>
#include <utility>
#include <vector>

#include "tlmg_kv8.cuh"

namespace tlmg {

struct Kv8Attn {
    Kv8View c;
    tlmg_kv8_batch b;
    int H, G;
    uint32_t inv_g;   // ceil(2^32 / G); 0 for G = 1
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
    int rt0;          // few query rows: the launch's first query tile
    // spans: partial outputs, maxima (log2 units) and sums [row][n_split], scores [row][s_stride]
    int n_split, tiles;
    float *po, *pm, *pl, *scores, *lse2;
    int64_t s_stride;
    // many query rows: the cache as the caller gave it; tile images of the sequences from s0 and the nkv KV heads from kv0,
    // n_img tiles for each pair, and what an image's code is worth
    tlmg_kv8 kv8;
    uint8_t *img, *heads;
    int s0, kv0, nkv, n_img;
    float unit;
    // its items: query tiles of a sequence and head; the items from n_full on go in pieces
    int q_tiles, n_full, pieces;
};

// tanh(x) = x (c0 + c1 x^2 + .. + c5 x^10) for |x| < TANH_X within 2e-7: fitted (reweighted least squares towards the
// smallest maximum) to tanh(x) / x over x^2 in [0, TANH_X^2]. Two issue slots and a half an element; the exponential
// form takes two of the slower special-function results.
constexpr float TANH_X = 0.8f;
__device__ constexpr float TANH_C[6] = { 0.9999999403953552f, -0.33332714438438416f, 0.13321532309055328f, -0.05313541740179062f, 0.019130872562527657f, -0.004378729499876499f };

__device__ __forceinline__ float kv8_tanh_small(float x) {
    const float y = x * x;
    float r = TANH_C[5];
#pragma unroll
    for (int k = 4; k >= 0; k--) r = __fmaf_rn(r, y, TANH_C[k]);
    return r * x;
}
__device__ __forceinline__ float kv8_ex2(float x) {   // 2^x, results below 2^-126 as 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The key tiles of TILE rows that a tile of queries at positions pmin ..
// pmax may see. Rows are positions when the cache has no position pool: then
// they are the rows below the prefix and those from the window's begin to
// the last query's position.
template <int TILE> struct Kv8Range {
    int nA, loB, n;   // tiles of the first part, first row of the second, tiles in all
    __device__ __forceinline__ int t0(int v) const { return v < nA ? v * TILE : loB + (v - nA) * TILE; }
    __device__ __forceinline__ bool has(int t) const { return t < nA * TILE || (t >= loB && t < loB + (n - nA) * TILE); }
};
template <int TILE>
__device__ __forceinline__ Kv8Range<TILE> kv8_range(const Kv8Attn &a, const Kv8Seq &q, int s, int pmin, int pmax) {
    int lo = 0, hi = q.L, pre = 0;
    if (!a.c.pos && (a.causal || a.window)) {
        pre = a.prefix ? min(max(a.prefix[s], 0), q.L) : 0;
        if (a.causal) hi = pmax >= q.L ? q.L : max(pmax, -1) + 1;
        if (a.window) lo = min(max((int)min((int64_t)pmin - a.window + 1, (int64_t)INT32_MAX), 0), hi);
    }
    Kv8Range<TILE> r;
    r.nA = (pre + TILE - 1) / TILE;
    r.loB = lo / TILE * TILE;
    const int nB = hi > r.loB ? (hi - r.loB + TILE - 1) / TILE : 0;
    if (r.nA * TILE >= r.loB) {      // one part
        r.n = max(r.nA, r.loB / TILE + nB);
        r.nA = r.n;
    } else {
        r.n = r.nA + nB;
    }
    return r;
}

inline int sm_count() {
    thread_local int dev = -1, n = 0;
    int d = 0;
    cudaGetDevice(&d);
    if (d != dev) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, d) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            n = 148;
        }
        dev = d;
    }
    return n;
}

// Lets a kernel take `bytes` of dynamic shared memory; asked for once a thread and device. Nothing leaves a C call as an
// exception: without memory for the note it is asked for again.
inline bool smem_opt_in(const void *fn, size_t bytes) {
    static thread_local std::vector<std::pair<const void *, int>> done;
    int dev = 0;
    cudaGetDevice(&dev);
    for (auto &d : done)
        if (d.first == fn && d.second == dev) return true;
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    try {
        done.push_back({ fn, dev });
    } catch (const std::bad_alloc &) {
    }
    return true;
}

// The form for many query rows (tlmg_kv8_prefill.cu): whether it serves a call, its workspace, and the call.
bool kv8_prefill_serves(const tlmg_kv8 &c, const tlmg_kv8_batch &b, int H);
size_t kv8_prefill_work_bytes(const tlmg_kv8 &c, const tlmg_kv8_batch &b, const tlmg_kv8_score &s, int H, int q_dt);
int kv8_prefill(const Kv8Attn &a, int q_dt, void *work, cudaStream_t st);

}  // namespace tlmg
