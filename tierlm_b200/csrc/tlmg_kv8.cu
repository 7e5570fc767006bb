// tlmg_kv8.cu - the 8-bit KV cache's append, read-back and eviction.
//
// A block (`block` consecutive rows of one head) is stored with one scale
// d = max(amax, 2^-100) * (1 / Q) and codes round(x / d); products and
// divisions are IEEE f32 and the rounding is to nearest even, so that codes are
// a function of the inputs alone. One warp owns one block of K or of V: it takes the maximum
// over the block's rows, then rounds them in a second pass that finds the
// rows in L1. All of these kernels move a few bytes per element. What bounds them
// is the chain of dependent loads or, for one token per sequence, the launch: 8,511
// bf16 rows of 4 heads of 128 in 14 us (26 MB, 1.9 TB/s: the rows of a block come
// twice, the maximum between), read back as f32 in 11 (44 MB, 4.0 TB/s); 64
// one-token sequences 2.7 us, 9 with the call from Python.
#include <algorithm>

#include "tlmg_dev.cuh"
#include "tlmg_internal.h"
#include "tlmg_kv8.cuh"

namespace tlmg {

static int log2i(int v) {
    int l = 0;
    while ((1 << l) < v) l++;
    return l;
}

int kv8_check(const char *who, const tlmg_kv8 *c) {
    if (!c) return set_error(TLMG_EINVAL, "%s: null cache", who);
    if (c->fmt != TLMG_KV8_INT8 && c->fmt != TLMG_KV8_E4M3)
        return set_error(TLMG_EINVAL, "%s: format %d (int8 1 or e4m3 2)", who, c->fmt);
    if (c->hd != 64 && c->hd != 128 && c->hd != 256)
        return set_error(TLMG_EINVAL, "%s: head_dim %d (64, 128 or 256)", who, c->hd);
    if (c->page <= 0 || c->page > (1 << 16) || (c->page & (c->page - 1)) || c->n_pages <= 0 || c->KV <= 0)
        return set_error(TLMG_EINVAL, "%s: page %d (a power of two up to 65536), %d pages, %d KV heads", who, c->page,
                         c->n_pages, c->KV);
    if (c->block <= 0 || c->block > 256 || c->block > c->page || (c->block & (c->block - 1)))
        return set_error(TLMG_EINVAL, "%s: block %d (a power of two, at most the page of %d rows and 256)", who, c->block,
                         c->page);
    if ((int64_t)c->n_pages * c->KV > (int64_t)0xFFFFFFFEu / c->page)
        return set_error(TLMG_ERANGE, "%s: %d pages x %d heads x %d rows pass 2^32 rows", who, c->n_pages, c->KV, c->page);
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return set_error(TLMG_EINVAL, "%s: null pool", who);
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15u)
        return set_error(TLMG_EINVAL, "%s: code pools must be 16-byte aligned", who);
    if (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale | (uintptr_t)c->pos) & 3u)
        return set_error(TLMG_EINVAL, "%s: scale and position pools must be 4-byte aligned", who);
    return TLMG_OK;
}

int kv8_check_batch(const char *who, const tlmg_kv8_batch *b) {
    if (!b || !b->page_table || !b->q_start || !b->kv_len) return set_error(TLMG_EINVAL, "%s: null batch array", who);
    if (b->n_seq <= 0 || b->n_seq > 65535 || b->table_stride <= 0 || b->total_q < 0 || b->max_q < 0 ||
        b->max_kv < 0 || b->max_kv > (1 << 30))
        return set_error(TLMG_EINVAL, "%s: %d sequences (1 .. 65535), table stride %d, %d tokens, max_q %d, max_kv %d", who,
                         b->n_seq, b->table_stride, b->total_q, b->max_q, b->max_kv);
    return TLMG_OK;
}

Kv8View kv8_view(const tlmg_kv8 *c) {
    return Kv8View{ (uint8_t *)c->k, (uint8_t *)c->v, c->k_scale, c->v_scale, c->pos, c->n_pages, c->KV, c->hd,
                    log2i(c->page), log2i(c->block) };
}

namespace {

// amax of |v| that a NaN survives (fmaxf would drop it): +inf and NaN both end as "not finite"
__device__ __forceinline__ float amax4(float a, float4 v) {
    const float m = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
    const bool nan = (v.x != v.x) | (v.y != v.y) | (v.z != v.z) | (v.w != v.w);
    return fmaxf(a, nan ? INFINITY : m);
}
__device__ __forceinline__ float warp_max(float a) {
    for (int o = 16; o; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xFFFFFFFFu, a, o));
    return a;
}
// The scale of a block from its amax; NaN where the block is not finite.
template <int FMT> __device__ __forceinline__ float scale_of(float amax) {
    return amax < INFINITY ? __fmul_rn(fmaxf(amax, KV8_FLOOR), 1.0f / kv8_qmax<FMT>()) : __uint_as_float(0x7FC00000u);
}
// The codes of x / d for four values. The quotient by the rounded reciprocal is within 2^-22 of the IEEE one; where
// 2^-21 more and less of it round to the same code, that is the code, else (one value in some ten thousand) the
// divisions are carried out.
template <int FMT> __device__ __noinline__ uint32_t codes4_div(float4 v, float d) {
    return kv8_code<FMT>(__fdiv_rn(v.x, d)) | (kv8_code<FMT>(__fdiv_rn(v.y, d)) << 8) | (kv8_code<FMT>(__fdiv_rn(v.z, d)) << 16) |
           (kv8_code<FMT>(__fdiv_rn(v.w, d)) << 24);
}
template <int FMT> __device__ __forceinline__ uint32_t pack4(float x, float y, float z, float w) {
    if constexpr (FMT == TLMG_KV8_INT8) {
        return __byte_perm(__byte_perm((uint32_t)__float2int_rn(x), (uint32_t)__float2int_rn(y), 0x0040),
                           __byte_perm((uint32_t)__float2int_rn(z), (uint32_t)__float2int_rn(w), 0x0040), 0x5410);
    } else {
        return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3) |
               ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(z, w), __NV_SATFINITE, __NV_E4M3) << 16);
    }
}
template <int FMT> __device__ __forceinline__ uint32_t codes4(float4 v, float d, float inv) {
    if (!(d == d)) return 0u;
    const float x = v.x * inv, y = v.y * inv, z = v.z * inv, w = v.w * inv;
    constexpr float lo = 1.0f - 0x1p-21f, hi = 1.0f + 0x1p-21f;
    const uint32_t c = pack4<FMT>(x * lo, y * lo, z * lo, w * lo);
    if (c != pack4<FMT>(x * hi, y * hi, z * hi, w * hi)) return codes4_div<FMT>(v, d);
    return c;
}
template <int FMT> __device__ __forceinline__ float4 values4(uint32_t w, float d) {
    return make_float4(__fmul_rn(kv8_value<FMT>(w & 255u), d), __fmul_rn(kv8_value<FMT>((w >> 8) & 255u), d),
                       __fmul_rn(kv8_value<FMT>((w >> 16) & 255u), d), __fmul_rn(kv8_value<FMT>(w >> 24), d));
}

constexpr int AP_WARPS = 4;

// grid (ceil(blocks a sequence can touch * 2 KV / 4 warps), n_seq)
template <int FMT, typename XT>
__global__ void __launch_bounds__(32 * AP_WARPS) k_kv8_append(const Kv8View c, const tlmg_kv8_batch b,
                                                              const XT *__restrict__ xk, const XT *__restrict__ xv,
                                                              int64_t x_stride) {
    const int s = blockIdx.y, lane = threadIdx.x & 31;
    Kv8Seq q;
    if (!kv8_seq(b, c.lp, s, q) || q.n == 0) return;
    const int unit = blockIdx.x * AP_WARPS + (threadIdx.x >> 5);
    const int is_v = unit & 1, kv = (unit >> 1) % c.KV, t_new = q.L - q.n;
    const int64_t blk = (int64_t)(t_new >> c.lb) + (unit >> 1) / c.KV;
    if (blk << c.lb >= q.L) return;
    const int t0 = (int)(blk << c.lb), t1 = min(q.L, t0 + (1 << c.lb)), ta = max(t0, t_new);
    const int32_t e = b.page_table[(size_t)s * b.table_stride + (t0 >> c.lp)];
    if (!c.ok(e)) return;
    const uint32_t r0 = c.row(e, kv, t0);
    uint8_t *codes = (is_v ? c.v : c.k) + (size_t)r0 * c.hd;
    float *scale = (is_v ? c.vs : c.ks) + (r0 >> c.lb);
    const XT *x = (is_v ? xv : xk) + (q.q0 + (int64_t)(ta - t_new)) * x_stride + (int64_t)kv * c.hd;
    const int per = c.hd >> 2, lper = 31 - __clz(per), n4 = (t1 - ta) << lper;
    float a = 0.0f;
#pragma unroll 8
    for (int i = lane; i < n4; i += 32) a = amax4(a, kv8_ld4(x + (int64_t)(i >> lper) * x_stride + 4 * (i & (per - 1))));
    float d = scale_of<FMT>(warp_max(a));
    float old = 0.0f;
    if (t0 < ta) {   // rows of an earlier call
        old = *scale;
        if (!(old <= d)) d = d == d ? old : d;     // max(old, d); a NaN of either side stays
    }
    const float inv = __frcp_rn(d);
    if (t0 < ta) {
        if (!(old == d)) {
            uint32_t *w = reinterpret_cast<uint32_t *>(codes);
            for (int i = lane; i < (ta - t0) << lper; i += 32) w[i] = codes4<FMT>(values4<FMT>(w[i], old), d, inv);
        }
        __syncwarp();                              // every lane has read the old scale
    }
    if (lane == 0) *scale = d;
    uint32_t *w = reinterpret_cast<uint32_t *>(codes + (size_t)(ta - t0) * c.hd);
#pragma unroll 4
    for (int i = lane; i < n4; i += 32)
        w[i] = codes4<FMT>(kv8_ld4(x + (int64_t)(i >> lper) * x_stride + 4 * (i & (per - 1))), d, inv);
    if (c.pos && !is_v)
        for (int t = ta + lane; t < t1; t += 32)
            c.pos[r0 + (uint32_t)(t - t0)] = b.q_pos ? b.q_pos[q.q0 + (t - t_new)] : t;
}

// One warp per (output row, KV head).
template <int FMT>
__global__ void __launch_bounds__(256) k_kv8_read(const Kv8View c, int n_seq, const int32_t *__restrict__ table,
                                                  int stride, const int32_t *__restrict__ row0,
                                                  const int32_t *__restrict__ start, int total, float *__restrict__ ko,
                                                  float *__restrict__ vo) {
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (unit >= (int64_t)total * c.KV) return;
    const int o = (int)(unit / c.KV), kv = (int)(unit - (int64_t)o * c.KV);
    int lo = 0, hi = n_seq;                        // the last sequence that starts at or before o
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (start[m] <= o) lo = m;
        else hi = m;
    }
    const int64_t t = (int64_t)row0[lo] + (o - start[lo]);
    int32_t e = -1;
    if (t >= 0 && (t >> c.lp) < stride) e = table[(size_t)lo * stride + (t >> c.lp)];
    const bool ok = c.ok(e);
    const uint32_t r = ok ? c.row(e, kv, (int)t) : 0u;
    const float nan = __uint_as_float(0x7FC00000u), dk = ok ? c.ks[r >> c.lb] : nan, dv = ok ? c.vs[r >> c.lb] : nan;
    const uint32_t *wk = reinterpret_cast<const uint32_t *>(c.k + (size_t)r * c.hd),
                   *wv = reinterpret_cast<const uint32_t *>(c.v + (size_t)r * c.hd);
    for (int i = lane; i < c.hd >> 2; i += 32) {
        kv8_st4(ko + unit * c.hd + 4 * i, values4<FMT>(wk[i], dk));
        kv8_st4(vo + unit * c.hd + 4 * i, values4<FMT>(wv[i], dv));
    }
}

// ---- eviction ----------------------------------------------------------------
// The order of weights as unsigned keys: larger weight, larger key; -0 is 0, a NaN is the lowest (key 0).
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int SEL_THREADS = 1024;
constexpr int SEL_BINS = 2048;
constexpr int SEL_CLUSTER = 8;
constexpr int SEL_KEEP = 4;       // keys a thread holds
constexpr int SEL_ALONE = 4096;   // rows up to which one CTA is as fast as a cluster

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
template <int CS> __device__ __forceinline__ void sync_all() {
    if constexpr (CS == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t ld_cluster(const uint32_t *p, uint32_t rank) {   // the word p of CTA `rank`'s shared memory
    uint32_t a, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// One CTA, or a cluster of CS over long caches, per (sequence, KV head). The
// m-th largest key of the rows between the first `sink` and the last `recent`
// is found digit by digit (11, 11 and 10 bits, a shared-memory count of each
// digit in every CTA's part, summed over the cluster), then one ordered pass
// writes the rows above it and as many rows equal to it, lowest first, as m
// leaves. Latency-bound: the weights are 4 bytes a row; 32,768 rows took 61 us
// with one CTA a head, 27 with a cluster of 8 (three passes with a cluster barrier
// each, and two more barriers after them).
template <int CS>
__global__ void __launch_bounds__(SEL_THREADS) k_kv8_select(int KV, const int32_t *__restrict__ kv_len, int max_kv,
                                                            const float *__restrict__ weights, int64_t w_stride,
                                                            int n_keep, int sink, int recent, int32_t *__restrict__ rows,
                                                            int32_t *__restrict__ lens) {
    __shared__ uint32_t hist[2][SEL_BINS];
    __shared__ uint32_t wsum[2][32], mine[2];
    __shared__ uint32_t pick_s, left_s;
    const int kv = blockIdx.x / CS, s = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = CS > 1 ? cluster_rank() : 0u;
    const int L = min(max(kv_len[s], 0), max_kv);
    int32_t *out = rows + ((size_t)s * KV + kv) * n_keep;
    const float *w = weights + ((size_t)s * KV + kv) * w_stride;
    const int first = (int)rank * SEL_THREADS + tid, step = CS * SEL_THREADS;
    if (kv == 0 && first == 0 && lens) lens[s] = min(L, n_keep);
    if (L <= n_keep) {   // the same for the whole cluster
        for (int j = first; j < n_keep; j += step) out[j] = j < L ? j : -1;
        return;
    }
    const int m = n_keep - sink - recent;
    for (int j = first; j < sink; j += step) out[j] = j;
    for (int j = first; j < recent; j += step) out[n_keep - recent + j] = L - recent + j;
    if (m == 0) return;
    // this CTA's part of the rows between, a multiple of the warp
    const int mid = L - recent - sink, part = ((mid + CS - 1) / CS + 31) / 32 * 32;
    const int lo = sink + min(mid, (int)rank * part), hi = sink + min(mid, ((int)rank + 1) * part);
    uint32_t key[SEL_KEEP];                    // the part's first keys stay in registers
#pragma unroll
    for (int u = 0; u < SEL_KEEP; u++) {
        const int t = lo + u * SEL_THREADS + tid;
        key[u] = t < hi ? weight_key(w[t]) : 0u;
    }
    uint32_t prefix = 0, left = (uint32_t)m;   // key bits found so far; rows still to take below them
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
        uint32_t *h = hist[pass & 1];          // the other one may still be read by the cluster
        for (int i = tid; i < bins; i += SEL_THREADS) h[i] = 0;
        __syncthreads();
        auto count = [&](uint32_t key, bool in) {
            if (in && (pass == 0 || (key >> (shift + (pass == 2 ? 10 : 11))) == prefix)) atomicAdd(&h[(key >> shift) & (uint32_t)(bins - 1)], 1u);
        };
#pragma unroll
        for (int u = 0; u < SEL_KEEP; u++) count(key[u], lo + u * SEL_THREADS + tid < hi);
        for (int t = lo + SEL_KEEP * SEL_THREADS + tid; t < hi; t += SEL_THREADS) count(weight_key(w[t]), true);
        sync_all<CS>();
        // counts from the top: thread i covers the bins / 1024 bins there
        const int per = bins / SEL_THREADS, b0 = bins - 1 - per * tid;
        uint32_t c0 = 0, c1 = 0;
#pragma unroll
        for (int r = 0; r < CS; r++) {
            c0 += CS == 1 ? h[b0] : ld_cluster(&h[b0], r);
            if (per == 2) c1 += CS == 1 ? h[b0 - 1] : ld_cluster(&h[b0 - 1], r);
        }
        const uint32_t sum = c0 + c1;
        uint32_t inc = sum;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) wsum[0][warp] = inc;
        __syncthreads();
        const uint32_t a = wsum[0][lane];
        const uint32_t upto = inc + __reduce_add_sync(0xFFFFFFFFu, lane < warp ? a : 0u), before = upto - sum;
        if (before < left && upto >= left) {       // exactly one thread
            const bool hit = before + c0 >= left;
            pick_s = (uint32_t)b0 - (hit ? 0u : 1u);
            left_s = left - before - (hit ? 0u : c0);
        }
        __syncthreads();
        prefix = (prefix << (pass == 2 ? 10 : 11)) | pick_s;
        left = left_s;
        __syncthreads();
    }
    // prefix is now the m-th largest key; `left` rows equal to it are taken
    uint32_t n_out = 0, n_eq = 0;
    if constexpr (CS > 1) {   // rows larger and equal in the parts before this one
        uint32_t g = 0, e = 0;
#pragma unroll
        for (int u = 0; u < SEL_KEEP; u++) {
            const bool in = lo + u * SEL_THREADS + tid < hi;
            g += in && key[u] > prefix;
            e += in && key[u] == prefix;
        }
        for (int t = lo + SEL_KEEP * SEL_THREADS + tid; t < hi; t += SEL_THREADS) {
            const uint32_t k = weight_key(w[t]);
            g += k > prefix;
            e += k == prefix;
        }
        g = __reduce_add_sync(0xFFFFFFFFu, g);
        e = __reduce_add_sync(0xFFFFFFFFu, e);
        if (tid < 2) mine[tid] = 0;
        __syncthreads();
        if (lane == 0) {
            atomicAdd(&mine[0], g);
            atomicAdd(&mine[1], e);
        }
        sync_all<CS>();
#pragma unroll
        for (uint32_t r = 0; r < CS; r++)
            if (r < rank) {
                n_out += ld_cluster(&mine[0], r);
                n_eq += ld_cluster(&mine[1], r);
            }
    }
    for (int t0 = lo; t0 < hi; t0 += SEL_THREADS) {
        const int t = t0 + tid;
        const uint32_t k = t < hi ? weight_key(w[t]) : 0u;
        const bool gt = t < hi && k > prefix, eq = t < hi && k == prefix;
        const uint32_t bg = __ballot_sync(0xFFFFFFFFu, gt), be = __ballot_sync(0xFFFFFFFFu, eq);
        if (lane == 0) {
            wsum[0][warp] = __popc(bg);
            wsum[1][warp] = __popc(be);
        }
        __syncthreads();
        const uint32_t a = wsum[0][lane], b = wsum[1][lane];
        const uint32_t g0 = n_out + __reduce_add_sync(0xFFFFFFFFu, lane < warp ? a : 0u);
        const uint32_t e0 = n_eq + __reduce_add_sync(0xFFFFFFFFu, lane < warp ? b : 0u);
        const uint32_t below = (1u << lane) - 1u;
        const uint32_t g = g0 + __popc(bg & below), q = e0 + __popc(be & below);   // larger / equal rows before t
        if (gt || (eq && q < left)) out[sink + (int)(g + min(q, left))] = t;
        n_out += __reduce_add_sync(0xFFFFFFFFu, a);
        n_eq += __reduce_add_sync(0xFFFFFFFFu, b);
        __syncthreads();
    }
    if constexpr (CS > 1) sync_all<CS>();   // no CTA leaves while another may read its shared memory
}

// One warp per (destination block, KV head, K or V). Kept rows lie apart, so
// that every row is two lines of its own: 4 heads x 4,096 rows of 128 in 11 us.
// Blocks of more than 32 rows, or than the registers hold, go over their rows
// twice (32,768 rows of 64 to 4,096, with the selection and the read-back: 44 us in
// blocks of 32, 50 in blocks of 64).
template <int FS, int FD>
__global__ void __launch_bounds__(32 * AP_WARPS) k_kv8_compact(const Kv8View c, const Kv8View d, const int32_t *__restrict__ table,
                                                               int stride, const int32_t *__restrict__ kv_len,
                                                               const int32_t *__restrict__ dtable, int dstride,
                                                               const int32_t *__restrict__ rows, int n_keep,
                                                               const float *__restrict__ weights, int64_t w_stride,
                                                               float *__restrict__ wout, int64_t wo_stride) {
    const int s = blockIdx.y, lane = threadIdx.x & 31;
    const int unit = blockIdx.x * AP_WARPS + (threadIdx.x >> 5);
    const int is_v = unit & 1, kv = (unit >> 1) % c.KV;
    const int64_t j0 = (int64_t)((unit >> 1) / c.KV) << d.lb;
    if (j0 >= n_keep) return;
    const int nj = (int)min((int64_t)1 << d.lb, n_keep - j0);
    const int L = kv_len[s];
    const int32_t *src = rows + ((size_t)s * c.KV + kv) * n_keep + j0;
    const int32_t de = (j0 >> d.lp) < dstride ? dtable[(size_t)s * dstride + (j0 >> d.lp)] : -1;
    const bool dok = d.ok(de);
    const uint32_t dr = dok ? d.row(de, kv, (int)j0) : 0u;
    const uint8_t *pool = is_v ? c.v : c.k;
    const float *sc = is_v ? c.vs : c.ks;
    // source row number of entry j
    auto source = [&](int j, uint32_t &r) {
        const int32_t t = j < nj ? src[j] : -1;
        if (t < 0 || t >= L || (t >> c.lp) >= stride) return false;
        const int32_t e = table[(size_t)s * stride + (t >> c.lp)];
        if (!c.ok(e)) return false;
        r = c.row(e, kv, t);
        return true;
    };
    // 32 rows a round: lane j finds row j's number and scale, then hd / 16 lanes share a row, 16 codes each
    const int lpr = c.hd >> 4, rpi = 32 / lpr, sub = lane / lpr, at = 16 * (lane - sub * lpr);
    auto rounds = [&](auto &&f) {
        for (int j0 = 0; j0 < nj; j0 += 32) {
            uint32_t r = 0;
            const bool ok = source(j0 + lane, r);
            const float v = ok ? sc[r >> c.lb] : 0.0f;
            const int left = min(32, nj - j0);
#pragma unroll 4
            for (int i = 0; i < left; i += rpi) {
                const uint32_t rr = __shfl_sync(0xFFFFFFFFu, r, i + sub);
                const float vv = __shfl_sync(0xFFFFFFFFu, v, i + sub);
                if (__shfl_sync(0xFFFFFFFFu, (int)ok, i + sub))
                    f(j0 + i + sub, *reinterpret_cast<const uint4 *>(pool + (size_t)rr * c.hd + at), vv);
            }
        }
    };
    float a = 0.0f;
    bool any = false;
    auto top = [&](uint4 w, float v) {
        any = true;
        a = amax4(amax4(amax4(amax4(a, values4<FS>(w.x, v)), values4<FS>(w.y, v)), values4<FS>(w.z, v)), values4<FS>(w.w, v));
    };
    uint8_t *to = (is_v ? d.v : d.k) + (size_t)dr * d.hd + at;
    float q = 0.0f, inv = 0.0f;
    auto put = [&](int j, uint4 w, float v) {
        *reinterpret_cast<uint4 *>(to + (size_t)j * d.hd) =
            make_uint4(codes4<FD>(values4<FS>(w.x, v), q, inv), codes4<FD>(values4<FS>(w.y, v), q, inv),
                       codes4<FD>(values4<FS>(w.z, v), q, inv), codes4<FD>(values4<FS>(w.w, v), q, inv));
    };
    auto scale = [&] {
        any = __any_sync(0xFFFFFFFFu, any);
        q = scale_of<FD>(warp_max(a));
        inv = __frcp_rn(q);
        any = any && dok;
        if (any && lane == 0) (is_v ? d.vs : d.ks)[dr >> d.lb] = q;
    };
    if (nj <= min(32, 8 * rpi)) {   // a row a lane, and the codes fit the warp's registers: all the block's loads at once, and once
        uint32_t r = 0;
        const bool ok = source(lane, r);
        const float v = ok ? sc[r >> c.lb] : 0.0f;
        uint4 w[8];
        float vv[8];
        bool have[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int j = i * rpi + sub;
            const uint32_t rr = __shfl_sync(0xFFFFFFFFu, r, j & 31);   // (from j = 32 on: no row, below)
            vv[i] = __shfl_sync(0xFFFFFFFFu, v, j & 31);
            have[i] = __shfl_sync(0xFFFFFFFFu, (int)ok, j & 31) && j < nj;
            if (have[i]) w[i] = *reinterpret_cast<const uint4 *>(pool + (size_t)rr * c.hd + at);
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (have[i]) top(w[i], vv[i]);
        scale();
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (have[i] && any) put(i * rpi + sub, w[i], vv[i]);
    } else {
        rounds([&](int, uint4 w, float v) { top(w, v); });
        scale();
        if (any) rounds(put);
    }
    if (!is_v)
        for (int j = lane; j < nj; j += 32) {
            uint32_t r;
            const bool ok = source(j, r);
            if (ok && dok) d.pos[dr + (uint32_t)j] = c.pos ? c.pos[r] : src[j];
            if (wout)
                wout[((size_t)s * c.KV + kv) * wo_stride + j0 + j] =
                    ok && src[j] < w_stride ? weights[((size_t)s * c.KV + kv) * w_stride + src[j]] : 0.0f;
        }
}

int launched(const char *what) {
    count_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? TLMG_OK : cuda_fail(e, what);
}

template <int FMT>
void append_launch(const Kv8View &v, const tlmg_kv8_batch &b, int x_dt, const void *k, const void *x, int64_t stride,
                   dim3 grid, cudaStream_t st) {
    if (x_dt == TLMG_DT_F32)
        k_kv8_append<FMT, float><<<grid, 32 * AP_WARPS, 0, st>>>(v, b, (const float *)k, (const float *)x, stride);
    else if (x_dt == TLMG_DT_F16)
        k_kv8_append<FMT, __half><<<grid, 32 * AP_WARPS, 0, st>>>(v, b, (const __half *)k, (const __half *)x, stride);
    else
        k_kv8_append<FMT, __nv_bfloat16><<<grid, 32 * AP_WARPS, 0, st>>>(v, b, (const __nv_bfloat16 *)k,
                                                                        (const __nv_bfloat16 *)x, stride);
}

}  // namespace
}  // namespace tlmg

using namespace tlmg;

extern "C" int tlmg_kv8_append(const tlmg_kv8 *c, const tlmg_kv8_batch *b, int x_dt, const void *k, const void *v,
                               int64_t x_stride, void *stream) {
    int rc = kv8_check("kv8_append", c);
    if (!rc) rc = kv8_check_batch("kv8_append", b);
    if (rc) return rc;
    if (x_dt != TLMG_DT_F32 && x_dt != TLMG_DT_F16 && x_dt != TLMG_DT_BF16)
        return set_error(TLMG_EINVAL, "kv8_append: row dtype %d (f32, f16 or bf16)", x_dt);
    if (b->total_q == 0 || b->max_q == 0) return TLMG_OK;
    if (!k || !v) return set_error(TLMG_EINVAL, "kv8_append: null pointer");
    const int64_t es = x_dt == TLMG_DT_F32 ? 4 : 2, st = x_stride ? x_stride : (int64_t)c->KV * c->hd;
    if (st < (int64_t)c->KV * c->hd || (st * es) % 16 || (((uintptr_t)k | (uintptr_t)v) & 15u))
        return set_error(TLMG_EINVAL, "kv8_append: rows must be 16-byte aligned, %lld elements apart or more (stride %lld)",
                         (long long)c->KV * c->hd, (long long)st);
    const Kv8View view = kv8_view(c);
    // n new rows touch at most this many blocks, whatever row they start at
    const int64_t blocks = ((int64_t)b->max_q + c->block - 2) / c->block + 1;
    const int64_t units = blocks * c->KV * 2;
    if (units > INT32_MAX - 64) return set_error(TLMG_ERANGE, "kv8_append: %lld blocks", (long long)units);
    const dim3 grid((unsigned)((units + AP_WARPS - 1) / AP_WARPS), b->n_seq);
    if (c->fmt == TLMG_KV8_INT8) append_launch<TLMG_KV8_INT8>(view, *b, x_dt, k, v, st, grid, pick_stream(stream));
    else append_launch<TLMG_KV8_E4M3>(view, *b, x_dt, k, v, st, grid, pick_stream(stream));
    return launched("kv8_append launch");
}

extern "C" int tlmg_kv8_read(const tlmg_kv8 *c, int n_seq, const int32_t *page_table, int table_stride,
                             const int32_t *row0, const int32_t *start, int total, float *k, float *v, void *stream) {
    int rc = kv8_check("kv8_read", c);
    if (rc) return rc;
    if (n_seq <= 0 || table_stride <= 0 || total < 0)
        return set_error(TLMG_EINVAL, "kv8_read: %d sequences, table stride %d, %d rows", n_seq, table_stride, total);
    if (total == 0) return TLMG_OK;
    if (!page_table || !row0 || !start || !k || !v) return set_error(TLMG_EINVAL, "kv8_read: null pointer");
    if (((uintptr_t)k | (uintptr_t)v) & 15u) return set_error(TLMG_EINVAL, "kv8_read: k and v must be 16-byte aligned");
    const int64_t grid = ((int64_t)total * c->KV + 7) / 8;
    if (grid > INT32_MAX) return set_error(TLMG_ERANGE, "kv8_read: %d rows x %d heads", total, c->KV);
    if (c->fmt == TLMG_KV8_INT8)
        k_kv8_read<TLMG_KV8_INT8><<<(unsigned)grid, 256, 0, pick_stream(stream)>>>(kv8_view(c), n_seq, page_table, table_stride,
                                                                                  row0, start, total, k, v);
    else
        k_kv8_read<TLMG_KV8_E4M3><<<(unsigned)grid, 256, 0, pick_stream(stream)>>>(kv8_view(c), n_seq, page_table, table_stride,
                                                                                  row0, start, total, k, v);
    return launched("kv8_read launch");
}

extern "C" int tlmg_kv8_select(int n_seq, int KV, const int32_t *kv_len, int max_kv, const float *weights, int64_t w_stride,
                               int n_keep, int sink, int recent, int32_t *rows, int32_t *lens, void *stream) {
    if (n_seq <= 0 || n_seq > 65535 || KV <= 0 || max_kv < 0 || w_stride < max_kv || n_keep <= 0 || sink < 0 ||
        recent < 0 || (int64_t)sink + recent > n_keep)
        return set_error(TLMG_EINVAL, "kv8_select: %d sequences x %d heads, max_kv %d, weight stride %lld, keep %d (%d first, %d last)",
                         n_seq, KV, max_kv, (long long)w_stride, n_keep, sink, recent);
    if (!kv_len || !weights || !rows) return set_error(TLMG_EINVAL, "kv8_select: null pointer");
    cudaStream_t st = pick_stream(stream);
    if (max_kv <= SEL_ALONE) {
        k_kv8_select<1><<<dim3(KV, n_seq), SEL_THREADS, 0, st>>>(KV, kv_len, max_kv, weights, w_stride, n_keep, sink, recent, rows, lens);
    } else {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)KV * SEL_CLUSTER, n_seq);
        cfg.blockDim = dim3(SEL_THREADS);
        cfg.stream = st;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = SEL_CLUSTER;
        at[0].val.clusterDim.y = 1;
        at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, k_kv8_select<SEL_CLUSTER>, KV, kv_len, max_kv, weights, w_stride, n_keep, sink, recent,
                                                 rows, lens);
        if (e != cudaSuccess) return cuda_fail(e, "kv8_select launch");
    }
    return launched("kv8_select launch");
}

extern "C" int tlmg_kv8_compact(const tlmg_kv8 *c, const tlmg_kv8 *dst, int n_seq, const int32_t *page_table,
                                int table_stride, const int32_t *kv_len, const int32_t *dst_table, int dst_stride,
                                const int32_t *rows, int n_keep, const float *weights, int64_t w_stride, float *weights_out,
                                int64_t wo_stride, void *stream) {
    int rc = kv8_check("kv8_compact", c);
    if (!rc) rc = kv8_check("kv8_compact (destination)", dst);
    if (rc) return rc;
    if (c->KV != dst->KV || c->hd != dst->hd)
        return set_error(TLMG_EINVAL, "kv8_compact: %d x %d heads into %d x %d", c->KV, c->hd, dst->KV, dst->hd);
    if (!dst->pos) return set_error(TLMG_EINVAL, "kv8_compact: the destination needs a position pool");
    if (n_seq <= 0 || n_seq > 65535 || table_stride <= 0 || dst_stride <= 0 || n_keep <= 0)
        return set_error(TLMG_EINVAL, "kv8_compact: %d sequences, table strides %d and %d, %d rows", n_seq, table_stride,
                         dst_stride, n_keep);
    if (!page_table || !kv_len || !dst_table || !rows) return set_error(TLMG_EINVAL, "kv8_compact: null pointer");
    if (weights_out && (!weights || wo_stride < n_keep))
        return set_error(TLMG_EINVAL, "kv8_compact: weights_out needs weights and a stride of %d (%lld)", n_keep, (long long)wo_stride);
    if (weights_out) {   // warps write it while others read the weights
        const int64_t rows_all = (int64_t)n_seq * c->KV;
        if (weights_out < weights + rows_all * std::max<int64_t>(w_stride, 0) && weights < weights_out + rows_all * wo_stride)
            return set_error(TLMG_EINVAL, "kv8_compact: weights_out overlaps weights");
    }
    const int64_t units = ((int64_t)(n_keep + dst->block - 1) / dst->block) * c->KV * 2;
    if (units > INT32_MAX - 64) return set_error(TLMG_ERANGE, "kv8_compact: %lld blocks", (long long)units);
    const dim3 grid((unsigned)((units + AP_WARPS - 1) / AP_WARPS), n_seq);
    const Kv8View a = kv8_view(c), d = kv8_view(dst);
    cudaStream_t st = pick_stream(stream);
#define TLMG_COMPACT(FS, FD)                                                                                              \
    if (c->fmt == FS && dst->fmt == FD)                                                                                   \
        k_kv8_compact<FS, FD><<<grid, 32 * AP_WARPS, 0, st>>>(a, d, page_table, table_stride, kv_len, dst_table, dst_stride, \
                                                              rows, n_keep, weights, w_stride, weights_out, wo_stride);
    TLMG_COMPACT(TLMG_KV8_INT8, TLMG_KV8_INT8)
    TLMG_COMPACT(TLMG_KV8_INT8, TLMG_KV8_E4M3)
    TLMG_COMPACT(TLMG_KV8_E4M3, TLMG_KV8_INT8)
    TLMG_COMPACT(TLMG_KV8_E4M3, TLMG_KV8_E4M3)
#undef TLMG_COMPACT
    return launched("kv8_compact launch");
}
