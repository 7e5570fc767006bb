// tlmg_kv8_attn.cu - attention over the 8-bit KV cache, split over the rows.
//
// One CTA takes a span of a sequence's rows, one KV head and a tile of query
// rows (a query row is one token's one head of the group; 8 rows, or 16 where
// a 16-bit call has more than 8 per KV head), and keeps a running maximum, sum
// and output per row; a second kernel joins the spans. This is the form for
// few query rows per KV head. A code byte of K or V feeds only 2 x 8
// multiply-adds, so HBM is the floor; what bounds it is the chain copy, f16,
// MMA, maximum, exponential, MMA of a tile (about 950 instructions for 32 rows)
// at the 8 to 12 warps that the registers allow: issue 41 %, HBM 41 %. One f32 query over 131,071 int8 rows
// of 4 heads of 128 takes 49 us (2.7 TB/s), 64 bf16 ones over 1 .. 8,192 e4m3
// rows 102 us (2.7 TB/s).
//
// Products run on mma.sync.m16n8k16 (f16 in, f32 out): the query rows of a
// group (1 .. 16) are below the 64-row minimum of tcgen05.mma, and at the HBM
// rate the K and V bytes of an SM need about a third of this instruction's
// rate. Codes become f16 exactly (tlmg_kv8.cuh), so the only roundings are
// the query's and the probabilities': an f32 query row is scaled by a power of
// two and enters as a high and a low f16 (22 bits) in rows r and r + 8 of one
// MMA, the probabilities likewise; 16-bit queries enter exactly, their
// probabilities as one f16 (11 bits, below the rounding of a 16-bit output).
//
// A warp owns tiles of 32 rows. Its lanes copy exactly the bytes that they
// themselves multiply (cp.async into a ring of two stages, no barrier between
// warps): contraction order is free, so lane (g, t4) holds the 16-byte pieces
// t4, t4 + 4, .. of key row g (mod 8) as its B fragments, and for V the hd / 8
// columns from g hd / 8 on of the four rows that its probabilities belong to.
//
// The product with V of one tile starts from zero and is added to the running
// output in f32 with the row's factor: probabilities times the rows' V scales
// are brought to f16 range by a power of two per row and tile, so that
// neither a large scale elsewhere in the cache nor a small one costs
// precision, and the tensor core's truncating sums stay short.
#include <algorithm>
#include <cmath>

#include "tlmg_dev.cuh"
#include "tlmg_internal.h"
#include "tlmg_kv8.cuh"
#include "tlmg_kv8_attn.cuh"

namespace tlmg {
namespace {

constexpr int TILE = 32;          // rows of a warp's tile
constexpr int NW = 4;             // warps of a CTA
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ uint32_t saddr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int N> __device__ __forceinline__ void cpN(uint32_t dst, const void *src, int src_bytes) {
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(src_bytes) : "memory");
}
template <int N> __device__ __forceinline__ void cpA(uint32_t dst, const void *src) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[2], uint32_t b0, uint32_t b1) {   // rows 8 .. 15 zero
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%6,%5,%6}, {%7,%8}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(0u), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the same with an accumulator that starts from zero
__device__ __forceinline__ void mma_f16_0(float (&c)[4], const uint32_t (&a)[2], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%6,%5,%6}, {%7,%8}, {%9,%9,%9,%9};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(0u), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_f16_0(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t pack_f16(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// x, y as f16 high parts and f16 remainders times 2^11 (LO makes up for it): the remainders of values near f16's
// smallest keep their bits
constexpr float LO = 0x1p-11f;
__device__ __forceinline__ void split_f16(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = pack_f16((x - f.x) * 0x1p11f, (y - f.y) * 0x1p11f);
}
// 2^e > |x| for finite x, e >= -100
__device__ __forceinline__ int exp_above(float x) { return max((int)((__float_as_uint(x) >> 23) & 255u) - 126, -100); }
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127

template <int HD> struct Plan {
    static constexpr int VB = HD / 8;                        // V bytes a lane takes of a row
    static constexpr int CH = VB > 16 ? 16 : VB;             // bytes of one copy
    static constexpr int VP = VB / CH;                       // copies per row
    static constexpr int META = 2 * TILE * HD;               // offset of scales, positions, documents
    static constexpr int STAGE = 2 * TILE * HD + 4 * TILE * 4;
    static constexpr int NST = 2;
    static constexpr int SMEM = NW * NST * STAGE;
};

__device__ __forceinline__ Kv8Range<TILE> key_range(const Kv8Attn &a, const Kv8Seq &q, int s, int i0, int i1) {
    int pmin = q.L - q.n + i0, pmax = q.L - q.n + i1 - 1;
    if (a.b.q_pos && !a.c.pos && (a.causal || a.window)) {
        pmin = INT32_MAX;
        pmax = INT32_MIN;
        for (int i = i0; i < i1; i++) {
            const int p = a.b.q_pos[q.q0 + i];
            pmin = min(pmin, p);
            pmax = max(pmax, p);
        }
    }
    return kv8_range<TILE>(a, q, s, pmin, pmax);
}

// CTAs of an SM, by registers: two f32 row tiles take 255; 16-bit queries over e4m3 rows spill at the 168 of three CTAs
// (64 ragged sequences: 121 us with three, 101 with two; int8 rows 99 and 106).
constexpr int split_ctas(int hd, bool f32, int rm, int fmt) {
    return hd > 128 ? 1 : f32 ? (rm == 2 ? 2 : 3) : fmt == TLMG_KV8_E4M3 && hd == 128 ? 2 : 3;
}

template <int HD, int FMT, typename QT, int RM>
__global__ void __launch_bounds__(32 * NW, split_ctas(HD, sizeof(QT) == 4, RM, FMT)) k_kv8_split(const __grid_constant__ Kv8Attn a) {
    constexpr bool F32 = sizeof(QT) == 4;
    constexpr int ROWS = 8 * RM;                             // query rows of the CTA (RM of a thread)
    constexpr int QR = F32 || RM == 2 ? 4 : 2;               // registers of a query fragment: rows 8 .. 15 may be zeros
    constexpr int MT = F32 ? RM : 1;                         // MMA row tiles (8 f32 rows or 16 others)
    constexpr int NT = HD / 8, KC = HD / 64, NST = Plan<HD>::NST;
    using P = Plan<HD>;
    extern __shared__ __align__(16) uint8_t sm[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int s = blockIdx.z, kvh = blockIdx.y % a.c.KV, rt = a.rt0 + blockIdx.y / a.c.KV, split = blockIdx.x;
    const int G = a.G, H = a.H;
    QT *out = static_cast<QT *>(a.out);
    Kv8Seq q;
    const float nan = __uint_as_float(0x7FC00000u);
    if (!kv8_seq(a.b, a.c.lp, s, q)) {
        // a sequence whose lengths do not fit: NaN for its tokens
        const int64_t i0 = max(q.q0, 0), i1 = min((int64_t)a.b.q_start[s + 1], (int64_t)a.b.total_q);
        const int64_t step = (int64_t)(gridDim.y / a.c.KV) * ROWS;
        for (int64_t R = rt * ROWS; R < (i1 - i0) * G; R += step) {
            for (int r = 0; r < ROWS && R + r < (i1 - i0) * G; r++) {
                const int64_t row = (i0 + (R + r) / G) * H + kvh * G + (R + r) % G;
                if (a.n_split > 1) {
                    if (tid == 0) {
                        a.pm[row * a.n_split + split] = -INFINITY;
                        a.pl[row * a.n_split + split] = nan;
                    }
                    for (int d = tid; d < HD; d += 32 * NW) a.po[(row * a.n_split + split) * HD + d] = nan;
                } else {
                    for (int d = 4 * tid; d < HD; d += 128 * NW) kv8_st4(out + row * HD + d, make_float4(nan, nan, nan, nan));
                    if (tid == 0 && a.lse) a.lse[row] = nan;
                    if (tid == 0 && a.lse2) a.lse2[row] = nan;
                }
            }
        }
        return;
    }
    const int R0 = rt * ROWS, n_rows = q.n * G;
    if (R0 >= n_rows) return;
    const int i0 = R0 / G, i1 = min(q.n, (R0 + ROWS - 1) / G + 1);
    const Kv8Range<TILE> rg = key_range(a, q, s, i0, i1);
    const int v0 = split * a.tiles, v1 = min(rg.n, v0 + a.tiles);
    const int n_my = v1 - v0 > warp ? (v1 - v0 - warp + NW - 1) / NW : 0;   // tiles v0 + warp + NW i

    const int32_t *table = a.b.page_table + (size_t)s * a.b.table_stride;
    const int32_t *docs = a.doc ? a.doc + (size_t)s * a.doc_stride : nullptr;
    uint8_t *ring = sm + (size_t)warp * NST * P::STAGE;
    int32_t te = -1;
    // pages of 32 rows and more hold a tile whole: one entry, offsets that the compiler knows
    const bool whole = a.c.lp >= 5;
    const int k_lane = g * HD + 16 * t4, v_lane = 2 * t4 * HD + g * P::VB;   // this lane's first K and V bytes of a tile
    auto load_te = [&](int i) {
        if (i < n_my) {
            const int t = rg.t0(v0 + warp + NW * i) + (whole ? 0 : lane);
            te = t < q.L ? __ldg(table + (t >> a.c.lp)) : -1;
        }
    };
    auto issue = [&](int i) {
        if (i < n_my) {
            const int t0 = rg.t0(v0 + warp + NW * i), t = t0 + lane;
            uint8_t *st = ring + (i % NST) * P::STAGE;
            const uint32_t sb = saddr(st), mb = sb + P::META + 4 * lane;
            const bool ok = t < q.L && a.c.ok(te);
            const uint32_t rid = ok ? a.c.row(te, kvh, t) : 0u;
            if (ok) {
                cpN<4>(mb, a.c.ks + (rid >> a.c.lb), 4);
                cpN<4>(mb + 4 * TILE, a.c.vs + (rid >> a.c.lb), 4);
                if (a.c.pos) cpN<4>(mb + 8 * TILE, a.c.pos + rid, 4);
            } else {   // past the end (masked below) or on a bad page (NaN for whoever sees it)
                float *m = reinterpret_cast<float *>(st + P::META);
                m[lane] = nan;
                m[TILE + lane] = nan;
                if (a.c.pos) reinterpret_cast<int *>(m)[2 * TILE + lane] = 0;
            }
            if (docs && !a.c.pos) {
                if (t < a.doc_stride) cpN<4>(mb + 12 * TILE, docs + t, 4);
                else reinterpret_cast<int *>(st + P::META)[3 * TILE + lane] = -1;
            }
            const uint32_t kd = sb + lane * 16, vd = sb + TILE * HD + lane * P::CH;
            if (whole && a.c.ok(te) && t0 + TILE <= q.L) {
                const uint8_t *ks = a.c.k + (size_t)a.c.row(te, kvh, t0) * HD, *vs = a.c.v + (ks - a.c.k) + v_lane;
                ks += k_lane;
#pragma unroll
                for (int nt = 0; nt < 4; nt++)
#pragma unroll
                    for (int c = 0; c < KC; c++) cpA<16>(kd + (nt * KC + c) * 512, ks + 8 * nt * HD + 64 * c);
#pragma unroll
                for (int kr = 0; kr < 8; kr++)   // rows 16 (kr / 4) + 2 t4 + {0, 1, 8, 9}
#pragma unroll
                    for (int c = 0; c < P::VP; c++)
                        cpA<P::CH>(vd + (kr * P::VP + c) * 32 * P::CH,
                                   vs + (16 * (kr >> 2) + (kr & 1) + 8 * ((kr >> 1) & 1)) * HD + 16 * c);
            } else {
#pragma unroll
                for (int nt = 0; nt < 4; nt++) {
                    const uint32_t r = __shfl_sync(0xFFFFFFFFu, rid, 8 * nt + g);
                    const int nb = __shfl_sync(0xFFFFFFFFu, ok ? 16 : 0, 8 * nt + g);
                    const uint8_t *src = a.c.k + (size_t)r * HD + 16 * t4;
#pragma unroll
                    for (int c = 0; c < KC; c++) cpN<16>(kd + (nt * KC + c) * 512, src + 64 * c, nb);
                }
#pragma unroll
                for (int kr = 0; kr < 8; kr++) {
                    const int row = 16 * (kr >> 2) + 2 * t4 + (kr & 1) + 8 * ((kr >> 1) & 1);
                    const uint32_t r = __shfl_sync(0xFFFFFFFFu, rid, row);
                    const int nb = __shfl_sync(0xFFFFFFFFu, ok ? P::CH : 0, row);
                    const uint8_t *src = a.c.v + (size_t)r * HD + g * P::VB;
#pragma unroll
                    for (int c = 0; c < P::VP; c++) cpN<P::CH>(vd + (kr * P::VP + c) * 32 * P::CH, src + 16 * c, nb);
                }
            }
        }
        cp_commit();   // an empty group past the end keeps the count uniform
    };
#pragma unroll
    for (int i = 0; i < NST - 1; i++) {
        load_te(i);
        issue(i);
    }
    load_te(NST - 1);

    // this thread's query rows: f16 fragments, the power of two taken out, masks
    uint32_t qa[MT][4 * KC][QR];
    float qs[RM], slope[RM];
    int qp[RM], qd[RM];
    {
        float4 x[RM][4 * KC];   // this lane's elements of its rows
        float up[RM];
#pragma unroll
        for (int r = 0; r < RM; r++) {
            const int R = R0 + g + 8 * r, tok = R / G, h = kvh * G + R % G;
            const bool live = R < n_rows;
            const int at = live ? tok : i0;   // a row past the end takes the first token's place
            const QT *qr = static_cast<const QT *>(a.q) + (q.q0 + (int64_t)at) * a.q_stride + (int64_t)(live ? h : kvh * G) * HD + 16 * t4;
#pragma unroll
            for (int c = 0; c < 4 * KC; c++) x[r][c] = kv8_ld4(qr + 64 * (c >> 2) + 4 * (c & 3));
            qp[r] = a.b.q_pos ? a.b.q_pos[q.q0 + at] : q.L - q.n + at;
            qd[r] = docs && live ? (qp[r] >= 0 && qp[r] < a.doc_stride ? docs[qp[r]] : -1) : -1;
            slope[r] = a.slopes && live ? a.slopes[h] * LOG2E : 0.0f;
            float m = 0.0f;
#pragma unroll
            for (int c = 0; c < 4 * KC; c++)
                m = fmaxf(m, fmaxf(fmaxf(fabsf(x[r][c].x), fabsf(x[r][c].y)), fmaxf(fabsf(x[r][c].z), fabsf(x[r][c].w))));
            m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
            // the row's largest element to 2^9 .. 2^10
            const int e = min(max(exp_above(m) - 10, -100), 100);
            up[r] = live ? pow2i(-e) : 0.0f;
            qs[r] = pow2i(e) * a.scale * kv8_cvt_unit<FMT>() * (a.softcap > 0.0f ? a.inv_cap : LOG2E);
        }
#pragma unroll
        for (int c = 0; c < 4 * KC; c++) {
#pragma unroll
            for (int r = 0; r < RM; r++) {
                x[r][c].x *= up[r];
                x[r][c].y *= up[r];
                x[r][c].z *= up[r];
                x[r][c].w *= up[r];
            }
            if constexpr (F32) {
#pragma unroll
                for (int r = 0; r < RM; r++) {
                    split_f16(x[r][c].x, x[r][c].y, qa[r][c][0], qa[r][c][1]);
                    split_f16(x[r][c].z, x[r][c].w, qa[r][c][2], qa[r][c][3]);
                }
            } else if constexpr (RM == 2) {
                qa[0][c][0] = pack_f16(x[0][c].x, x[0][c].y);
                qa[0][c][1] = pack_f16(x[1][c].x, x[1][c].y);
                qa[0][c][2] = pack_f16(x[0][c].z, x[0][c].w);
                qa[0][c][3] = pack_f16(x[1][c].z, x[1][c].w);
            } else {
                qa[0][c][0] = pack_f16(x[0][c].x, x[0][c].y);
                qa[0][c][1] = pack_f16(x[0][c].z, x[0][c].w);
            }
        }
    }
    const float capl = a.softcap * LOG2E;
    const int pre = a.prefix ? a.prefix[s] : 0;
    int pmin = qp[0], pmax = qp[0];
    if constexpr (RM == 2) {
        pmin = min(pmin, qp[1]);
        pmax = max(pmax, qp[1]);
    }

    float o[NT][2 * RM], mrun[RM], lrun[RM];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int r = 0; r < 2 * RM; r++) o[j][r] = 0.0f;
#pragma unroll
    for (int r = 0; r < RM; r++) mrun[r] = -INFINITY, lrun[r] = 0.0f;

    for (int i = 0; i < n_my; i++) {
        cp_wait<NST - 2>();
        __syncwarp();
        const uint8_t *st = ring + (i % NST) * P::STAGE;
        const int t0 = rg.t0(v0 + warp + NW * i);
        float sc[MT][4][4];
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int nt = 0; nt < 4; nt++) {
                const uint4 w = *reinterpret_cast<const uint4 *>(st + ((nt * KC + c) * 32 + lane) * 16);
                const uint32_t x[4] = { kv8_bias<FMT>(w.x), kv8_bias<FMT>(w.y), kv8_bias<FMT>(w.z), kv8_bias<FMT>(w.w) };
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t b0 = kv8_cvt2<FMT, 0, false>(x[j]), b1 = kv8_cvt2<FMT, 1, false>(x[j]);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if (c == 0 && j == 0) mma_f16_0(sc[mt][nt], qa[mt][0], b0, b1);
                        else mma_f16(sc[mt][nt], qa[mt][4 * c + j], b0, b1);
                    }
                }
            }
        // scores in log2 units (with a cap: over it, until the tanh), masked ones -inf
        const float *ms = reinterpret_cast<const float *>(st + P::META);
        const int *mi = reinterpret_cast<const int *>(ms);
        const bool full = !docs && !a.c.pos && t0 + TILE <= q.L &&
                          __all_sync(0xFFFFFFFFu, (!a.causal || t0 + TILE - 1 <= pmin) && (!a.window || pmax - t0 < a.window));
        float z[RM][8], vs[8];
#pragma unroll
        for (int nt = 0; nt < 4; nt++) {
            const float2 ks2 = *reinterpret_cast<const float2 *>(ms + 8 * nt + 2 * t4);
            const float2 vs2 = *reinterpret_cast<const float2 *>(ms + TILE + 8 * nt + 2 * t4);
            vs[2 * nt] = vs2.x;
            vs[2 * nt + 1] = vs2.y;
#pragma unroll
            for (int r = 0; r < RM; r++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const float dot = F32 ? __fmaf_rn(sc[F32 ? r : 0][nt][2 + u], LO, sc[F32 ? r : 0][nt][u]) : sc[0][nt][F32 ? 0 : 2 * r + u];
                    z[r][2 * nt + u] = dot * ((u ? ks2.y : ks2.x) * qs[r]);
                }
        }
        if (a.softcap > 0.0f) {
            float big = 0.0f;
#pragma unroll
            for (int r = 0; r < RM; r++)
#pragma unroll
                for (int j = 0; j < 8; j++) big = fmaxf(big, fabsf(z[r][j]));
            if (__all_sync(0xFFFFFFFFu, big < TANH_X)) {   // (a NaN may pass: the polynomial keeps it)
#pragma unroll
                for (int r = 0; r < RM; r++)
#pragma unroll
                    for (int j = 0; j < 8; j++) z[r][j] = capl * kv8_tanh_small(z[r][j]);
            } else {
#pragma unroll
                for (int r = 0; r < RM; r++)
#pragma unroll
                    for (int j = 0; j < 8; j++) z[r][j] = capl * tanhf(z[r][j]);
            }
        }
        if (a.slopes) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int col = 8 * (j >> 1) + 2 * t4 + (j & 1), kp = a.c.pos ? mi[2 * TILE + col] : t0 + col;
#pragma unroll
                for (int r = 0; r < RM; r++) z[r][j] = z[r][j] - slope[r] * fabsf((float)(qp[r] - kp));
            }
        }
        if (!full) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int col = 8 * (j >> 1) + 2 * t4 + (j & 1), t = t0 + col, kp = a.c.pos ? mi[2 * TILE + col] : t;
                int kd = -1;
                if (docs) kd = a.c.pos ? (kp >= 0 && kp < a.doc_stride ? __ldg(docs + kp) : -1) : mi[3 * TILE + col];
#pragma unroll
                for (int r = 0; r < RM; r++) {
                    bool see = kp < pre || ((!a.causal || kp <= qp[r]) && (!a.window || qp[r] - kp < a.window));
                    see = see && t < q.L && (!docs || kd == qd[r]);
                    z[r][j] = see ? z[r][j] : -INFINITY;
                }
            }
        }
        if (a.scores) {
#pragma unroll
            for (int r = 0; r < RM; r++) {
                const int R = R0 + g + 8 * r;
                if (R < n_rows) {
                    float *d = a.scores + ((q.q0 + (int64_t)(R / G)) * H + kvh * G + R % G) * a.s_stride + t0 + 2 * t4;
#pragma unroll
                    for (int nt = 0; nt < 4; nt++) *reinterpret_cast<float2 *>(d + 8 * nt) = make_float2(z[r][2 * nt], z[r][2 * nt + 1]);
                }
            }
        }
        float alpha[RM], back[RM];
        uint32_t pa[MT][2][QR];
#pragma unroll
        for (int r = 0; r < RM; r++) {
            float m = fmaxf(fmaxf(fmaxf(z[r][0], z[r][1]), fmaxf(z[r][2], z[r][3])), fmaxf(fmaxf(z[r][4], z[r][5]), fmaxf(z[r][6], z[r][7])));
            m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
            m = fmaxf(m, mrun[r]);
            const float sub = m == -INFINITY ? 0.0f : m;
            alpha[r] = m == -INFINITY ? 1.0f : kv8_ex2(mrun[r] - m);
            mrun[r] = m;
            float sum = 0.0f, top = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float p = kv8_ex2(z[r][j] - sub);
                sum += p;
                // a masked key's scale has no part in this, whatever it is
                z[r][j] = z[r][j] == -INFINITY ? 0.0f : p * vs[j];
                top = fmaxf(top, z[r][j]);
            }
            lrun[r] = __fmaf_rn(lrun[r], alpha[r], sum);
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const int e = exp_above(top);
            // p vs 2^(15 - e) < 2^15
            const float up = pow2i(min(15 - e, 100));
            back[r] = pow2i(max(e - 15, -100)) * kv8_cvt_unit<FMT>();
#pragma unroll
            for (int j = 0; j < 8; j++) z[r][j] *= up;
        }
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            if constexpr (F32) {
#pragma unroll
                for (int r = 0; r < RM; r++) {
                    split_f16(z[r][4 * kk], z[r][4 * kk + 1], pa[r][kk][0], pa[r][kk][1]);
                    split_f16(z[r][4 * kk + 2], z[r][4 * kk + 3], pa[r][kk][2], pa[r][kk][3]);
                }
            } else if constexpr (RM == 2) {
                pa[0][kk][0] = pack_f16(z[0][4 * kk], z[0][4 * kk + 1]);
                pa[0][kk][1] = pack_f16(z[RM - 1][4 * kk], z[RM - 1][4 * kk + 1]);
                pa[0][kk][2] = pack_f16(z[0][4 * kk + 2], z[0][4 * kk + 3]);
                pa[0][kk][3] = pack_f16(z[RM - 1][4 * kk + 2], z[RM - 1][4 * kk + 3]);
            } else {
                pa[0][kk][0] = pack_f16(z[0][4 * kk], z[0][4 * kk + 1]);
                pa[0][kk][1] = pack_f16(z[0][4 * kk + 2], z[0][4 * kk + 3]);
            }
        }
        bool same = alpha[0] == 1.0f;
        if constexpr (RM == 2) same = same && alpha[1] == 1.0f;
        if (!__all_sync(0xFFFFFFFFu, same)) {
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int r = 0; r < 2 * RM; r++) o[j][r] *= alpha[r >> 1];
        }
        asm volatile("" ::: "memory");   // V's words are not fetched before here: their registers are the probabilities'
        const uint8_t *vt = st + TILE * HD;
#pragma unroll
        for (int c = 0; c < P::VP; c++) {
            constexpr int CW = P::CH / 4;   // words of one copy
            uint32_t w[8][CW];
#pragma unroll
            for (int kr = 0; kr < 8; kr++) {
                const uint8_t *p = vt + ((kr * P::VP + c) * 32 + lane) * P::CH;
                if constexpr (CW == 4) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(p);
                    w[kr][0] = kv8_bias<FMT>(v.x);
                    w[kr][1] = kv8_bias<FMT>(v.y);
                    w[kr][2] = kv8_bias<FMT>(v.z);
                    w[kr][3] = kv8_bias<FMT>(v.w);
                } else {
                    const uint2 v = *reinterpret_cast<const uint2 *>(p);
                    w[kr][0] = kv8_bias<FMT>(v.x);
                    w[kr][1] = kv8_bias<FMT>(v.y);
                }
            }
#pragma unroll
            for (int x = 0; x < CW; x++) {
                // bytes of rows 2 t4 and 2 t4 + 1 (8 further: the second register) side by side
                uint32_t ev[4], od[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    ev[k] = __byte_perm(w[2 * k][x], w[2 * k + 1][x], 0x5140);
                    od[k] = __byte_perm(w[2 * k][x], w[2 * k + 1][x], 0x7362);
                }
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    float acc[MT][4];
#pragma unroll
                    for (int kk = 0; kk < 2; kk++) {
                        const uint32_t *u = y < 2 ? ev : od;
                        const uint32_t b0 = (y & 1) ? kv8_cvt2<FMT, 1, true>(u[2 * kk]) : kv8_cvt2<FMT, 0, true>(u[2 * kk]);
                        const uint32_t b1 = (y & 1) ? kv8_cvt2<FMT, 1, true>(u[2 * kk + 1]) : kv8_cvt2<FMT, 0, true>(u[2 * kk + 1]);
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            if (kk == 0) mma_f16_0(acc[mt], pa[mt][kk], b0, b1);
                            else mma_f16(acc[mt], pa[mt][kk], b0, b1);
                        }
                    }
                    float (&oj)[2 * RM] = o[16 * c + 4 * x + y];
                    if constexpr (F32) {
#pragma unroll
                        for (int r = 0; r < RM; r++) {
                            oj[2 * r] = __fmaf_rn(__fmaf_rn(acc[r][2], LO, acc[r][0]), back[r], oj[2 * r]);
                            oj[2 * r + 1] = __fmaf_rn(__fmaf_rn(acc[r][3], LO, acc[r][1]), back[r], oj[2 * r + 1]);
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < 2 * RM; r++) oj[r] = __fmaf_rn(acc[0][r], back[r >> 1], oj[r]);
                    }
                }
            }
        }
        __syncwarp();              // every lane has read this stage's scales before one copies over them
        issue(i + NST - 1);
        load_te(i + NST);
    }
    cp_wait<0>();
    __syncthreads();
    // join the warps: per row weights 2^(m_w - M). A row's HD columns lie in four runs (one per t4) of HD / 4 + 4
    // floats, HD + 16 in all, so that the eight lanes of a 16-byte store phase take different banks.
    constexpr int RUN = HD / 4 + 4, ROW = HD + 16;
    float *wo = reinterpret_cast<float *>(sm);                  // [NW][ROWS][ROW]
    float *wm = wo + NW * ROWS * ROW, *wl = wm + NW * ROWS;     // [NW][ROWS]
#pragma unroll
    for (int r = 0; r < RM; r++) {
        float l = lrun[r];
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
        float *d = wo + (warp * ROWS + g + 8 * r) * ROW + t4 * RUN;
#pragma unroll
        for (int j = 0; j < NT; j += 4) {
            kv8_st4(d + j, make_float4(o[j][2 * r], o[j + 1][2 * r], o[j + 2][2 * r], o[j + 3][2 * r]));
            kv8_st4(d + P::VB + j, make_float4(o[j][2 * r + 1], o[j + 1][2 * r + 1], o[j + 2][2 * r + 1], o[j + 3][2 * r + 1]));
        }
        if (t4 == 0) {
            wm[warp * ROWS + g + 8 * r] = mrun[r];
            wl[warp * ROWS + g + 8 * r] = l;
        }
    }
    __syncthreads();
    constexpr int TR = 32 * NW / ROWS;      // threads of a row, 4 columns each and TR * 4 further
    const int r = tid / TR, R = R0 + r, col0 = 4 * (tid % TR);
    if (R >= n_rows) return;
    float M = -INFINITY, L = 0.0f, f[NW];
#pragma unroll
    for (int w = 0; w < NW; w++) M = fmaxf(M, wm[w * ROWS + r]);
#pragma unroll
    for (int w = 0; w < NW; w++) {
        const float mw = wm[w * ROWS + r];
        f[w] = mw == -INFINITY ? 1.0f : kv8_ex2(mw - M);   // an empty warp holds zeros
        L = __fmaf_rn(wl[w * ROWS + r], f[w], L);
    }
    const int64_t row = (q.q0 + (int64_t)(R / G)) * H + kvh * G + R % G;
    const float inv = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
#pragma unroll 2
    for (int d = col0; d < HD; d += 4 * TR) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float4 u = *reinterpret_cast<const float4 *>(wo + (w * ROWS + r) * ROW + d + 4 * (d / (HD / 4)));
            v.x = __fmaf_rn(u.x, f[w], v.x);
            v.y = __fmaf_rn(u.y, f[w], v.y);
            v.z = __fmaf_rn(u.z, f[w], v.z);
            v.w = __fmaf_rn(u.w, f[w], v.w);
        }
        if (a.n_split > 1) kv8_st4(a.po + (row * a.n_split + split) * HD + d, v);
        else kv8_st4(out + row * HD + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    }
    if (col0 == 0) {
        if (a.n_split > 1) {
            a.pm[row * a.n_split + split] = M;
            a.pl[row * a.n_split + split] = L;
        } else {
            const float l2 = M + log2f(L);
            if (a.lse) a.lse[row] = l2 * LN2;
            if (a.lse2) a.lse2[row] = l2;
        }
    }
}

// out[row] = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M): one CTA per output row, HD / 4 column groups times the
// slices of the spans that 256 threads leave. Every warp finds M by itself. (111 spans of one long sequence: one
// slice of 4 with a serial maximum took 22 us.)
constexpr int JOIN_THREADS = 256;
template <int HD, typename QT>
__global__ void __launch_bounds__(JOIN_THREADS) k_kv8_join(const __grid_constant__ Kv8Attn a) {
    constexpr int CG = HD / 4, SL = JOIN_THREADS / CG;
    pdl_enter();
    __shared__ __align__(16) float ro[SL][HD];
    __shared__ float rl[SL];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, sl = tid / CG, d = 4 * (tid % CG), n = a.n_split;
    const float *m = a.pm + row * n, *l = a.pl + row * n, *po = a.po + row * n * HD + d;
    float M = -INFINITY;
    for (int i = tid & 31; i < n; i += 32) M = fmaxf(M, m[i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
    float L = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = sl; i < n; i += SL) {
        const float mi = m[i], li = l[i];
        if (mi == -INFINITY && li == 0.0f) continue;                // a span without visible keys
        const float f = mi == -INFINITY ? 1.0f : kv8_ex2(mi - M);   // -inf with a sum: a NaN, which stays
        const float4 u = *reinterpret_cast<const float4 *>(po + (size_t)i * HD);
        L = __fmaf_rn(li, f, L);
        v.x = __fmaf_rn(u.x, f, v.x);
        v.y = __fmaf_rn(u.y, f, v.y);
        v.z = __fmaf_rn(u.z, f, v.z);
        v.w = __fmaf_rn(u.w, f, v.w);
    }
    kv8_st4(&ro[sl][d], v);
    if (d == 0) rl[sl] = L;
    __syncthreads();
    if (sl) return;
#pragma unroll
    for (int k = 1; k < SL; k++) {
        const float4 u = *reinterpret_cast<const float4 *>(&ro[k][d]);
        v.x += u.x;
        v.y += u.y;
        v.z += u.z;
        v.w += u.w;
        L += rl[k];
    }
    const float inv = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
    kv8_st4(static_cast<QT *>(a.out) + row * HD + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    if (tid == 0) {
        const float l2 = M + log2f(L);
        if (a.lse) a.lse[row] = l2 * LN2;
        if (a.lse2) a.lse2[row] = l2;
    }
}

// weights[s][kv][t] += sum over the sequence's tokens and the group's heads
// of 2^(score - lse): one thread per row t, rows of a query tile read only
// where its CTAs wrote scores. 16 sequences of 2,000 .. 4,099 rows and 64
// heads: 13 us, bound by the scores' traffic (16 f32 a row in and out).
constexpr int WG_THREADS = 128;
template <int ROWS>
__global__ void __launch_bounds__(WG_THREADS) k_kv8_weights(const __grid_constant__ Kv8Attn a) {
    pdl_enter();
    __shared__ float l2[64 * 16];
    __shared__ int end_a[64 * 16 / 8], lo_b[64 * 16 / 8], end_b[64 * 16 / 8];
    const int s = blockIdx.z, kvh = blockIdx.y, tid = threadIdx.x;
    Kv8Seq q;
    if (!kv8_seq(a.b, a.c.lp, s, q) || q.n == 0) return;
    const int n_rows = q.n * a.G, n_rt = (n_rows + ROWS - 1) / ROWS;
    for (int R = tid; R < n_rows; R += WG_THREADS) l2[R] = a.lse2[(q.q0 + (int64_t)(R / a.G)) * a.H + kvh * a.G + R % a.G];
    for (int r = tid; r < n_rt; r += WG_THREADS) {
        const Kv8Range<TILE> rg = key_range(a, q, s, r * ROWS / a.G, min(q.n, (r * ROWS + ROWS - 1) / a.G + 1));
        end_a[r] = rg.nA * TILE;
        lo_b[r] = rg.loB;
        end_b[r] = rg.loB + (rg.n - rg.nA) * TILE;
    }
    __syncthreads();
    const int t = blockIdx.x * WG_THREADS + tid;
    if (t >= q.L) return;
    float sum = 0.0f;
    for (int r = 0; r < n_rt; r++) {
        if (!(t < end_a[r] || (t >= lo_b[r] && t < end_b[r]))) continue;
        const int R1 = min(n_rows, (r + 1) * ROWS);
        for (int R = r * ROWS; R < R1; R++) {
            const float z = a.scores[((q.q0 + (int64_t)(R / a.G)) * a.H + kvh * a.G + R % a.G) * a.s_stride + t];
            sum += z == -INFINITY ? 0.0f : kv8_ex2(z - l2[R]);
        }
    }
    a.weights[((int64_t)s * a.c.KV + kvh) * a.w_stride + t] += sum;
}

struct Split {
    bool wide;             // the tcgen05 kernel serves the call
    int rm;                // query rows of a CTA / 8
    int n, tiles;          // spans, 32-row tiles per span
    int64_t rtiles;        // query tiles
    size_t part, scores, total;   // floats of the partial results / scores, bytes in all
    int64_t s_stride;
};

Split split_plan(const tlmg_kv8 &c, const tlmg_kv8_batch &b, const tlmg_kv8_score &s, int H, int q_dt, bool weights) {
    Split p{};
    const int G = H / c.KV;
    p.wide = !weights && kv8_prefill_serves(c, b, H);
    if (p.wide) {
        p.total = kv8_prefill_work_bytes(c, b, s, H, q_dt) + 16;
        return p;
    }
    // 16 query rows a CTA where there are more than 8 (not for f32 ones of 256 dims: no registers)
    p.rm = (int64_t)b.max_q * G > 8 && (q_dt != TLMG_DT_F32 || c.hd <= 128) ? 2 : 1;
    const int rows = 8 * p.rm;
    p.rtiles = ((int64_t)std::min(b.max_q, b.total_q) * G + rows - 1) / rows;
    // rows that a query tile can see at most (the prefix is only known to the device)
    int64_t vis = b.max_kv;
    if (s.window > 0 && s.causal && !c.pos && !s.prefix && !b.q_pos)
        vis = std::min<int64_t>(vis, (int64_t)s.window + (rows + G - 1) / G + TILE);
    // Spans: one round of the CTAs that the SMs hold for one sequence; four for a batch, whose lengths differ.
    const int64_t slots = (int64_t)sm_count() * split_ctas(c.hd, q_dt == TLMG_DT_F32, p.rm, c.fmt) * (b.n_seq > 1 ? 4 : 1);
    const int64_t tiles = std::max<int64_t>(1, (vis + TILE - 1) / TILE), base = p.rtiles * c.KV * b.n_seq;
    const int64_t want = std::max<int64_t>(1, slots / base);
    p.tiles = (int)std::max<int64_t>(NW, (tiles + want - 1) / want);
    p.n = (int)((tiles + p.tiles - 1) / p.tiles);
    const size_t rows_all = (size_t)b.total_q * H;
    p.part = p.n > 1 ? rows_all * p.n * (2 + (size_t)c.hd) : 0;
    p.s_stride = ((int64_t)b.max_kv + TILE - 1) / TILE * TILE;
    p.scores = weights ? rows_all * ((size_t)p.s_stride + 1) : 0;
    p.total = ((p.part + 3) / 4 * 4 + p.scores) * 4 + 16;
    return p;
}

template <typename F> cudaError_t launch_dep(F fn, dim3 grid, int block, const Kv8Attn &a, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, a);
}

template <int HD, int FMT, typename QT, int RM>
int launch_split_rows(const Kv8Attn &a, const Split &p, cudaStream_t st) {
    auto fn = k_kv8_split<HD, FMT, QT, RM>;
    constexpr int ROWS = 8 * RM;
    constexpr size_t join = (size_t)NW * ROWS * (HD + 18) * 4, sm = std::max<size_t>(Plan<HD>::SMEM, join);
    if (!smem_opt_in((const void *)fn, sm)) return set_error(TLMG_EIO, "kv8_attend: shared memory opt-in failed");
    // query tiles and KV heads are the grid's y, which ends at 65,535: longer calls take launches of whole tiles in turn
    Kv8Attn part = a;
    const int64_t step = 65535 / a.c.KV;
    cudaError_t e = cudaSuccess;
    for (int64_t t = 0; e == cudaSuccess && t < p.rtiles; t += step) {
        part.rt0 = (int)t;
        fn<<<dim3(p.n, (unsigned)(std::min(step, p.rtiles - t) * a.c.KV), a.b.n_seq), 32 * NW, sm, st>>>(part);
        count_launch();
        e = cudaGetLastError();
    }
    if (e == cudaSuccess && p.n > 1) {
        e = launch_dep(k_kv8_join<HD, QT>, dim3((unsigned)((int64_t)a.b.total_q * a.H)), JOIN_THREADS, a, st);
        count_launch();
    }
    if (e == cudaSuccess && a.weights && a.b.max_kv > 0) {
        const dim3 grid((a.b.max_kv + WG_THREADS - 1) / WG_THREADS, a.c.KV, a.b.n_seq);
        e = launch_dep(k_kv8_weights<ROWS>, grid, WG_THREADS, a, st);
        count_launch();
    }
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? TLMG_OK : cuda_fail(e, "kv8_attend launch");
}
template <int HD, int FMT, typename QT> int launch_split(const Kv8Attn &a, const Split &p, cudaStream_t st) {
    if constexpr (sizeof(QT) == 2 || HD <= 128)
        if (p.rm == 2) return launch_split_rows<HD, FMT, QT, 2>(a, p, st);
    return launch_split_rows<HD, FMT, QT, 1>(a, p, st);
}

template <int HD, int FMT> int launch_split_q(const Kv8Attn &a, const Split &p, int q_dt, cudaStream_t st) {
    if (q_dt == TLMG_DT_F32) return launch_split<HD, FMT, float>(a, p, st);
    if (q_dt == TLMG_DT_F16) return launch_split<HD, FMT, __half>(a, p, st);
    return launch_split<HD, FMT, __nv_bfloat16>(a, p, st);
}
template <int FMT> int launch_split_hd(const Kv8Attn &a, const Split &p, int q_dt, cudaStream_t st) {
    if (a.c.hd == 64) return launch_split_q<64, FMT>(a, p, q_dt, st);
    if (a.c.hd == 128) return launch_split_q<128, FMT>(a, p, q_dt, st);
    return launch_split_q<256, FMT>(a, p, q_dt, st);
}

int check_attend(const tlmg_kv8 *c, const tlmg_kv8_batch *b, const tlmg_kv8_score *s, int H, int q_dt) {
    int rc = kv8_check("kv8_attend", c);
    if (!rc) rc = kv8_check_batch("kv8_attend", b);
    if (rc) return rc;
    if (!s) return set_error(TLMG_EINVAL, "kv8_attend: null score");
    if (H <= 0 || H % c->KV || H / c->KV > 16)
        return set_error(TLMG_EINVAL, "kv8_attend: %d heads over %d KV heads (at most 16 per KV head)", H, c->KV);
    if (q_dt != TLMG_DT_F32 && q_dt != TLMG_DT_F16 && q_dt != TLMG_DT_BF16)
        return set_error(TLMG_EINVAL, "kv8_attend: query dtype %d (f32, f16 or bf16)", q_dt);
    if (!(s->scale >= 0.0f) || !std::isfinite(s->scale) || !(s->softcap >= 0.0f) || !std::isfinite(s->softcap) ||
        s->window < 0 || (s->doc && s->doc_stride <= 0))
        return set_error(TLMG_EINVAL, "kv8_attend: scale %g, softcap %g, window %d, document stride %d", (double)s->scale,
                         (double)s->softcap, s->window, s->doc_stride);
    if ((int64_t)b->total_q * H > INT32_MAX || c->KV > 65535 ||
        (kv8_prefill_serves(*c, *b, H) && (int64_t)b->max_q * (H / c->KV) >= 1 << 28))
        return set_error(TLMG_ERANGE, "kv8_attend: %d tokens x %d heads on %d, at most %d tokens a sequence", b->total_q, H, c->KV, b->max_q);
    return TLMG_OK;
}

}  // namespace
}  // namespace tlmg

using namespace tlmg;

extern "C" size_t tlmg_kv8_attend_work_bytes(const tlmg_kv8 *c, const tlmg_kv8_batch *b, const tlmg_kv8_score *s, int H,
                                             int q_dt, int with_weights) {
    if (check_attend(c, b, s, H, q_dt)) return 0;
    if (b->total_q == 0 || b->max_q == 0) return 16;   // nothing to do
    return split_plan(*c, *b, *s, H, q_dt, with_weights != 0).total;
}

extern "C" int tlmg_kv8_attend(const tlmg_kv8 *c, const tlmg_kv8_batch *b, const tlmg_kv8_score *s, int H, int q_dt,
                               const void *q, int64_t q_stride, void *out, float *lse, float *weights, int64_t w_stride,
                               void *work, size_t work_bytes, void *stream) {
    int rc = check_attend(c, b, s, H, q_dt);
    if (rc) return rc;
    if (b->total_q == 0 || b->max_q == 0) return TLMG_OK;
    if (!q || !out) return set_error(TLMG_EINVAL, "kv8_attend: null pointer");
    const int64_t es = q_dt == TLMG_DT_F32 ? 4 : 2, st = q_stride ? q_stride : (int64_t)H * c->hd;
    if (st < (int64_t)H * c->hd || (st * es) % 16 || (((uintptr_t)q | (uintptr_t)out) & 15u))
        return set_error(TLMG_EINVAL, "kv8_attend: query rows must be 16-byte aligned, %lld elements apart or more (stride %lld)",
                         (long long)H * c->hd, (long long)st);
    if (weights && (b->max_q > 64 || w_stride < b->max_kv))
        return set_error(TLMG_EINVAL, "kv8_attend: weights of at most 64 tokens a sequence (%d), stride %lld for %d rows",
                         b->max_q, (long long)w_stride, b->max_kv);
    const Split p = split_plan(*c, *b, *s, H, q_dt, weights != nullptr);
    if (p.total > 16 && (!work || ((uintptr_t)work & 15u) || work_bytes < p.total))
        return set_error(work && work_bytes < p.total ? TLMG_ERANGE : TLMG_EINVAL,
                         "kv8_attend: work holds %zu bytes at %p, needs %zu, 16-byte aligned", work_bytes, work, p.total);
    Kv8Attn a{};
    a.c = kv8_view(c);
    a.kv8 = *c;
    a.b = *b;
    a.H = H;
    a.G = H / c->KV;
    a.inv_g = a.G > 1 ? (uint32_t)((0x100000000ull + a.G - 1) / a.G) : 0u;
    a.q = q;
    a.q_stride = st;
    a.out = out;
    a.lse = lse;
    a.weights = weights;
    a.w_stride = w_stride;
    a.scale = s->scale > 0.0f ? s->scale : 1.0f / sqrtf((float)c->hd);
    a.softcap = s->softcap;
    a.inv_cap = s->softcap > 0.0f ? 1.0f / s->softcap : 0.0f;
    a.slopes = s->slopes;
    a.prefix = s->prefix;
    a.doc = s->doc;
    a.doc_stride = s->doc_stride;
    a.causal = s->causal;
    a.window = s->window;
    a.n_split = p.n;
    a.tiles = p.tiles;
    float *w = static_cast<float *>(work);
    const size_t rows = (size_t)b->total_q * H;
    if (p.n > 1) {
        a.po = w;
        a.pm = a.po + rows * p.n * c->hd;
        a.pl = a.pm + rows * p.n;
    }
    if (weights) {
        a.scores = w + (p.part + 3) / 4 * 4;
        a.s_stride = p.s_stride;
        a.lse2 = a.scores + rows * p.s_stride;
    }
    cudaStream_t cs = pick_stream(stream);
    if (p.wide) return kv8_prefill(a, q_dt, work, cs);
    return c->fmt == TLMG_KV8_INT8 ? launch_split_hd<TLMG_KV8_INT8>(a, p, q_dt, cs) : launch_split_hd<TLMG_KV8_E4M3>(a, p, q_dt, cs);
}
