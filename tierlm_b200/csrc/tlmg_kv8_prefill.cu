// tlmg_kv8_prefill.cu - attention over the 8-bit KV cache for many query rows,
// on tcgen05 (head_dim 64 and 128).
//
// out = sum_t p_t v_t / sum_t p_t with p_t = 2^(score_t - reference): 4 hd flops a visible pair, so the tensor core is
// the floor (2,048 clocks a key tile of 256 rows at hd 128). What is reached is set by the way from a tile's scores to its
// weights: 2,600 clocks of softmax and 1,700 of MMAs and signals, half of each under the other tile's. 65,536 rows x 2,048
// tokens x 32 heads of 128: 2,055 us, 1,053 TFLOP/s; a chunk of 2,048 on 16,384 rows 642 us, with a soft cap 1,046.
//
// 16-bit queries: one CTA per SM takes 256 query rows (token, head of the
// group) of one KV head in two tiles A and B of 128, and walks the visible keys
// in tiles of 128. Warps:
//   0-7, 8-15  softmax of tile A, B: two threads per query row (= TMEM lane), each with half of the keys
//   16-23      K and V codes -> f16 in shared memory, once for both tiles; or, where enough query tiles share them
//              (IMG), none: a kernel before this one wrote every key tile as the tensor core reads it, and
//              one thread brings K, V and scales by bulk copies (converting in every CTA: 18k chunk 1,398 us,
//              images 1,184; the softmax threads get 104 registers in place of 80)
//   last four  the first issues the MMAs (a warpgroup, for its share of the registers)
// Items that would leave SMs idle are cut along the keys (tail_plan) and joined by k_kv8_pieces.
// Per key tile and query tile: S = Q K^T (8 x tcgen05.mma M128 N128 K16 at
// hd 128, operands in shared memory, S f32 in TMEM); the softmax warps read S
// and write P as f16 over it (each half over its own columns); O += P V (A operand P from TMEM, V from shared
// memory, O f32 in TMEM). While one tile's softmax runs, the tensor core
// works for the other: TMEM is full at 2 x (S 128 + O 128) columns.
//
// Scales. A key's score is S * k_scale (per column) * the row's factor; the
// weight that multiplies V's code is p * v_scale. Each row keeps a reference
// w = max over its visible keys of score + log2(v_scale) and stores
// p'' = 2^(score - w + 14), so p'' * v_scale < 2^16 fits f16 whatever the scales
// of other rows, and the row sum of p'' divides the result. The reference
// follows the maximum when it grew by more than a factor of 2^1.9; then the
// warp multiplies its O rows in TMEM (its MMAs are done: the commit that
// announced S covers the PV before it).
//
// Layouts. Shared-memory operands are 8 x 16-byte core matrices without
// swizzle: chunk c (8 dims) of row r at (r / 8) * hd * 16 + c * 128 + (r % 8) *
// 16, so 8 lanes write 8 rows of one chunk, 128 contiguous bytes. The same
// bytes are K as a K-major B operand (contraction over dims) and V as an
// MN-major one (contraction over keys).
//
// O's sums truncate: after RUN tiles O goes into an f32 sum of the softmax threads and starts again from zero.
//
// f32 queries (one query tile a CTA): Q and P are two f16 each, the high part and the remainder (P's times 2^11); S
// sums the two products of Q, O's two products stay apart, start from zero at every key tile and are added to f32
// registers a tile later, since the tensor core's sums truncate. S has two buffers, so the next tile's scores form
// while this one's are weighed.
//
// Every wait is bounded: a role whose wait runs out sets a flag, all roles
// leave, and the CTA's outputs are NaN.
#include <cstdint>

#include "tlmg_dev.cuh"
#include "tlmg_internal.h"
#include "tlmg_kv8.cuh"
#include "tlmg_kv8_attn.cuh"

namespace tlmg {
namespace {

constexpr int TK = 128;           // keys of a tile
constexpr int TQ = 128;           // query rows of a tile
constexpr int HC = TK / 2;        // keys of a softmax thread: two threads share a query row
constexpr int CV = 256;           // converting threads
// What differs between 16-bit queries (two query tiles in turn) and f32 ones (one tile of which every operand but K and V
// has a high and a low part), with converting warps or with tile images. Registers a thread: 16-bit 72 at launch (896 x 72 =
// 64,512), then 512 x 80 + 256 x 56 + 128 x 72 = 64,512; f32 96 at launch (640 x 96 = 61,440), then 256 x 144 + 256 x 56 +
// 128 x 72 = 60,416. Images: 16-bit 96 at launch (640 x 96 = 61,440), then 512 x 104 + 128 x 64 = 61,440; f32 168 at
// launch (384 x 168 = 64,512), then 256 x 200 + 128 x 96 = 63,488.
template <bool F32, bool IMG> struct Role {
    static constexpr int TILES = F32 ? 1 : 2;                 // query tiles of a CTA
    static constexpr int SW = 8 * TILES;                      // softmax warps; then those that convert and 4 for the MMAs
    static constexpr int MW = SW + (IMG ? 0 : 8);             // the MMAs' first warp
    static constexpr int THREADS = 32 * (MW + 4);
    static constexpr int REGS_SOFTMAX = IMG ? (F32 ? 200 : 104) : F32 ? 144 : 80, REGS_CONVERT = 56,
                         REGS_MMA = IMG ? (F32 ? 96 : 64) : 72;
};
template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
constexpr int META = 4;           // buffers of per-key scales
// Key tiles (262,144 rows) up to which those that no query of the CTA sees are left out by a list, where a position pool or
// documents mask: 8,192 tokens of 32 heads on 4 with a pool took 3,350 us with every tile read.
constexpr int LIST = 2048;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ uint32_t saddr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// What the softmax needs of a tile's keys: scales (of V also log2 and 1 / scale), positions and documents.
struct Meta {
    float ks[TK], vs[TK], lv[TK], rv[TK];
    int pos[TK], doc[TK];
};
// A tile as an image in global memory: K and V as the tensor core reads them, then Meta; and what decides whether it is read.
template <int HD> constexpr size_t IMAGE = 2 * (size_t)TK * HD * 2 + sizeof(Meta);
struct alignas(16) Kv8Head {
    int pmin, pmax, dmin, dmax;   // of its rows: positions and documents
    int tame, pad[3];
};

template <int HD> struct Smem {
    alignas(128) uint8_t q[2][TQ * HD * 2];
    alignas(128) uint8_t k[2][TK * HD * 2];
    alignas(128) uint8_t v[2][TK * HD * 2];
    alignas(128) Meta m[META];
    // per quarter of a tile: no scale is extreme; with a table to mask by: every row of the CTA sees every key
    alignas(4) uint8_t tame[META][4], seen[META][4];
    uint32_t row[2][TK];
    float qs[2][TQ], part[2][2][TQ], sums[2][2][TQ];     // [tile (f32 queries' maxima: key tile & 1)][half][row]: the halves' maxima; in the end their sums
    uint64_t q_full, k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2], p_full[2], p_half[2], x_full[2], o_full[2], meta_full[META], drain;
    uint32_t tmem;
    int abort, pmin, pmax, dmin, dmax, n_list;
    uint16_t list[LIST];      // the key tiles that hold a key which a query may see
};

__device__ __forceinline__ void mbar_init(uint64_t *b, uint32_t n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(saddr(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(saddr(b)) : "memory");
}
// Waits for phase `parity`; false when it did not come in about a second or another role gave up.
__device__ __forceinline__ bool mbar_wait(uint64_t *b, uint32_t parity, int *abort) {
#pragma unroll 1
    for (uint32_t i = 0; i < (1u << 20); i++) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
                     : "=r"(done)
                     : "r"(saddr(b)), "r"(parity)
                     : "memory");
        if (done) return true;
        if ((i & 63u) == 63u && abort && *(volatile int *)abort) return false;
    }
    if (abort) *(volatile int *)abort = 1;
    return false;
}
// The same with one outcome for a warp. (One lane polling and a shuffle of its result took 1.6 times as long over all:
// a shuffle waits in the queue that the MMAs are issued through; 18k case 1,087 us, with the vote 1,004.)
__device__ __forceinline__ bool mbar_wait_warp(uint64_t *b, uint32_t parity, int *abort) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(b, parity, abort));
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Shared-memory operand descriptor, no swizzle, version 1: start, leading and stride byte offsets.
__device__ __forceinline__ uint64_t umma_desc(uint32_t start, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((start >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}
// Instruction descriptor: D f32, A and B f16, A K-major, B K-major or MN-major, M 128.
constexpr uint32_t idesc(int n, bool b_mn) {
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TQ >> 4) << 24);
}
// The whole warp runs the issuing code, converged and on warp-uniform values (descriptors then live in uniform
// registers); `lead` is set in one lane, which alone issues. Code that one lane runs by itself takes about 200 clocks
// per MMA to move its operands, three times what the MMA takes.
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc, uint32_t lead) {
    const uint32_t z = 0;
    asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(id), "r"(acc), "r"(z), "r"(lead)
                 : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc, uint32_t lead) {
    const uint32_t z = 0;
    asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(id), "r"(acc), "r"(z), "r"(lead)
                 : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t *b, uint32_t lead) {
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(saddr(b)), "r"(lead)
                 : "memory");
}

#define TLMG_R32(V)                                                                                                       \
    V(0), V(1), V(2), V(3), V(4), V(5), V(6), V(7), V(8), V(9), V(10), V(11), V(12), V(13), V(14), V(15), V(16), V(17),   \
        V(18), V(19), V(20), V(21), V(22), V(23), V(24), V(25), V(26), V(27), V(28), V(29), V(30), V(31)
#define TLMG_OUT(I) "=r"(v[I])
#define TLMG_IN(I) "r"(v[I])
// 32 columns of the warp's lanes; the load and its wait are one statement
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
                 "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
                 "tcgen05.wait::ld.sync.aligned;\n"
                 : TLMG_R32(TLMG_OUT)
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ldc(uint32_t addr, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
                 "[%16];\n\ttcgen05.wait::ld.sync.aligned;\n"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                   "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};\n" ::"r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld4(uint32_t addr, uint32_t (&v)[4]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];\n\ttcgen05.wait::ld.sync.aligned;\n"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t addr, const uint32_t (&v)[4]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%4], {%0, %1, %2, %3};\n" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st2(uint32_t addr, const uint32_t (&v)[2]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%2], {%0, %1};\n" ::"r"(v[0]), "r"(v[1]), "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                 "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};\n" ::TLMG_R32(TLMG_IN),
                 "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                 "%14, %15};\n" ::"r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
                 "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ldc(uint32_t a, uint32_t (&v)[32]) { tmem_ld32(a, v); }
__device__ __forceinline__ void tmem_stc(uint32_t a, const uint32_t (&v)[8]) { tmem_st8(a, v); }
__device__ __forceinline__ void tmem_stc(uint32_t a, const uint32_t (&v)[16]) { tmem_st16(a, v); }
__device__ __forceinline__ void tmem_stc(uint32_t a, const uint32_t (&v)[32]) { tmem_st32(a, v); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void mbar_expect(uint64_t *b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(saddr(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *b) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(saddr(dst)), "l"(src), "r"(bytes),
                 "r"(saddr(b))
                 : "memory");
}

// packed pairs of f32 (one issue slot for two)
typedef unsigned long long f2;
__device__ __forceinline__ f2 pk(float x, float y) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ f2 pku(uint32_t x, uint32_t y) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(x), "r"(y));
    return r;
}
__device__ __forceinline__ void upk(f2 a, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a)); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float ex2(float x) { return kv8_ex2(x); }
__device__ __forceinline__ uint32_t pack_f16(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// what the f16 pair h leaves of x, y, times `mul`, as f16
__device__ __forceinline__ uint32_t rest_f16(float x, float y, uint32_t h, float mul) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
    return pack_f16((x - f.x) * mul, (y - f.y) * mul);
}

// softcap * log2(e) * tanh(y) by the exponential. The approximate division and exponential, of 2 units
// in the last place each, keep it within 2^-20 of the cap: 1 / (1 + e^2y) is at most 1 and no steeper than 1 / 4 in 2y.
__device__ __forceinline__ float cap_exp(float y, float capl) {
    return __fmaf_rn(-2.0f * capl, __fdividef(1.0f, ex2(y * (2.0f * LOG2E)) + 1.0f), capl);
}

constexpr float TOP = 14.0f;   // log2 of the largest p * v_scale right after a row's reference moved
constexpr float GROW = 1.9f;   // how far it may grow before the reference moves again: 2^15.9 is an f16 (65,504 its largest)
// 16-bit queries: key tiles whose products O adds up in the tensor core before they go into an f32 sum of rounded
// additions. The tensor core's own sums truncate, 8 a tile and 2^-23 at most each, all towards zero: a run loses 2^-13 of
// sum p |v| at most (1e-4 measured, at 131,072 and at 524,288 positive rows; as one sum 8.3e-4 and 3.3e-3).
constexpr int RUN = 128;

// The CTAs' work: one item a query tile and KV head, last tokens first since they see the most keys; the items from a.n_full
// on are cut along the keys.
struct Kv8Item {
    int s, kvh, rt, piece, pieces;
};
__device__ __forceinline__ Kv8Item kv8_item(const Kv8Attn &a, int b) {
    Kv8Item r;
    r.pieces = b < a.n_full ? 1 : a.pieces;
    r.piece = b < a.n_full ? 0 : (b - a.n_full) % a.pieces;
    const int i = b < a.n_full ? b : a.n_full + (b - a.n_full) / a.pieces, per = a.q_tiles * a.nkv, x = i % per;
    r.s = a.s0 + i / per;
    r.kvh = a.kv0 + x % a.nkv;
    r.rt = a.q_tiles - 1 - x / a.nkv;
    return r;
}

// Joins the pieces: out = sum_p o_p 2^(w_p - W) / sum_p l_p 2^(w_p - W), W the largest reference; one warp a query row.
template <int HD, typename QT>
__global__ void __launch_bounds__(256) k_kv8_pieces(const __grid_constant__ Kv8Attn a) {
    constexpr int RPC = Role<sizeof(QT) == 4, true>::TILES * TQ;
    const int lane = threadIdx.x & 31, t = blockIdx.x / (RPC / 8), r = blockIdx.x % (RPC / 8) * 8 + (threadIdx.x >> 5);
    const Kv8Item it = kv8_item(a, a.n_full + t * a.pieces);
    Kv8Seq q;
    const int R = it.rt * RPC + r;
    if (!kv8_seq(a.b, a.c.lp, it.s, q) || R >= q.n * a.G) return;     // (a bad sequence's rows are NaN already)
    const int64_t row = (q.q0 + (int64_t)(R / a.G)) * a.H + it.kvh * a.G + R % a.G;
    const size_t p0 = (size_t)t * a.pieces * RPC + r;
    float W = -INFINITY, L = 0.0f;
    for (int p = 0; p < a.pieces; p++) W = fmaxf(W, a.pm[p0 + (size_t)p * RPC]);
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int p = 0; p < a.pieces; p++) {
        const size_t at = p0 + (size_t)p * RPC;
        const float w = a.pm[at], l = a.pl[at];
        if (w == -INFINITY && l == 0.0f) continue;                 // no visible keys
        const float f = w == -INFINITY ? 1.0f : ex2(w - W);        // -inf with a sum: a NaN, which stays
        L = __fmaf_rn(l, f, L);
        if (lane < HD / 4) {
            const float4 u = *reinterpret_cast<const float4 *>(a.po + at * HD + 4 * lane);
            v = make_float4(__fmaf_rn(u.x, f, v.x), __fmaf_rn(u.y, f, v.y), __fmaf_rn(u.z, f, v.z), __fmaf_rn(u.w, f, v.w));
        }
    }
    const float inv = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
    if (lane < HD / 4)
        kv8_st4(static_cast<QT *>(a.out) + row * HD + 4 * lane, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    if (lane == 0 && a.lse) a.lse[row] = L == 0.0f ? -INFINITY : (log2f(L) - (W == -INFINITY ? 0.0f : TOP - W)) * LN2;
}

// Smallest and largest position of a sequence's tokens (by all threads of the CTA).
__device__ __forceinline__ void token_span(const Kv8Attn &a, const Kv8Seq &q, int *mm, int &pmin, int &pmax) {
    pmin = q.L - q.n, pmax = q.L - 1;
    if (!a.b.q_pos) return;
    if (threadIdx.x == 0) mm[0] = INT32_MAX, mm[1] = INT32_MIN;
    __syncthreads();
    int lo = INT32_MAX, hi = INT32_MIN;
    for (int i = threadIdx.x; i < q.n; i += blockDim.x) {
        const int p = a.b.q_pos[q.q0 + i];
        lo = min(lo, p), hi = max(hi, p);
    }
    lo = __reduce_min_sync(0xFFFFFFFFu, lo), hi = __reduce_max_sync(0xFFFFFFFFu, hi);
    if ((threadIdx.x & 31) == 0) atomicMin(&mm[0], lo), atomicMax(&mm[1], hi);
    __syncthreads();
    pmin = mm[0], pmax = mm[1];
}
// Whether a row between these positions may be seen by a token between those.
__device__ __forceinline__ bool may_see(const Kv8Attn &a, int pre, int kmin, int kmax, int pmin, int pmax) {
    return kmin < pre || ((!a.causal || kmin <= pmax) && (!a.window || (int64_t)pmin - kmax < a.window));
}

// Tile images: every key tile that a token of its sequence may see, converted once for all of the query tiles. One CTA a
// tile and KV head.
template <int HD, int FMT>
__global__ void __launch_bounds__(256) k_kv8_images(const __grid_constant__ Kv8Attn a) {
    constexpr int SBO = HD * 16, PC = HD / 16, NP = TK * PC / 128;
    __shared__ int mm[2], span[4][4], ok4[4];
    __shared__ uint32_t row[TK];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, s = a.s0 + blockIdx.z, kvh = a.kv0 + blockIdx.y, t0 = blockIdx.x * TK;
    Kv8Seq q;
    if (!kv8_seq(a.b, a.c.lp, s, q) || t0 >= q.L || q.n == 0) return;
    int pmin, pmax;
    token_span(a, q, mm, pmin, pmax);
    const Kv8Range<TK> rg = kv8_range<TK>(a, q, s, pmin, pmax);
    if (!rg.has(t0)) return;
    const size_t at = ((size_t)blockIdx.z * gridDim.y + blockIdx.y) * a.n_img + blockIdx.x;
    uint8_t *img = a.img + at * IMAGE<HD>;
    Kv8Head *head = reinterpret_cast<Kv8Head *>(a.heads) + at;
    const int32_t *table = a.b.page_table + (size_t)s * a.b.table_stride;
    if (tid < TK) {
        const int t = t0 + tid;
        const int32_t e = t < q.L ? __ldg(table + (t >> a.c.lp)) : -1;
        const bool have = a.c.ok(e);
        const uint32_t rid = have ? a.c.row(e, kvh, t) : 0xFFFFFFFFu;
        row[tid] = rid;
        const float none = t < q.L ? __uint_as_float(0x7FC00000u) : 1.0f;   // a bad page: NaN for whoever sees it
        const float ks = have ? __ldg(a.c.ks + (rid >> a.c.lb)) : none, vs = have ? __ldg(a.c.vs + (rid >> a.c.lb)) : none;
        const int p = a.c.pos ? (have ? __ldg(a.c.pos + rid) : 0) : t;
        const int d = a.doc && p >= 0 && p < a.doc_stride ? __ldg(a.doc + (size_t)s * a.doc_stride + p) : -1;
        Meta *m = reinterpret_cast<Meta *>(img + 4 * TK * HD);
        m->ks[tid] = ks, m->vs[tid] = vs, m->lv[tid] = fmaxf(log2f(vs), -60.0f), m->rv[tid] = __frcp_rn(vs);
        m->pos[tid] = p, m->doc[tid] = d;
        const bool in = t < q.L, tame = __all_sync(0xFFFFFFFFu, vs > 0x1p-60f && vs < 0x1p60f);
        const int x0 = __reduce_min_sync(0xFFFFFFFFu, in ? p : INT32_MAX), x1 = __reduce_max_sync(0xFFFFFFFFu, in ? p : INT32_MIN),
                  x2 = __reduce_min_sync(0xFFFFFFFFu, in ? d : INT32_MAX), x3 = __reduce_max_sync(0xFFFFFFFFu, in ? d : INT32_MIN);
        if (lane == 0) span[warp][0] = x0, span[warp][1] = x1, span[warp][2] = x2, span[warp][3] = x3, ok4[warp] = tame;
    }
    __syncthreads();
    Kv8Head hd;
    hd.pmin = min(min(span[0][0], span[1][0]), min(span[2][0], span[3][0]));
    hd.pmax = max(max(span[0][1], span[1][1]), max(span[2][1], span[3][1]));
    hd.dmin = min(min(span[0][2], span[1][2]), min(span[2][2], span[3][2]));
    hd.dmax = max(max(span[0][3], span[1][3]), max(span[2][3], span[3][3]));
    hd.tame = ok4[0] && ok4[1] && ok4[2] && ok4[3];
    hd.pad[0] = hd.pad[1] = hd.pad[2] = 0;
    if (tid == 0) *head = hd;
    // hidden by the position pool from every token: no list takes it (a sequence too long for lists reads all tiles)
    if (a.c.pos && rg.n <= LIST && !may_see(a, a.prefix ? a.prefix[s] : 0, hd.pmin, hd.pmax, pmin, pmax)) return;
    const int h = tid & 127, prow = (h & 7) + 8 * (h / (8 * PC)), piece = (h >> 3) % PC;
    constexpr int RSTEP = 8 * (128 / (8 * PC));
    const uint8_t *pool = tid >= 128 ? a.c.v : a.c.k;
    uint8_t *dst = img + (tid >= 128 ? 2 * TK * HD : 0) + (prow >> 3) * SBO + piece * 256 + (prow & 7) * 16;
    uint4 x[NP];
#pragma unroll
    for (int i = 0; i < NP; i++) {
        const uint32_t rid = row[prow + RSTEP * i];
        x[i] = rid != 0xFFFFFFFFu ? __ldg(reinterpret_cast<const uint4 *>(pool + (size_t)rid * HD + 16 * piece)) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < NP; i++, dst += RSTEP / 8 * SBO) {
        const uint32_t b0 = kv8_bias<FMT>(x[i].x), b1 = kv8_bias<FMT>(x[i].y), b2 = kv8_bias<FMT>(x[i].z), b3 = kv8_bias<FMT>(x[i].w);
        *reinterpret_cast<uint4 *>(dst) = make_uint4(kv8_half2<FMT, 0>(b0), kv8_half2<FMT, 1>(b0), kv8_half2<FMT, 0>(b1), kv8_half2<FMT, 1>(b1));
        *reinterpret_cast<uint4 *>(dst + 128) = make_uint4(kv8_half2<FMT, 0>(b2), kv8_half2<FMT, 1>(b2), kv8_half2<FMT, 0>(b3), kv8_half2<FMT, 1>(b3));
    }
}

// IMG: K and V come as tile images (whose codes' unit is a.unit) by bulk copies; else by 8 converting warps.
// SHAPED: softcap, slopes, documents or a position pool; without them the code is half the size, and the instruction
// cache is what these roles share most tightly.
template <int HD, int FMT, typename QT, bool SHAPED, bool IMG>
__global__ void __launch_bounds__(Role<sizeof(QT) == 4, IMG>::THREADS, 1) k_kv8_prefill(const __grid_constant__ Kv8Attn a) {
    extern __shared__ __align__(128) uint8_t raw[];
    Smem<HD> &sm = *reinterpret_cast<Smem<HD> *>(raw);
    constexpr bool F32 = sizeof(QT) == 4;
    using RL = Role<F32, IMG>;
    constexpr int THREADS = RL::THREADS, SW = RL::SW, MW = RL::MW, RPC = RL::TILES * TQ;   // query rows of the CTA
    constexpr int SBO = HD * 16;              // bytes between 8-row groups of an operand
    constexpr int PC = HD / 16;               // 16-byte pieces of a code row
    constexpr int NP = TK * PC / CV;          // pieces of half a tile per converting thread
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Kv8Item it = kv8_item(a, blockIdx.x);
    const int s = it.s, kvh = it.kvh, tiles = a.q_tiles, rt = it.rt;
    const float unit = IMG ? a.unit : kv8_f16_unit<FMT>();
    const size_t slot = IMG ? ((size_t)(s - a.s0) * a.nkv + kvh - a.kv0) * a.n_img : 0;
    const Kv8Head *heads = reinterpret_cast<const Kv8Head *>(a.heads) + slot;
    QT *out = static_cast<QT *>(a.out);
    Kv8Seq q;
    if (!kv8_seq(a.b, a.c.lp, s, q)) {
        const float nan = __uint_as_float(0x7FC00000u);
        const int64_t i0 = max(q.q0, 0), i1 = min((int64_t)a.b.q_start[s + 1], (int64_t)a.b.total_q);
        for (int64_t R = (int64_t)rt * (THREADS / 32) + warp; R < (i1 - i0) * a.G; R += (int64_t)tiles * (THREADS / 32)) {
            const int64_t row = (i0 + R / a.G) * a.H + kvh * a.G + R % a.G;
            for (int d = 4 * lane; d < HD; d += 128) kv8_st4(out + row * HD + d, make_float4(nan, nan, nan, nan));
            if (lane == 0 && a.lse) a.lse[row] = nan;
        }
        return;
    }
    // R / G for the rows of a call (fewer than 2^28, G at most 16): the division's own code would be a good part of the start
    auto token_of = [&](int R) { return (int)__umulhi((uint32_t)R, a.inv_g) + (a.G == 1 ? R : 0); };
    const int n_rows = q.n * a.G, R0 = rt * RPC;
    if (R0 >= n_rows) return;
    const bool two = !F32 && R0 + TQ < n_rows;
    const int i0 = token_of(R0), i1 = min(q.n, token_of(R0 + RPC - 1) + 1);
    // the query rows set out for L2 while the CTA finds its tiles
    constexpr int LINES = HD * (int)sizeof(QT) / 128;
    for (int i = tid; i < min(RPC, n_rows - R0) * LINES; i += THREADS) {
        const int R = R0 + i / LINES, tk = token_of(R);
        const QT *x = static_cast<const QT *>(a.q) + (q.q0 + (int64_t)tk) * a.q_stride + (kvh * a.G + R - tk * a.G) * HD;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(x + i % LINES * (128 / (int)sizeof(QT))));
    }
    if (tid == 0) {
        sm.abort = 0;
        sm.pmin = INT32_MAX;
        sm.pmax = INT32_MIN;
        sm.dmin = INT32_MAX;
        sm.dmax = INT32_MIN;
        mbar_init(&sm.q_full, two ? 4 * TQ : 2 * TQ);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sm.k_full[i], IMG ? 1 : CV / 2);
            mbar_init(&sm.v_full[i], IMG ? 1 : CV / 2);
            mbar_init(&sm.k_empty[i], 1);
            mbar_init(&sm.v_empty[i], 1);
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.p_full[i], 2 * TQ);
            mbar_init(&sm.p_half[i], 2 * TQ);
            mbar_init(&sm.x_full[i], 2 * TQ);
            mbar_init(&sm.o_full[i], 1);
        }
        for (int i = 0; i < META; i++) mbar_init(&sm.meta_full[i], IMG ? 1 : 128);
        mbar_init(&sm.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&sm.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    for (int i = i0 + tid; i < i1; i += THREADS) {
        const int p = a.b.q_pos ? a.b.q_pos[q.q0 + i] : q.L - q.n + i;
        atomicMin(&sm.pmin, p);
        atomicMax(&sm.pmax, p);
        if constexpr (SHAPED)
            if (a.doc) {
                const int d = p >= 0 && p < a.doc_stride ? a.doc[(size_t)s * a.doc_stride + p] : -1;
                atomicMin(&sm.dmin, d);
                atomicMax(&sm.dmax, d);
            }
    }
    __syncthreads();
    const int pmin = sm.pmin, pmax = sm.pmax;
    const Kv8Range<TK> rg = kv8_range<TK>(a, q, s, pmin, pmax);
    const uint32_t tmem = sm.tmem;
    const int32_t *docs = a.doc ? a.doc + (size_t)s * a.doc_stride : nullptr;
    // A piece takes its share of the tiles: of those listed where a tile's header says who sees it, else of all of them (a
    // list of all for each of 37 pieces cost a third of 32 tokens over 131,072 rows).
    int n = rg.n, first = 0;
    auto share = [&] {
        first = (int)((int64_t)n * it.piece / it.pieces);
        n = (int)((int64_t)n * (it.piece + 1) / it.pieces) - first;
    };
    if (!IMG) share();
    const int v_0 = first;
    bool listed = false;
    if constexpr (SHAPED) {
        listed = n <= LIST && (docs || (a.c.pos && (a.causal || a.window)));
        if (listed) {
            // a tile takes part if one of its keys lies where the rows' positions allow, and its document between the
            // queries' smallest and largest (a bad page's rows stand at 0, as below)
            const int lo = sm.dmin, hi = sm.dmax, pre = a.prefix ? a.prefix[s] : 0;
            const int32_t *table = a.b.page_table + (size_t)s * a.b.table_stride;
            if constexpr (IMG) {
                for (int v = tid; v < n; v += THREADS) {
                    const int4 x = __ldg(reinterpret_cast<const int4 *>(heads + rg.t0(v) / TK));
                    sm.list[v] = may_see(a, pre, x.x, x.y, pmin, pmax) && (!docs || (x.w >= lo && x.z <= hi));
                }
            }
            for (int v = warp; !IMG && v < n; v += THREADS / 32) {
                const int tv = rg.t0(v_0 + v);
                bool any = false;
                int kp[TK / 32];
#pragma unroll
                for (int i = 0; i < TK / 32; i++) {
                    const int t = tv + 32 * i + lane;
                    kp[i] = t;
                    if (a.c.pos) {
                        const int32_t e = t < q.L ? __ldg(table + (t >> a.c.lp)) : -1;
                        kp[i] = a.c.ok(e) ? __ldg(a.c.pos + a.c.row(e, kvh, t)) : 0;
                    }
                }
#pragma unroll
                for (int i = 0; i < TK / 32; i++) {
                    bool see = kp[i] < pre || ((!a.causal || kp[i] <= pmax) && (!a.window || (int64_t)pmin - kp[i] < a.window));
                    if (docs) {
                        const int d = kp[i] >= 0 && kp[i] < a.doc_stride ? __ldg(docs + kp[i]) : -1;
                        see = see && d >= lo && d <= hi;
                    }
                    any = any || (see && tv + 32 * i + lane < q.L);
                }
                any = __any_sync(0xFFFFFFFFu, any);
                if (lane == 0) sm.list[v] = any;
            }
            __syncthreads();
            if (warp == 0) {   // the flags become the tiles' numbers, in place and in order
                int at = 0;
                for (int v0 = 0; v0 < n; v0 += 32) {
                    const bool in = v0 + lane < n && sm.list[v0 + lane];
                    const uint32_t b = __ballot_sync(0xFFFFFFFFu, in);
                    __syncwarp();
                    if (in) sm.list[at + __popc(b & ((1u << lane) - 1u))] = (uint16_t)(v0 + lane);
                    __syncwarp();
                    at += __popc(b);
                }
                if (lane == 0) sm.n_list = at;
            }
            __syncthreads();
            n = sm.n_list;
            first = 0;
        }
    }
    if (IMG) share();
    auto tile_at = [&](int j) { return rg.t0(SHAPED && listed ? v_0 + sm.list[first + j] : first + j); };

    if (warp < SW) {
        // ---- softmax of one query tile ----
        regs_up<RL::REGS_SOFTMAX>();
        const int w = warp >> 3, half = (warp >> 2) & 1, r = tid & (TQ - 1), k0 = half * HC;
        if (w == 0 || two) {
            const int R = R0 + w * TQ + r;
            const bool live = R < n_rows;
            const int tok = live ? token_of(R) : i0, h = kvh * a.G + (live ? R - tok * a.G : 0);
            const int qp = a.b.q_pos ? a.b.q_pos[q.q0 + tok] : q.L - q.n + tok;
            const int qd = docs ? (qp >= 0 && qp < a.doc_stride ? docs[qp] : -1) : -1;
            const float slope = a.slopes ? a.slopes[h] * LOG2E : 0.0f;
            const int pre = a.prefix ? a.prefix[s] : 0;
            const int64_t orow = (q.q0 + (int64_t)tok) * a.H + h;
            {   // query rows as f16, each row's largest element brought to 2^9 .. 2^10: a warp takes 8 rows at a time, four
                // lanes a row, and writes 128 contiguous bytes per chunk
                const int r8 = lane & 7, cq = lane >> 3;
#pragma unroll 1
                for (int g = 0; g < 2; g++) {
                    float4 x[F32 ? HD / 32 : 1][2];
                    uint4 x16[HD / 32];
                    const int rr = R0 + w * TQ + (warp & 7) * 16 + 8 * g + r8;
                    const int tk = rr < n_rows ? token_of(rr) : i0, hh = kvh * a.G + (rr < n_rows ? rr - tk * a.G : 0);
                    const QT *src = static_cast<const QT *>(a.q) + (q.q0 + (int64_t)tk) * a.q_stride + hh * HD + 8 * cq;
                    // elements 8 i .. of chunk i
                    auto get = [&](int i, float4 &u, float4 &v) {
                        if constexpr (F32) u = x[i][0], v = x[i][1];
                        else u = kv8_ld4(reinterpret_cast<const QT *>(&x16[i])), v = kv8_ld4(reinterpret_cast<const QT *>(&x16[i]) + 4);
                    };
#pragma unroll
                    for (int i = 0; i < HD / 32; i++) {
                        if constexpr (F32) x[i][0] = kv8_ld4(src + 32 * i), x[i][1] = kv8_ld4(src + 32 * i + 4);
                        else x16[i] = *reinterpret_cast<const uint4 *>(src + 32 * i);
                    }
                    const int row = (warp & 7) * 16 + 8 * g + r8;
                    float m = 0.0f;
#pragma unroll
                    for (int i = 0; i < HD / 32; i++) {
                        float4 u, v;
                        get(i, u, v);
                        m = fmaxf(m, fmaxf(fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(u.z), fabsf(u.w))),
                                           fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)))));
                    }
                    m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 16));
                    const int e = min(max((int)((__float_as_uint(m) >> 23) & 255u) - 136, -100), 100);
                    const float up = R0 + w * TQ + row < n_rows ? __int_as_float((127 - e) << 23) : 0.0f;
                    if (cq == 0) sm.qs[w][row] = __int_as_float((127 + e) << 23) * a.scale * unit;
                    uint8_t *dst = sm.q[w] + (row >> 3) * SBO + (row & 7) * 16 + cq * 128;
#pragma unroll
                    for (int i = 0; i < HD / 32; i++) {
                        float4 u, v;
                        get(i, u, v);
                        const uint4 hi = make_uint4(pack_f16(u.x * up, u.y * up), pack_f16(u.z * up, u.w * up),
                                                    pack_f16(v.x * up, v.y * up), pack_f16(v.z * up, v.w * up));
                        *reinterpret_cast<uint4 *>(dst + 512 * i) = hi;
                        if constexpr (F32)
                            *reinterpret_cast<uint4 *>(dst + TQ * HD * 2 + 512 * i) =
                                make_uint4(rest_f16(u.x * up, u.y * up, hi.x, 1.0f), rest_f16(u.z * up, u.w * up, hi.y, 1.0f),
                                           rest_f16(v.x * up, v.y * up, hi.z, 1.0f), rest_f16(v.z * up, v.w * up, hi.w, 1.0f));
                    }
                }
                fence_async_smem();
                mbar_arrive(&sm.q_full);
            }
            bool ok = mbar_wait_warp(&sm.q_full, 0, &sm.abort);
            const float qsc = sm.qs[w][r];
            const uint32_t lanes = (uint32_t)(warp & 3) << 21;           // this warp's 32 TMEM lanes
            const uint32_t to = tmem + lanes + 2 * TK + w * HD;          // O (f32 queries: then O of the remainders)
            const bool lists = SHAPED && (docs || a.c.pos);        // masks that go by a table
            const float qs2 = qsc * LOG2E, capl = a.softcap * LOG2E, capx = qsc * a.inv_cap;
            const float mul = SHAPED && a.softcap > 0.0f ? capx : qs2;
            float wref = -INFINITY, lsum = 0.0f;
            // f32 queries: this thread's half of the row's output, and what the reference's last move multiplies it by
            float o[F32 ? HD / 2 : 1], fo = 1.0f;
            // 16-bit queries: this thread's half of O of the runs so far and the reference it goes by, in local memory: none of
            // it takes a register of the tile loop (the index is one that the compiler cannot know)
            float4 runs[F32 ? 1 : HD / 8 + 1];
            auto run_at = [&]() -> float4 * {
                int zero = 0;
                if constexpr (!F32) asm volatile("" : "+r"(zero));
                return runs + zero;
            };
            auto run_factor = [&](const float4 *rs) { return rs[HD / 8].x == -INFINITY ? 0.0f : ex2(rs[HD / 8].x - wref); };
            auto add_o = [&] {
#pragma unroll
                for (int c = 0; c < (F32 ? HD / 2 : 0); c += 16) {
                    uint32_t hi[16], lo[16];
                    tmem_ldc(to + half * (HD / 2) + c, hi);
                    tmem_ldc(to + HD + half * (HD / 2) + c, lo);
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        o[c + i] = __fmaf_rn(o[c + i], fo, __fmaf_rn(__uint_as_float(lo[i]), 0x1p-11f, __uint_as_float(hi[i])));
                }
            };
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < HD / 2; i++) o[i] = 0.0f;
            }
            // columns of a round of these loops: as many as the registers take (18k chunk without cap: 16 columns 702 us, 32 676)
            constexpr int CK = IMG && !F32 ? 32 : 16;
            int j = 0, j_end = F32 ? n : min(n, RUN);
            for (;;) {
#pragma unroll 1
                for (; ok && j < j_end; j++) {
                    const int t0 = tile_at(j), mb = j & (META - 1);
                    const int sb = F32 ? j & 1 : w;                     // buffer of S
                    const uint32_t ts = tmem + lanes + sb * TK;
                    ok = mbar_wait_warp(&sm.meta_full[mb], (j / META) & 1, &sm.abort) && mbar_wait_warp(&sm.s_full[sb], F32 ? (j >> 1) & 1 : j & 1, &sm.abort);
                    if (!ok) break;
                    tc_after();
                    const float *ks = sm.m[mb].ks, *vs = sm.m[mb].vs, *lv = sm.m[mb].lv;
                    // every key of the tile is seen by every row of the CTA
                    const bool open = lists ? *reinterpret_cast<const uint32_t *>(sm.seen[mb]) == 0x01010101u
                                            : t0 + TK <= q.L && (!a.causal || t0 + TK - 1 <= pmin) && (!a.window || pmax - t0 < a.window);
                    // one scale for 8 keys, none of them extreme: the scales come in per group
                    const bool grp = a.c.lb >= 3 && *reinterpret_cast<const uint32_t *>(sm.tame[mb]) == 0x01010101u;
                    const bool rawS = open && grp && !(SHAPED && (a.softcap > 0.0f || a.slopes));
                    // Without tables a row sees the columns below c_pre and those in [c_lo, c_hi).
                    const int c_hi = min(a.causal ? (qp >= t0 + TK ? TK : qp + 1 - t0) : TK, q.L - t0);
                    const int c_lo = a.window ? (int)max((int64_t)qp - a.window + 1 - t0, (int64_t)0) : 0;
                    const int c_pre = min(pre - t0, q.L - t0);
                    float m0 = -INFINITY;
                    uint32_t xa[CK];
                    if (rawS) {
#pragma unroll 1
                        for (int c = k0; c < k0 + HC; c += CK) {
                            tmem_ldc(ts + c, xa);
#pragma unroll
                            for (int g = 0; g < CK; g += 8) {
                                float y = __uint_as_float(xa[g]), y1 = __uint_as_float(xa[g + 1]);
#pragma unroll
                                for (int i = 2; i < 8; i += 2) {
                                    y = fmaxf(y, __uint_as_float(xa[g + i]));
                                    y1 = fmaxf(y1, __uint_as_float(xa[g + i + 1]));
                                }
                                m0 = fmaxf(m0, __fmaf_rn(fmaxf(y, y1), ks[c + g] * qs2, lv[c + g]));
                            }
                        }
                    } else if (grp) {
                        // scores in log2 units, masked ones -inf, written back over S
#pragma unroll 1
                        for (int c = k0; c < k0 + HC; c += CK) {
                            // (the flags are made to look new in every round: the compiler would copy the loop for each of them)
                            int cap = SHAPED && a.softcap > 0.0f, ali = SHAPED && a.slopes, by_pos = SHAPED && a.c.pos, by_doc = SHAPED && docs, shut = !open;
                            if constexpr (SHAPED) asm volatile("" : "+r"(cap), "+r"(ali), "+r"(by_pos), "+r"(by_doc), "+r"(shut));
                            tmem_ldc(ts + c, xa);
                            float z[CK];
#pragma unroll
                            for (int g = 0; g < CK; g += 8) {
                                const float k = ks[c + g] * mul;
#pragma unroll
                                for (int i = 0; i < 8; i += 2) upk(mul2(pku(xa[g + i], xa[g + i + 1]), pk(k, k)), z[g + i], z[g + i + 1]);
                            }
                            if (cap) {
                                float big = 0.0f;
#pragma unroll
                                for (int i = 0; i < CK; i++) big = fmaxf(big, fabsf(z[i]));
                                if (__all_sync(0xFFFFFFFFu, big < TANH_X)) {   // (a NaN may pass: the polynomial keeps it)
                                    const f2 cl = pk(capl, capl);
#pragma unroll
                                    for (int i = 0; i < CK; i += 2) {
                                        const f2 y = pk(z[i], z[i + 1]), y2 = mul2(y, y);
                                        f2 r = pk(TANH_C[5], TANH_C[5]);
#pragma unroll
                                        for (int k = 4; k >= 0; k--) r = fma2(r, y2, pk(TANH_C[k], TANH_C[k]));
                                        upk(mul2(mul2(r, y), cl), z[i], z[i + 1]);
                                    }
                                } else {   // tanh(y) = 1 - 2 / (e^2y + 1)
#pragma unroll
                                    for (int i = 0; i < CK; i++) z[i] = cap_exp(z[i], capl);
                                }
                            }
                            if (ali) {
                                if (by_pos) {
#pragma unroll
                                    for (int i = 0; i < CK; i++) z[i] = __fmaf_rn(-slope, fabsf((float)(qp - sm.m[mb].pos[c + i])), z[i]);
                                } else {
                                    const float far = (float)(qp - t0 - c);
#pragma unroll
                                    for (int i = 0; i < CK; i++) z[i] = __fmaf_rn(-slope, fabsf(far - (float)i), z[i]);
                                }
                            }
                            if (shut) {
                                const int lo = c_lo - c, hi = c_hi - c, pr = c_pre - c;
                                if (by_pos) {
#pragma unroll
                                    for (int i = 0; i < CK; i++) {
                                        const int kp = sm.m[mb].pos[c + i];
                                        const bool see = kp < pre || ((!a.causal || kp <= qp) && (!a.window || qp - kp < a.window));
                                        z[i] = see && t0 + c + i < q.L ? z[i] : -INFINITY;
                                    }
                                } else {
#pragma unroll
                                    for (int i = 0; i < CK; i++) z[i] = (i >= lo && i < hi) || i < pr ? z[i] : -INFINITY;
                                }
                                if (by_doc) {
#pragma unroll
                                    for (int i = 0; i < CK; i += 4) {
                                        const int4 d = *reinterpret_cast<const int4 *>(&sm.m[mb].doc[c + i]);
                                        z[i] = d.x == qd ? z[i] : -INFINITY;
                                        z[i + 1] = d.y == qd ? z[i + 1] : -INFINITY;
                                        z[i + 2] = d.z == qd ? z[i + 2] : -INFINITY;
                                        z[i + 3] = d.w == qd ? z[i + 3] : -INFINITY;
                                    }
                                }
                            }
#pragma unroll
                            for (int g = 0; g < CK; g += 8) {
                                const float y = fmaxf(fmaxf(z[g], z[g + 1]), z[g + 2]), y1 = fmaxf(fmaxf(z[g + 3], z[g + 4]), z[g + 5]);
                                m0 = fmaxf(m0, fmaxf(fmaxf(fmaxf(y, y1), z[g + 6]), z[g + 7]) + lv[c + g]);
                            }
#pragma unroll
                            for (int i = 0; i < CK; i++) xa[i] = __float_as_uint(z[i]);
                            tmem_stc(ts + c, xa);
                        }
                        tmem_wait_st();
                    } else {
                        // scales of single keys: the same, four columns a round
#pragma unroll 1
                        for (int c = k0; c < k0 + HC; c += 4) {
                            uint32_t x[4];
                            tmem_ld4(ts + c, x);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int col = c + i, t = t0 + col, kp = SHAPED && a.c.pos ? sm.m[mb].pos[col] : t;
                                float z = __uint_as_float(x[i]) * (ks[col] * mul);
                                if (SHAPED && a.softcap > 0.0f) z = cap_exp(z, capl);
                                if (SHAPED && a.slopes) z = __fmaf_rn(-slope, fabsf((float)(qp - kp)), z);
                                bool see = kp < pre || ((!a.causal || kp <= qp) && (!a.window || qp - kp < a.window));
                                see = see && t < q.L && (!(SHAPED && docs) || sm.m[mb].doc[col] == qd);
                                z = see ? z : -INFINITY;
                                m0 = fmaxf(m0, z + lv[col]);
                                x[i] = __float_as_uint(z);
                            }
                            tmem_st4(ts + c, x);
                        }
                        tmem_wait_st();
                    }
                    // The other half's maximum: both threads of a row go by the same reference. 16-bit queries: this tile's
                    // scores came after the last tile's weights of all threads, so the entries of that tile have been read.
                    // f32 ones: S of this tile may have come before; two buffers in turn, and x_full of the tile between
                    // says that they have.
                    const int pb = F32 ? j & 1 : w;
                    sm.part[pb][half][r] = m0;
                    mbar_arrive(&sm.x_full[w]);
                    ok = mbar_wait_warp(&sm.x_full[w], j & 1, &sm.abort);
                    if (!ok) break;
                    m0 = fmaxf(m0, sm.part[pb][half ^ 1][r]);
                    const bool grow = m0 > wref + GROW;
                    float fnew = 1.0f;
                    if (__any_sync(0xFFFFFFFFu, grow)) {
                        const float f = grow && wref != -INFINITY ? ex2(wref - m0) : 1.0f;
                        if (grow) wref = m0;
                        lsum *= f;
                        fnew = f;
                        if (!F32 && j > 0) {
#pragma unroll 1
                            for (int c = half * (HD / 2); c < (half + 1) * (HD / 2); c += CK) {
                                tmem_ldc(to + c, xa);
#pragma unroll
                                for (int i = 0; i < CK; i++) xa[i] = __float_as_uint(__uint_as_float(xa[i]) * f);
                                tmem_stc(to + c, xa);
                            }
                            tmem_wait_st();
                        }
                    }
                    const float sub = wref == -INFINITY ? 0.0f : TOP - wref;
                    if (grp) {
                        // p * v_scale = 2^(score + sub + log2 v_scale); the group's sum over v_scale is the sum of its p
#pragma unroll 1
                        for (int c = k0; c < k0 + HC; c += CK) {
                            uint32_t p[CK / 2];
                            tmem_ldc(ts + c, xa);
#pragma unroll
                            for (int g = 0; g < CK; g += 8) {
                                const float k = rawS ? ks[c + g] * qs2 : 1.0f, off = sub + lv[c + g];
                                const f2 k2 = pk(k, k), o2 = pk(off, off);
                                float y[8];
#pragma unroll
                                for (int i = 0; i < 8; i += 2) {
                                    upk(fma2(pku(xa[g + i], xa[g + i + 1]), k2, o2), y[i], y[i + 1]);
                                    y[i] = ex2(y[i]), y[i + 1] = ex2(y[i + 1]);
                                    p[(g + i) / 2] = pack_f16(y[i], y[i + 1]);
                                    if constexpr (F32) xa[(g + i) / 2] = rest_f16(y[i], y[i + 1], p[(g + i) / 2], 0x1p11f);
                                }
                                float u0, u1;
                                upk(add2(add2(pk(y[0], y[1]), pk(y[2], y[3])), add2(pk(y[4], y[5]), pk(y[6], y[7]))), u0, u1);
                                lsum = __fmaf_rn(u0 + u1, sm.m[mb].rv[c + g], lsum);
                            }
                            if constexpr (F32) {   // high parts and remainders of 16 keys over their 16 scores
                                tmem_stc(ts + c, p);
#pragma unroll
                                for (int i = 0; i < CK / 2; i++) p[i] = xa[i];
                                tmem_stc(ts + c + 8, p);
                            } else {
                                tmem_stc(ts + (c + k0) / 2, p);   // columns whose scores are read already
                                if (c == k0 + HC / 2 - CK) {        // the first half of these weights: their product can start
                                    tmem_wait_st();
                                    tc_before();
                                    mbar_arrive(&sm.p_half[w]);
                                }
                            }
                        }
                    } else if constexpr (F32) {
#pragma unroll 1
                        for (int c = k0; c < k0 + HC; c += CK) {
                            uint32_t p[CK / 2];
                            tmem_ldc(ts + c, xa);
#pragma unroll
                            for (int i = 0; i < CK; i += 2) {
                                const float y0 = __uint_as_float(xa[i]), y1 = __uint_as_float(xa[i + 1]), e0 = ex2(y0 + sub), e1 = ex2(y1 + sub);
                                lsum += e0 + e1;
                                const float u0 = y0 == -INFINITY ? 0.0f : e0 * vs[c + i], u1 = y1 == -INFINITY ? 0.0f : e1 * vs[c + i + 1];
                                p[i / 2] = pack_f16(u0, u1);
                                xa[i / 2] = rest_f16(u0, u1, p[i / 2], 0x1p11f);
                            }
                            tmem_stc(ts + c, p);
#pragma unroll
                            for (int i = 0; i < CK / 2; i++) p[i] = xa[i];
                            tmem_stc(ts + c + 8, p);
                        }
                    } else {
#pragma unroll 1
                        for (int c = k0; c < k0 + HC; c += 4) {
                            uint32_t x[4], p[2];
                            tmem_ld4(ts + c, x);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const float y = __uint_as_float(x[i]), e = ex2(y + sub);
                                lsum += e;
                                // a masked key's scale has no part in this, whatever it is
                                x[i] = __float_as_uint(y == -INFINITY ? 0.0f : e * vs[c + i]);
                            }
                            p[0] = pack_f16(__uint_as_float(x[0]), __uint_as_float(x[1]));
                            p[1] = pack_f16(__uint_as_float(x[2]), __uint_as_float(x[3]));
                            tmem_st2(ts + (c + k0) / 2, p);
                        }
                        tmem_wait_st();
                        tc_before();
                        mbar_arrive(&sm.p_half[w]);
                    }
                    tmem_wait_st();
                    if constexpr (F32) {   // the last tile's product: the next one starts over it
                        if (j > 0) {
                            ok = mbar_wait_warp(&sm.o_full[0], (j - 1) & 1, &sm.abort);
                            if (!ok) break;
                            tc_after();
                            add_o();
                        }
                        fo = fnew;
                    }
                    tc_before();
                    mbar_arrive(&sm.p_full[w]);
                }
                if (F32 || !ok || j_end == n) break;
                // a run ends, and more are to come: its products join the sum, and the next one starts O from zero
                ok = mbar_wait_warp(&sm.o_full[w], (j / RUN - 1) & 1, &sm.abort);
                if (!ok) break;
                tc_after();
                float4 *rs = run_at();
                const float f = j > RUN ? run_factor(rs) : 0.0f;
#pragma unroll 1
                for (int c = 0; c < HD / 2; c += 16) {
                    uint32_t x[16];
                    tmem_ldc(to + half * (HD / 2) + c, x);
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        float4 &v = rs[(c + i) / 4];
                        const float4 u = j > RUN ? v : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        v = make_float4(__fmaf_rn(u.x, f, __uint_as_float(x[i])), __fmaf_rn(u.y, f, __uint_as_float(x[i + 1])),
                                        __fmaf_rn(u.z, f, __uint_as_float(x[i + 2])), __fmaf_rn(u.w, f, __uint_as_float(x[i + 3])));
                    }
                }
                rs[HD / 8].x = wref;
                j_end = min(n, j_end + RUN);
            }
            float l = 0.0f;
            if (ok && n > 0) {
                sm.sums[w][half][r] = lsum;
                mbar_arrive(&sm.x_full[w]);
                ok = mbar_wait_warp(&sm.x_full[w], n & 1, &sm.abort) && mbar_wait_warp(&sm.o_full[w], (F32 ? n - 1 : (n - 1) / RUN) & 1, &sm.abort);
                l = lsum + sm.sums[w][half ^ 1][r];
            }
            tc_after();
            const bool part = it.pieces > 1;     // the sums go to the workspace, for the join
            const float inv = !ok ? __uint_as_float(0x7FC00000u) : part ? unit : l == 0.0f ? 0.0f : __fdiv_rn(unit, l);
            const size_t prow = part ? ((size_t)(blockIdx.x - a.n_full) * RPC + w * TQ + r) : 0;
            // The warp's 32 half rows go through its share of the queries' buffer (their products are done), 16-byte chunks
            // crossed so that neither side meets a bank twice, and out in whole lines: one row a lane, as they lie in TMEM,
            // took 4,500 clocks a CTA.
            constexpr int CH = HD / 2 * (int)sizeof(QT) / 16;
            auto cross = [](int row) { return CH == 4 ? (row >> 1) & 3 : row & 7; };
            uint8_t *stage = sm.q[F32 ? 0 : w] + (warp & 7) * (32 * CH * 16);
            auto put = [&](int ch, uint4 v) { *reinterpret_cast<uint4 *>(stage + lane * CH * 16 + ((ch ^ cross(lane)) * 16)) = v; };
            if constexpr (F32) {
                if (ok && n > 0) add_o();
#pragma unroll
                for (int i = 0; i < HD / 2; i += 4) {
                    const float4 v = make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv);
                    put(i / 4, *reinterpret_cast<const uint4 *>(&v));
                }
            }
#pragma unroll 1
            for (int c = half * (HD / 2); !F32 && c < (half + 1) * (HD / 2); c += 32) {
                uint32_t x[32];
                if (ok && n > 0) {
                    tmem_ld32(to + c, x);
                    if (n > RUN) {
                        const float4 *rs = run_at();
                        const float f = run_factor(rs);
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 u = rs[(c - half * (HD / 2) + i) / 4];
                            x[i] = __float_as_uint(__fmaf_rn(u.x, f, __uint_as_float(x[i])));
                            x[i + 1] = __float_as_uint(__fmaf_rn(u.y, f, __uint_as_float(x[i + 1])));
                            x[i + 2] = __float_as_uint(__fmaf_rn(u.z, f, __uint_as_float(x[i + 2])));
                            x[i + 3] = __float_as_uint(__fmaf_rn(u.w, f, __uint_as_float(x[i + 3])));
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) x[i] = 0;
                }
                if (part) {
                    if (live)
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            kv8_st4(a.po + prow * HD + c + i, make_float4(__uint_as_float(x[i]) * inv, __uint_as_float(x[i + 1]) * inv,
                                                                          __uint_as_float(x[i + 2]) * inv, __uint_as_float(x[i + 3]) * inv));
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint4 o;
                        kv8_st4(reinterpret_cast<QT *>(&o), make_float4(__uint_as_float(x[i]) * inv, __uint_as_float(x[i + 1]) * inv,
                                                                        __uint_as_float(x[i + 2]) * inv, __uint_as_float(x[i + 3]) * inv));
                        kv8_st4(reinterpret_cast<QT *>(&o) + 4, make_float4(__uint_as_float(x[i + 4]) * inv, __uint_as_float(x[i + 5]) * inv,
                                                                            __uint_as_float(x[i + 6]) * inv, __uint_as_float(x[i + 7]) * inv));
                        put((c - half * (HD / 2) + i) / 8, o);
                    }
                }
            }
            if (F32 || !part) {
                __syncwarp();
                QT *to_rows = F32 && part ? reinterpret_cast<QT *>(a.po) : out;
                const long long my = !live ? -1 : F32 && part ? (long long)prow : (long long)orow;
#pragma unroll 4
                for (int i = 0; i < CH; i++) {
                    const int row = (32 * i + lane) / CH, ch = (32 * i + lane) % CH;
                    const long long at = __shfl_sync(0xFFFFFFFFu, my, row);
                    const uint4 v = *reinterpret_cast<const uint4 *>(stage + row * CH * 16 + ((ch ^ cross(row)) * 16));
                    if (at >= 0) *reinterpret_cast<uint4 *>(to_rows + at * HD + half * (HD / 2) + ch * (16 / (int)sizeof(QT))) = v;
                }
            }
            if (live && half == 0 && part) {
                a.pm[prow] = wref;
                a.pl[prow] = ok ? l : __uint_as_float(0x7FC00000u);
            } else if (live && half == 0 && a.lse)
                a.lse[orow] = !ok ? __uint_as_float(0x7FC00000u) : l == 0.0f ? -INFINITY : (log2f(l) - (wref == -INFINITY ? 0.0f : TOP - wref)) * LN2;
        }
    } else if (!IMG && warp < MW) {
        // ---- codes to f16 ----
        regs_down<RL::REGS_CONVERT>();
        const int c = tid - 32 * SW;
        const bool is_v = c >= CV / 2;            // half of the warps convert K, half V: the same code
        const int h = c & (CV / 2 - 1);
        const int prow = (h & 7) + 8 * (h / (8 * PC)), piece = (h >> 3) % PC;   // first row and piece of this thread
        constexpr int RSTEP = 8 * (CV / 2 / (8 * PC));                             // its next row
        const uint8_t *pool = is_v ? a.c.v : a.c.k;
        uint8_t *dst0 = (is_v ? sm.v[0] : sm.k[0]) + (prow >> 3) * SBO + piece * 256 + (prow & 7) * 16;
        uint64_t *full = is_v ? sm.v_full : sm.k_full, *empty = is_v ? sm.v_empty : sm.k_empty;
        const int32_t *table = a.b.page_table + (size_t)s * a.b.table_stride;
        const float nan = __uint_as_float(0x7FC00000u);
        uint4 xa[NP], xb[NP];
        int32_t te = -1, te_next = -1;
        auto entry = [&](int j) {
            if (j >= n || !is_v) return -1;
            const int t = tile_at(j) + h;
            return t < q.L ? __ldg(table + (t >> a.c.lp)) : -1;
        };
        float mk = 0.0f, mv = 0.0f;
        int mp = 0, md = -1;
        auto rows_of = [&](int j, int32_t e) {   // row numbers of tile j; its scales into registers
            if (!is_v) return;   // (V's threads: what they wait for covers the last use of a buffer of scales)
            const int t = tile_at(j) + h;
            const bool have = t < q.L && a.c.ok(e);
            const uint32_t rid = have ? a.c.row(e, kvh, t) : 0xFFFFFFFFu;
            sm.row[j & 1][h] = rid;
            const float none = t < q.L ? nan : 1.0f;   // a bad page: NaN for whoever sees it
            mk = have ? __ldg(a.c.ks + (rid >> a.c.lb)) : none;
            mv = have ? __ldg(a.c.vs + (rid >> a.c.lb)) : none;
            if (a.c.pos) mp = have ? __ldg(a.c.pos + rid) : 0;
            if (docs) {
                const int p = a.c.pos ? mp : t;
                md = p >= 0 && p < a.doc_stride ? __ldg(docs + p) : -1;
            }
        };
        auto put_meta = [&](int j) {
            if (!is_v) return;
            const int mb = j & (META - 1);
            sm.m[mb].ks[h] = mk;
            sm.m[mb].vs[h] = mv;
            sm.m[mb].lv[h] = fmaxf(log2f(mv), -60.0f);
            sm.m[mb].rv[h] = __frcp_rn(mv);
            const bool tame = __all_sync(0xFFFFFFFFu, mv > 0x1p-60f && mv < 0x1p60f);
            if (lane == 0) sm.tame[mb][warp - SW - 4] = tame;
            if constexpr (SHAPED) {
                if (a.c.pos || docs) {
                    const int t = tile_at(j) + h, p = a.c.pos ? mp : t;
                    bool see = t < q.L && (!a.causal || p <= pmin) && (!a.window || (int64_t)pmax - p < a.window);
                    see = see && (!docs || (sm.dmin == md && sm.dmax == md));
                    see = __all_sync(0xFFFFFFFFu, see);
                    if (lane == 0) sm.seen[mb][warp - SW - 4] = see;
                    sm.m[mb].pos[h] = mp;
                    sm.m[mb].doc[h] = md;
                }
            }
            mbar_arrive(&sm.meta_full[mb]);
        };
        auto load = [&](int j, int i0, uint4 (&x)[NP]) {   // pieces i0 .. i0 + NP - 1 of the thread
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const uint32_t rid = sm.row[j & 1][prow + RSTEP * (i0 + i)];
                x[i] = rid != 0xFFFFFFFFu ? __ldg(reinterpret_cast<const uint4 *>(pool + (size_t)rid * HD + 16 * piece)) : make_uint4(0, 0, 0, 0);
            }
        };
        auto convert = [&](int j, int i0, const uint4 (&x)[NP]) {
            uint8_t *d = dst0 + (j & 1) * (TK * HD * 2) + i0 * (RSTEP / 8) * SBO;
#pragma unroll
            for (int i = 0; i < NP; i++, d += RSTEP / 8 * SBO) {
                const uint32_t b0 = kv8_bias<FMT>(x[i].x), b1 = kv8_bias<FMT>(x[i].y), b2 = kv8_bias<FMT>(x[i].z), b3 = kv8_bias<FMT>(x[i].w);
                *reinterpret_cast<uint4 *>(d) = make_uint4(kv8_half2<FMT, 0>(b0), kv8_half2<FMT, 1>(b0), kv8_half2<FMT, 0>(b1), kv8_half2<FMT, 1>(b1));
                *reinterpret_cast<uint4 *>(d + 128) = make_uint4(kv8_half2<FMT, 0>(b2), kv8_half2<FMT, 1>(b2), kv8_half2<FMT, 0>(b3), kv8_half2<FMT, 1>(b3));
            }
        };
        auto bar = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
        bool ok = true;
        if (n > 0) {
            rows_of(0, entry(0));
            te = entry(1);
            bar();
            load(0, 0, xa);
            load(0, NP, xb);
            put_meta(0);
        }
#pragma unroll 1
        for (int j = 0; j < n; j++) {
            te_next = entry(j + 2);
            // row numbers of the next tile while this one waits for its buffer
            if (j + 1 < n) rows_of(j + 1, te);
            te = te_next;
            bar();
            // after a wait that ran out the thread goes on to the barriers, without work
            if (j >= 2) ok = mbar_wait_warp(&empty[j & 1], ((j >> 1) - 1) & 1, &sm.abort) && ok;
            if (ok) {
                convert(j, 0, xa);
                convert(j, NP, xb);
                fence_async_smem();
                mbar_arrive(&full[j & 1]);
                if (j + 1 < n) {
                    load(j + 1, 0, xa);
                    load(j + 1, NP, xb);
                    put_meta(j + 1);
                }
            }
        }
    } else {
        // ---- MMAs ----
        regs_down<RL::REGS_MMA>();
        if (warp == MW) {
            // One warp for both query tiles: with a warp each the tiles' phases drift together, and the tensor core and the
            // softmax warps wait for each other in turn (18k chunk without cap 902 us, in turn 739).
            constexpr uint32_t id_qk = idesc(TK, false), id_pv = idesc(HD, true);
            const uint32_t lead = lane == 0, tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
            const int nt = __shfl_sync(0xFFFFFFFFu, n, 0), nw = __shfl_sync(0xFFFFFFFFu, two ? 2 : 1, 0);
            // operand descriptors of the first step; a step further is a constant added to the start address (16-byte units)
            const uint64_t dq = umma_desc(saddr(sm.q[0]), 128, SBO), dk = umma_desc(saddr(sm.k[0]), 128, SBO),
                           dv = umma_desc(saddr(sm.v[0]), SBO, 128);
            constexpr int BUF = TK * HD * 2 / 16;   // from a first buffer to its second
            auto qk = [&](int w, int j) {
                const uint64_t qa = dq + w * BUF, ka = dk + (j & 1) * BUF;
                const int sb = F32 ? j & 1 : w;
#pragma unroll
                for (int k = 0; k < HD / 16; k++) umma_ss(tm + sb * TK, qa + 16 * k, ka + 16 * k, id_qk, k > 0, lead);
                if constexpr (F32) {
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) umma_ss(tm + sb * TK, qa + BUF + 16 * k, ka + 16 * k, id_qk, 1, lead);
                }
                umma_commit(&sm.s_full[sb], lead);
            };
            auto pv = [&](int w, int j, int part) {
                const uint64_t va = dv + (j & 1) * BUF;
                if constexpr (F32) {
#pragma unroll
                    for (int part = 0; part < 2; part++)
#pragma unroll
                        for (int k = 0; k < TK / 16; k++)
                            umma_ts(tm + 2 * TK + part * HD, tm + (j & 1) * TK + 16 * k + 8 * part, va + 2 * SBO / 16 * k, id_pv, k > 0, lead);
                } else {
#pragma unroll
                    for (int i = 0; i < TK / 32; i++) {
                        const int k = (i & 1) + (i & 2) * 2, kk = k + 2 * part;
                        umma_ts(tm + 2 * TK + w * HD, tm + w * TK + 8 * kk + (k >= HC / 16 ? HC / 2 : 0), va + 2 * SBO / 16 * kk, id_pv, (j & (RUN - 1)) != 0 || part > 0 || i > 0, lead);
                    }
                }
            };
            bool ok = nt == 0 || (mbar_wait(&sm.q_full, 0, &sm.abort) && mbar_wait(&sm.k_full[0], 0, &sm.abort));
            if (ok && nt > 0) {
                tc_after();
                for (int w = 0; w < nw; w++) qk(w, 0);
                umma_commit(&sm.k_empty[0], lead);
            }
            if constexpr (F32) {
#pragma unroll 1
                for (int j = 0; ok && j < nt; j++) {
                    if (j + 1 < nt) {
                        ok = mbar_wait(&sm.k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, &sm.abort);
                        if (!ok) break;
                        tc_after();
                        qk(0, j + 1);
                        umma_commit(&sm.k_empty[(j + 1) & 1], lead);
                    }
                    ok = mbar_wait(&sm.p_full[0], j & 1, &sm.abort) && mbar_wait(&sm.v_full[j & 1], (j >> 1) & 1, &sm.abort);
                    if (!ok) break;
                    tc_after();
                    pv(0, j, 0);
                    umma_commit(&sm.o_full[0], lead);
                    umma_commit(&sm.v_empty[j & 1], lead);
                }
            }
#pragma unroll 1
            for (int j = 0; !F32 && ok && j < nt; j++) {
                // V of this tile and K of the next are there long before the weights: those waits come first, once
                ok = mbar_wait(&sm.v_full[j & 1], (j >> 1) & 1, &sm.abort) &&
                     (j + 1 == nt || mbar_wait(&sm.k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, &sm.abort));
#pragma unroll 1
                for (int w = 0; ok && w < nw; w++) {
                    ok = mbar_wait(&sm.p_half[w], j & 1, &sm.abort);
                    if (!ok) break;
                    tc_after();
                    pv(w, j, 0);
                    ok = mbar_wait(&sm.p_full[w], j & 1, &sm.abort);
                    if (!ok) break;
                    tc_after();
                    pv(w, j, 1);
                    if (w == nw - 1) umma_commit(&sm.v_empty[j & 1], lead);
                    if (j + 1 == nt || ((j + 1) & (RUN - 1)) == 0) umma_commit(&sm.o_full[w], lead);
                    if (j + 1 < nt) {
                        qk(w, j + 1);
                        if (w == nw - 1) umma_commit(&sm.k_empty[(j + 1) & 1], lead);
                    }
                }
            }
            // nothing may be in flight when the TMEM goes
            umma_commit(&sm.drain, lead);
            mbar_wait(&sm.drain, 0, nullptr);
        } else if (IMG && warp == MW + 1 && lane == 0) {
            // ---- tile images to shared memory ----
            const uint8_t *img = a.img + slot * IMAGE<HD>;
            constexpr uint32_t HALF = TK * HD * 2;
            const uint32_t meta_bytes = SHAPED ? sizeof(Meta) : 4 * TK * 4;
            auto meta = [&](int j) {
                const int t0 = tile_at(j), v = t0 / TK, mb = j & (META - 1);
                const Kv8Head x = heads[v];
                *reinterpret_cast<uint32_t *>(sm.tame[mb]) = x.tame ? 0x01010101u : 0u;
                if (SHAPED && (docs || a.c.pos)) {
                    const bool see = t0 + TK <= q.L && (!a.causal || x.pmax <= pmin) && (!a.window || (int64_t)pmax - x.pmin < a.window) &&
                                     (!docs || (sm.dmin == x.dmin && sm.dmax == x.dmin && x.dmax == x.dmin));
                    *reinterpret_cast<uint32_t *>(sm.seen[mb]) = see ? 0x01010101u : 0u;
                }
                mbar_expect(&sm.meta_full[mb], meta_bytes);
                bulk_load(&sm.m[mb], img + (size_t)v * IMAGE<HD> + 2 * HALF, meta_bytes, &sm.meta_full[mb]);
            };
            if (n > 0) meta(0);
            if (n > 1) meta(1);
            bool ok = true;
            int j = 0;
#pragma unroll 1
            for (; j < n; j++) {
                const int b = j & 1;
                const uint8_t *src = img + (size_t)(tile_at(j) / TK) * IMAGE<HD>;
                if (j >= 2) ok = mbar_wait(&sm.k_empty[b], ((j >> 1) - 1) & 1, &sm.abort);
                if (!ok) break;
                mbar_expect(&sm.k_full[b], HALF);
                bulk_load(sm.k[b], src, HALF, &sm.k_full[b]);
                if (j >= 2) ok = mbar_wait(&sm.v_empty[b], ((j >> 1) - 1) & 1, &sm.abort);
                if (!ok) break;
                mbar_expect(&sm.v_full[b], HALF);
                bulk_load(sm.v[b], src + HALF, HALF, &sm.v_full[b]);
                // PV of tile j - 2 is done: its scales' buffer is free
                if (j + 2 < n) meta(j + 2);
            }
            if (!ok) {   // nothing may be in flight when the shared memory goes
                for (int i = max(j - 2, 0); i <= j; i++) {
                    mbar_wait(&sm.k_full[i & 1], (i >> 1) & 1, nullptr);
                    if (i < j) mbar_wait(&sm.v_full[i & 1], (i >> 1) & 1, nullptr);
                }
                for (int i = max(j - 2, 0); i < min(j + 2, n); i++) mbar_wait(&sm.meta_full[i & (META - 1)], (i / META) & 1, nullptr);
            }
        }
    }
    __syncwarp();
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == MW) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// Key tiles of a sequence, and (sequence, KV head) pairs whose images one launch holds; 0 pairs: converting warps. Images
// pay from IMG_TILES query tiles on (131,072 rows, 1 / 2 / 4 / 8 tiles a head: 190 / 245 / 368 / 637 us with them, 153 /
// 244 / 430 / 841 without). Above IMG_BYTES the pairs go in turns, each of which has to fill the SMs twice.
constexpr int IMG_TILES = 3;
constexpr size_t IMG_BYTES = (size_t)512 << 20;
struct Images {
    int n_img, n_seq, n_kv;   // sequences and KV heads of a launch
    size_t bytes;
};
Images images(const tlmg_kv8 &c, const tlmg_kv8_batch &b, int H, int q_dt) {
    Images r{};
    const int64_t rows = q_dt == TLMG_DT_F32 ? TQ : 2 * TQ, tiles = ((int64_t)b.max_q * (H / c.KV) + rows - 1) / rows;
    if (tiles < IMG_TILES) return r;
    r.n_img = (b.max_kv + TK - 1) / TK;
    const size_t one = (size_t)r.n_img * ((c.hd == 64 ? IMAGE<64> : IMAGE<128>) + sizeof(Kv8Head));
    const int64_t fit = std::max<int64_t>(1, (int64_t)(IMG_BYTES / std::max<size_t>(one, 1)));
    if (fit >= c.KV) r.n_kv = c.KV, r.n_seq = (int)std::min<int64_t>(b.n_seq, fit / c.KV);
    else r.n_kv = (int)fit, r.n_seq = 1;
    const bool all = r.n_kv == c.KV && r.n_seq == b.n_seq;
    if (!all && r.n_kv * r.n_seq * tiles < 2 * sm_count()) return Images{};
    r.bytes = (size_t)r.n_kv * r.n_seq * one;
    return r;
}

// Items on the SMs: whole rounds of them as they are, the rest (all of them where they leave SMs idle) cut along the keys
// into pieces of PIECE tiles or more. In units of a tile's time (2.4 us) a CTA's start and end cost about 5, the join 3 and
// what a piece writes and the join reads 1 / 50. Beyond ROUNDS rounds the last one is too small a part. Without and with
// pieces: 18k chunk (256 items, 108 of them in 4 pieces) 1,073 and 1,028 us, 65,536 rows 2,344 and 2,071, 32 tokens of 32
// heads on 4 over 131,072 rows (4 items in 37) 159 with.
constexpr int ROUNDS = 8, PIECE = 4;
struct Tail {
    int n_full, pieces, n_tail;
};
Tail tail_plan(const tlmg_kv8 &c, const tlmg_kv8_batch &b, bool causal, int window, int64_t items, int rows) {
    const int64_t sms = sm_count(), full = items / sms * sms, left = items - full;
    Tail r{ (int)items, 1, 0 };
    if (full > ROUNDS * sms || left == 0) return r;
    // key tiles of such an item: its tokens are among the first ones where whole rounds came before
    int64_t keys = b.max_kv;
    if (causal) keys = std::max<int64_t>(b.max_kv - b.max_q, 0) + (full ? b.max_q * left / items : b.max_q / 2);
    if (window > 0 && causal && !c.pos) keys = std::min<int64_t>(keys, (int64_t)window + rows);
    const int64_t kt = std::max<int64_t>(1, keys / TK);
    int64_t best = kt + 5;
    for (int64_t s = 2; s <= kt / PIECE && left * s <= 4 * sms; s++) {
        const int64_t cost = (left * s + sms - 1) / sms * ((kt + s - 1) / s + 5) + 3 + left * s / 50;
        if (cost < best) best = cost, r = { (int)full, (int)s, (int)left };
    }
    return r;
}

template <int HD, int FMT, typename QT, bool SHAPED, bool IMG> int launch_shape(const Kv8Attn &a, unsigned grid, cudaStream_t st) {
    auto fn = k_kv8_prefill<HD, FMT, QT, SHAPED, IMG>;
    constexpr size_t bytes = sizeof(Smem<HD>);
    static_assert(bytes <= 227 * 1024, "shared memory");
    if (!smem_opt_in((const void *)fn, bytes)) return set_error(TLMG_EIO, "kv8_attend: shared memory opt-in failed");
    fn<<<grid, Role<sizeof(QT) == 4, IMG>::THREADS, bytes, st>>>(a);
    count_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? TLMG_OK : cuda_fail(e, "kv8_attend launch");
}
// What a call does, from its sizes alone: workspace = images, then the pieces' outputs, references and sums.
struct Wide {
    Images im;
    Tail tail;
    int q_tiles;
    size_t part, bytes;   // rows of partial results
};
Wide wide_plan(const tlmg_kv8 &c, const tlmg_kv8_batch &b, int H, int q_dt, bool causal, int window) {
    Wide p;
    p.im = images(c, b, H, q_dt);
    const int rows = q_dt == TLMG_DT_F32 ? TQ : 2 * TQ;
    p.q_tiles = (int)(((int64_t)b.max_q * (H / c.KV) + rows - 1) / rows);
    const int64_t items = (int64_t)p.q_tiles * c.KV * b.n_seq;
    p.tail = Tail{ (int)std::min<int64_t>(items, INT32_MAX), 1, 0 };
    if (!p.im.n_kv || (p.im.n_kv == c.KV && p.im.n_seq == b.n_seq)) p.tail = tail_plan(c, b, causal, window, items, rows);
    p.part = (size_t)p.tail.n_tail * p.tail.pieces * rows;
    p.bytes = p.im.bytes + p.part * (c.hd + 2) * 4;
    return p;
}

template <int HD, int FMT, typename QT> int launch(const Kv8Attn &a0, void *work, cudaStream_t st) {
    Kv8Attn a = a0;
    const bool shaped = a.softcap > 0.0f || a.slopes || a.doc || a.c.pos;
    const Wide p = wide_plan(a.kv8, a.b, a.H, sizeof(QT) == 4 ? TLMG_DT_F32 : TLMG_DT_F16, a.causal, a.window);
    const Images &im = p.im;
    if ((int64_t)p.q_tiles * a.c.KV * a.b.n_seq > INT32_MAX)
        return set_error(TLMG_ERANGE, "kv8_attend: %d sequences of %d KV heads and %d tokens are too many for a call", a.b.n_seq, a.c.KV, a.b.max_q);
    a.q_tiles = p.q_tiles;
    a.pieces = p.tail.pieces;
    a.po = reinterpret_cast<float *>(static_cast<uint8_t *>(work) + im.bytes);
    a.pm = a.po + p.part * HD;
    a.pl = a.pm + p.part;
    a.s0 = a.kv0 = 0;
    int rc = TLMG_OK;
    if (!im.n_kv) {
        a.nkv = a.c.KV;
        a.n_full = p.tail.n_full;
        const unsigned grid = (unsigned)(a.n_full + p.tail.n_tail * a.pieces);
        rc = shaped ? launch_shape<HD, FMT, QT, true, false>(a, grid, st) : launch_shape<HD, FMT, QT, false, false>(a, grid, st);
    } else {
        a.unit = kv8_f16_unit<FMT>();
        a.n_img = im.n_img;
        a.img = static_cast<uint8_t *>(work);
        a.heads = a.img + (size_t)im.n_kv * im.n_seq * im.n_img * IMAGE<HD>;
        for (a.s0 = 0; !rc && a.s0 < a.b.n_seq; a.s0 += im.n_seq)
            for (a.kv0 = 0; !rc && a.kv0 < a.c.KV; a.kv0 += im.n_kv) {
                const int ns = std::min(im.n_seq, a.b.n_seq - a.s0);
                a.nkv = std::min(im.n_kv, a.c.KV - a.kv0);
                k_kv8_images<HD, FMT><<<dim3(im.n_img, a.nkv, ns), 256, 0, st>>>(a);
                count_launch();
                a.n_full = p.tail.n_tail ? p.tail.n_full : a.q_tiles * a.nkv * ns;
                const unsigned grid = (unsigned)(a.n_full + p.tail.n_tail * a.pieces);
                rc = shaped ? launch_shape<HD, TLMG_KV8_INT8, QT, true, true>(a, grid, st)
                            : launch_shape<HD, TLMG_KV8_INT8, QT, false, true>(a, grid, st);
            }
        a.s0 = a.kv0 = 0;
    }
    if (rc || !p.tail.n_tail) return rc;
    constexpr int rows = Role<sizeof(QT) == 4, true>::TILES * TQ;
    a.nkv = a.c.KV;
    k_kv8_pieces<HD, QT><<<p.tail.n_tail * (rows / 8), 256, 0, st>>>(a);
    count_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? TLMG_OK : cuda_fail(e, "kv8_attend launch");
}
template <int HD, int FMT> int launch_q(const Kv8Attn &a, int q_dt, void *work, cudaStream_t st) {
    if (q_dt == TLMG_DT_F32) return launch<HD, FMT, float>(a, work, st);
    return q_dt == TLMG_DT_F16 ? launch<HD, FMT, __half>(a, work, st) : launch<HD, FMT, __nv_bfloat16>(a, work, st);
}
template <int HD> int launch_fmt(const Kv8Attn &a, int q_dt, void *work, cudaStream_t st) {
    return a.kv8.fmt == TLMG_KV8_INT8 ? launch_q<HD, TLMG_KV8_INT8>(a, q_dt, work, st) : launch_q<HD, TLMG_KV8_E4M3>(a, q_dt, work, st);
}

}  // namespace

bool kv8_prefill_serves(const tlmg_kv8 &c, const tlmg_kv8_batch &b, int H) {
    // 32 heads on 4 of 128, a call as Python makes it: 16 tokens over 701 / 2,048 / 8,192 / 131,072 rows take 36 / 43 / 49 /
    // 135 us here and 20 / 25 / 40 / 318 us in the kernel for few rows; 32 tokens over 2,048 / 8,192 rows 51 / 57 and 32 / 64,
    // 64 tokens over 2,048 rows 51 and 45. The two meet where rows x keys x dims of all heads come to WIDE_WORK. Other
    // layouts (8 on 2, 64 on 4; dims 64 and 128; f32 and bf16; 701 .. 131,072 rows) meet between half of it and it for one
    // sequence: at 2/3 of it 34 .. 51 us here and 29 .. 43 there, at 4/3 39 .. 60 and 49 .. 76. Batches of short sequences
    // meet at a fourth of it (8 x 32 tokens over 701 rows, 32 on 4 of 128, 0.9 of it: 35 here, 70 there).
    constexpr int64_t WIDE_WORK = (int64_t)3 << 28;
    const int64_t rows = (int64_t)b.max_q * (H / c.KV);
    return c.hd <= 128 && rows >= TQ && (double)rows * c.KV * b.n_seq * b.max_kv * c.hd >= (double)WIDE_WORK;
}

size_t kv8_prefill_work_bytes(const tlmg_kv8 &c, const tlmg_kv8_batch &b, const tlmg_kv8_score &s, int H, int q_dt) {
    return wide_plan(c, b, H, q_dt, s.causal, s.window).bytes;
}

int kv8_prefill(const Kv8Attn &a, int q_dt, void *work, cudaStream_t st) {
    return a.c.hd == 64 ? launch_fmt<64>(a, q_dt, work, st) : launch_fmt<128>(a, q_dt, work, st);
}

}  // namespace tlmg
