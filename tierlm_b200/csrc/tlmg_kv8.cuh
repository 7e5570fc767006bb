// tlmg_kv8.cuh - the 8-bit KV cache: code formats and what its kernels share.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "../../include/tlmg.h"

namespace tlmg {

constexpr float KV8_FLOOR = 0x1p-100f;   // smallest amax a scale is made from: no division by zero, no subnormal scale

template <int FMT> __host__ __device__ constexpr float kv8_qmax() { return FMT == TLMG_KV8_INT8 ? 127.0f : 448.0f; }

// The value a code byte stands for (before the scale). The e4m3 pattern
// s eeee mmm, moved to the top of an f32's exponent and mantissa, is the
// value times 2^-120 (biases 7 and 127), subnormals included.
template <int FMT> __device__ __forceinline__ float kv8_value(uint32_t c) {
    if constexpr (FMT == TLMG_KV8_INT8) return (float)(int8_t)c;
    return __fmul_rn(__uint_as_float(((c & 0x80u) << 24) | ((c & 0x7Fu) << 20)), 0x1p120f);
}

// round-to-nearest-even code of y = x / d, |y| <= Q up to the division's rounding
template <int FMT> __device__ __forceinline__ uint32_t kv8_code(float y) {
    if constexpr (FMT == TLMG_KV8_INT8) return (uint32_t)__float2int_rn(y) & 0xFFu;
    return (uint32_t)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}

// Two code bytes of word w as f16x2. int8: the byte plus 128 in the
// low bits of 1024.0 (0x6400) is 1152 + code, less 1152 (exact). e4m3:
// exponent and mantissa moved into the f16 fields give the value times 2^-8
// (biases 7 and 15; f16 subnormals hold the small ones exactly), which the
// scale makes up for (kv8_f16_unit). Both are exact for every code, and no
// code, whatever a masked or unwritten row holds, becomes a NaN or infinity.
// kv8_cvt2 is the same for e4m3 by the conversion instruction: one instruction
// for four, at a fourth of their rate, the better bargain where issue slots are
// short (64 ragged sequences: 134 us with bit fields, 101 with it; the prefill's
// converting warps: 994 us and 1,051). The code that is no number, which
// nothing writes, stays one: clean = true makes it 448.
template <int FMT> constexpr float kv8_f16_unit() { return FMT == TLMG_KV8_INT8 ? 1.0f : 256.0f; }
template <int FMT> __device__ __forceinline__ uint32_t kv8_bias(uint32_t w) {
    return FMT == TLMG_KV8_INT8 ? w ^ 0x80808080u : w;
}
template <int FMT, int HI> __device__ __forceinline__ uint32_t kv8_half2(uint32_t w) {   // bytes 2 HI, 2 HI + 1 of a biased word
    if constexpr (FMT == TLMG_KV8_INT8) {
        const uint32_t h = __byte_perm(w, 0x64646464u, HI ? 0x4342 : 0x4140);
        const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&h), __half2half2(__ushort_as_half(0x6480)));
        return *reinterpret_cast<const uint32_t *>(&r);
    } else {
        const uint32_t h = __byte_perm(w, 0u, HI ? 0x3424 : 0x1404);
        return (h & 0x80008000u) | ((h >> 1) & 0x3F803F80u);
    }
}

template <int FMT> constexpr float kv8_cvt_unit() { return 1.0f; }
template <int FMT, int HI, bool clean> __device__ __forceinline__ uint32_t kv8_cvt2(uint32_t w) {
    if constexpr (FMT == TLMG_KV8_INT8) return kv8_half2<FMT, HI>(w);
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)(HI ? w >> 16 : w)));
    if constexpr (clean) {
        const __half2 m = __hmin2(*reinterpret_cast<const __half2 *>(&r), __half2half2(__ushort_as_half(0x5F00)));
        r = *reinterpret_cast<const uint32_t *>(&m);
    }
    return r;
}

// Four consecutive elements of an activation row as floats (16- or 8-byte aligned).
__device__ __forceinline__ float4 kv8_ld4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 kv8_ld4(const __half *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)),
                 b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 kv8_ld4(const __nv_bfloat16 *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xFFFF0000u));
}
__device__ __forceinline__ void kv8_st4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void kv8_st4(__half *p, float4 v) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
__device__ __forceinline__ void kv8_st4(__nv_bfloat16 *p, float4 v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

// Device view of a cache with shifts for its powers of two.
struct Kv8View {
    uint8_t *k, *v;
    float *ks, *vs;
    int32_t *pos;
    int n_pages, KV, hd;
    int lp, lb;               // log2(page), log2(block)
    // row number of (page entry e, head, row r in the page): fewer than 2^32 (checked on the host)
    __device__ __forceinline__ uint32_t row(int32_t e, int kv, int t) const {
        return (((uint32_t)e * (uint32_t)KV + (uint32_t)kv) << lp) + ((uint32_t)t & ((1u << lp) - 1u));
    }
    __device__ __forceinline__ bool ok(int32_t e) const { return e >= 0 && e < n_pages; }
};

// A sequence of a batch: its rows and its new tokens; false when the lengths break the batch's bounds.
struct Kv8Seq {
    int q0, n, L;
};
__device__ __forceinline__ bool kv8_seq(const tlmg_kv8_batch &b, int lp, int s, Kv8Seq &o) {
    o.q0 = b.q_start[s];
    o.L = b.kv_len[s];
    const int64_t n = (int64_t)b.q_start[s + 1] - o.q0;
    const bool ok = o.q0 >= 0 && n >= 0 && n <= b.max_q && o.q0 + n <= b.total_q && o.L >= n && o.L <= b.max_kv &&
                    (int64_t)o.L <= ((int64_t)b.table_stride << lp);
    o.n = (int)n;
    return ok;
}

// Host: checks (return a TLMG code with the message set) and the device view.
int kv8_check(const char *who, const tlmg_kv8 *c);
int kv8_check_batch(const char *who, const tlmg_kv8_batch *b);
Kv8View kv8_view(const tlmg_kv8 *c);

}  // namespace tlmg
