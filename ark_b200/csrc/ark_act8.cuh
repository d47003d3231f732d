// ark_act8.cuh -- building blocks of the activation kernels: 8-element loads
// and stores of FP16 / BF16 / FP32 rows, and the 8-bit checkpoint format.
//
// Checkpoint of a [rows, cols] activation: one byte per element in rows of
// `pitch` bytes (cols rounded up to 128, so that every row starts on a
// 128-byte boundary and its scale bytes on a 4-byte one), and one scale byte
// per 32 columns.  The scale is a power of two 2^k, k the smallest integer >=
// -126 with max|x| <= top * 2^k (top: 448 for e4m3, 127 for int8); the scale
// byte is k + 127.  A power of two makes x * 2^-k and q * 2^k exact in FP32,
// so the only rounding of the format is the one to 8 bits (nearest even), the
// bytes do not depend on who computes them, and the matrix kernel can turn a
// byte back into a 16-bit operand without a second rounding, within that type's
// range (operand16).  Against a scale max|x| / top it costs int8 half a bit on
// average and e4m3 nothing.
// A block that holds an infinity or a NaN gets scale byte 255 and bytes 0 and
// reads back as NaN: an overflowed forward still makes the step a skipped one.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "ark_device.cuh"
#include "ark_internal.h"

namespace ark {

constexpr int kActBlock = 32;    // columns per scale
constexpr int kActPitch = 128;   // row pitch granule in bytes
constexpr uint32_t kActBad = 255;

enum : int { kE4M3 = ARK_ACT8_E4M3, kInt8 = ARK_ACT8_INT8 };

__host__ __device__ inline uint64_t act8_pitch(uint64_t cols) {
    return (cols + kActPitch - 1) / kActPitch * kActPitch;
}

// ------------------------------------------------------------ element types
template <class T>
struct Elem;
template <>
struct Elem<__half> {
    static constexpr float kMax = 65504.0f;
    static __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr float kMax = 3.38953138925153547590e38f;
    static __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
};
template <>
struct Elem<float> {
    static constexpr float kMax = 3.40282346638528859812e38f;
    static __device__ __forceinline__ float to_f(float x) { return x; }
    static __device__ __forceinline__ float from_f(float x) { return x; }
};

// finite values saturate at the type's largest, a NaN stays one
template <class T>
__device__ __forceinline__ float saturate(float x) {
    x = x > Elem<T>::kMax ? Elem<T>::kMax : x;
    return x < -Elem<T>::kMax ? -Elem<T>::kMax : x;
}

__device__ __forceinline__ void widen2(uint32_t w, float& a, float& b, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x;
    b = f.y;
}
__device__ __forceinline__ void widen2(uint32_t w, float& a, float& b, __nv_bfloat16) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// N consecutive elements (N = 4 or 8) at an address aligned to their size
template <int N>
__device__ __forceinline__ void load_vec(const float* p, float* v) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 q = *reinterpret_cast<const float4*>(p + i);
        v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
    }
}
template <int N, class T>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
    if constexpr (N == 8) {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        widen2(q.x, v[0], v[1], T());
        widen2(q.y, v[2], v[3], T());
        widen2(q.z, v[4], v[5], T());
        widen2(q.w, v[6], v[7], T());
    } else {
        const uint2 q = *reinterpret_cast<const uint2*>(p);
        widen2(q.x, v[0], v[1], T());
        widen2(q.y, v[2], v[3], T());
    }
}
template <int N>
__device__ __forceinline__ void store_vec(float* p, const float* v) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
        *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
template <int N, class T>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
    if constexpr (N == 8)
        *reinterpret_cast<uint4*>(p) =
            make_uint4(narrow2(v[0], v[1], T()), narrow2(v[2], v[3], T()),
                       narrow2(v[4], v[5], T()), narrow2(v[6], v[7], T()));
    else
        *reinterpret_cast<uint2*>(p) = make_uint2(narrow2(v[0], v[1], T()), narrow2(v[2], v[3], T()));
}

// 8 elements of a row of which the first n are there (the others read as 0)
template <class T>
__device__ __forceinline__ void load8(const T* p, int n, bool vec, float* v) {
    if (vec && n >= 8) {
        load_vec<8>(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? Elem<T>::to_f(p[i]) : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, int n, bool vec, const float* v) {
    if (vec && n >= 8) {
        store_vec<8>(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = Elem<T>::from_f(v[i]);
    }
}

// ------------------------------------------------------------ the 8-bit format
template <int N>
__device__ __forceinline__ uint32_t abs_max(const float* v) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
}

// The block's scale byte from the bits of its largest magnitude.  448 is
// 1.75 * 2^8 and 127 is 1.984375 * 2^6: adding the mantissa's distance to the
// next power of two carries into the exponent exactly when 2^k must be one larger.
template <int KIND>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7F800000u) return kActBad;
    const int b = KIND == kE4M3 ? (int)((amax_bits + 0x1FFFFFu) >> 23) - 8
                                : (int)((amax_bits + 0x01FFFFu) >> 23) - 6;
    return (uint32_t)max(b, 1);
}
// 2^-k for a scale byte of 1 to 253
__device__ __forceinline__ float inv_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// 2^k; NaN for the byte of a block that held an infinity or a NaN
__device__ __forceinline__ float scale_of(uint32_t byte) {
    return byte == kActBad ? __uint_as_float(0x7FC00000u) : __uint_as_float(byte << 23);
}

// Four values to four bytes, nearest even.
template <int KIND>
__device__ __forceinline__ uint32_t quant4(const float* v, float inv) {
    if constexpr (KIND == kE4M3) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
            : "=h"(lo)
            : "f"(__fmul_rn(v[1], inv)), "f"(__fmul_rn(v[0], inv)));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
            : "=h"(hi)
            : "f"(__fmul_rn(v[3], inv)), "f"(__fmul_rn(v[2], inv)));
        return pack16(lo, hi);
    } else {
        // |v * inv| <= 127: adding 1.5 * 2^23 rounds to the nearest even
        // integer, whose two's complement is then the low byte
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[i] = __float_as_uint(__fadd_rn(__fmul_rn(v[i], inv), 12582912.0f));
        return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
    }
}

// Eight values of a block with scale byte `byte`.
template <int KIND>
__device__ __forceinline__ uint2 quant8(const float* v, uint32_t byte) {
    if (byte == kActBad) return make_uint2(0u, 0u);
    const float inv = inv_scale(byte);
    return make_uint2(quant4<KIND>(v, inv), quant4<KIND>(v + 4, inv));
}

// Four bytes back to the integers or e4m3 values that they hold (not scaled).
template <int KIND>
__device__ __forceinline__ void bytes4(uint32_t w, float* v) {
    if constexpr (KIND == kE4M3) {
        uint32_t lo, hi;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)(w & 0xFFFFu)));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(w >> 16)));
        widen2(lo, v[0], v[1], __half());
        widen2(hi, v[2], v[3], __half());
    } else {
        // byte ^ 0x80 is q + 128; as the low mantissa byte of 2^23 it is 2^23 + q + 128
        const uint32_t u = w ^ 0x80808080u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = __fsub_rn(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + i)), 8388736.0f);
    }
}
template <int KIND>
__device__ __forceinline__ void dequant8(uint2 w, uint32_t byte, float* v) {
    const float s = scale_of(byte);
    bytes4<KIND>(w.x, v);
    bytes4<KIND>(w.y, v + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], s);
}

// ------------------------------------------------------------ bytes to 16-bit values
// Two FP32 values to a pair of T, saturating (a NaN stays one).
__device__ __forceinline__ uint32_t pair_of(float a, float b, __half) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t pair_of(float a, float b, __nv_bfloat16) {
    uint32_t r;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// Scale bytes between which q * 2^k needs neither saturation nor a scale
// outside of T; every block of ordinary activations lies between them.  The
// others (and NaN blocks) go through FP32, but for operands up to kNone, where every
// value rounds to zero: a row's padding makes such blocks (scale byte 1).
template <class T, int KIND>
struct Fast;
template <>
struct Fast<__half, kE4M3> {
    // 2^-24 is the smallest FP16; 448 * 2^7 is below 65504
    static constexpr uint32_t kLo = 127 - 24, kHi = 127 + 7, kNone = 127 - 37;
    __half2 s;
    __device__ __forceinline__ explicit Fast(uint32_t byte) {
        s = __float2half2_rn(__uint_as_float(byte << 23));
    }
    __device__ __forceinline__ uint32_t pair(uint32_t w, int at) const {   // bytes at, at + 1
        uint32_t h;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w >> (8 * at))));
        const __half2 r = __hmul2_rn(*reinterpret_cast<__half2*>(&h), s);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};
template <>
struct Fast<__half, kInt8> {
    static constexpr uint32_t kLo = 127 - 24, kHi = 127 + 5, kNone = 127 - 37;
    __half2 s, t;   // 2^k and -1152 * 2^k
    __device__ __forceinline__ explicit Fast(uint32_t byte) {
        const float f = __uint_as_float(byte << 23);
        s = __float2half2_rn(f);
        t = __float2half2_rn(__fmul_rn(f, -1152.0f));
    }
    __device__ __forceinline__ uint32_t pair(uint32_t w, int at) const {
        // (q + 128) as the low byte of 1024 is 1152 + q: one fused operation
        // takes the offset off and scales, exactly
        const uint32_t h = __byte_perm(w ^ 0x80808080u, 0x64646464u, at ? 0x4342 : 0x4140);
        const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&h), s, t);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};
template <>
struct Fast<__nv_bfloat16, kE4M3> {
    // exponent and mantissa of e4m3 moved to BF16's, whose bias is 120 larger:
    // the value times 2^-120, subnormals included
    static constexpr uint32_t kLo = 1, kHi = 127 + 7, kNone = 0;
    __nv_bfloat162 s;
    __device__ __forceinline__ explicit Fast(uint32_t byte) {
        s = __float2bfloat162_rn(__uint_as_float((byte + 120u) << 23));
    }
    __device__ __forceinline__ uint32_t pair(uint32_t w, int at) const {
        const uint32_t h = __byte_perm(w, 0u, at ? 0x3424 : 0x1404);   // bytes to the high halves
        const uint32_t v = (h & 0x80008000u) | ((h >> 4) & 0x07F007F0u);
        const __nv_bfloat162 r = __hmul2_rn(*reinterpret_cast<const __nv_bfloat162*>(&v), s);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};
template <>
struct Fast<__nv_bfloat16, kInt8> {
    static constexpr uint32_t kLo = 1, kHi = 127 + 120, kNone = 0;
    __nv_bfloat162 s;
    __device__ __forceinline__ explicit Fast(uint32_t byte) {
        s = __float2bfloat162_rn(__uint_as_float(byte << 23));
    }
    __device__ __forceinline__ uint32_t pair(uint32_t w, int at) const {
        // under the exponent of 128 the low 7 bits are 128 + (q mod 128), and the
        // sign bit alone is 128 or 256: their difference is q
        const uint32_t h = __byte_perm(w, 0x43434343u, at ? 0x4342 : 0x4140);
        const uint32_t lo = h & 0xFF7FFF7Fu, hi = h & 0xFF80FF80u;
        const __nv_bfloat162 r =
            __hmul2_rn(__hsub2_rn(*reinterpret_cast<const __nv_bfloat162*>(&lo),
                                  *reinterpret_cast<const __nv_bfloat162*>(&hi)),
                       s);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};
// The same for an operand of the matrix kernels: a magnitude above 65536 becomes an
// infinity in FP16, so that the gradient shows it.  65536 itself is what the 8-bit
// rounding makes of the largest FP16 numbers; 65504 is as near to them.  BF16 has the
// FP32 range, and saturates only what 8 bits rounded up to 2^128.
__device__ __forceinline__ uint32_t operand_pair(float a, float b, __half) {
    a = fabsf(a) == 65536.0f ? copysignf(65504.0f, a) : a;
    b = fabsf(b) == 65536.0f ? copysignf(65504.0f, b) : b;
    return narrow2(a, b, __half());
}
__device__ __forceinline__ uint32_t operand_pair(float a, float b, __nv_bfloat16) {
    return pair_of(a, b, __nv_bfloat16());
}
// Sixteen bytes of one block to 16-bit values in order.  OPERAND: out of range as
// operand_pair, else saturating.  Every value of a checkpoint of FP16 numbers is an
// FP16 number (but for 65536), down to 2^-24: the 8-bit rounding takes low bits off and
// puts none on.  Values of a checkpoint of a wider type are rounded once.
template <class T, int KIND, bool OPERAND>
__device__ __forceinline__ void operand16(uint4 w, uint32_t byte, uint4& lo, uint4& hi) {
    using F = Fast<T, KIND>;
    if (byte >= F::kLo && byte <= F::kHi) {
        const F f(byte);
        lo = make_uint4(f.pair(w.x, 0), f.pair(w.x, 2), f.pair(w.y, 0), f.pair(w.y, 2));
        hi = make_uint4(f.pair(w.z, 0), f.pair(w.z, 2), f.pair(w.w, 0), f.pair(w.w, 2));
    } else if (OPERAND && byte <= F::kNone) {
        lo = hi = make_uint4(0u, 0u, 0u, 0u);
    } else {
        auto two = [](float x, float y) {
            return OPERAND ? operand_pair(x, y, T()) : pair_of(x, y, T());
        };
        float v[8];
        dequant8<KIND>(make_uint2(w.x, w.y), byte, v);
        lo = make_uint4(two(v[0], v[1]), two(v[2], v[3]), two(v[4], v[5]), two(v[6], v[7]));
        dequant8<KIND>(make_uint2(w.z, w.w), byte, v);
        hi = make_uint4(two(v[0], v[1]), two(v[2], v[3]), two(v[4], v[5]), two(v[6], v[7]));
    }
}

// ------------------------------------------------------------ pairs of FP32
// One instruction for two products or sums, each rounded as the single one is.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t twice(float a) { return pair(a, a); }
__device__ __forceinline__ uint64_t neg2(uint64_t v) { return v ^ 0x8000000080000000ull; }
__device__ __forceinline__ float sum2(uint64_t v) {
    float a, b;
    unpair(v, a, b);
    return __fadd_rn(a, b);
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// ------------------------------------------------------------ 16-bit values to bytes
// The largest magnitudes of N words' low and high halves.
template <int N>
__device__ __forceinline__ uint32_t pairs_max(const uint32_t* w) {
    uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
    for (int i = 1; i < N; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
    return m;
}
// The FP32 bits of the larger half.
template <class T>
__device__ __forceinline__ uint32_t pairs_bits(uint32_t m, T) {
    float a, b;
    widen2(max(m & 0xFFFFu, m >> 16), a, b, T());
    return __float_as_uint(a);
}
// N words of two values of a block with scale byte `byte` to N / 2 words of four bytes.
template <class T, int KIND, int N>
__device__ __forceinline__ void quant_words(const uint32_t* w, uint32_t byte, uint32_t* o) {
    if constexpr (std::is_same<T, __half>::value) {
        // 2^-k is an FP16 number, and x * 2^-k as FP16 keeps every bit that rounding
        // to 8 bits looks at: below 2^-14, where it may not, all values round to 0
        if (byte >= 127 - 15 && byte <= 127 + 14) {
            const __half2 inv = __float2half2_rn(inv_scale(byte));
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const __half2 a = *reinterpret_cast<const __half2*>(&w[2 * i]);
                const __half2 b = *reinterpret_cast<const __half2*>(&w[2 * i + 1]);
                if constexpr (KIND == kE4M3) {
                    const __half2 x = __hmul2_rn(a, inv), y = __hmul2_rn(b, inv);
                    uint16_t lo, hi;
                    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;"
                        : "=h"(lo)
                        : "r"(*reinterpret_cast<const uint32_t*>(&x)));
                    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;"
                        : "=h"(hi)
                        : "r"(*reinterpret_cast<const uint32_t*>(&y)));
                    o[i] = pack16(lo, hi);
                } else {
                    // 1536 + x * 2^-k rounds once, to a whole number; its low byte is
                    // the integer's two's complement
                    const __half2 magic = __float2half2_rn(1536.0f);
                    const __half2 x = __hfma2(a, inv, magic), y = __hfma2(b, inv, magic);
                    o[i] = __byte_perm(*reinterpret_cast<const uint32_t*>(&x),
                                       *reinterpret_cast<const uint32_t*>(&y), 0x6420);
                }
            }
            return;
        }
    }
    if (byte == kActBad) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) o[i] = 0;
        return;
    }
    const uint64_t inv = twice(inv_scale(byte));
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        float a, b, c, d;
        widen2(w[2 * i], a, b, T());
        widen2(w[2 * i + 1], c, d, T());
        if constexpr (KIND == kE4M3) {
            unpair(mul2(pair(a, b), inv), a, b);
            unpair(mul2(pair(c, d), inv), c, d);
            uint16_t lo, hi;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
            o[i] = pack16(lo, hi);
        } else {
            // as quant4, the product exact and the sum rounded once
            const uint64_t magic = twice(12582912.0f);
            unpair(fma2(pair(a, b), inv, magic), a, b);
            unpair(fma2(pair(c, d), inv, magic), c, d);
            o[i] = __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                               __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
        }
    }
}

// ------------------------------------------------------------ host checks
inline uint64_t type_size(int32_t type) {
    return type == ARK_TYPE_F32 ? 4u : (type == ARK_TYPE_F16 || type == ARK_TYPE_BF16) ? 2u : 0u;
}
inline bool aligned_to(const void* p, uint64_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}
// f called with a value of the element type
template <class F>
int by_type(int32_t type, F f) {
    if (type == ARK_TYPE_F16) return f(__half());
    if (type == ARK_TYPE_BF16) return f(__nv_bfloat16());
    if (type == ARK_TYPE_F32) return f(float());
    return ARK_E_INVALID_ARG;
}

// null data is fine for an empty checkpoint
int act8_check(const ark_act8* c);
// act8_unpack to 16-bit operands of the matrix kernels (operand16), rows of whole vectors
int act8_operands(const ark_act8* c, void* y, int32_t type, uint64_t ldy, cudaStream_t s);
// 16-bit rows that start on any element, copied to rows of whole 16-byte vectors
int realign_rows(const void* src, uint64_t ld, uint64_t rows, uint32_t cols, void* dst, uint64_t ldd,
                 cudaStream_t s);

}  // namespace ark
