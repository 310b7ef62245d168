// Conversions of the 8-bit key/value cache's codes (see kv8.cu for its layout).
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace msgl {

MSGL_DEVICE void kv8_load_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// mbar_wait for the roles of a stream of data: few instructions (many such waits' code has to fit the instruction cache), and no
// look at the clock, which takes long to read. A try takes 0.1 to 4 us, so that a wait gives up after 0.3 to 17 s; the role
// then ends, and says where by kv8_gave_up.
MSGL_DEVICE bool kv8_wait(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (uint32_t i = 0; i < (1u << 22); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred P;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, P;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(4000u)  // (suspended for up to 4 us)
        : "memory");
    if (ok) return true;
  }
  return false;
}
// The same for a whole warp: its lanes go on or give up together.
MSGL_DEVICE bool kv8_wait_warp(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, kv8_wait(bar, parity)); }
MSGL_DEVICE void kv8_gave_up(int where) { report_error(kErrMbarTimeout, where); }

// two values to two e4m3 codes, nearest, ties to even (the first one in the low byte)
MSGL_DEVICE uint16_t kv8_e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// A row x has scale = max|x| / Q with Q = 127 (int8) or 448 (e4m3), and codes = nearest(x Q / max|x|), ties
// to even. The quotient has to be rounded as in exact arithmetic: it can lie on a tie (x = max / 2 gives 63.5), and
// where it does not it is at least 2^-16 of its size away from one: x and max have 8 bits, a tie t = odd / 2 has 8 (int8; 5 in
// e4m3, whose Q is 7 times a power of two), so 2 x Q and 2 t max are different multiples of x's unit, below 2^16 of it.
// An fp32 quotient that is exact where it is representable suffices.
// pairs of fp32 in one register pair
MSGL_DEVICE uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
MSGL_DEVICE float2 f2_unpack(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
MSGL_DEVICE uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
MSGL_DEVICE uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
MSGL_DEVICE uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

template <bool FP8>
struct Kv8Quant {
  float scale, by, a, inv;
  bool codes;  // the row has any: not one of zeros, nor one with an infinity or a NaN, whose scale is NaN
  MSGL_DEVICE explicit Kv8Quant(float top) {
    constexpr float Q = FP8 ? 448.f : 127.f;
    codes = top > 0.f && top < INFINITY;
    if (top > 0x1p-100f && codes) {
      // top / Q by Q's reciprocal and one Newton step on the remainder, which fma gives exactly: within 2^-46 of the quotient,
      // which is 2^-33 or more away from where fp32's rounding turns (8 bits over 7)
      scale = top * (1.f / Q);
      scale = fmaf(fmaf(-scale, Q, top), 1.f / Q, scale);
    } else {
      scale = top == 0.f || codes ? __fdiv_rn(top, Q) : __int_as_float(0x7fc00000);
    }
    // x Q must not overflow, and products with the remainder below not underflow: both sides of the quotient
    // are moved to the middle of the range, by a power of two, which changes neither
    by = Q;
    a = top;
    if (top > 0x1p+100f) by *= 0x1p-64f, a *= 0x1p-64f;
    if (top < 0x1p-60f) by *= 0x1p+64f, a *= 0x1p+64f;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(a));  // (to 1 ulp)
  }
  // x Q / max of two values: by the reciprocal, then a Newton step on the remainder x - q a, which fma gives exactly:
  // within 2^-45 of the quotient before its rounding to fp32, so exact where it is representable
  MSGL_DEVICE uint64_t quotients(float lo, float hi) const {
    const uint64_t i2 = f2_pack(inv, inv), x = f2_mul(f2_pack(lo, hi), f2_pack(by, by)), q = f2_mul(x, i2);
    return f2_fma(f2_fma(f2_mul(q, f2_pack(-1.f, -1.f)), f2_pack(a, a), x), i2, q);
  }
  // two values of the row to two codes (the first one in the low byte; what is above them is not theirs)
  MSGL_DEVICE uint32_t pair(float lo, float hi) const {
    if constexpr (FP8) {
      const float2 q = f2_unpack(quotients(lo, hi));
      return codes ? kv8_e4m3x2(q.x, q.y) : 0u;
    } else {  // 1.5 2^23 more has the nearest whole number in its low bits
      const float2 q = f2_unpack(f2_add(quotients(lo, hi), f2_pack(12582912.f, 12582912.f)));
      return codes ? __byte_perm(__float_as_uint(q.x), __float_as_uint(q.y), 0x0040) : 0u;
    }
  }
};

// the two values of a pair of codes (the low 16 bits)
template <bool FP8>
MSGL_DEVICE float2 kv8_decode2(uint32_t pair) {
  if constexpr (FP8) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(pair & 0xffffu), __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
  } else {
    return make_float2((float)(int8_t)(pair & 255u), (float)(int8_t)((pair >> 8) & 255u));
  }
}

// Four codes (one register) to two fp16 pairs, exactly: lo holds the first two values, hi the others. int8: the byte
// with its sign bit turned is the low mantissa of 1024 + (code + 128), from which 1152 is taken.
template <bool FP8>
MSGL_DEVICE void kv8_to_half(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  if constexpr (FP8) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(codes));
  } else {
    const uint32_t u = codes ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off), y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}

// The same to two bf16 pairs, exactly: every code has at most 8 significant bits.
template <bool FP8>
MSGL_DEVICE void kv8_to_bf16(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  if constexpr (FP8) {
    uint32_t a, b;
    kv8_to_half<true>(codes, a, b);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    lo = pack_bf16(x.x, x.y);
    hi = pack_bf16(y.x, y.y);
  } else {  // 128 + the low seven bits, less 128 or, with the sign bit, 256
    const uint32_t a = __byte_perm(codes, 0x43434343u, 0x4140), b = __byte_perm(codes, 0x43434343u, 0x4342);
    const uint32_t x = a & 0xff7fff7fu, y = a & 0xff80ff80u, z = b & 0xff7fff7fu, w = b & 0xff80ff80u;
    const __nv_bfloat162 c = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&z), *reinterpret_cast<const __nv_bfloat162*>(&w));
    lo = *reinterpret_cast<const uint32_t*>(&c);
    hi = *reinterpret_cast<const uint32_t*>(&d);
  }
}

// 2^x, to 2^-22 of it (2^-126 and below: zero)
MSGL_DEVICE float kv8_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

MSGL_DEVICE uint32_t pack_half(float a, float b) {
  const __half2 t = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}

// The power of two that brings a row of queries with this largest magnitude to [2^14, 2^15), where fp16 holds them
// exactly down to 2^-31 of the largest; 1 for rows of zeros and rows that are not finite.
MSGL_DEVICE float kv8_q_factor(float top) {
  if (!(top > 0.f) || !(top < INFINITY)) return 1.f;
  const int e = (int)(__float_as_uint(top) >> 23);  // biased
  return __uint_as_float((uint32_t)min(268 - e, 253) << 23);
}
MSGL_DEVICE float kv8_reciprocal(float power_of_two) { return __uint_as_float((254u << 23) - __float_as_uint(power_of_two)); }

// A softmax weight times its value's scale is rounded to fp16, so it is that product which must lie in fp16's range, not
// the probability: a token that takes nearly all of a softmax often has a value row of nearly nothing. So a row's
// running offset m is the maximum of s_j + log2 s^v_j, less kKv8Top, not that of the logits s_j: products
// 2^(s_j - m) s^v_j are at most 2^14, and 11 bits hold down to 2^-28 of the largest. The sum of the 2^(s_j - m) is fp32, with
// the same m, and keeps its own range as long as a row's scales are between 2^-96 and 2^96; smaller ones (a row of zeros has
// 0) are taken for 2^-96 in m, which leaves the products right but smaller.
constexpr float kKv8Top = 14.f;
MSGL_DEVICE float kv8_log_scale(float scale) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(scale));
  return fminf(fmaxf(y, -96.f), 96.f);
}

}  // namespace msgl
