// Device arithmetic of the per-token symmetric quantizer, shared by the quantizers (quantize.cu, whose
// file comment gives the sequence and the proof of the fast quotient) and the paged append (append_paged.cu).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace fqkv {
namespace {

template <int Q>
__device__ __forceinline__ int quant_code(float x, float s) {
  const float r = __half2float(__float2half_rn(__fdiv_rn(x, s)));
  const float rr = rintf(r);
  if (isnan(rr)) return 0;
  return static_cast<int>(fminf(fmaxf(rr, -float(Q)), float(Q)));
}

// fp32 quotient x / s for a normal fp16 scale s (y = approximate 1/s), rounded as IEEE division.
__device__ __forceinline__ float quot_fast(float x, float s, float y) {
  const float q0 = x * y;
  return fmaf(fmaf(-s, q0, x), y, q0);
}

// Codes of two fp32 quotients with |q| <= 128: fp16(q) (the reference's rounding of X / s),
// then round half to even to an integer by one fp16 addition of 1536 = 1.5 * 2^10 (the sums
// lie in [1408, 1664], where fp16 spacing is 1 and 1536 is even); each code is then the low
// byte of its half's bit pattern (1536 + k has mantissa 512 + k: low byte = k mod 256).
__device__ __forceinline__ uint32_t code_pair_bits(float q_lo, float q_hi) {
  const __half2 r = __floats2half2_rn(q_lo, q_hi);
  const __half2 m = __hadd2(r, __half2half2(__ushort_as_half(0x6600u)));  // + 1536
  return *reinterpret_cast<const uint32_t*>(&m);  // byte 0: code(q_lo), byte 2: code(q_hi)
}

__device__ __forceinline__ float rcp_approx(float s) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(s));
  return y;
}

// s is a normal fp16 number: the fast division applies (see the file comment)
__device__ __forceinline__ bool normal_fp16_scale(float s) { return s >= 6.103515625e-05f && s <= 65504.f; }

template <int Q>
__device__ __forceinline__ __half quant_scale(float amax, bool any_nan) {
  const float a = any_nan ? __int_as_float(0x7fc00000) : amax;
  return __float2half_rn(__fdiv_rn(a, float(Q)));
}

// The same scale for a finite amax by the FMA-corrected division (amax and Q are
// fp16 values, so the argument of the file comment applies); inf / NaN take
// quant_scale's IEEE path.
template <int Q>
__device__ __forceinline__ __half quant_scale_fast(float amax, bool any_nan) {
  if (any_nan || !(amax <= 65504.f)) return quant_scale<Q>(amax, any_nan);
  constexpr float kY = 1.0f / float(Q);  // within half an ulp of 1/Q
  const float q0 = amax * kY;
  return __float2half_rn(fmaf(fmaf(-float(Q), q0, amax), kY, q0));
}

__device__ __forceinline__ unsigned long long f32x2_pack(float lo, float hi) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f32x2_unpack(unsigned long long v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ unsigned long long f32x2_mul(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long f32x2_fma(unsigned long long a, unsigned long long b,
                                                        unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Codes of the fp16 pair h for a normal fp16 scale s (ns2 = (-s, -s), y2 = (1/s~, 1/s~)):
// quot_fast on both lanes, then code_pair_bits.
__device__ __forceinline__ uint32_t code_pair_fast(__half2 h, unsigned long long ns2, unsigned long long y2) {
  const float2 f = __half22float2(h);
  const unsigned long long x2 = f32x2_pack(f.x, f.y);
  const unsigned long long q0 = f32x2_mul(x2, y2);
  const unsigned long long q1 = f32x2_fma(f32x2_fma(ns2, q0, x2), y2, q0);
  float lo, hi;
  f32x2_unpack(q1, lo, hi);
  return code_pair_bits(lo, hi);
}

}  // namespace
}  // namespace fqkv
