// Eight neighbouring values of a row and their E4M3 codes (fp8_rows.cu says what they are).
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "axb_common.cuh"

namespace {

template <typename T>
AXB_DEVICE float to_f32(T v);
template <>
AXB_DEVICE float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
AXB_DEVICE float to_f32(__half v) { return __half2float(v); }
template <>
AXB_DEVICE float to_f32(float v) { return v; }
// two neighbouring values as they are stored
AXB_DEVICE void put2(__nv_bfloat16* o, float2 f) { *reinterpret_cast<uint32_t*>(o) = pack_bf16x2(f.x, f.y); }
// The largest fp16 numbers have a code that stands for 2^16, which fp16 does not have: its largest one, so that they stay finite.
AXB_DEVICE float in_fp16(float v) { return fabsf(v) == 65536.f ? copysignf(65504.f, v) : v; }
AXB_DEVICE void put2(__half* o, float2 f) { *reinterpret_cast<__half2*>(o) = __floats2half2_rn(in_fp16(f.x), in_fp16(f.y)); }
AXB_DEVICE void put2(float* o, float2 f) { *reinterpret_cast<float2*>(o) = f; }

// Eight values of a row as they are stored. The largest magnitude is taken in the stored type, two values an instruction: with every
// value widened first the kernel was bound by its arithmetic (32768 x 4096 in bf16: 112 us, 70 like this, 64 with codes4 below).
template <typename T>
struct Eight {
  uint4 raw[sizeof(T) / 2];
  AXB_DEVICE void load(const T* p) {
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h) raw[h] = __ldg(reinterpret_cast<const uint4*>(p) + h);
  }
  AXB_DEVICE void load_some(const T* p, int n) {     // the first n, zeros behind them
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h) raw[h] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) reinterpret_cast<T*>(raw)[j] = p[j];
  }
  AXB_DEVICE float at(int j) const { return to_f32<T>(reinterpret_cast<const T*>(raw)[j]); }
  AXB_DEVICE float top() const;                      // of those that are not NaN (NaN: there is none)
  // with m the largest of `top` over the block, and the biased exponent of its scale; 16 lanes hold the block. odd: m is not finite in
  // some lane of the warp
  AXB_DEVICE uint2 codes(float m, bool odd, int& e) const;
};
template <>
AXB_DEVICE float Eight<__nv_bfloat16>::top() const {
  const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(raw);
  const __nv_bfloat162 m = __hmax2(__hmax2(__habs2(v[0]), __habs2(v[1])), __hmax2(__habs2(v[2]), __habs2(v[3])));
  return __bfloat162float(__hmax(m.x, m.y));
}
template <>
AXB_DEVICE float Eight<__half>::top() const {
  const __half2* v = reinterpret_cast<const __half2*>(raw);
  const __half2 m = __hmax2(__hmax2(__habs2(v[0]), __habs2(v[1])), __hmax2(__habs2(v[2]), __habs2(v[3])));
  return __half2float(__hmax(__low2half(m), __high2half(m)));
}
template <>
AXB_DEVICE float Eight<float>::top() const {
  float m = fabsf(at(0));
#pragma unroll
  for (int j = 1; j < 8; ++j) m = fmaxf(m, fabsf(at(j)));
  return m;
}

AXB_DEVICE float group_max(float m) {     // over the 16 lanes that hold a block of 128 columns
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

AXB_DEVICE bool odd_max(float m) { return !(m <= 3.402823466e38f); }

template <typename T>
AXB_DEVICE uint2 Eight<T>::codes(float m, bool odd, int& e) const {
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = at(j);
  if (odd) {
    // an infinity, or nothing but NaN: the maximum of the finite values, and NaN for the others
    m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (fabsf(f[j]) <= 3.402823466e38f) m = fmaxf(m, fabsf(f[j]));
      else f[j] = __uint_as_float(0x7FC00000u);
    }
    m = group_max(m);
  }
  e = fp8_scale_exponent(m);
  const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
  if (e >= 247) {                                    // scale 2^120: the code 256 would stand for 2^128
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (fabsf(f[j]) > 240.f * 0x1p120f) f[j] = copysignf(240.f * 0x1p120f, f[j]);
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * h] * inv, f[4 * h + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * h + 2] * inv, f[4 * h + 3] * inv), __NV_SATFINITE, __NV_E4M3);
    w[h] = lo | (hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// Codes of four blocks and the biased exponents of their scales; 16 lanes hold a block each time.
template <typename T>
AXB_DEVICE void codes4(const Eight<T> (&v)[4], uint2 (&w)[4], int (&e)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float m = group_max(v[i].top());
    w[i] = v[i].codes(m, __any_sync(0xffffffffu, odd_max(m)), e[i]);
  }
}
// The four maxima travel together, two to a register, and half of the lanes finish two of them each: five shuffles instead of sixteen, and
// the exponents are worked out once for two blocks. Values are scaled two an instruction: a power of two is exact in bf16, and what falls
// below its range has the code 0 either way. Where the largest value is 2^127 or more, an infinity or NaN, the blocks go one by one.
AXB_DEVICE void codes4(const Eight<__nv_bfloat16> (&v)[4], uint2 (&w)[4], int (&e)[4]) {
  uint32_t t[4];                          // the lane's largest of each block in both halves
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162* u = reinterpret_cast<const __nv_bfloat162*>(v[i].raw);
    const __nv_bfloat162 m = __hmax2(__hmax2(__habs2(u[0]), __habs2(u[1])), __hmax2(__habs2(u[2]), __habs2(u[3])));
    t[i] = *reinterpret_cast<const uint32_t*>(&m);
  }
  auto max2 = [](uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  };
  const bool hi = threadIdx.x & 8;
  const uint32_t t01 = max2(__byte_perm(t[0], t[1], 0x5410), __byte_perm(t[0], t[1], 0x7632));
  const uint32_t t23 = max2(__byte_perm(t[2], t[3], 0x5410), __byte_perm(t[2], t[3], 0x7632));
  uint32_t m = max2(hi ? t23 : t01, __shfl_xor_sync(0xffffffffu, hi ? t01 : t23, 8));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) m = max2(m, __shfl_xor_sync(0xffffffffu, m, o));
  const int a = m & 0x7FFF, b = (m >> 16) & 0x7FFF;
  if (__any_sync(0xffffffffu, max(a, b) >= 0x7F00)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = v[i].codes(group_max(v[i].top()), true, e[i]);
    return;
  }
  // fp8_scale_exponent of a bf16 number: 0x60 is the mantissa of 1.75
  const int ea = a == 0 ? 127 : max(((a + 0x1F) >> 7) - 8, 1), eb = b == 0 ? 127 : max(((b + 0x1F) >> 7) - 8, 1);
  const uint32_t mine = (uint32_t)ea | ((uint32_t)eb << 16), other = __shfl_xor_sync(0xffffffffu, mine, 8);
  const uint32_t e01 = hi ? other : mine, e23 = hi ? mine : other;
  e[0] = e01 & 0xFFFF;
  e[1] = e01 >> 16;
  e[2] = e23 & 0xFFFF;
  e[3] = e23 >> 16;
  const uint32_t i01 = (0x00FE00FEu - e01) << 7, i23 = (0x00FE00FEu - e23) << 7;      // 2^(127 - e) in bf16; no borrow: e < 247
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t inv = __byte_perm(i < 2 ? i01 : i23, 0u, i & 1 ? 0x3232 : 0x1010);
    const __nv_bfloat162* u = reinterpret_cast<const __nv_bfloat162*>(v[i].raw);
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __bfloat1622float2(__hmul2(u[j], *reinterpret_cast<const __nv_bfloat162*>(&inv)));
      c[j] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
    }
    w[i] = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
  }
}

}  // namespace
