// Encoding of a block of 128 values as e4m3 codes with one fp32 scale.
//
//   scale = max|x| / 448 (1 where that is 0),  q = e4m3(x / scale)
//
// The quotient is the correctly rounded one. Where the scale is far from the ends of the
// exponent range it comes from the block's reciprocal by Markstein's final step: with r the
// correctly rounded 1 / s and q0 = x r, the sum q0 + r (x - q0 s) in two fused operations is
// x / s correctly rounded. That is 3 operations per value; the division is about 12, and
// made the quantizer take 53 us instead of 21 for 8192 x 4096 bf16 values.
#pragma once
#include "common.cuh"

namespace sb {

// |v| as an integer that orders like |v|, NaN above infinity, infinity above every number.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct BlockScale {
  float s, r;
  bool fast;  // 2^-90 < s < 2^90: no operand of the fused steps under- or overflows
  __device__ __forceinline__ explicit BlockScale(uint32_t amax_bits) {
    s = __uint_as_float(amax_bits) / 448.0f;
    s = s == 0.f ? 1.f : s;
    r = __frcp_rn(s);
    fast = s > 8.0779357e-28f && s < 1.2379400e27f;
  }
  template <bool FAST>
  __device__ __forceinline__ float quotient(float v) const {
    if (!FAST) return v / s;
    const float q0 = v * r;
    return fmaf(fmaf(-q0, s, v), r, q0);
  }
  // four magnitudes to four codes without their signs
  template <bool FAST>
  __device__ __forceinline__ uint32_t encode4(const float* f) const {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(quotient<FAST>(f[0]), quotient<FAST>(f[1])), __NV_SATFINITE,
                                                 __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(quotient<FAST>(f[2]), quotient<FAST>(f[3])), __NV_SATFINITE,
                                                 __NV_E4M3);
    return lo | hi << 16;
  }
  // eight magnitudes
  __device__ __forceinline__ uint2 encode8(const float (&f)[8]) const {
    return fast ? make_uint2(encode4<true>(f), encode4<true>(f + 4)) : make_uint2(encode4<false>(f), encode4<false>(f + 4));
  }
  __device__ __forceinline__ uint2 encode_signed8(const float (&f)[8]) const {
    float m[8];
    uint32_t sign[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] = fabsf(f[i]);
      sign[i >> 2] |= (__float_as_uint(f[i]) & 0x80000000u) >> (24 - 8 * (i & 3));
    }
    const uint2 c = encode8(m);
    return make_uint2(c.x | sign[0], c.y | sign[1]);
  }
};

// 8 neighbouring values of a row as loaded, their largest magnitude, and their codes.
template <typename T>
struct Vals8 {
  uint4 u;
  __device__ __forceinline__ void load(const T* p) { u = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void set(int i, T v) { reinterpret_cast<T*>(&u)[i] = v; }
  // bits of the largest |value| as fp32 (16-bit magnitudes order like their bits)
  __device__ __forceinline__ uint32_t amax() const {
    const uint32_t m = __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu),
                                __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
    const uint16_t h = (uint16_t)max(m & 0xffffu, m >> 16);
    return __float_as_uint(to_f32<T>(*reinterpret_cast<const T*>(&h)));
  }
  // the codes: the signs go past the arithmetic, from the words' own sign bits
  __device__ __forceinline__ uint2 encode(const BlockScale& s) const {
    const uint4 m = make_uint4(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu, u.z & 0x7fff7fffu, u.w & 0x7fff7fffu);
    float f[8];
    unpack8<T>(m, f);
    const uint2 c = s.encode8(f);
    return make_uint2(c.x | (__byte_perm(u.x, u.y, 0x7531) & 0x80808080u),
                      c.y | (__byte_perm(u.z, u.w, 0x7531) & 0x80808080u));
  }
};
template <>
struct Vals8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void set(int i, float v) { (i < 4 ? reinterpret_cast<float*>(&a) : reinterpret_cast<float*>(&b))[i & 3] = v; }
  __device__ __forceinline__ uint32_t amax() const {
    return max(max(max(abs_bits(a.x), abs_bits(a.y)), max(abs_bits(a.z), abs_bits(a.w))),
               max(max(abs_bits(b.x), abs_bits(b.y)), max(abs_bits(b.z), abs_bits(b.w))));
  }
  __device__ __forceinline__ uint2 encode(const BlockScale& s) const {
    const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    return s.encode_signed8(f);
  }
};

}  // namespace sb
