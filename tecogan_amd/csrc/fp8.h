// 8-bit floating point with a power-of-two scale for each block of 128: what the quantiser and the product that quantises on the way
// share.
#pragma once
#include "common.h"

typedef short s16x2q __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2q __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2q __attribute__((ext_vector_type(2)));

// biased exponent of a block's scale, from the bits of its largest absolute value (fp32, finite)
template <int FMT>
__device__ __forceinline__ uint32_t fp8_scale_code(uint32_t b) {
  if (b == 0) return 127;
  const int e = (int)(b >> 23) - 127 - (FMT == TG_FP8_E4M3 ? 8 : 15) + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)((e < -126 ? -126 : e) + 127);
}
constexpr uint32_t FP8_INF = 0x7f800000u;

// Two values -> two bytes of w, divided by 2^(code - 127), rounded to nearest even in one instruction.
template <int FMT, bool HI>
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w, float a, float b, uint32_t code) {
  const s16x2q o = __builtin_bit_cast(s16x2q, w);
  const float s = __uint_as_float(code << 23);
  if constexpr (FMT == TG_FP8_E4M3) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, a, b, s, HI));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(o, a, b, s, HI));
}
template <int FMT, bool HI>
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w, uint32_t ab /*two bf16*/, uint32_t code) {
  const s16x2q o = __builtin_bit_cast(s16x2q, w);
  const bf16x2q v = __builtin_bit_cast(bf16x2q, ab);
  const float s = __uint_as_float(code << 23);
  if constexpr (FMT == TG_FP8_E4M3) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, v, s, HI));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(o, v, s, HI));
}

// 8 neighbouring values as they lie in memory.  BAD (one choice for a wave): a NaN or an infinity is among the wave's values; they
// are left out of the largest absolute value, and infinities of e4m3, which has none, become NaN before the conversion.
struct Fp8In16 {
  uint4 w;
  __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const u16* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void load(const u16* p, int have, bool vec) {
    if (have >= 8) {
      w = vec ? *reinterpret_cast<const uint4*>(p) : ld128_any(p);
    } else {
      uint32_t q[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = (2 * k < have ? p[2 * k] : 0u) | ((2 * k + 1 < have ? (uint32_t)p[2 * k + 1] : 0u) << 16);
      w = make_uint4(q[0], q[1], q[2], q[3]);
    }
  }
  __device__ __forceinline__ uint32_t word(int k) const { return k == 0 ? w.x : k == 1 ? w.y : k == 2 ? w.z : w.w; }
  // |values| of word k, two bf16
  template <bool BAD>
  __device__ __forceinline__ u16x2q abs2(int k) const {
    uint32_t a = word(k) & 0x7fff7fffu;
    if constexpr (BAD) {
      if ((a & 0xffffu) >= 0x7f80u) a &= 0xffff0000u;
      if ((a >> 16) >= 0x7f80u) a &= 0xffffu;
    }
    return __builtin_bit_cast(u16x2q, a);
  }
  template <bool BAD>
  __device__ __forceinline__ uint32_t most() const {                   // bits of the largest absolute value
    const u16x2q m = __builtin_elementwise_max(__builtin_elementwise_max(abs2<BAD>(0), abs2<BAD>(1)), __builtin_elementwise_max(abs2<BAD>(2), abs2<BAD>(3)));
    return (uint32_t)(m[0] > m[1] ? m[0] : m[1]) << 16;
  }
  template <int FMT, bool BAD>
  static __device__ __forceinline__ uint32_t storable(uint32_t ab) {
    if constexpr (BAD && FMT == TG_FP8_E4M3) {
      if ((ab & 0x7fffu) == 0x7f80u) ab |= 0x40u;
      if ((ab & 0x7fff0000u) == 0x7f800000u) ab |= 0x400000u;
    }
    return ab;
  }
  template <int FMT, bool BAD>
  __device__ __forceinline__ uint2 pack(uint32_t code) const {
    uint2 o;
    o.x = fp8_pair<FMT, true>(fp8_pair<FMT, false>(0, storable<FMT, BAD>(w.x), code), storable<FMT, BAD>(w.y), code);
    o.y = fp8_pair<FMT, true>(fp8_pair<FMT, false>(0, storable<FMT, BAD>(w.z), code), storable<FMT, BAD>(w.w), code);
    return o;
  }
};
struct Fp8In32 {
  f32x4 a, b;
  __device__ __forceinline__ void zero() { a = b = f32x4{0.f, 0.f, 0.f, 0.f}; }
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const f32x4*>(p);
    b = *reinterpret_cast<const f32x4*>(p + 4);
  }
  __device__ __forceinline__ void load(const float* p, int have, bool vec) {
    if (have >= 8) {
      a = vec ? *reinterpret_cast<const f32x4*>(p) : __builtin_bit_cast(f32x4, ld128_any(p));
      b = vec ? *reinterpret_cast<const f32x4*>(p + 4) : __builtin_bit_cast(f32x4, ld128_any(p + 4));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a[k] = k < have ? p[k] : 0.f;
        b[k] = 4 + k < have ? p[4 + k] : 0.f;
      }
    }
  }
  __device__ __forceinline__ float value(int k) const { return k < 4 ? a[k & 3] : b[k & 3]; }
  template <bool BAD>
  __device__ __forceinline__ uint32_t abs1(int k) const {
    const uint32_t v = __float_as_uint(value(k)) & 0x7fffffffu;
    return BAD && v >= FP8_INF ? 0u : v;
  }
  template <bool BAD>
  __device__ __forceinline__ uint32_t most() const {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t v = abs1<BAD>(k);
      m = m > v ? m : v;
    }
    return m;
  }
  template <int FMT, bool BAD>
  static __device__ __forceinline__ float storable(float v) {
    return BAD && FMT == TG_FP8_E4M3 && (__float_as_uint(v) & 0x7fffffffu) == FP8_INF ? __builtin_nanf("") : v;
  }
  template <int FMT, bool BAD>
  __device__ __forceinline__ uint2 pack(uint32_t code) const {
    uint2 o;
    o.x = fp8_pair<FMT, true>(fp8_pair<FMT, false>(0, storable<FMT, BAD>(a[0]), storable<FMT, BAD>(a[1]), code), storable<FMT, BAD>(a[2]), storable<FMT, BAD>(a[3]), code);
    o.y = fp8_pair<FMT, true>(fp8_pair<FMT, false>(0, storable<FMT, BAD>(b[0]), storable<FMT, BAD>(b[1]), code), storable<FMT, BAD>(b[2]), storable<FMT, BAD>(b[3]), code);
    return o;
  }
};
template <typename T> struct Fp8In;
template <> struct Fp8In<u16> { using type = Fp8In16; };
template <> struct Fp8In<float> { using type = Fp8In32; };

// the larger of v and its partner's, lane exchanges inside the vector unit: over the 16 lanes of a row of lanes, and across the rows
template <int CTRL>
__device__ __forceinline__ uint32_t fp8_max_dpp(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
  return v > o ? v : o;
}
__device__ __forceinline__ uint32_t fp8_max16(uint32_t v) {
  v = fp8_max_dpp<0xB1>(v);                                             // lane ^ 1
  v = fp8_max_dpp<0x4E>(v);                                             // lane ^ 2
  v = fp8_max_dpp<0x141>(v);                                            // 7 - lane: the other four of eight
  return fp8_max_dpp<0x128>(v);                                         // lane ^ 8
}
