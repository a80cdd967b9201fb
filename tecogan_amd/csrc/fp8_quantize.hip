// 8-bit floating point with one power-of-two scale for each block of 128 along the reduction.
//
// The scale of a block is 2^e, e the smallest integer in [-126, 127] with amax <= largest(type) 2^e (448 = 1.75 2^8 for e4m3,
// 57344 = 1.75 2^15 for e5m2); a value is stored as round-to-nearest-even(x 2^-e).  Powers of two make the division exact, so the
// rounding to 8 bits is the only one, and gfx950's scaled matrix instruction takes the biased exponent (e + 127, one byte) as
// its operand: the product needs no multiplication by scales.  amax is taken over the finite values of a block; a NaN or an
// infinity stays one (e4m3 has no infinity: NaN) and does not touch its neighbours.  A block of zeros has e = 0.
//
// One workgroup takes a 128 x 128 tile, 64 values a thread in registers: the matrix is read once for both orders that a training
// step needs (blocks along the columns for y and dx, along the rows for dW), 2 + 1 + 1 bytes a value: bound by HBM.  The transposed
// copy goes through LDS as bytes (rows of 144 bytes), so both copies are written as whole 128-byte lines.
#include "common.h"

namespace {

constexpr int FQ_PITCH = 144;

template <typename T>
__device__ __forceinline__ void load8q(const T* __restrict__ p, int have, bool vec, float (&f)[8]) {
  if (vec && have >= 8) {
    if constexpr (sizeof(T) == 2) {
      bf8_unpack(*reinterpret_cast<const uint4*>(p), f);
    } else {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = k < have ? Elem<T>::ld(p + k) : 0.f;
  }
}

__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a < __builtin_inff() ? a : 0.f;
}

// biased exponent of a block's scale
template <int FMT>
__device__ __forceinline__ uint32_t scale_code(float amax) {
  const uint32_t b = __float_as_uint(amax);
  if (b == 0) return 127;
  const int e = (int)(b >> 23) - 127 - (FMT == TG_FP8_E4M3 ? 8 : 15) + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)((e < -126 ? -126 : e) + 127);
}
__device__ __forceinline__ float inverse_scale(uint32_t code) { return __uint_as_float((254u - code) << 23); }

// four values -> four bytes; |v| <= largest(type) but for NaN and infinity
template <int FMT>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int w = 0;
  if constexpr (FMT == TG_FP8_E4M3) {
    w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
  }
  return (uint32_t)w;
}

// infinities of e4m3 become NaN before the conversion, so that nothing depends on its overflow mode
template <int FMT>
__device__ __forceinline__ float storable(float v) {
  if (FMT == TG_FP8_E4M3 && fabsf(v) == __builtin_inff()) return __builtin_nanf("");
  return v;
}

struct FqP {
  const void* x;
  unsigned char *q, *s, *qt, *st;
  int64_t rows, cols, ldx, cp, rp, sp, stp;                          // padded columns / rows, scale pitches
  int tiles_c, tile, vec;
};

template <typename T, int FMT>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(FqP p) {
  __shared__ __attribute__((aligned(16))) unsigned char sh[128 * FQ_PITCH];
  __shared__ float smax[4][128];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, wave = tid >> 6;
  const int64_t tr = blockIdx.x / p.tiles_c, tc = blockIdx.x - tr * p.tiles_c;
  const int64_t r0 = tr * 128 + ty * 8, c0 = tc * 128 + tx * 8;
  const int have = p.cols - c0 >= 8 ? 8 : (p.cols - c0 > 0 ? (int)(p.cols - c0) : 0);
  float v[8][8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    load8q<T>(static_cast<const T*>(p.x) + (r0 + j) * p.ldx + c0, r0 + j < p.rows ? have : 0, p.vec != 0, v[j]);

  uint32_t code_tile = 0;
  if (p.tile) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmaxf(m, finite_abs(v[j][k]));
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((tid & 63) == 0) smax[wave][0] = m;
    __syncthreads();
    m = fmaxf(fmaxf(smax[0][0], smax[1][0]), fmaxf(smax[2][0], smax[3][0]));
    code_tile = scale_code<FMT>(m);
    if (tid == 0) {
      if (p.q) p.s[tr * p.sp + tc] = (unsigned char)code_tile;
      if (p.qt) p.st[tc * p.stp + tr] = (unsigned char)code_tile;
    }
  }
  if (p.q) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t code = code_tile;
      if (!p.tile) {
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, finite_abs(v[j][k]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        code = scale_code<FMT>(m);
      }
      const float i = inverse_scale(code);
      if (r0 + j < p.rows) {
        uint2 w;
        w.x = pack4<FMT>(storable<FMT>(v[j][0] * i), storable<FMT>(v[j][1] * i), storable<FMT>(v[j][2] * i), storable<FMT>(v[j][3] * i));
        w.y = pack4<FMT>(storable<FMT>(v[j][4] * i), storable<FMT>(v[j][5] * i), storable<FMT>(v[j][6] * i), storable<FMT>(v[j][7] * i));
        *reinterpret_cast<uint2*>(p.q + (r0 + j) * p.cp + c0) = w;
        if (!p.tile && tx == 0) p.s[(r0 + j) * p.sp + tc] = (unsigned char)code;
      }
    }
  }
  if (p.qt) {
    float inv[8];
    if (p.tile) {
#pragma unroll
      for (int k = 0; k < 8; ++k) inv[k] = inverse_scale(code_tile);
    } else {
      float m[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        m[k] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m[k] = fmaxf(m[k], finite_abs(v[j][k]));
        m[k] = fmaxf(m[k], __shfl_xor(m[k], 16, 64));
        m[k] = fmaxf(m[k], __shfl_xor(m[k], 32, 64));
      }
      if ((tid & 63) < 16) {
#pragma unroll
        for (int k = 0; k < 8; ++k) smax[wave][tx * 8 + k] = m[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = tx * 8 + k;
        const uint32_t code = scale_code<FMT>(fmaxf(fmaxf(smax[0][c], smax[1][c]), fmaxf(smax[2][c], smax[3][c])));
        inv[k] = inverse_scale(code);
        if (ty == 0 && c0 + k < p.cols) p.st[(c0 + k) * p.stp + tr] = (unsigned char)code;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint2 w;
      w.x = pack4<FMT>(storable<FMT>(v[0][k] * inv[k]), storable<FMT>(v[1][k] * inv[k]), storable<FMT>(v[2][k] * inv[k]), storable<FMT>(v[3][k] * inv[k]));
      w.y = pack4<FMT>(storable<FMT>(v[4][k] * inv[k]), storable<FMT>(v[5][k] * inv[k]), storable<FMT>(v[6][k] * inv[k]), storable<FMT>(v[7][k] * inv[k]));
      *reinterpret_cast<uint2*>(sh + (tx * 8 + k) * FQ_PITCH + ty * 8) = w;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int slot = tid + 256 * i, c = slot >> 3, ch = slot & 7;
      if (tc * 128 + c < p.cols)
        *reinterpret_cast<uint4*>(p.qt + (tc * 128 + c) * p.rp + tr * 128 + ch * 16) = *reinterpret_cast<const uint4*>(sh + c * FQ_PITCH + ch * 16);
    }
  }
  // the unused bytes behind the last block of a scale row
  if (p.q && tc == p.tiles_c - 1) {
    const int pad = (int)(p.sp - p.tiles_c);
    if (p.tile) {
      if (tid < pad) p.s[tr * p.sp + p.tiles_c + tid] = 127;
    } else {
      for (int e = tid; e < 128 * pad; e += 256)
        if (tr * 128 + e / pad < p.rows) p.s[(tr * 128 + e / pad) * p.sp + p.tiles_c + e % pad] = 127;
    }
  }
  const int64_t tiles_r = p.rp / 128;
  if (p.qt && tr == tiles_r - 1) {
    const int pad = (int)(p.stp - tiles_r);
    if (p.tile) {
      if (tid < pad) p.st[tc * p.stp + tiles_r + tid] = 127;
    } else {
      for (int e = tid; e < 128 * pad; e += 256)
        if (tc * 128 + e / pad < p.cols) p.st[(tc * 128 + e / pad) * p.stp + tiles_r + e % pad] = 127;
    }
  }
}

}  // namespace

#define ST(s) static_cast<hipStream_t>(s)

extern "C" int tg_fp8_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int fmt, int tile, void* q,
                               void* scale, void* qt, void* scale_t, void* stream) {
  TG_CHECK_ARG(dtype == TG_F32 || dtype == TG_BF16, "bad dtype");
  TG_CHECK_ARG(fmt == TG_FP8_E4M3 || fmt == TG_FP8_E5M2, "bad 8-bit type");
  TG_CHECK_ARG(rows >= 0 && cols >= 0 && rows < ((int64_t)1 << 31) && cols < ((int64_t)1 << 31), "rows and cols must lie in [0, 2^31)");
  if (rows == 0 || cols == 0) return TG_OK;
  TG_CHECK_ARG(x != nullptr && ldx >= cols, "x is missing, or its row stride is below cols");
  TG_CHECK_ARG(q != nullptr || qt != nullptr, "neither order is asked for");
  TG_CHECK_ARG((q == nullptr) == (scale == nullptr) && (qt == nullptr) == (scale_t == nullptr), "a copy goes with its scales");
  TG_CHECK_ARG((((uintptr_t)q | (uintptr_t)qt) & 15) == 0 && (((uintptr_t)scale | (uintptr_t)scale_t) & 3) == 0,
               "q, qt must be 16-byte and their scales 4-byte aligned");
  const int64_t tiles_r = cdiv64(rows, 128), tiles_c = cdiv64(cols, 128);
  TG_CHECK_ARG(tiles_r * tiles_c < ((int64_t)1 << 31), "too many 128 x 128 tiles");
  FqP p = {};
  p.x = x;
  p.q = static_cast<unsigned char*>(q); p.s = static_cast<unsigned char*>(scale);
  p.qt = static_cast<unsigned char*>(qt); p.st = static_cast<unsigned char*>(scale_t);
  p.rows = rows; p.cols = cols; p.ldx = ldx;
  p.cp = tiles_c * 128; p.rp = tiles_r * 128;
  p.sp = cdiv64(tiles_c, 4) * 4; p.stp = cdiv64(tiles_r, 4) * 4;
  p.tiles_c = (int)tiles_c;
  p.tile = tile != 0;
  const int es = dtype == TG_F32 ? 4 : 2;
  p.vec = ((uintptr_t)x & 15) == 0 && (ldx * es) % 16 == 0;
  const char* const name = "fp8_quantize";
  const double n = (double)rows * cols, bytes = n * (es + (q ? 1 : 0) + (qt ? 1 : 0));
  const dim3 grid((unsigned)(tiles_r * tiles_c)), block(256);
  if (dtype == TG_F32) {
    if (fmt == TG_FP8_E4M3) TG_LAUNCH(name, 4 * n, bytes, (fp8_quantize_kernel<float, TG_FP8_E4M3>), grid, block, 0, ST(stream), p);
    else TG_LAUNCH(name, 4 * n, bytes, (fp8_quantize_kernel<float, TG_FP8_E5M2>), grid, block, 0, ST(stream), p);
  } else {
    if (fmt == TG_FP8_E4M3) TG_LAUNCH(name, 4 * n, bytes, (fp8_quantize_kernel<u16, TG_FP8_E4M3>), grid, block, 0, ST(stream), p);
    else TG_LAUNCH(name, 4 * n, bytes, (fp8_quantize_kernel<u16, TG_FP8_E5M2>), grid, block, 0, ST(stream), p);
  }
  TG_CHECK_LAUNCH();
}
