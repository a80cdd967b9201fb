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
//
// Measured on one device: [8192, 4096] bf16 28 us in one order = 3.6 TB/s, 34 us in both = 3.9.
#include "fp8.h"

namespace {

constexpr int FQ_PITCH = 144;

struct FqP {
  const void* x;
  unsigned char *q, *s, *qt, *st;
  int64_t rows, cols, ldx, cp, rp, sp, stp;                          // padded columns / rows, scale pitches
  int tiles_c, tile, vec;
};

// bits of the largest absolute values of a thread's 8 columns, over the wave's 32 rows
template <bool BAD>
__device__ __forceinline__ void column_most(const Fp8In16 (&v)[8], uint32_t (&m)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    u16x2q a = v[0].abs2<BAD>(k);
#pragma unroll
    for (int j = 1; j < 8; ++j) a = __builtin_elementwise_max(a, v[j].abs2<BAD>(k));
    a = __builtin_elementwise_max(a, __builtin_bit_cast(u16x2q, __shfl_xor(__builtin_bit_cast(int, a), 16, 64)));
    a = __builtin_elementwise_max(a, __builtin_bit_cast(u16x2q, __shfl_xor(__builtin_bit_cast(int, a), 32, 64)));
    m[2 * k] = (uint32_t)a[0] << 16;
    m[2 * k + 1] = (uint32_t)a[1] << 16;
  }
}
template <bool BAD>
__device__ __forceinline__ void column_most(const Fp8In32 (&v)[8], uint32_t (&m)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    m[k] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m[k] = max(m[k], v[j].abs1<BAD>(k));
    m[k] = max(m[k], (uint32_t)__shfl_xor((int)m[k], 16, 64));
    m[k] = max(m[k], (uint32_t)__shfl_xor((int)m[k], 32, 64));
  }
}
// a thread's 8 columns of 8 rows as bytes, column by column
template <int FMT, bool BAD>
__device__ __forceinline__ void columns_out(const Fp8In16 (&v)[8], const uint32_t (&code)[8], unsigned char* out) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    uint32_t d[4];                                                      // column k of rows 2 i, 2 i + 1
#pragma unroll
    for (int i = 0; i < 4; ++i)
      d[i] = Fp8In16::storable<FMT, BAD>(__builtin_amdgcn_perm(v[2 * i + 1].word(k >> 1), v[2 * i].word(k >> 1), k & 1 ? 0x07060302u : 0x05040100u));
    uint2 w;
    w.x = fp8_pair<FMT, true>(fp8_pair<FMT, false>(0, d[0], code[k]), d[1], code[k]);
    w.y = fp8_pair<FMT, true>(fp8_pair<FMT, false>(0, d[2], code[k]), d[3], code[k]);
    *reinterpret_cast<uint2*>(out + k * FQ_PITCH) = w;
  }
}
template <int FMT, bool BAD>
__device__ __forceinline__ void columns_out(const Fp8In32 (&v)[8], const uint32_t (&code)[8], unsigned char* out) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    float d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = Fp8In32::storable<FMT, BAD>(v[j].value(k));
    uint2 w;
    w.x = fp8_pair<FMT, true>(fp8_pair<FMT, false>(0, d[0], d[1], code[k]), d[2], d[3], code[k]);
    w.y = fp8_pair<FMT, true>(fp8_pair<FMT, false>(0, d[4], d[5], code[k]), d[6], d[7], code[k]);
    *reinterpret_cast<uint2*>(out + k * FQ_PITCH) = w;
  }
}

template <typename T, int FMT>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(FqP p) {
  __shared__ __attribute__((aligned(16))) unsigned char sh[128 * FQ_PITCH];
  __shared__ uint32_t smax[4][128];
  using In = typename Fp8In<T>::type;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, wave = tid >> 6;
  const int64_t tr = blockIdx.x / p.tiles_c, tc = blockIdx.x - tr * p.tiles_c;
  const int64_t r0 = tr * 128 + ty * 8, c0 = tc * 128 + tx * 8;
  const int have = p.cols - c0 >= 8 ? 8 : (p.cols - c0 > 0 ? (int)(p.cols - c0) : 0);
  In v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (r0 + j < p.rows && have > 0) v[j].load(static_cast<const T*>(p.x) + (r0 + j) * p.ldx + c0, have, p.vec != 0);
    else v[j].zero();
  }
  uint32_t mr[8], ma = 0;                                               // bits of the largest absolute value: of each row, of all
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    mr[j] = v[j].template most<false>();
    ma = ma > mr[j] ? ma : mr[j];
  }
  const bool bad = __any(ma >= FP8_INF);
  if (bad) {
    ma = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mr[j] = v[j].template most<true>();
      ma = ma > mr[j] ? ma : mr[j];
    }
  }
  uint32_t code_tile = 0;
  if (p.tile) {
    ma = fp8_max16(ma);
    ma = max(ma, (uint32_t)__shfl_xor((int)ma, 16, 64));
    ma = max(ma, (uint32_t)__shfl_xor((int)ma, 32, 64));
    if ((tid & 63) == 0) smax[wave][0] = ma;
    __syncthreads();
    code_tile = fp8_scale_code<FMT>(max(max(smax[0][0], smax[1][0]), max(smax[2][0], smax[3][0])));
    if (tid == 0) {
      if (p.q) p.s[tr * p.sp + tc] = (unsigned char)code_tile;
      if (p.qt) p.st[tc * p.stp + tr] = (unsigned char)code_tile;
    }
  }
  if (p.q) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t code = p.tile ? code_tile : fp8_scale_code<FMT>(fp8_max16(mr[j]));
      if (r0 + j < p.rows) {
        *reinterpret_cast<uint2*>(p.q + (r0 + j) * p.cp + c0) = bad ? v[j].template pack<FMT, true>(code) : v[j].template pack<FMT, false>(code);
        if (!p.tile && tx == 0) p.s[(r0 + j) * p.sp + tc] = (unsigned char)code;
      }
    }
  }
  if (p.qt) {
    uint32_t code[8];
    if (p.tile) {
#pragma unroll
      for (int k = 0; k < 8; ++k) code[k] = code_tile;
    } else {
      uint32_t m[8];                                                    // of the 8 columns, over the wave's 32 rows
      if (bad) column_most<true>(v, m);
      else column_most<false>(v, m);
      if ((tid & 63) < 16) {
#pragma unroll
        for (int k = 0; k < 8; ++k) smax[wave][tx * 8 + k] = m[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = tx * 8 + k;
        code[k] = fp8_scale_code<FMT>(max(max(smax[0][c], smax[1][c]), max(smax[2][c], smax[3][c])));
        if (ty == 0 && c0 + k < p.cols) p.st[(c0 + k) * p.stp + tr] = (unsigned char)code[k];
      }
    }
    if (bad) columns_out<FMT, true>(v, code, sh + tx * 8 * FQ_PITCH + ty * 8);
    else columns_out<FMT, false>(v, code, sh + tx * 8 * FQ_PITCH + ty * 8);
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
