// out[m][n] = sum over blocks kb of 128 of 2^(ea[m, kb] + eb[n, kb]) sum_k a[m][k] b[n][k]  (+ bias[n]) (+ out[m][n])
//
// a [M][K], b [N][K] in 8-bit floating point (e4m3 or e5m2 each), K a multiple of 128 (tg_fp8_quantize pads rows with zeros); the
// scales' biased exponents one byte for a row and 128 columns, or for a tile of 128 x 128.  Two ways through the matrix unit, chosen
// by the output's type:
//
//   bf16 outputs: v_mfma_scale_f32_16x16x128 covers 16 x 16 outputs over exactly one block of K with the scales of its 16 rows and 16
//     columns as operands (4.2 PFLOP/s issued back to back on one device).  The products of 8 neighbouring k are aligned to the largest
//     sum of exponents E among them and cut to multiples of 2^(E - 13) before they are added (found by adding small products to a
//     large one; the unscaled 8-bit instructions do the same): measured 1.5e-5 of the result for normal operands, 7e-5 where a few
//     channels carry it, the same for any K.  That is 25 - 100 times less than the rounding of the result to bf16; the sums over
//     the groups and blocks are fp32.
//   f32 outputs: the operands are widened to bf16 with their scales in registers (v_cvt_scalef32_pk_bf16_fp8: exact, 4 bits of
//     mantissa) and multiplied by v_mfma_f32_16x16x32_bf16, whose sums are fp32 throughout: half the rate, the accuracy that the type
//     promises (a weight gradient that is accumulated).
//
// The instruction's rows are n and its columns m: a lane holds four neighbouring n of one m.
#include "common.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4m __attribute__((ext_vector_type(4)));

struct MmP {
  const unsigned char *a, *b, *sa, *sb;
  const float* bias;
  void* out;
  int64_t M, N, ldo;
  int K, sp;                                                          // bytes of a row, of a row of scales
  int sh_a, sh_b;                                                     // row -> row of scales: 0, or 7 for tiles
  int out_bf16, accumulate, vec;
};

// the instruction's format codes: 0 e4m3, 1 e5m2
template <int FB, int FA>
__device__ __forceinline__ f32x4 mfma_block(i32x8 b, i32x8 a, f32x4 c, int sb, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, FB, FA, 0, sb, 0, sa);
}

typedef __bf16 bf16x2m __attribute__((ext_vector_type(2)));

// the 8 values of two dwords, times 2^(code - 127), as bf16
template <int F>
__device__ __forceinline__ bf16x8 widen(int lo, int hi, float scale) {
  bf16x2m v[4];
  if constexpr (F == 0) {
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  } else {
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, scale, false);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, scale, true);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, scale, false);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, scale, true);
  }
  return bf16x8{v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
}

// 128 x 128 outputs, four waves of 64 x 64.  LDS rows are the 128 bytes of one block of K; the 16-byte chunk c of row r sits at
// chunk c ^ ((r >> 1) & 7).  A lane's 32 bytes are chunks g and g + 4 (g = lane / 16) in both operands: any order of k serves.
template <int FB, int FA, bool WIDE>
__global__ __launch_bounds__(256) void fp8_matmul_kernel(MmP p) {
  __shared__ __attribute__((aligned(16))) unsigned char sA[128 * 128], sB[128 * 128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, g = lane >> 4;
  const int64_t nb = (p.N + 127) / 128, m0 = (int64_t)(blockIdx.x / nb) * 128, n0 = (int64_t)(blockIdx.x % nb) * 128;
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const unsigned char *ra[4], *rb[4];                                 // this thread's rows, clamped: what is past the end is not stored
  int64_t qa[4], qb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (tid + 256 * i) >> 3;
    const int64_t m = m0 + row < p.M ? m0 + row : p.M - 1, n = n0 + row < p.N ? n0 + row : p.N - 1;
    ra[i] = p.a + m * p.K + (tid & 7) * 16;
    rb[i] = p.b + n * p.K + (tid & 7) * 16;
    const int64_t ms = m0 + wm + 16 * i + r16, ns = n0 + wn + 16 * i + r16;
    qa[i] = ((ms < p.M ? ms : p.M - 1) >> p.sh_a) * p.sp;
    qb[i] = ((ns < p.N ? ns : p.N - 1) >> p.sh_b) * p.sp;
  }
  for (int k = 0; k < p.K; k += 128) {
    uint4 va[4], vb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      va[i] = *reinterpret_cast<const uint4*>(ra[i] + k);
      vb[i] = *reinterpret_cast<const uint4*>(rb[i] + k);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = tid + 256 * i, row = s >> 3, at = row * 128 + (((s & 7) ^ ((row >> 1) & 7)) << 4);
      *reinterpret_cast<uint4*>(sA + at) = va[i];
      *reinterpret_cast<uint4*>(sB + at) = vb[i];
    }
    __syncthreads();
    i32x8 fa[4], fb[4];
    int ca[4], cb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row_a = wm + 16 * i + r16, row_b = wn + 16 * i + r16;
      const i32x4m a0 = *reinterpret_cast<const i32x4m*>(sA + row_a * 128 + ((g ^ ((row_a >> 1) & 7)) << 4));
      const i32x4m a1 = *reinterpret_cast<const i32x4m*>(sA + row_a * 128 + (((g + 4) ^ ((row_a >> 1) & 7)) << 4));
      const i32x4m b0 = *reinterpret_cast<const i32x4m*>(sB + row_b * 128 + ((g ^ ((row_b >> 1) & 7)) << 4));
      const i32x4m b1 = *reinterpret_cast<const i32x4m*>(sB + row_b * 128 + (((g + 4) ^ ((row_b >> 1) & 7)) << 4));
      fa[i] = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
      fb[i] = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
      ca[i] = p.sa[qa[i] + (k >> 7)];
      cb[i] = p.sb[qb[i] + (k >> 7)];
    }
    if constexpr (WIDE) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        bf16x8 wa[4], wb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          wa[i] = widen<FA>(fa[i][2 * s], fa[i][2 * s + 1], __int_as_float(ca[i] << 23));
          wb[i] = widen<FB>(fb[i][2 * s], fb[i][2 * s + 1], __int_as_float(cb[i] << 23));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[j], wa[i], acc[i][j], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mfma_block<FB, FA>(fb[j], fa[i], acc[i][j], cb[j], ca[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + wm + 16 * i + r16;
    if (m >= p.M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t n = n0 + wn + 16 * j + 4 * g + q;
        if (n >= p.N) continue;
        float v = acc[i][j][q] + (p.bias ? p.bias[n] : 0.f);
        if (p.out_bf16) {
          static_cast<u16*>(p.out)[m * p.ldo + n] = f2bf(v);
        } else {
          float* o = static_cast<float*>(p.out) + m * p.ldo + n;
          *o = p.accumulate ? *o + v : v;
        }
      }
    }
  }
}

bool al16m(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool fmt_ok(int f) { return f == TG_FP8_E4M3 || f == TG_FP8_E5M2; }

}  // namespace

#define ST(s) static_cast<hipStream_t>(s)

extern "C" int tg_fp8_matmul(const tg_fp8_matmul_desc* d, const void* a, const void* scale_a, const void* b, const void* scale_b,
                             const float* bias, void* out, void* stream) {
  TG_CHECK_ARG(d != nullptr, "null descriptor");
  TG_CHECK_ARG(d->M >= 0 && d->N >= 0 && d->M < ((int64_t)1 << 31) && d->N < ((int64_t)1 << 31), "M and N must lie in [0, 2^31)");
  TG_CHECK_ARG(d->K >= 0 && d->K % 128 == 0 && d->K <= (1 << 24), "K must be a multiple of 128 in [0, 2^24] (rows padded with zeros)");
  TG_CHECK_ARG(fmt_ok(d->a_fmt) && fmt_ok(d->b_fmt), "bad 8-bit type");
  TG_CHECK_ARG(d->out_dtype == TG_F32 || d->out_dtype == TG_BF16, "bad output type");
  TG_CHECK_ARG(!d->accumulate || d->out_dtype == TG_F32, "accumulation needs an f32 output");
  if (d->M == 0 || d->N == 0) return TG_OK;
  TG_CHECK_ARG(out && (d->K == 0 || (a && scale_a && b && scale_b)), "null pointer");   // K == 0: the empty sum
  TG_CHECK_ARG(al16m(a) && al16m(b) && ((((uintptr_t)scale_a | (uintptr_t)scale_b) & 3) == 0), "a, b must be 16-byte and their scales 4-byte aligned");
  TG_CHECK_ARG(d->ldo >= d->N, "a row stride of out below N");
  MmP p = {};
  p.a = static_cast<const unsigned char*>(a); p.b = static_cast<const unsigned char*>(b);
  p.sa = static_cast<const unsigned char*>(scale_a); p.sb = static_cast<const unsigned char*>(scale_b);
  p.bias = bias; p.out = out;
  p.M = d->M; p.N = d->N; p.ldo = d->ldo;
  p.K = (int)d->K;
  p.sp = (int)cdiv64(d->K / 128, 4) * 4;
  p.sh_a = d->a_tile ? 7 : 0;
  p.sh_b = d->b_tile ? 7 : 0;
  p.out_bf16 = d->out_dtype == TG_BF16;
  p.accumulate = d->accumulate;
  const char* const name = "fp8_matmul";
  const double flops = 2.0 * d->M * d->N * d->K, bytes = (double)d->M * d->K + (double)d->N * d->K + (double)d->M * d->N * (p.out_bf16 ? 2 : 4);
  const int64_t blocks = cdiv64(d->M, 128) * cdiv64(d->N, 128);
  TG_CHECK_ARG(blocks < ((int64_t)1 << 31), "too many output tiles");
  const dim3 grid((unsigned)blocks), block(256);
  const int fa = d->a_fmt == TG_FP8_E5M2, fb = d->b_fmt == TG_FP8_E5M2;
#define MM_PICK(WIDEV)                                                                                                   \
  do {                                                                                                                   \
    if (fa && fb) TG_LAUNCH(name, flops, bytes, (fp8_matmul_kernel<1, 1, WIDEV>), grid, block, 0, ST(stream), p);        \
    else if (fa) TG_LAUNCH(name, flops, bytes, (fp8_matmul_kernel<0, 1, WIDEV>), grid, block, 0, ST(stream), p);         \
    else if (fb) TG_LAUNCH(name, flops, bytes, (fp8_matmul_kernel<1, 0, WIDEV>), grid, block, 0, ST(stream), p);         \
    else TG_LAUNCH(name, flops, bytes, (fp8_matmul_kernel<0, 0, WIDEV>), grid, block, 0, ST(stream), p);                 \
  } while (0)
  if (p.out_bf16) MM_PICK(false);
  else MM_PICK(true);
  TG_CHECK_LAUNCH();
}

namespace {
int64_t linear_ws(int64_t M, int64_t K) {
  const int64_t kb = cdiv64(K, 128);
  return (M * kb * 128 + M * cdiv64(kb, 4) * 4 + 15) / 16 * 16;
}
}  // namespace

extern "C" int tg_fp8_linear_ws(int64_t M, int64_t N, int64_t K, int64_t* bytes) {
  TG_CHECK_ARG(bytes != nullptr, "null pointer");
  TG_CHECK_ARG(M >= 0 && N >= 0 && K >= 1 && M < ((int64_t)1 << 31) && N < ((int64_t)1 << 31) && K <= (1 << 24), "M, N in [0, 2^31) and K in [1, 2^24] are wanted");
  *bytes = linear_ws(M, K);
  return TG_OK;
}

extern "C" int tg_fp8_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* w, const void* scale_w, int64_t N,
                             int w_fmt, const float* bias, void* out, int out_dtype, int64_t ldo, void* ws, int64_t ws_bytes,
                             void* stream) {
  TG_CHECK_ARG(M >= 0 && N >= 0 && K >= 1 && M < ((int64_t)1 << 31) && N < ((int64_t)1 << 31) && K <= (1 << 24), "M, N in [0, 2^31) and K in [1, 2^24] are wanted");
  if (M == 0 || N == 0) return TG_OK;
  TG_CHECK_ARG(ws != nullptr && al16m(ws) && ws_bytes >= linear_ws(M, K), "a workspace of tg_fp8_linear_ws() bytes is missing");
  const int64_t kb = cdiv64(K, 128);
  unsigned char* q = static_cast<unsigned char*>(ws);
  unsigned char* s = q + M * kb * 128;
  // the product's own checks first: nothing is launched where they fail
  tg_fp8_matmul_desc d = {};
  d.M = M; d.N = N; d.K = kb * 128; d.ldo = ldo;
  d.a_fmt = TG_FP8_E4M3; d.b_fmt = w_fmt; d.b_tile = 1; d.out_dtype = out_dtype;
  TG_CHECK_ARG(fmt_ok(w_fmt) && w && scale_w && out && al16m(w) && ((uintptr_t)scale_w & 3) == 0 && ldo >= N &&
                   (out_dtype == TG_F32 || out_dtype == TG_BF16), "bad weight or output");
  const int rc = tg_fp8_quantize(x, dtype, M, K, ldx, TG_FP8_E4M3, 0, q, s, nullptr, nullptr, stream);
  if (rc != TG_OK) return rc;
  return tg_fp8_matmul(&d, q, s, w, scale_w, bias, out, stream);
}
