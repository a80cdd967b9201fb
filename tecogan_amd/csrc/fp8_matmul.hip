// out[m][n] = sum over blocks kb of 128 of 2^(ea[m, kb] + eb[n, kb]) sum_k a[m][k] b[n][k]  (+ bias[n]) (+ out[m][n])
//
// a [M][K], b [N][K] in 8-bit floating point (e4m3 or e5m2 each), K a multiple of 128 (tg_fp8_quantize pads rows with zeros); the
// scales' biased exponents one byte for a row and 128 columns, or for a tile of 128 x 128.  Two ways through the matrix unit:
//
//   whole sums: the operands are widened to bf16 with their scales in registers (v_cvt_scalef32_pk_bf16_fp8: exact, 4 bits of mantissa,
//     as long as the scaled values lie in fp32's normal range) and multiplied by v_mfma_f32_16x16x32_bf16, whose sums are fp32
//     throughout: half the rate of the 8-bit instruction.
//   fast (bf16 outputs, asked for by the caller): v_mfma_scale_f32_16x16x128 covers 16 x 16 outputs over exactly one block of K with the
//     scales of its 16 rows and 16 columns as operands.  The products of 8 neighbouring k are aligned to the largest sum of exponents E
//     among them and cut to multiples of 2^(E - 13) before they are added (found by adding small products to a large one; the unscaled
//     8-bit instructions do the same); the sums over the groups and blocks are fp32.  Measured 1.5e-5 of the result for normal operands,
//     7e-5 where a few channels carry it, the same for any K -- but where large products of one group cancel, what is left of the others
//     is lost (256 - 256 + 6 x 15 x 2^-9: 0, not 0.18).  Hence the caller's choice.
//
// Measured on one device, 8192 x 8192 x 4096: whole sums 371 - 394 us = 1480 - 1400 TFLOP/s (bf16 out), 398 - 416 us (f32 out);
// fast 212 - 250 us = 2600 - 2200.  1 x 4096 x 4096 from bf16 rows 9 us.
//
// The instruction's rows are n and its columns m: a lane holds four neighbouring n of one m.
#include "fp8.h"
#include <type_traits>

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4m __attribute__((ext_vector_type(4)));

struct MmP {
  const unsigned char *a, *b, *sa, *sb;
  const float* bias;
  void* out;
  int64_t M, N, ldo;
  int tiles_m, tiles_n, tiles;
  int K, sp;                                                          // bytes of a row, of a row of scales
  int sh_a, sh_b;                                                     // row -> row of scales: 0, or 7 for tiles
  int out_bf16, accumulate, vec;
};

// c += b a over a block of K, in place: written as assembly because the compiler, left to choose, gives the 64 accumulators of the
// largest tile other registers from one product to the next and copies them back (1300 moves a block of K).  The wait states in
// front cover a scale or a widened operand that vector instructions have just written (two states; the matrix unit is busy with the
// product before, so they cost nothing); results are read by nothing but the next product into the same registers until settle().
// The instruction's format codes: 0 e4m3, 1 e5m2.
template <int FB, int FA>
__device__ __forceinline__ void mfma_block(f32x4& c, i32x8 b, i32x8 a, int sb, int sa) {
#ifdef __HIP_DEVICE_COMPILE__                                           // the host pass does not know the registers
  asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:%5 blgp:%6"
               : "+a"(c) : "v"(b), "v"(a), "v"(sb), "v"(sa), "n"(FB), "n"(FA));
#endif
}
__device__ __forceinline__ void mfma_wide(f32x4& c, bf16x8 b, bf16x8 a) {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(b), "v"(a));
#endif
}
// Results are whole from here on: 32 wait states behind the last product (16 passes at most), then every accumulator passes an
// empty statement so that no read of it is moved in front.
template <int N>
__device__ __forceinline__ void settle(f32x4 (&c)[N]) {
#ifdef __HIP_DEVICE_COMPILE__
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+a"(c[i]));
#endif
}

typedef __bf16 bf16x2m __attribute__((ext_vector_type(2)));

// Values that have been loaded are there from here on: without it every branch behind waits for them again, and for all stores with them.
template <int N>
__device__ __forceinline__ void arrived(f32x4 (&c)[N]) {
#ifdef __HIP_DEVICE_COMPILE__
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(c[i]));
#endif
}

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

// the lane's number, counted anew where this stands
__device__ __forceinline__ int lane_again() {
#ifdef __HIP_DEVICE_COMPILE__
  uint32_t all = ~0u;
  asm volatile("" : "+s"(all));
  return (int)__builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0u));
#else
  return 0;
#endif
}

typedef __attribute__((address_space(3))) void lds_void_m;
// 16 (4) bytes a lane from rsrc[voff + soff] to lds + 16 (4) lane
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rsrc, unsigned char* lds, int voff, int soff) {   // 4 bytes a lane
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_m*)lds, 4, voff, soff, 0, 0);
}
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rsrc, unsigned char* lds, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_m*)lds, 16, voff, soff, 0, 0);
}

// 32 MF x 32 NF outputs, four waves of 16 MF x 16 NF.  A stage of LDS holds one block of K of both operands, rows of 128 bytes, filled
// by 16-byte DMA from global memory, and the scale dwords of its rows; S stages in turn.  The 16-byte chunk c of row r sits at chunk
// c ^ ((r >> 1) & 7) (chosen on the global side): a lane's 32 bytes are chunks g and g + 4 (g = lane / 16) in both operands -- any
// order of k serves -- and the 16 lanes that a ds_read_b128 serves together cover all 64 banks once.
//
// A block of K is four quarters: half of the wave's rows x half of its columns, (a0, b0), (a0, b1), (a1, b1), (a1, b0).  Between a
// quarter's products the fragments that the next quarters need are read, each into the registers of the one that has just been used
// up: b1, a1 of this block, then a0 and -- column by column, as (a1, b0) finishes with them -- b0 of the next.  The one barrier of a
// block sits in its middle: there every wave has read the last of this stage and its own DMA of the next stage has landed; the DMA
// of block kb + S goes out between the products of the second half.
//
// G groups of four waves share a tile: group j takes the blocks j, j + G, ... of K through stages of its own, and the groups' sums meet in
// LDS in the groups' order.  A block of the smallest tile costs its waves
// about 800 cycles, most of them waits (barrier, LDS, products, in turn); G groups wait at the same time.
// WIDE: whole sums, either output type; otherwise the 8-bit instruction's, bf16 outputs.
template <int FB, int FA, bool WIDE, int MF, int NF, int S, int G>
__global__ __launch_bounds__(256 * G, MF * NF >= 64 || G > 1 ? 1 : 2) void fp8_tile_kernel(MmP p) {
  constexpr int TM = 32 * MF, TN = 32 * NF, STAGE = (TM + TN) * 132, HM = MF / 2, HN = NF / 2;
  extern __shared__ __attribute__((aligned(16))) unsigned char tile_lds[];
  const int tid = threadIdx.x;
  int lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int grp = G > 1 ? __builtin_amdgcn_readfirstlane(tid >> 8) : 0, wave = __builtin_amdgcn_readfirstlane((tid >> 6) & 3);
  const int wm = wave >> 1, wn = wave & 1;
  unsigned char* const smem = tile_lds + grp * S * STAGE;
  // tile of this workgroup: XCD x (linear id % 8) owns consecutive tiles of an order that walks 8 tile rows down before the next column
  int t = blockIdx.x;
  {
    const int full = p.tiles / 8 * 8;
    if (t < full) t = (t & 7) * (full / 8) + (t >> 3);
  }
  const int band = t / (8 * p.tiles_n), rest = t - band * 8 * p.tiles_n, left = p.tiles_m - band * 8, deep = left < 8 ? left : 8;
  const int64_t m0 = (int64_t)__builtin_amdgcn_readfirstlane(band * 8 + rest % deep) * TM;
  const int64_t n0 = (int64_t)__builtin_amdgcn_readfirstlane(rest / deep) * TN;

  const int rows_a = (int)(p.M - m0 < TM ? p.M - m0 : TM), rows_b = (int)(p.N - n0 < TN ? p.N - n0 : TN);
  const int all = p.K >> 7, turns = (all + G - 1) / G, nkb = (all - grp + G - 1) / G;   // blocks of K, of the busiest group, of this one
  const auto rsrcA = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.a + m0 * p.K), 0, rows_a * p.K, 0x00020000);
  const auto rsrcB = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.b + n0 * p.K), 0, rows_b * p.K, 0x00020000);
  int oa[MF], ob[NF];                                                 // DMA sources: rows past the end read the last one (not stored)
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int row = (wave * MF + i) * 8 + (lane >> 3);
    oa[i] = (row < rows_a ? row : rows_a - 1) * p.K + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  }
#pragma unroll
  for (int i = 0; i < NF; ++i) {
    const int row = (wave * NF + i) * 8 + (lane >> 3);
    ob[i] = (row < rows_b ? row : rows_b - 1) * p.K + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  }
  auto dma_at = [&](int q, int stage, int i) {                        // instruction q of the group's block i into stage % S
    const int kb = grp + G * i;
    unsigned char* const st = smem + (stage & (S - 1)) * STAGE;
    if (q < MF) dma16(rsrcA, st + (wave * MF + q) * 1024, oa[q < MF ? q : 0], kb * 128);
    else dma16(rsrcB, st + TM * 128 + (wave * NF + q - MF) * 1024, ob[q < MF ? 0 : q - MF], kb * 128);
  };
  // scales: a dword DMA takes the four bytes around block kb of 64 rows
  const auto rsrcSA = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.sa + (m0 >> p.sh_a) * p.sp), 0, (((rows_a - 1) >> p.sh_a) + 1) * p.sp, 0x00020000);
  const auto rsrcSB = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.sb + (n0 >> p.sh_b) * p.sp), 0, (((rows_b - 1) >> p.sh_b) + 1) * p.sp, 0x00020000);
  constexpr int NCH = (TM + TN) / 64, NS = NCH >= 4 ? NCH / 4 : 1;     // 64 rows each; with fewer than four, waves fetch the same
  int os[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int ch = (wave + 4 * i) % NCH, row = (ch * 64 < TM ? ch * 64 : ch * 64 - TM) + lane;
    if (ch * 64 < TM) os[i] = ((row < rows_a ? row : rows_a - 1) >> p.sh_a) * p.sp;
    else os[i] = ((row < rows_b ? row : rows_b - 1) >> p.sh_b) * p.sp;
  }
  auto dma_scales_at = [&](int stage, int k) {
    const int at = (grp + G * k) & ~3;
    unsigned char* const st = smem + (stage & (S - 1)) * STAGE + (TM + TN) * 128;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int ch = (wave + 4 * i) % NCH;
      if (ch * 64 < TM) dma4(rsrcSA, st + ch * 256, os[i], at);
      else dma4(rsrcSB, st + ch * 256, os[i], at);
    }
  };

  f32x4 acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  i32x8 fa[2][HM], fb[2][HN];
  int ca[2][HM], cb[2][HN];
  // this lane's addresses in the stage that is read: low and high chunks of a fragment, its scale
  const int la = r16 * 128 + ((g ^ (r16 >> 1)) << 4);
  const unsigned char* const bal = smem + wm * 16 * MF * 128 + la;
  const unsigned char* const bah = smem + ((wm * 16 * MF * 128 + la) ^ 64);
  const unsigned char* const bbl = smem + TM * 128 + wn * 16 * NF * 128 + la;
  const unsigned char* const bbh = smem + ((TM * 128 + wn * 16 * NF * 128 + la) ^ 64);
  const unsigned char* const psa = smem + (TM + TN) * 128 + (wm * 16 * MF + r16) * 4;
  const unsigned char* const psb = smem + (TM + TN) * 128 + (TM + wn * 16 * NF + r16) * 4;
  const unsigned char *pal = bal, *pah = bah, *pbl = bbl, *pbh = bbh, *qsa = psa + (G > 1 ? grp & 3 : 0), *qsb = psb + (G > 1 ? grp & 3 : 0);
  auto frag = [](const unsigned char* lo, const unsigned char* hi) {
    return __builtin_shufflevector(*reinterpret_cast<const i32x4m*>(lo), *reinterpret_cast<const i32x4m*>(hi), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto read_a = [&](int h, int u) {
    fa[h][u] = frag(pal + (h * HM + u) * 2048, pah + (h * HM + u) * 2048);
    ca[h][u] = qsa[(h * HM + u) * 64];
  };
  auto read_b = [&](int h, int u) {
    fb[h][u] = frag(pbl + (h * HN + u) * 2048, pbh + (h * HN + u) * 2048);
    cb[h][u] = qsb[(h * HN + u) * 64];
  };
  // what is read from here on is the group's block kb
  int shift = STAGE;
  auto turn = [&](int kb) {
    const int st = (kb & (S - 1)) * STAGE;
    if constexpr (S == 2) {                                           // no second set of addresses: the largest tile has no registers for it
      pal += shift; pah += shift; pbl += shift; pbh += shift;
      shift = -shift;
    } else {
      pal = bal + st; pah = bah + st; pbl = bbl + st; pbh = bbh + st;
    }
    qsa = psa + st + ((grp + G * kb) & 3);
    qsb = psb + st + ((grp + G * kb) & 3);
  };
  // A quarter's products, columns outermost; after(x) follows product x of HM HN
  auto quarter = [&](int ha, int hb, auto after) {
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < HN; ++j) {
        bf16x8 wb[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) wb[s] = widen<FB>(fb[hb][j][2 * s], fb[hb][j][2 * s + 1], __int_as_float(cb[hb][j] << 23));
#pragma unroll
        for (int i = 0; i < HM; ++i) {
          f32x4& c = acc[ha * HM + i][hb * HN + j];
#pragma unroll
          for (int s = 0; s < 4; ++s)
            mfma_wide(c, wb[s], widen<FA>(fa[ha][i][2 * s], fa[ha][i][2 * s + 1], __int_as_float(ca[ha][i] << 23)));
          after(j * HM + i);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < HN; ++j) {
#pragma unroll
        for (int i = 0; i < HM; ++i) {
          f32x4& c = acc[ha * HM + i][hb * HN + j];
          mfma_block<FB, FA>(c, fb[hb][j], fa[ha][i], cb[hb][j], ca[ha][i]);
          after(j * HM + i);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };
  constexpr int ND = MF + NF, N1 = HM * HN;
  if (nkb > 0) {
#pragma unroll
    for (int k = 0; k < S; ++k) {
      const int kb = k < nkb ? k : nkb - 1;
#pragma unroll
      for (int q = 0; q < ND; ++q) dma_at(q, k, kb);
      dma_scales_at(k, kb);
    }
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * (ND + NS)) : "memory");   // the first block has landed
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int u = 0; u < HM; ++u) read_a(0, u);
#pragma unroll
    for (int u = 0; u < HN; ++u) read_b(0, u);
    for (int kb = 0; kb < nkb; ++kb) {
      // behind the last block the DMA and the reads go on with the last block's data: nobody uses it
      const int ahead = kb + S < nkb ? kb + S : nkb - 1;
      quarter(0, 0, [&](int x) {
#pragma unroll
        for (int u = x * HN / N1; u < (x + 1) * HN / N1; ++u) read_b(1, u);
      });
      quarter(0, 1, [&](int x) {
#pragma unroll
        for (int u = x * HM / N1; u < (x + 1) * HM / N1; ++u) read_a(1, u);
      });
      // this wave's DMA of the next block has landed: at most that of the S - 2 blocks behind it may be under way
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 2) * (ND + NS)) : "memory");
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      turn(kb + 1);
      quarter(1, 1, [&](int x) {
#pragma unroll
        for (int u = x * HM / N1; u < (x + 1) * HM / N1; ++u) read_a(0, u);
#pragma unroll
        for (int q = x * MF / N1; q < (x + 1) * MF / N1; ++q) dma_at(q, kb, ahead);
        if (x == N1 - 1) dma_scales_at(kb, ahead);
      });
      quarter(1, 0, [&](int x) {
        if (x % HM == HM - 1) read_b(0, x / HM);
#pragma unroll
        for (int q = x * NF / N1; q < (x + 1) * NF / N1; ++q) dma_at(MF + q, kb, ahead);
      });
    }
    asm volatile("s_waitcnt vmcnt(0)\n\ts_nop 15\n\ts_nop 15" ::: "memory");   // no DMA outlives the workgroup
#pragma unroll
    for (int i = 0; i < MF; ++i) settle(acc[i]);
  } else if (G > 1 && all > 0) {                                       // a group without a block: the barrier in front of the loop
    __builtin_amdgcn_s_barrier();
  }
  lane = lane_again();                                                  // not kept over the loop: the largest tile has no register for it
  r16 = lane & 15;
  g = lane >> 4;
  if constexpr (G > 1) {
    if (nkb < turns) __builtin_amdgcn_s_barrier();                     // a group with one block less than the others
    __syncthreads();
    f32x4* const mine = reinterpret_cast<f32x4*>(tile_lds) + (grp * 4 + wave) * MF * NF * 64 + lane;
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) mine[(i * NF + j) * 64] = acc[i][j];
    __syncthreads();
  }
  auto sum_of = [&](int i, int j) {
    f32x4 v = acc[i][j];
    if constexpr (G > 1) {
      const f32x4* const sums = reinterpret_cast<const f32x4*>(tile_lds) + (wave * MF * NF + i * NF + j) * 64 + lane;
      v = sums[0];
#pragma unroll
      for (int q = 1; q < G; ++q) v += sums[q * 4 * MF * NF * 64];
    }
    return v;
  };
  // Everything that is loaded stands in front of the stores: a wait for a load waits for the stores before it too (8192 x 4096 x 2048 with a
  // bias: 81 us, read between them 102; 8192 x 8192 x 4096: 226 and 275)
  f32x4 bias[NF];
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    const int64_t n = n0 + wn * 16 * NF + 16 * j + 4 * g;
    bias[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (p.bias) {
      if (p.vec) {
        bias[j] = *reinterpret_cast<const f32x4*>(p.bias + (n < p.N ? n : p.N - 4));
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) bias[j][q] = p.bias[n + q < p.N ? n + q : p.N - 1];
      }
    }
  }
  arrived(bias);
  if (p.vec) {
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const int64_t m = m0 + wm * 16 * MF + 16 * i + r16;
      if (m >= p.M) continue;
      f32x4 prior[WIDE ? NF : 1];
      if constexpr (WIDE) {
        if (p.accumulate) {
#pragma unroll
          for (int j = 0; j < NF; ++j) {
            const int64_t n = n0 + wn * 16 * NF + 16 * j + 4 * g;
            prior[j] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p.out) + m * p.ldo + (n < p.N ? n : p.N - 4));
          }
          arrived(prior);
        }
      }
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        const int64_t n = n0 + wn * 16 * NF + 16 * j + 4 * g;
        if (n >= p.N || (G > 1 && (i * NF + j) % G != grp)) continue;   // each group writes its share
        f32x4 v = sum_of(i, j) + bias[j];
        if (!WIDE || p.out_bf16) {
          const bf16x2m lo = {(__bf16)v[0], (__bf16)v[1]}, hi = {(__bf16)v[2], (__bf16)v[3]};
          *reinterpret_cast<uint2*>(static_cast<u16*>(p.out) + m * p.ldo + n) = make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
        } else {
          if (p.accumulate) v += prior[j];
          *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + m * p.ldo + n) = v;
        }
      }
    }
    return;
  }
  // Rows of odd lengths: 16 rows at a time through a piece of LDS of this wave, so that a store instruction writes whole stretches of a row
  // ([6541, 2203] bf16, K = 128: 21 us, 2204 columns 15; values stored from where the products leave them, 2 bytes in 16 rows at once, 45)
  constexpr int WC = G > 1 ? 16 : 16 * NF, PITCH = WC + 4;
  __syncthreads();                                                     // the stages are free; the groups' sums stay
  float* const slab = reinterpret_cast<float*>(tile_lds + (G > 1 ? G * 4 * MF * NF * 1024 : 0)) + (grp * 4 + wave) * 16 * PITCH;
#pragma unroll
  for (int i = 0; i < MF; ++i) {
#pragma unroll
    for (int j0 = 0; j0 < NF; j0 += WC / 16) {
      if (G > 1 && (i * NF + j0) % G != grp) continue;
#pragma unroll
      for (int j = j0; j < j0 + WC / 16; ++j) *reinterpret_cast<f32x4*>(slab + r16 * PITCH + 16 * (j - j0) + 4 * g) = sum_of(i, j) + bias[j];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");               // between the lanes of a wave: in order
      const int64_t mr = m0 + wm * 16 * MF + 16 * i, nc = n0 + wn * 16 * NF + 16 * j0;
      const int cols = (int)(p.N - nc < WC ? p.N - nc : WC), rows = (int)(p.M - mr < 16 ? p.M - mr : 16);
      // this lane's columns (two where a row of the piece is wider than a wave) and, in every RS rows, its row
      constexpr int NB = WC > 64 ? WC / 64 : 1, RS = WC < 64 ? 64 / WC : 1;
      const int r0 = WC < 64 ? lane / WC : 0;
#pragma unroll
      for (int h = 0; h < NB; ++h) {
        const int c = (WC < 64 ? lane % WC : lane) + 64 * h;
        const float* const from = slab + r0 * PITCH + c;
        const int64_t at = (mr + r0) * p.ldo + nc + c;
        const int left = c < cols ? rows - r0 : 0;
        float v[16 / RS];
#pragma unroll
        for (int r = 0; r < 16; r += RS) v[r / RS] = from[r * PITCH];
        asm volatile("" ::: "memory");                                 // one wait for all of them
        if (left <= 0) continue;
        if (!WIDE || p.out_bf16) {
#pragma unroll
          for (int r = 0; r < 16; r += RS)
            if (r < left) (static_cast<u16*>(p.out) + at)[r * p.ldo] = f2bf(v[r / RS]);
        } else {
          float* const o = static_cast<float*>(p.out) + at;
          if (p.accumulate) {
            float prior[16 / RS];
#pragma unroll
            for (int r = 0; r < 16; r += RS) prior[r / RS] = o[(r < left ? r : 0) * p.ldo];
#pragma unroll
            for (int r = 0; r < 16; r += RS) v[r / RS] += prior[r / RS];
          }
#pragma unroll
          for (int r = 0; r < 16; r += RS)
            if (r < left) o[r * p.ldo] = v[r / RS];
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
}

// hipFuncAttributeMaxDynamicSharedMemorySize is not needed on this device; a launch may ask for up to 160 KB.
template <int FB, int FA, bool WIDE, int MF, int NF, int S, int G>
void launch_tile(MmP p, const char* name, double flops, double bytes, hipStream_t st) {
  p.tiles_m = (int)cdiv64(p.M, 32 * MF);
  p.tiles_n = (int)cdiv64(p.N, 32 * NF);
  p.tiles = p.tiles_m * p.tiles_n;
  constexpr int lds = G * S * (32 * MF + 32 * NF) * 132;
  static_assert(G == 1 || (MF * NF >= G && lds >= G * 4 * MF * NF * 1024), "the groups' sums lie in the stages");
  static_assert(lds >= (G > 1 ? G * 4 * MF * NF * 1024 : 0) + G * 4 * 16 * ((G > 1 ? 16 : 16 * NF) + 4) * 4, "and so do the rows on their way out");
  TG_LAUNCH(name, flops, bytes, (fp8_tile_kernel<FB, FA, WIDE, MF, NF, S, G>), dim3((unsigned)p.tiles), dim3(256 * G), lds, st, p);
}

// The largest tile that still gives most compute units one -- of the two larger ones (one and two a unit) the one whose last round of
// tiles is not the emptier by more than it is the faster (bf16 out, whole sums: 8192 x 8192 x 4096 394 and 438 us, 4096^3, one full round,
// 98 and 109; 4352 x 4096 x 4096, a second round of 16 tiles, 182 and 129, fast sums 103 and 95).  Over few blocks of K it is faster by
// less, since two tiles a unit hide each other's way out (K = 384, 6207 x 5696: 60 and 45, fast 48 and 42), for whole sums of several
// rounds not enough to count on (8192 x 8192 x 1024: f32 out 189 and 161, bf16 out 130 and 138).
// And what else of a unit a tile leaves free.  Fast sums: with at most one tile a unit its LDS holds more stages (1024 x 4096 x 4096: 28 us
// with two, 23 with four; whole sums 37 both) or a second group of waves (64 x 4096 x 4096: 12.1 us with one group, 10.8 with two, 12.5 with
// four of two stages).  Whole sums, where the widening takes its time: 19.5, 16.9 and 14.9; 512 rows, two tiles a unit, 26.5, 24 and 28.
template <int FB, int FA, bool WIDE>
void launch_formats(const MmP& p, const char* name, double flops, double bytes, hipStream_t st) {
  const int64_t cus = tg_num_cus();
  const int64_t t256 = cdiv64(p.M, 256) * cdiv64(p.N, 256), t128 = cdiv64(p.M, 128) * cdiv64(p.N, 128), t64 = cdiv64(p.M, 64) * cdiv64(p.N, 64);
  const int64_t places256 = cdiv64(t256, cus) * cus, places128 = cdiv64(t128, 2 * cus) * 2 * cus;
  const bool brief = p.K <= 1024;
  const int64_t gain = brief ? 114 : 125;                              // per cent
  const bool large = t256 * 5 >= cus * 4 && gain * t256 * places128 >= 100 * t128 * places256 && !(WIDE && brief && t256 > cus);
  if (large) {
    launch_tile<FB, FA, WIDE, 8, 8, 2, 1>(p, name, flops, bytes, st);
  } else if constexpr (WIDE) {
    if (t128 * 5 >= cus * 4) launch_tile<FB, FA, true, 4, 4, 2, 1>(p, name, flops, bytes, st);
    else if (t64 > 2 * cus) launch_tile<FB, FA, true, 2, 2, 4, 1>(p, name, flops, bytes, st);
    else if (t64 > cus) launch_tile<FB, FA, true, 2, 2, 2, 2>(p, name, flops, bytes, st);
    else launch_tile<FB, FA, true, 2, 2, 2, 4>(p, name, flops, bytes, st);
  } else {
    if (t128 > cus) launch_tile<FB, FA, false, 4, 4, 2, 1>(p, name, flops, bytes, st);
    else if (t128 * 5 >= cus * 4) launch_tile<FB, FA, false, 4, 4, 4, 1>(p, name, flops, bytes, st);
    else if (t64 > cus) launch_tile<FB, FA, false, 2, 2, 4, 1>(p, name, flops, bytes, st);
    else launch_tile<FB, FA, false, 2, 2, 4, 2>(p, name, flops, bytes, st);
  }
}

// Few rows of a: 16 columns n of the output for a workgroup, all M (at most 16 MF) rows.  Here the weight's bytes count: every wave
// streams its blocks of K (wave w those with kb % 8 = w: the waves of a workgroup read 1 KB of a row together) from memory straight
// into the operand's registers, four blocks in flight, and the waves' sums meet in LDS in a fixed order.  Both operands are widened to
// bf16 (there is time: fp32 sums for either output type).
// SRC: where a comes from -- 0, 1: 8-bit e4m3 / e5m2; 2, 3: bf16 / f32 values that are quantised here, as tg_fp8_quantize does it (at
// most 16 rows: one launch instead of two).
struct SkP {
  MmP m;
  const void* x;
  int64_t ldx;
  int cols, plain;                                                    // columns of x before padding; whole blocks, 16-byte aligned
};

constexpr int SK_WAVES = 8;

template <int FB, int SRC, int MF>
__global__ __launch_bounds__(64 * SK_WAVES) void fp8_skinny_kernel(SkP s) {
  constexpr int AHEAD = 4;                                              // blocks of K in flight
  using T = std::conditional_t<SRC == 3, float, u16>;
  using In = typename Fp8In<T>::type;
  const MmP& p = s.m;
  __shared__ float join[SK_WAVES][MF][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16, n = n0 + r16 < p.N ? n0 + r16 : p.N - 1;
  const int nkb = p.K >> 7;
  const unsigned char* const pb = p.b + n * p.K + g * 16;
  const unsigned char* const qb = p.sb + (n >> p.sh_b) * p.sp;
  int64_t m[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) m[i] = 16 * i + r16 < p.M ? 16 * i + r16 : p.M - 1;
  const T* const row = static_cast<const T*>(s.x) + (SRC >= 2 ? m[0] * s.ldx : 0);
  f32x4 acc[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k0 = wave; k0 < nkb; k0 += SK_WAVES * AHEAD) {
    i32x4m wl[AHEAD], wh[AHEAD], al[AHEAD][MF], ah[AHEAD][MF];
    In f[SRC >= 2 ? AHEAD : 1][4];
    int ws[AHEAD], as[AHEAD][MF];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int kb = k0 + u * SK_WAVES < nkb ? k0 + u * SK_WAVES : k0;   // past the end: loaded again, not used
      wl[u] = *reinterpret_cast<const i32x4m*>(pb + kb * 128);
      wh[u] = *reinterpret_cast<const i32x4m*>(pb + kb * 128 + 64);
      ws[u] = qb[kb];
      if constexpr (SRC >= 2) {
        const T* const at = row + kb * 128 + g * 16;                     // chunks g and g + 4 of the block: 2 x 16 values
        if (s.plain) {
#pragma unroll
          for (int h = 0; h < 4; ++h) f[u][h].load(at + (h >> 1) * 64 + (h & 1) * 8);
        } else {
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const int o = (h >> 1) * 64 + (h & 1) * 8, have = s.cols - (kb * 128 + g * 16 + o);
            f[u][h].load(at + o, have < 0 ? 0 : (have > 8 ? 8 : have), false);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < MF; ++i) {
          const unsigned char* const pa = p.a + m[i] * p.K + kb * 128 + g * 16;
          al[u][i] = *reinterpret_cast<const i32x4m*>(pa);
          ah[u][i] = *reinterpret_cast<const i32x4m*>(pa + 64);
          as[u][i] = p.sa[(m[i] >> p.sh_a) * p.sp + kb];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (k0 + u * SK_WAVES >= nkb) break;
      const float sb = __int_as_float(ws[u] << 23);
      const bf16x8 b[4] = {widen<FB>(wl[u][0], wl[u][1], sb), widen<FB>(wl[u][2], wl[u][3], sb), widen<FB>(wh[u][0], wh[u][1], sb),
                           widen<FB>(wh[u][2], wh[u][3], sb)};
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        i32x4m lo, hi;
        float sa;
        if constexpr (SRC < 2) {
          lo = al[u][i];
          hi = ah[u][i];
          sa = __int_as_float(as[u][i] << 23);
        } else {
          uint32_t most = max(max(f[u][0].template most<false>(), f[u][1].template most<false>()),
                              max(f[u][2].template most<false>(), f[u][3].template most<false>()));
          const bool bad = __any(most >= FP8_INF);
          if (bad)
            most = max(max(f[u][0].template most<true>(), f[u][1].template most<true>()),
                       max(f[u][2].template most<true>(), f[u][3].template most<true>()));
          most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));    // the four lanes of a row
          most = max(most, (uint32_t)__shfl_xor((int)most, 32, 64));
          const uint32_t code = fp8_scale_code<TG_FP8_E4M3>(most);
          sa = __uint_as_float(code << 23);
          uint2 w[4];
          if (bad) {
#pragma unroll
            for (int h = 0; h < 4; ++h) w[h] = f[u][h].template pack<TG_FP8_E4M3, true>(code);
          } else {
#pragma unroll
            for (int h = 0; h < 4; ++h) w[h] = f[u][h].template pack<TG_FP8_E4M3, false>(code);
          }
          lo = i32x4m{(int)w[0].x, (int)w[0].y, (int)w[1].x, (int)w[1].y};
          hi = i32x4m{(int)w[2].x, (int)w[2].y, (int)w[3].x, (int)w[3].y};
        }
        constexpr int FA = SRC == 1 ? 1 : 0;
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[0], widen<FA>(lo[0], lo[1], sa), acc[i], 0, 0, 0);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[1], widen<FA>(lo[2], lo[3], sa), acc[i], 0, 0, 0);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[2], widen<FA>(hi[0], hi[1], sa), acc[i], 0, 0, 0);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[3], widen<FA>(hi[2], hi[3], sa), acc[i], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MF; ++i) *reinterpret_cast<f32x4*>(&join[wave][i][r16 * 16 + 4 * g]) = acc[i];   // [m][n]
  __syncthreads();
  for (int e = tid; e < MF * 256; e += 64 * SK_WAVES) {
    const int64_t m = e >> 4, no = n0 + (e & 15);
    if (m >= p.M || no >= p.N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < SK_WAVES; ++w) v += join[w][e >> 8][e & 255];
    if (p.bias) v += p.bias[no];
    if (p.out_bf16) {
      static_cast<u16*>(p.out)[m * p.ldo + no] = f2bf(v);
    } else {
      float* const o = static_cast<float*>(p.out) + m * p.ldo + no;
      *o = p.accumulate ? *o + v : v;
    }
  }
}

template <int FB, int SRC>
void launch_skinny(const SkP& s, const char* name, double flops, double bytes, hipStream_t st) {
  const dim3 grid((unsigned)cdiv64(s.m.N, 16)), block(64 * SK_WAVES);
  const int mf = (int)cdiv64(s.m.M, 16);
  if (mf <= 1) TG_LAUNCH(name, flops, bytes, (fp8_skinny_kernel<FB, SRC, 1>), grid, block, 0, st, s);
  if constexpr (SRC < 2) {
    if (mf == 2) TG_LAUNCH(name, flops, bytes, (fp8_skinny_kernel<FB, SRC, 2>), grid, block, 0, st, s);
  }
}
// Up to 32 rows (4096 x 4096: 6.5 us with 1, 10 with 32 rows; with 64 the 64 x 64 tiles take 13, this kernel 15).  Quantising on the way
// costs every workgroup the whole of x again: with 4 blocks of K a wave in one round of workgroups 3.6 us, twice or four times that 8 - 12,
// against about 4.5 us for a launch of the quantiser.
constexpr int SK_ROWS = 32, SK_FUSED = 16;
bool skinny_fuses(int64_t M, int64_t N, int64_t nkb) {
  return M <= SK_FUSED && cdiv64(cdiv64(N, 16), tg_num_cus()) * cdiv64(nkb, SK_WAVES) <= 4;
}

bool al16m(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool tiles_ok(int64_t M, int64_t N) { return cdiv64(M, 64) * cdiv64(N, 64) < ((int64_t)1 << 27); }
bool fmt_ok(int f) { return f == TG_FP8_E4M3 || f == TG_FP8_E5M2; }

}  // namespace

#define ST(s) static_cast<hipStream_t>(s)

extern "C" int tg_fp8_matmul(const tg_fp8_matmul_desc* d, const void* a, const void* scale_a, const void* b, const void* scale_b,
                             const float* bias, void* out, void* stream) {
  TG_CHECK_ARG(d != nullptr, "null descriptor");
  TG_CHECK_ARG(d->M >= 0 && d->N >= 0 && d->M < ((int64_t)1 << 31) && d->N < ((int64_t)1 << 31), "M and N must lie in [0, 2^31)");
  TG_CHECK_ARG(d->K >= 0 && d->K % 128 == 0 && d->K <= (1 << 22), "K must be a multiple of 128 in [0, 2^22] (rows padded with zeros)");
  TG_CHECK_ARG(fmt_ok(d->a_fmt) && fmt_ok(d->b_fmt), "bad 8-bit type");
  TG_CHECK_ARG(d->out_dtype == TG_F32 || d->out_dtype == TG_BF16, "bad output type");
  TG_CHECK_ARG(!d->accumulate || d->out_dtype == TG_F32, "accumulation needs an f32 output");
  TG_CHECK_ARG(!d->fast || d->out_dtype == TG_BF16, "fast sums are for bf16 outputs");
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
  TG_CHECK_ARG(tiles_ok(d->M, d->N), "too many output tiles");
  const int oe = p.out_bf16 ? 2 : 4;
  p.vec = d->N % 4 == 0 && ((uintptr_t)out & (4 * oe - 1)) == 0 && d->ldo % 4 == 0 && al16m(bias);
  const int fa = d->a_fmt == TG_FP8_E5M2, fb = d->b_fmt == TG_FP8_E5M2;
  if (d->M <= SK_ROWS) {
    SkP k = {};
    k.m = p;
    if (fa && fb) launch_skinny<1, 1>(k, "fp8_skinny", flops, bytes, ST(stream));
    else if (fa) launch_skinny<0, 1>(k, "fp8_skinny", flops, bytes, ST(stream));
    else if (fb) launch_skinny<1, 0>(k, "fp8_skinny", flops, bytes, ST(stream));
    else launch_skinny<0, 0>(k, "fp8_skinny", flops, bytes, ST(stream));
    TG_CHECK_LAUNCH();
  }
#define MM_PICK(WIDEV)                                                                     \
  do {                                                                                     \
    if (fa && fb) launch_formats<1, 1, WIDEV>(p, name, flops, bytes, ST(stream));          \
    else if (fa) launch_formats<0, 1, WIDEV>(p, name, flops, bytes, ST(stream));           \
    else if (fb) launch_formats<1, 0, WIDEV>(p, name, flops, bytes, ST(stream));           \
    else launch_formats<0, 0, WIDEV>(p, name, flops, bytes, ST(stream));                   \
  } while (0)
  if (d->fast) MM_PICK(false);
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
  TG_CHECK_ARG(M >= 0 && N >= 0 && K >= 1 && M < ((int64_t)1 << 31) && N < ((int64_t)1 << 31) && K <= (1 << 22), "M, N in [0, 2^31) and K in [1, 2^22] are wanted");
  *bytes = linear_ws(M, K);
  return TG_OK;
}

extern "C" int tg_fp8_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* w, const void* scale_w, int64_t N,
                             int w_fmt, const float* bias, void* out, int out_dtype, int64_t ldo, void* ws, int64_t ws_bytes,
                             void* stream) {
  TG_CHECK_ARG(M >= 0 && N >= 0 && K >= 1 && M < ((int64_t)1 << 31) && N < ((int64_t)1 << 31) && K <= (1 << 22), "M, N in [0, 2^31) and K in [1, 2^22] are wanted");
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
  TG_CHECK_ARG(tiles_ok(M, N), "too many output tiles");
  if (skinny_fuses(M, N, kb)) {
    TG_CHECK_ARG(x != nullptr && ldx >= K && (dtype == TG_F32 || dtype == TG_BF16), "x is missing, its type unknown or its row stride below K");
    SkP k = {};
    k.m.b = static_cast<const unsigned char*>(w); k.m.sb = static_cast<const unsigned char*>(scale_w);
    k.m.bias = bias; k.m.out = out;
    k.m.M = M; k.m.N = N; k.m.ldo = ldo;
    k.m.K = (int)(kb * 128);
    k.m.sp = (int)cdiv64(kb, 4) * 4;
    k.m.sh_b = 7;
    k.m.out_bf16 = out_dtype == TG_BF16;
    k.x = x;
    k.ldx = ldx;
    k.cols = (int)K;
    k.plain = K % 128 == 0 && al16m(x) && (ldx * (dtype == TG_F32 ? 4 : 2)) % 16 == 0;
    const double flops = 2.0 * M * N * K, bytes = (double)N * K + (double)M * K * (dtype == TG_F32 ? 4 : 2) + (double)M * N * (k.m.out_bf16 ? 2 : 4);
    const char* const name = "fp8_skinny<quantise>";
    if (dtype == TG_BF16) {
      if (w_fmt == TG_FP8_E5M2) launch_skinny<1, 2>(k, name, flops, bytes, ST(stream));
      else launch_skinny<0, 2>(k, name, flops, bytes, ST(stream));
    } else {
      if (w_fmt == TG_FP8_E5M2) launch_skinny<1, 3>(k, name, flops, bytes, ST(stream));
      else launch_skinny<0, 3>(k, name, flops, bytes, ST(stream));
    }
    TG_CHECK_LAUNCH();
  }
  const int rc = tg_fp8_quantize(x, dtype, M, K, ldx, TG_FP8_E4M3, 0, q, s, nullptr, nullptr, stream);
  if (rc != TG_OK) return rc;
  return tg_fp8_matmul(&d, q, s, w, scale_w, bias, out, stream);
}
