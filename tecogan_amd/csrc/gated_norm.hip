// The boundary between two blocks of a network over rows of features, as one launch per direction:
//
//   u = post(o)                      norm after the block that ends        (none / RMS / layer)
//   v = alpha scale[c] act(gate) u   its gate and its residual scale
//   y = x + v                        the residual stream
//   h = pre(y)                       norm before the block that begins     (none / RMS / layer)
//
// with post, pre: z^ w + b, z^ = z / sqrt(mean(z^2) + eps) (RMS) or (z - mean) / sqrt(var + eps) (layer).
//
// About 14 (forward) / 40 (backward) operations a value against 10 - 32 bytes: bound by HBM.  Every tensor is read once and written
// once; a row stays in registers between its reductions.  A row belongs to LPR lanes (a power of two, 1 - 512) with 8 NV values
// each: 16-byte loads, reductions by lane exchange inside a wave and through LDS between the waves of a row.  All sums, statistics
// and gradients are fp32; h is taken from the fp32 y before y is rounded to its type (one rounding per output).  The backward pass
// takes the statistics again from y and o, which it has to read anyway: nothing is kept between the passes but the tensors.
// Parameter gradients: per-lane sums over the rows of a workgroup, one partial row per workgroup, then a second launch adds the
// partials in a fixed order (no atomics: the same inputs give the same bits).
//
// Measured on one device (a large copy: 5.17 TB/s): forward [16384, 4096] bf16 with a gate per row 132 us = 5.07 TB/s; [8, 2048] 3.8 us;
// backward [8192, 2048] bf16 beside an fp32 stream, shared gate rows, 70 + 4.8 us (rows, sums) = 4.3 TB/s; [77824, 64] fp32 29.4 + 4.5 us.
#include "common.h"

namespace {

typedef float f4v __attribute__((ext_vector_type(4)));

// A lane's 8 values of a vector: neighbours (VEC: 16-byte loads), or, where a row's length, stride or address is no multiple of 8
// values, every lpr-th: single loads in which a wave still reads one stretch of memory, and no case for a row's end (52600 rows of 775
// bf16 values: 162 us; 16 bytes at a time from odd addresses 401, and 776 values 83).
template <bool VEC> struct Cols {
  static __device__ __forceinline__ int first(int v, int lane, int lpr) { return VEC ? (v * lpr + lane) * 8 : v * lpr * 8 + lane; }
  static __device__ __forceinline__ int step(int lpr) { return VEC ? 1 : lpr; }
};

// The 8 values as they lie in memory: what is fetched a row ahead.  C: the row's columns, 0 for a row past the end, which reads nothing;
// values past them are 0.
template <typename T, bool VEC> struct Raw8;
template <> struct Raw8<u16, true> {
  uint4 w;
  __device__ __forceinline__ void load(const u16* __restrict__ row, int c, int, int C) {
    w = make_uint4(0, 0, 0, 0);
    if (c < C) w = *reinterpret_cast<const uint4*>(row + c);
  }
  __device__ __forceinline__ void values(float (&v)[8]) const { bf8_unpack(w, v); }
};
template <> struct Raw8<float, true> {
  f4v a, b;
  __device__ __forceinline__ void load(const float* __restrict__ row, int c, int, int C) {
    a = b = f4v{0.f, 0.f, 0.f, 0.f};
    if (c < C) {
      a = *reinterpret_cast<const f4v*>(row + c);
      b = *reinterpret_cast<const f4v*>(row + c + 4);
    }
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    v[0] = a[0]; v[1] = a[1]; v[2] = a[2]; v[3] = a[3];
    v[4] = b[0]; v[5] = b[1]; v[6] = b[2]; v[7] = b[3];
  }
};
template <typename T> struct Raw8<T, false> {
  T w[8];
  int left, step;
  __device__ __forceinline__ void load(const T* __restrict__ row, int c, int st, int C) {
    left = C - c;
    step = st;
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = T(0);
    if (C > 0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = row[min(c + k * st, C - 1)];
    }
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k * step < left ? Elem<T>::ld(&w[k]) : 0.f;
  }
};

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ row, int c, int st, int C, const float (&f)[8]) {
  if constexpr (VEC) {
    if (c >= C) return;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(row + c) = bf8_pack(f);
    } else {
      *reinterpret_cast<f4v*>(row + c) = f4v{f[0], f[1], f[2], f[3]};
      *reinterpret_cast<f4v*>(row + c + 4) = f4v{f[4], f[5], f[6], f[7]};
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k * st < C) Elem<T>::st(row + c + k * st, f[k]);
  }
}

// fp32 parameter vector (nullable): its 8 values, or `other`
template <bool VEC>
__device__ __forceinline__ void param8(const float* __restrict__ p, int c, int st, int C, float other, float (&f)[8]) {
  if (p) {
    Raw8<float, VEC> raw;
    raw.load(p, c, st, C);
    raw.values(f);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = other;
  }
}

// sigmoid(v) and sigmoid(-v) without a difference: e = exp(-|v|), 1 / (1 + e) and e / (1 + e)
template <typename T>
__device__ __forceinline__ void sigmoids(float v, float& up, float& down) {
  const float e = gate_exp<T>(-fabsf(v)), r = __builtin_amdgcn_rcpf(1.f + e), q = e * r;
  up = v >= 0.f ? r : (v != v ? v : q);
  down = v >= 0.f ? q : r;
}
// tanh(v) = sign(v) (1 - e) / (1 + e) with e = exp(-2 |v|); below 0.3, where 1 - e cancels, its power series to v^9 (the next term is
// 9e-3 v^10 = 5e-8 of the value)
__device__ __forceinline__ float tanh_of(float v, float e, float r) {
  const float s = v * v;
  const float small = v + v * s * (-0.333333333f + s * (0.133333333f + s * (-0.0539682540f + s * 0.0218694885f)));
  return fabsf(v) < 0.3f ? small : copysignf((1.f - e) * r, v);
}
// g = act(g), one choice for the eight; T: the gate's type
template <typename T>
__device__ __forceinline__ void gate_values(float (&g)[8], int act) {
  if (act == TG_ACT_SIGMOID || act == TG_ACT_SILU) {
    const bool silu = act == TG_ACT_SILU;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float up = __builtin_amdgcn_rcpf(1.f + gate_exp<T>(-g[k]));
      g[k] = silu ? g[k] * up : up;
    }
  } else if (act == TG_ACT_TANH) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float e = gate_exp<T>(-2.f * fabsf(g[k]));
      g[k] = tanh_of(g[k], e, __builtin_amdgcn_rcpf(1.f + e));
    }
  }
}
// value = act(g), slope = act'(g)
template <typename T>
__device__ __forceinline__ void gate_slopes(const float (&g)[8], int act, float (&value)[8], float (&slope)[8]) {
  if (act == TG_ACT_SIGMOID || act == TG_ACT_SILU) {
    const bool silu = act == TG_ACT_SILU;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float up, down;
      sigmoids<T>(g[k], up, down);
      value[k] = silu ? g[k] * up : up;
      slope[k] = silu ? up + g[k] * up * down : up * down;
    }
  } else if (act == TG_ACT_TANH) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float e = gate_exp<T>(-2.f * fabsf(g[k])), r = __builtin_amdgcn_rcpf(1.f + e);
      value[k] = tanh_of(g[k], e, r);
      slope[k] = 4.f * e * r * r;                                   // 1 - tanh^2
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      value[k] = g[k];
      slope[k] = 1.f;
    }
  }
}

// row / rows_per_gate by a multiplication: n < 2^31, q = (mulhi(n, magic) + n) >> shift
struct Divide {
  uint32_t magic;
  int shift;
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return shift == 0 ? n : (__umulhi(n, magic) + n) >> shift; }
};
Divide divide_by(uint32_t d) {
  Divide r = {0, 0};
  while (r.shift < 32 && ((uint64_t)1 << r.shift) < d) ++r.shift;
  r.magic = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << r.shift) - d)) / d + 1);
  return r;
}

constexpr int GN_MAX_LPR = 512;

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float plus_row16(float v) {           // + the other row of 16 lanes
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float plus_half32(float v) {          // + the other half of the wave
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Sums over the lanes whose numbers differ in the bits from `from` up to below `to` (powers of two up to 64), by lane exchanges inside
// the vector unit; every lane gets its sum, all lanes of a group the same bits.
template <int N>
__device__ __forceinline__ void lane_sums(float (&v)[N], int from, int to) {
  if (from < 2 && to >= 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += dpp<0xB1>(v[i]);         // lane ^ 1
  }
  if (from < 4 && to >= 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += dpp<0x4E>(v[i]);         // lane ^ 2
  }
  if (from < 8 && to >= 8) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += from == 1 ? dpp<0x141>(v[i]) : __shfl_xor(v[i], 4, 64);   // 7 - lane serves where four agree
  }
  if (from < 16 && to >= 16) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += dpp<0x128>(v[i]);        // lane ^ 8
  }
  if (from < 32 && to >= 32) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = plus_row16(v[i]);
  }
  if (from < 64 && to >= 64) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = plus_half32(v[i]);
  }
}

// Sums v[0..N) over the lanes of this lane's row.  Rows wider than a wave meet in `red` (two buffers used in turn: a buffer is
// written again two calls later, behind the other buffer's barrier).
template <int N>
__device__ __forceinline__ void row_sums(float (&v)[N], int lpr, float* red, int& turn) {
  if (lpr < 64) {
    lane_sums(v, 1, lpr);
    return;
  }
  lane_sums(v, 1, 64);                                           // constant bounds: six steps without branches
  if (lpr > 64) {
    const int wave = threadIdx.x >> 6, w0 = wave & ~((lpr >> 6) - 1);
    float* buf = red + turn * (8 * 4);                           // [value][wave]
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) buf[i * 8 + wave] = v[i];
    }
    __syncthreads();
    if (lpr == 512) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const f4v a = *reinterpret_cast<const f4v*>(buf + i * 8), b = *reinterpret_cast<const f4v*>(buf + i * 8 + 4);
        v[i] = ((a[0] + a[1]) + (a[2] + a[3])) + ((b[0] + b[1]) + (b[2] + b[3]));
      }
    } else if (lpr == 256) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const f4v a = *reinterpret_cast<const f4v*>(buf + i * 8 + w0);
        v[i] = (a[0] + a[1]) + (a[2] + a[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = buf[i * 8 + w0] + buf[i * 8 + w0 + 1];
    }
    turn ^= 1;
  }
}

struct GnP {
  tg_gated_norm_desc d;
  const void *x, *o, *gate, *y, *d_y, *d_h;
  const float *w_post, *b_post, *scale, *w_pre, *b_pre;
  void *out_y, *out_h, *d_x, *d_o, *d_gate;
  float *part, *gate_part;                   // [blocks][5][C], [items][C]
  Divide gate_of;
  int lpr_log2;
  int item_rows, pieces;                     // rows of an item; > 0: pieces of a gate row's rows (an item is one piece)
  int64_t items;
  int want;                                  // bit p: parameter p's gradient is asked for
  float inv_c;
};

// MODE: what there is beside x -- 0 nothing, 1 a block's output, 2 that and a gate, 3 asked at run time (the widest rows).  A norm
// that is not wanted is one with mean 0 and deviation 1: no branches around the values.
// Parameters stay in registers over a workgroup's rows where they fit (one or two vectors a lane), and the next row's tensors are on
// their way while a row's sums are made.
template <typename TO, typename TX, int NV, bool VEC, int MODE>
__global__ __launch_bounds__(512) void gated_norm_fwd_kernel(GnP p) {
  __shared__ __attribute__((aligned(16))) float red[2 * 8 * 4];
  constexpr bool KEEP = NV <= (VEC ? 2 : 1);                      // wider rows: no registers for the parameters or a second row
  const bool HO = MODE == 3 ? p.o != nullptr : MODE >= 1, HG = MODE == 3 ? p.gate != nullptr : MODE == 2;
  const tg_gated_norm_desc& d = p.d;
  const int lpr = NV > 1 ? GN_MAX_LPR : 1 << p.lpr_log2, lane = threadIdx.x & (lpr - 1), sub = threadIdx.x >> p.lpr_log2, rpb = blockDim.x >> p.lpr_log2;
  const int C = d.C, st = Cols<VEC>::step(lpr);
  constexpr int NP = KEEP ? NV : 1;
  float wpo[NP][8], bpo[NP][8], sc[NP][8], wpr[NP][8], bpr[NP][8];
  auto params_post = [&](int v, int a) {
    const int c = Cols<VEC>::first(v, lane, lpr);
    param8<VEC>(p.w_post, c, st, C, 1.f, wpo[a]);
    param8<VEC>(p.b_post, c, st, C, 0.f, bpo[a]);
    param8<VEC>(p.scale, c, st, C, 1.f, sc[a]);
#pragma unroll
    for (int k = 0; k < 8; ++k) sc[a][k] *= d.alpha;
  };
  auto params_pre = [&](int v, int a) {
    const int c = Cols<VEC>::first(v, lane, lpr);
    param8<VEC>(p.w_pre, c, st, C, 1.f, wpr[a]);
    param8<VEC>(p.b_pre, c, st, C, 0.f, bpr[a]);
  };
  const int64_t row0 = (int64_t)blockIdx.x * rpb + sub, step = (int64_t)gridDim.x * rpb;
  const TX* px = static_cast<const TX*>(p.x) + row0 * d.ldx;      // the row that is fetched next
  const TO* po = static_cast<const TO*>(p.o) + row0 * d.ldo;
  TX* py = static_cast<TX*>(p.out_y) + row0 * d.ldy;              // the row that is written next
  TO* ph = static_cast<TO*>(p.out_h) + row0 * d.ldh;
  const int64_t sx = step * d.ldx, so = step * d.ldo, sy = step * d.ldy, sh = step * d.ldh;
  Raw8<TX, VEC> rx[NV];
  Raw8<TO, VEC> ro[NV], rg[NV];
  auto fetch = [&](int64_t row) {                                 // a row past the end reads nothing
    const int Cr = row < d.rows ? C : 0;
    const TO* pg = static_cast<const TO*>(p.gate) + (int64_t)p.gate_of.of((uint32_t)row) * d.ldg;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = Cols<VEC>::first(v, lane, lpr);
      rx[v].load(px, c, st, Cr);
      if (HO) ro[v].load(po, c, st, Cr);
      if (HG) rg[v].load(pg, c, st, Cr);
    }
    px += sx;
    po += so;
  };
  int turn = 0;
  int64_t row = row0;
  if constexpr (KEEP) {
    fetch(row);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (HO) params_post(v, v);
      params_pre(v, v);
    }
  }
  for (int64_t base = (int64_t)blockIdx.x * rpb; base < d.rows; base += step, row += step, py += sy, ph += sh) {
    const int Cr = row < d.rows ? C : 0;
    if constexpr (!KEEP) fetch(row);
    float x[NV][8], u[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      rx[v].values(x[v]);
      if (HO) ro[v].values(u[v]);
    }
    float g[NP][8];
    if (KEEP && HG) {
#pragma unroll
      for (int v = 0; v < NV; ++v) rg[v].values(g[KEEP ? v : 0]);
    }
    if (KEEP && base + step < d.rows) fetch(row + step);
    if (HO) {
      float mu = 0.f, r = 1.f;
      if (d.post == TG_NORM_LAYER) {
        float s[1] = {0.f};
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int k = 0; k < 8; ++k) s[0] += u[v][k];
        row_sums(s, lpr, red, turn);
        mu = s[0] * p.inv_c;
      }
      if (d.post != TG_NORM_NONE) {
        float s[1] = {0.f};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int c = Cols<VEC>::first(v, lane, lpr);
          const float mv = c < Cr ? mu : 0.f;                       // values past the end are 0 and stay 0
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float t = u[v][k] - (VEC || c + k * st < Cr ? mv : 0.f);
            s[0] += t * t;
          }
        }
        row_sums(s, lpr, red, turn);
        r = rsqrtf(s[0] * p.inv_c + d.eps);
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = Cols<VEC>::first(v, lane, lpr);
        const int a = KEEP ? v : 0;
        if (!KEEP) {
          params_post(v, 0);
          if (HG) rg[v].values(g[0]);
        }
        if (HG) gate_values<TO>(g[a], d.gate_act);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float t = (u[v][k] - mu) * (r * wpo[a][k]) + bpo[a][k];
          x[v][k] += (HG ? sc[a][k] * g[a][k] : sc[a][k]) * t;
        }
        store8<TX, VEC>(py, c, st, Cr, x[v]);
      }
    }
    if (d.pre != TG_NORM_NONE) {
      float mu = 0.f;
      if (d.pre == TG_NORM_LAYER) {
        float s[1] = {0.f};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int c = Cols<VEC>::first(v, lane, lpr);
          float t = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) t += VEC || c + k * st < Cr ? x[v][k] : 0.f;
          s[0] += c < Cr ? t : 0.f;
        }
        row_sums(s, lpr, red, turn);
        mu = s[0] * p.inv_c;
      }
      float s[1] = {0.f};
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = Cols<VEC>::first(v, lane, lpr);
        float q = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float t = x[v][k] - mu;
          q += VEC || c + k * st < Cr ? t * t : 0.f;
        }
        s[0] += c < Cr ? q : 0.f;
      }
      row_sums(s, lpr, red, turn);
      const float r = rsqrtf(s[0] * p.inv_c + d.eps);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int a = KEEP ? v : 0;
        if (!KEEP) params_pre(v, 0);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[v][k] = (x[v][k] - mu) * (r * wpr[a][k]) + bpr[a][k];
        store8<TO, VEC>(ph, Cols<VEC>::first(v, lane, lpr), st, Cr, x[v]);
      }
    }
  }
}

// One item = item_rows consecutive rows of one sub-row of lanes: whole gate rows, or a piece of one (pieces > 0).
template <typename TO, typename TX, int NV, bool VEC, int MODE>
__global__ __launch_bounds__(512) void gated_norm_bwd_kernel(GnP p) {
  const bool HO = MODE == 3 ? p.o != nullptr : MODE >= 1, HG = MODE == 3 ? p.gate != nullptr : MODE == 2;
  __shared__ __attribute__((aligned(16))) float red[2 * 8 * 4];
  extern __shared__ __attribute__((aligned(16))) float join[];      // [rows of the workgroup][8 lpr]: only where it has several
  constexpr bool IN_LDS = NV > 1;                                   // the parameter sums of wide rows: no registers for them
  const tg_gated_norm_desc& d = p.d;
  const int lpr = NV > 1 ? GN_MAX_LPR : 1 << p.lpr_log2, lane = threadIdx.x & (lpr - 1), sub = threadIdx.x >> p.lpr_log2, rpb = blockDim.x >> p.lpr_log2;
  const int C = d.C, st = Cols<VEC>::step(lpr);
  const int64_t item = (int64_t)blockIdx.x * rpb + sub;
  int64_t start, end;
  if (p.pieces > 0) {
    const int64_t group = item / p.pieces, piece = item - group * p.pieces;
    const int64_t last = (group + 1) * d.rows_per_gate;
    start = group * d.rows_per_gate + piece * p.item_rows;
    end = start + p.item_rows < last ? start + p.item_rows : last;
  } else {
    start = item * p.item_rows;
    end = start + p.item_rows;
  }
  end = item < p.items ? (end < d.rows ? end : d.rows) : start;
  const bool layer = d.pre == TG_NORM_LAYER || d.post == TG_NORM_LAYER;
  // sums of w_post, b_post, scale, w_pre, b_pre, and of the gate row; in LDS every lane has its own places, 16 bytes apart
  float acc[IN_LDS ? 1 : 5][IN_LDS ? 1 : NV][8] = {}, dga[NV][8] = {};
  auto place_of = [&](int q, int v) { return reinterpret_cast<f4v*>(join) + (__popc(p.want & ((1 << q) - 1)) * NV + v) * 2 * GN_MAX_LPR + threadIdx.x; };
  auto add = [&](int q, int v, const float (&t)[8]) {
    if constexpr (IN_LDS) {
      if (p.want >> q & 1) {
        f4v* const at = place_of(q, v);
        at[0] += f4v{t[0], t[1], t[2], t[3]};
        at[GN_MAX_LPR] += f4v{t[4], t[5], t[6], t[7]};
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[q][v][k] += t[k];
    }
  };
  if constexpr (IN_LDS) {
#pragma unroll
    for (int q = 0; q < 5; ++q)
      if (p.want >> q & 1) {
#pragma unroll
        for (int v = 0; v < NV; ++v) place_of(q, v)[0] = place_of(q, v)[GN_MAX_LPR] = f4v{0.f, 0.f, 0.f, 0.f};
      }
  }
  Raw8<TX, VEC> ry[NV], rdy[NV];
  Raw8<TO, VEC> rdh[NV], ro[NV], rg[NV];
  auto fetch = [&](int64_t row) {
    const int Cr = row < end ? C : 0;
    const int64_t r = row < end ? row : 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = Cols<VEC>::first(v, lane, lpr);
      ry[v].load(static_cast<const TX*>(p.y) + r * d.ldy, c, st, Cr);
      if (p.d_h) rdh[v].load(static_cast<const TO*>(p.d_h) + r * d.ldh, c, st, Cr);
      if (p.d_y) rdy[v].load(static_cast<const TX*>(p.d_y) + r * d.ld_dy, c, st, Cr);
      if (HO) ro[v].load(static_cast<const TO*>(p.o) + r * d.ldo, c, st, Cr);
      if (HG) rg[v].load(static_cast<const TO*>(p.gate) + (int64_t)p.gate_of.of((uint32_t)r) * d.ldg, c, st, Cr);
    }
  };
  float ga[8], gs[8];                                               // the gate's activation and its derivative
  int64_t gate_row = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) { ga[k] = 1.f; gs[k] = 0.f; }
  // of one vector of a lane: wider rows have no registers for all of them, nor for a second row
  float wpre[8], wpost[8], bpost[8], sc[8];
  auto params_pre = [&](int v) { param8<VEC>(p.w_pre, Cols<VEC>::first(v, lane, lpr), st, C, 1.f, wpre); };
  auto params_post = [&](int v) {
    const int c = Cols<VEC>::first(v, lane, lpr);
    param8<VEC>(p.w_post, c, st, C, 1.f, wpost);
    param8<VEC>(p.b_post, c, st, C, 0.f, bpost);
    param8<VEC>(p.scale, c, st, C, 1.f, sc);
  };
  auto gate_of = [&](int v) {
    float g[8];
    rg[v].values(g);
    gate_slopes<TO>(g, d.gate_act, ga, gs);
  };
  int turn = 0;
  if constexpr (NV == 1) {
    fetch(start);
    params_pre(0);
    params_post(0);
  }
  // the workgroup's longest item: without pieces its first one
  int jn = p.item_rows;
  if (p.pieces == 0) {
    const int64_t rows = d.rows - (int64_t)blockIdx.x * rpb * p.item_rows;
    if (rows < jn) jn = (int)rows;
  }
  for (int j = 0; j < jn; ++j) {
    const bool on = start + j < end;
    const int64_t row = on ? start + j : 0;
    const int Cr = on ? C : 0;
    const int64_t grow = p.gate_of.of((uint32_t)row);
    if constexpr (NV > 1) fetch(start + j);
    float y[NV][8], o[NV][8], dh[NV][8], G[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      ry[v].values(y[v]);
      rdh[v].values(dh[v]);
      rdy[v].values(G[v]);
      if (HO) ro[v].values(o[v]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (!p.d_h) dh[v][k] = 0.f;
        if (!p.d_y) G[v][k] = 0.f;
        if (!HO) o[v][k] = 0.f;
      }
    }
    if (NV == 1 && HG && (j == 0 || grow != gate_row)) {        // a shared gate row: its activation once
      gate_row = grow;
      gate_of(0);
    }
    if (NV == 1 && j + 1 < jn) fetch(start + j + 1);
    float mu_y = 0.f, mu_o = 0.f;
    if (layer) {
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int k = 0; k < 8; ++k) { s[0] += y[v][k]; s[1] += o[v][k]; }
      row_sums(s, lpr, red, turn);
      mu_y = d.pre == TG_NORM_LAYER ? s[0] * p.inv_c : 0.f;
      mu_o = d.post == TG_NORM_LAYER ? s[1] * p.inv_c : 0.f;
    }
    float s[4] = {0.f, 0.f, 0.f, 0.f};                              // |y - mu|^2, t (y - mu), t, |o - mu|^2 with t = dh w_pre
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = Cols<VEC>::first(v, lane, lpr);
      const float my = c < Cr ? mu_y : 0.f, mo = c < Cr ? mu_o : 0.f;   // values past the end are 0 and stay 0
      if (NV > 1) params_pre(v);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        y[v][k] -= VEC || c + k * st < Cr ? my : 0.f;
        o[v][k] -= VEC || c + k * st < Cr ? mo : 0.f;
        const float t = dh[v][k] * wpre[k];
        s[0] += y[v][k] * y[v][k];
        s[1] += t * y[v][k];
        s[2] += t;
        s[3] += o[v][k] * o[v][k];
      }
    }
    row_sums(s, lpr, red, turn);
    const float r_y = rsqrtf(s[0] * p.inv_c + d.eps), r_o = d.post != TG_NORM_NONE ? rsqrtf(s[3] * p.inv_c + d.eps) : 1.f;
    const float m1 = s[1] * r_y * p.inv_c, m2 = d.pre == TG_NORM_LAYER ? s[2] * p.inv_c : 0.f;
    float q[2] = {0.f, 0.f};                                        // t o^, t with t = du w_post
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = Cols<VEC>::first(v, lane, lpr);
      float dg[8], t0[8], t1[8], t2[8];
      const float mp = c < Cr ? m2 : 0.f;
      if (NV > 1) params_pre(v);
#pragma unroll
      for (int k = 0; k < 8; ++k) {                                  // no pre norm: dh = 0
        const float n = y[v][k] * r_y;
        t0[k] = dh[v][k] * n;
        G[v][k] += r_y * (dh[v][k] * wpre[k] - n * m1 - (VEC || c + k * st < Cr ? mp : 0.f));
      }
      add(3, v, t0);
      add(4, v, dh[v]);
      if (p.d_x) store8<TX, VEC>(static_cast<TX*>(p.d_x) + row * d.ldx, c, st, Cr, G[v]);
      if (HO) {
        if (NV > 1) {
          params_post(v);
          if (HG) gate_of(v);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float n = o[v][k] * r_o;                             // no post norm: deviation 1, weight 1, bias 0
          const float u = n * wpost[k] + bpost[k];
          const float a = ga[k], D = d.alpha * G[v][k];
          t2[k] = D * a * u;
          dg[k] = D * sc[k] * u * gs[k];
          t1[k] = D * sc[k] * a;
          t0[k] = t1[k] * n;
          o[v][k] = n;
          G[v][k] = t1[k] * wpost[k];
          q[0] += G[v][k] * n;
          q[1] += G[v][k];
        }
        add(0, v, t0);
        add(1, v, t1);
        add(2, v, t2);
        if (p.d_gate) {
          if (d.rows_per_gate == 1) {
            store8<TO, VEC>(static_cast<TO*>(p.d_gate) + row * d.ld_dg, c, st, Cr, dg);
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) dga[v][k] += dg[k];
          }
        }
      }
    }
    if (HO) {
      if (d.post != TG_NORM_NONE) row_sums(q, lpr, red, turn);
      if (p.d_o) {
        const float n1 = d.post != TG_NORM_NONE ? q[0] * p.inv_c : 0.f, n2 = d.post == TG_NORM_LAYER ? q[1] * p.inv_c : 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int c = Cols<VEC>::first(v, lane, lpr);
          float out[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) out[k] = r_o * (G[v][k] - o[v][k] * n1 - n2);
          store8<TO, VEC>(static_cast<TO*>(p.d_o) + row * d.ld_do, c, st, Cr, out);
        }
      }
      // the last row of a gate row in this item: its sum is complete (whole gate rows only)
      if (p.d_gate && p.pieces == 0 && d.rows_per_gate > 1 && on && (row + 1 == d.rows || (row + 1) % d.rows_per_gate == 0)) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          store8<TO, VEC>(static_cast<TO*>(p.d_gate) + grow * d.ld_dg, Cols<VEC>::first(v, lane, lpr), st, C, dga[v]);
#pragma unroll
          for (int k = 0; k < 8; ++k) dga[v][k] = 0.f;
        }
      }
    }
  }
  if (p.pieces > 0 && item < p.items) {
#pragma unroll
    for (int v = 0; v < NV; ++v) store8<float, VEC>(p.gate_part + item * C, Cols<VEC>::first(v, lane, lpr), st, C, dga[v]);
  }
  // the workgroup's parameter sums: over the rows of a wave by lane exchange, then over the waves through LDS
#pragma unroll
  for (int q = 0; q < 5; ++q) {
    if (!(p.want >> q & 1)) continue;
    float* out = p.part + ((int64_t)blockIdx.x * 5 + q) * C;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = Cols<VEC>::first(v, lane, lpr);
      if (!IN_LDS && rpb > 1) {                                     // several rows only where a row is narrow
        if (lpr < 64) lane_sums(acc[IN_LDS ? 0 : q][IN_LDS ? 0 : v], lpr, 64);
        const int held = lpr < 64 ? blockDim.x >> 6 : rpb;          // sums left per column
        const bool mine = lpr < 64 ? (threadIdx.x & 63) < lpr : true;
        const int slot = lpr < 64 ? threadIdx.x >> 6 : sub;
        __syncthreads();
        if (mine) {
#pragma unroll
          for (int k = 0; k < 8; ++k) join[slot * lpr * 8 + Cols<VEC>::first(0, lane, lpr) + k * st] = acc[IN_LDS ? 0 : q][IN_LDS ? 0 : v][k];
        }
        __syncthreads();
        for (int e = threadIdx.x; e < lpr * 8 && e < C; e += blockDim.x) {
          float t = 0.f;
          for (int s = 0; s < held; ++s) t += join[s * lpr * 8 + e];
          out[e] = t;
        }
      } else if constexpr (IN_LDS) {
        const f4v a = place_of(q, v)[0], b = place_of(q, v)[GN_MAX_LPR];
        const float t[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        store8<float, VEC>(out, c, st, C, t);
      } else {
        store8<float, VEC>(out, c, st, C, acc[q][v]);
      }
    }
  }
}

// The second launch: sums of partial rows in a fixed order -- the five parameters over the workgroups, then (pieces > 0) every gate
// row over its pieces.  A workgroup takes 64 columns of one of them: 16 strided sums a column, then a tree over those.
struct GnSum {
  float* param[5];
  const float *part, *gate_part;
  void* d_gate;
  int64_t ld;
  int blocks, pieces, C, ncb;
};
template <typename TO>
__global__ __launch_bounds__(1024) void gated_norm_sums_kernel(GnSum p) {
  __shared__ float sm[16][64];
  const int64_t q = blockIdx.x / p.ncb;
  const int cl = threadIdx.x & 63, c = (int)(blockIdx.x - q * p.ncb) * 64 + cl, w = threadIdx.x >> 6;
  if (q < 5 && !p.param[q]) return;
  const float* src = q < 5 ? p.part + q * p.C : p.gate_part + (q - 5) * p.pieces * p.C;
  const int64_t stride = q < 5 ? 5 * (int64_t)p.C : p.C;
  const int n = q < 5 ? p.blocks : p.pieces;
  float s = 0.f;
  if (c < p.C) {
#pragma unroll 8
    for (int b = w; b < n; b += 16) s += src[b * stride + c];
  }
  sm[w][cl] = s;
  __syncthreads();
#pragma unroll
  for (int h = 8; h > 0; h >>= 1) {
    if (w < h) sm[w][cl] += sm[w + h][cl];
    __syncthreads();
  }
  if (w == 0 && c < p.C) {
    if (q < 5) p.param[q][c] = sm[0][cl];
    else Elem<TO>::st(static_cast<TO*>(p.d_gate) + (q - 5) * p.ld + c, sm[0][cl]);
  }
}

struct Geo {
  int lpr_log2, lpr, block, nv, rpb, item_rows, pieces, blocks;
  int64_t items;
};

void row_geometry(int C, int block, Geo* g) {
  const int oct = (C + 7) / 8;
  int l = 0;
  while ((1 << l) < oct && (1 << l) < GN_MAX_LPR) ++l;
  g->lpr_log2 = l;
  g->lpr = 1 << l;
  g->nv = oct <= g->lpr ? 1 : (oct <= 2 * g->lpr ? 2 : 4);
  g->block = g->lpr < block ? block : g->lpr;
  g->rpb = g->block / g->lpr;
}

// The backward pass's split of the rows: workgroups of 512 lanes, one per compute unit (their registers leave room for one or two), as
// few rows as that gives to each: every row costs its workgroup 2 - 9 us of latency, while partial sums, up to 5 C values a workgroup,
// are read once from near by (64 rows of 1024 bf16 values: at least one row an item 10.7 us, at least four 18.7; 2048 x 2048: 25 both).
// The split fixes the workspace's size and the order of the sums, which a host may ask for where no device is: it takes the 256 compute
// units of a whole MI355X instead of asking (a partition of one gets the same results, several rounds of workgroups).
// A gate row that several rows share stays with one item, or is cut into even pieces where that would double the item (72352 x 88,
// 13 rows a gate row: whole ones 37 us, 9 and 4 rows 75).
constexpr int64_t GN_UNITS = 256;
void item_geometry(int64_t rows, int C, int64_t k, Geo* g) {
  row_geometry(C, 512, g);
  int64_t m = rows > 0 ? cdiv64(rows, GN_UNITS * g->rpb) : 1;
  g->pieces = 0;
  if (k > 1 && k <= 2 * m) {
    m = k <= m ? cdiv64(m, k) * k : k;
  } else if (k > m) {
    k = k < rows ? k : rows;
    g->pieces = (int)cdiv64(k, m);
    m = cdiv64(k, g->pieces);
  }
  g->item_rows = (int)m;
  g->items = g->pieces > 0 ? cdiv64(rows, k) * g->pieces : cdiv64(rows, m);
  g->blocks = (int)cdiv64(g->items, g->rpb);
}

int64_t part_floats(const Geo& g, int C) { return ((int64_t)g.blocks * 5 * C + 3) / 4 * 4; }

bool shape_ok(int64_t rows, int C, int64_t k) {
  return rows >= 0 && rows < ((int64_t)1 << 31) && C >= 1 && C <= TG_GATED_NORM_MAX_C && k >= 1 && k < ((int64_t)1 << 31);
}

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// dtype pairs (rows of the blocks, residual stream): bf16 / bf16, bf16 / f32, f32 / f32
bool types_ok(const tg_gated_norm_desc* d) {
  return (d->dtype == TG_BF16 && (d->res_dtype == TG_BF16 || d->res_dtype == TG_F32)) || (d->dtype == TG_F32 && d->res_dtype == TG_F32);
}
bool codes_ok(const tg_gated_norm_desc* d) {
  auto kind = [](int k) { return k == TG_NORM_NONE || k == TG_NORM_RMS || k == TG_NORM_LAYER; };
  return kind(d->post) && kind(d->pre) &&
         (d->gate_act == TG_ACT_NONE || d->gate_act == TG_ACT_SIGMOID || d->gate_act == TG_ACT_TANH || d->gate_act == TG_ACT_SILU);
}
// eps keeps 1 / sqrt(0 + eps) finite: the lanes past a row's end and rows of zeros rely on it
bool eps_ok(const tg_gated_norm_desc* d) { return d->eps >= 1e-30f && d->eps <= 1e30f; }

}  // namespace

#define ST(s) static_cast<hipStream_t>(s)

#define GN_PICK(KERN, VECV, ...)                                                                                \
  do {                                                                                                          \
    if (d->dtype == TG_F32) { GN_NV(KERN, float, float, VECV, __VA_ARGS__); }                                   \
    else if (d->res_dtype == TG_F32) { GN_NV(KERN, u16, float, VECV, __VA_ARGS__); }                            \
    else { GN_NV(KERN, u16, u16, VECV, __VA_ARGS__); }                                                          \
  } while (0)
#define GN_NV(KERN, TO, TX, VECV, ...)                                                                          \
  do {                                                                                                          \
    if (g.nv == 1) { GN_MODE(KERN, TO, TX, 1, VECV, __VA_ARGS__); }                                             \
    else if (g.nv == 2) { GN_MODE(KERN, TO, TX, 2, VECV, __VA_ARGS__); }                                        \
    else { TG_LAUNCH(name, flops, bytes, (KERN<TO, TX, 4, VECV, 3>), __VA_ARGS__); }                            \
  } while (0)
#define GN_MODE(KERN, TO, TX, NVV, VECV, ...)                                                                   \
  do {                                                                                                          \
    if (gate) { TG_LAUNCH(name, flops, bytes, (KERN<TO, TX, NVV, VECV, 2>), __VA_ARGS__); }                     \
    else if (o) { TG_LAUNCH(name, flops, bytes, (KERN<TO, TX, NVV, VECV, 1>), __VA_ARGS__); }                   \
    else { TG_LAUNCH(name, flops, bytes, (KERN<TO, TX, NVV, VECV, 0>), __VA_ARGS__); }                          \
  } while (0)

extern "C" int tg_gated_norm_forward(const tg_gated_norm_desc* d, const void* x, const void* o, const void* gate, const float* w_post,
                                     const float* b_post, const float* scale, const float* w_pre, const float* b_pre, void* y, void* h,
                                     void* stream) {
  TG_CHECK_ARG(d != nullptr, "null descriptor");
  TG_CHECK_ARG(shape_ok(d->rows, d->C, d->rows_per_gate), "rows in [0, 2^31), C in [1, TG_GATED_NORM_MAX_C], rows_per_gate in [1, 2^31)");
  TG_CHECK_ARG(types_ok(d), "types: bf16 rows with a bf16 or f32 residual stream, or f32 rows with an f32 one");
  TG_CHECK_ARG(eps_ok(d), "eps must lie in [1e-30, 1e30]");
  TG_CHECK_ARG(codes_ok(d), "unknown norm kind or gate activation (none, sigmoid, tanh, silu)");
  if (d->rows == 0) return TG_OK;                                   // an empty tensor has no address
  TG_CHECK_ARG(o != nullptr || (d->post == TG_NORM_NONE && gate == nullptr && y == nullptr), "a post norm, a gate or y without a block output");
  TG_CHECK_ARG((o == nullptr || y != nullptr) && (h != nullptr) == (d->pre != TG_NORM_NONE), "y goes with the block output, h with a pre norm");
  TG_CHECK_ARG(o != nullptr || h != nullptr, "nothing to do: neither a block output nor a pre norm");
  TG_CHECK_ARG(x != nullptr, "x is missing");
  const int C = d->C;
  TG_CHECK_ARG(d->ldx >= C && (!o || (d->ldo >= C && d->ldy >= C)) && (!gate || d->ldg >= C) && (!h || d->ldh >= C), "a row stride below C");
  Geo g;
  row_geometry(C, 256, &g);
  GnP p = {};
  p.d = *d;
  p.x = x; p.o = o; p.gate = gate;
  p.w_post = w_post; p.b_post = b_post; p.scale = scale; p.w_pre = w_pre; p.b_pre = b_pre;
  p.out_y = y; p.out_h = h;
  p.lpr_log2 = g.lpr_log2;
  p.inv_c = 1.f / (float)C;
  p.gate_of = divide_by((uint32_t)d->rows_per_gate);
  const bool vec = C % 8 == 0 && al16(x) && al16(o) && al16(gate) && al16(y) && al16(h) && al16(w_post) && al16(b_post) && al16(scale) &&
                   al16(w_pre) && al16(b_pre) && d->ldx % 8 == 0 && (!o || (d->ldo % 8 == 0 && d->ldy % 8 == 0)) &&
                   (!gate || d->ldg % 8 == 0) && (!h || d->ldh % 8 == 0);
  const char* const name = "gated_norm_fwd";
  const double n = (double)d->rows * C, flops = 14 * n, ex = d->res_dtype == TG_F32 ? 4 : 2, eo = d->dtype == TG_F32 ? 4 : 2;
  const double bytes = n * (ex + (o ? ex + eo : 0) + (gate && d->rows_per_gate == 1 ? eo : 0) + (h ? eo : 0));
  const int64_t resident = (int64_t)tg_num_cus() * (1024 / g.block);  // workgroups that stay on the device and walk over the rows
  const dim3 grid((unsigned)(cdiv64(d->rows, g.rpb) < resident ? cdiv64(d->rows, g.rpb) : resident)), block(g.block);
  if (vec) GN_PICK(gated_norm_fwd_kernel, true, grid, block, 0, ST(stream), p);
  else GN_PICK(gated_norm_fwd_kernel, false, grid, block, 0, ST(stream), p);
  TG_CHECK_LAUNCH();
}

extern "C" int tg_gated_norm_ws(int64_t rows, int C, int64_t rows_per_gate, int64_t* floats) {
  TG_CHECK_ARG(floats != nullptr, "null pointer");
  TG_CHECK_ARG(shape_ok(rows, C, rows_per_gate), "rows in [0, 2^31), C in [1, TG_GATED_NORM_MAX_C], rows_per_gate in [1, 2^31)");
  Geo g;
  item_geometry(rows, C, rows_per_gate, &g);
  *floats = part_floats(g, C) + (g.pieces > 0 ? g.items * C : 0);
  return TG_OK;
}

extern "C" int tg_gated_norm_backward(const tg_gated_norm_desc* d, const void* d_y, const void* d_h, const void* y, const void* o,
                                      const void* gate, const float* w_post, const float* b_post, const float* scale,
                                      const float* w_pre, const float* b_pre, void* d_x, void* d_o, void* d_gate, float* d_w_post,
                                      float* d_b_post, float* d_scale, float* d_w_pre, float* d_b_pre, float* ws, int64_t ws_floats,
                                      void* stream) {
  TG_CHECK_ARG(d != nullptr, "null descriptor");
  TG_CHECK_ARG(shape_ok(d->rows, d->C, d->rows_per_gate), "rows in [0, 2^31), C in [1, TG_GATED_NORM_MAX_C], rows_per_gate in [1, 2^31)");
  TG_CHECK_ARG(types_ok(d), "types: bf16 rows with a bf16 or f32 residual stream, or f32 rows with an f32 one");
  TG_CHECK_ARG(eps_ok(d), "eps must lie in [1e-30, 1e30]");
  TG_CHECK_ARG(codes_ok(d), "unknown norm kind or gate activation (none, sigmoid, tanh, silu)");
  TG_CHECK_ARG(d->rows == 0 || o != nullptr || (d->post == TG_NORM_NONE && gate == nullptr && !d_o && !d_scale),
               "a post norm, a gate, d_o or d_scale without a block output");   // rows == 0: an empty tensor has no address
  TG_CHECK_ARG(d->rows == 0 || d_gate == nullptr || gate != nullptr, "d_gate without a gate");
  TG_CHECK_ARG(d->pre != TG_NORM_NONE || (d_h == nullptr && !d_w_pre && !d_b_pre), "d_h, d_w_pre or d_b_pre without a pre norm");
  TG_CHECK_ARG(d->post != TG_NORM_NONE || (!d_w_post && !d_b_post), "d_w_post or d_b_post without a post norm");
  const int C = d->C;
  Geo g;
  item_geometry(d->rows, C, d->rows_per_gate, &g);
  const int64_t pf = part_floats(g, C), need = pf + (g.pieces > 0 ? g.items * C : 0);
  TG_CHECK_ARG(d->rows == 0 || (y != nullptr && ws != nullptr && al16(ws) && ws_floats >= need), "y, or a workspace of tg_gated_norm_ws() floats, is missing");
  TG_CHECK_ARG((!d_y || d->ld_dy >= C) && (!d_h || d->ldh >= C) && d->ldy >= C && (!o || d->ldo >= C) && (!gate || d->ldg >= C) &&
                   (!d_x || d->ldx >= C) && (!d_o || d->ld_do >= C) && (!d_gate || d->ld_dg >= C),
               "a row stride below C");
  const int want = (d_w_post ? 1 : 0) | (d_b_post ? 2 : 0) | (d_scale ? 4 : 0) | (d_w_pre ? 8 : 0) | (d_b_pre ? 16 : 0);
  if (d->rows > 0) {
    GnP p = {};
    p.d = *d;
    p.y = y; p.o = o; p.gate = gate; p.d_y = d_y; p.d_h = d_h;
    p.w_post = w_post; p.b_post = b_post; p.scale = scale; p.w_pre = w_pre; p.b_pre = b_pre;
    p.d_x = d_x; p.d_o = d_o; p.d_gate = d_gate;
    p.part = ws;
    p.gate_part = ws + pf;
    p.lpr_log2 = g.lpr_log2;
    p.item_rows = g.item_rows; p.pieces = g.pieces; p.items = g.items;
    p.want = want;
    p.inv_c = 1.f / (float)C;
    p.gate_of = divide_by((uint32_t)d->rows_per_gate);
    const bool vec = C % 8 == 0 && al16(d_y) && al16(d_h) && al16(y) && al16(o) && al16(gate) && al16(w_post) && al16(b_post) &&
                     al16(scale) && al16(w_pre) && al16(d_x) && al16(d_o) && al16(d_gate) && (!d_y || d->ld_dy % 8 == 0) &&
                     (!d_h || d->ldh % 8 == 0) && d->ldy % 8 == 0 && (!o || d->ldo % 8 == 0) && (!gate || d->ldg % 8 == 0) &&
                     (!d_x || d->ldx % 8 == 0) && (!d_o || d->ld_do % 8 == 0) && (!d_gate || d->ld_dg % 8 == 0);
    const char* const name = "gated_norm_bwd";
    const double n = (double)d->rows * C, flops = 40 * n, ex = d->res_dtype == TG_F32 ? 4 : 2, eo = d->dtype == TG_F32 ? 4 : 2;
    const double bytes = n * (ex * (1 + (d_y ? 1 : 0) + (d_x ? 1 : 0)) + eo * ((d_h ? 1 : 0) + (o ? 1 : 0) + (d_o ? 1 : 0)));
    const dim3 grid((unsigned)g.blocks), block(g.block);
    // Wide rows: as many parameter sums at a time as LDS holds beside the row sums' buffers (4 up to 8192 columns, 2 above); passes
    // that only sum come first, since the outputs may lie over the inputs.
    const int room = g.nv > 1 ? (int)(159 * 1024 / ((size_t)g.nv * GN_MAX_LPR * 32)) : 5;
    int left = want;
    do {
      p.want = 0;
      for (int n = 0; left && n < room; ++n) {
        const int bit = left & -left;
        p.want |= bit;
        left ^= bit;
      }
      p.d_x = left ? nullptr : d_x;
      p.d_o = left ? nullptr : d_o;
      p.d_gate = left ? nullptr : d_gate;
      const size_t lds = g.nv > 1 ? (size_t)__builtin_popcount(p.want) * g.nv * GN_MAX_LPR * 32 : (g.rpb > 1 ? (size_t)g.block * 8 * sizeof(float) : 0);
      if (vec) GN_PICK(gated_norm_bwd_kernel, true, grid, block, lds, ST(stream), p);
      else GN_PICK(gated_norm_bwd_kernel, false, grid, block, lds, ST(stream), p);
    } while (left);
  }
  const bool gates = d->rows > 0 && d_gate && g.pieces > 0;
  if (want || gates) {
    const GnSum q = {{d_w_post, d_b_post, d_scale, d_w_pre, d_b_pre}, ws, ws + pf, d_gate, d->ld_dg, d->rows > 0 ? g.blocks : 0, g.pieces, C, (C + 63) / 64};
    const dim3 grid((unsigned)(q.ncb * (5 + (gates ? cdiv64(d->rows, d->rows_per_gate) : 0))));
    if (d->dtype == TG_F32) hipLaunchKernelGGL((gated_norm_sums_kernel<float>), grid, dim3(1024), 0, ST(stream), q);
    else hipLaunchKernelGGL((gated_norm_sums_kernel<u16>), grid, dim3(1024), 0, ST(stream), q);
  }
  TG_CHECK_LAUNCH();
}
