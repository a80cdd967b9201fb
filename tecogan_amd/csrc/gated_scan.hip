// Gated linear recurrence along a sequence, channel by channel:
//
//   f[t] = floor + (1 - floor) sigmoid(g[t]),   h[t] = f[t] h[t-1] + (1 - f[t]) x[t],   y = h,  hT = h[last]
//   backward:  D[t] = dy[t] + f[t+1] D[t+1];  dx = (1 - f) D;  df = D (h[t-1] - x);  dg = df (1 - floor) s(g) s(-g);
//              dfloor = sum df s(-g);  dh0 = f[0] D[0]
//
// A step is an affine map of the state, h -> P h + L, and maps compose: (P2, L2) after (P1, L1) = (P1 P2, P2 L1 + L2).  A sequence
// is cut into chunks, each chunk into tiles of 8 W steps (W waves, 8 steps each in registers): every wave composes its 8 steps,
// the maps meet in LDS, every wave enters its steps with the right state and writes them.  Where the channels alone fill the
// device there is one chunk and x, g are read once; otherwise a first launch composes the chunks, a second one runs over the
// chunks' maps (few values), a third one writes the outputs.  About 14 / 50 operations a value: bound by HBM.  States, maps and
// gradient sums are fp32; 1 - f is (1 - floor) sigmoid(-g), not a difference.  The forward pass keeps the state before every
// tile (fp32, 1 value in 64): the backward pass makes the states of a tile again from it instead of reading rounded ones.
//
// A reset (a new sequence begins at step t) drops the state by selection, not by a product with 0: what was in it, NaN included,
// does not get past.  In a composed map P = -1 says that a reset is inside (P is a product of values in [0, 1] otherwise).
// Steps at and behind a row's length keep the state, write y = 0 and zero gradients, and their x, g, dy are not looked at.
#include "common.h"

namespace {

constexpr int GS_L = 8;                                            // steps of a wave in a tile
constexpr int GS_MAXW = 8;

struct GsP {
  tg_gated_scan_desc d;
  const void *x, *g, *d_y;
  const float *h0, *floor, *d_hT;
  const int32_t* lengths;
  const unsigned char* reset;
  void *y, *d_x, *d_g;
  float *hT, *d_h0;
  float *tiles;                              // [B][ntiles][D] state before each tile
  float *agg_p, *agg_l;                      // [B][nc][D] the chunks' maps
  float *rev_l, *rev_in;                     // [B][nc][D] backward: chunk's part, gradient that enters a chunk from behind
  float *floor_part;                         // [B * nc][D]
  int ncb, nc, tpc, ntiles, W;               // channel blocks, chunks, tiles of a chunk, tiles, waves
  int keep_tiles;
};

template <typename T, int V>
__device__ __forceinline__ void ldv(const T* p, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = Elem<T>::ld(p);
  } else if constexpr (sizeof(T) == 2) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    f[0] = __uint_as_float(w << 16);
    f[1] = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 w = *reinterpret_cast<const float2*>(p);
    f[0] = w.x;
    f[1] = w.y;
  }
}
template <typename T, int V>
__device__ __forceinline__ void stv(T* p, const float (&f)[V]) {
  if constexpr (V == 1) {
    Elem<T>::st(p, f[0]);
  } else if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint32_t*>(p) = (uint32_t)f2bf(f[0]) | ((uint32_t)f2bf(f[1]) << 16);
  } else {
    *reinterpret_cast<float2*>(p) = make_float2(f[0], f[1]);
  }
}

// sigmoid(g) and sigmoid(-g) without a difference: e = exp(-|g|), 1 / (1 + e) and e / (1 + e)
__device__ __forceinline__ void sigmoids(float g, float& up, float& down) {
  const float e = __expf(-fabsf(g));
  const float r = __builtin_amdgcn_rcpf(1.f + e), q = e * r;
  up = g >= 0.f ? r : q;
  down = g >= 0.f ? q : r;
  if (g != g) up = down = g;
}

// state -> P state + L; P = -1: a reset inside
__device__ __forceinline__ float apply(float P, float L, float h) { return P < 0.f ? L : P * h + L; }
__device__ __forceinline__ void compose(float& P, float& L, float P2, float L2) {
  L = apply(P2, L2, L);
  P = P < 0.f || P2 < 0.f ? -1.f : P * P2;
}

struct Steps {                                                     // the 8 steps of a wave: which are live, which begin a sequence
  int live;
  unsigned reset;
};
__device__ __forceinline__ Steps steps_of(const GsP& p, int b, int64_t t0, int len) {
  Steps s;
  const int64_t left = len - t0;
  s.live = left < 0 ? 0 : (left > GS_L ? GS_L : (int)left);
  s.reset = 0;
  if (p.reset) {
    const int lane = threadIdx.x & 63;
    const bool r = lane < s.live && p.reset[(int64_t)b * p.d.T + t0 + lane] != 0;
    s.reset = (unsigned)__ballot(r);
  }
  return s;
}

// Forward.  OUT false: the chunk's map only (each wave a contiguous part of it); true: states and outputs.
template <typename T, int V, bool OUT>
__global__ __launch_bounds__(512) void gated_scan_fwd_kernel(GsP p) {
  __shared__ float sP[GS_MAXW][64 * V], sL[GS_MAXW][64 * V];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = p.W;
  const int cb = blockIdx.x % p.ncb, rest = blockIdx.x / p.ncb, chunk = rest % p.nc, b = rest / p.nc;
  const int c = (cb * 64 + lane) * V, D = p.d.D, Tn = p.d.T;
  const bool on = c < D;
  int len = Tn;
  if (p.lengths) {
    const int n = p.lengths[b];
    len = n < 0 ? 0 : (n < Tn ? n : Tn);
  }
  const T* xr = static_cast<const T*>(p.x) + (int64_t)b * p.d.x_b + c;
  const T* gr = static_cast<const T*>(p.g) + (int64_t)b * p.d.g_b + c;
  T* yr = static_cast<T*>(p.y) + (int64_t)b * p.d.y_b + c;
  float low[V];
#pragma unroll
  for (int v = 0; v < V; ++v) low[v] = p.floor && on ? p.floor[c + v] : 0.f;
  const int64_t first = (int64_t)chunk * p.tpc;
  const int ntiles = (int)(p.ntiles - first < p.tpc ? p.ntiles - first : p.tpc);
  const int64_t state = ((int64_t)b * p.ntiles + first) * D + c;  // of p.tiles

  float H[V], P[V], L[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { H[v] = 0.f; P[v] = 1.f; L[v] = 0.f; }
  if (OUT && on) {
#pragma unroll
    for (int v = 0; v < V; ++v) H[v] = p.nc > 1 ? p.tiles[state + v] : (p.h0 ? p.h0[(int64_t)b * D + c + v] : 0.f);
  }
  for (int i = 0; i < ntiles; ++i) {
    // OUT: tile i, wave after wave; otherwise this wave's i-th group of 8 steps of its contiguous part of the chunk
    const int64_t t0 = OUT ? ((first + i) * W + wave) * GS_L : (first * W + (int64_t)wave * ntiles + i) * GS_L;
    const Steps st = steps_of(p, b, t0, len);
    float f[GS_L][V], a[GS_L][V];
#pragma unroll
    for (int j = 0; j < GS_L; ++j) {
      const bool ok = on && j < st.live;
      float g[V], x[V];
#pragma unroll
      for (int v = 0; v < V; ++v) { g[v] = 0.f; x[v] = 0.f; }
      if (ok) {
        ldv<T, V>(gr + (t0 + j) * p.d.g_t, g);
        ldv<T, V>(xr + (t0 + j) * p.d.x_t, x);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float up, down;
        sigmoids(g[v], up, down);
        f[j][v] = ok ? low[v] + (1.f - low[v]) * up : 1.f;
        a[j][v] = ok ? (1.f - low[v]) * down * x[v] : 0.f;
      }
    }
    if (OUT) {
#pragma unroll
      for (int v = 0; v < V; ++v) { P[v] = 1.f; L[v] = 0.f; }
    }
#pragma unroll
    for (int j = 0; j < GS_L; ++j) {
      const bool r = st.reset >> j & 1;
#pragma unroll
      for (int v = 0; v < V; ++v) compose(P[v], L[v], r ? -1.f : f[j][v], a[j][v]);
    }
    if constexpr (OUT) {
      if (i > 0) __syncthreads();                                  // the last tile's maps have been read
#pragma unroll
      for (int v = 0; v < V; ++v) { sP[wave][lane * V + v] = P[v]; sL[wave][lane * V + v] = L[v]; }
      __syncthreads();
      float h[V];
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = H[v];
      if (p.keep_tiles && wave == 0 && on && !(p.nc > 1 && i == 0)) {
#pragma unroll
        for (int v = 0; v < V; ++v) p.tiles[state + (int64_t)i * D + v] = H[v];
      }
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (w == wave) h[v] = H[v];
          H[v] = apply(sP[w][lane * V + v], sL[w][lane * V + v], H[v]);
        }
      }
#pragma unroll
      for (int j = 0; j < GS_L; ++j) {
        const bool r = st.reset >> j & 1;
        float o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h[v] = (r ? 0.f : f[j][v] * h[v]) + a[j][v];
          o[v] = j < st.live ? h[v] : 0.f;
        }
        if (on && t0 + j < Tn) stv<T, V>(yr + (t0 + j) * p.d.y_t, o);
      }
    }
  }
  if constexpr (OUT) {
    if (p.hT && chunk == p.nc - 1 && wave == 0 && on) {
#pragma unroll
      for (int v = 0; v < V; ++v) p.hT[(int64_t)b * D + c + v] = H[v];
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) { sP[wave][lane * V + v] = P[v]; sL[wave][lane * V + v] = L[v]; }
    __syncthreads();
    if (wave == 0 && on) {
      for (int w = 1; w < W; ++w) {
#pragma unroll
        for (int v = 0; v < V; ++v) compose(P[v], L[v], sP[w][lane * V + v], sL[w][lane * V + v]);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int64_t at = ((int64_t)b * p.nc + chunk) * D + c + v;
        p.agg_p[at] = P[v];
        p.agg_l[at] = L[v];
      }
    }
  }
}

// The states before the chunks, from h0 over the chunks' maps; written where the outputs' launch looks for them.
__global__ __launch_bounds__(64) void gated_scan_carry_kernel(GsP p) {
  const int64_t e = (int64_t)blockIdx.x * 64 + threadIdx.x;
  const int D = p.d.D;
  if (e >= (int64_t)p.d.B * D) return;
  const int64_t b = e / D, c = e - b * D;
  float H = p.h0 ? p.h0[e] : 0.f;
#pragma unroll 8
  for (int k = 0; k < p.nc; ++k) {
    const int64_t at = (b * p.nc + k) * D + c;
    p.tiles[(b * p.ntiles + (int64_t)k * p.tpc) * D + c] = H;
    H = apply(p.agg_p[at], p.agg_l[at], H);
  }
}

// The gradient that enters each chunk from behind, and what is left of it before the first step.
__global__ __launch_bounds__(64) void gated_scan_rcarry_kernel(GsP p) {
  const int64_t e = (int64_t)blockIdx.x * 64 + threadIdx.x;
  const int D = p.d.D;
  if (e >= (int64_t)p.d.B * D) return;
  const int64_t b = e / D, c = e - b * D;
  float R = p.d_hT ? p.d_hT[e] : 0.f;
#pragma unroll 8
  for (int k = p.nc - 1; k >= 0; --k) {
    const int64_t at = (b * p.nc + k) * D + c;
    p.rev_in[at] = R;
    R = apply(p.agg_p[at], p.rev_l[at], R);
  }
  if (p.d_h0) p.d_h0[e] = R;
}

// Backward.  OUT false: what a chunk adds to the gradient that leaves it in front; true: the gradients.
template <typename T, int V, bool OUT>
__global__ __launch_bounds__(512) void gated_scan_bwd_kernel(GsP p) {
  __shared__ float sP[GS_MAXW][64 * V], sL[GS_MAXW][64 * V], sR[GS_MAXW][64 * V];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = p.W;
  const int cb = blockIdx.x % p.ncb, rest = blockIdx.x / p.ncb, chunk = rest % p.nc, b = rest / p.nc;
  const int c = (cb * 64 + lane) * V, D = p.d.D, Tn = p.d.T;
  const bool on = c < D;
  int len = Tn;
  if (p.lengths) {
    const int n = p.lengths[b];
    len = n < 0 ? 0 : (n < Tn ? n : Tn);
  }
  const T* xr = static_cast<const T*>(p.x) + (int64_t)b * p.d.x_b + c;
  const T* gr = static_cast<const T*>(p.g) + (int64_t)b * p.d.g_b + c;
  const T* er = static_cast<const T*>(p.d_y) + (int64_t)b * p.d.dy_b + c;
  T* dxr = static_cast<T*>(p.d_x) + (int64_t)b * p.d.dx_b + c;
  T* dgr = static_cast<T*>(p.d_g) + (int64_t)b * p.d.dg_b + c;
  float low[V];
#pragma unroll
  for (int v = 0; v < V; ++v) low[v] = p.floor && on ? p.floor[c + v] : 0.f;
  const int64_t first = (int64_t)chunk * p.tpc;
  const int ntiles = (int)(p.ntiles - first < p.tpc ? p.ntiles - first : p.tpc);
  const int64_t chunk_at = ((int64_t)b * p.nc + chunk) * D + c;

  float R[V], dlow[V], P[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { R[v] = 0.f; dlow[v] = 0.f; P[v] = 1.f; }
  if (OUT && on) {
#pragma unroll
    for (int v = 0; v < V; ++v) R[v] = p.nc > 1 ? p.rev_in[chunk_at + v] : (p.d_hT ? p.d_hT[(int64_t)b * D + c + v] : 0.f);
  }
  for (int i = ntiles - 1; i >= 0; --i) {
    const int64_t t0 = OUT ? ((first + i) * W + wave) * GS_L : (first * W + (int64_t)wave * ntiles + i) * GS_L;
    const Steps st = steps_of(p, b, t0, len);
    float up[GS_L][V], down[GS_L][V], x[GS_L][V], e[GS_L][V];
#pragma unroll
    for (int j = 0; j < GS_L; ++j) {
      const bool ok = on && j < st.live;
      float g[V];
#pragma unroll
      for (int v = 0; v < V; ++v) { g[v] = 0.f; x[j][v] = 0.f; e[j][v] = 0.f; }
      if (ok) {
        ldv<T, V>(gr + (t0 + j) * p.d.g_t, g);
        if (p.d_y) ldv<T, V>(er + (t0 + j) * p.d.dy_t, e[j]);
        if (OUT) ldv<T, V>(xr + (t0 + j) * p.d.x_t, x[j]);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        sigmoids(g[v], up[j][v], down[j][v]);
        if (!OUT) x[j][v] = ok ? low[v] + (1.f - low[v]) * up[j][v] : 1.f;            // f: x is not needed
      }
    }
    if constexpr (!OUT) {
#pragma unroll
      for (int j = GS_L - 1; j >= 0; --j) {
        const bool r = st.reset >> j & 1;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          R[v] = r ? 0.f : x[j][v] * (e[j][v] + R[v]);
          P[v] = r || P[v] < 0.f ? -1.f : P[v] * x[j][v];
        }
      }
    } else {
      float h[GS_L][V], Lf[V], Lr[V];
#pragma unroll
      for (int v = 0; v < V; ++v) { P[v] = 1.f; Lf[v] = 0.f; Lr[v] = 0.f; }
#pragma unroll
      for (int j = 0; j < GS_L; ++j) {
        const bool r = st.reset >> j & 1, ok = j < st.live;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float f = ok ? low[v] + (1.f - low[v]) * up[j][v] : 1.f;
          const float a = ok ? (1.f - low[v]) * down[j][v] * x[j][v] : 0.f;
          compose(P[v], Lf[v], r ? -1.f : f, a);
        }
      }
#pragma unroll
      for (int j = GS_L - 1; j >= 0; --j) {
        const bool r = st.reset >> j & 1, ok = j < st.live;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float f = ok ? low[v] + (1.f - low[v]) * up[j][v] : 1.f;
          Lr[v] = r ? 0.f : f * (e[j][v] + Lr[v]);
        }
      }
      if (i < ntiles - 1) __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        sP[wave][lane * V + v] = P[v];
        sL[wave][lane * V + v] = Lf[v];
        sR[wave][lane * V + v] = Lr[v];
      }
      float H[V];
#pragma unroll
      for (int v = 0; v < V; ++v) H[v] = on ? p.tiles[((int64_t)b * p.ntiles + first + i) * D + c + v] : 0.f;
      __syncthreads();
      for (int w = 0; w < wave; ++w) {
#pragma unroll
        for (int v = 0; v < V; ++v) H[v] = apply(sP[w][lane * V + v], sL[w][lane * V + v], H[v]);
      }
      float Rw[V];
#pragma unroll
      for (int v = 0; v < V; ++v) Rw[v] = R[v];
      for (int w = W - 1; w >= 0; --w) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (w == wave) Rw[v] = R[v];
          R[v] = apply(sP[w][lane * V + v], sR[w][lane * V + v], R[v]);
        }
      }
#pragma unroll
      for (int j = 0; j < GS_L; ++j) {                              // the state before each step
        const bool r = st.reset >> j & 1, ok = j < st.live;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h[j][v] = r ? 0.f : H[v];
          if (ok) H[v] = (low[v] + (1.f - low[v]) * up[j][v]) * h[j][v] + (1.f - low[v]) * down[j][v] * x[j][v];
        }
      }
#pragma unroll
      for (int j = GS_L - 1; j >= 0; --j) {
        const bool r = st.reset >> j & 1, ok = j < st.live;
        float ox[V], og[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float k = 1.f - low[v], Dt = e[j][v] + Rw[v], df = Dt * (h[j][v] - x[j][v]);
          ox[v] = ok ? k * down[j][v] * Dt : 0.f;
          og[v] = ok ? df * k * up[j][v] * down[j][v] : 0.f;
          if (ok) {
            dlow[v] += df * down[j][v];
            Rw[v] = r ? 0.f : (low[v] + k * up[j][v]) * Dt;
          }
        }
        if (on && t0 + j < Tn) {
          stv<T, V>(dxr + (t0 + j) * p.d.dx_t, ox);
          stv<T, V>(dgr + (t0 + j) * p.d.dg_t, og);
        }
      }
    }
  }
  if constexpr (!OUT) {
#pragma unroll
    for (int v = 0; v < V; ++v) { sP[wave][lane * V + v] = P[v]; sR[wave][lane * V + v] = R[v]; }
    __syncthreads();
    if (wave == 0 && on) {
      float t[V];
#pragma unroll
      for (int v = 0; v < V; ++v) t[v] = 0.f;
      for (int w = W - 1; w >= 0; --w) {
#pragma unroll
        for (int v = 0; v < V; ++v) t[v] = apply(sP[w][lane * V + v], sR[w][lane * V + v], t[v]);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) p.rev_l[chunk_at + v] = t[v];
    }
  } else {
    if (p.d_h0 && p.nc == 1 && wave == 0 && on) {
#pragma unroll
      for (int v = 0; v < V; ++v) p.d_h0[(int64_t)b * D + c + v] = R[v];
    }
    if (p.floor_part) {
      __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v) sP[wave][lane * V + v] = dlow[v];
      __syncthreads();
      if (wave == 0 && on) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float s = 0.f;
          for (int w = 0; w < W; ++w) s += sP[w][lane * V + v];
          p.floor_part[chunk_at + v] = s;
        }
      }
    }
  }
}

// d_floor[c] = sum over (row, chunk) of their parts, fixed order
__global__ __launch_bounds__(1024) void gated_scan_floor_kernel(const float* __restrict__ part, int64_t n, int D, float* __restrict__ out) {
  __shared__ float sm[16][64];
  const int cl = threadIdx.x & 63, c = blockIdx.x * 64 + cl, w = threadIdx.x >> 6;
  float s = 0.f;
  if (c < D) {
#pragma unroll 4
    for (int64_t k = w; k < n; k += 16) s += part[k * D + c];
  }
  sm[w][cl] = s;
  __syncthreads();
  for (int h = 8; h > 0; h >>= 1) {
    if (w < h) sm[w][cl] += sm[w + h][cl];
    __syncthreads();
  }
  if (w == 0 && c < D) out[c] = sm[0][cl];
}

struct Plan {
  int W, tile, ntiles, nc, tpc;
};
// Waves of a tile by the sequence's length; chunks by how many workgroups the channels alone give (128 channels each): about 1024
// workgroups fill the device.
Plan plan_of(int64_t B, int64_t T, int64_t D) {
  Plan p;
  p.W = T <= 8 ? 1 : (T <= 16 ? 2 : (T <= 32 ? 4 : 8));
  p.tile = p.W * GS_L;
  p.ntiles = (int)cdiv64(T, p.tile);
  const int64_t units = B * cdiv64(D, 128);
  int64_t nc = units >= 1024 || units == 0 ? 1 : cdiv64(1024, units);
  if (nc > p.ntiles) nc = p.ntiles;
  p.tpc = (int)cdiv64(p.ntiles, nc);
  p.nc = (int)cdiv64(p.ntiles, p.tpc);
  return p;
}

bool sizes_ok(int64_t B, int64_t T, int64_t D) {
  return B >= 0 && T >= 1 && D >= 0 && B <= (1 << 24) && T <= (1 << 30) && D <= (1 << 24) && B * cdiv64(D, 64) < ((int64_t)1 << 20);
}

int64_t tile_floats(const Plan& pl, int64_t B, int64_t D) { return (B * pl.ntiles * D + 3) / 4 * 4; }
int64_t chunk_floats(const Plan& pl, int64_t B, int64_t D) { return (B * pl.nc * D + 3) / 4 * 4; }

template <typename P>
bool al(const P* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace

#define ST(s) static_cast<hipStream_t>(s)

extern "C" int tg_gated_scan_sizes(int B, int T, int D, int64_t* carry_floats, int64_t* ws_floats) {
  TG_CHECK_ARG(carry_floats != nullptr && ws_floats != nullptr, "null pointer");
  TG_CHECK_ARG(sizes_ok(B, T, D), "B >= 0, T >= 1, D >= 0 and B * ceil(D / 64) < 2^20 are wanted");
  const Plan pl = plan_of(B, T, D);
  *carry_floats = tile_floats(pl, B, D) + (pl.nc > 1 ? 2 * chunk_floats(pl, B, D) : 0);
  *ws_floats = chunk_floats(pl, B, D) * (pl.nc > 1 ? 3 : 1);
  return TG_OK;
}

namespace {
void set_plan(GsP* p, const Plan& pl, int V, float* carry) {
  const tg_gated_scan_desc& d = p->d;
  p->W = pl.W;
  p->ntiles = pl.ntiles;
  p->nc = pl.nc;
  p->tpc = pl.tpc;
  p->ncb = (int)cdiv64(d.D, 64 * V);
  p->tiles = carry;
  if (pl.nc > 1) {
    p->agg_p = carry + tile_floats(pl, d.B, d.D);
    p->agg_l = p->agg_p + chunk_floats(pl, d.B, d.D);
  }
}
}  // namespace

#define GS_PICK(KERN, OUTV, GRID)                                                                                                   \
  do {                                                                                                                              \
    if (d->dtype == TG_F32) {                                                                                                       \
      if (V == 2) TG_LAUNCH(name, flops, bytes, (KERN<float, 2, OUTV>), dim3(GRID), dim3(64 * pl.W), 0, ST(stream), p);             \
      else TG_LAUNCH(name, flops, bytes, (KERN<float, 1, OUTV>), dim3(GRID), dim3(64 * pl.W), 0, ST(stream), p);                    \
    } else {                                                                                                                        \
      if (V == 2) TG_LAUNCH(name, flops, bytes, (KERN<u16, 2, OUTV>), dim3(GRID), dim3(64 * pl.W), 0, ST(stream), p);               \
      else TG_LAUNCH(name, flops, bytes, (KERN<u16, 1, OUTV>), dim3(GRID), dim3(64 * pl.W), 0, ST(stream), p);                      \
    }                                                                                                                               \
  } while (0)

extern "C" int tg_gated_scan_forward(const tg_gated_scan_desc* d, const void* x, const void* g, const float* h0, const float* floor,
                                     const int32_t* lengths, const unsigned char* reset, void* y, float* hT, float* carry,
                                     int64_t carry_floats, int keep, void* stream) {
  TG_CHECK_ARG(d != nullptr, "null descriptor");
  TG_CHECK_ARG(sizes_ok(d->B, d->T, d->D), "B >= 0, T >= 1, D >= 0 and B * ceil(D / 64) < 2^20 are wanted");
  TG_CHECK_ARG(d->dtype == TG_F32 || d->dtype == TG_BF16, "bad dtype");
  if (d->B == 0 || d->D == 0) return TG_OK;
  TG_CHECK_ARG(x && g && y, "x, g or y is missing");
  TG_CHECK_ARG(d->x_t >= d->D && d->g_t >= d->D && d->y_t >= d->D, "a step stride below D");
  const Plan pl = plan_of(d->B, d->T, d->D);
  const int64_t need = tile_floats(pl, d->B, d->D) + (pl.nc > 1 ? 2 * chunk_floats(pl, d->B, d->D) : 0);
  TG_CHECK_ARG((pl.nc == 1 && !keep) || (carry != nullptr && carry_floats >= need && al(carry, 16)), "the carry of tg_gated_scan_sizes() floats is missing");
  const int es = d->dtype == TG_F32 ? 4 : 2;
  const bool even = d->D % 2 == 0 && al(x, 2 * es) && al(g, 2 * es) && al(y, 2 * es) &&
                    ((d->x_t | d->x_b | d->g_t | d->g_b | d->y_t | d->y_b) & 1) == 0;
  const int V = even ? 2 : 1;
  GsP p = {};
  p.d = *d;
  p.x = x; p.g = g; p.h0 = h0; p.floor = floor; p.lengths = lengths; p.reset = reset; p.y = y; p.hT = hT;
  p.keep_tiles = keep;
  set_plan(&p, pl, V, carry);
  const double n = (double)d->B * d->T * d->D;
  const int64_t blocks = (int64_t)p.ncb * p.nc * d->B;
  if (pl.nc > 1) {
    const char* const name = "gated_scan_fwd<map>";
    const double flops = 10 * n, bytes = 2 * es * n;
    GS_PICK(gated_scan_fwd_kernel, false, (unsigned)blocks);
    hipLaunchKernelGGL(gated_scan_carry_kernel, dim3((unsigned)cdiv64((int64_t)d->B * d->D, 64)), dim3(64), 0, ST(stream), p);
  }
  const char* const name = "gated_scan_fwd";
  const double flops = 14 * n, bytes = 3 * es * n;
  GS_PICK(gated_scan_fwd_kernel, true, (unsigned)blocks);
  TG_CHECK_LAUNCH();
}

extern "C" int tg_gated_scan_backward(const tg_gated_scan_desc* d, const void* x, const void* g, const float* floor,
                                      const int32_t* lengths, const unsigned char* reset, const void* d_y, const float* d_hT,
                                      const float* carry, int64_t carry_floats, void* d_x, void* d_g, float* d_h0, float* d_floor,
                                      float* ws, int64_t ws_floats, void* stream) {
  TG_CHECK_ARG(d != nullptr, "null descriptor");
  TG_CHECK_ARG(sizes_ok(d->B, d->T, d->D), "B >= 0, T >= 1, D >= 0 and B * ceil(D / 64) < 2^20 are wanted");
  TG_CHECK_ARG(d->dtype == TG_F32 || d->dtype == TG_BF16, "bad dtype");
  TG_CHECK_ARG(d_floor == nullptr || floor != nullptr, "d_floor without a floor");
  const Plan pl = plan_of(d->B, d->T, d->D);
  if (d->D == 0) return TG_OK;
  if (d->B > 0) {
    TG_CHECK_ARG(x && g && d_x && d_g, "x, g, d_x or d_g is missing");
    TG_CHECK_ARG(d->x_t >= d->D && d->g_t >= d->D && d->dx_t >= d->D && d->dg_t >= d->D && (!d_y || d->dy_t >= d->D), "a step stride below D");
    const int64_t need = tile_floats(pl, d->B, d->D) + (pl.nc > 1 ? 2 * chunk_floats(pl, d->B, d->D) : 0);
    TG_CHECK_ARG(carry != nullptr && carry_floats >= need && al(carry, 16), "the carry of the forward pass is missing");
    const int64_t cf = chunk_floats(pl, d->B, d->D), want = cf * (pl.nc > 1 ? 3 : 1);
    TG_CHECK_ARG((pl.nc == 1 && !d_floor) || (ws != nullptr && ws_floats >= want && al(ws, 16)), "a workspace of tg_gated_scan_sizes() floats is missing");
    const int es = d->dtype == TG_F32 ? 4 : 2;
    const bool even = d->D % 2 == 0 && al(x, 2 * es) && al(g, 2 * es) && al(d_y, 2 * es) && al(d_x, 2 * es) && al(d_g, 2 * es) &&
                      ((d->x_t | d->x_b | d->g_t | d->g_b | d->dx_t | d->dx_b | d->dg_t | d->dg_b) & 1) == 0 &&
                      (!d_y || ((d->dy_t | d->dy_b) & 1) == 0);
    const int V = even ? 2 : 1;
    GsP p = {};
    p.d = *d;
    p.x = x; p.g = g; p.floor = floor; p.lengths = lengths; p.reset = reset; p.d_y = d_y; p.d_hT = d_hT;
    p.d_x = d_x; p.d_g = d_g; p.d_h0 = d_h0;
    set_plan(&p, pl, V, const_cast<float*>(carry));                // only read by this pass
    p.floor_part = d_floor ? ws : nullptr;
    if (pl.nc > 1) {
      p.rev_l = ws + cf;
      p.rev_in = ws + 2 * cf;
    }
    const double n = (double)d->B * d->T * d->D;
    const int64_t blocks = (int64_t)p.ncb * p.nc * d->B;
    if (pl.nc > 1) {
      const char* const name = "gated_scan_bwd<map>";
      const double flops = 12 * n, bytes = 2 * es * n;
      GS_PICK(gated_scan_bwd_kernel, false, (unsigned)blocks);
      hipLaunchKernelGGL(gated_scan_rcarry_kernel, dim3((unsigned)cdiv64((int64_t)d->B * d->D, 64)), dim3(64), 0, ST(stream), p);
    }
    const char* const name = "gated_scan_bwd";
    const double flops = 40 * n, bytes = 5 * es * n;
    GS_PICK(gated_scan_bwd_kernel, true, (unsigned)blocks);
  }
  if (d_floor)
    hipLaunchKernelGGL(gated_scan_floor_kernel, dim3((unsigned)cdiv64(d->D, 64)), dim3(1024), 0, ST(stream), ws, d->B > 0 ? (int64_t)d->B * pl.nc : 0, d->D, d_floor);
  TG_CHECK_LAUNCH();
}
