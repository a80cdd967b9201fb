// Gated linear recurrence along a sequence, channel by channel:
//
//   f[t] = floor + (1 - floor) sigmoid(g[t]),   h[t] = f[t] h[t-1] + (1 - f[t]) x[t],   y = h,  hT = h[last]
//   backward:  D[t] = dy[t] + f[t+1] D[t+1];  dx = (1 - f) D;  df = D (h[t-1] - x);  dg = df (1 - floor) s(g) s(-g);
//              dfloor = sum df s(-g);  dh0 = f[0] D[0]
//
// A step is an affine map of the state, h -> P h + L, and maps compose: (P2, L2) after (P1, L1) = (P1 P2, P2 L1 + L2).  A sequence
// is cut into chunks, each chunk into tiles of 8 W steps (W waves, 8 steps each in registers): every wave composes its 8 steps,
// the maps meet in LDS, every wave enters its steps with the right state and writes them; the next tile is fetched meanwhile.  Where
// the channels alone fill the device there is one chunk and x, g are read once; otherwise a first launch composes each chunk's map
// and the second one's workgroups compose the maps in front of their chunk (behind it, backward) before they begin: x and g are
// read twice, the second time from the chunk that was read last on, so that the memory-side cache still holds most of them.
// About 14 / 50 operations a value: bound by HBM.  States, maps and gradient sums are fp32; 1 - f is (1 - floor) sigmoid(-g), not a
// difference.  The forward pass keeps the state before every tile (fp32, 1 value in 32): the backward pass makes the states of a tile
// again from it instead of reading rounded ones.
//
// A reset (a new sequence begins at step t) drops the state by selection, not by a product with 0: what was in it, NaN included,
// does not get past.  In a composed map one NaN of its own says that a reset is inside; P may have any other value (a floor outside [0, 1)
// makes f one outside [0, 1]).
// Steps at and behind a row's length keep the state, write y = 0 and zero gradients, and their x, g, dy are not looked at.
//
// Measured on one device: [1, 65536, 1024] bf16 in chunks 141 us (its bytes once 78 us, as read 130); [64, 1, 4096] one step 3.6 us;
// [8, 4096, 1536] bf16 forward 47 + 54, backward 37 + 108 + 5 us; [4, 19, 65536] fp32 in one pass 15.5 and 25.5 us.
#include "common.h"

namespace {

constexpr int GS_L = 8;                                            // steps of a wave in a tile; N = 1 in the kernels where T = 1
constexpr int GS_MAXW = 4;                                         // waves of a workgroup: two small ones on a unit cover each other's
                                                                   // barriers (backward pass 128 us with 8 waves, 109 us with 4)

struct GsP {
  tg_gated_scan_desc d;
  const void *x, *g, *d_y;
  const float *h0, *floor, *d_hT;
  const int32_t* lengths;
  const unsigned char* reset;
  void *y, *d_x, *d_g;
  float *hT, *d_h0;
  float *tiles;                              // [B][ntiles][D] state before each tile
  float *agg_p, *agg_l;                      // [B][nc][D] the chunks' maps (in the last one's L the state in front of the sequence)
  float *rev_l;                              // [B][nc][D] backward: what a chunk adds to the gradient that leaves it in front
  float *floor_part;                         // [B * nc][D]
  int ncb, nc, tpc, ntiles, W;               // channel blocks, chunks, tiles of a chunk, tiles, waves
  int keep_tiles;
};

// V neighbouring channels of one step, as they lie in memory
template <typename T, int V> struct Raw;
template <> struct Raw<u16, 1> {
  u16 w;
  __device__ __forceinline__ void load(const u16* p) { w = *p; }
  __device__ __forceinline__ void zero() { w = 0; }
  __device__ __forceinline__ void values(float (&f)[1]) const { f[0] = bf2f(w); }
  static __device__ __forceinline__ void store(u16* p, const float (&f)[1]) { *p = f2bf(f[0]); }
};
template <> struct Raw<u16, 2> {
  uint32_t w;
  __device__ __forceinline__ void load(const u16* p) { w = reinterpret_cast<const Any32*>(p)->w; }
  __device__ __forceinline__ void zero() { w = 0; }
  __device__ __forceinline__ void values(float (&f)[2]) const {
    f[0] = __uint_as_float(w << 16);
    f[1] = __uint_as_float(w & 0xffff0000u);
  }
  static __device__ __forceinline__ void store(u16* p, const float (&f)[2]) {
    reinterpret_cast<Any32*>(p)->w = (uint32_t)f2bf(f[0]) | ((uint32_t)f2bf(f[1]) << 16);
  }
};
template <> struct Raw<float, 1> {
  float w;
  __device__ __forceinline__ void load(const float* p) { w = *p; }
  __device__ __forceinline__ void zero() { w = 0.f; }
  __device__ __forceinline__ void values(float (&f)[1]) const { f[0] = w; }
  static __device__ __forceinline__ void store(float* p, const float (&f)[1]) { *p = f[0]; }
};
template <> struct Raw<float, 2> {
  float2 w;
  __device__ __forceinline__ void load(const float* p) {
    const Any64 a = *reinterpret_cast<const Any64*>(p);
    w = make_float2(__uint_as_float(a.w[0]), __uint_as_float(a.w[1]));
  }
  __device__ __forceinline__ void zero() { w = make_float2(0.f, 0.f); }
  __device__ __forceinline__ void values(float (&f)[2]) const {
    f[0] = w.x;
    f[1] = w.y;
  }
  static __device__ __forceinline__ void store(float* p, const float (&f)[2]) {
    *reinterpret_cast<Any64*>(p) = Any64{{__float_as_uint(f[0]), __float_as_uint(f[1])}};
  }
};

// sigmoid(g) and sigmoid(-g) without a difference: e = exp(-g), 1 / (1 + e) and e / (1 + e); e past 2^100: 1 (e may be infinite)
template <typename T>
__device__ __forceinline__ void sigmoids(float g, float& up, float& down) {
  const float e = gate_exp<T>(-g);
  up = __builtin_amdgcn_rcpf(1.f + e);
  down = e > 0x1p100f ? 1.f : e * up;
}

// state -> P state + L; P = the NaN of these bits: a reset inside.  Only selected, stored and compared, never calculated with; a NaN of g or of
// the floor has other bits, as long as nobody chooses these.
constexpr uint32_t GS_RESET = 0x7fd1c3a5u;
__device__ __forceinline__ float reset_inside() { return __uint_as_float(GS_RESET); }
__device__ __forceinline__ bool has_reset(float P) { return __float_as_uint(P) == GS_RESET; }
__device__ __forceinline__ float apply(float P, float L, float h) { return has_reset(P) ? L : P * h + L; }
__device__ __forceinline__ float product(float P, float P2) { return has_reset(P) || has_reset(P2) ? reset_inside() : P * P2; }
__device__ __forceinline__ void compose(float& P, float& L, float P2, float L2) {
  L = apply(P2, L2, L);
  P = product(P, P2);
}

// The waves' maps of a tile, read at once (the chain over them waits for LDS one time); where there are fewer than 4 waves the others'
// places hold the identity.
template <int V>
struct Maps {
  float P[GS_MAXW][V], L[GS_MAXW][V];
  __device__ __forceinline__ void read(float (*sP)[64 * V], float (*sL)[64 * V], int lane, int W) {
#pragma unroll
    for (int w = 0; w < GS_MAXW; ++w)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        P[w][v] = sP[w < W ? w : 0][lane * V + v];
        L[w][v] = sL[w < W ? w : 0][lane * V + v];
      }
#pragma unroll
    for (int w = 1; w < GS_MAXW; ++w)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (w >= W) { P[w][v] = 1.f; L[w][v] = 0.f; }
      }
  }
  __device__ __forceinline__ void read_l(float (*sL)[64 * V], int lane, int W) {
#pragma unroll
    for (int w = 0; w < GS_MAXW; ++w)
#pragma unroll
      for (int v = 0; v < V; ++v) L[w][v] = w < W ? sL[w < W ? w : 0][lane * V + v] : 0.f;
  }
};

// What the kernels know of their place: channels, chunk, steps.  Everything but the channel is the same for a whole wave.
template <int V>
struct Place {
  int lane, wave, b, chunk, c, cl, len, ntiles;
  bool on;
  int64_t first;
  __device__ __forceinline__ Place(const GsP& p, int block) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cb = block % p.ncb, rest = block / p.ncb;
    chunk = rest % p.nc;
    b = rest / p.nc;
    c = (cb * 64 + lane) * V;
    on = c < p.d.D;
    cl = on ? c : p.d.D - V;                                       // lanes past the end read the last channels and write nothing
    len = p.d.T;
    if (p.lengths) {
      const int n = p.lengths[b];
      len = n < 0 ? 0 : (n < p.d.T ? n : p.d.T);
    }
    first = (int64_t)chunk * p.tpc;
    ntiles = (int)(p.ntiles - first < p.tpc ? p.ntiles - first : p.tpc);
  }
  // of a wave's 8 steps from t0: how many are live, and (a byte a lane, looked at later) which begin a sequence
  __device__ __forceinline__ int live(int64_t t0) const {
    const int64_t left = len - t0;
    return left < 0 ? 0 : (left > GS_L ? GS_L : (int)left);
  }
  __device__ __forceinline__ unsigned resets(const GsP& p, int64_t t0, int n) const {
    return p.reset && lane < n ? p.reset[(int64_t)b * p.d.T + t0 + lane] : 0;
  }
};

// N steps of one tensor; `base`: its row of the batch (the same for a wave), cl: the lane's channel
template <typename T, int V, int N>
__device__ __forceinline__ void fetch(Raw<T, V> (&r)[N], const T* base, int64_t t0, int64_t stride, int cl, int live) {
  const T* at = base + t0 * stride;
  if (live == N) {
#pragma unroll
    for (int j = 0; j < N; ++j) r[j].load(at + j * stride + cl);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      r[j].zero();
      if (j < live) r[j].load(at + j * stride + cl);
    }
  }
}

// The state that enters a chunk (or, backward, the gradient): `start` carried over the maps of the chunks from..to (step +1 or -1),
// each wave a part of them, the parts joined in LDS.  Every wave returns the same values.
template <int V>
__device__ __forceinline__ void enter(const GsP& p, const Place<V>& q, const float* mp, const float* ml, int count, int from, int step,
                                      float (&h)[V], float (*sP)[64 * V], float (*sL)[64 * V]) {
  const int W = p.W, per = (count + W - 1) / W, i0 = q.wave * per, i1 = i0 + per < count ? i0 + per : count;
  float P[V], L[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { P[v] = 1.f; L[v] = 0.f; }
#pragma unroll 4
  for (int i = i0; i < i1; ++i) {
    const int64_t at = ((int64_t)q.b * p.nc + from + i * step) * p.d.D + q.cl;
#pragma unroll
    for (int v = 0; v < V; ++v) compose(P[v], L[v], mp[at + v], ml[at + v]);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) { sP[q.wave][q.lane * V + v] = P[v]; sL[q.wave][q.lane * V + v] = L[v]; }
  __syncthreads();
  for (int w = 0; w < W; ++w) {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = apply(sP[w][q.lane * V + v], sL[w][q.lane * V + v], h[v]);
  }
  __syncthreads();
}

// Forward.  OUT false: the chunk's map only (each wave a contiguous part of it); true: states and outputs.
template <typename T, int V, bool OUT, int N>
__global__ __launch_bounds__(256) void gated_scan_fwd_kernel(GsP p) {
  __shared__ float sP[GS_MAXW][64 * V], sL[GS_MAXW][64 * V];
  const Place<V> q(p, OUT ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x);
  const int W = p.W, D = p.d.D, lane = q.lane, wave = q.wave;
  const T* const xr = static_cast<const T*>(p.x) + (int64_t)q.b * p.d.x_b;
  const T* const gr = static_cast<const T*>(p.g) + (int64_t)q.b * p.d.g_b;
  T* const yr = static_cast<T*>(p.y) + (int64_t)q.b * p.d.y_b;
  // OUT: tile i, wave after wave; otherwise this wave's i-th group of 8 steps of its contiguous part of the chunk
  auto step0 = [&](int i) -> int64_t { return OUT ? ((q.first + i) * W + wave) * N : (q.first * W + (int64_t)wave * q.ntiles + i) * N; };
  Raw<T, V> rx[N], rg[N];
  int64_t t0 = step0(0);
  int live = q.live(t0);
  fetch<T, V, N>(rg, gr, t0, p.d.g_t, q.cl, live);
  fetch<T, V, N>(rx, xr, t0, p.d.x_t, q.cl, live);
  unsigned rr = q.resets(p, t0, live);
  // The state in front: with chunks from the first launch's copy, since hT may lie over h0 and be written while other chunks begin.  The
  // copy has the place of the last chunk's L, which nothing is composed with (its P the backward pass needs).
  const int64_t last = ((int64_t)q.b * p.nc + p.nc - 1) * D;
  const float* const start = p.nc > 1 ? p.agg_l + last : (p.h0 ? p.h0 + (int64_t)q.b * D : nullptr);
  float low[V], k[V], H[V], P[V], L[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    low[v] = p.floor ? p.floor[q.cl + v] : 0.f;
    k[v] = 1.f - low[v];
    H[v] = OUT && start ? start[q.cl + v] : 0.f;
    P[v] = 1.f;
    L[v] = 0.f;
  }
  if (OUT && q.chunk > 0) enter<V>(p, q, p.agg_p, p.agg_l, q.chunk, 0, 1, H, sP, sL);
  for (int i = 0; i < q.ntiles; ++i) {
    const unsigned fresh = p.reset ? (unsigned)__ballot(rr != 0) : 0;
    const int now = live;
    const int64_t tn = t0;
    float f[N][V], a[N][V];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float g[V], x[V];
      rg[j].values(g);
      rx[j].values(x);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float up, down;
        sigmoids<T>(g[v], up, down);
        f[j][v] = low[v] + k[v] * up;
        a[j][v] = k[v] * down * x[v];
      }
    }
    if (i + 1 < q.ntiles) {
      t0 = step0(i + 1);
      live = q.live(t0);
      fetch<T, V, N>(rg, gr, t0, p.d.g_t, q.cl, live);
      fetch<T, V, N>(rx, xr, t0, p.d.x_t, q.cl, live);
      rr = q.resets(p, t0, live);
    }
    if (now < N) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j >= now) {
#pragma unroll
          for (int v = 0; v < V; ++v) { f[j][v] = 1.f; a[j][v] = 0.f; }
        }
    }
    if (OUT) {
#pragma unroll
      for (int v = 0; v < V; ++v) { P[v] = 1.f; L[v] = 0.f; }
    }
    if (fresh == 0) {
      float Q[V];
#pragma unroll
      for (int v = 0; v < V; ++v) Q[v] = 1.f;
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          L[v] = f[j][v] * L[v] + a[j][v];
          Q[v] *= f[j][v];
        }
#pragma unroll
      for (int v = 0; v < V; ++v) P[v] = has_reset(P[v]) ? P[v] : P[v] * Q[v];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) compose(P[v], L[v], fresh >> j & 1 ? reset_inside() : f[j][v], a[j][v]);
    }
    if constexpr (OUT) {
      float h[V];
      if (W > 1) {
        if (i > 0) __syncthreads();                                // the last tile's maps have been read
#pragma unroll
        for (int v = 0; v < V; ++v) { sP[wave][lane * V + v] = P[v]; sL[wave][lane * V + v] = L[v]; }
        __syncthreads();
      }
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = H[v];
      if (p.keep_tiles && wave == 0 && q.on) {
        float* const st = p.tiles + ((int64_t)q.b * p.ntiles + q.first + i) * D + q.c;
#pragma unroll
        for (int v = 0; v < V; ++v) st[v] = H[v];
      }
      if (W > 1) {
        Maps<V> m;
        m.read(sP, sL, lane, W);
#pragma unroll
        for (int w = 0; w < GS_MAXW; ++w)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            if (w == wave) h[v] = H[v];
            H[v] = apply(m.P[w][v], m.L[w][v], H[v]);
          }
      }
      T* const out = yr + tn * p.d.y_t;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h[v] = (fresh >> j & 1 ? 0.f : f[j][v] * h[v]) + a[j][v];
          o[v] = j < now ? h[v] : 0.f;
        }
        if (tn + j < p.d.T && q.on) Raw<T, V>::store(out + j * p.d.y_t + q.c, o);
      }
      if (W == 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) H[v] = h[v];
      }
    }
  }
  if constexpr (OUT) {
    if (p.hT && q.chunk == p.nc - 1 && wave == 0 && q.on) {
#pragma unroll
      for (int v = 0; v < V; ++v) p.hT[(int64_t)q.b * D + q.c + v] = H[v];
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) { sP[wave][lane * V + v] = P[v]; sL[wave][lane * V + v] = L[v]; }
    __syncthreads();
    if (wave == 0 && q.on) {
      for (int w = 1; w < W; ++w) {
#pragma unroll
        for (int v = 0; v < V; ++v) compose(P[v], L[v], sP[w][lane * V + v], sL[w][lane * V + v]);
      }
      const int64_t at = ((int64_t)q.b * p.nc + q.chunk) * D + q.c;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        p.agg_p[at + v] = P[v];
        p.agg_l[at + v] = q.chunk < p.nc - 1 ? L[v] : (p.h0 ? p.h0[(int64_t)q.b * D + q.c + v] : 0.f);
      }
    }
  }
}

// Backward.  OUT false: what a chunk adds to the gradient that leaves it in front; true: the gradients.
template <typename T, int V, bool OUT, int N>
__global__ __launch_bounds__(256) void gated_scan_bwd_kernel(GsP p) {
  __shared__ float sP[GS_MAXW][64 * V], sL[GS_MAXW][64 * V], sR[GS_MAXW][64 * V];
  const Place<V> q(p, OUT ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x);
  const int W = p.W, D = p.d.D, lane = q.lane, wave = q.wave;
  const T* const xr = static_cast<const T*>(p.x) + (int64_t)q.b * p.d.x_b;
  const T* const gr = static_cast<const T*>(p.g) + (int64_t)q.b * p.d.g_b;
  const T* const er = static_cast<const T*>(p.d_y) + (int64_t)q.b * p.d.dy_b;
  T* const dxr = static_cast<T*>(p.d_x) + (int64_t)q.b * p.d.dx_b;
  T* const dgr = static_cast<T*>(p.d_g) + (int64_t)q.b * p.d.dg_b;
  auto step0 = [&](int i) -> int64_t { return OUT ? ((q.first + i) * W + wave) * N : (q.first * W + (int64_t)wave * q.ntiles + i) * N; };
  Raw<T, V> rx[N], rg[N], re[N];
  float rH[V];
  auto fetch_all = [&](int i, int64_t t0, int live) {
    fetch<T, V, N>(rg, gr, t0, p.d.g_t, q.cl, live);
    fetch<T, V, N>(re, er, t0, p.d.dy_t, q.cl, p.d_y ? live : 0);
    if (OUT) {
      fetch<T, V, N>(rx, xr, t0, p.d.x_t, q.cl, live);
      const float* const st = p.tiles + ((int64_t)q.b * p.ntiles + q.first + i) * D + q.cl;
#pragma unroll
      for (int v = 0; v < V; ++v) rH[v] = st[v];
    }
  };
  int64_t t0 = step0(q.ntiles - 1);
  int live = q.live(t0);
  fetch_all(q.ntiles - 1, t0, live);
  unsigned rr = q.resets(p, t0, live);
  float low[V], k[V], R[V], dlow[V], P[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    low[v] = p.floor ? p.floor[q.cl + v] : 0.f;
    k[v] = 1.f - low[v];
    R[v] = OUT && p.d_hT ? p.d_hT[(int64_t)q.b * D + q.cl + v] : 0.f;
    dlow[v] = 0.f;
    P[v] = 1.f;
  }
  if (OUT && q.chunk < p.nc - 1) enter<V>(p, q, p.agg_p, p.rev_l, p.nc - 1 - q.chunk, p.nc - 1, -1, R, sP, sL);
  for (int i = q.ntiles - 1; i >= 0; --i) {
    const unsigned fresh = p.reset ? (unsigned)__ballot(rr != 0) : 0;
    const int now = live;
    const int64_t tn = t0;
    float up[N][V], down[N][V], x[N][V], e[N][V], H[V];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float g[V];
      rg[j].values(g);
      re[j].values(e[j]);
      if (OUT) rx[j].values(x[j]);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        sigmoids<T>(g[v], up[j][v], down[j][v]);
        H[v] = rH[v];
      }
    }
    if (i > 0) {
      t0 = step0(i - 1);
      live = q.live(t0);
      fetch_all(i - 1, t0, live);
      rr = q.resets(p, t0, live);
    }
    if constexpr (!OUT) {
#pragma unroll
      for (int j = N - 1; j >= 0; --j) {
        if (j < now) {
          const bool r = fresh >> j & 1;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float f = low[v] + k[v] * up[j][v];
            R[v] = r ? 0.f : f * (e[j][v] + R[v]);
            P[v] = r || has_reset(P[v]) ? reset_inside() : P[v] * f;
          }
        }
      }
    } else {
      float Lf[V], Lr[V];
#pragma unroll
      for (int v = 0; v < V; ++v) { P[v] = 1.f; Lf[v] = 0.f; Lr[v] = 0.f; }
      if (now == N && fresh == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float f = low[v] + k[v] * up[j][v];
            Lf[v] = f * Lf[v] + k[v] * down[j][v] * x[j][v];
            P[v] *= f;
          }
#pragma unroll
        for (int j = N - 1; j >= 0; --j)
#pragma unroll
          for (int v = 0; v < V; ++v) Lr[v] = (low[v] + k[v] * up[j][v]) * (e[j][v] + Lr[v]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (j < now) {
#pragma unroll
            for (int v = 0; v < V; ++v) compose(P[v], Lf[v], fresh >> j & 1 ? reset_inside() : low[v] + k[v] * up[j][v], k[v] * down[j][v] * x[j][v]);
          }
#pragma unroll
        for (int j = N - 1; j >= 0; --j)
          if (j < now) {
#pragma unroll
            for (int v = 0; v < V; ++v) Lr[v] = fresh >> j & 1 ? 0.f : (low[v] + k[v] * up[j][v]) * (e[j][v] + Lr[v]);
          }
      }
      float Rw[V];
      if (W > 1) {
        if (i < q.ntiles - 1) __syncthreads();                     // the last tile's maps have been read
#pragma unroll
        for (int v = 0; v < V; ++v) {
          sP[wave][lane * V + v] = P[v];
          sL[wave][lane * V + v] = Lf[v];
          sR[wave][lane * V + v] = Lr[v];
        }
        __syncthreads();
        Maps<V> m;
        m.read(sP, sL, lane, W);
#pragma unroll
        for (int w = 0; w < GS_MAXW; ++w)
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (w < wave) H[v] = apply(m.P[w][v], m.L[w][v], H[v]);
        m.read_l(sR, lane, W);
#pragma unroll
        for (int v = 0; v < V; ++v) Rw[v] = R[v];
#pragma unroll
        for (int w = GS_MAXW - 1; w >= 0; --w)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            if (w == wave) Rw[v] = R[v];
            R[v] = apply(m.P[w][v], m.L[w][v], R[v]);
          }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) Rw[v] = R[v];
      }
      float h[N][V];
#pragma unroll
      for (int j = 0; j < N; ++j) {                              // the state before each step
        const bool r = fresh >> j & 1;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h[j][v] = r ? 0.f : H[v];
          H[v] = (low[v] + k[v] * up[j][v]) * h[j][v] + k[v] * down[j][v] * x[j][v];   // behind the live steps nobody looks at it
        }
      }
      T* const ox = dxr + tn * p.d.dx_t;
      T* const og = dgr + tn * p.d.dg_t;
#pragma unroll
      for (int j = N - 1; j >= 0; --j) {
        float vx[V], vg[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { vx[v] = 0.f; vg[v] = 0.f; }
        if (j < now) {
          const bool r = fresh >> j & 1;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float Dt = e[j][v] + Rw[v], df = Dt * (h[j][v] - x[j][v]) * down[j][v];
            vx[v] = k[v] * down[j][v] * Dt;
            vg[v] = k[v] * df * up[j][v];
            dlow[v] += df;
            Rw[v] = r ? 0.f : (low[v] + k[v] * up[j][v]) * Dt;
          }
        }
        if (tn + j < p.d.T && q.on) {
          Raw<T, V>::store(ox + j * p.d.dx_t + q.c, vx);
          Raw<T, V>::store(og + j * p.d.dg_t + q.c, vg);
        }
      }
      if (W == 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) R[v] = Rw[v];
      }
    }
  }
  const int64_t chunk_at = ((int64_t)q.b * p.nc + q.chunk) * D + q.c;
  if constexpr (!OUT) {
#pragma unroll
    for (int v = 0; v < V; ++v) { sP[wave][lane * V + v] = P[v]; sR[wave][lane * V + v] = R[v]; }
    __syncthreads();
    (void)sL;
    if (wave == 0 && q.on) {
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
    if (p.d_h0 && q.chunk == 0 && wave == 0 && q.on) {
#pragma unroll
      for (int v = 0; v < V; ++v) p.d_h0[(int64_t)q.b * D + q.c + v] = R[v];
    }
    if (p.floor_part) {
      __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v) sP[wave][lane * V + v] = dlow[v];
      __syncthreads();
      if (wave == 0 && q.on) {
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
// Waves of a tile by the sequence's length.  Chunks: the time goes as tiles of a chunk x rounds of 512 workgroups (two a compute unit:
// 128 channels x one chunk each; fewer than four a unit reach about 1 / 1.3 of the bandwidth) x bytes a value (3 tensors in one pass,
// 5 in two), and the second launch of a chunked pass costs about as much as 13 of these units (measured: a tile and a round about
// 0.8 us, a launch with its gap 4 us).  The fewest chunks at the least of it.  The plan fixes the scratch buffers' sizes and the order of the
// sums, which a host may ask for where no device is: it takes the 256 compute units of a whole MI355X instead of asking.
constexpr int GS_PLACES = 2 * 256;
Plan plan_of(int64_t B, int64_t T, int64_t D) {
  Plan p;
  p.W = T <= 24 ? (int)cdiv64(T, GS_L) : GS_MAXW;
  p.tile = p.W * GS_L;
  p.ntiles = (int)cdiv64(T, p.tile);
  const int64_t units = B * cdiv64(D, 128);
  double best = 0.0;
  p.nc = p.tpc = 0;
  for (int64_t n = 1, tpc = p.ntiles; n == 1 || units * n <= 4096; n = cdiv64(p.ntiles, tpc - 1), tpc = cdiv64(p.ntiles, n)) {
    const int64_t blocks = units * n;                              // n: the fewest chunks of tpc tiles
    const double rounds = (double)cdiv64(blocks, GS_PLACES);
    const double cost = tpc * rounds * (blocks < 2 * GS_PLACES ? 1.3 : 1.0) * (n == 1 ? 3 : 5) + (n == 1 ? 0 : 13 + 0.08 * n * rounds);
    if (p.nc == 0 || cost < best) {
      best = cost;
      p.nc = (int)n;
      p.tpc = (int)tpc;
    }
    if (tpc == 1) break;
  }
  return p;
}

// Channels of a lane: two, but one where D is odd or a wave of single ones covers it.  [64, 4096, 40] bf16, forward and backward: 60 and
// 87 us with two, 44 and 53 with one; [4, 4096, 4096]: 122 and 201 with two, 149 and 208 with one.
int lane_channels(int D) { return D % 2 == 0 && D > 64 ? 2 : 1; }

bool sizes_ok(int64_t B, int64_t T, int64_t D) {
  return B >= 0 && T >= 1 && D >= 0 && B <= (1 << 24) && T <= (1 << 30) && D <= (1 << 24) && B * cdiv64(D, 64) < ((int64_t)1 << 20);
}

int64_t tile_floats(const Plan& pl, int64_t B, int64_t D) { return (B * pl.ntiles * D + 3) / 4 * 4; }
int64_t chunk_floats(const Plan& pl, int64_t B, int64_t D) { return (B * pl.nc * D + 3) / 4 * 4; }

// rows of D values at strides t (T of them) and b (B of them): no two share one.  Outputs only: inputs may be windows over one another.
bool apart(int64_t t, int64_t b, int64_t B, int64_t T, int64_t D) {
  return (B == 1 || b >= D) && (B == 1 || T == 1 || b >= (T - 1) * t + D || t >= (B - 1) * b + D);
}

template <typename P>
bool al(const P* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace

#define ST(s) static_cast<hipStream_t>(s)

extern "C" int tg_gated_scan_sizes(int B, int T, int D, int64_t* carry_floats, int64_t* ws_floats) {
  TG_CHECK_ARG(carry_floats != nullptr && ws_floats != nullptr, "null pointer");
  TG_CHECK_ARG(sizes_ok(B, T, D), "B >= 0, T >= 1, D >= 0 and B * ceil(D / 64) < 2^20 are wanted");
  const Plan pl = plan_of(B, T, D);
  *carry_floats = tile_floats(pl, B, D) + (pl.nc > 1 ? 2 * chunk_floats(pl, B, D) : 0);
  *ws_floats = chunk_floats(pl, B, D) * (pl.nc > 1 ? 2 : 1);
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

#define GS_PICK(KERN, OUTV, NV, GRID)                                                                                               \
  do {                                                                                                                              \
    if (d->dtype == TG_F32) {                                                                                                       \
      if (V == 2) TG_LAUNCH(name, flops, bytes, (KERN<float, 2, OUTV, NV>), dim3(GRID), dim3(64 * pl.W), 0, ST(stream), p);         \
      else TG_LAUNCH(name, flops, bytes, (KERN<float, 1, OUTV, NV>), dim3(GRID), dim3(64 * pl.W), 0, ST(stream), p);                \
    } else {                                                                                                                        \
      if (V == 2) TG_LAUNCH(name, flops, bytes, (KERN<u16, 2, OUTV, NV>), dim3(GRID), dim3(64 * pl.W), 0, ST(stream), p);           \
      else TG_LAUNCH(name, flops, bytes, (KERN<u16, 1, OUTV, NV>), dim3(GRID), dim3(64 * pl.W), 0, ST(stream), p);                  \
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
  TG_CHECK_ARG(apart(d->y_t, d->y_b, d->B, d->T, d->D), "batch rows of y overlap");
  const int es = d->dtype == TG_F32 ? 4 : 2;
  const int V = lane_channels(d->D);
  GsP p = {};
  p.d = *d;
  p.x = x; p.g = g; p.h0 = h0; p.floor = floor; p.lengths = lengths; p.reset = reset; p.y = y; p.hT = hT;
  p.keep_tiles = keep != 0;
  set_plan(&p, pl, V, carry);
  const double n = (double)d->B * d->T * d->D;
  const int64_t blocks = (int64_t)p.ncb * p.nc * d->B;
  if (pl.nc > 1) {
    const char* const name = "gated_scan_fwd<map>";
    const double flops = 10 * n, bytes = 2 * es * n;
    GS_PICK(gated_scan_fwd_kernel, false, GS_L, (unsigned)blocks);
  }
  const char* const name = "gated_scan_fwd";
  const double flops = 14 * n, bytes = 3 * es * n;
  // single steps: seven more that are not there cost their exponentials ([256, 1, 8192] bf16: 10.6 us, with them 17.6; backward 11.3 and 29.4)
  if (d->T == 1) GS_PICK(gated_scan_fwd_kernel, true, 1, (unsigned)blocks);
  else GS_PICK(gated_scan_fwd_kernel, true, GS_L, (unsigned)blocks);
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
    const int64_t cf = chunk_floats(pl, d->B, d->D), want = cf * (pl.nc > 1 ? 2 : 1);
    TG_CHECK_ARG((pl.nc == 1 && !d_floor) || (ws != nullptr && ws_floats >= want && al(ws, 16)), "a workspace of tg_gated_scan_sizes() floats is missing");
    TG_CHECK_ARG(apart(d->dx_t, d->dx_b, d->B, d->T, d->D) && apart(d->dg_t, d->dg_b, d->B, d->T, d->D), "batch rows of d_x or d_g overlap");
    const int es = d->dtype == TG_F32 ? 4 : 2;
    // Three waves of two channels: their 200 - 225 registers leave a quarter of a unit's places empty, one channel needs 122 ([64, 20, 8192]
    // bf16 40.5 us with two, 35 with one; four waves 41; with 32 steps 37.5 and 41)
    const int V = pl.W == 3 ? 1 : lane_channels(d->D);
    GsP p = {};
    p.d = *d;
    p.x = x; p.g = g; p.floor = floor; p.lengths = lengths; p.reset = reset; p.d_y = d_y; p.d_hT = d_hT;
    p.d_x = d_x; p.d_g = d_g; p.d_h0 = d_h0;
    set_plan(&p, pl, V, const_cast<float*>(carry));                // only read by this pass
    p.floor_part = d_floor ? ws : nullptr;
    if (pl.nc > 1) p.rev_l = ws + cf;
    const double n = (double)d->B * d->T * d->D;
    const int64_t blocks = (int64_t)p.ncb * p.nc * d->B;
    if (pl.nc > 1) {
      const char* const name = "gated_scan_bwd<map>";
      const double flops = 12 * n, bytes = 2 * es * n;
      GS_PICK(gated_scan_bwd_kernel, false, GS_L, (unsigned)blocks);
    }
    const char* const name = "gated_scan_bwd";
    const double flops = 40 * n, bytes = 5 * es * n;
    if (d->T == 1) GS_PICK(gated_scan_bwd_kernel, true, 1, (unsigned)blocks);
    else GS_PICK(gated_scan_bwd_kernel, true, GS_L, (unsigned)blocks);
  }
  if (d_floor)
    hipLaunchKernelGGL(gated_scan_floor_kernel, dim3((unsigned)cdiv64(d->D, 64)), dim3(1024), 0, ST(stream), ws, d->B > 0 ? (int64_t)d->B * pl.nc : 0, d->D, d_floor);
  TG_CHECK_LAUNCH();
}
