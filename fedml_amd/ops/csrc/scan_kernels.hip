// Gated linear recurrence (driven by ops/scan_ops.py), per sequence and feature:
//   f_t = σ(gate_t),  h_t = f_t h_{t−1} + (1 − f_t) x_t,  y_t = h_t
//   backward, with G_t = f_t δ_t handed on to step t − 1:  δ_t = dy_t + G_{t+1} (dh_T for the last step)
//   dx_t = (1 − f_t) δ_t,  dgate_t = δ_t (h_{t−1} − x_t) f_t (1 − f_t),  dh_0 = G_1
// A masked step has f = 1 and takes nothing: the state passes it, y, dx and dgate are zero there.
//
// Any run of steps is an affine map of the state, h → A h + B, and maps compose: a workgroup owns 32·V features of one
// sequence and walks the time in tiles of 32 steps; 8 groups of 32 lanes take 4 steps each in registers, put their maps
// into LDS, and every group composes those before it. The carried state stays in fp32 registers; x and gate are read
// once. The forward leaves the state before every tile (fp32, 1/32 of the states): the backward recomputes the
// others in registers from there, so it reads x, gate and dy only and loses nothing to the rounding of y.
// Few features and a long time: the time is cut into segments, whose maps a first kernel forms (same reads); the
// workgroups of the second compose those before (after, backward) their segment. Order fixed, no atomics.
//
// Bound by bandwidth. Measured on MI355X (a large copy: 4.94 TB/s), bf16, forward / backward (3 / 5 streams):
// [1, 2048, 64, 1024] 177 / 318 us = 4.5 / 4.2 TB/s; [8, 2048, 16, 670] 310 / 565 us = 3.4 / 3.1 TB/s, where rows of 1340
// bytes split every line between two workgroups (672 features: 254 / 467 us); [1, 16384, 4, 1024] cut into 16 segments
// 77 / 136 us + 78 / 62 for the maps. Tiles of 64 steps (8 a thread) took the forward of 670 features 420 us: 95
// registers left 5 workgroups a CU for the 5.5 that there are.
#include "common.h"

namespace scan {

constexpr int kTile = 32, kGroups = 8, kSteps = kTile / kGroups;
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const void *x, *gate, *dy;
  void *y, *dx, *dgate;
  const float *h0, *dh;
  float *hT, *dh0, *ckpt, *agg;
  const uint8_t* mask;
  int64_t xs[3], gs[3], dys[3], ys[3], ms[3];   // element strides over client, time and sequence; y, dx and dgate share ys
  int C, T, B, H, nseg, tps;                    // tps: tiles of a segment, even if there are several
};

template <typename T, int V> struct Vec;
template <> struct Vec<uint16_t, 2> {
  typedef uint32_t raw;
  static __device__ __forceinline__ void get(raw u, float* f) {
    f[0] = __uint_as_float(u << 16);
    f[1] = __uint_as_float(u & 0xffff0000u);
  }
  static __device__ __forceinline__ raw put(const float* f) {
    return (uint32_t)f32_to_bf16(f[0]) | ((uint32_t)f32_to_bf16(f[1]) << 16);
  }
};
template <> struct Vec<uint16_t, 1> {
  typedef uint16_t raw;
  static __device__ __forceinline__ void get(raw u, float* f) { f[0] = bf16_to_f32(u); }
  static __device__ __forceinline__ raw put(const float* f) { return f32_to_bf16(f[0]); }
};
template <> struct Vec<float, 2> {
  typedef float2 raw;
  static __device__ __forceinline__ void get(raw u, float* f) {
    f[0] = u.x;
    f[1] = u.y;
  }
  static __device__ __forceinline__ raw put(const float* f) { return make_float2(f[0], f[1]); }
};
template <> struct Vec<float, 1> {
  typedef float raw;
  static __device__ __forceinline__ void get(raw u, float* f) { f[0] = u; }
  static __device__ __forceinline__ raw put(const float* f) { return f[0]; }
};

// f = σ(g) and 1 − f = e^−g f, without the cancellation of the difference; below −80 f is smaller than any state's
// last bit (and e^−g stays finite)
__device__ __forceinline__ void gates(float g, float& f, float& keep) {
  const float c = g < -80.f ? -80.f : g;
  const float e = __builtin_amdgcn_exp2f(c * -kLog2e);
  f = __builtin_amdgcn_rcpf(1.f + e);
  keep = e * f;
}

// where a workgroup and a thread stand
template <int V> struct At {
  int c, b, seg, lane, grp, j0, j, jr;   // features: the workgroup's first, the thread's, one that exists
  bool on;
  __device__ __forceinline__ explicit At(const Args& a) {
    const int nft = (a.H + 32 * V - 1) / (32 * V);
    // consecutive work items to the same XCD (workgroup ids go round the 8 of them): where rows are no whole cache
    // lines, the two workgroups that share one meet in one L2
    const int per = gridDim.x >> 3, wg = blockIdx.x;
    int id = wg < per * 8 ? (wg & 7) * per + (wg >> 3) : wg;
    const int ft = id % nft;
    id /= nft;
    seg = id % a.nseg;
    id /= a.nseg;
    b = id % a.B;
    c = id / a.B;
    lane = threadIdx.x & 31;
    grp = threadIdx.x >> 5;
    j0 = ft * 32 * V;
    j = j0 + lane * V;
    on = j < a.H;
    jr = on ? j : 0;
  }
};

// one stream of a thread's N steps; every load is made, of steps up to the last and features that exist
template <typename T, int V, int N> struct Steps {
  typename Vec<T, V>::raw r[N];
  __device__ __forceinline__ void load(const T* p, int64_t st, int t0, int T_) {
    if (t0 + N <= T_) {
      const T* q = p + t0 * st;
#pragma unroll
      for (int i = 0; i < N; ++i, q += st) r[i] = *reinterpret_cast<const typename Vec<T, V>::raw*>(q);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        r[i] = *reinterpret_cast<const typename Vec<T, V>::raw*>(p + (t0 + i < T_ ? t0 + i : T_ - 1) * st);
    }
  }
};

// lane i < N of a group: is step t0 + i one of the text's
template <int N> __device__ __forceinline__ int real_step(const uint8_t* m, int64_t st, int t0, int T_, int lane) {
  const int t = t0 + (lane & (N - 1));
  const int r = m ? m[(t < T_ ? t : T_ - 1) * st] : 1;
  return t < T_ ? r : 0;
}
// bit i: step t0 + i of this thread's group
template <int N> __device__ __forceinline__ uint32_t real_bits(int real) {
  return (uint32_t)((uint64_t)__ballot(real != 0) >> (threadIdx.x & 32)) & ((1u << N) - 1);
}

template <typename T, int V, int N>
__device__ __forceinline__ void values(const Steps<T, V, N>& x, const Steps<T, V, N>& g, uint32_t bits, float (*f)[V],
                                       float (*keep)[V], float (*xv)[V]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float gv[V];
    Vec<T, V>::get(g.r[i], gv);
    Vec<T, V>::get(x.r[i], xv[i]);
#pragma unroll
    for (int v = 0; v < V; ++v) gates(gv[v], f[i][v], keep[i][v]);
  }
  if (__any(bits != (1u << N) - 1)) {      // padding somewhere: a step of it keeps the state and takes nothing
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const bool real = (bits >> i) & 1;
        f[i][v] = real ? f[i][v] : 1.f;
        keep[i][v] = real ? keep[i][v] : 0.f;
        xv[i][v] = real ? xv[i][v] : 0.f;
      }
  }
}

// The first 32·V threads carry the states of the workgroup's features, one each, from group to group and tile to tile
// (the last ones, in the backward, the gradients that go the other way); a group gets what it starts from through LDS.
// With every thread composing the maps before its own, their reads took the backward's registers (134 instead of 95, 3
// waves a SIMD instead of 5): 162 instead of 137 us at 16384 steps of 4096 features.
template <typename T, int V> __global__ __launch_bounds__(256) void fwd_kernel(const Args a) {
  __shared__ float sA[kGroups][32 * V], sB[kGroups][32 * V], sS[kGroups][32 * V];
  const At<V> at(a);
  const int ntile = (a.T + kTile - 1) / kTile;
  const int k0 = at.seg * a.tps, k1 = k0 + a.tps < ntile ? k0 + a.tps : ntile;
  const T* x = (const T*)a.x + at.c * a.xs[0] + at.b * a.xs[2] + at.jr;
  const T* g = (const T*)a.gate + at.c * a.gs[0] + at.b * a.gs[2] + at.jr;
  T* y = (T*)a.y + at.c * a.ys[0] + at.b * a.ys[2] + at.j;
  const uint8_t* m = a.mask ? a.mask + at.c * a.ms[0] + at.b * a.ms[2] : nullptr;
  const int q = threadIdx.x, jq = at.j0 + q;           // a carrying thread's feature
  const bool carries = q < 32 * V, onq = carries && jq < a.H;
  const int64_t seq = (int64_t)at.c * a.B + at.b;
  float h = onq && a.h0 ? a.h0[seq * a.H + jq] : 0.f;
  for (int s = 0; s < at.seg && onq; ++s) {            // the segments before this one
    const float* p = a.agg + (seq * a.nseg + s) * 2 * a.H + jq;
    h = fmaf(p[0], h, p[a.H]);
  }
  Steps<T, V, kSteps> rx, rg;
  int real;
  auto load = [&](int k) {
    const int t0 = k * kTile + at.grp * kSteps;
    real = real_step<kSteps>(m, a.ms[1], t0, a.T, at.lane);
    rx.load(x, a.xs[1], t0, a.T);
    rg.load(g, a.gs[1], t0, a.T);
  };
  load(k0);
  for (int k = k0; k < k1; ++k) {
    const int t0 = k * kTile + at.grp * kSteps;
    const uint32_t bits = real_bits<kSteps>(real);
    float f[kSteps][V], keep[kSteps][V], in[kSteps][V], A[V], Bv[V];
    values<T, V, kSteps>(rx, rg, bits, f, keep, in);
    if (k + 1 < k1) load(k + 1);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      A[v] = 1.f;
      Bv[v] = 0.f;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        in[i][v] *= keep[i][v];
        A[v] *= f[i][v];
        Bv[v] = fmaf(f[i][v], Bv[v], in[i][v]);
      }
      sA[at.grp][at.lane * V + v] = A[v];
      sB[at.grp][at.lane * V + v] = Bv[v];
    }
    __syncthreads();
    if (carries) {
      if (onq && a.ckpt) a.ckpt[(((int64_t)at.c * ntile + k) * a.B + at.b) * a.H + jq] = h;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        sS[i][q] = h;
        h = fmaf(sA[i][q], h, sB[i][q]);
      }
    }
    __syncthreads();
    float s[V];
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = sS[at.grp][at.lane * V + v];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      float o[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        s[v] = fmaf(f[i][v], s[v], in[i][v]);
        o[v] = (bits >> i) & 1 ? s[v] : 0.f;
      }
      if (at.on && t0 + i < a.T)
        *reinterpret_cast<typename Vec<T, V>::raw*>(y + (t0 + i) * a.ys[1]) = Vec<T, V>::put(o);
    }
  }
  if (onq && k1 == ntile) a.hT[seq * a.H + jq] = h;
}

template <typename T, int V> __global__ __launch_bounds__(256) void bwd_kernel(const Args a) {
  __shared__ float sA[kGroups][32 * V], sB[kGroups][32 * V], sG[kGroups][32 * V], sS[kGroups][32 * V],
      sE[kGroups][32 * V];
  const At<V> at(a);
  const int ntile = (a.T + kTile - 1) / kTile;
  const int k0 = at.seg * a.tps, k1 = k0 + a.tps < ntile ? k0 + a.tps : ntile;
  const T* x = (const T*)a.x + at.c * a.xs[0] + at.b * a.xs[2] + at.jr;
  const T* g = (const T*)a.gate + at.c * a.gs[0] + at.b * a.gs[2] + at.jr;
  const T* dy = (const T*)a.dy + at.c * a.dys[0] + at.b * a.dys[2] + at.jr;
  T* dx = (T*)a.dx + at.c * a.ys[0] + at.b * a.ys[2] + at.j;
  T* dg = (T*)a.dgate + at.c * a.ys[0] + at.b * a.ys[2] + at.j;
  const uint8_t* m = a.mask ? a.mask + at.c * a.ms[0] + at.b * a.ms[2] : nullptr;
  // the first threads carry states, the last ones gradients
  const bool fore = threadIdx.x < 32 * V, aft = threadIdx.x >= 256 - 32 * V;
  const int q = fore ? threadIdx.x : threadIdx.x - (256 - 32 * V), jq = at.j0 + q;
  const bool onq = (fore || aft) && jq < a.H;
  const int64_t seq = (int64_t)at.c * a.B + at.b;
  float G = 0.f, hn = 0.f;
  if (aft && onq) {
    if (a.dh) G = a.dh[seq * a.H + jq];
    for (int s = a.nseg - 1; s > at.seg; --s) {              // the segments after this one
      const float* p = a.agg + (seq * a.nseg + s) * 2 * a.H + jq;
      G = fmaf(p[0], G, p[a.H]);
    }
  }
  Steps<T, V, kSteps> rx, rg, rd;
  int real;
  auto load = [&](int k) {
    const int t0 = k * kTile + at.grp * kSteps;
    real = real_step<kSteps>(m, a.ms[1], t0, a.T, at.lane);
    rx.load(x, a.xs[1], t0, a.T);
    rg.load(g, a.gs[1], t0, a.T);
    rd.load(dy, a.dys[1], t0, a.T);
    if (fore && onq) hn = a.ckpt[(((int64_t)at.c * ntile + k) * a.B + at.b) * a.H + jq];   // the state before the tile
  };
  load(k1 - 1);
  for (int k = k1 - 1; k >= k0; --k) {
    const int t0 = k * kTile + at.grp * kSteps;
    const uint32_t bits = real_bits<kSteps>(real);
    float f[kSteps][V], keep[kSteps][V], xv[kSteps][V], d[kSteps][V];
    values<T, V, kSteps>(rx, rg, bits, f, keep, xv);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      Vec<T, V>::get(rd.r[i], d[i]);
#pragma unroll
      for (int v = 0; v < V; ++v) d[i][v] = (bits >> i) & 1 ? d[i][v] : 0.f;
    }
    float h = hn;
    if (k > k0) load(k - 1);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float A = 1.f, Bv = 0.f, Gv = 0.f;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        A *= f[i][v];
        Bv = fmaf(f[i][v], Bv, keep[i][v] * xv[i][v]);
      }
#pragma unroll
      for (int i = kSteps - 1; i >= 0; --i) Gv = f[i][v] * (d[i][v] + Gv);
      sA[at.grp][at.lane * V + v] = A;
      sB[at.grp][at.lane * V + v] = Bv;
      sG[at.grp][at.lane * V + v] = Gv;
    }
    __syncthreads();
    if (fore) {
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        sS[i][q] = h;
        h = fmaf(sA[i][q], h, sB[i][q]);
      }
    } else if (aft) {
#pragma unroll
      for (int i = kGroups - 1; i >= 0; --i) {
        sE[i][q] = G;
        G = fmaf(sA[i][q], G, sG[i][q]);
      }
    }
    __syncthreads();
    // dgate without δ, (h_{t−1} − x_t) f_t (1 − f_t), is formed on the way forward, in x's place
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s = sS[at.grp][at.lane * V + v];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const float n = fmaf(f[i][v], s, keep[i][v] * xv[i][v]);
        xv[i][v] = (s - xv[i][v]) * (f[i][v] * keep[i][v]);
        s = n;
      }
    }
    float e[V];
#pragma unroll
    for (int v = 0; v < V; ++v) e[v] = sE[at.grp][at.lane * V + v];
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) {
      float ox[V], og[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float dl = d[i][v] + e[v];
        ox[v] = keep[i][v] * dl;
        og[v] = xv[i][v] * dl;
        e[v] = f[i][v] * dl;
      }
      if (at.on && t0 + i < a.T) {
        *reinterpret_cast<typename Vec<T, V>::raw*>(dx + (t0 + i) * a.ys[1]) = Vec<T, V>::put(ox);
        *reinterpret_cast<typename Vec<T, V>::raw*>(dg + (t0 + i) * a.ys[1]) = Vec<T, V>::put(og);
      }
    }
  }
  if (aft && onq && k0 == 0 && a.dh0) a.dh0[seq * a.H + jq] = G;
}

// the map of every segment: forward h → A h + B (from x), backward G → A G + B (from dy)
template <typename T, int V, bool BWD> __global__ __launch_bounds__(256) void agg_kernel(const Args a) {
  __shared__ float sA[kGroups][32 * V], sB[kGroups][32 * V];
  const At<V> at(a);
  const int ntile = (a.T + kTile - 1) / kTile;
  const int k0 = at.seg * a.tps, k1 = k0 + a.tps < ntile ? k0 + a.tps : ntile;
  const T* g = (const T*)a.gate + at.c * a.gs[0] + at.b * a.gs[2] + at.jr;
  const T* o = BWD ? (const T*)a.dy + at.c * a.dys[0] + at.b * a.dys[2] + at.jr
                   : (const T*)a.x + at.c * a.xs[0] + at.b * a.xs[2] + at.jr;
  const int64_t ot = BWD ? a.dys[1] : a.xs[1];
  const uint8_t* m = a.mask ? a.mask + at.c * a.ms[0] + at.b * a.ms[2] : nullptr;
  // a group walks a run of the segment of its own: its map is formed without a barrier
  constexpr int N = 8;
  const int run = ((k1 - k0) * kTile / kGroups + N - 1) / N * N;     // whole tiles of it but in the last segment
  const int ta = k0 * kTile + at.grp * run, tb = ta + run;
  float A[V], Bv[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = 1.f;
    Bv[v] = 0.f;
  }
  Steps<T, V, N> rg, ro;
  int real;
  const int n = run / N;
  auto load = [&](int i) {
    const int t0 = BWD ? tb - (i + 1) * N : ta + i * N;
    real = real_step<N>(m, a.ms[1], t0, a.T, at.lane);
    rg.load(g, a.gs[1], t0, a.T);
    ro.load(o, ot, t0, a.T);
  };
  load(0);
  for (int i = 0; i < n; ++i) {
    float f[N][V], keep[N][V], ov[N][V];
    values<T, V, N>(ro, rg, real_bits<N>(real), f, keep, ov);
    if (i + 1 < n) load(i + 1);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int r = BWD ? N - 1 - u : u;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        A[v] *= f[r][v];
        Bv[v] = BWD ? f[r][v] * (ov[r][v] + Bv[v]) : fmaf(f[r][v], Bv[v], keep[r][v] * ov[r][v]);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sA[at.grp][at.lane * V + v] = A[v];
    sB[at.grp][at.lane * V + v] = Bv[v];
  }
  __syncthreads();
  if (at.grp || !at.on) return;
  float* p = a.agg + (((int64_t)at.c * a.B + at.b) * a.nseg + at.seg) * 2 * a.H + at.j;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float A1 = 1.f, B1 = 0.f;
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
      const int i = BWD ? kGroups - 1 - u : u;
      B1 = fmaf(sA[i][at.lane * V + v], B1, sB[i][at.lane * V + v]);
      A1 *= sA[i][at.lane * V + v];
    }
    p[v] = A1;
    p[a.H + v] = B1;
  }
}

template <typename T, int V> int launch(const Args& a, bool bwd, hipStream_t st) {
  const int64_t n = (int64_t)a.C * a.B * a.nseg * ((a.H + 32 * V - 1) / (32 * V));
  const dim3 grid((unsigned)n), block(256);
  if (a.nseg > 1) {
    if (bwd) hipLaunchKernelGGL((agg_kernel<T, V, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((agg_kernel<T, V, false>), grid, block, 0, st, a);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
  }
  if (bwd) hipLaunchKernelGGL((bwd_kernel<T, V>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((fwd_kernel<T, V>), grid, block, 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace scan

// vec: 2 where every row starts at a multiple of two elements and H is even, else 1
FA_EXPORT int fa_gated_scan(const scan::Args* a, int bf16, int vec, int bwd, hipStream_t stream) {
  if (bf16) return vec == 2 ? scan::launch<uint16_t, 2>(*a, bwd, stream) : scan::launch<uint16_t, 1>(*a, bwd, stream);
  return vec == 2 ? scan::launch<float, 2>(*a, bwd, stream) : scan::launch<float, 1>(*a, bwd, stream);
}
