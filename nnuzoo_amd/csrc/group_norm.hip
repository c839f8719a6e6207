// Group norm with an activation, channels last (gfx950), forward and backward:
//   z = (x - mu[n,g]) * r[n,g] * w[c] + b[c],  y = act(z),  mu / r over the S positions and C / G channels of a group;
//   dz = dy act'(z),  db = sum dz,  dw = sum dz xhat,  dx = r (w dz - <w dz> - xhat <w dz xhat>)  with <.> the group's mean.
// Bound by HBM: a group does not fit on chip, so forward reads x twice and writes y, backward reads x and dy twice and writes dx.
// 2 x 128^3 x 32 f16 (268 MB a tensor), SiLU: sums 66 us (4.1 TB/s), write pass 90 (6.0), backward sums 127 (4.2, the logistic
// function's share shows), write pass 149 (5.4), finishing launches 5 each.
//
// A thread owns V consecutive channels (16 bytes) and walks the rows, a workgroup has a share of the rows of one sample: every access
// is a run of whole rows whatever the group width, and the group's members meet only after the rows are summed.  The forward's sums
// are fp64 (whose vector rate is that of plain fp32 here): E[x^2] - mu^2 then costs about 2^-53 (mu / sigma)^2 of the variance, less than
// its rounding to fp32 up to mu / sigma = 2^14 and 2^-13 at 2^20, where x itself has 4 bits left for the spread.  Partial sums go
// through a workspace and are added in a fixed order: results are bit-identical from run to run.
// No atomics.
#include "elem_io.hpp"

namespace nnz {

enum GnAct { GN_NONE = 0, GN_RELU = 1, GN_LEAKY = 2, GN_SILU = 3 };
constexpr int GN_NT = 256;

struct GnArgs {
  const void* x;      // [N][S][C] with strides xb, xs, 1
  const void* dy;     // [N][S][C] contiguous
  const float* w;     // [C] or null (ones)
  const float* b;     // [C] or null (zeros)
  void* out;          // y or dx, [N][S][C] contiguous; backward: null where x needs no gradient
  float* stats;       // [N][G][2]: mean, 1 / sqrt(var + eps)
  double* gpart;      // [N][nblk][G][2]
  float* cpart;       // backward: [N][nblk][C][2]: sum dz, sum dz xhat
  float* cc;          // backward: [N][G][2]: <w dz>, <w dz xhat>
  float* dw;          // [C] or null
  float* db;
  long N, S, xb, xs;
  int nblk, C, G, q;        // q = C / G
  int act;
  float slope, eps;
};

__device__ __forceinline__ float gn_act(float z, int act, float slope) {
  switch (act) {
    case GN_RELU: return z < 0.f ? 0.f : z;  // NaN stays
    case GN_LEAKY: return z > 0.f ? z : z * slope;
    case GN_SILU: return z * sigmoid_hw(z);
    default: return z;
  }
}
__device__ __forceinline__ float gn_dact(float z, float dy, int act, float slope) {
  switch (act) {
    case GN_RELU: return z > 0.f ? dy : 0.f;
    case GN_LEAKY: return z > 0.f ? dy : dy * slope;
    case GN_SILU: {
      const float s = sigmoid_hw(z);
      return dy * (s * (1.f + z * (1.f - s)));
    }
    default: return dy;
  }
}

// a workgroup takes the parts (samples x a.nblk) of a launch in turn; more parts than a grid may have workgroups are rare
#define GN_FOR_EACH_PART(a) for (long part = blockIdx.x; part < (a).N * (a).nblk; part += gridDim.x)
constexpr long GN_MAX_WG = 1L << 22;   // 2^32 threads are too many

// a thread's place: vector columns [c0, c0 + cw) of the row are dealt out over the workgroup, R rows at a time
struct GnPlace {
  int col, rr, R;
  bool on;
};
template <int NT = GN_NT>
__device__ __forceinline__ GnPlace gn_place(int cw, int tid = threadIdx.x) {
  GnPlace p;
  p.R = NT / cw;
  p.rr = tid / cw;
  p.col = tid - p.rr * cw;
  p.on = p.rr < p.R;
  return p;
}

// per-channel sums over the workgroup's row threads, of a pair of values: s[V], t[V] of every thread -> dst_s[channel],
// dst_t[channel], in a fixed order.  stage: [2 * NT * V].  All threads first share out the rows of a channel, then its partial sums
// are added.
template <class A, int V, int NT = GN_NT>
__device__ __forceinline__ void gn_fold_rows(A* stage, A* dst_s, A* dst_t, const A (&s)[V], const A (&t)[V], const GnPlace& p,
                                             int cw) {
  A* st2 = stage + NT * V;
  const int ch = cw * V;
  __syncthreads();
  if (p.on) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      stage[threadIdx.x * V + j] = s[j];
      st2[threadIdx.x * V + j] = t[j];
    }
  }
  __syncthreads();
  if (ch > NT) {
    for (int c = threadIdx.x; c < ch; c += NT) {
      A u = 0, v = 0;
      for (int r = 0; r < p.R; ++r) {
        u += stage[r * ch + c];
        v += st2[r * ch + c];
      }
      if (dst_s) dst_s[c] = u;
      if (dst_t) dst_t[c] = v;
    }
    return;
  }
  const int parts = NT / ch, part = threadIdx.x / ch, c = threadIdx.x - part * ch;
  A u = 0, v = 0;
  if (part < parts)
    for (int r = part; r < p.R; r += parts) {
      u += stage[r * ch + c];
      v += st2[r * ch + c];
    }
  __syncthreads();
  if (part < parts) {
    stage[threadIdx.x] = u;
    st2[threadIdx.x] = v;
  }
  __syncthreads();
  if (part == 0) {
    const int n = parts < p.R ? parts : p.R;
    for (int k = 1; k < n; ++k) {
      u += stage[k * ch + c];
      v += st2[k * ch + c];
    }
    if (dst_s) dst_s[c] = u;
    if (dst_t) dst_t[c] = v;
  }
}

// per-group sums of two per-channel sums [2][C], weighted by w, in fp64 and in a fixed order: up to 64 lanes a group
template <class A>
__device__ __forceinline__ void gn_fold_groups(const GnArgs& a, const A* sums, const float* w, double* out) {
  int lp = 1;
  while (2 * lp <= a.q && lp < 64) lp *= 2;
  const int li = threadIdx.x & (lp - 1);
  for (int g = threadIdx.x / lp; g < a.G; g += GN_NT / lp) {
    double u = 0.0, v = 0.0;
    for (int c = g * a.q + li; c < (g + 1) * a.q; c += lp) {
      const double k = w ? w[c] : 1.0;
      u = fma(k, (double)sums[c], u);
      v = fma(k, (double)sums[a.C + c], v);
    }
    for (int o = lp / 2; o > 0; o >>= 1) {
      u += __shfl_xor(u, o, 64);
      v += __shfl_xor(v, o, 64);
    }
    if (li == 0) {
      out[2 * g] = u;
      out[2 * g + 1] = v;
    }
  }
}

// fp64 throughout: fp32 sums about a thread's own first value took as long (the kernel waits for memory) and are at the mercy of
// that value.
template <class TI, int V>
__global__ __launch_bounds__(GN_NT) void gn_stats_kernel(GnArgs a) {
  extern __shared__ __attribute__((aligned(16))) double gn_lds_d[];
  double* stage = gn_lds_d;                 // [2][GN_NT * V]
  double* sums = gn_lds_d + 2 * GN_NT * V;  // [2][C]
  GN_FOR_EACH_PART(a) {
    const long n = part / a.nblk, blk = part - n * a.nblk;
    const TI* xn = (const TI*)a.x + n * a.xb;
    const int CV = a.C / V;
    for (int c0 = 0; c0 < CV; c0 += GN_NT) {
      const int cw = CV - c0 < GN_NT ? CV - c0 : GN_NT;
      const GnPlace p = gn_place(cw);
      double s[V], sq[V];
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = sq[j] = 0.0;
      if (p.on) {
        const TI* xc = xn + (long)(c0 + p.col) * V;
#pragma unroll 2
        for (long r = blk * p.R + p.rr; r < a.S; r += (long)a.nblk * p.R) {
          float v[V];
          ld_elems<TI, V>(xc + r * a.xs, v);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const double d = (double)v[j];
            s[j] += d;
            sq[j] = fma(d, d, sq[j]);
          }
        }
      }
      gn_fold_rows<double, V>(stage, sums + c0 * V, sums + a.C + c0 * V, s, sq, p, cw);
    }
    __syncthreads();
    gn_fold_groups(a, sums, nullptr, a.gpart + part * a.G * 2);
  }
}

// pairs [nblk] of one (sample, group) summed by one wave
__device__ __forceinline__ void gn_sum_parts(const double* p, int nblk, int G, double& s, double& t) {
  s = t = 0.0;
  for (int k = threadIdx.x & 63; k < nblk; k += 64) {
    s += p[(long)k * G * 2];
    t += p[(long)k * G * 2 + 1];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    t += __shfl_xor(t, o, 64);
  }
}

__global__ __launch_bounds__(64) void gn_stats_finish_kernel(GnArgs a) {
  for (long pair = blockIdx.x; pair < a.N * a.G; pair += gridDim.x) {
    const long n = pair / a.G;
    const int g = (int)(pair - n * a.G);
    double s, sq;
    gn_sum_parts(a.gpart + (n * a.nblk * a.G + g) * 2, a.nblk, a.G, s, sq);
    if (threadIdx.x == 0) {
      const double m = (double)a.S * a.q, mean = s / m;
      double var = sq / m - mean * mean;
      if (var < 0.0) var = 0.0;  // NaN stays
      a.stats[pair * 2] = (float)mean;
      a.stats[pair * 2 + 1] = (float)(1.0 / sqrt(var + (double)a.eps));
    }
  }
}

// constants of a thread's V channels, which lie in GV groups of V / GV channels (registers decide how many waves hide the loads)
template <int V, int GV>
struct GnChan {
  float mean[GV], rstd[GV], w[V], b[V];
  __device__ __forceinline__ void load(const GnArgs& a, long n, int c) {
#pragma unroll
    for (int i = 0; i < GV; ++i) {
      const float* st = a.stats + (n * a.G + (c + i * (V / GV)) / a.q) * 2;
      mean[i] = st[0];
      rstd[i] = st[1];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[j] = a.w ? a.w[c + j] : 1.f;
      b[j] = a.b ? a.b[c + j] : 0.f;
    }
  }
  __device__ __forceinline__ float xhat(int j, float v) const { return (v - mean[j / (V / GV)]) * rstd[j / (V / GV)]; }
  __device__ __forceinline__ float z(int j, float xh) const { return fmaf(xh, w[j], b[j]); }
};

template <class TI, class TO, int V, int GV>
__global__ __launch_bounds__(GN_NT) void gn_apply_kernel(GnArgs a) {
  GN_FOR_EACH_PART(a) {
    const long n = part / a.nblk, blk = part - n * a.nblk;
    const TI* xn = (const TI*)a.x + n * a.xb;
    TO* yn = (TO*)a.out + n * a.S * a.C;
    const int CV = a.C / V;
    for (int c0 = 0; c0 < CV; c0 += GN_NT) {
      const int cw = CV - c0 < GN_NT ? CV - c0 : GN_NT;
      const GnPlace p = gn_place(cw);
      if (!p.on) continue;
      const int c = (c0 + p.col) * V;
      GnChan<V, GV> k;
      k.load(a, n, c);
#pragma unroll 1
      for (long r = blk * p.R + p.rr; r < a.S; r += (long)a.nblk * p.R) {
        float v[V];
        ld_elems<TI, V>(xn + r * a.xs + c, v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = gn_act(k.z(j, k.xhat(j, v[j])), a.act, a.slope);
        st_elems<TO, V>(yn + r * a.C + c, v);
      }
    }
  }
}

// backward sums: per channel sum dz and sum dz xhat of the workgroup's rows, and their weighted sums per group
template <class TI, class TO, int V, int GV>
__global__ __launch_bounds__(GN_NT) void gn_bwd_reduce_kernel(GnArgs a) {
  extern __shared__ __attribute__((aligned(16))) float gn_lds_f[];
  float* stage = gn_lds_f;                 // [2][GN_NT * V]
  float* sums = gn_lds_f + 2 * GN_NT * V;  // [2][C]
  GN_FOR_EACH_PART(a) {
    const long n = part / a.nblk, blk = part - n * a.nblk;
    const TI* xn = (const TI*)a.x + n * a.xb;
    const TO* gn = (const TO*)a.dy + n * a.S * a.C;
    const int CV = a.C / V;
    for (int c0 = 0; c0 < CV; c0 += GN_NT) {
      const int cw = CV - c0 < GN_NT ? CV - c0 : GN_NT;
      const GnPlace p = gn_place(cw);
      float s[V], t[V];
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = t[j] = 0.f;
      if (p.on) {
        const int c = (c0 + p.col) * V;
        GnChan<V, GV> k;
        k.load(a, n, c);
#pragma unroll 2
        for (long r = blk * p.R + p.rr; r < a.S; r += (long)a.nblk * p.R) {
          float v[V], g[V];
          ld_elems<TI, V>(xn + r * a.xs + c, v);
          ld_elems<TO, V>(gn + r * a.C + c, g);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float xh = k.xhat(j, v[j]);
            const float dz = gn_dact(k.z(j, xh), g[j], a.act, a.slope);
            s[j] += dz;
            t[j] = fmaf(dz, xh, t[j]);
          }
        }
      }
      gn_fold_rows<float, V>(stage, sums + c0 * V, sums + a.C + c0 * V, s, t, p, cw);
    }
    __syncthreads();
    float* cp = a.cpart + part * a.C * 2;
    for (int c = threadIdx.x; c < a.C; c += GN_NT) {
      cp[2 * c] = sums[c];
      cp[2 * c + 1] = sums[a.C + c];
    }
    gn_fold_groups(a, sums, a.w, a.gpart + part * a.G * 2);
  }
}

constexpr int GN_FC = 4;  // channels of a finishing workgroup: 4 x 64 threads share the partial sums of 4 channels
// workgroups 0 .. pair_wgs - 1: <w dz>, <w dz xhat> of the (sample, group) pairs, a wave each; the rest: dw and db
__global__ __launch_bounds__(GN_NT) void gn_bwd_finish_kernel(GnArgs a, long pair_wgs) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((long)blockIdx.x < pair_wgs) {
    for (long pair = (long)blockIdx.x * 4 + wave; pair < a.N * a.G; pair += pair_wgs * 4) {
      const long n = pair / a.G;
      double s, t;
      gn_sum_parts(a.gpart + (n * a.nblk * a.G + (pair - n * a.G)) * 2, a.nblk, a.G, s, t);
      if (lane == 0) {
        const double m = (double)a.S * a.q;
        a.cc[pair * 2] = (float)(s / m);
        a.cc[pair * 2 + 1] = (float)(t / m);
      }
    }
    return;
  }
  // lanes 4k + i of the workgroup's 256: partial k, k + 64, .. of channel i
  const int c = (int)((long)blockIdx.x - pair_wgs) * GN_FC + (threadIdx.x & (GN_FC - 1));
  const long parts = a.N * a.nblk;
  double s = 0.0, t = 0.0;
  if (c < a.C) {
    const float* cp = a.cpart + 2 * (long)c;
#pragma unroll 8
    for (long k = threadIdx.x / GN_FC; k < parts; k += GN_NT / GN_FC) {
      s += cp[k * a.C * 2];
      t += cp[k * a.C * 2 + 1];
    }
  }
#pragma unroll
  for (int o = 32; o >= GN_FC; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    t += __shfl_xor(t, o, 64);
  }
  __shared__ double red[4][GN_FC][2];
  if (lane < GN_FC) {
    red[wave][lane][0] = s;
    red[wave][lane][1] = t;
  }
  __syncthreads();
  if (threadIdx.x < GN_FC && c < a.C) {
    if (a.db) a.db[c] = (float)((red[0][lane][0] + red[1][lane][0]) + (red[2][lane][0] + red[3][lane][0]));
    if (a.dw) a.dw[c] = (float)((red[0][lane][1] + red[1][lane][1]) + (red[2][lane][1] + red[3][lane][1]));
  }
}

template <class TI, class TO, int V, int GV>
__global__ __launch_bounds__(GN_NT) void gn_bwd_apply_kernel(GnArgs a) {
  GN_FOR_EACH_PART(a) {
    const long n = part / a.nblk, blk = part - n * a.nblk;
    const TI* xn = (const TI*)a.x + n * a.xb;
    const TO* gn = (const TO*)a.dy + n * a.S * a.C;
    TI* on = (TI*)a.out + n * a.S * a.C;
    const int CV = a.C / V;
    for (int c0 = 0; c0 < CV; c0 += GN_NT) {
      const int cw = CV - c0 < GN_NT ? CV - c0 : GN_NT;
      const GnPlace p = gn_place(cw);
      if (!p.on) continue;
      const int c = (c0 + p.col) * V;
      GnChan<V, GV> k;
      k.load(a, n, c);
      float m1[GV], m2[GV];
#pragma unroll
      for (int i = 0; i < GV; ++i) {
        const float* cc = a.cc + (n * a.G + (c + i * (V / GV)) / a.q) * 2;
        m1[i] = cc[0];
        m2[i] = cc[1];
      }
#pragma unroll 1
      for (long r = blk * p.R + p.rr; r < a.S; r += (long)a.nblk * p.R) {
        float v[V], g[V];
        ld_elems<TI, V>(xn + r * a.xs + c, v);
        ld_elems<TO, V>(gn + r * a.C + c, g);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          constexpr int Q = V / GV;
          const float xh = k.xhat(j, v[j]);
          const float dz = gn_dact(k.z(j, xh), g[j], a.act, a.slope);
          v[j] = k.rstd[j / Q] * (k.w[j] * dz - m1[j / Q] - xh * m2[j / Q]);
        }
        st_elems<TI, V>(on + r * a.C + c, v);
      }
    }
  }
}

// ---- small groups ------------------------------------------------------------------------------------------------------------
// A team of T threads - a workgroup, or a wave where groups are many and tiny - owns the C / G channels of a
// group: of one sample at a time in the forward, of every K-th sample in turn in the backward (K = 1 for few samples: the weight
// gradients then need no second stage).  One launch in the forward, one or two in the backward; the row segments are short, but
// everything stays in L2.
constexpr int GN_SNT = 512;
// sum over a team of a pair, the same bits in all its threads; red: [2 * GN_SNT / 64]
template <int T>
__device__ __forceinline__ void gn_team_sum(double& s, double& t, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    t += __shfl_xor(t, o, 64);
  }
  if constexpr (T > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      red[2 * (threadIdx.x >> 6)] = s;
      red[2 * (threadIdx.x >> 6) + 1] = t;
    }
    __syncthreads();
    s = t = 0.0;
#pragma unroll
    for (int w = 0; w < GN_SNT / 64; ++w) {
      s += red[2 * w];
      t += red[2 * w + 1];
    }
  }
}

template <class TI, class TO, int V, int T>
__global__ __launch_bounds__(GN_SNT) void gn_small_fwd_kernel(GnArgs a) {
  __shared__ double red[2 * GN_SNT / 64];
  constexpr int TEAMS = GN_SNT / T;
  const int cw = a.q / V;
  const GnPlace p = gn_place<T>(cw, threadIdx.x % T);
  for (long pair = (long)blockIdx.x * TEAMS + threadIdx.x / T; pair < a.N * a.G; pair += (long)gridDim.x * TEAMS) {
    const long n = pair / a.G;
    const int c = (int)(pair - n * a.G) * a.q + p.col * V;
    const TI* x = (const TI*)a.x + n * a.xb + c;
    double s = 0.0, sq = 0.0;
    if (p.on) {
#pragma unroll 4
      for (long r = p.rr; r < a.S; r += p.R) {
        float v[V];
        ld_elems<TI, V>(x + r * a.xs, v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const double d = (double)v[j];
          s += d;
          sq = fma(d, d, sq);
        }
      }
    }
    gn_team_sum<T>(s, sq, red);
    const double m = (double)a.S * a.q, mean = s / m;
    double var = sq / m - mean * mean;
    if (var < 0.0) var = 0.0;  // NaN stays
    const float mu = (float)mean, rstd = (float)(1.0 / sqrt(var + (double)a.eps));
    if (threadIdx.x % T == 0) {
      a.stats[pair * 2] = mu;
      a.stats[pair * 2 + 1] = rstd;
    }
    if (!p.on) continue;
    float w[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[j] = a.w ? a.w[c + j] : 1.f;
      b[j] = a.b ? a.b[c + j] : 0.f;
    }
    TO* y = (TO*)a.out + n * a.S * a.C + c;
#pragma unroll 4
    for (long r = p.rr; r < a.S; r += p.R) {
      float v[V];
      ld_elems<TI, V>(x + r * a.xs, v);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = gn_act(fmaf((v[j] - mu) * rstd, w[j], b[j]), a.act, a.slope);
      st_elems<TO, V>(y + r * a.C, v);
    }
  }
}

// teams: K of a group; a.cpart: [K][C][2] where K > 1
template <class TI, class TO, int V, int T>
__global__ __launch_bounds__(GN_SNT) void gn_small_bwd_kernel(GnArgs a, int K) {
  __shared__ double red[2 * GN_SNT / 64];
  __shared__ float stage[2 * GN_SNT * V];
  constexpr int TEAMS = GN_SNT / T;
  const int team = threadIdx.x / T;
  const long id = (long)blockIdx.x * TEAMS + team;
  if (T == 64 && id >= (long)K * a.G) return;   // a wave on its own: no barrier follows
  const int k = (int)(id / a.G), g = (int)(id - (long)k * a.G), cw = a.q / V;
  const GnPlace p = gn_place<T>(cw, threadIdx.x % T);
  const int c = g * a.q + p.col * V;
  float w[V], b[V], sw[V], sb[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    w[j] = a.w && p.on ? a.w[c + j] : 1.f;
    b[j] = a.b && p.on ? a.b[c + j] : 0.f;
    sw[j] = sb[j] = 0.f;
  }
  const double m = (double)a.S * a.q;
  for (long n = k; n < a.N; n += K) {
    const TI* x = (const TI*)a.x + n * a.xb + c;
    const TO* dy = (const TO*)a.dy + n * a.S * a.C + c;
    TI* dx = a.out ? (TI*)a.out + n * a.S * a.C + c : nullptr;
    const float mu = a.stats[(n * a.G + g) * 2], rstd = a.stats[(n * a.G + g) * 2 + 1];
    double s = 0.0, t = 0.0;
    if (p.on) {
#pragma unroll 2
      for (long r = p.rr; r < a.S; r += p.R) {
        float v[V], d[V];
        ld_elems<TI, V>(x + r * a.xs, v);
        ld_elems<TO, V>(dy + r * a.C, d);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xh = (v[j] - mu) * rstd;
          const float dz = gn_dact(fmaf(xh, w[j], b[j]), d[j], a.act, a.slope);
          sb[j] += dz;
          sw[j] = fmaf(dz, xh, sw[j]);
          const double wdz = (double)w[j] * dz;
          s += wdz;
          t = fma(wdz, (double)xh, t);
        }
      }
    }
    gn_team_sum<T>(s, t, red);
    const float m1 = (float)(s / m), m2 = (float)(t / m);
    if (p.on && a.out) {
#pragma unroll 2
      for (long r = p.rr; r < a.S; r += p.R) {
        float v[V], d[V];
        ld_elems<TI, V>(x + r * a.xs, v);
        ld_elems<TO, V>(dy + r * a.C, d);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xh = (v[j] - mu) * rstd;
          const float dz = gn_dact(fmaf(xh, w[j], b[j]), d[j], a.act, a.slope);
          v[j] = rstd * (w[j] * dz - m1 - xh * m2);
        }
        st_elems<TI, V>(dx + r * a.C, v);
      }
    }
  }
  // per-channel sums over the team's rows, in a fixed order: to dw and db, or to the team's row of partial sums
  float* st1 = stage + team * T * V;
  float* st2 = st1 + GN_SNT * V;
  const int tid = threadIdx.x % T, ch = cw * V;
  if (p.on) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      st1[tid * V + j] = sb[j];
      st2[tid * V + j] = sw[j];
    }
  }
  if (T == 64) wave_lds_sync();
  else __syncthreads();
  for (int i = tid; i < ch; i += T) {
    float u = 0.f, v = 0.f;
    for (int r = 0; r < p.R; ++r) {
      u += st1[r * ch + i];
      v += st2[r * ch + i];
    }
    const int o = g * a.q + i;
    if (K > 1) {
      a.cpart[((long)k * a.C + o) * 2] = u;
      a.cpart[((long)k * a.C + o) * 2 + 1] = v;
    } else {
      if (a.db) a.db[o] = u;
      if (a.dw) a.dw[o] = v;
    }
  }
}

constexpr int GN_MAX_C = 4096;    // C and 256 x V fp64 pairs fit LDS
constexpr long GN_TARGET = 1024;  // workgroups of a launch that sums
constexpr long GN_TARGET_APPLY = 4096;  // of one that writes (1 024: 119 us instead of 89 for the forward at 2 x 128^3 x 32 f16)
// Workgroups of a sample: enough to fill the chip, with at least 8 passes over the rows that their threads cover at once.  The rows
// are dealt out in turn, so that the chip reads one moving window: runs of rows a workgroup lie a power of two apart on the usual
// sizes, and their streams then meet in the same memory channels (the forward's sums and write pass at 2 x 128^3 x 32 f16: 70 and 97 us
// that way, 66 and 90 in turn; the backward's 128 and 145 us, and 126 and 149).
inline void gn_split(GnArgs& a, int V, long target) {
  const int CV = a.C / V;
  const long R = CV >= GN_NT ? 1 : GN_NT / CV;
  long per = (target + a.N - 1) / a.N;
  const long most = (a.S + 8 * R - 1) / (8 * R);
  if (per > most) per = most;
  a.nblk = (int)(per < 1 ? 1 : per);
}
// Which kernels a call takes, by forward + backward on the device, fp32 unless said otherwise (32 channels in 8 groups, other shapes alike):
// - one launch each way (small groups) up to GN_ROWS rows: 2 x 512 x 32: 20 us against 25 by rows, 2 x 1024: 24 against 26, 2 x 2048: 33
//   against 26, 2 x 4096: 49 against 26;
// - and up to GN_SEGS row segments altogether, for a segment narrower than a line costs as much as a line: 16 x 512: 21 against 26, 32 x 512
//   (2^17): 26 against 26, 32 x 1024: 46 against 27, 128 x 1024: 143 against 37.  From 64 channels a group on a segment is whole lines
//   (64 x 128 x 512 in 8 groups: 27 against 41);
// - a wave is team enough for GN_WAVE elements once there are more pairs than workgroups to keep the chip busy: 128 x 128 x 32: 15 us by
//   waves, 34 by workgroups, 23 by rows; 32 x 32 x 32: 12, 19, 18.  Few pairs of 1 024 elements are quicker by workgroups (32 x 102 x 60 in
//   6 groups: 13 by workgroups, 20 by waves), so up to 256 pairs half as many elements count.
constexpr long GN_SMALL = 16384, GN_WAVE = 1024, GN_ROWS = 1024, GN_SEGS = 1L << 17;
inline bool gn_by_wave(long N, long S, int G, int q) {
  return q <= 64 && S * q <= (N * G > 256 ? GN_WAVE : GN_WAVE / 2) && N * G > 64;
}
inline bool gn_small(long N, long S, int G, int q) {
  return q <= GN_SNT && S * q <= GN_SMALL && (gn_by_wave(N, S, G, q) || (S <= GN_ROWS && (q >= 64 || N * G * S <= GN_SEGS)));
}
// teams of a group in the backward: one walks up to four samples (4 x 128 x 32, forward + backward: 22 us on the device against 18 by a
// team a sample, but the launch that adds partial weight gradients is spared, 7 us of a call by itself); else as many as fill the chip
// (8 x 512 x 32: 20 us, by one team 36)
inline int gn_teams(long N, long S, int G, int q) {
  if (N <= 4) return 1;
  long k = (gn_by_wave(N, S, G, q) ? 8192 : 1024) / G;
  if (k > N) k = N;
  return (int)(k < 1 ? 1 : k);
}
inline dim3 gn_grid(long wgs) { return dim3((unsigned)(wgs < GN_MAX_WG ? wgs : GN_MAX_WG)); }
inline long gn_align(long v) { return (v + 255) & ~255L; }
// layout of the workspace, the same whatever V a call's alignment allows
struct GnWs {
  long gpart, cpart, cc, bytes;
};
inline GnWs gn_ws(long N, long S, int C, int G, bool bwd) {
  if (gn_small(N, S, G, C / G)) {
    const int k = bwd ? gn_teams(N, S, G, C / G) : 1;
    return GnWs{0, 0, 0, k > 1 ? (long)k * C * 8 : 0};
  }
  long parts = (GN_TARGET + N - 1) / N;   // no split has more parts a sample
  if (parts > S) parts = S;
  GnWs w;
  w.gpart = 0;
  w.cpart = gn_align(N * parts * G * 16);
  w.cc = w.cpart + (bwd ? gn_align(N * parts * C * 8) : 0);
  w.bytes = w.cc + (bwd ? gn_align(N * G * 8) : 0);
  return w;
}

// one function, and so one cache, a kernel: the callers differ in the output's type and the groups of a vector
template <class TI, int V>
static int gn_stats(const GnArgs& a, hipStream_t s) {
  static DynLdsCache cache;
  const int lds = (GN_NT * V + a.C) * 2 * 8;
  hipError_t e = ensure_dyn_lds((const void*)gn_stats_kernel<TI, V>, lds, cache);
  if (e != hipSuccess) return (int)e;
  NNZ_LAUNCH((gn_stats_kernel<TI, V>), gn_grid(a.N * a.nblk), dim3(GN_NT), lds, s, a);
  NNZ_LAUNCH_CHECK();
  return NNZ_OK;
}
template <class TI, class TO, int V, int GV>
static int gn_large_fwd(GnArgs a, hipStream_t s) {
  gn_split(a, V, GN_TARGET);
  const int rc = gn_stats<TI, V>(a, s);
  if (rc) return rc;
  NNZ_LAUNCH(gn_stats_finish_kernel, gn_grid(a.N * a.G), dim3(64), 0, s, a);
  NNZ_LAUNCH_CHECK();
  gn_split(a, V, GN_TARGET_APPLY);
  NNZ_LAUNCH((gn_apply_kernel<TI, TO, V, GV>), gn_grid(a.N * a.nblk), dim3(GN_NT), 0, s, a);
  NNZ_LAUNCH_CHECK();
  return NNZ_OK;
}
template <class TI, class TO, int V, int GV>
static int gn_large_bwd(GnArgs a, hipStream_t s) {
  static DynLdsCache cache;
  gn_split(a, V, GN_TARGET);
  const int lds = (GN_NT * V + a.C) * 2 * 4;
  hipError_t e = ensure_dyn_lds((const void*)gn_bwd_reduce_kernel<TI, TO, V, GV>, lds, cache);
  if (e != hipSuccess) return (int)e;
  NNZ_LAUNCH((gn_bwd_reduce_kernel<TI, TO, V, GV>), gn_grid(a.N * a.nblk), dim3(GN_NT), lds, s, a);
  NNZ_LAUNCH_CHECK();
  const long pairs4 = (a.N * a.G + 3) / 4, pair_wgs = pairs4 < GN_MAX_WG ? pairs4 : GN_MAX_WG;
  NNZ_LAUNCH(gn_bwd_finish_kernel, dim3((unsigned)(pair_wgs + (a.C + GN_FC - 1) / GN_FC)), dim3(GN_NT), 0, s, a, pair_wgs);
  NNZ_LAUNCH_CHECK();
  if (!a.out) return NNZ_OK;
  gn_split(a, V, GN_TARGET_APPLY);
  NNZ_LAUNCH((gn_bwd_apply_kernel<TI, TO, V, GV>), gn_grid(a.N * a.nblk), dim3(GN_NT), 0, s, a);
  NNZ_LAUNCH_CHECK();
  return NNZ_OK;
}
template <class TI, class TO, int V>
static int gn_run_small(const GnArgs& a, bool bwd, hipStream_t s) {
  const bool wave = gn_by_wave(a.N, a.S, a.G, a.q);
  constexpr int TEAMS = GN_SNT / 64;
  if (!bwd) {
    const long pairs = a.N * a.G;
    if (wave) NNZ_LAUNCH((gn_small_fwd_kernel<TI, TO, V, 64>), gn_grid((pairs + TEAMS - 1) / TEAMS), dim3(GN_SNT), 0, s, a);
    else NNZ_LAUNCH((gn_small_fwd_kernel<TI, TO, V, GN_SNT>), gn_grid(pairs), dim3(GN_SNT), 0, s, a);
    NNZ_LAUNCH_CHECK();
    return NNZ_OK;
  }
  const int K = gn_teams(a.N, a.S, a.G, a.q);
  const long teams = (long)K * a.G;   // at most 8 192, or G
  if (wave) NNZ_LAUNCH((gn_small_bwd_kernel<TI, TO, V, 64>), dim3((unsigned)((teams + TEAMS - 1) / TEAMS)), dim3(GN_SNT), 0, s, a, K);
  else NNZ_LAUNCH((gn_small_bwd_kernel<TI, TO, V, GN_SNT>), dim3((unsigned)teams), dim3(GN_SNT), 0, s, a, K);
  NNZ_LAUNCH_CHECK();
  if (K > 1 && (a.dw || a.db)) {
    GnArgs f = a;   // K rows of partial sums, no pairs to finish
    f.N = K;
    f.nblk = 1;
    NNZ_LAUNCH(gn_bwd_finish_kernel, dim3((a.C + GN_FC - 1) / GN_FC), dim3(GN_NT), 0, s, f, 0L);
    NNZ_LAUNCH_CHECK();
  }
  return NNZ_OK;
}
template <class TI, class TO, int V>
static int gn_run(const GnArgs& a, bool bwd, hipStream_t s) {
  if (gn_small(a.N, a.S, a.G, a.q)) {
    // a vector lies within a group or is one element
    if (V > 1 && a.q % V != 0) return gn_run_small<TI, TO, 1>(a, bwd, s);
    return gn_run_small<TI, TO, V>(a, bwd, s);
  }
  // a vector's channels in one group, in two, or anyhow
  if (a.q % V == 0) return bwd ? gn_large_bwd<TI, TO, V, 1>(a, s) : gn_large_fwd<TI, TO, V, 1>(a, s);
  if constexpr (V > 2)
    if (2 * a.q == V) return bwd ? gn_large_bwd<TI, TO, V, 2>(a, s) : gn_large_fwd<TI, TO, V, 2>(a, s);
  return bwd ? gn_large_bwd<TI, TO, V, V>(a, s) : gn_large_fwd<TI, TO, V, V>(a, s);
}

// V: the widest of 16 bytes, 4 elements and 1 that the channel count, the strides and the pointers allow
template <class TI, class TO>
static int gn_dispatch(const GnArgs& a, bool bwd, hipStream_t s) {
  auto fits = [&](int v) {
    const uintptr_t ai = (v * sizeof(TI) < 16 ? v * sizeof(TI) : 16) - 1, ao = (v * sizeof(TO) < 16 ? v * sizeof(TO) : 16) - 1;
    const uintptr_t out = (uintptr_t)a.out & (bwd ? ai : ao), dy = bwd ? ((uintptr_t)a.dy & ao) : 0;
    return a.C % v == 0 && a.xs % v == 0 && a.xb % v == 0 && ((uintptr_t)a.x & ai) == 0 && out == 0 && dy == 0;
  };
  constexpr int FULL = 16 / (int)sizeof(TI);
  if (fits(FULL)) return gn_run<TI, TO, FULL>(a, bwd, s);
  if (FULL != 4 && fits(4)) return gn_run<TI, TO, 4>(a, bwd, s);
  return gn_run<TI, TO, 1>(a, bwd, s);
}
static int gn_go(const GnArgs& a, int ti, int to, bool bwd, hipStream_t s) {
  if (ti == ELEM_F32 && to == ELEM_F32) return gn_dispatch<float, float>(a, bwd, s);
  if (ti == ELEM_F16 && to == ELEM_F16) return gn_dispatch<f16, f16>(a, bwd, s);
  if (ti == ELEM_F16 && to == ELEM_F32) return gn_dispatch<f16, float>(a, bwd, s);
  if (ti == ELEM_BF16 && to == ELEM_BF16) return gn_dispatch<bf16, bf16>(a, bwd, s);
  if (ti == ELEM_BF16 && to == ELEM_F32) return gn_dispatch<bf16, float>(a, bwd, s);
  return NNZ_EINVAL;
}
static bool gn_shape_ok(long N, long S, int C, int G) {
  return N >= 1 && S >= 1 && C >= 1 && C <= GN_MAX_C && G >= 1 && C % G == 0 && N <= (1L << 40) / C && S <= (1L << 40) / C / N;
}

}  // namespace nnz

extern "C" long nnz_group_norm_act_workspace_bytes(long N, long S, int C, int G, int backward) {
  using namespace nnz;
  if (!gn_shape_ok(N, S, C, G)) return NNZ_EINVAL;
  return gn_ws(N, S, C, G, backward != 0).bytes;
}

extern "C" int nnz_group_norm_act_forward(const void* x, int x_type, long x_batch_stride, long x_row_stride, const float* weight,
                                          const float* bias, void* y, int y_type, float* stats, void* workspace,
                                          long workspace_bytes, long N, long S, int C, int G, float eps, int act, float slope,
                                          void* stream) {
  using namespace nnz;
  if (!x || !y || !stats || !gn_shape_ok(N, S, C, G) || act < GN_NONE || act > GN_SILU) return NNZ_EINVAL;
  const GnWs w = gn_ws(N, S, C, G, false);
  if (w.bytes && (!workspace || workspace_bytes < w.bytes)) return NNZ_EINVAL;
  GnArgs a = {};
  a.x = x; a.w = weight; a.b = bias; a.out = y; a.stats = stats; a.gpart = (double*)workspace;
  a.N = N; a.S = S; a.xb = x_batch_stride; a.xs = x_row_stride; a.C = C; a.G = G; a.q = C / G;
  a.act = act; a.slope = slope; a.eps = eps;
  return gn_go(a, x_type, y_type, false, (hipStream_t)stream);
}

extern "C" int nnz_group_norm_act_backward(const void* x, int x_type, long x_batch_stride, long x_row_stride, const void* dy,
                                           int dy_type, const float* weight, const float* bias, const float* stats, void* dx,
                                           float* dweight, float* dbias, void* workspace, long workspace_bytes, long N, long S,
                                           int C, int G, int act, float slope, void* stream) {
  using namespace nnz;
  if (!x || !dy || !(dx || dweight || dbias) || !stats || !gn_shape_ok(N, S, C, G) || act < GN_NONE || act > GN_SILU) return NNZ_EINVAL;
  const GnWs w = gn_ws(N, S, C, G, true);
  if (w.bytes && (!workspace || workspace_bytes < w.bytes)) return NNZ_EINVAL;
  GnArgs a = {};
  a.x = x; a.dy = dy; a.w = weight; a.b = bias; a.out = dx; a.stats = (float*)stats;
  if (w.bytes) {
    a.gpart = (double*)workspace; a.cpart = (float*)((char*)workspace + w.cpart); a.cc = (float*)((char*)workspace + w.cc);
  }
  a.dw = dweight; a.db = dbias;
  a.N = N; a.S = S; a.xb = x_batch_stride; a.xs = x_row_stride; a.C = C; a.G = G; a.q = C / G;
  a.act = act; a.slope = slope;
  return gn_go(a, x_type, dy_type, true, (hipStream_t)stream);
}
