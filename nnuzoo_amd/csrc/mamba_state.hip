// The state-carrying operators of a Mamba block (gfx950), token-major, for prompts and for single tokens:
//   short causal convolution   y_t = act(bias + sum_j w_j x_{t-W+1+j}); inputs before the first come from conv_state (the last W
//                              inputs of the sequence), which is brought up to date in place;
//   selective scan             D_t = [softplus](dt_t + dt_bias);  h_t = exp(D_t A) h_{t-1} + D_t x_t B_t;
//                              y_t = <C_t, h_t> + D x_t, times silu(z_t);  h starts from `state` and is left there.
// Rows are (B, L, D) with the channels innermost, as the projections around them write and read them: nothing is transposed.
// Every sequence has its own length; nothing behind it is read, its outputs are 0, and a sequence of length 0 keeps its states.
// Sums and states are fp32 whatever the activations' type.
#include "elem_io.hpp"

#include <type_traits>

namespace nnz {

// ---------------------------------------------------------------------------------------------------------------
// causal convolution
// ---------------------------------------------------------------------------------------------------------------
struct ConvStateArgs {
  const void* x;       // [B][L][D], strides xb, xt, 1 (token form: xt unused)
  const float* w;      // [D][W]
  const float* bias;   // [D] or null
  void* y;             // [B][L][D] contiguous
  void* st;            // [B][D][W], strides sb, sd, sw, or null (zeros before the first token, nothing kept)
  const void* len;     // [B] int32 / int64, or null (all L); token form: [B] bool, or null (all active)
  long xb, xt, sb, sd, sw;
  int B, L, D, silu, len64, st_type;
  int tt;              // tokens of a thread
};

__device__ __forceinline__ int seq_len(const void* len, int len64, int b, int L) {
  if (!len) return L;
  const long v = len64 ? ((const long long*)len)[b] : (long)((const int*)len)[b];
  return v < 0 ? 0 : v > L ? L : (int)v;
}

// V elements of a row as they were loaded
template <class T, int V>
struct RowVec {
  ElemVec<T, V> r;
  __device__ __forceinline__ void load(const T* p) { r = *reinterpret_cast<const ElemVec<T, V>*>(p); }
  __device__ __forceinline__ float get(int v) const { return (float)r[v]; }
};
template <class T>
struct RowVec<T, 1> {
  T r;
  __device__ __forceinline__ void load(const T* p) { r = *p; }
  __device__ __forceinline__ float get(int) const { return (float)r; }
};

// A thread: V adjacent channels, tt consecutive tokens, the window in registers.  Bound by HBM (x in, y out); a load in front of every
// token's stores waited for those as well; with loads U tokens ahead 51 us = 3.9 TB/s at 2 x 262144 x 96 f16, W = 4, where x is one
// half of rows of 384 bytes, so that a third of every second line fetched is not x.
template <class T, int W, int V>
__global__ __launch_bounds__(256) void conv_prompt_kernel(ConvStateArgs a) {
  const int CV = a.D / V;
  const int chunks = (a.L + a.tt - 1) / a.tt;
  const unsigned id = blockIdx.x * 256 + threadIdx.x;   // a launch has less than 2^32 threads
  if (id >= (unsigned long)CV * chunks * a.B) return;
  const unsigned rest = id / CV;
  const int d = (int)(id - rest * CV) * V;
  const int b = (int)(rest / chunks), t0 = (int)(rest - (unsigned)b * chunks) * a.tt;
  const int len = seq_len(a.len, a.len64, b, a.L);
  const int t1 = t0 + a.tt < a.L ? t0 + a.tt : a.L;
  const T* x = (const T*)a.x + (long)b * a.xb + d;
  T* y = (T*)a.y + ((long)b * a.L) * a.D + d;
  constexpr int U = 4;           // tokens whose loads are in flight while the U before them are computed
  float w[V][W], bias[V], win[W - 1 + U][V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    bias[v] = a.bias ? a.bias[d + v] : 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) w[v][j] = a.w[(long)(d + v) * W + j];
  }
  // the W - 1 inputs before t0; inputs before the sequence: the state's last columns
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const int t = t0 - (W - 1) + j;
    if (t >= 0) {
      if (t < len) ld_elems<T, V>(x + (long)t * a.xt, win[j]);
      else {
#pragma unroll
        for (int v = 0; v < V; ++v) win[j][v] = 0.f;
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
        win[j][v] = a.st ? ld_any(a.st, b * a.sb + (long)(d + v) * a.sd + (long)(W + t) * a.sw, a.st_type) : 0.f;
    }
  }
  // the first chunk's thread alone touches the state: it has read its history above (the new state may keep part of it)
  if (a.st && t0 == 0 && len > 0) {
    float keep[W][V];   // the new state's columns
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const int t = len - W + k;
      if (t >= 0) ld_elems<T, V>(x + (long)t * a.xt, keep[k]);
      else {
#pragma unroll
        for (int v = 0; v < V; ++v) keep[k][v] = ld_any(a.st, b * a.sb + (long)(d + v) * a.sd + (long)(W + t) * a.sw, a.st_type);
      }
    }
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) st_any(a.st, b * a.sb + (long)(d + v) * a.sd + k * a.sw, a.st_type, keep[k][v]);
  }
  const int te = t1 < len ? t1 : len;
  RowVec<T, V> next[U];
  const T* xn = x + (long)t0 * a.xt;
  auto fetch = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t + u < te) next[u].load(xn + u * a.xt);
    xn += U * a.xt;
  };
  fetch(t0);
  T* yt = y + (long)t0 * a.D;
  for (int t = t0; t < te; t += U) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int v = 0; v < V; ++v) win[W - 1 + u][v] = next[u].get(v);
    fetch(t + U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float o[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float s = bias[v];
#pragma unroll
        for (int j = 0; j < W; ++j) s = fmaf(w[v][j], win[u + j][v], s);
        o[v] = a.silu ? s * sigmoid_hw(s) : s;
      }
      if (t + u < te) st_elems<T, V>(yt + (long)u * a.D, o);
    }
    yt += (long)U * a.D;
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) win[j][v] = win[U + j][v];
  }
  const float zero[V] = {};
  for (int t = te > t0 ? te : t0; t < t1; ++t) st_elems<T, V>(y + (long)t * a.D, zero);
}

// One token: a thread per (sequence, channel); 3 us, the smallest launch's time, at the sizes of a decoder's step.
template <class T, int W>
__global__ __launch_bounds__(256) void conv_token_kernel(ConvStateArgs a) {
  const unsigned id = blockIdx.x * 256 + threadIdx.x;   // B * D < 2^32
  if (id >= (unsigned long)a.B * a.D) return;
  const unsigned b = id / (unsigned)a.D;
  const int d = (int)(id - b * a.D);
  T* y = (T*)a.y;
  if (a.len && !((const unsigned char*)a.len)[b]) {
    y[id] = (T)0.f;
    return;
  }
  const long s0 = b * a.sb + d * a.sd;
  float win[W];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) win[j] = ld_any(a.st, s0 + (j + 1) * a.sw, a.st_type);
  win[W - 1] = (float)((const T*)a.x)[b * a.xb + d];
  float s = a.bias ? a.bias[d] : 0.f;
#pragma unroll
  for (int j = 0; j < W; ++j) s = fmaf(a.w[(long)d * W + j], win[j], s);
  y[id] = (T)(a.silu ? s * sigmoid_hw(s) : s);
#pragma unroll
  for (int j = 0; j < W; ++j) st_any(a.st, s0 + j * a.sw, a.st_type, win[j]);
}

template <class T, int W>
static int conv_state_run(ConvStateArgs a, bool token, hipStream_t s) {
  if (token) {
    const long wg = ((long)a.B * a.D + 255) / 256;
    NNZ_LAUNCH((conv_token_kernel<T, W>), dim3((unsigned)wg), dim3(256), 0, s, a);
    NNZ_LAUNCH_CHECK();
    return NNZ_OK;
  }
  constexpr int FULL = 4;   // 8 f16 a thread: 178 registers at W = 4 instead of 100, 57 us instead of 51 at 2 x 262144 x 96
  const bool vec = a.D % FULL == 0 && a.xb % FULL == 0 && a.xt % FULL == 0 &&
                   (((uintptr_t)a.x | (uintptr_t)a.y) & (FULL * sizeof(T) - 1)) == 0;
  const int CV = vec ? a.D / FULL : a.D;
  // a thread re-reads W - 1 tokens (from L2): 16 tokens each once that leaves enough threads, 8 on short inputs and no fewer: only
  // a sequence's first chunk may need the state, for its thread writes the new one (8 >= W - 1)
  a.tt = (long)CV * a.B * ((a.L + 15) / 16) < 256L * 512 ? 8 : 16;
  const long wg = ((long)CV * a.B * ((a.L + a.tt - 1) / a.tt) + 255) / 256;
  if (wg >= 1L << 24) return NNZ_EINVAL;   // 2^32 threads
  if (vec) NNZ_LAUNCH((conv_prompt_kernel<T, W, FULL>), dim3((unsigned)wg), dim3(256), 0, s, a);
  else NNZ_LAUNCH((conv_prompt_kernel<T, W, 1>), dim3((unsigned)wg), dim3(256), 0, s, a);
  NNZ_LAUNCH_CHECK();
  return NNZ_OK;
}
template <class T>
static int conv_state_width(const ConvStateArgs& a, int W, bool token, hipStream_t s) {
  switch (W) {
    case 1: return conv_state_run<T, 1>(a, token, s);
    case 2: return conv_state_run<T, 2>(a, token, s);
    case 3: return conv_state_run<T, 3>(a, token, s);
    case 4: return conv_state_run<T, 4>(a, token, s);
    case 5: return conv_state_run<T, 5>(a, token, s);
    case 6: return conv_state_run<T, 6>(a, token, s);
    case 7: return conv_state_run<T, 7>(a, token, s);
    case 8: return conv_state_run<T, 8>(a, token, s);
  }
  return NNZ_EINVAL;
}
static int conv_state_go(const ConvStateArgs& a, int type, int W, bool token, hipStream_t s) {
  if (type == ELEM_F32) return conv_state_width<float>(a, W, token, s);
  if (type == ELEM_F16) return conv_state_width<f16>(a, W, token, s);
  if (type == ELEM_BF16) return conv_state_width<bf16>(a, W, token, s);
  return NNZ_EINVAL;
}

// ---------------------------------------------------------------------------------------------------------------
// selective scan
// ---------------------------------------------------------------------------------------------------------------
struct ScanStateArgs {
  const void* x;         // [B][L][D], strides xb, xt, 1
  const void* dt;        // [B][L][H], strides db, dt_t, 1
  const void* Bm;        // [B][L][G][N], strides bb, bt, bg, 1
  const void* Cm;        // strides cb, ct, cg, 1
  const void* z;         // [B][L][D], strides zb, zt, 1, or null
  const float* A;        // [H][N] (a_n = 1) or [H] (a_n = 0); with a_log its entries are log(-A)
  const float* Dv;       // [H] or null
  const float* dt_bias;  // [H] or null
  float* state;          // [B][D][N], batch stride sb, rows contiguous; or null (zeros, nothing kept)
  void* y;               // [B][L][D] contiguous
  const void* len;       // as above
  float* part_h;         // [chunks][B][D][N]: end state of chunk c from a zero entry, then (scan_join_kernel) the true entry state of
                         // c; without that kernel the last slot, whose summary nobody needs, keeps the sequence's entry state
  float* part_d;         // [chunks][B][D]: sum of D_t over chunk c
  long xb, xt, db, dtt, bb, bt, bg, cb, ct, cg, zb, zt, sb;
  int B, L, D, H, G, softplus, len64, a_n, a_log;
  int rep;               // channels of a head
  int dg;                // channels of a group
  int nch, wpg;          // channels of a workgroup, workgroups of a group
  int cl, chunks, joined;  // tokens of a chunk; joined: scan_join_kernel runs between MODE 1 and MODE 2
  int pair, pair_dt;     // x and z / dt: two adjacent channels are one aligned access
};

// e^x with the rounding of x * log2(e) put right
__device__ __forceinline__ float exp_fine(float x) {
  const float p = x * 1.4426950408889634f;
  const float r = fmaf(x, 1.9259629911266175e-8f, fmaf(x, 1.4426950408889634f, -p));
  const float e = __builtin_amdgcn_exp2f(p);
  return fmaf(e * 0.6931471805599453f, r, e);
}
// softplus(x) = max(x, 0) + log(1 + e), e = exp(-|x|) <= 1; w = 1 + e is rounded, and what the rounding lost is added to log w
// (v_log_f32 keeps 1 ulp of its result down to w = 1 + 2^-23): relative accuracy for small e, too - a time step is often softplus of
// -5, and the states' decay takes its relative error.  e is 0 beyond -110.
__device__ __forceinline__ float softplus_hw(float x) {
  const float e = exp_fine(-fminf(fabsf(x), 110.f));
  const float w = 1.f + e;
  const float l = fmaf(__builtin_amdgcn_logf(w), 0.6931471805599453f, e - (w - 1.f));
  return l + (x < 0.f ? 0.f : x);   // NaN stays
}

constexpr float LOG2E = 1.4426950408889634f;
// decays of NS states from n on, in units of log 2; an infinite one becomes huge, so that a padding token's D_t = 0 leaves the state
// alone.  All are loaded before the first is used.
template <int N, int NS>
__device__ __forceinline__ void load_decays(const ScanStateArgs& a, int head, int n, float (&A2)[NS]) {
  const float* p = a.a_n ? a.A + (long)head * N + n : a.A + head;
#pragma unroll
  for (int i = 0; i < NS; ++i) A2[i] = p[i * a.a_n];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    // exp_fine takes no infinity (its rounding of x log2 e would be inf - inf); exp(-110) is 0; NaN stays
    if (a.a_log) A2[i] = -exp_fine(A2[i] > 88.f ? 88.f : A2[i] < -110.f ? -110.f : A2[i]);
    const float v = A2[i] * LOG2E;
    A2[i] = v < -3.0e38f ? -3.0e38f : v;
  }
}
// sum over the 4 lanes of a channel (quad_perm: no LDS, unlike a shuffle)
__device__ __forceinline__ float quad_sum(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
  return v;
}
template <class T>
__device__ __forceinline__ ElemVec<T, 2> ld_pair(const T* p, bool aligned, int second) {
  if (aligned) return *reinterpret_cast<const ElemVec<T, 2>*>(p);
  return ElemVec<T, 2>{p[0], p[second]};
}

// 4 lanes share CPL channels and hold N / 4 states of each; a workgroup has nch = 16 CPL channels a wave of one group and walks
// its tokens in tiles: every (token, channel) of a tile is loaded and turned into D_t, D_t x_t once, B and C are widened once, all
// through LDS.  Bound by the vector unit: per token, channel and state a 2^x (quarter rate), two products and two FMAs - 32 cycles a
// wave of 64 states, 165 us for one pass at 2 x 262144 x 96, N = 16; measured there (f16): summaries 200 us, joining 21, outputs 270.
// MODE 0: whole sequences in one launch.  Long sequences of few channels are cut into chunks that run in parallel: MODE 1 leaves
// every chunk's summary (end state from a zero entry, sum of D_t: a chunk multiplies its entry state by exp(A sum D)), and MODE 2 runs
// the chunks from the entry states that the summaries in front of them make: each workgroup joins up to SC_JOIN - 1 of them by
// itself, scan_join_kernel more.
constexpr int SC_TT = 16;   // tokens of a tile
// chunks from which on a kernel of its own joins them.  Us a call with it / without, chunks of 64 tokens, fp32, 16 states: 4 x 768 channels,
// 16 chunks 65 / 41, 31: 90 / 76, 40: 105 / 98, 64: 145 / 158; 8 x 1024 channels, 31 chunks (as many as they get): 213 / 162; 1 x 512, 16:
// 27 / 25, 40: 34 / 34, 64: 37 / 46.  Only few channels would want it earlier: 2 x 96, 16: 24 / 26, 31: 25 / 33
constexpr int SC_JOIN = 32;

template <class T, int N, int CPL, int MODE>
__global__ __launch_bounds__(256) void scan_prompt_kernel(ScanStateArgs a) {
  constexpr int NS = N / 4;
  constexpr int IT = SC_TT * CPL / 8;    // token rows of a thread in the staging passes
  constexpr int ROWS = SC_TT / IT;       // their distance: NT / (nch / 2)
  extern __shared__ __attribute__((aligned(16))) float sc_lds[];
  const int nch = a.nch, np = nch / 2;
  float4* s_du = reinterpret_cast<float4*>(sc_lds);     // [SC_TT][nch / 2]: {D, D x} of two channels
  float* s_b = sc_lds + SC_TT * nch * 2;                // [SC_TT][N]
  float* s_c = s_b + SC_TT * N;                         // [SC_TT][N], not in MODE 1
  float* s_y = s_c + SC_TT * N;                         // [SC_TT][nch], not in MODE 1
  const int tid = threadIdx.x, NT = blockDim.x;
  const int g = blockIdx.x / a.wpg;
  const int ch0 = (blockIdx.x - g * a.wpg) * nch;       // within the group
  const int chunk = blockIdx.y, b = blockIdx.z;
  const int len = seq_len(a.len, a.len64, b, a.L);
  const int t0 = chunk * a.cl;
  const int tend = t0 + a.cl < a.L ? t0 + a.cl : a.L;
  const int te = tend < len ? tend : len;
  // staging role: two adjacent channels, tokens st + ROWS * i
  const int st = tid / np, sp = tid - st * np;
  const int sc0 = ch0 + 2 * sp;
  const bool on0 = sc0 < a.dg, on1 = sc0 + 1 < a.dg;
  const int sd = g * a.dg + (on0 ? sc0 : a.dg - 1), sd1 = on1 ? 1 : 0;
  const int hd = sd / a.rep, hd1 = (sd + sd1) / a.rep - hd;
  const bool pair = a.pair && on1, pair_dt = a.pair_dt && on1;
  const float bias0 = a.dt_bias ? a.dt_bias[hd] : 0.f, bias1 = a.dt_bias ? a.dt_bias[hd + hd1] : 0.f;
  const float D0 = a.Dv ? a.Dv[hd] : 0.f, D1 = a.Dv ? a.Dv[hd + hd1] : 0.f;
  // state role
  const int sub = tid & 3, mc = (tid >> 2) * CPL;       // the quad's first channel, within the workgroup
  float A2[CPL][NS], h[CPL][NS];
  long prow[CPL], srow[CPL];
  bool m_on[CPL];
#pragma unroll
  for (int q = 0; q < CPL; ++q) {
    m_on[q] = ch0 + mc + q < a.dg;
    const int md = g * a.dg + (m_on[q] ? ch0 + mc + q : a.dg - 1), mh = md / a.rep;
    srow[q] = (long)b * a.sb + (long)md * N + sub * NS;
    prow[q] = (((long)chunk * a.B + b) * a.D + md) * N + sub * NS;
    load_decays<N, NS>(a, mh, sub * NS, A2[q]);
#pragma unroll
    for (int n = 0; n < NS; ++n) h[q][n] = MODE == 0 && a.state ? a.state[srow[q] + n] : 0.f;
    // MODE 2 never reads `state`: the workgroup of the last token may have written it already
    if (MODE == 2 && t0 < te) {
      const long step = (long)a.B * a.D * N;
      const float* own = a.part_h + prow[q];
      const float* first = a.joined ? own : own + (a.chunks - 1 - chunk) * step;
#pragma unroll
      for (int n = 0; n < NS; ++n) h[q][n] = first[n];
      if (!a.joined) {
        const float* p = own - chunk * step;
        const float* pd = a.part_d + (long)b * a.D + md;
#pragma unroll 4
        for (int c = 0; c < chunk; ++c) {
          const float sum = pd[(long)c * a.B * a.D];
#pragma unroll
          for (int n = 0; n < NS; ++n) h[q][n] = fmaf(__builtin_amdgcn_exp2f(sum * A2[q][n]), h[q][n], p[c * step + n]);
        }
      }
    }
    if (MODE == 1 && !a.joined && chunk == 0 && m_on[q]) {
      float* keep = a.part_h + prow[q] + (long)(a.chunks - 1) * a.B * a.D * N;
#pragma unroll
      for (int n = 0; n < NS; ++n) keep[n] = a.state ? a.state[srow[q] + n] : 0.f;
    }
  }
  float dsum[CPL] = {};
  // every access walks its rows by a constant step
  const T* xp = (const T*)a.x + (long)b * a.xb + (long)(t0 + st) * a.xt + sd;
  const T* zp = (const T*)a.z + (a.z ? (long)b * a.zb + (long)(t0 + st) * a.zt + sd : 0);
  const T* dp = (const T*)a.dt + (long)b * a.db + (long)(t0 + st) * a.dtt + hd;
  T* yp = (T*)a.y + ((long)b * a.L + t0 + st) * a.D + sd;
  const int bn = tid % N, b0 = tid / N, brows = NT / N;   // N <= 32 divides NT
  const T* bp = (const T*)a.Bm + (long)b * a.bb + g * a.bg + (long)(t0 + b0) * a.bt + bn;
  const T* cp = (const T*)a.Cm + (long)b * a.cb + g * a.cg + (long)(t0 + b0) * a.ct + bn;
  const long xs = ROWS * a.xt, zs = ROWS * a.zt, dls = ROWS * a.dtt, ys = (long)ROWS * a.D;
  // a tile's loads are issued before the tile in front of it is computed
  constexpr int BI = SC_TT * N / 64;
  typedef ElemVec<T, 2> Pair;
  Pair xr[IT], zr[IT], dr[IT];
  T br[BI], cr[BI];
  const Pair none = {(T)0.f, (T)0.f};
  auto fetch_rows = [&](int tile, auto whole) __attribute__((always_inline)) {
    constexpr bool W = decltype(whole)::value;   // all rows of the tile exist
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const bool in = W || tile + st + ROWS * i < te;
      xr[i] = in ? ld_pair<T>(xp, pair, sd1) : none;
      dr[i] = in ? ld_pair<T>(dp, pair_dt, hd1) : none;
      if (MODE != 1) zr[i] = in && a.z ? ld_pair<T>(zp, pair, sd1) : none;
      xp += xs;
      dp += dls;
      if (MODE != 1) zp += zs;
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
      const int tt = b0 + i * brows;
      const bool in = tt < SC_TT && (W || tile + tt < te);
      br[i] = in ? bp[(long)i * brows * a.bt] : (T)0.f;
      if (MODE != 1) cr[i] = in ? cp[(long)i * brows * a.ct] : (T)0.f;
    }
    bp += SC_TT * a.bt;
    cp += SC_TT * a.ct;
  };
  auto fetch = [&](int tile) __attribute__((always_inline)) {
    if (tile + SC_TT <= te) fetch_rows(tile, std::true_type{});
    else fetch_rows(tile, std::false_type{});
  };
  if (t0 < te) fetch(t0);
  for (int tile = t0; tile < te; tile += SC_TT) {
    float2 xv[IT], zv[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      xv[i] = make_float2((float)xr[i][0], (float)xr[i][1]);
      if (MODE != 1) zv[i] = make_float2((float)zr[i][0], (float)zr[i][1]);
      float dl0 = (float)dr[i][0] + bias0, dl1 = (float)dr[i][1] + bias1;
      if (a.softplus) {
        dl0 = softplus_hw(dl0);
        dl1 = softplus_hw(dl1);
      }
      if (tile + st + ROWS * i >= te) dl0 = dl1 = 0.f;
      s_du[(st + ROWS * i) * np + sp] = make_float4(dl0, dl0 * xv[i].x, dl1, dl1 * xv[i].y);
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
      const int tt = b0 + i * brows;
      if (tt < SC_TT) {
        s_b[tt * N + bn] = (float)br[i];
        if (MODE != 1) s_c[tt * N + bn] = (float)cr[i];
      }
    }
    if (tile + SC_TT < te) fetch(tile + SC_TT);
    __syncthreads();
    const int cnt = te - tile < SC_TT ? te - tile : SC_TT;
    // 4 tokens at a time; a tile's tokens behind the end have D = 0 and change nothing
    for (int tt = 0; tt < cnt; tt += 4) {
      float yv[CPL];
      if constexpr (CPL == 1) {
        // few waves: 4 tokens' reads and decays before their recurrence, so that the latencies overlap
        float d[4], u[4], bv[4][NS], cv[4][NS], e[4][NS];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 v = reinterpret_cast<const float2*>(s_du)[(tt + k) * nch + mc];
          d[k] = v.x;
          u[k] = v.y;
          ld_elems<float, NS>(s_b + (tt + k) * N + sub * NS, bv[k]);
          if (MODE != 1) ld_elems<float, NS>(s_c + (tt + k) * N + sub * NS, cv[k]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int n = 0; n < NS; ++n) e[k][n] = __builtin_amdgcn_exp2f(d[k] * A2[0][n]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float acc = 0.f;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            h[0][n] = fmaf(e[k][n], h[0][n], u[k] * bv[k][n]);
            if (MODE != 1) acc = n ? fmaf(h[0][n], cv[k][n], acc) : h[0][n] * cv[k][n];
          }
          if (MODE == 1) dsum[0] += d[k];
          else {
            acc = quad_sum(acc);
            yv[0] = k == 0 || sub == k ? acc : yv[0];   // lane k of the quad keeps token k
          }
        }
      } else {
        // many waves hide the latencies, and registers count
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 v = s_du[(tt + k) * np + (mc >> 1)];
          const float d[2] = {v.x, v.z}, u[2] = {v.y, v.w};
          float bv[NS], cv[NS];
          ld_elems<float, NS>(s_b + (tt + k) * N + sub * NS, bv);
          if (MODE != 1) ld_elems<float, NS>(s_c + (tt + k) * N + sub * NS, cv);
#pragma unroll
          for (int q = 0; q < CPL; ++q) {
            float acc = 0.f;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
              h[q][n] = fmaf(__builtin_amdgcn_exp2f(d[q] * A2[q][n]), h[q][n], u[q] * bv[n]);
              if (MODE != 1) acc = n ? fmaf(h[q][n], cv[n], acc) : h[q][n] * cv[n];
            }
            if (MODE == 1) dsum[q] += d[q];
            else {
              acc = quad_sum(acc);
              yv[q] = k == 0 || sub == k ? acc : yv[q];
            }
          }
        }
      }
      if (MODE != 1) {
        if constexpr (CPL == 2) *reinterpret_cast<float2*>(s_y + (tt + sub) * nch + mc) = make_float2(yv[0], yv[1]);
        else s_y[(tt + sub) * nch + mc] = yv[0];
      }
    }
    __syncthreads();
    if (MODE != 1) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int tt = st + ROWS * i, t = tile + tt;
        if (t < te && on0) {
          const float2 yy = *reinterpret_cast<const float2*>(s_y + tt * nch + 2 * sp);
          float v0 = yy.x, v1 = yy.y;
          if (a.Dv) {
            v0 = fmaf(D0, xv[i].x, v0);
            v1 = fmaf(D1, xv[i].y, v1);
          }
          if (a.z) {
            v0 *= zv[i].x * sigmoid_hw(zv[i].x);
            v1 *= zv[i].y * sigmoid_hw(zv[i].y);
          }
          T* o = yp + i * ys;
          if (pair) {
            ElemVec<T, 2> r;
            r[0] = (T)v0;
            r[1] = (T)v1;
            *reinterpret_cast<ElemVec<T, 2>*>(o) = r;
          } else {
            o[0] = (T)v0;
            if (on1) o[1] = (T)v1;
          }
        }
      }
      yp += IT * ys;
    }
  }
  if (MODE == 1) {
#pragma unroll
    for (int q = 0; q < CPL; ++q)
      if (m_on[q]) {
#pragma unroll
        for (int n = 0; n < NS; ++n) a.part_h[prow[q] + n] = h[q][n];
        if (sub == 0) a.part_d[prow[q] / N] = dsum[q];
      }
    return;
  }
  if (on0) {
    T* y0 = (T*)a.y + (long)b * a.L * a.D + sd;
    for (int t = (te > t0 ? te : t0) + st; t < tend; t += ROWS) {
      y0[(long)t * a.D] = (T)0.f;
      if (on1) y0[(long)t * a.D + 1] = (T)0.f;
    }
  }
  // the chunk that holds the last token leaves the state (MODE 2 reads the copies that scan_join_kernel or MODE 1's first chunk made)
  if (a.state && len > t0 && len <= tend) {
#pragma unroll
    for (int q = 0; q < CPL; ++q)
      if (m_on[q]) {
#pragma unroll
        for (int n = 0; n < NS; ++n) a.state[srow[q] + n] = h[q][n];
      }
  }
}

// chunk summaries -> entry states, in place: E_0 = state, E_{c+1} = exp(A sum_c) E_c + S_c.  SEG threads a (channel, state) share the
// chunks: each joins its own run, then starts again from the runs before it (1 261 chunks of 2 x 96 x 16 states: 21 us with 64
// runs, 26 us with 16).
template <int N, int LN, int SEG>
__global__ __launch_bounds__(LN * SEG) void scan_join_kernel(ScanStateArgs a) {
  __shared__ float s_p[SEG][LN], s_h[SEG][LN];
  const int lane = threadIdx.x % LN, seg = threadIdx.x / LN, b = blockIdx.y;
  const long dn = (long)a.D * N, i = (long)blockIdx.x * LN + lane;
  const long at = i < dn ? i : dn - 1;
  const int d = (int)(at / N), hd = d / a.rep;
  float A1[1];
  load_decays<N, 1>(a, hd, (int)(at % N), A1);
  const float A2 = A1[0];
  const int per = (a.chunks + SEG - 1) / SEG;
  const int c0 = seg * per, c1 = c0 + per < a.chunks ? c0 + per : a.chunks;
  float* ph = a.part_h + (long)b * dn + at;
  const float* pd = a.part_d + (long)b * a.D + d;
  const long hs = (long)a.B * dn, ds = (long)a.B * a.D;
  float e = a.state ? a.state[(long)b * a.sb + at] : 0.f;
  float p = 0.f, h = 0.f;
#pragma unroll 8
  for (int c = c0; c < c1; ++c) {
    const float sum = pd[c * ds];
    h = fmaf(__builtin_amdgcn_exp2f(sum * A2), h, ph[c * hs]);
    p += sum;
  }
  s_p[seg][lane] = p;
  s_h[seg][lane] = h;
  __syncthreads();
  for (int s = 0; s < seg; ++s) e = fmaf(__builtin_amdgcn_exp2f(s_p[s][lane] * A2), e, s_h[s][lane]);
  if (i >= dn) return;
#pragma unroll 8
  for (int c = c0; c < c1; ++c) {
    const float own = ph[c * hs], sum = pd[c * ds];
    ph[c * hs] = e;
    e = fmaf(__builtin_amdgcn_exp2f(sum * A2), e, own);
  }
}

// One token: 4 lanes a channel, each its N / 4 states in one access.  Bound by HBM (the states in and out): 128 x 1536 x 16: 9.1 us =
// 3 TB/s, of which 2.8 us is what the smallest launch takes (11.8 us with 64-bit indices and loads behind branches).
template <class T, int N>
__global__ __launch_bounds__(256) void scan_token_kernel(ScanStateArgs a) {
  constexpr int NS = N / 4;
  const unsigned id = (blockIdx.x * 256 + threadIdx.x) >> 2;   // 4 B * D < 2^32
  const int sub = threadIdx.x & 3;
  if (id >= (unsigned long)a.B * a.D) return;     // all 4 lanes of a channel leave together
  const unsigned b = id / (unsigned)a.D;
  const int d = (int)(id - b * a.D);
  T* y = (T*)a.y;
  if (a.len && !((const unsigned char*)a.len)[b]) {
    if (sub == 0) y[id] = (T)0.f;
    return;
  }
  const int head = d / a.rep, g = d / a.dg;
  float* st = a.state + (long)b * a.sb + (long)d * N + sub * NS;
  const T* bp = (const T*)a.Bm + (long)b * a.bb + g * a.bg + sub * NS;
  const T* cp = (const T*)a.Cm + (long)b * a.cb + g * a.cg + sub * NS;
  // all loads first, of absent inputs from a place that is there: neither stores nor branches stand between them
  const T* xp = (const T*)a.x + b * a.xb + d;
  const T* zp = a.z ? (const T*)a.z + b * a.zb + d : xp;
  const T xr = *xp, zr = *zp, dr = ((const T*)a.dt)[b * a.db + head];
  const float Dr = a.Dv ? a.Dv[head] : 0.f, br = a.dt_bias ? a.dt_bias[head] : 0.f;
  float h[NS], A2[NS];
  T bv[NS], cv[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) h[n] = st[n];
#pragma unroll
  for (int n = 0; n < NS; ++n) bv[n] = bp[n];
#pragma unroll
  for (int n = 0; n < NS; ++n) cv[n] = cp[n];
  load_decays<N, NS>(a, head, sub * NS, A2);
  const float x = (float)xr, z = (float)zr;
  float dl = (float)dr + br;
  if (a.softplus) dl = softplus_hw(dl);
  const float u = dl * x;
  float acc = 0.f;
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    h[n] = fmaf(__builtin_amdgcn_exp2f(dl * A2[n]), h[n], u * (float)bv[n]);
    acc = fmaf(h[n], (float)cv[n], acc);
  }
#pragma unroll
  for (int n = 0; n < NS; ++n) st[n] = h[n];
  acc = quad_sum(acc);
  if (sub == 0) {
    const float v = a.Dv ? fmaf(Dr, x, acc) : acc;
    y[id] = (T)(a.z ? v * (z * sigmoid_hw(z)) : v);
  }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------
struct ScanSplit {
  int cpl, nch, wpg, cl, chunks;
};
// Chunks cost a second pass over the states, so sequences are cut only where whole ones leave most of the chip idle: into chunks of
// at least 64 tokens until there are about 8 192 waves (8 a SIMD, so that their uneven spread over the CUs does not count: 4 096 took
// 1.35 times as long at 2 x 262144 x 96), and only if that makes at least 4 chunks.
// Two channels a quad (half the LDS reads of B and C) once there are enough waves; one where the latency of few waves counts.
inline ScanSplit scan_split(int B, int L, int D, int G) {
  ScanSplit s;
  const int dg = D / G;
  const long waves2 = (long)B * G * ((dg + 31) / 32);
  long want = 8192 / waves2;
  const long most = (L + 63) / 64;
  if (want > most) want = most;
  if (want < 4) want = 1;
  s.cpl = waves2 * want >= 4096 ? 2 : 1;
  long cl = (L + want - 1) / want;
  cl = (cl + SC_TT - 1) / SC_TT * SC_TT;
  s.cl = (int)cl;
  s.chunks = (int)((L + cl - 1) / cl);
  // up to 4 waves a workgroup, as many as pad the group's channels least
  const int wch = 16 * s.cpl, need = (dg + wch - 1) / wch;
  int best = 1;
  for (int w = 2; w <= 4; ++w)
    if ((need + w - 1) / w * w <= (need + best - 1) / best * best) best = w;
  s.nch = best * wch;
  s.wpg = (dg + s.nch - 1) / s.nch;
  return s;
}
template <class T, int N, int CPL>
static int scan_prompt_run(const ScanStateArgs& a, hipStream_t s) {
  const dim3 grid(a.G * a.wpg, a.chunks, a.B), block(a.nch * 4 / CPL);
  const int lds = SC_TT * (3 * a.nch + 2 * N) * 4, lds1 = SC_TT * (2 * a.nch + N) * 4;
  static DynLdsCache c0, c1, c2;
  hipError_t e;
  if (a.chunks == 1) {
    if ((e = ensure_dyn_lds((const void*)scan_prompt_kernel<T, N, CPL, 0>, lds, c0)) != hipSuccess) return (int)e;
    NNZ_LAUNCH((scan_prompt_kernel<T, N, CPL, 0>), grid, block, lds, s, a);
  } else {
    if ((e = ensure_dyn_lds((const void*)scan_prompt_kernel<T, N, CPL, 1>, lds1, c1)) != hipSuccess) return (int)e;
    if ((e = ensure_dyn_lds((const void*)scan_prompt_kernel<T, N, CPL, 2>, lds, c2)) != hipSuccess) return (int)e;
    const dim3 sums(a.G * a.wpg, a.joined ? a.chunks : a.chunks - 1, a.B);
    NNZ_LAUNCH((scan_prompt_kernel<T, N, CPL, 1>), sums, block, lds1, s, a);
    NNZ_LAUNCH_CHECK();
    if (a.joined) {
      const long dn = (long)a.D * N;
      NNZ_LAUNCH((scan_join_kernel<N, 16, 64>), dim3((unsigned)((dn + 15) / 16), a.B), dim3(1024), 0, s, a);
      NNZ_LAUNCH_CHECK();
    }
    NNZ_LAUNCH((scan_prompt_kernel<T, N, CPL, 2>), grid, block, lds, s, a);
  }
  NNZ_LAUNCH_CHECK();
  return NNZ_OK;
}
template <class T, int N>
static int scan_state_run(const ScanStateArgs& a, int cpl, bool token, hipStream_t s) {
  if (token) {
    const long wg = ((long)a.B * a.D * 4 + 255) / 256;
    if (wg >= 1L << 24) return NNZ_EINVAL;   // 2^32 threads
    NNZ_LAUNCH((scan_token_kernel<T, N>), dim3((unsigned)wg), dim3(256), 0, s, a);
    NNZ_LAUNCH_CHECK();
    return NNZ_OK;
  }
  return cpl == 2 ? scan_prompt_run<T, N, 2>(a, s) : scan_prompt_run<T, N, 1>(a, s);
}
template <class T>
static int scan_state_n(const ScanStateArgs& a, int N, int cpl, bool token, hipStream_t s) {
  switch (N) {
    case 4: return scan_state_run<T, 4>(a, cpl, token, s);
    case 8: return scan_state_run<T, 8>(a, cpl, token, s);
    case 16: return scan_state_run<T, 16>(a, cpl, token, s);
    case 32: return scan_state_run<T, 32>(a, cpl, token, s);
  }
  return NNZ_EINVAL;
}
static int scan_state_go(const ScanStateArgs& a, int type, int N, int cpl, bool token, hipStream_t s) {
  if (type == ELEM_F32) return scan_state_n<float>(a, N, cpl, token, s);
  if (type == ELEM_F16) return scan_state_n<f16>(a, N, cpl, token, s);
  if (type == ELEM_BF16) return scan_state_n<bf16>(a, N, cpl, token, s);
  return NNZ_EINVAL;
}
static bool scan_shape_ok(int B, int L, int D, int H, int G, int N) {
  return B >= 1 && L >= 1 && L <= (1 << 30) && D >= 1 && H >= 1 && G >= 1 && D % H == 0 && D % G == 0 &&
         H % G == 0 && (N == 4 || N == 8 || N == 16 || N == 32);
}

}  // namespace nnz

extern "C" int nnz_causal_conv1d_prompt(const void* x, int type, long x_batch_stride, long x_token_stride, const float* weight,
                                        const float* bias, void* y, void* conv_state, int state_type, long state_batch_stride,
                                        long state_channel_stride, long state_column_stride, const void* lengths,
                                        int lengths_are_int64, int B, int L, int D, int W, int silu, void* stream) {
  using namespace nnz;
  if (!x || !weight || !y || B < 1 || L < 1 || L > (1 << 30) || D < 1 || (conv_state && !elem_ok(state_type))) return NNZ_EINVAL;
  ConvStateArgs a = {};
  a.x = x; a.w = weight; a.bias = bias; a.y = y; a.st = conv_state; a.len = lengths;
  a.xb = x_batch_stride; a.xt = x_token_stride;
  a.sb = state_batch_stride; a.sd = state_channel_stride; a.sw = state_column_stride;
  a.B = B; a.L = L; a.D = D; a.silu = silu; a.len64 = lengths_are_int64; a.st_type = state_type;
  return conv_state_go(a, type, W, false, (hipStream_t)stream);
}

extern "C" int nnz_causal_conv1d_token(const void* x, int type, long x_batch_stride, const float* weight, const float* bias, void* y,
                                       void* conv_state, int state_type, long state_batch_stride, long state_channel_stride,
                                       long state_column_stride, const void* active, int B, int D, int W, int silu,
                                       void* stream) {
  using namespace nnz;
  if (!x || !weight || !y || !conv_state || B < 1 || D < 1 || (long)B * D > 0xFFFFFF00L || !elem_ok(state_type)) return NNZ_EINVAL;
  ConvStateArgs a = {};
  a.x = x; a.w = weight; a.bias = bias; a.y = y; a.st = conv_state; a.len = active;
  a.xb = x_batch_stride; a.sb = state_batch_stride; a.sd = state_channel_stride; a.sw = state_column_stride;
  a.B = B; a.L = 1; a.D = D; a.silu = silu; a.st_type = state_type;
  return conv_state_go(a, type, W, true, (hipStream_t)stream);
}

extern "C" long nnz_selective_scan_prompt_workspace_bytes(int B, int L, int D, int H, int G, int N) {
  using namespace nnz;
  if (!scan_shape_ok(B, L, D, H, G, N)) return NNZ_EINVAL;
  const ScanSplit s = scan_split(B, L, D, G);
  return s.chunks == 1 ? 0 : (long)s.chunks * B * D * (N + 1) * 4;
}

extern "C" int nnz_selective_scan_prompt(const void* x, const void* dt, const void* Bm, const void* Cm, const void* z, int type,
                                         const long* strides, const float* A, int A_form, const float* D_skip,
                                         const float* dt_bias, int softplus, float* state, long state_batch_stride, void* y,
                                         const void* lengths, int lengths_are_int64, void* workspace, long workspace_bytes,
                                         int B, int L, int D, int H, int G, int N, void* stream) {
  using namespace nnz;
  if (!x || !dt || !Bm || !Cm || !A || !y || !strides || B > 65535 || !scan_shape_ok(B, L, D, H, G, N)) return NNZ_EINVAL;
  const ScanSplit sp = scan_split(B, L, D, G);
  if (sp.chunks > 1 && (!workspace || workspace_bytes < (long)sp.chunks * B * D * (N + 1) * 4)) return NNZ_EINVAL;
  ScanStateArgs a = {};
  a.x = x; a.dt = dt; a.Bm = Bm; a.Cm = Cm; a.z = z; a.A = A; a.a_n = A_form & 1; a.a_log = A_form >> 1 & 1; a.Dv = D_skip; a.dt_bias = dt_bias;
  a.state = state; a.sb = state_batch_stride; a.y = y; a.len = lengths; a.len64 = lengths_are_int64;
  a.xb = strides[0]; a.xt = strides[1]; a.db = strides[2]; a.dtt = strides[3]; a.bb = strides[4]; a.bt = strides[5];
  a.bg = strides[6]; a.cb = strides[7]; a.ct = strides[8]; a.cg = strides[9]; a.zb = strides[10]; a.zt = strides[11];
  a.part_h = (float*)workspace;
  a.part_d = a.part_h + (long)sp.chunks * B * D * N;
  a.B = B; a.L = L; a.D = D; a.H = H; a.G = G; a.softplus = softplus;
  a.rep = D / H; a.dg = D / G; a.nch = sp.nch; a.wpg = sp.wpg; a.cl = sp.cl; a.chunks = sp.chunks;
  a.joined = sp.chunks >= SC_JOIN;
  const uintptr_t m = 2 * (uintptr_t)elem_size(type) - 1;   // a pair's alignment; a group begins at an even channel
  a.pair = (((uintptr_t)x | (uintptr_t)z | (uintptr_t)y) & m) == 0 && ((a.xb | a.xt | a.zb | a.zt | D | a.dg) & 1) == 0;
  a.pair_dt = a.rep == 1 && ((uintptr_t)dt & m) == 0 && ((a.db | a.dtt | a.dg) & 1) == 0;
  return scan_state_go(a, type, N, sp.cpl, false, (hipStream_t)stream);
}

extern "C" int nnz_selective_scan_token(const void* x, const void* dt, const void* Bm, const void* Cm, const void* z, int type,
                                        const long* strides, const float* A, int A_form, const float* D_skip,
                                        const float* dt_bias, int softplus, float* state, long state_batch_stride, void* y,
                                        const void* active, int B, int D, int H, int G, int N, void* stream) {
  using namespace nnz;
  if (!x || !dt || !Bm || !Cm || !A || !y || !state || !strides || !scan_shape_ok(B, 1, D, H, G, N)) return NNZ_EINVAL;
  ScanStateArgs a = {};
  a.x = x; a.dt = dt; a.Bm = Bm; a.Cm = Cm; a.z = z; a.A = A; a.a_n = A_form & 1; a.a_log = A_form >> 1 & 1; a.Dv = D_skip; a.dt_bias = dt_bias;
  a.state = state; a.sb = state_batch_stride; a.y = y; a.len = active;
  a.xb = strides[0]; a.db = strides[1]; a.bb = strides[2]; a.bg = strides[3]; a.cb = strides[4]; a.cg = strides[5];
  a.zb = strides[6];
  a.B = B; a.L = 1; a.D = D; a.H = H; a.G = G; a.softplus = softplus;
  a.rep = D / H; a.dg = D / G;
  return scan_state_go(a, type, N, 0, true, (hipStream_t)stream);
}
