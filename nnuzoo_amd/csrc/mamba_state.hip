// The state-carrying operators of a Mamba block (gfx950), token-major, for prompts and for single tokens:
//   short causal convolution   y_t = act(bias + sum_j w_j x_{t-W+1+j}); inputs before the first come from conv_state (the last W
//                              inputs of the sequence), which is brought up to date in place;
//   selective scan             D_t = [softplus](dt_t + dt_bias);  h_t = exp(D_t A) h_{t-1} + D_t x_t B_t;
//                              y_t = <C_t, h_t> + D x_t, times silu(z_t);  h starts from `state` and is left there.
// Rows are (B, L, D) with the channels innermost, as the projections around them write and read them: nothing is transposed.
// Every sequence has its own length; nothing behind it is read, its outputs are 0, and a sequence of length 0 keeps its states.
// Sums and states are fp32 whatever the activations' type.
#include "elem_io.hpp"

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

// a thread: V adjacent channels, tt consecutive tokens, the window in registers
template <class T, int W, int V>
__global__ __launch_bounds__(256) void conv_prompt_kernel(ConvStateArgs a) {
  const int CV = a.D / V;
  const int chunks = (a.L + a.tt - 1) / a.tt;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long)CV * chunks * a.B) return;
  const int d = (int)(id % CV) * V;
  const long rest = id / CV;
  const int t0 = (int)(rest % chunks) * a.tt;
  const int b = (int)(rest / chunks);
  const int len = seq_len(a.len, a.len64, b, a.L);
  const int t1 = t0 + a.tt < a.L ? t0 + a.tt : a.L;
  const T* x = (const T*)a.x + (long)b * a.xb + d;
  T* y = (T*)a.y + ((long)b * a.L) * a.D + d;
  float w[V][W], bias[V], win[W][V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    bias[v] = a.bias ? a.bias[d + v] : 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) w[v][j] = a.w[(long)(d + v) * W + j];
  }
  // the W - 1 inputs before t0 (win[W - 1] is the current one); inputs before the sequence: the state's last columns
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const int t = t0 - (W - 1) + j;
    if (t >= 0) {
      if (t < len) ld_elems<T, V>(x + (long)t * a.xt, win[j + 1]);
      else {
#pragma unroll
        for (int v = 0; v < V; ++v) win[j + 1][v] = 0.f;
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
        win[j + 1][v] = a.st ? ld_any(a.st, b * a.sb + (long)(d + v) * a.sd + (long)(W + t) * a.sw, a.st_type) : 0.f;
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
  int t = t0;
#pragma unroll 4
  for (; t < te; ++t) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) win[j][v] = win[j + 1][v];
    ld_elems<T, V>(x + (long)t * a.xt, win[W - 1]);
    float o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s = bias[v];
#pragma unroll
      for (int j = 0; j < W; ++j) s = fmaf(w[v][j], win[j][v], s);
      o[v] = a.silu ? s * sigmoid_hw(s) : s;
    }
    st_elems<T, V>(y + (long)t * a.D, o);
  }
  const float zero[V] = {};
  for (; t < t1; ++t) st_elems<T, V>(y + (long)t * a.D, zero);
}

// one token: a thread per (sequence, channel)
template <class T, int W>
__global__ __launch_bounds__(256) void conv_token_kernel(ConvStateArgs a) {
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long)a.B * a.D) return;
  const int b = (int)(id / a.D), d = (int)(id % a.D);
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
  constexpr int FULL = 16 / (int)sizeof(T);
  const bool vec = a.D % FULL == 0 && a.xb % FULL == 0 && a.xt % FULL == 0 && (((uintptr_t)a.x | (uintptr_t)a.y) & 15) == 0;
  const int CV = vec ? a.D / FULL : a.D;
  // a thread re-reads W - 1 tokens (from L2): 16 tokens each once that leaves enough threads, 8 on short inputs and no fewer: only
  // a sequence's first chunk may need the state, for its thread writes the new one (8 >= W - 1)
  a.tt = (long)CV * a.B * ((a.L + 15) / 16) < 256L * 512 ? 8 : 16;
  const long wg = ((long)CV * a.B * ((a.L + a.tt - 1) / a.tt) + 255) / 256;
  if (wg > 0x7FFFFFFFL) return NNZ_EINVAL;
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
  const float* A;        // [H][N] (a_n = 1) or [H] (a_n = 0)
  const float* Dv;       // [H] or null
  const float* dt_bias;  // [H] or null
  float* state;          // [B][D][N], batch stride sb, rows contiguous; or null (zeros, nothing kept)
  void* y;               // [B][L][D] contiguous
  const void* len;       // as above
  float* part_h;         // [chunks][B][D][N]: slot 0 the entry state of the sequence, slot c + 1 the end state of chunk c from a zero
                         // entry (chunk 0: from the true one)
  float* part_d;         // [chunks][B][D]: slot c + 1 the sum of D_t over chunk c
  long xb, xt, db, dtt, bb, bt, bg, cb, ct, cg, zb, zt, sb;
  int B, L, D, H, G, softplus, len64, a_n;
  int rep;               // channels of a head
  int dg;                // channels of a group
  int wpg;               // workgroups (channel blocks) of a group
  int cl, chunks;        // tokens of a chunk
};

// e^x with the rounding of x * log2(e) put right
__device__ __forceinline__ float exp_fine(float x) {
  const float p = x * 1.4426950408889634f;
  const float r = fmaf(x, 1.9259629911266175e-8f, fmaf(x, 1.4426950408889634f, -p));
  const float e = __builtin_amdgcn_exp2f(p);
  return fmaf(e * 0.6931471805599453f, r, e);
}
// softplus(x) = max(x, 0) + log(1 + e), e = exp(-|x|) <= 1, by log(1 + e) = 2 atanh(s), s = e / (2 + e) <= 1/3: relative accuracy
// for small e, too (a time step is often softplus of -5, and the states' decay takes its relative error)
__device__ __forceinline__ float softplus_hw(float x) {
  const float e = x == x ? exp_fine(-fabsf(x)) : x;
  const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
  float p = fmaf(q, 1.f / 13.f, 1.f / 11.f);
  p = fmaf(q, p, 1.f / 9.f);
  p = fmaf(q, p, 1.f / 7.f);
  p = fmaf(q, p, 1.f / 5.f);
  p = fmaf(q, p, 1.f / 3.f);
  p = fmaf(q, p, 1.f);
  return fmaf(2.f * s, p, x > 0.f ? x : 0.f);
}

constexpr float LOG2E = 1.4426950408889634f;

// 4 lanes share a channel and hold N / 4 states each; a workgroup has NCH channels of one group and walks its tokens in tiles:
// every (token, channel) of a tile is loaded and turned into D_t, D_t x_t once, B and C are widened once, all through LDS.
// MODE 0: whole sequences in one launch.  Long sequences of few channels are cut into chunks: MODE 1 leaves every chunk's summary
// (end state, sum of D_t: the chunk multiplies its entry state by exp(A sum D)), MODE 2 joins the summaries before its chunk and
// runs it from the true entry state.
constexpr int SC_TT = 32;   // tokens of a tile

template <class T, int N, int NCH, int MODE>
__global__ __launch_bounds__(NCH * 4) void scan_prompt_kernel(ScanStateArgs a) {
  constexpr int NT = NCH * 4, NS = N / 4;
  constexpr int IT = SC_TT * NCH / NT;   // elements of a thread in the staging passes
  __shared__ float2 s_du[SC_TT][NCH];
  __shared__ __attribute__((aligned(16))) float s_b[SC_TT][N];
  __shared__ __attribute__((aligned(16))) float s_c[SC_TT][N];
  __shared__ float s_y[SC_TT][NCH];
  const int tid = threadIdx.x;
  const int g = blockIdx.x / a.wpg;
  const int ch0 = (blockIdx.x % a.wpg) * NCH;       // within the group
  const int chunk = blockIdx.y, b = blockIdx.z;
  const int len = seq_len(a.len, a.len64, b, a.L);
  const int t0 = chunk * a.cl;
  const int tend = t0 + a.cl < a.L ? t0 + a.cl : a.L;
  const int te = tend < len ? tend : len;
  // staging role: one channel, tokens (tid / NCH) + 4 i
  const int sch = tid % NCH, st = tid / NCH;
  const bool s_on = ch0 + sch < a.dg;
  const int sd = g * a.dg + (s_on ? ch0 + sch : a.dg - 1);
  const int shead = sd / a.rep;
  const float sbias = a.dt_bias ? a.dt_bias[shead] : 0.f;
  const float sD = a.Dv ? a.Dv[shead] : 0.f;
  // state role: 4 lanes a channel
  const int sub = tid & 3, mch = tid >> 2;
  const bool m_on = ch0 + mch < a.dg;
  const int md = g * a.dg + (m_on ? ch0 + mch : a.dg - 1);
  const int mhead = md / a.rep;
  float A2[NS], h[NS];
  const long srow = (long)b * a.sb + (long)md * N + sub * NS;
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    A2[n] = (a.a_n ? a.A[(long)mhead * N + sub * NS + n] : a.A[mhead]) * LOG2E;
    h[n] = 0.f;
  }
  const long prow = ((long)b * a.D + md) * N + sub * NS, pstep = (long)a.B * a.D * N;
  if (MODE == 2) {
    // never from `state`: the workgroup of the last token may have written it already
    if (t0 < te) {
      const float* p = a.part_h + (chunk > 0 ? pstep : 0) + prow;
#pragma unroll
      for (int n = 0; n < NS; ++n) h[n] = p[n];
#pragma unroll 4
      for (int c = 2; c <= chunk; ++c) {
        const float sum = a.part_d[((long)c * a.B + b) * a.D + md];
#pragma unroll
        for (int n = 0; n < NS; ++n) h[n] = fmaf(__builtin_amdgcn_exp2f(sum * A2[n]), h[n], a.part_h[c * pstep + prow + n]);
      }
    }
  } else if (chunk == 0 && a.state) {
#pragma unroll
    for (int n = 0; n < NS; ++n) h[n] = a.state[srow + n];
  }
  if (MODE == 1 && chunk == 0 && m_on) {
#pragma unroll
    for (int n = 0; n < NS; ++n) a.part_h[prow + n] = h[n];
  }
  float dsum = 0.f;
  const T* xp = (const T*)a.x + (long)b * a.xb + sd;
  const T* zp = a.z ? (const T*)a.z + (long)b * a.zb + sd : nullptr;
  const T* dp = (const T*)a.dt + (long)b * a.db + shead;
  const T* bp = (const T*)a.Bm + (long)b * a.bb + g * a.bg;
  const T* cp = (const T*)a.Cm + (long)b * a.cb + g * a.cg;
  T* yp = (T*)a.y + (long)b * a.L * a.D + sd;
  for (int tile = t0; tile < te; tile += SC_TT) {
    float xv[IT], zv[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int t = tile + st + 4 * i;
      float dl = 0.f;
      xv[i] = 0.f;
      zv[i] = 0.f;
      if (t < te) {
        xv[i] = (float)xp[(long)t * a.xt];
        if (MODE != 1 && zp) zv[i] = (float)zp[(long)t * a.zt];
        dl = (float)dp[(long)t * a.dtt] + sbias;
        if (a.softplus) dl = softplus_hw(dl);
      }
      s_du[st + 4 * i][sch] = make_float2(dl, dl * xv[i]);
    }
    for (int i = tid; i < SC_TT * N; i += NT) {
      const int tt = i / N, n = i % N, t = tile + tt;
      s_b[tt][n] = t < te ? (float)bp[(long)t * a.bt + n] : 0.f;
      if (MODE != 1) s_c[tt][n] = t < te ? (float)cp[(long)t * a.ct + n] : 0.f;
    }
    __syncthreads();
    const int cnt = te - tile < SC_TT ? te - tile : SC_TT;
#pragma unroll 4
    for (int tt = 0; tt < cnt; ++tt) {
      const float2 du = s_du[tt][mch];
      float acc = 0.f;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        h[n] = fmaf(__builtin_amdgcn_exp2f(du.x * A2[n]), h[n], du.y * s_b[tt][sub * NS + n]);
        if (MODE != 1) acc = fmaf(h[n], s_c[tt][sub * NS + n], acc);
      }
      if (MODE == 1) dsum += du.x;
      else {
        acc += __shfl_xor(acc, 1, 64);
        acc += __shfl_xor(acc, 2, 64);
        if (sub == 0) s_y[tt][mch] = acc;
      }
    }
    __syncthreads();
    if (MODE != 1) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int t = tile + st + 4 * i;
        if (t < te && s_on) {
          float v = fmaf(sD, xv[i], s_y[st + 4 * i][sch]);
          if (zp) v *= zv[i] * sigmoid_hw(zv[i]);
          yp[(long)t * a.D] = (T)v;
        }
      }
    }
  }
  if (MODE == 1) {
    if (m_on) {
      float* o = a.part_h + (chunk + 1) * pstep + prow;
#pragma unroll
      for (int n = 0; n < NS; ++n) o[n] = h[n];
      if (sub == 0) a.part_d[((long)(chunk + 1) * a.B + b) * a.D + md] = dsum;
    }
    return;
  }
  if (s_on)
    for (int t = (te > t0 ? te : t0) + st; t < tend; t += 4) yp[(long)t * a.D] = (T)0.f;
  // the chunk that holds the last token leaves the state
  if (a.state && m_on && len > 0 && t0 < len && len <= tend) {
#pragma unroll
    for (int n = 0; n < NS; ++n) a.state[srow + n] = h[n];
  }
}

// one token: 4 lanes a channel
template <class T, int N>
__global__ __launch_bounds__(256) void scan_token_kernel(ScanStateArgs a) {
  constexpr int NS = N / 4;
  const long id = ((long)blockIdx.x * 256 + threadIdx.x) >> 2;
  const int sub = threadIdx.x & 3;
  if (id >= (long)a.B * a.D) return;     // all 4 lanes of a channel leave together
  const int b = (int)(id / a.D), d = (int)(id % a.D);
  T* y = (T*)a.y;
  if (a.len && !((const unsigned char*)a.len)[b]) {
    if (sub == 0) y[id] = (T)0.f;
    return;
  }
  const int head = d / a.rep, g = d / a.dg;
  float* st = a.state + (long)b * a.sb + (long)d * N + sub * NS;
  const T* bp = (const T*)a.Bm + (long)b * a.bb + g * a.bg + sub * NS;
  const T* cp = (const T*)a.Cm + (long)b * a.cb + g * a.cg + sub * NS;
  float dl = (float)((const T*)a.dt)[b * a.db + head] + (a.dt_bias ? a.dt_bias[head] : 0.f);
  if (a.softplus) dl = softplus_hw(dl);
  const float x = (float)((const T*)a.x)[b * a.xb + d];
  const float u = dl * x;
  float acc = 0.f;
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const float A2 = (a.a_n ? a.A[(long)head * N + sub * NS + n] : a.A[head]) * LOG2E;
    const float h = fmaf(__builtin_amdgcn_exp2f(dl * A2), st[n], u * (float)bp[n]);
    st[n] = h;
    acc = fmaf(h, (float)cp[n], acc);
  }
  acc += __shfl_xor(acc, 1, 64);
  acc += __shfl_xor(acc, 2, 64);
  if (sub == 0) {
    float v = a.Dv ? fmaf(a.Dv[head], x, acc) : acc;
    if (a.z) {
      const float z = (float)((const T*)a.z)[b * a.zb + d];
      v *= z * sigmoid_hw(z);
    }
    y[id] = (T)v;
  }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------
constexpr int SC_MAX_CHUNKS = 128;
// channels of a workgroup: the widest block that pads the group's channels least
inline int scan_nch(int dg) {
  int best = 16;
  for (int c = 32; c <= 64; c *= 2)
    if ((dg + c - 1) / c * c <= (dg + best - 1) / best * best) best = c;
  return best;
}
struct ScanSplit {
  int nch, wpg, cl, chunks;
};
// Chunks cost a second pass over the states, so sequences are cut only where whole ones leave most of the chip idle
// (256 CUs x 4 SIMDs: under 512 waves), into chunks of at least 4 tiles, until there are about 2 048 waves.
inline ScanSplit scan_split(int B, int L, int D, int G) {
  ScanSplit s;
  const int dg = D / G;
  s.nch = scan_nch(dg);
  s.wpg = (dg + s.nch - 1) / s.nch;
  const long waves = (long)B * G * s.wpg * (s.nch / 16);
  long want = waves >= 512 ? 1 : (2048 + waves - 1) / waves;
  const long most = (L + 4 * SC_TT - 1) / (4 * SC_TT);
  if (want > most) want = most;
  if (want > SC_MAX_CHUNKS) want = SC_MAX_CHUNKS;
  if (want < 1) want = 1;
  long cl = (L + want - 1) / want;
  cl = (cl + SC_TT - 1) / SC_TT * SC_TT;
  s.cl = (int)cl;
  s.chunks = (int)((L + cl - 1) / cl);
  return s;
}
template <class T, int N, int NCH>
static int scan_prompt_run(const ScanStateArgs& a, hipStream_t s) {
  const dim3 grid(a.G * a.wpg, a.chunks, a.B);
  if (a.chunks == 1) {
    NNZ_LAUNCH((scan_prompt_kernel<T, N, NCH, 0>), grid, dim3(NCH * 4), 0, s, a);
  } else {
    // the last chunk's summary is not needed
    NNZ_LAUNCH((scan_prompt_kernel<T, N, NCH, 1>), dim3(a.G * a.wpg, a.chunks - 1, a.B), dim3(NCH * 4), 0, s, a);
    NNZ_LAUNCH_CHECK();
    NNZ_LAUNCH((scan_prompt_kernel<T, N, NCH, 2>), grid, dim3(NCH * 4), 0, s, a);
  }
  NNZ_LAUNCH_CHECK();
  return NNZ_OK;
}
template <class T, int N>
static int scan_state_run(const ScanStateArgs& a, int nch, bool token, hipStream_t s) {
  if (token) {
    const long wg = ((long)a.B * a.D * 4 + 255) / 256;
    if (wg > 0x7FFFFFFFL) return NNZ_EINVAL;
    NNZ_LAUNCH((scan_token_kernel<T, N>), dim3((unsigned)wg), dim3(256), 0, s, a);
    NNZ_LAUNCH_CHECK();
    return NNZ_OK;
  }
  if (nch == 64) return scan_prompt_run<T, N, 64>(a, s);
  if (nch == 32) return scan_prompt_run<T, N, 32>(a, s);
  return scan_prompt_run<T, N, 16>(a, s);
}
template <class T>
static int scan_state_n(const ScanStateArgs& a, int N, int nch, bool token, hipStream_t s) {
  switch (N) {
    case 4: return scan_state_run<T, 4>(a, nch, token, s);
    case 8: return scan_state_run<T, 8>(a, nch, token, s);
    case 16: return scan_state_run<T, 16>(a, nch, token, s);
    case 32: return scan_state_run<T, 32>(a, nch, token, s);
  }
  return NNZ_EINVAL;
}
static int scan_state_go(const ScanStateArgs& a, int type, int N, int nch, bool token, hipStream_t s) {
  if (type == ELEM_F32) return scan_state_n<float>(a, N, nch, token, s);
  if (type == ELEM_F16) return scan_state_n<f16>(a, N, nch, token, s);
  if (type == ELEM_BF16) return scan_state_n<bf16>(a, N, nch, token, s);
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
  if (!x || !weight || !y || !conv_state || B < 1 || D < 1 || (long)B * D > (1L << 38) || !elem_ok(state_type)) return NNZ_EINVAL;
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
                                         const long* strides, const float* A, int A_per_state, const float* D_skip,
                                         const float* dt_bias, int softplus, float* state, long state_batch_stride, void* y,
                                         const void* lengths, int lengths_are_int64, void* workspace, long workspace_bytes,
                                         int B, int L, int D, int H, int G, int N, void* stream) {
  using namespace nnz;
  if (!x || !dt || !Bm || !Cm || !A || !y || !strides || B > 65535 || !scan_shape_ok(B, L, D, H, G, N)) return NNZ_EINVAL;
  const ScanSplit sp = scan_split(B, L, D, G);
  if (sp.chunks > 1 && (!workspace || workspace_bytes < (long)sp.chunks * B * D * (N + 1) * 4)) return NNZ_EINVAL;
  ScanStateArgs a = {};
  a.x = x; a.dt = dt; a.Bm = Bm; a.Cm = Cm; a.z = z; a.A = A; a.a_n = A_per_state; a.Dv = D_skip; a.dt_bias = dt_bias;
  a.state = state; a.sb = state_batch_stride; a.y = y; a.len = lengths; a.len64 = lengths_are_int64;
  a.xb = strides[0]; a.xt = strides[1]; a.db = strides[2]; a.dtt = strides[3]; a.bb = strides[4]; a.bt = strides[5];
  a.bg = strides[6]; a.cb = strides[7]; a.ct = strides[8]; a.cg = strides[9]; a.zb = strides[10]; a.zt = strides[11];
  a.part_h = (float*)workspace;
  a.part_d = a.part_h + (long)sp.chunks * B * D * N;
  a.B = B; a.L = L; a.D = D; a.H = H; a.G = G; a.softplus = softplus;
  a.rep = D / H; a.dg = D / G; a.wpg = sp.wpg; a.cl = sp.cl; a.chunks = sp.chunks;
  return scan_state_go(a, type, N, sp.nch, false, (hipStream_t)stream);
}

extern "C" int nnz_selective_scan_token(const void* x, const void* dt, const void* Bm, const void* Cm, const void* z, int type,
                                        const long* strides, const float* A, int A_per_state, const float* D_skip,
                                        const float* dt_bias, int softplus, float* state, long state_batch_stride, void* y,
                                        const void* active, int B, int D, int H, int G, int N, void* stream) {
  using namespace nnz;
  if (!x || !dt || !Bm || !Cm || !A || !y || !state || !strides || !scan_shape_ok(B, 1, D, H, G, N)) return NNZ_EINVAL;
  ScanStateArgs a = {};
  a.x = x; a.dt = dt; a.Bm = Bm; a.Cm = Cm; a.z = z; a.A = A; a.a_n = A_per_state; a.Dv = D_skip; a.dt_bias = dt_bias;
  a.state = state; a.sb = state_batch_stride; a.y = y; a.len = active;
  a.xb = strides[0]; a.db = strides[1]; a.bb = strides[2]; a.bg = strides[3]; a.cb = strides[4]; a.cg = strides[5];
  a.zb = strides[6];
  a.B = B; a.L = 1; a.D = D; a.H = H; a.G = G; a.softplus = softplus;
  a.rep = D / H; a.dg = D / G;
  return scan_state_go(a, type, N, 0, true, (hipStream_t)stream);
}
