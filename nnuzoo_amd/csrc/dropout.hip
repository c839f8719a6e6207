// Dropout whose mask comes from a counter-based generator and is never stored (gfx950): forward, forward with a residual,
// backward.
//   element e is kept iff u(e) >= T, T = round(p 2^32);  y = kept ? x / (1 - p) : 0  [+ residual];  dx = kept ? dy / (1 - p) : 0
//   u(e): the call Philox-4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC'11) with key =
//   seed and counter (e / 8 low, e / 8 high, site, step) gives 128 bits = the HIGH halves of the 8 draws of block e / 8; their low
//   halves come from a second call (top bit of the second counter word set).
// The mask depends on (seed, step, site, e) alone: not on the type, the launch or the alignment.  Seed and step are read from
// device memory, so a captured graph draws anew at every replay once the step has been advanced inside it.
//
// Bound by HBM, with integer multiplication close behind: a call is 20 products of 32 x 32 -> 64 bits at a quarter of the vector
// rate.  One call serves 8 elements because a 16-bit half already decides unless it EQUALS the threshold's upper half; that
// happens once in 65 536 elements, and only the waves that meet it make the second call - the probability is exact to 2^-32 at
// half the price of 32-bit draws.  2 x 512^2 x 128 f16: 50 us each way = 5.4 TB/s, what a copy of that size reaches.
#include "elem_io.hpp"

namespace nnz {

struct DropArgs {
  const void* x;           // forward: x, backward: dy
  const void* res;         // residual or null
  void* y;                 // y or dx
  const long long* state;  // {seed, step}
  long long* used;         // where the forward leaves the pair for its backward, or null
  long n;
  unsigned t_hi, t_lo;     // the threshold's halves; t_hi = 65536: everything is dropped
  float scale;
  unsigned site;
  int vec;                 // all pointers are 16-byte aligned
};

struct Philox4 {
  unsigned w[4];
};
__device__ __forceinline__ Philox4 philox10(unsigned c0, unsigned c1, unsigned c2, unsigned c3, unsigned k0, unsigned k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(p1 >> 32) ^ c1 ^ k0;
    c1 = (unsigned)p1;
    c2 = (unsigned)(p0 >> 32) ^ c3 ^ k1;
    c3 = (unsigned)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Philox4{{c0, c1, c2, c3}};
}

// bit j: element 8 blk + j is kept
__device__ __forceinline__ unsigned kept8(const DropArgs& a, uint64_t blk, unsigned k0, unsigned k1, unsigned step) {
  const Philox4 h = philox10((unsigned)blk, (unsigned)(blk >> 32), a.site, step, k0, k1);
  unsigned kept = 0, tie = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const unsigned u = (h.w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu;
    kept |= (u > a.t_hi ? 1u : 0u) << j;
    tie |= (u == a.t_hi ? 1u : 0u) << j;
  }
  if (tie) {
    const Philox4 l = philox10((unsigned)blk, (unsigned)(blk >> 32) | 0x80000000u, a.site, step, k0, k1);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned u = (l.w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu;
      kept |= (((tie >> j) & 1u) && u >= a.t_lo ? 1u : 0u) << j;
    }
  }
  return kept;
}

template <class TX, class TR, class TY, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs a) {
  const long long seed = a.state[0], st = a.state[1];
  const unsigned k0 = (unsigned)seed, k1 = (unsigned)((unsigned long long)seed >> 32), step = (unsigned)st;
  if (a.used && blockIdx.x == 0 && threadIdx.x == 0) {
    a.used[0] = seed;
    a.used[1] = st;
  }
  const TX* x = (const TX*)a.x;
  const TR* res = (const TR*)a.res;
  TY* y = (TY*)a.y;
  const long nblk = (a.n + 7) / 8;
  for (long blk = (long)blockIdx.x * 256 + threadIdx.x; blk < nblk; blk += (long)gridDim.x * 256) {
    const long i = blk * 8;
    const int cnt = a.n - i < 8 ? (int)(a.n - i) : 8;
    const bool whole = a.vec && cnt == 8;
    float v[8], r[8];
    if (whole) {
      ld_elems<TX, 8>(x + i, v);
      if (RES) ld_elems<TR, 8>(res + i, r);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = j < cnt ? (float)x[i + j] : 0.f;
        if (RES) r[j] = j < cnt ? (float)res[i + j] : 0.f;
      }
    }
    const unsigned kept = kept8(a, (uint64_t)blk, k0, k1, step);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = (kept >> j) & 1u ? v[j] * a.scale : 0.f;   // a dropped inf or NaN is 0, too
      if (RES) v[j] += r[j];
    }
    if (whole) {
      st_elems<TY, 8>(y + i, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < cnt) y[i + j] = (TY)v[j];
    }
  }
}

template <class TX, class TR, class TY, bool RES>
static int drop_run(const DropArgs& a, hipStream_t s) {
  long wg = (a.n + 2047) / 2048;
  if (wg > 8192) wg = 8192;
  NNZ_LAUNCH((dropout_kernel<TX, TR, TY, RES>), dim3((unsigned)wg), dim3(256), 0, s, a);
  NNZ_LAUNCH_CHECK();
  return NNZ_OK;
}
template <class A, class B>
struct Wider {   // fp32 unless the two are one type
  typedef float type;
};
template <class A>
struct Wider<A, A> {
  typedef A type;
};
template <class TX>
static int drop_res(const DropArgs& a, int rt, hipStream_t s) {
  if (rt == ELEM_F32) return drop_run<TX, float, typename Wider<TX, float>::type, true>(a, s);
  if (rt == ELEM_F16) return drop_run<TX, f16, typename Wider<TX, f16>::type, true>(a, s);
  return drop_run<TX, bf16, typename Wider<TX, bf16>::type, true>(a, s);
}
// backward: dy has the forward's output type, dx the type of x
template <class TD>
static int drop_bwd(const DropArgs& a, int xt, hipStream_t s) {
  if (xt == ELEM_F32) return drop_run<TD, float, float, false>(a, s);
  if (xt == ELEM_F16) return drop_run<TD, float, f16, false>(a, s);
  return drop_run<TD, float, bf16, false>(a, s);
}
static bool drop_args(DropArgs& a, const void* x, const void* res, void* y, long n, long threshold, float scale, int site,
                      const long long* state) {
  if (!x || !y || !state || n < 1 || threshold < 0 || threshold > (1L << 32)) return false;
  a.x = x; a.res = res; a.y = y; a.state = state; a.n = n;
  a.t_hi = (unsigned)(threshold >> 16); a.t_lo = (unsigned)(threshold & 0xFFFF);
  a.scale = scale; a.site = (unsigned)site;
  a.vec = (((uintptr_t)x | (uintptr_t)res | (uintptr_t)y) & 15) == 0;
  return true;
}

}  // namespace nnz

extern "C" int nnz_dropout_forward(const void* x, int x_type, const void* residual, int residual_type, void* y, long n,
                                   long threshold, float scale, int site, const long long* state, long long* used,
                                   void* stream) {
  using namespace nnz;
  DropArgs a = {};
  if (!drop_args(a, x, residual, y, n, threshold, scale, site, state) || !elem_ok(x_type) || (residual && !elem_ok(residual_type)))
    return NNZ_EINVAL;
  a.used = used;
  hipStream_t s = (hipStream_t)stream;
  if (!residual) {
    if (x_type == ELEM_F32) return drop_run<float, float, float, false>(a, s);
    if (x_type == ELEM_F16) return drop_run<f16, float, f16, false>(a, s);
    return drop_run<bf16, float, bf16, false>(a, s);
  }
  if (x_type == ELEM_F32) return drop_res<float>(a, residual_type, s);
  if (x_type == ELEM_F16) return drop_res<f16>(a, residual_type, s);
  return drop_res<bf16>(a, residual_type, s);
}

extern "C" int nnz_dropout_backward(const void* dy, int dy_type, void* dx, int dx_type, long n, long threshold, float scale,
                                    int site, const long long* used, void* stream) {
  using namespace nnz;
  DropArgs a = {};
  if (!drop_args(a, dy, nullptr, dx, n, threshold, scale, site, used) || !elem_ok(dy_type) || !elem_ok(dx_type)) return NNZ_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  if (dy_type == ELEM_F32) return drop_bwd<float>(a, dx_type, s);
  if (dy_type == ELEM_F16) return drop_bwd<f16>(a, dx_type, s);
  return drop_bwd<bf16>(a, dx_type, s);
}
