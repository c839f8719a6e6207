// Element access of the operators that take fp32, fp16 and bf16 tensors: V consecutive elements <-> fp32 registers.
// Widening is exact; narrowing rounds once, to nearest even (v_cvt_f16_f32 / v_cvt_pk_bf16_f32).
#pragma once
#include "common.hpp"

typedef __bf16 bf16;

namespace nnz {

// element types as they cross the C boundary
enum ElemType { ELEM_F32 = 0, ELEM_F16 = 1, ELEM_BF16 = 2 };
inline int elem_size(int t) { return t == ELEM_F32 ? 4 : 2; }
inline bool elem_ok(int t) { return t == ELEM_F32 || t == ELEM_F16 || t == ELEM_BF16; }

template <class T, int V>
using ElemVec = T __attribute__((ext_vector_type(V)));

// V elements at p, p aligned to min(16, V * sizeof(T)) bytes: accesses of at most 16 bytes
template <class T, int V>
__device__ __forceinline__ void ld_elems(const T* __restrict__ p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = (float)p[0];
  } else {
    constexpr int W = V * (int)sizeof(T) <= 16 ? V : 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < V; i += W) {
      const ElemVec<T, W> r = *reinterpret_cast<const ElemVec<T, W>*>(p + i);
#pragma unroll
      for (int j = 0; j < W; ++j) v[i + j] = (float)r[j];
    }
  }
}
template <class T, int V>
__device__ __forceinline__ void st_elems(T* __restrict__ p, const float (&v)[V]) {
  if constexpr (V == 1) {
    p[0] = (T)v[0];
  } else {
    constexpr int W = V * (int)sizeof(T) <= 16 ? V : 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < V; i += W) {
      ElemVec<T, W> r;
#pragma unroll
      for (int j = 0; j < W; ++j) r[j] = (T)v[i + j];
      *reinterpret_cast<ElemVec<T, W>*>(p + i) = r;
    }
  }
}

// one element of a type known at run time (state and parameter reads, off the hot loops)
__device__ __forceinline__ float ld_any(const void* p, long i, int t) {
  if (t == ELEM_F32) return ((const float*)p)[i];
  if (t == ELEM_F16) return (float)((const f16*)p)[i];
  return (float)((const bf16*)p)[i];
}
__device__ __forceinline__ void st_any(void* p, long i, int t, float v) {
  if (t == ELEM_F32) ((float*)p)[i] = v;
  else if (t == ELEM_F16) ((f16*)p)[i] = (f16)v;
  else ((bf16*)p)[i] = (bf16)v;
}

// exp and the logistic function on the hardware's 2^x and reciprocal (1 ulp each): exp(x) is off by |x| * 2^-24 relative, for
// the product x * log2(e) is rounded once
__device__ __forceinline__ float exp_hw(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float sigmoid_hw(float x) { return __builtin_amdgcn_rcpf(1.f + exp_hw(-x)); }

}  // namespace nnz
