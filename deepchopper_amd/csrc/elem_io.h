// Element types, vector loads / stores and wavefront reductions shared by the sequence-layer kernels
// (gated_scan.hip, block_norm.hip, token_logprobs.hip).
#pragma once
#include "dc_common.h"

namespace dc {

using f32 = float;
using f16 = _Float16;
using bf16 = __bf16;

template <typename T, int N>
using vec_t = T __attribute__((ext_vector_type(N)));

// N consecutive elements at p (aligned to N * sizeof(T)) as fp32
template <int N, typename T>
__device__ __forceinline__ void load_vec(const T* __restrict__ p, float (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = (float)p[0];
  } else {
    const vec_t<T, N> r = *reinterpret_cast<const vec_t<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)r[i];
  }
}

// ... and back, each rounded once to nearest even (the only rounding below fp32 these kernels do)
template <int N, typename T>
__device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&v)[N]) {
  if constexpr (N == 1) {
    p[0] = (T)v[0];
  } else {
    vec_t<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = (T)v[i];
    *reinterpret_cast<vec_t<T, N>*>(p) = r;
  }
}

static inline size_t dtype_size(int32_t dtype) { return dtype == DC_DTYPE_F32 ? 4 : 2; }
static inline bool dtype_ok(int32_t dtype) { return dtype == DC_DTYPE_F32 || dtype == DC_DTYPE_F16 || dtype == DC_DTYPE_BF16; }
static inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// calls f with a value of the element type `dtype` names
template <typename F>
static inline int with_dtype(int32_t dtype, F&& f) {
  switch (dtype) {
    case DC_DTYPE_F32: return f(f32{});
    case DC_DTYPE_F16: return f(f16{});
    default: return f(bf16{});
  }
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32: 1 ulp, 0 below 2^-126
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }    // v_rcp_f32: 1 ulp
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// p = min(sigmoid(f), 1 - sigmoid(f)) = e / (1 + e) with e = exp(-|f|): of the two weights of a gate the one that has full
// relative accuracy; the other is 1 - p.
__device__ __forceinline__ float gate_minor(float f) {
  const float e = fast_exp2(-__builtin_fabsf(f) * kLog2e);
  return e * fast_rcp(1.0f + e);
}

// sum over the 64 lanes, the same bits in every lane (butterfly: fixed order)
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
  return v;
}

}  // namespace dc
