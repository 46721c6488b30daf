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

// ... at any element's address (gfx950 takes unaligned vector accesses to global memory)
template <typename T, int N>
struct loose_vec {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

// N consecutive elements at p as fp32
template <int N, typename T>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = (float)p[0];
  } else {
    const typename loose_vec<T, N>::type r = *reinterpret_cast<const typename loose_vec<T, N>::type*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)r[i];
  }
}

// ... and back, each rounded once to nearest even (the only rounding below fp32 these kernels do)
template <int N, typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[N]) {
  if constexpr (N == 1) {
    p[0] = (T)v[0];
  } else {
    typename loose_vec<T, N>::type r;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = (T)v[i];
    *reinterpret_cast<typename loose_vec<T, N>::type*>(p) = r;
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

// p = min(sigmoid(f), 1 - sigmoid(f)) = 1 / (1 + exp(|f|)): of the two weights of a gate the one that has full relative accuracy; the
// other is 1 - p.
__device__ __forceinline__ float gate_minor(float f) { return fast_rcp(1.0f + fast_exp2(__builtin_fabsf(f) * kLog2e)); }

// The value of another lane by a fixed pattern of lanes, without a trip through LDS.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E, kMirror8 = 0x141, kMirror16 = 0x140;  // quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror, row_mirror

// op over the 2^bits neighbouring lanes (bits 0 .. 6, uniform): the same bits in every one of them, in a fixed order.  After a step
// all lanes of a group of 2, 4, 8, 16 hold its value, so that a mirror image is as good as a swap; rows of 16 and halves of 32 are
// exchanged by the permlane swaps (both results together are the two halves).
template <typename Op>
__device__ __forceinline__ float lanes_reduce(float v, int bits, Op op) {
  if (bits > 0) v = op(v, dpp<kSwap1>(v));
  if (bits > 1) v = op(v, dpp<kSwap2>(v));
  if (bits > 2) v = op(v, dpp<kMirror8>(v));
  if (bits > 3) v = op(v, dpp<kMirror16>(v));
  if (bits > 4) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if (bits > 5) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}
__device__ __forceinline__ float lanes_sum(float v, int bits) {
  return lanes_reduce(v, bits, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float lanes_max(float v, int bits) {
  return lanes_reduce(v, bits, [](float a, float b) { return __builtin_fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float v) { return lanes_sum(v, 6); }

}  // namespace dc
