// dc_block_norm: the norm behind a block, its gate and residual scale, and the norm in front of the next block, in one pass
// over the rows, and its backward pass.
//
// HBM-bound: forward 5 row elements of traffic per element (y, gate, residual in; r', n out), backward 8 (y, gate, residual, both
// gradients in; three out) for 4 row reductions each.  A row stays in registers between its passes: 4 elements a lane and step of 256
// columns, a row in 2 to 64 lanes of a wavefront up to 256 columns, in one wavefront up to 1 024 (backward 512), in up to 16 of them
// beyond.  Mean and deviation are taken one after the other (no E[x^2] - E[x]^2: a mean far from 0 costs no digits).  Backward, nothing of
// the forward pass is read back: r', u and both norms' statistics cost less to take again from the inputs than to load.
// The vectors' gradients: every lane sums its own columns over the rows of its workgroup, the workgroups' sums go to the workspace
// and are added in order by a second kernel (no atomics).
#include <type_traits>

#include "elem_io.h"

namespace dc {
namespace {

constexpr int V = 4;  // columns of one vector

struct NormArgs {
  int64_t n_rows;
  int32_t width, kind, act, post_norm;
  float eps, inv_width;
  int64_t y_stride, gate_stride, residual_stride;
  const float *scale, *post_w, *post_b, *pre_w, *pre_b;
  int32_t lane_bits;  // log2 of the lanes a row takes (6 where it takes whole wavefronts)
  int32_t n_waves;    // wavefronts a row takes
};

__device__ __forceinline__ float sigmoid(float x) { return fast_rcp(1.0f + fast_exp2(-x * kLog2e)); }
__device__ __forceinline__ float act_of(int act, float x) {
  return act == DC_ACT_IDENTITY ? x : act == DC_ACT_SIGMOID ? sigmoid(x) : x * sigmoid(x);
}

// One row's columns of this thread: K vectors of V, 256 * n_waves apart.  Elements beyond the width are 0 and not stored.
template <int K>
struct Part {
  float v[K][V];
};

// Where a thread's columns and rows lie.
struct Spot {
  int lane, column, step, group, n_groups;  // first column, columns between vectors, row group of the workgroup
  __device__ __forceinline__ Spot(const NormArgs& a) {
    const int wave = threadIdx.x >> 6, per_row = a.n_waves;
    if (per_row == 1) {
      lane = threadIdx.x & ((1 << a.lane_bits) - 1);
      group = threadIdx.x >> a.lane_bits;
      n_groups = blockDim.x >> a.lane_bits;
      column = lane * V;
    } else {
      lane = threadIdx.x & 63;
      group = wave / per_row;
      n_groups = (int)(blockDim.x >> 6) / per_row;
      column = (wave % per_row * 64 + lane) * V;
    }
    step = per_row * 64 * V;
  }
};

template <int K, typename T>
__device__ __forceinline__ void load_part(const T* row, const NormArgs& a, const Spot& at, Part<K>& p) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = at.column + k * at.step;
    if (c + V <= a.width) {
      load_vec<V>(row + c, p.v[k]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p.v[k][i] = c + i < a.width ? (float)row[c + i] : 0.0f;
    }
  }
}
template <int K, typename T>
__device__ __forceinline__ void store_part(T* row, const NormArgs& a, const Spot& at, const Part<K>& p) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = at.column + k * at.step;
    if (c + V <= a.width) {
      store_vec<V>(row + c, p.v[k]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c + i < a.width) row[c + i] = (T)p.v[k][i];
    }
  }
}
// a vector of the width, or a constant
template <int K>
__device__ __forceinline__ void load_weights(const float* w, float other, const NormArgs& a, const Spot& at, Part<K>& p) {
  if (w) {
    load_part<K>(w, a, at, p);
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) p.v[k][i] = other;
  }
}

// Sum over the row.  MULTI: its wavefronts meet in `scratch` (one slot a wavefront, two halves used in turn: one barrier a sum).
template <bool MULTI>
__device__ __forceinline__ float row_sum(float v, const NormArgs& a, float (*scratch)[16], int& turn) {
  v = lanes_sum(v, MULTI ? 6 : a.lane_bits);
  if constexpr (MULTI) {
    const int wave = threadIdx.x >> 6, first = wave / a.n_waves * a.n_waves;
    if ((threadIdx.x & 63) == 0) scratch[turn][wave] = v;
    __syncthreads();
    v = scratch[turn][first];
    for (int w = 1; w < a.n_waves; ++w) v += scratch[turn][first + w];
    turn ^= 1;
  }
  return v;
}

// mean (RMS: 0) and 1 / deviation of a row; elements beyond the width are 0
template <int K, bool MULTI>
__device__ __forceinline__ float2 row_stats(const Part<K>& p, const NormArgs& a, const Spot& at, float (*scratch)[16], int& turn) {
  float mean = 0.0f;
  if (a.kind == DC_NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) s += p.v[k][i];
    mean = row_sum<MULTI>(s, a, scratch, turn) * a.inv_width;
  }
  float q = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = at.column + k * at.step;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = c + i < a.width ? p.v[k][i] - mean : 0.0f;
      q = __builtin_fmaf(d, d, q);
    }
  }
  return {mean, 1.0f / sqrtf(row_sum<MULTI>(q, a, scratch, turn) * a.inv_width + a.eps)};
}

constexpr int kMaxThreads = 1024;

template <typename T, typename R, int K, bool MULTI>
__global__ __launch_bounds__(MULTI ? kMaxThreads : 256) void block_norm_kernel(NormArgs a, const T* y, const T* gate, const R* residual, R* residual_out,
                                                                              int64_t residual_out_stride, T* normed, int64_t normed_stride) {
  __shared__ float scratch[2][16];
  int turn = 0;
  const Spot at(a);
  Part<K> sc, w1, b1, w2, b2;
  load_weights(a.scale, 1.0f, a, at, sc);
  load_weights(a.post_w, 1.0f, a, at, w1);
  load_weights(a.post_b, 0.0f, a, at, b1);
  load_weights(a.pre_w, 1.0f, a, at, w2);
  load_weights(a.pre_b, 0.0f, a, at, b2);
  // (all row groups of a workgroup take the same number of turns: a MULTI row sum has barriers)
  for (int64_t first = (int64_t)blockIdx.x * at.n_groups; first < a.n_rows; first += (int64_t)gridDim.x * at.n_groups) {
    const int64_t row = first + at.group;
    const bool live = row < a.n_rows;
    const int64_t r0 = live ? row : a.n_rows - 1;  // a group without a row reads the last one
    Part<K> v, g, r;
    if (y) load_part<K>(y + r0 * a.y_stride, a, at, v);
    if (gate) load_part<K>(gate + r0 * a.gate_stride, a, at, g);
    if (residual) load_part<K>(residual + r0 * a.residual_stride, a, at, r);
    else load_weights<K>(nullptr, 0.0f, a, at, r);
    if (y) {
      float2 st{0.0f, 1.0f};
      if (a.post_norm) st = row_stats<K, MULTI>(v, a, at, scratch, turn);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = at.column + k * at.step;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float u = v.v[k][i];
          if (a.post_norm) u = __builtin_fmaf((u - st.x) * st.y, w1.v[k][i], b1.v[k][i]);
          if (gate) u *= act_of(a.act, g.v[k][i]);
          r.v[k][i] = c + i < a.width ? __builtin_fmaf(sc.v[k][i], u, r.v[k][i]) : 0.0f;
        }
      }
    }
    if (residual_out && live) store_part<K>(residual_out + row * residual_out_stride, a, at, r);
    if (normed) {
      const float2 st = row_stats<K, MULTI>(r, a, at, scratch, turn);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[k][i] = __builtin_fmaf((r.v[k][i] - st.x) * st.y, w2.v[k][i], b2.v[k][i]);
      if (live) store_part<K>(normed + row * normed_stride, a, at, r);
    }
  }
}

// The gradient g of a normalised row, in place, to that of the row: factor (g - mean(g) - hat mean(g hat)).
template <int K, bool MULTI>
__device__ __forceinline__ void norm_back(Part<K>& g, const Part<K>& hat, const NormArgs& a, float factor, float (*scratch)[16], int& turn) {
  float s = 0.0f, q = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) s += g.v[k][i], q = __builtin_fmaf(g.v[k][i], hat.v[k][i], q);
  s = a.kind == DC_NORM_LAYER ? row_sum<MULTI>(s, a, scratch, turn) * a.inv_width : 0.0f;
  q = row_sum<MULTI>(q, a, scratch, turn) * a.inv_width;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) g.v[k][i] = factor * (g.v[k][i] - s - hat.v[k][i] * q);
}

// Rows blockIdx.x * groups + group, ... ; the workgroup's sums over them, [5][width] in the order scale, post_w, post_b, pre_w, pre_b,
// go to sums[blockIdx.x].
template <typename T, typename R, int K, bool MULTI>
__global__ __launch_bounds__(MULTI ? kMaxThreads : 256) void block_norm_backward_kernel(NormArgs a, const T* y, const T* gate, const R* residual,
                                                                                       const R* g_out, int64_t g_out_stride, const T* g_normed,
                                                                                       int64_t g_normed_stride, T* g_y, T* g_gate, R* g_residual,
                                                                                       float* __restrict__ sums) {
  extern __shared__ float lds[];  // one vector per row group
  __shared__ float scratch[2][16];
  int turn = 0;
  const Spot at(a);
  Part<K> acc[5];
#pragma unroll
  for (int n = 0; n < 5; ++n) load_weights<K>(nullptr, 0.0f, a, at, acc[n]);
  for (int64_t first = (int64_t)blockIdx.x * at.n_groups; first < a.n_rows; first += (int64_t)gridDim.x * at.n_groups) {
    const int64_t row = first + at.group;
    const bool live = row < a.n_rows;
    const int64_t r0 = live ? row : a.n_rows - 1;
    const float on = live ? 1.0f : 0.0f;  // (a group without a row adds nothing)
    Part<K> hat, g, t, r, w;
    float2 st{0.0f, 1.0f};
    if (residual) load_part<K>(residual + r0 * a.residual_stride, a, at, r);
    else load_weights<K>(nullptr, 0.0f, a, at, r);
    if (g_normed) load_part<K>(g_normed + r0 * g_normed_stride, a, at, t);
    if (y) {  // hat: the normalised block output (or the output itself)
      load_part<K>(y + r0 * a.y_stride, a, at, hat);
      if (gate) load_part<K>(gate + r0 * a.gate_stride, a, at, g);
      if (a.post_norm) {
        st = row_stats<K, MULTI>(hat, a, at, scratch, turn);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) hat.v[k][i] = (hat.v[k][i] - st.x) * st.y;
      }
      Part<K> sc, b;
      load_weights(a.scale, 1.0f, a, at, sc);
      load_weights(a.post_w, 1.0f, a, at, w);
      load_weights(a.post_b, 0.0f, a, at, b);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = at.column + k * at.step;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float u = a.post_norm ? __builtin_fmaf(hat.v[k][i], w.v[k][i], b.v[k][i]) : hat.v[k][i];
          if (gate) u *= act_of(a.act, g.v[k][i]);
          r.v[k][i] = c + i < a.width ? __builtin_fmaf(sc.v[k][i], u, r.v[k][i]) : 0.0f;
        }
      }
    }
    if (g_normed) {  // r becomes the normalised r', t the gradient of r' through the norm
      const float2 st2 = row_stats<K, MULTI>(r, a, at, scratch, turn);
      load_weights(a.pre_w, 1.0f, a, at, w);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = at.column + k * at.step;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          r.v[k][i] = c + i < a.width ? (r.v[k][i] - st2.x) * st2.y : 0.0f;
          acc[3].v[k][i] = __builtin_fmaf(on * t.v[k][i], r.v[k][i], acc[3].v[k][i]);
          acc[4].v[k][i] = __builtin_fmaf(on, t.v[k][i], acc[4].v[k][i]);
          t.v[k][i] *= w.v[k][i];
        }
      }
      norm_back<K, MULTI>(t, r, a, st2.y, scratch, turn);
    } else {
      load_weights<K>(nullptr, 0.0f, a, at, t);
    }
    if (g_out) {
      load_part<K>(g_out + r0 * g_out_stride, a, at, r);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) t.v[k][i] += r.v[k][i];
    }
    if (g_residual && live) store_part<K>(g_residual + row * a.width, a, at, t);
    if (!y) continue;
    Part<K> sc, b;
    load_weights(a.scale, 1.0f, a, at, sc);
    load_weights(a.post_w, 1.0f, a, at, w);
    load_weights(a.post_b, 0.0f, a, at, b);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = at.column + k * at.step;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = a.post_norm ? __builtin_fmaf(hat.v[k][i], w.v[k][i], b.v[k][i]) : hat.v[k][i];
        const float gv = t.v[k][i] * sc.v[k][i];
        float av = 1.0f;
        if (gate) {
          const float x = g.v[k][i], s = sigmoid(x);
          av = a.act == DC_ACT_IDENTITY ? x : a.act == DC_ACT_SIGMOID ? s : x * s;
          const float slope = a.act == DC_ACT_IDENTITY ? 1.0f : a.act == DC_ACT_SIGMOID ? s * (1.0f - s) : s * (1.0f + x * (1.0f - s));
          g.v[k][i] = gv * u * slope;
        }
        const float gu = c + i < a.width ? gv * av : 0.0f;
        acc[0].v[k][i] = __builtin_fmaf(on * t.v[k][i], av * u, acc[0].v[k][i]);
        acc[1].v[k][i] = __builtin_fmaf(on * gu, hat.v[k][i], acc[1].v[k][i]);
        acc[2].v[k][i] = __builtin_fmaf(on, gu, acc[2].v[k][i]);
        t.v[k][i] = a.post_norm ? gu * w.v[k][i] : gu;
      }
    }
    if (gate && g_gate && live) store_part<K>(g_gate + row * a.width, a, at, g);
    if (g_y) {
      if (a.post_norm) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = at.column + k * at.step;
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (c + i >= a.width) hat.v[k][i] = 0.0f;
        }
        norm_back<K, MULTI>(t, hat, a, st.y, scratch, turn);
      }
      if (live) store_part<K>(g_y + row * a.width, a, at, t);
    }
  }
  if (!sums) return;
  float* own = sums + (int64_t)blockIdx.x * 5 * a.width;
#pragma unroll
  for (int n = 0; n < 5; ++n) {
    __syncthreads();
    store_part<K>(lds + at.group * a.width, a, at, acc[n]);
    __syncthreads();
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
      float s = lds[c];
      for (int q = 1; q < at.n_groups; ++q) s += lds[q * a.width + c];
      own[n * a.width + c] = s;
    }
  }
}

struct SumOut {
  float* p[5];
};

// 32 columns of one vector, the parts divided over 32 rows of threads.
__global__ __launch_bounds__(1024) void block_norm_sums_kernel(const float* __restrict__ sums, int32_t n_parts, int32_t width, SumOut out) {
  __shared__ float lds[32][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, k = blockIdx.y;
  if (!out.p[k]) return;
  float s = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (int i = part; i < n_parts; i += 32) s += sums[((int64_t)i * 5 + k) * width + c];
  }
  lds[part][lane] = s;
  __syncthreads();
  if (part == 0 && c < width) {
    for (int q = 1; q < 32; ++q) s += lds[q][lane];
    out.p[k][c] = s;
  }
}

// How many lanes, wavefronts and vectors a row takes.  Backward: 5 sums a column besides the row, so half as many columns a lane.
struct RowPlan {
  int lane_bits, n_waves, k, threads;
};
RowPlan row_plan(int32_t width, bool backward) {
  RowPlan p{6, 1, 1, 256};
  if (width <= 64 * V) {
    const int lanes = (width + V - 1) / V;
    p.lane_bits = 1;
    while ((1 << p.lane_bits) < lanes) ++p.lane_bits;
    return p;
  }
#ifndef BW_MOST
#define BW_MOST 1
#endif
#ifndef FW_MOST
#define FW_MOST 2
#endif
  const int most = backward ? BW_MOST : FW_MOST;
  while (p.k < most && width > 64 * V * p.k) p.k *= 2;
  while (width > 64 * V * p.k * p.n_waves && p.n_waves < 16) p.n_waves *= 2;
  if (width > 64 * V * p.k * p.n_waves) p.k *= 2;
  if (p.n_waves > 4) p.threads = 64 * p.n_waves;
  return p;
}

// workgroups of the backward pass = parts of the vectors' sums
int parts_of(int64_t n_rows, int32_t width) {
  const RowPlan p = row_plan(width, true);
  const int groups = p.n_waves > 1 ? p.threads / 64 / p.n_waves : p.threads >> p.lane_bits;
  int64_t most = (1 << 21) / width;  // at most 40 MB of them, ...
  most = most > 1024 ? 1024 : most < 256 ? 256 : most;
  const int64_t need = (n_rows + groups - 1) / groups;
  return (int)(need < most ? need : most);
}

int check_norm(int32_t dtype, int32_t residual_dtype, int64_t n_rows, int32_t width, int32_t kind, float eps, const void* y, int64_t y_stride,
               const void* gate, int64_t gate_stride, int32_t act, const void* residual, int64_t residual_stride) {
  DC_REQUIRE(dtype_ok(dtype), "unknown element type");
  DC_REQUIRE(residual_dtype == DC_DTYPE_F32 || residual_dtype == dtype, "the residual stream is fp32 or of the activations' type");
  DC_REQUIRE(n_rows >= 0, "negative size");
  DC_REQUIRE(width >= 1 && width <= DC_MAX_NORM_WIDTH, "width must be in [1, 8192]");
  DC_REQUIRE(kind == DC_NORM_LAYER || kind == DC_NORM_RMS, "unknown norm");
  DC_REQUIRE(act >= DC_ACT_IDENTITY && act <= DC_ACT_SILU, "unknown gate activation");
  DC_REQUIRE(eps >= 0.0f && eps <= 3.0e38f, "eps must be finite and not negative");
  DC_REQUIRE(n_rows == 0 || y || residual, "neither a block's output nor a residual");
  DC_REQUIRE(!gate || y, "a gate without a block's output");
  DC_REQUIRE(y_stride >= 0 && gate_stride >= 0 && residual_stride >= 0, "negative stride");
  DC_REQUIRE(aligned(y, dtype_size(dtype)) && aligned(gate, dtype_size(dtype)) && aligned(residual, dtype_size(residual_dtype)), "misaligned pointer");
  return DC_OK;
}

// calls f with the element types, the vectors a lane and whether a row takes several wavefronts
template <typename F>
int with_row(int32_t dtype, int32_t residual_dtype, const RowPlan& p, F&& f) {
  return with_dtype(dtype, [&](auto t) {
    auto g = [&](auto r) {
      if (p.k == 1) return p.n_waves > 1 ? f(t, r, std::integral_constant<int, 1>{}, std::true_type{}) : f(t, r, std::integral_constant<int, 1>{}, std::false_type{});
      return p.n_waves > 1 ? f(t, r, std::integral_constant<int, 2>{}, std::true_type{}) : f(t, r, std::integral_constant<int, 2>{}, std::false_type{});
    };
    return residual_dtype == dtype ? g(t) : g(f32{});
  });
}

}  // namespace
}  // namespace dc

extern "C" int64_t dc_block_norm_workspace(int64_t n_rows, int32_t width) {
  return n_rows > 0 && width > 0 ? (int64_t)dc::parts_of(n_rows, width) * 5 * width * 4 : 0;
}

extern "C" int dc_block_norm(void* stream, int32_t dtype, int32_t residual_dtype, int64_t n_rows, int32_t width, int32_t kind, float eps,
                             const void* d_y, int64_t y_stride, const void* d_gate, int64_t gate_stride, int32_t gate_act,
                             const void* d_residual, int64_t residual_stride, const float* d_scale, int32_t post_norm, const float* d_post_w,
                             const float* d_post_b, const float* d_pre_w, const float* d_pre_b, void* d_residual_out,
                             int64_t residual_out_stride, void* d_normed, int64_t normed_stride) {
  using namespace dc;
  if (int rc = check_norm(dtype, residual_dtype, n_rows, width, kind, eps, d_y, y_stride, d_gate, gate_stride, gate_act, d_residual, residual_stride)) return rc;
  DC_REQUIRE(!d_residual_out || residual_out_stride >= width, "rows of an output overlap");
  DC_REQUIRE(!d_normed || normed_stride >= width, "rows of an output overlap");
  DC_REQUIRE(aligned(d_residual_out, dtype_size(residual_dtype)) && aligned(d_normed, dtype_size(dtype)), "misaligned pointer");
  if (n_rows == 0 || (!d_residual_out && !d_normed)) return DC_OK;
  const RowPlan p = row_plan(width, false);
  const NormArgs a{n_rows, width, kind, gate_act, post_norm, eps, 1.0f / width, y_stride, gate_stride, residual_stride,
                   d_scale, d_post_w, d_post_b, d_pre_w, d_pre_b, p.lane_bits, p.n_waves};
  const int groups = p.n_waves > 1 ? p.threads / 64 / p.n_waves : p.threads >> p.lane_bits;
  const int64_t need = (n_rows + groups - 1) / groups;
  const int grid = (int)(need < 4096 ? need : 4096);
  return with_row(dtype, residual_dtype, p, [&](auto t, auto r, auto k, auto multi) {
    using T = decltype(t);
    using R = decltype(r);
    block_norm_kernel<T, R, decltype(k)::value, decltype(multi)::value><<<dim3(grid), dim3(p.threads), 0, as_stream(stream)>>>(
        a, (const T*)d_y, (const T*)d_gate, (const R*)d_residual, (R*)d_residual_out, residual_out_stride, (T*)d_normed, normed_stride);
    DC_LAUNCH_CHECK();
    return DC_OK;
  });
}

extern "C" int dc_block_norm_backward(void* stream, int32_t dtype, int32_t residual_dtype, int64_t n_rows, int32_t width, int32_t kind, float eps,
                                      const void* d_y, int64_t y_stride, const void* d_gate, int64_t gate_stride, int32_t gate_act,
                                      const void* d_residual, int64_t residual_stride, const float* d_scale, int32_t post_norm,
                                      const float* d_post_w, const float* d_post_b, const float* d_pre_w, const void* d_grad_residual_out,
                                      int64_t grad_residual_out_stride, const void* d_grad_normed, int64_t grad_normed_stride, void* d_grad_y,
                                      void* d_grad_gate, void* d_grad_residual, float* d_grad_scale, float* d_grad_post_w, float* d_grad_post_b,
                                      float* d_grad_pre_w, float* d_grad_pre_b, void* d_workspace, int64_t workspace_bytes) {
  using namespace dc;
  if (int rc = check_norm(dtype, residual_dtype, n_rows, width, kind, eps, d_y, y_stride, d_gate, gate_stride, gate_act, d_residual, residual_stride)) return rc;
  DC_REQUIRE(grad_residual_out_stride >= 0 && grad_normed_stride >= 0, "negative stride");
  DC_REQUIRE(aligned(d_grad_residual_out, dtype_size(residual_dtype)) && aligned(d_grad_residual, dtype_size(residual_dtype)) &&
                 aligned(d_grad_normed, dtype_size(dtype)) && aligned(d_grad_y, dtype_size(dtype)) && aligned(d_grad_gate, dtype_size(dtype)),
             "misaligned pointer");
  DC_REQUIRE(workspace_bytes >= dc_block_norm_workspace(n_rows, width) && (n_rows == 0 || d_workspace) && aligned(d_workspace, 16), "workspace too small");
  const RowPlan p = row_plan(width, true);
  const NormArgs a{n_rows, width, kind, gate_act, post_norm, eps, 1.0f / width, y_stride, gate_stride, residual_stride,
                   d_scale, d_post_w, d_post_b, d_pre_w, nullptr, p.lane_bits, p.n_waves};
  const int groups = p.n_waves > 1 ? p.threads / 64 / p.n_waves : p.threads >> p.lane_bits;
  const int grid = parts_of(n_rows, width);
  const bool any = d_grad_scale || d_grad_post_w || d_grad_post_b || d_grad_pre_w || d_grad_pre_b;
  return with_row(dtype, residual_dtype, p, [&](auto t, auto r, auto k, auto multi) {
    using T = decltype(t);
    using R = decltype(r);
    if (grid > 0) {
      auto kernel = block_norm_backward_kernel<T, R, decltype(k)::value, decltype(multi)::value>;
      DC_SET_MAX_SMEM_ONCE_PER_DEVICE(kernel, DC_MAX_NORM_WIDTH * 4);
      kernel<<<dim3(grid), dim3(p.threads), groups * width * 4, as_stream(stream)>>>(
          a, (const T*)d_y, (const T*)d_gate, (const R*)d_residual, (const R*)d_grad_residual_out, grad_residual_out_stride,
          (const T*)d_grad_normed, grad_normed_stride, (T*)d_grad_y, (T*)d_grad_gate, (R*)d_grad_residual, any ? (float*)d_workspace : nullptr);
      DC_LAUNCH_CHECK();
    }
    if (any) {
      block_norm_sums_kernel<<<dim3((width + 31) / 32, 5), dim3(1024), 0, as_stream(stream)>>>(
          (const float*)d_workspace, grid, width, SumOut{{d_grad_scale, d_grad_post_w, d_grad_post_b, d_grad_pre_w, d_grad_pre_b}});
      DC_LAUNCH_CHECK();
    }
    return DC_OK;
  });
}
