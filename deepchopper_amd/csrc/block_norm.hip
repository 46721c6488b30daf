// dc_block_norm: the norm behind a block, its gate and residual scale, and the norm in front of the next block, in one pass
// over the rows, and its backward pass.
#include "elem_io.h"

namespace dc {
namespace {

constexpr int kRowThreads = 256;

struct NormArgs {
  int64_t n_rows;
  int32_t width, kind, act, post_norm;
  float eps;
  int64_t y_stride, gate_stride, residual_stride;
  const float *scale, *post_w, *post_b, *pre_w, *pre_b;
};

__device__ __forceinline__ float sigmoid(float x) { return fast_rcp(1.0f + fast_exp2(-x * kLog2e)); }
__device__ __forceinline__ float act_of(int act, float x) {
  return act == DC_ACT_IDENTITY ? x : act == DC_ACT_SIGMOID ? sigmoid(x) : x * sigmoid(x);
}
// d act / dx
__device__ __forceinline__ float slope_of(int act, float x) {
  const float s = sigmoid(x);
  return act == DC_ACT_IDENTITY ? 1.0f : act == DC_ACT_SIGMOID ? s * (1.0f - s) : s * (1.0f + x * (1.0f - s));
}

__device__ float block_sum(float v, float* scratch) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
}

// mean (0 for RMS) and 1 / deviation of the block's row, held in LDS
__device__ float2 row_stats(const float* row, const NormArgs& a, float* scratch) {
  float mean = 0.0f;
  if (a.kind == DC_NORM_LAYER) {
    float s = 0.0f;
    for (int c = threadIdx.x; c < a.width; c += kRowThreads) s += row[c];
    mean = block_sum(s, scratch) / a.width;
  }
  float q = 0.0f;
  for (int c = threadIdx.x; c < a.width; c += kRowThreads) q += (row[c] - mean) * (row[c] - mean);
  return {mean, 1.0f / sqrtf(block_sum(q, scratch) / a.width + a.eps)};
}

// A block per row.
template <typename T, typename R>
__global__ __launch_bounds__(kRowThreads) void block_norm_kernel(NormArgs a, const T* y, const T* gate, const R* residual, R* residual_out,
                                                                 int64_t residual_out_stride, T* normed, int64_t normed_stride) {
  extern __shared__ float row[];
  __shared__ float scratch[4];
  for (int64_t i = blockIdx.x; i < a.n_rows; i += gridDim.x) {
    float2 st{0.0f, 1.0f};
    __syncthreads();
    if (y) {
      for (int c = threadIdx.x; c < a.width; c += kRowThreads) row[c] = (float)y[i * a.y_stride + c];
      if (a.post_norm) st = row_stats(row, a, scratch);
    }
    for (int c = threadIdx.x; c < a.width; c += kRowThreads) {
      float r = residual ? (float)residual[i * a.residual_stride + c] : 0.0f;
      if (y) {
        float v = row[c];
        if (a.post_norm) v = (v - st.x) * st.y * (a.post_w ? a.post_w[c] : 1.0f) + (a.post_b ? a.post_b[c] : 0.0f);
        if (gate) v *= act_of(a.act, (float)gate[i * a.gate_stride + c]);
        r += (a.scale ? a.scale[c] : 1.0f) * v;
      }
      row[c] = r;
      if (residual_out) residual_out[i * residual_out_stride + c] = (R)r;
    }
    if (normed) {
      st = row_stats(row, a, scratch);
      for (int c = threadIdx.x; c < a.width; c += kRowThreads)
        normed[i * normed_stride + c] = (T)((row[c] - st.x) * st.y * (a.pre_w ? a.pre_w[c] : 1.0f) + (a.pre_b ? a.pre_b[c] : 0.0f));
    }
  }
}

// the gradient g of a normalised row, in place, to that of the row: factor (g - mean(g) - hat mean(g hat))
__device__ void norm_back(float* g, const float* hat, const NormArgs& a, float factor, float* scratch) {
  float s = 0.0f, q = 0.0f;
  for (int c = threadIdx.x; c < a.width; c += kRowThreads) s += g[c], q += g[c] * hat[c];
  s = a.kind == DC_NORM_LAYER ? block_sum(s, scratch) / a.width : 0.0f;
  q = block_sum(q, scratch) / a.width;
  for (int c = threadIdx.x; c < a.width; c += kRowThreads) g[c] = factor * (g[c] - s - hat[c] * q);
}

// A block for every gridDim.x-th row; its sums over them, [5][width] in the order scale, post_w, post_b, pre_w, pre_b, go to `sums`.
template <typename T, typename R>
__global__ __launch_bounds__(kRowThreads) void block_norm_backward_kernel(NormArgs a, const T* y, const T* gate, const R* residual,
                                                                          const R* g_out, int64_t g_out_stride, const T* g_normed,
                                                                          int64_t g_normed_stride, T* g_y, T* g_gate, R* g_residual, float* sums) {
  extern __shared__ float lds[];
  __shared__ float scratch[4];
  float *hat = lds, *t = lds + a.width;  // normalised r', gradient of r'
  float* own = sums + (int64_t)blockIdx.x * 5 * a.width;
  for (int c = threadIdx.x; c < 5 * a.width; c += kRowThreads) own[c] = 0.0f;
  for (int64_t i = blockIdx.x; i < a.n_rows; i += gridDim.x) {
    __syncthreads();
    float2 st{0.0f, 1.0f}, st2{0.0f, 1.0f};
    if (y && a.post_norm) {
      for (int c = threadIdx.x; c < a.width; c += kRowThreads) hat[c] = (float)y[i * a.y_stride + c];
      st = row_stats(hat, a, scratch);
    }
    for (int c = threadIdx.x; c < a.width; c += kRowThreads) {
      float r = residual ? (float)residual[i * a.residual_stride + c] : 0.0f;
      if (y) {
        float v = (float)y[i * a.y_stride + c];
        if (a.post_norm) v = (v - st.x) * st.y * (a.post_w ? a.post_w[c] : 1.0f) + (a.post_b ? a.post_b[c] : 0.0f);
        if (gate) v *= act_of(a.act, (float)gate[i * a.gate_stride + c]);
        r += (a.scale ? a.scale[c] : 1.0f) * v;
      }
      hat[c] = r;
      t[c] = 0.0f;
    }
    if (g_normed) {
      st2 = row_stats(hat, a, scratch);
      for (int c = threadIdx.x; c < a.width; c += kRowThreads) {
        const float g = (float)g_normed[i * g_normed_stride + c];
        hat[c] = (hat[c] - st2.x) * st2.y;
        own[3 * a.width + c] += g * hat[c];
        own[4 * a.width + c] += g;
        t[c] = g * (a.pre_w ? a.pre_w[c] : 1.0f);
      }
      norm_back(t, hat, a, st2.y, scratch);
    }
    for (int c = threadIdx.x; c < a.width; c += kRowThreads) {
      if (g_out) t[c] += (float)g_out[i * g_out_stride + c];
      if (g_residual) g_residual[i * a.width + c] = (R)t[c];
    }
    if (!y) continue;
    for (int c = threadIdx.x; c < a.width; c += kRowThreads) {
      const float x = (float)y[i * a.y_stride + c], w = a.post_norm && a.post_w ? a.post_w[c] : 1.0f;
      const float h = a.post_norm ? (x - st.x) * st.y : x, u = a.post_norm ? h * w + (a.post_b ? a.post_b[c] : 0.0f) : x;
      const float gt = gate ? (float)gate[i * a.gate_stride + c] : 0.0f, av = gate ? act_of(a.act, gt) : 1.0f;
      const float gv = t[c] * (a.scale ? a.scale[c] : 1.0f), gu = gv * av;
      own[c] += t[c] * av * u;
      own[a.width + c] += gu * h;
      own[2 * a.width + c] += gu;
      if (gate && g_gate) g_gate[i * a.width + c] = (T)(gv * u * slope_of(a.act, gt));
      hat[c] = h;
      t[c] = gu * w;
    }
    if (!g_y) continue;
    if (a.post_norm) norm_back(t, hat, a, st.y, scratch);
    for (int c = threadIdx.x; c < a.width; c += kRowThreads) g_y[i * a.width + c] = (T)t[c];
  }
}

struct SumOut {
  float* p[5];
};

__global__ __launch_bounds__(256) void block_norm_sums_kernel(const float* sums, int32_t n_parts, int32_t width, SumOut out) {
  const int c = blockIdx.x * 256 + threadIdx.x, k = blockIdx.y;
  if (c >= width || !out.p[k]) return;
  float s = 0.0f;
  for (int i = 0; i < n_parts; ++i) s += sums[((int64_t)i * 5 + k) * width + c];
  out.p[k][c] = s;
}

constexpr int kParts = 512;  // blocks of the backward pass = partial sums
int parts_of(int64_t n_rows) { return (int)(n_rows < kParts ? n_rows : kParts); }

int check_norm(int32_t dtype, int32_t residual_dtype, int64_t n_rows, int32_t width, int32_t kind, float eps, const void* y, int64_t y_stride,
               const void* gate, int64_t gate_stride, int32_t act, const void* residual, int64_t residual_stride) {
  DC_REQUIRE(dtype_ok(dtype), "unknown element type");
  DC_REQUIRE(residual_dtype == DC_DTYPE_F32 || residual_dtype == dtype, "the residual stream is fp32 or of the activations' type");
  DC_REQUIRE(n_rows >= 0, "negative size");
  DC_REQUIRE(width >= 1 && width <= DC_MAX_NORM_WIDTH, "width must be in [1, 16384]");
  DC_REQUIRE(kind == DC_NORM_LAYER || kind == DC_NORM_RMS, "unknown norm");
  DC_REQUIRE(act >= DC_ACT_IDENTITY && act <= DC_ACT_SILU, "unknown gate activation");
  DC_REQUIRE(eps >= 0.0f && eps <= 3.0e38f, "eps must be finite and not negative");
  DC_REQUIRE(n_rows == 0 || y || residual, "neither a block's output nor a residual");
  DC_REQUIRE(!gate || y, "a gate without a block's output");
  DC_REQUIRE(y_stride >= 0 && gate_stride >= 0 && residual_stride >= 0, "negative stride");
  DC_REQUIRE(aligned(y, dtype_size(dtype)) && aligned(gate, dtype_size(dtype)) && aligned(residual, dtype_size(residual_dtype)), "misaligned pointer");
  return DC_OK;
}

template <typename F>
int with_types(int32_t dtype, int32_t residual_dtype, F&& f) {
  return with_dtype(dtype, [&](auto t) { return residual_dtype == dtype ? f(t, t) : f(t, f32{}); });
}

}  // namespace
}  // namespace dc

extern "C" int64_t dc_block_norm_workspace(int64_t n_rows, int32_t width) {
  return n_rows > 0 && width > 0 ? (int64_t)dc::parts_of(n_rows) * 5 * width * 4 : 0;
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
  const NormArgs a{n_rows, width, kind, gate_act, post_norm, eps, y_stride, gate_stride, residual_stride, d_scale, d_post_w, d_post_b, d_pre_w, d_pre_b};
  const int grid = (int)(n_rows < 65536 ? n_rows : 65536);
  return with_types(dtype, residual_dtype, [&](auto t, auto r) {
    using T = decltype(t);
    using R = decltype(r);
    DC_SET_MAX_SMEM_ONCE_PER_DEVICE((block_norm_kernel<T, R>), DC_MAX_NORM_WIDTH * 4);
    block_norm_kernel<T, R><<<dim3(grid), dim3(kRowThreads), width * 4, as_stream(stream)>>>(
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
  const NormArgs a{n_rows, width, kind, gate_act, post_norm, eps, y_stride, gate_stride, residual_stride, d_scale, d_post_w, d_post_b, d_pre_w, nullptr};
  const int grid = parts_of(n_rows);
  return with_types(dtype, residual_dtype, [&](auto t, auto r) {
    using T = decltype(t);
    using R = decltype(r);
    if (grid > 0) {
      DC_SET_MAX_SMEM_ONCE_PER_DEVICE((block_norm_backward_kernel<T, R>), DC_MAX_NORM_WIDTH * 8);
      block_norm_backward_kernel<T, R><<<dim3(grid), dim3(kRowThreads), width * 8, as_stream(stream)>>>(
          a, (const T*)d_y, (const T*)d_gate, (const R*)d_residual, (const R*)d_grad_residual_out, grad_residual_out_stride,
          (const T*)d_grad_normed, grad_normed_stride, (T*)d_grad_y, (T*)d_grad_gate, (R*)d_grad_residual, (float*)d_workspace);
      DC_LAUNCH_CHECK();
    }
    block_norm_sums_kernel<<<dim3((width + 255) / 256, 5), dim3(256), 0, as_stream(stream)>>>(
        (const float*)d_workspace, grid, width, SumOut{{d_grad_scale, d_grad_post_w, d_grad_post_b, d_grad_pre_w, d_grad_pre_b}});
    DC_LAUNCH_CHECK();
    return DC_OK;
  });
}
