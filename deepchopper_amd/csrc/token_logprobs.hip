// dc_token_logprobs: log probabilities of given tokens, entropy and top alternatives of rows of logits, and their gradient.
#include "elem_io.h"

namespace dc {
namespace {

struct Tokens {
  const void* p;  // or null: no token, no row is skipped
  int32_t type;
  int64_t ignore;
};

__device__ __forceinline__ int64_t token_at(const Tokens& t, int64_t i) {
  switch (t.type) {
    case DC_TOKENS_I8: return ((const int8_t*)t.p)[i];
    case DC_TOKENS_U8: return ((const uint8_t*)t.p)[i];
    case DC_TOKENS_I32: return ((const int32_t*)t.p)[i];
    default: return ((const int64_t*)t.p)[i];
  }
}

// a float's place in ascending order as an unsigned number: -0 with +0, every NaN above +inf, none 0xffffffff
__device__ __forceinline__ uint32_t order_key(float z) {
  if (!(z == z)) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(z + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct RowStats {
  float m, log_sum, entropy;  // max, log sum exp(z - m), entropy
};

// One wavefront per row, three passes over it.
template <typename T>
__device__ RowStats row_stats(const T* z, int n) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  bool bad = false;
  for (int j = lane; j < n; j += 64) {
    const float v = (float)z[j];
    bad |= !(v == v) || v == INFINITY;
    m = fmaxf(m, v);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  if (__any(bad)) return {__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
  if (m == -INFINITY) return {m, 0.0f, 0.0f};
  // the sum without the largest term's 1, so that log S = log1p(...) keeps its digits where one class has all the weight
  float s = 0.0f, u = 0.0f, ones = 0.0f;
  for (int j = lane; j < n; j += 64) {
    const float d = (float)z[j] - m, e = fast_exp2(d * kLog2e);
    if (d == 0.0f) {
      ones += 1.0f;
    } else if (e > 0.0f) {
      s += e;
      u += e * d;
    }
  }
  s = wave_sum(s) + (wave_sum(ones) - 1.0f);
  u = wave_sum(u);
  const float log_sum = log1pf(s);
  return {m, log_sum, log_sum - u / (1.0f + s)};
}

__device__ __forceinline__ float log_prob(const RowStats& r, float z) {
  return r.m == -INFINITY ? -INFINITY : (z - r.m) - r.log_sum;
}

template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_kernel(const T* __restrict__ logits, int64_t n_rows, int32_t n, int64_t ld, Tokens tok, int32_t n_top,
                                                             float* logprob, float* entropy, float* stats, int32_t* top_ids, float* top_logprob) {
  const int lane = threadIdx.x & 63;
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < n_rows; i += (int64_t)gridDim.x * 4) {
    const int64_t t = tok.p ? token_at(tok, i) : 0;
    const bool skip = tok.p && t == tok.ignore;
    const T* z = logits + i * ld;
    RowStats r{0.0f, 0.0f, 0.0f};
    if (!skip) r = row_stats(z, n);
    if (lane == 0) {
      if (logprob && tok.p) logprob[i] = skip ? 0.0f : t >= 0 && t < n ? log_prob(r, (float)z[t]) : __builtin_nanf("");
      if (entropy) entropy[i] = r.entropy;
      if (stats) stats[3 * i] = r.m, stats[3 * i + 1] = r.log_sum, stats[3 * i + 2] = r.entropy;
    }
    uint64_t below = ~0ull;  // (key, ~class) of the alternative found last
    for (int k = 0; k < n_top; ++k) {
      uint64_t best = 0;
      if (!skip) {
        for (int j = lane; j < n; j += 64) {
          const uint64_t c = (uint64_t)order_key((float)z[j]) << 32 | (uint32_t)~j;
          if (c < below && c > best) best = c;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const uint64_t o = __shfl_xor(best, d, 64);
          if (o > best) best = o;
        }
      }
      below = best;
      if (lane == 0) {
        const int id = skip ? -1 : (int)~(uint32_t)best;
        top_ids[i * n_top + k] = id;
        top_logprob[i * n_top + k] = skip ? 0.0f : log_prob(r, (float)z[id]);
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_backward_kernel(const T* logits, int64_t n_rows, int32_t n, int64_t ld, Tokens tok,
                                                                      const float* stats, const float* g_logprob, const float* g_entropy, T* out,
                                                                      int64_t ld_out) {
  const int lane = threadIdx.x & 63;
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < n_rows; i += (int64_t)gridDim.x * 4) {
    const int64_t t = tok.p ? token_at(tok, i) : -1;
    const bool skip = tok.p && t == tok.ignore;
    const T* z = logits + i * ld;
    RowStats r{0.0f, 0.0f, 0.0f};
    if (!skip) r = stats ? RowStats{stats[3 * i], stats[3 * i + 1], stats[3 * i + 2]} : row_stats(z, n);
    const float g = g_logprob ? g_logprob[i] : 0.0f, h = g_entropy ? g_entropy[i] : 0.0f;
    const bool wrong = g_logprob && !(t >= 0 && t < n);
    for (int j = lane; j < n; j += 64) {
      float d = 0.0f;
      if (!skip && r.m != -INFINITY) {
        const float lp = log_prob(r, (float)z[j]), p = fast_exp2(lp * kLog2e);
        d = p > 0.0f || p != p ? -p * (g + h * (lp + r.entropy)) : 0.0f;
        if (j == t) d += g;
        if (wrong) d = __builtin_nanf("");
      }
      out[i * ld_out + j] = (T)d;
    }
  }
}

int check_logits(const void* logits, int32_t dtype, int64_t n_rows, int32_t n_classes, int64_t row_stride, const void* tokens, int32_t token_type) {
  DC_REQUIRE(dtype_ok(dtype), "unknown element type");
  DC_REQUIRE(n_rows >= 0 && n_classes >= 1, "negative size");
  DC_REQUIRE(n_rows == 0 || logits, "null pointer");
  DC_REQUIRE(row_stride >= 0, "negative stride");
  DC_REQUIRE(token_type >= DC_TOKENS_I8 && token_type <= DC_TOKENS_I64, "unknown token type");
  DC_REQUIRE(aligned(logits, dtype_size(dtype)), "misaligned pointer");
  DC_REQUIRE(aligned(tokens, token_type == DC_TOKENS_I64 ? 8 : token_type == DC_TOKENS_I32 ? 4 : 1), "misaligned pointer");
  return DC_OK;
}

unsigned row_grid(int64_t n_rows) {
  const int64_t b = (n_rows + 3) / 4;
  return (unsigned)(b < (1 << 20) ? b : 1 << 20);
}

}  // namespace
}  // namespace dc

extern "C" int64_t dc_token_logprobs_workspace(int64_t, int32_t, int32_t) { return 0; }

extern "C" int dc_token_logprobs(void* stream, const void* d_logits, int32_t dtype, int64_t n_rows, int32_t n_classes, int64_t row_stride,
                                 const void* d_tokens, int32_t token_type, int64_t ignore_token, int32_t n_top, float* d_logprob, float* d_entropy,
                                 float* d_stats, int32_t* d_top_ids, float* d_top_logprob, void* d_workspace, int64_t workspace_bytes) {
  using namespace dc;
  if (int rc = check_logits(d_logits, dtype, n_rows, n_classes, row_stride, d_tokens, token_type)) return rc;
  DC_REQUIRE(n_top >= 0 && n_top <= n_classes && n_top <= DC_MAX_TOP, "n_top must be in [0, min(n_classes, 32)]");
  DC_REQUIRE(n_rows == 0 || n_top == 0 || (d_top_ids && d_top_logprob), "null pointer");
  (void)d_workspace, (void)workspace_bytes;
  if (n_rows == 0) return DC_OK;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    token_logprobs_kernel<T><<<dim3(row_grid(n_rows)), dim3(256), 0, as_stream(stream)>>>((const T*)d_logits, n_rows, n_classes, row_stride,
                                                                                          Tokens{d_tokens, token_type, ignore_token}, n_top, d_logprob,
                                                                                          d_entropy, d_stats, d_top_ids, d_top_logprob);
    DC_LAUNCH_CHECK();
    return DC_OK;
  });
}

extern "C" int dc_token_logprobs_backward(void* stream, const void* d_logits, int32_t dtype, int64_t n_rows, int32_t n_classes, int64_t row_stride,
                                          const void* d_tokens, int32_t token_type, int64_t ignore_token, const float* d_stats,
                                          const float* d_grad_logprob, const float* d_grad_entropy, void* d_grad_logits, int64_t grad_stride) {
  using namespace dc;
  if (int rc = check_logits(d_logits, dtype, n_rows, n_classes, row_stride, d_tokens, token_type)) return rc;
  DC_REQUIRE(n_rows == 0 || d_grad_logits, "null pointer");
  DC_REQUIRE(d_tokens || !d_grad_logprob, "a gradient of log probabilities without tokens");
  DC_REQUIRE(n_rows == 0 || d_stats || n_classes < DC_STATS_FROM, "the forward call's statistics are needed from 513 classes on");
  DC_REQUIRE(grad_stride >= n_classes, "rows of the output overlap");
  DC_REQUIRE(aligned(d_grad_logits, dtype_size(dtype)), "misaligned pointer");
  if (n_rows == 0) return DC_OK;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    token_logprobs_backward_kernel<T><<<dim3(row_grid(n_rows)), dim3(256), 0, as_stream(stream)>>>(
        (const T*)d_logits, n_rows, n_classes, row_stride, Tokens{d_tokens, token_type, ignore_token}, d_stats, d_grad_logprob, d_grad_entropy,
        (T*)d_grad_logits, grad_stride);
    DC_LAUNCH_CHECK();
    return DC_OK;
  });
}
