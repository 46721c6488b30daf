// dc_gated_scan: h_t = a_t h_(t-1) + (1 - a_t) x_t with a = sigmoid(f), per channel of every sequence, and its backward pass.
//
// A gate has two weights, a and 1 - a, and fp32 holds only the smaller of them to full relative accuracy:
// p = min(a, 1 - a) = e / (1 + e), e = exp(-|f|).  Each step is written as a move by p from the one operand towards the other,
//   f > 0: h' = h + p (x - h)        f <= 0: h' = x + p (h - x)
// so a gate that keeps 99.99 % for thousands of tokens loses no more than one that forgets at once (a * h + (1 - a) * x with
// a rounded to 1 - 2^-24 steps drifts by 2^-25 / (1 - a)).  p = 0 selects its operand: a gate of +-inf never touches the other.
#include "elem_io.h"

namespace dc {
namespace {

constexpr int kTile = 128;  // tokens between two states of d_saved

struct ScanArgs {
  const int64_t* begin;  // or null: dense sequences of max_len tokens
  const int64_t* end;
  int64_t n_tokens, max_len;
  int32_t n_seqs, n_channels, reverse;
};

// [b, e) of sequence s; false: the sequence breaks the contract
__device__ __forceinline__ bool seq_range(const ScanArgs& a, int s, int64_t* b, int64_t* e) {
  *b = a.begin ? a.begin[s] : s * a.max_len;
  *e = a.end ? a.end[s] : *b + a.max_len;
  return *b >= 0 && *e >= *b && *e <= a.n_tokens && *e - *b <= a.max_len;
}

__device__ __forceinline__ float step(float h, float x, float f) {
  const float p = gate_minor(f);
  const float base = f > 0.0f ? h : x, other = f > 0.0f ? x : h;
  return p == 0.0f ? base : __builtin_fmaf(p, other - base, base);
}

// A thread per channel of a sequence.
template <typename T>
__global__ __launch_bounds__(64) void scan_walk_kernel(ScanArgs a, const T* __restrict__ x, int64_t ldx, const T* __restrict__ f, int64_t ldf,
                                                       const float* h0, T* __restrict__ y, int64_t ldy, float* h_last,
                                                       float* __restrict__ saved) {
  const int blocks = (a.n_channels + 63) / 64;
  const int s = blockIdx.x / blocks, c = blockIdx.x % blocks * 64 + threadIdx.x;
  if (c >= a.n_channels) return;
  int64_t b, e;
  const bool ok = seq_range(a, s, &b, &e);
  float h = h0 ? h0[(int64_t)s * a.n_channels + c] : 0.0f;
  if (ok) {
    for (int64_t i = 0; i < e - b; ++i) {
      const int64_t t = a.reverse ? e - 1 - i : b + i;
      if (saved && (a.reverse ? t % kTile == kTile - 1 : t % kTile == 0)) saved[t / kTile * a.n_channels + c] = h;
      h = step(h, (float)x[t * ldx + c], (float)f[t * ldf + c]);
      y[t * ldy + c] = (T)h;
    }
  }
  if (h_last) h_last[(int64_t)s * a.n_channels + c] = ok ? h : __builtin_nanf("");
}

// A thread per channel of a sequence, tile by tile from its last token on: the states of a tile again from the one it was
// entered with, kept in LDS, then the gradients against the direction of the recurrence.
template <typename T>
__global__ __launch_bounds__(64) void scan_walk_backward_kernel(ScanArgs a, const T* __restrict__ x, int64_t ldx, const T* __restrict__ f, int64_t ldf,
                                                                const float* __restrict__ h0, const float* __restrict__ saved,
                                                                const T* __restrict__ gy, int64_t ldgy, const float* g_last,
                                                                T* __restrict__ gx, int64_t ldgx, T* __restrict__ gf, int64_t ldgf, float* g_h0) {
  __shared__ float before[kTile][64];
  const int blocks = (a.n_channels + 63) / 64;
  const int s = blockIdx.x / blocks, c = blockIdx.x % blocks * 64 + threadIdx.x;
  if (c >= a.n_channels) return;
  int64_t b, e;
  const bool ok = seq_range(a, s, &b, &e);
  const int64_t sc = (int64_t)s * a.n_channels + c;
  float g = g_last ? g_last[sc] : 0.0f;
  if (ok) {
    for (int64_t left = e - b; left > 0;) {  // tokens i = 0 .. left - 1 (in the recurrence's order) are still to do
      const int64_t last = a.reverse ? e - left : b + left - 1;
      const int64_t tile = last / kTile;
      const int64_t in_tile = a.reverse ? (tile + 1) * kTile - last : last - tile * kTile + 1;
      const int n = (int)(in_tile < left ? in_tile : left);
      float h = in_tile <= left ? saved[tile * a.n_channels + c] : h0 ? h0[sc] : 0.0f;
      for (int k = 0; k < n; ++k) {
        const int64_t i = left - n + k, t = a.reverse ? e - 1 - i : b + i;
        before[k][threadIdx.x] = h;
        h = step(h, (float)x[t * ldx + c], (float)f[t * ldf + c]);
      }
      for (int k = n - 1; k >= 0; --k) {
        const int64_t i = left - n + k, t = a.reverse ? e - 1 - i : b + i;
        const float xt = (float)x[t * ldx + c], ft = (float)f[t * ldf + c];
        const float p = gate_minor(ft);
        g += (float)gy[t * ldgy + c];
        const float pg = p == 0.0f ? 0.0f : p * g, rest = g - pg;
        gx[t * ldgx + c] = (T)(ft > 0.0f ? pg : rest);
        gf[t * ldgf + c] = (T)(p == 0.0f ? 0.0f : pg * (1.0f - p) * (before[k][threadIdx.x] - xt));
        g = ft > 0.0f ? rest : pg;
      }
      left -= n;
    }
  }
  if (g_h0) g_h0[sc] = ok ? g : __builtin_nanf("");
}

// zeros in the tokens in front of the first and behind the last sequence (rows blockIdx.x, blockIdx.x + gridDim.x, ... of them)
template <typename T>
__global__ __launch_bounds__(256) void zero_rest_kernel(ScanArgs a, T* y, int64_t ldy, T* y2, int64_t ldy2) {
  int64_t b = a.n_tokens, e = a.n_tokens;
  if (a.n_seqs > 0) {
    b = a.begin ? a.begin[0] : 0;
    e = a.end ? a.end[a.n_seqs - 1] : a.n_seqs * a.max_len;
    b = b < 0 ? 0 : b > a.n_tokens ? a.n_tokens : b;
    e = e < b ? b : e > a.n_tokens ? a.n_tokens : e;
  }
  for (int64_t i = blockIdx.x; i < b + a.n_tokens - e; i += gridDim.x) {
    const int64_t t = i < b ? i : i - b + e;
    for (int c = threadIdx.x; c < a.n_channels; c += blockDim.x) {
      y[t * ldy + c] = (T)0.0f;
      if (y2) y2[t * ldy2 + c] = (T)0.0f;
    }
  }
}

int check_scan(int32_t dtype, const void* x, int64_t x_stride, const void* f, int64_t f_stride, int64_t n_tokens, int32_t n_channels,
               const int64_t* begin, const int64_t* end, int32_t n_seqs, int64_t max_len) {
  DC_REQUIRE(dtype_ok(dtype), "unknown element type");
  DC_REQUIRE(n_tokens >= 0 && n_channels > 0 && n_seqs >= 0 && max_len >= 0, "negative size");
  DC_REQUIRE((begin == nullptr) == (end == nullptr), "begin and end come together");
  DC_REQUIRE(begin || max_len == 0 || n_seqs <= n_tokens / max_len, "dense sequences exceed the tokens");
  DC_REQUIRE(n_tokens == 0 || (x && f), "null pointer");
  DC_REQUIRE(x_stride >= 0 && f_stride >= 0, "negative stride");
  DC_REQUIRE((int64_t)n_seqs * ((n_channels + 63) / 64) < ((int64_t)1 << 25), "more than 2^25 blocks of 64 channels");
  DC_REQUIRE(aligned(x, dtype_size(dtype)) && aligned(f, dtype_size(dtype)), "misaligned pointer");
  return DC_OK;
}

}  // namespace
}  // namespace dc

extern "C" int64_t dc_gated_scan_saved(int64_t n_tokens, int32_t n_channels) {
  return n_tokens > 0 && n_channels > 0 ? (n_tokens + dc::kTile - 1) / dc::kTile * n_channels : 0;
}

extern "C" int64_t dc_gated_scan_workspace(int64_t, int32_t, int32_t, int64_t) { return 0; }

extern "C" int dc_gated_scan(void* stream, int32_t dtype, const void* d_x, int64_t x_stride, const void* d_f, int64_t f_stride,
                             int64_t n_tokens, int32_t n_channels, const int64_t* d_begin, const int64_t* d_end, int32_t n_seqs,
                             int64_t max_len, int32_t reverse, const float* d_h0, void* d_y, int64_t y_stride, int32_t zero_rest,
                             float* d_h_last, float* d_saved, void* d_workspace, int64_t workspace_bytes) {
  using namespace dc;
  if (int rc = check_scan(dtype, d_x, x_stride, d_f, f_stride, n_tokens, n_channels, d_begin, d_end, n_seqs, max_len)) return rc;
  DC_REQUIRE(n_tokens == 0 || d_y, "null pointer");
  DC_REQUIRE(y_stride >= n_channels, "rows of the output overlap");
  DC_REQUIRE(aligned(d_y, dtype_size(dtype)), "misaligned pointer");
  (void)d_workspace, (void)workspace_bytes;
  const ScanArgs a{d_begin, d_end, n_tokens, max_len, n_seqs, n_channels, reverse};
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (zero_rest && n_tokens > 0) zero_rest_kernel<T><<<dim3(64), dim3(256), 0, as_stream(stream)>>>(a, (T*)d_y, y_stride, nullptr, 0);
    if (n_seqs > 0) scan_walk_kernel<T><<<dim3(n_seqs * ((n_channels + 63) / 64)), dim3(64), 0, as_stream(stream)>>>(
        a, (const T*)d_x, x_stride, (const T*)d_f, f_stride, d_h0, (T*)d_y, y_stride, d_h_last, d_saved);
    DC_LAUNCH_CHECK();
    return DC_OK;
  });
}

extern "C" int dc_gated_scan_backward(void* stream, int32_t dtype, const void* d_x, int64_t x_stride, const void* d_f, int64_t f_stride,
                                      int64_t n_tokens, int32_t n_channels, const int64_t* d_begin, const int64_t* d_end, int32_t n_seqs,
                                      int64_t max_len, int32_t reverse, const float* d_h0, const float* d_saved, const void* d_grad_y,
                                      int64_t grad_y_stride, const float* d_grad_h_last, void* d_grad_x, int64_t grad_x_stride, void* d_grad_f,
                                      int64_t grad_f_stride, int32_t zero_rest, float* d_grad_h0, void* d_workspace, int64_t workspace_bytes) {
  using namespace dc;
  if (int rc = check_scan(dtype, d_x, x_stride, d_f, f_stride, n_tokens, n_channels, d_begin, d_end, n_seqs, max_len)) return rc;
  DC_REQUIRE(n_tokens == 0 || (d_saved && d_grad_y && d_grad_x && d_grad_f), "null pointer");
  DC_REQUIRE(grad_y_stride >= 0, "negative stride");
  DC_REQUIRE(grad_x_stride >= n_channels && grad_f_stride >= n_channels, "rows of an output overlap");
  DC_REQUIRE(aligned(d_grad_y, dtype_size(dtype)) && aligned(d_grad_x, dtype_size(dtype)) && aligned(d_grad_f, dtype_size(dtype)), "misaligned pointer");
  (void)d_workspace, (void)workspace_bytes;
  const ScanArgs a{d_begin, d_end, n_tokens, max_len, n_seqs, n_channels, reverse};
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (zero_rest && n_tokens > 0) zero_rest_kernel<T><<<dim3(64), dim3(256), 0, as_stream(stream)>>>(a, (T*)d_grad_x, grad_x_stride, (T*)d_grad_f, grad_f_stride);
    if (n_seqs > 0) scan_walk_backward_kernel<T><<<dim3(n_seqs * ((n_channels + 63) / 64)), dim3(64), 0, as_stream(stream)>>>(
        a, (const T*)d_x, x_stride, (const T*)d_f, f_stride, d_h0, d_saved, (const T*)d_grad_y, grad_y_stride, d_grad_h_last, (T*)d_grad_x,
        grad_x_stride, (T*)d_grad_f, grad_f_stride, d_grad_h0);
    DC_LAUNCH_CHECK();
    return DC_OK;
  });
}
