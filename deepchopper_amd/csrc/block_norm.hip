// dc_block_norm: the norm behind a block, its gate and residual scale, and the norm in front of the next block, in one pass
// over the rows, and its backward pass.
//
// HBM-bound: forward 5 row elements of traffic per element (y, gate, residual in; r', n out), backward 8 (y, gate, residual, both
// gradients in; three out) for 4 row reductions each.  A row stays in registers between its passes: 4 elements a lane and step of 256
// columns, a row in 2 to 64 lanes of a wavefront up to 256 columns, in one wavefront up to 512 (forward), in up to 16 of them
// beyond.  Mean and deviation are taken one after the other (no E[x^2] - E[x]^2: a mean far from 0 costs no digits).  Backward, nothing of
// the forward pass is read back: r', u and both norms' statistics cost less to take again from the inputs than to load.
// The vectors' gradients: every lane sums its own columns over the rows of its workgroup, the workgroups' sums go to the workspace
// and are added in order by a second kernel (no atomics).
// Measured (a large copy: 4.7 TB/s): 524 288 x 256 bf16 on an fp32 residual forward 384 us = 4.9 TB/s, backward 592 us = 5.0 TB/s (fp32 throughout
// 562 us = 4.8 TB/s, 851 us = 5.0 TB/s); 65 537 x 1000 bf16 forward 137 us = 4.8 TB/s, backward 266 us = 3.9 TB/s: bound by vector work, 55
// operations a column and four exchanges a row.  Beyond 4 096 columns the backward pass spills: 8 192 x 8 192 bf16 824 us = 1.3 TB/s.
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
  // what a team's wavefronts told each other is added up one after the other (forward, two wavefronts: 65 536 x 1000 bf16 153 us against
  // 200 us) or by the lanes of 16 (backward and more wavefronts: 131 072 x 512 bf16 265 us against 293 us, 32 768 x 2048 292 us against 396 us)
  int32_t serial;
};

// One row's columns of this thread: K vectors of V, 256 * n_waves apart.  Elements beyond the width are 0 and not stored.
template <int K>
struct Part {
  float v[K][V];
};
// ... as they lie in memory: the next row is on its way while one is worked on
template <typename T, int K>
struct RawPart {
  typename loose_vec<T, V>::type r[K];
};

// How a row lies in a workgroup: several rows in a wavefront (at most 128 columns), a row in one, a row in several.
enum Form { kSub, kWave, kTeam };

// columns that wavefront w of a row has (w >= n_waves: 0)
template <int K>
__device__ __forceinline__ float columns_of(const NormArgs& a, int w) {
  int n = 0;
  if (w >= a.n_waves) return 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int left = a.width - (w + k * a.n_waves) * 64 * V;
    n += left < 0 ? 0 : left < 64 * V ? left : 64 * V;
  }
  return (float)n;
}

// Where a thread's columns and rows lie.  Outside kSub the row is the wavefront's, kept in scalar registers.
template <int K, Form F>
struct Spot {
  int column, step, wave, group, n_groups;  // first column, columns between vectors, row group of the workgroup
  float inv_own, of_lane;                   // a team's: 1 / columns of this wavefront, columns of wavefront (lane mod 16) of the row
  __device__ __forceinline__ Spot(const NormArgs& a) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if constexpr (F == kSub) {
      column = (threadIdx.x & ((1 << a.lane_bits) - 1)) * V;
      group = threadIdx.x >> a.lane_bits;
      n_groups = blockDim.x >> a.lane_bits;
    } else {
      const int per_row = F == kTeam ? a.n_waves : 1;
      column = (wave % per_row * 64 + (threadIdx.x & 63)) * V;
      group = wave / per_row;
      n_groups = (int)(blockDim.x >> 6) / per_row;
    }
    step = a.n_waves * 64 * V;
    if constexpr (F == kTeam) {
      inv_own = 1.0f / __builtin_fmaxf(columns_of<K>(a, wave - group * a.n_waves), 1.0f);
      of_lane = columns_of<K>(a, threadIdx.x & 15);
    }
  }
};

// the thread's whole vectors of a row, or the single elements of the one that the width cuts
template <typename T, int K>
__device__ __forceinline__ void load_whole(const T* row, int c, int k, RawPart<T, K>& p) {
  p.r[k] = *reinterpret_cast<const typename loose_vec<T, V>::type*>(row + c);
}
template <typename T, int K>
__device__ __forceinline__ void load_cut(const T* row, int c, int k, int width, RawPart<T, K>& p) {
#pragma unroll
  for (int i = 0; i < V - 1; ++i)
    if (c + i < width) p.r[k][i] = row[c + i];
}
template <typename T, int K>
__device__ __forceinline__ void clear(RawPart<T, K>& p) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) p.r[k][i] = (T)0.0f;
}
template <typename T, int K>
__device__ __forceinline__ void store_whole(T* row, int c, int k, const Part<K>& p) {
  store_vec<V>(row + c, p.v[k]);
}
template <typename T, int K>
__device__ __forceinline__ void store_cut(T* row, int c, int k, int width, const Part<K>& p) {
#pragma unroll
  for (int i = 0; i < V - 1; ++i)
    if (c + i < width) row[c + i] = (T)p.v[k][i];
}
// f(whole, c, k) for every vector of the thread that has elements of the row
template <int K, typename At, typename Fn>
__device__ __forceinline__ void for_vectors(const NormArgs& a, const At& at, Fn&& f) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = at.column + k * at.step;
    if (c + V <= a.width) f(std::true_type{}, c, k);
    else if (c < a.width) f(std::false_type{}, c, k);
  }
}
template <typename T, int K>
__device__ __forceinline__ void widen(const RawPart<T, K>& p, Part<K>& out) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) out.v[k][i] = (float)p.r[k][i];
}
// The gate's activation, in place; with `slope`, its derivative.  With e = exp(-x) and s = 1 / (1 + e), 1 - s is e s, which keeps its digits
// where s is next to 1 (and is 1 where e is infinite).
template <int K>
__device__ __forceinline__ void activate(const NormArgs& a, Part<K>& g, Part<K>* slope) {
  if (a.act == DC_ACT_IDENTITY) {
    if (slope) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) slope->v[k][i] = 1.0f;
    }
    return;
  }
  const bool silu = a.act == DC_ACT_SILU;
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float x = g.v[k][i], e = fast_exp2(-x * kLog2e), s = fast_rcp(1.0f + e);
      if (slope) {
        const float rest = __builtin_fminf(e * s, 1.0f);
        slope->v[k][i] = s * (silu ? __builtin_fmaf(x, rest, 1.0f) : rest);
      }
      g.v[k][i] = silu ? x * s : s;
    }
  }
}
template <int K>
__device__ __forceinline__ void fill(Part<K>& p, float x) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) p.v[k][i] = x;
}
// a vector of the width, or a constant; 0 beyond the width, which keeps what stands there out of every sum
template <int K, typename At>
__device__ __forceinline__ void load_weights(const float* w, float other, const NormArgs& a, const At& at, Part<K>& p) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = at.column + k * at.step + i;
      p.v[k][i] = c >= a.width ? 0.0f : w ? w[c] : other;
    }
  }
}

// What the wavefronts of a row tell each other, one slot a wavefront, two halves used in turn: one barrier an exchange.
struct Meeting {
  float2 slot[2][16];
  // lane l of every 16: what wavefront l of the row said
  __device__ __forceinline__ float2 of_lane(int turn, int first, int n_waves) const {
    const int l = threadIdx.x & 15;
    return l < n_waves ? slot[turn][first + l] : float2{0.0f, 0.0f};
  }
};

// Sums over the row of one or two values.
template <int K, Form F>
__device__ __forceinline__ float2 row_sums(float x, float y, bool two, const NormArgs& a, const Spot<K, F>& at, Meeting& m, int& turn) {
  const int bits = F == kSub ? a.lane_bits : 6;
  float2 s{lanes_sum(x, bits), two ? lanes_sum(y, bits) : 0.0f};
  if constexpr (F == kTeam) {
    if ((threadIdx.x & 63) == 0) m.slot[turn][at.wave] = s;
    __syncthreads();
    const int first = at.group * a.n_waves;
    if (a.serial) {
      s = m.slot[turn][first];
      for (int w = 1; w < a.n_waves; ++w) s.x += m.slot[turn][first + w].x, s.y += m.slot[turn][first + w].y;
    } else {
      s = m.of_lane(turn, first, a.n_waves);
      s = {lanes_sum(s.x, 4), two ? lanes_sum(s.y, 4) : 0.0f};
    }
    turn ^= 1;
  }
  return s;
}

// mean (RMS: 0) and 1 / deviation of a row; elements beyond the width are 0.  The squares are taken about the mean: of the wavefront's own
// columns first, moved to the row's mean when the wavefronts meet (sum (x - m)^2 = sum (x - m_w)^2 + n_w (m_w - m)^2).
template <int K, Form F>
__device__ __forceinline__ float2 row_stats(const Part<K>& p, const NormArgs& a, const Spot<K, F>& at, Meeting& m, int& turn) {
  const int bits = F == kSub ? a.lane_bits : 6;
  float mean = 0.0f, q = 0.0f;
  if (a.kind == DC_NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) s += p.v[k][i];
    s = lanes_sum(s, bits);
    mean = s * (F == kTeam ? at.inv_own : a.inv_width);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = at.column + k * at.step;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = c + i < a.width ? p.v[k][i] - mean : 0.0f;
      q = __builtin_fmaf(d, d, q);
    }
  }
  q = lanes_sum(q, bits);
  if constexpr (F == kTeam) {
    if ((threadIdx.x & 63) == 0) m.slot[turn][at.wave] = {mean, q};
    __syncthreads();
    const int first = at.group * a.n_waves;
    if (a.serial) {
      q = 0.0f;
      if (a.kind == DC_NORM_LAYER) {
        float all = 0.0f;
        for (int w = 0; w < a.n_waves; ++w) all = __builtin_fmaf(m.slot[turn][first + w].x, columns_of<K>(a, w), all);
        mean = all * a.inv_width;
        for (int w = 0; w < a.n_waves; ++w) {
          const float2 o = m.slot[turn][first + w];
          q += __builtin_fmaf((o.x - mean) * (o.x - mean), columns_of<K>(a, w), o.y);
        }
      } else {
        for (int w = 0; w < a.n_waves; ++w) q += m.slot[turn][first + w].y;
      }
      turn ^= 1;
      return {mean, __builtin_amdgcn_rsqf(__builtin_fmaf(q, a.inv_width, a.eps))};
    }
    const float2 o = m.of_lane(turn, first, a.n_waves);
    if (a.kind == DC_NORM_LAYER) {
      mean = lanes_sum(o.x * at.of_lane, 4) * a.inv_width;
      q = lanes_sum(__builtin_fmaf((o.x - mean) * (o.x - mean), at.of_lane, o.y), 4);
    } else {
      q = lanes_sum(o.y, 4);
    }
    turn ^= 1;
  }
  return {mean, __builtin_amdgcn_rsqf(__builtin_fmaf(q, a.inv_width, a.eps))};  // (v_rsq_f32: 1 ulp)
}

// The rows of a workgroup's group: blockIdx.x * n_groups + group, ...; all groups take the same number of turns (a team's sums have
// barriers), one without a row in the last turn works on the last row again and stores nothing.
struct Rows {
  int64_t first, step, n;
  int group;
  template <int K, Form F>
  __device__ __forceinline__ Rows(const NormArgs& a, const Spot<K, F>& at)
      : first((int64_t)blockIdx.x * at.n_groups), step((int64_t)gridDim.x * at.n_groups), n(a.n_rows), group(at.group) {}
  __device__ __forceinline__ int64_t clamped(int64_t f) const { return f + group < n ? f + group : n - 1; }
};

template <typename T, typename R, int K, Form F, int THREADS>
__global__ __launch_bounds__(THREADS) void block_norm_kernel(NormArgs a, const T* y, const T* gate, const R* residual, R* residual_out,
                                                                              int64_t residual_out_stride, T* normed, int64_t normed_stride) {
  __shared__ Meeting meeting;
  int turn = 0;
  const Spot<K, F> at(a);
  const Rows rows(a, at);
  RawPart<T, K> raw_y, raw_g;
  RawPart<R, K> raw_r;
  clear(raw_y), clear(raw_g), clear(raw_r);
  auto fetch = [&](int64_t row) {
    const T *py = y + row * a.y_stride, *pg = gate + row * a.gate_stride;
    const R* pr = residual + row * a.residual_stride;
    for_vectors<K>(a, at, [&](auto whole, int c, int k) {
      if constexpr (decltype(whole)::value) {
        if (y) load_whole(py, c, k, raw_y);
        if (gate) load_whole(pg, c, k, raw_g);
        if (residual) load_whole(pr, c, k, raw_r);
      } else {
        if (y) load_cut(py, c, k, a.width, raw_y);
        if (gate) load_cut(pg, c, k, a.width, raw_g);
        if (residual) load_cut(pr, c, k, a.width, raw_r);
      }
    });
  };
  if (rows.first < rows.n) fetch(rows.clamped(rows.first));
  Part<K> sc, w1, b1, w2, b2;
  load_weights(a.scale, 1.0f, a, at, sc);
  load_weights(a.post_w, 1.0f, a, at, w1);
  load_weights(a.post_b, 0.0f, a, at, b1);
  load_weights(a.pre_w, 1.0f, a, at, w2);
  load_weights(a.pre_b, 0.0f, a, at, b2);
  for (int64_t f = rows.first; f < rows.n; f += rows.step) {
    const int64_t row = f + at.group;
    const bool live = row < rows.n;
    Part<K> v, g, r;
    fill(r, 0.0f);
    if (y) widen(raw_y, v);
    if (gate) widen(raw_g, g);
    if (residual) widen(raw_r, r);
    if (f + rows.step < rows.n) fetch(rows.clamped(f + rows.step));
    if (y) {
      if (gate) activate<K>(a, g, nullptr);
      else fill(g, 1.0f);
      float2 st{0.0f, 1.0f};
      if (a.post_norm) st = row_stats<K, F>(v, a, at, meeting, turn);
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float u = v.v[k][i];
          if (a.post_norm) u = __builtin_fmaf((u - st.x) * st.y, w1.v[k][i], b1.v[k][i]);
          r.v[k][i] = __builtin_fmaf(sc.v[k][i], g.v[k][i] * u, r.v[k][i]);
        }
      }
    }
    if (normed) {
      const float2 st = row_stats<K, F>(r, a, at, meeting, turn);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) v.v[k][i] = __builtin_fmaf((r.v[k][i] - st.x) * st.y, w2.v[k][i], b2.v[k][i]);
    }
    if (!live) continue;
    R* po = residual_out + row * residual_out_stride;
    T* pn = normed + row * normed_stride;
    for_vectors<K>(a, at, [&](auto whole, int c, int k) {
      if constexpr (decltype(whole)::value) {
        if (residual_out) store_whole(po, c, k, r);
        if (normed) store_whole(pn, c, k, v);
      } else {
        if (residual_out) store_cut(po, c, k, a.width, r);
        if (normed) store_cut(pn, c, k, a.width, v);
      }
    });
  }
}

// The gradient g of a normalised row, in place, to that of the row: factor (g - mean(g) - hat mean(g hat)).
template <int K, Form F>
__device__ __forceinline__ void norm_back(Part<K>& g, const Part<K>& hat, const NormArgs& a, const Spot<K, F>& at, float factor, Meeting& m, int& turn) {
  float s = 0.0f, q = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) s += g.v[k][i], q = __builtin_fmaf(g.v[k][i], hat.v[k][i], q);
  const bool layer = a.kind == DC_NORM_LAYER;
  const float2 t = row_sums<K, F>(q, s, layer, a, at, m, turn);
  q = t.x * a.inv_width;
  s = layer ? t.y * a.inv_width : 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) g.v[k][i] = factor * (g.v[k][i] - s - hat.v[k][i] * q);
}

// Five workgroups a CU where 16-bit rows leave the registers for it: 262 144 x 256 bf16 320 -> 278 us; with fp32 rows it would spill.
constexpr int waves_a_simd(int row_bytes, int k, Form f, int threads) { return row_bytes == 2 && k == 1 && f != kSub && threads == 256 ? 5 : 1; }

// Rows as in the forward pass; the workgroup's sums over them, [5][width] in the order scale, post_w, post_b, pre_w, pre_b, go to
// sums[blockIdx.x].
template <typename T, typename R, int K, Form F, int THREADS>
__global__ __launch_bounds__(THREADS, waves_a_simd(sizeof(R), K, F, THREADS)) void block_norm_backward_kernel(
    NormArgs a, const T* y, const T* gate, const R* residual, const R* g_out, int64_t g_out_stride, const T* g_normed, int64_t g_normed_stride, T* g_y,
    T* g_gate, R* g_residual, float* __restrict__ sums) {
  extern __shared__ __align__(16) float lds[];  // a team's weights, and at the end a vector per row group
  __shared__ Meeting meeting;
  int turn = 0;
  const Spot<K, F> at(a);
  const Rows rows(a, at);
  RawPart<T, K> raw_y, raw_g, raw_n;
  RawPart<R, K> raw_r, raw_o;
  clear(raw_y), clear(raw_g), clear(raw_n), clear(raw_r), clear(raw_o);
  auto fetch = [&](int64_t row) {
    const T *py = y + row * a.y_stride, *pg = gate + row * a.gate_stride, *pn = g_normed + row * g_normed_stride;
    const R *pr = residual + row * a.residual_stride, *po = g_out + row * g_out_stride;
    for_vectors<K>(a, at, [&](auto whole, int c, int k) {
      if constexpr (decltype(whole)::value) {
        if (y) load_whole(py, c, k, raw_y);
        if (residual) load_whole(pr, c, k, raw_r);
        if (gate) load_whole(pg, c, k, raw_g);
        if (g_normed) load_whole(pn, c, k, raw_n);
        if (g_out) load_whole(po, c, k, raw_o);
      } else {
        if (y) load_cut(py, c, k, a.width, raw_y);
        if (residual) load_cut(pr, c, k, a.width, raw_r);
        if (gate) load_cut(pg, c, k, a.width, raw_g);
        if (g_normed) load_cut(pn, c, k, a.width, raw_n);
        if (g_out) load_cut(po, c, k, a.width, raw_o);
      }
    });
  };
  if (rows.first < rows.n) fetch(rows.clamped(rows.first));
  // The weights: a team keeps them in LDS (its lanes have no registers to spare), others in registers.
  Part<K> acc[5], held[F == kTeam ? 1 : 4];
#pragma unroll
  for (int n = 0; n < 5; ++n) fill(acc[n], 0.0f);
  const int span = a.n_waves * 64 * V * K;
  if constexpr (F == kTeam) {
    for (int c = threadIdx.x; c < span; c += blockDim.x) {
      const bool in = c < a.width;
      lds[c] = in ? a.scale ? a.scale[c] : 1.0f : 0.0f;
      lds[span + c] = in ? a.post_w ? a.post_w[c] : 1.0f : 0.0f;
      lds[2 * span + c] = in && a.post_b ? a.post_b[c] : 0.0f;
      lds[3 * span + c] = in ? a.pre_w ? a.pre_w[c] : 1.0f : 0.0f;
    }
    __syncthreads();
  } else {
    load_weights(a.scale, 1.0f, a, at, held[0]);
    load_weights(a.post_w, 1.0f, a, at, held[1]);
    load_weights(a.post_b, 0.0f, a, at, held[2]);
    load_weights(a.pre_w, 1.0f, a, at, held[3]);
  }
  enum { kScale, kPostW, kPostB, kPreW };
  auto weights = [&](int n) {
    if constexpr (F == kTeam) {
      Part<K> p;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float4 q = *reinterpret_cast<const float4*>(lds + n * span + at.column + k * at.step);
        p.v[k][0] = q.x, p.v[k][1] = q.y, p.v[k][2] = q.z, p.v[k][3] = q.w;
      }
      return p;
    } else {
      return held[n];
    }
  };
  for (int64_t f = rows.first; f < rows.n; f += rows.step) {
    const int64_t row = f + at.group;
    const bool live = row < rows.n;
    Part<K> hat, g, slope, t, r, o;  // g: act(gate)
    fill(r, 0.0f);
    fill(o, 0.0f);
    if (y) widen(raw_y, hat);
    if (residual) widen(raw_r, r);
    if (gate) widen(raw_g, g);
    if (g_normed) widen(raw_n, t);
    if (g_out) widen(raw_o, o);
    if (f + rows.step < rows.n) fetch(rows.clamped(f + rows.step));
    float2 st{0.0f, 1.0f};
    if (y) {  // hat: the normalised block output (or the output itself); r: r'
      if (gate) activate<K>(a, g, &slope);
      else fill(g, 1.0f);
      if (a.post_norm) {
        st = row_stats<K, F>(hat, a, at, meeting, turn);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) hat.v[k][i] = (hat.v[k][i] - st.x) * st.y;
      }
      const Part<K> sc = weights(kScale), w1 = weights(kPostW), b1 = weights(kPostB);
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float u = a.post_norm ? __builtin_fmaf(hat.v[k][i], w1.v[k][i], b1.v[k][i]) : hat.v[k][i];
          r.v[k][i] = __builtin_fmaf(sc.v[k][i], g.v[k][i] * u, r.v[k][i]);
        }
      }
    }
    if (g_normed) {  // r becomes the normalised r', t the gradient of r' through the norm
      const float2 st2 = row_stats<K, F>(r, a, at, meeting, turn);
      const Part<K> w2 = weights(kPreW);
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          r.v[k][i] = (r.v[k][i] - st2.x) * st2.y;
          if (live) {
            acc[3].v[k][i] = __builtin_fmaf(t.v[k][i], r.v[k][i], acc[3].v[k][i]);
            acc[4].v[k][i] += t.v[k][i];
          }
          t.v[k][i] *= w2.v[k][i];
        }
      }
      norm_back<K, F>(t, r, a, at, st2.y, meeting, turn);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) t.v[k][i] += o.v[k][i];
    } else {
      t = o;
    }
    r = t;  // the gradient of the residual
    if (y) {
      const Part<K> sc = weights(kScale), w1 = weights(kPostW), b1 = weights(kPostB);
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float u = a.post_norm ? __builtin_fmaf(hat.v[k][i], w1.v[k][i], b1.v[k][i]) : hat.v[k][i];
          const float gv = t.v[k][i] * sc.v[k][i];
          const float gu = gv * g.v[k][i];
          if (live) {
            acc[0].v[k][i] = __builtin_fmaf(t.v[k][i], g.v[k][i] * u, acc[0].v[k][i]);
            acc[1].v[k][i] = __builtin_fmaf(gu, hat.v[k][i], acc[1].v[k][i]);
            acc[2].v[k][i] += gu;
          }
          slope.v[k][i] *= gv * u;
          t.v[k][i] = a.post_norm ? gu * w1.v[k][i] : gu;
        }
      }
      if (g_y && a.post_norm) norm_back<K, F>(t, hat, a, at, st.y, meeting, turn);
    }
    if (!live) continue;
    R* pr = g_residual + row * a.width;
    T *pg = g_gate + row * a.width, *py = g_y + row * a.width;
    for_vectors<K>(a, at, [&](auto whole, int c, int k) {
      if constexpr (decltype(whole)::value) {
        if (g_residual) store_whole(pr, c, k, r);
        if (gate && g_gate) store_whole(pg, c, k, slope);
        if (y && g_y) store_whole(py, c, k, t);
      } else {
        if (g_residual) store_cut(pr, c, k, a.width, r);
        if (gate && g_gate) store_cut(pg, c, k, a.width, slope);
        if (y && g_y) store_cut(py, c, k, a.width, t);
      }
    });
  }
  if (!sums) return;
  float* own = sums + (int64_t)blockIdx.x * 5 * a.width;
#pragma unroll
  for (int n = 0; n < 5; ++n) {
    __syncthreads();
    for_vectors<K>(a, at, [&](auto whole, int c, int k) {
      if constexpr (decltype(whole)::value) store_whole(lds + at.group * a.width, c, k, acc[n]);
      else store_cut(lds + at.group * a.width, c, k, a.width, acc[n]);
    });
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
  int32_t n_parts[5];  // 0: a vector that the call did not use
};

// 32 columns of one vector, the parts divided over 32 rows of threads.
__global__ __launch_bounds__(1024) void block_norm_sums_kernel(const float* __restrict__ sums, int32_t width, SumOut out) {
  __shared__ float lds[32][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, k = blockIdx.y;
  if (!out.p[k]) return;
  float s = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (int i = part; i < out.n_parts[k]; i += 32) s += sums[((int64_t)i * 5 + k) * width + c];
  }
  lds[part][lane] = s;
  __syncthreads();
  if (part == 0 && c < width) {
    for (int q = 1; q < 32; ++q) s += lds[q][lane];
    out.p[k][c] = s;
  }
}

// How many lanes, wavefronts and vectors a row takes: lanes of a wavefront up to 256 columns, then (forward) two vectors a lane, then up to
// 16 wavefronts.  Backward there are 5 sums a column besides the row: one vector a lane while 16 wavefronts suffice (two would leave 2
// instead of 4 or 5 workgroups a CU: 131 072 x 512 bf16 548 us against 265 us).
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
  const int one = (width + 64 * V - 1) / (64 * V), two = (width + 128 * V - 1) / (128 * V);  // wavefronts with one or two vectors a lane
  p.k = backward ? one > 16 ? 2 : 1 : one <= 16 && 5 * one < 8 * two ? 1 : 2;                // (forward: two, unless a fifth of them would be idle)
  p.n_waves = p.k == 1 ? one : two;
  p.threads = p.n_waves <= 2 ? 256 : 64 * p.n_waves;
  return p;
}

// workgroups of the backward pass = parts of the vectors' sums
int parts_of(int64_t n_rows, int32_t width, int32_t residual_dtype) {
  const RowPlan p = row_plan(width, true);
  const int groups = p.n_waves > 1 ? p.threads / 64 / p.n_waves : p.threads >> p.lane_bits;
  int64_t most = (1 << 21) / width;  // at most 40 MB of them, but one for every CU
  const int full = residual_dtype != DC_DTYPE_F32 && (p.n_waves > 1 || p.lane_bits == 6) && p.n_waves <= 4 ? 1280 : 1024;  // (what runs at once)
  most = most > full ? full : most < 256 ? 256 : most;
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

// calls f with the element types, the vectors a lane and whether a row takes several wavefronts.  (Of the forms only those that row_plan
// gives: two vectors a lane forward in one wavefront or more, backward only beyond 16; one of 5 to 16 wavefronts only backward.)
template <bool BACK, typename F>
int with_row(int32_t dtype, int32_t residual_dtype, const RowPlan& p, F&& f) {
  return with_dtype(dtype, [&](auto t) {
    auto g = [&](auto r) {
      using One = std::integral_constant<int, 1>;
      using Two = std::integral_constant<int, 2>;
      using Wave = std::integral_constant<Form, kWave>;
      using Team = std::integral_constant<Form, kTeam>;
      using Small = std::integral_constant<int, 256>;
      using Large = std::integral_constant<int, 1024>;
      if (p.n_waves == 1 && p.lane_bits < 6) return f(t, r, One{}, std::integral_constant<Form, kSub>{}, Small{});
      if constexpr (BACK) {
        if (p.n_waves == 1) return f(t, r, One{}, Wave{}, Small{});
        if (p.n_waves <= 4) return f(t, r, One{}, Team{}, Small{});
        return p.k == 1 ? f(t, r, One{}, Team{}, Large{}) : f(t, r, Two{}, Team{}, Large{});
      } else {
        if (p.n_waves == 1) return p.k == 1 ? f(t, r, One{}, Wave{}, Small{}) : f(t, r, Two{}, Wave{}, Small{});
        if (p.n_waves <= 4) return p.k == 1 ? f(t, r, One{}, Team{}, Small{}) : f(t, r, Two{}, Team{}, Small{});
        return f(t, r, Two{}, Team{}, Large{});
      }
    };
    return residual_dtype == dtype ? g(t) : g(f32{});
  });
}

}  // namespace
}  // namespace dc

extern "C" int64_t dc_block_norm_workspace(int64_t n_rows, int32_t width, int32_t residual_dtype) {
  return n_rows > 0 && width > 0 ? (int64_t)dc::parts_of(n_rows, width, residual_dtype) * 5 * width * 4 : 0;
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
                   d_scale, d_post_w, d_post_b, d_pre_w, d_pre_b, p.lane_bits, p.n_waves, p.n_waves == 2};
  const int groups = p.n_waves > 1 ? p.threads / 64 / p.n_waves : p.threads >> p.lane_bits;
  const int64_t need = (n_rows + groups - 1) / groups;
  const int grid = (int)(need < 4096 ? need : 4096);
  return with_row<false>(dtype, residual_dtype, p, [&](auto t, auto r, auto k, auto form, auto threads) {
    using T = decltype(t);
    using R = decltype(r);
    block_norm_kernel<T, R, decltype(k)::value, decltype(form)::value, decltype(threads)::value><<<dim3(grid), dim3(p.threads), 0, as_stream(stream)>>>(
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
  DC_REQUIRE(workspace_bytes >= dc_block_norm_workspace(n_rows, width, residual_dtype) && (n_rows == 0 || d_workspace) && aligned(d_workspace, 16), "workspace too small");
  const RowPlan p = row_plan(width, true);
  const NormArgs a{n_rows, width, kind, gate_act, post_norm, eps, 1.0f / width, y_stride, gate_stride, residual_stride,
                   d_scale, d_post_w, d_post_b, d_pre_w, nullptr, p.lane_bits, p.n_waves, 0};
  const int groups = p.n_waves > 1 ? p.threads / 64 / p.n_waves : p.threads >> p.lane_bits;
  const int grid = parts_of(n_rows, width, residual_dtype);
  const bool any = d_grad_scale || d_grad_post_w || d_grad_post_b || d_grad_pre_w || d_grad_pre_b;
  return with_row<true>(dtype, residual_dtype, p, [&](auto t, auto r, auto k, auto form, auto threads) {
    using T = decltype(t);
    using R = decltype(r);
    if (grid > 0) {
      auto kernel = block_norm_backward_kernel<T, R, decltype(k)::value, decltype(form)::value, decltype(threads)::value>;
      DC_SET_MAX_SMEM_ONCE_PER_DEVICE(kernel, DC_MAX_NORM_WIDTH * 16);
      const int held = p.n_waves > 1 ? 4 * p.n_waves * 64 * V * p.k : 0, floats = held > groups * width ? held : groups * width;
      kernel<<<dim3(grid), dim3(p.threads), floats * 4, as_stream(stream)>>>(
          a, (const T*)d_y, (const T*)d_gate, (const R*)d_residual, (const R*)d_grad_residual_out, grad_residual_out_stride,
          (const T*)d_grad_normed, grad_normed_stride, (T*)d_grad_y, (T*)d_grad_gate, (R*)d_grad_residual, any ? (float*)d_workspace : nullptr);
      DC_LAUNCH_CHECK();
    }
    if (any) {
      block_norm_sums_kernel<<<dim3((width + 31) / 32, 5), dim3(1024), 0, as_stream(stream)>>>(
          (const float*)d_workspace, width,
          SumOut{{d_grad_scale, d_grad_post_w, d_grad_post_b, d_grad_pre_w, d_grad_pre_b}, {grid, post_norm ? grid : 0, post_norm ? grid : 0, grid, grid}});
      DC_LAUNCH_CHECK();
    }
    return DC_OK;
  });
}
