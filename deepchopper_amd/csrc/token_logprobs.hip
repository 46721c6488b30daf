// dc_token_logprobs: log probabilities of given tokens, entropy and top alternatives of rows of logits, and their gradient.
//
// HBM-bound: a row is read once (backward: read once, written once).  With m the row's maximum, S = sum exp(z - m) and
// U = sum exp(z - m) (z - m):   log p_j = (z_j - m) - log S    H = log S - U / S    dz_j = p_j (-g - h (log p_j + H)) + g [j = t]
//
// Up to 512 classes a row lives in the registers of 1 to 32 lanes (2 to 16 classes a lane), forward and backward:
// the two-class logits of a predict batch are one lane a row.  There S is summed without its largest term's 1 and log S = log1p(S - 1), so a
// row that is sure of its class keeps the digits of -log p.
// Beyond, a wavefront walks the row (or, where there are few rows, one of up to 64 slices of it, joined by a second kernel) in pieces of
// 64 x 64 bytes kept in registers: running maximum, S and U per lane, joined at the end.
// Top alternatives of a walk: the n-th largest of the lanes' (or quads') maxima bounds the n-th largest class from below, so one comparison
// a class against that bound leaves a few candidates, which are collected in LDS and ranked by counting; the bound only rises from
// there on.  Ties go to the lower class throughout: candidates are ordered by (logit, class).
// Measured (a large copy: 4.7 TB/s): 2 050 048 x 2 fp32 with one alternative 13.6 us (47 MB); 4 096 x 100 003 bf16 forward 188 us = 4.4 TB/s,
// backward 270 us = 6 TB/s; 16 384 x 4 096 bf16 with four alternatives 50 us (vector work, 22 operations a class); 5 x 50 257 fp16 with
// twenty 9.4 + 5.9 us (latency).  A piece is worked in full whatever of it the row fills: 16 384 x 600 bf16 16.1 us, as x 1 024.
#include <type_traits>

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

// a float's place in ascending order as an unsigned number, never 0 or 0xffffffff: -0 with +0, every NaN above +inf
__device__ __forceinline__ uint32_t order_key(float z) {
  if (!(z == z)) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(z + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return k == 0xfffffffeu ? __builtin_nanf("") : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct RowStats {
  float m, log_sum, entropy;  // max, log sum exp(z - m), entropy
};
__device__ __forceinline__ float log_prob(const RowStats& r, float z) { return r.m == -INFINITY ? -INFINITY : (z - r.m) - r.log_sum; }

// dz of the other classes
__device__ __forceinline__ float grad_at(const RowStats& r, float z, float g, float h) {
  const float lp = (z - r.m) - r.log_sum, p = fast_exp2(lp * kLog2e);
  return p == 0.0f ? 0.0f : -p * __builtin_fmaf(h, lp + r.entropy, g);
}
// dz of the given one, g (1 - p) - h p (lp + H): for p next to 1 its 1 - p is the series of -expm1(lp) (below 1/4 to 2^-29), not a difference
__device__ __forceinline__ float grad_of_given(const RowStats& r, float z, float g, float h) {
  const float lp = (z - r.m) - r.log_sum, p = fast_exp2(lp * kLog2e), u = -lp;
  float rest = __builtin_fmaf(u, 1.0f / 5040, -1.0f / 720);
  rest = __builtin_fmaf(u, rest, 1.0f / 120);
  rest = __builtin_fmaf(u, rest, -1.0f / 24);
  rest = __builtin_fmaf(u, rest, 1.0f / 6);
  rest = __builtin_fmaf(u, rest, -0.5f);
  rest = __builtin_fmaf(u, rest, 1.0f) * u;
  return p == 0.0f ? g : __builtin_fmaf(g, u < 0.25f ? rest : 1.0f - p, -h * p * (lp + r.entropy));
}

// what a row's gradient is: as the formula says, zeros (skipped, or nothing is possible), or NaN (a token outside the classes)
enum RowGrad { kFormula, kZeros, kNans };
__device__ __forceinline__ RowGrad row_grad(bool skip, const RowStats& r, bool wrong) {
  return skip || r.m == -INFINITY ? kZeros : wrong ? kNans : kFormula;
}

template <typename Op>
__device__ __forceinline__ uint32_t lanes_reduce_u32(uint32_t v, int bits, Op op) {
  return __float_as_uint(lanes_reduce(__uint_as_float(v), bits, [&](float a, float b) { return __uint_as_float(op(__float_as_uint(a), __float_as_uint(b))); }));
}

// ---- up to 512 classes: a row in the registers of 2^bits lanes ------------------------------------------------------------------
template <int E>
struct Few {
  static constexpr int W = E < 4 ? E : 4;  // neighbouring classes of a lane
  float z[E];
  int c[E];  // their class numbers
};

// -inf beyond the classes
template <int E, typename T>
__device__ __forceinline__ void load_few(const T* row, int n, int lane, int bits, Few<E>& f) {
  constexpr int W = Few<E>::W;
#pragma unroll
  for (int k = 0; k < E / W; ++k) {
    const int c = ((k << bits) + lane) * W;
    float v[W];
    if (c + W <= n) {
      load_vec<W>(row + c, v);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = c + i < n ? (float)row[c + i] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) f.z[k * W + i] = v[i], f.c[k * W + i] = c + i;
  }
}

// log(1 + s) for s >= 0 to the last digits of s: what 1 + s rounds away comes back as c / (1 + s)
__device__ __forceinline__ float log_one_plus(float s) {
  const float u = 1.0f + s, c = s - (u - 1.0f);
  return __builtin_fmaf(c, fast_rcp(u), __builtin_amdgcn_logf(u) * kLn2);
}

template <int E>
__device__ __forceinline__ RowStats few_stats(const Few<E>& f, int bits) {
  float m = f.z[0];
#pragma unroll
  for (int i = 1; i < E; ++i) m = __builtin_fmaxf(m, f.z[i]);
  m = lanes_max(m, bits);
  const float ref = m == -INFINITY ? 0.0f : m;
  float s = 0.0f, u = 0.0f, ones = 0.0f;  // (a NaN, or the NaN of inf - inf, reaches s and all that comes of it)
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float d = f.z[i] - ref, e = fast_exp2(d * kLog2e);
    ones += d == 0.0f ? 1.0f : 0.0f;
    s += d == 0.0f ? 0.0f : e;
    u = __builtin_fmaf(e, __builtin_fmaxf(d, -150.0f), u);  // (e is 0 there, and 0 x -inf is not wanted)
  }
  s = lanes_sum(s, bits);
  ones = lanes_sum(ones, bits);
  u = lanes_sum(u, bits);
  if (m == -INFINITY && s == 0.0f) return {m, 0.0f, 0.0f};
  s += ones - 1.0f;
  const float log_sum = log_one_plus(s);
  return {ref, log_sum, log_sum - u * fast_rcp(1.0f + s)};
}

// ONE: a row is one lane's (bits = 0, known to the compiler)
template <typename T, int E, bool ONE, bool TOP>
__global__ __launch_bounds__(256) void few_classes_kernel(const T* __restrict__ logits, int64_t n_rows, int32_t n, int64_t ld, int32_t lane_bits, Tokens tok,
                                                          int32_t n_top, float* __restrict__ logprob, float* __restrict__ entropy,
                                                          float* __restrict__ stats, int32_t* __restrict__ top_ids, float* __restrict__ top_logprob) {
  const int bits = ONE ? 0 : lane_bits, lane = threadIdx.x & ((1 << bits) - 1);
  const int64_t step = (int64_t)gridDim.x * (256 >> bits);
  for (int64_t i = (int64_t)blockIdx.x * (256 >> bits) + (threadIdx.x >> bits); i < n_rows; i += step) {
    const int64_t t = tok.p ? token_at(tok, i) : 0;
    const bool skip = tok.p && t == tok.ignore;
    RowStats r{0.0f, 0.0f, 0.0f};
    Few<E> f;
    if (!skip) {
      load_few<E>(logits + i * ld, n, lane, bits, f);
      r = few_stats<E>(f, bits);
    }
    if (logprob && tok.p) {
      float lp = 0.0f;
      if (!skip) {
        lp = __builtin_nanf("");
        bool mine = lane == 0 && !(t >= 0 && t < n);  // the lane that holds the token's class, or the first one for a wrong token
#pragma unroll
        for (int k = 0; k < E; ++k)
          if (f.c[k] == t && t < n) lp = log_prob(r, f.z[k]), mine = true;
        if (mine) logprob[i] = lp;
      } else if (lane == 0) {
        logprob[i] = lp;
      }
    }
    if (lane == 0) {
      if (entropy) entropy[i] = r.entropy;
      if (stats) stats[3 * i] = r.m, stats[3 * i + 1] = r.log_sum, stats[3 * i + 2] = r.entropy;
    }
    if constexpr (!TOP) continue;
    if (skip) {
      for (int k = lane; k < n_top; k += 1 << bits) top_ids[i * n_top + k] = -1, top_logprob[i * n_top + k] = 0.0f;
      continue;
    }
    uint32_t key[E];  // 0: no class
#pragma unroll
    for (int q = 0; q < E; ++q) key[q] = f.c[q] < n ? order_key(f.z[q]) : 0;
    if constexpr (E <= 4) {
      if (3 * n_top > 2 << bits) {  // (a lane's classes are counted in two thirds of the time of a round below)
        // Every class counts how many are better -- of an equal logit, those of lower classes -- and writes itself to that place.  Classes go
        // by (vector, lane, place in the vector).
        constexpr int W = Few<E>::W;
        int rank[E];
#pragma unroll
        for (int q = 0; q < E; ++q) {
          rank[q] = 0;
#pragma unroll
          for (int o = 0; o < E; ++o) rank[q] += o < q ? key[o] >= key[q] : key[o] > key[q];
        }
        if constexpr (!ONE) {
          for (int l = 0; l < 1 << bits; ++l) {
            uint32_t least[E];  // what a class of lane l in the same vector has to exceed
#pragma unroll
            for (int q = 0; q < E; ++q) least[q] = key[q] - (l < lane ? 1 : 0);
#pragma unroll
            for (int o = 0; o < E; ++o) {
              uint32_t other = (uint32_t)__shfl((int)key[o], l, 1 << bits);
              if (l == lane) other = 0;
#pragma unroll
              for (int q = 0; q < E; ++q) rank[q] += other > (o / W < q / W ? key[q] - 1 : o / W > q / W ? key[q] : least[q]);
            }
          }
        }
#pragma unroll
        for (int q = 0; q < E; ++q) {
          if (key[q] != 0 && rank[q] < n_top)
            top_ids[i * n_top + rank[q]] = f.c[q], top_logprob[i * n_top + rank[q]] = log_prob(r, key_value(key[q]));
        }
        continue;
      }
    }
    for (int k = 0; k < n_top; ++k) {  // the best one that is left, n_top times
      uint32_t mine = key[0];
      int c = f.c[0];
#pragma unroll
      for (int q = 1; q < E; ++q)
        if (key[q] > mine) mine = key[q], c = f.c[q];
      const uint32_t best = lanes_reduce_u32(mine, bits, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
      const int id = (int)lanes_reduce_u32(mine == best ? (uint32_t)c : 0x7fffffffu, bits, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
#pragma unroll
      for (int q = 0; q < E; ++q)
        if (f.c[q] == id) key[q] = 0;
      if (lane == 0) top_ids[i * n_top + k] = id, top_logprob[i * n_top + k] = log_prob(r, key_value(best));
    }
  }
}

template <typename T, int E, bool ONE>
__global__ __launch_bounds__(256) void few_classes_backward_kernel(const T* logits, int64_t n_rows, int32_t n, int64_t ld, int32_t lane_bits, Tokens tok,
                                                                   const float* __restrict__ g_logprob, const float* __restrict__ g_entropy, T* out,
                                                                   int64_t ld_out) {
  constexpr int W = Few<E>::W;
  const int bits = ONE ? 0 : lane_bits, lane = threadIdx.x & ((1 << bits) - 1);
  const int64_t step = (int64_t)gridDim.x * (256 >> bits);
  for (int64_t i = (int64_t)blockIdx.x * (256 >> bits) + (threadIdx.x >> bits); i < n_rows; i += step) {
    const int64_t t = tok.p ? token_at(tok, i) : -1;
    const bool skip = tok.p && t == tok.ignore;
    RowStats r{-INFINITY, 0.0f, 0.0f};
    Few<E> f;
    float g = 0.0f, h = 0.0f;
    if (!skip) {
      g = g_logprob ? g_logprob[i] : 0.0f, h = g_entropy ? g_entropy[i] : 0.0f;
      load_few<E>(logits + i * ld, n, lane, bits, f);
      r = few_stats<E>(f, bits);
    }
    const RowGrad what = row_grad(skip, r, g_logprob && !(t >= 0 && t < n));
    float given = 0.0f;
#pragma unroll
    for (int k = 0; k < E; ++k) given = f.c[k] == t ? f.z[k] : given;
    given = grad_of_given(r, given, g, h);
#pragma unroll
    for (int k = 0; k < E / W; ++k) {
      const int c = ((k << bits) + lane) * W;
      float v[W];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        v[w] = what == kZeros ? 0.0f : what == kNans ? __builtin_nanf("") : c + w == t ? given : grad_at(r, f.z[k * W + w], g, h);
      }
      T* o = out + i * ld_out + c;
      if (c + W <= n) {
        store_vec<W>(o, v);
      } else {
#pragma unroll
        for (int w = 0; w < W; ++w)
          if (c + w < n) o[w] = (T)v[w];
      }
    }
  }
}

// ---- more classes: a wavefront walks a row or a slice of it ---------------------------------------------------------------------
constexpr int kVectors = 4;  // 16-byte vectors of a lane in a piece
constexpr int kMaxSlices = 64;

// A row in aligned 16-byte vectors and what is left at its two ends.
template <typename T>
struct Layout {
  static constexpr int W = 16 / sizeof(T);
  int head, n_vec, tail;
  __device__ __forceinline__ Layout(const T* row, int n) {
    head = (int)((-(reinterpret_cast<uintptr_t>(row) / sizeof(T))) & (W - 1));
    if (head > n) head = n;
    n_vec = (n - head) / W;
    tail = n - head - n_vec * W;
  }
};

// The maximum m, and S = sum 2^d, U = sum 2^d d over d = (z - m) log2(e); m = -inf, S = 0: nothing yet.  (The difference is taken first:
// z log2(e) - m log2(e) in one FMA would overflow for logits of the type's lowest value.)
struct Running {
  float m, s, u;
};
// x's sums moved to the maximum m >= x.m.  (S of a part that has seen only -inf is 0, or NaN; 2^-200 counts for nothing, and 0 x -inf is
// not wanted.)
__device__ __forceinline__ Running moved(const Running& x, float m) {
  const float ref = m == -INFINITY ? 0.0f : m;
  const float d = x.m == -INFINITY ? 0.0f : __builtin_fmaxf((x.m - ref) * kLog2e, -200.0f), f = fast_exp2(d);
  return {m, f * x.s, f * __builtin_fmaf(d, x.s, x.u)};
}
__device__ __forceinline__ Running merged(const Running& a, const Running& b) {
  const float m = __builtin_fmaxf(a.m, b.m);
  const Running x = moved(a, m), y = moved(b, m);
  return {m, x.s + y.s, x.u + y.u};
}
__device__ __forceinline__ Running wave_merged(const Running& r) {
  const Running x = moved(r, lanes_max(r.m, 6));
  return {x.m, wave_sum(x.s), wave_sum(x.u)};
}
__device__ __forceinline__ RowStats finish(const Running& r) {
  if (r.m == -INFINITY && r.s == 0.0f) return {r.m, 0.0f, 0.0f};
  const float log_sum = logf(r.s);
  return {r.m == -INFINITY ? 0.0f : r.m, log_sum, log_sum - kLn2 * r.u / r.s};
}

// What the lanes of a wavefront have stored to LDS, all of them read from here on.  (A wavefront's LDS accesses are carried out in order: this
// keeps the compiler from changing it.)
__device__ __forceinline__ void wave_meets() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Candidates of one wavefront in LDS: (key, ~class) as one number, larger is better.
struct Candidates {
  uint64_t* list;  // [128]
  int n, k;        // collected, wanted
  float bound;     // a class below it is none of the k best
  uint64_t worst;  // the k-th best of those ranked so far, or 0
  int ranked;      // how many at the list's front are in order already

  __device__ __forceinline__ void start(uint64_t* lds, int wanted) { list = lds, n = 0, k = wanted, bound = -INFINITY, worst = 0, ranked = 0; }

  // the lanes of `has` add theirs; a full list is ranked first
  __device__ __forceinline__ void add(bool has, uint64_t cand) {
    uint64_t mask = __ballot(has && cand > worst);
    if (!mask) return;
    if (n > 64) {
      rank();
      mask = __ballot(has && cand > worst);
    }
    if (mask >> (threadIdx.x & 63) & 1) list[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = cand;
    n += __popcll(mask);
    wave_meets();
  }

  // the k best, in order, to the front of the list: everyone counts how many are better than its one or two
  __device__ void rank() {
    if (n == ranked) return;
    const int lane = threadIdx.x & 63;
    wave_meets();
    const uint64_t a = lane < n ? list[lane] : 0, b = lane + 64 < n ? list[lane + 64] : 0;
    int ra = 0, rb = 0;
    if (n <= 64) {
#pragma unroll 8
      for (int i = 0; i < n; ++i) ra += list[i] > a;
    } else {
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const uint64_t o = list[i];
        ra += o > a, rb += o > b;
      }
    }
    wave_meets();
    if (lane < n && ra < k) list[ra] = a;
    if (lane + 64 < n && rb < k) list[rb] = b;
    wave_meets();
    if (n >= k) {
      n = k;
      worst = list[k - 1];
      const float v = key_value((uint32_t)(worst >> 32));
      bound = v;  // (a NaN bound lets every class through to the comparison with `worst`)
    }
    ranked = n;
  }
};
__device__ __forceinline__ uint64_t candidate(float z, int c) { return (uint64_t)order_key(z) << 32 | (uint32_t)~c; }

// The k-th largest of the maxima of 64 lanes, or of 16 quads where that is enough: at least k classes are no smaller.
__device__ __forceinline__ float first_bound(float lane_max, int k) {
  int rank = 0;
  const int lane = threadIdx.x & 63;
  if (k <= 8) {
    const float q = lanes_max(lane_max, 2);
    for (int i = 0; i < 64; i += 4) {
      const float o = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(q), i));
      rank += o > q || (o == q && i < (lane & ~3));
    }
    lane_max = q;
    const uint64_t hit = __ballot(rank == k - 1);
    return hit ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(lane_max), __builtin_ctzll(hit))) : -INFINITY;
  }
  for (int i = 0; i < 64; ++i) {
    const float o = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(lane_max), i));
    rank += o > lane_max || (o == lane_max && i < lane);
  }
  const uint64_t hit = __ballot(rank == k - 1);
  return hit ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(lane_max), __builtin_ctzll(hit))) : -INFINITY;
}

// What a slice leaves for the join: m, S, U and its k best candidates.
struct Slices {
  int32_t n;        // of a row; 1: no join
  float* running;   // [row][slice][3]
  uint64_t* best;   // [row][slice][n_top]
};

struct ManyOut {
  float *logprob, *entropy, *stats;
  int32_t* top_ids;
  float* top_logprob;
};

// one row's results, by the lanes of one wavefront
template <typename T>
__device__ __forceinline__ void write_row(const ManyOut& out, int64_t i, const T* row, int n, int64_t t, bool have_token, const RowStats& r, int n_top,
                                          const uint64_t* best) {
  const int lane = threadIdx.x & 63;
  if (lane == 0) {
    if (out.logprob && have_token) out.logprob[i] = t >= 0 && t < n ? log_prob(r, (float)row[t]) : __builtin_nanf("");
    if (out.entropy) out.entropy[i] = r.entropy;
    if (out.stats) out.stats[3 * i] = r.m, out.stats[3 * i + 1] = r.log_sum, out.stats[3 * i + 2] = r.entropy;
  }
  if (lane < n_top) {
    out.top_ids[i * n_top + lane] = (int)~(uint32_t)best[lane];
    out.top_logprob[i * n_top + lane] = log_prob(r, key_value((uint32_t)(best[lane] >> 32)));
  }
}
__device__ __forceinline__ void write_skipped(const ManyOut& out, int64_t i, int n_top) {
  const int lane = threadIdx.x & 63;
  if (lane == 0) {
    if (out.logprob) out.logprob[i] = 0.0f;
    if (out.entropy) out.entropy[i] = 0.0f;
    if (out.stats) out.stats[3 * i] = out.stats[3 * i + 1] = out.stats[3 * i + 2] = 0.0f;
  }
  if (lane < n_top) out.top_ids[i * n_top + lane] = -1, out.top_logprob[i * n_top + lane] = 0.0f;
}

template <typename T, bool TOP>
__global__ __launch_bounds__(256) void many_classes_kernel(const T* __restrict__ logits, int64_t n_rows, int32_t n, int64_t ld, Tokens tok, int32_t n_top,
                                                           Slices sl, ManyOut out) {
  constexpr int W = 16 / sizeof(T);
  using Vec = vec_t<T, W>;
  __shared__ uint64_t lds[4][128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n_units = n_rows * sl.n;
  for (int64_t unit = (int64_t)blockIdx.x * 4 + wave; unit < n_units; unit += (int64_t)gridDim.x * 4) {
    const int64_t i = unit / sl.n;
    const int slice = (int)(unit - i * sl.n);
    const int64_t t = tok.p ? token_at(tok, i) : 0;
    if (tok.p && t == tok.ignore) {
      if (sl.n == 1) write_skipped(out, i, n_top);
      continue;
    }
    const T* row = logits + i * ld;
    const Layout<T> at(row, n);
    const Vec* vecs = reinterpret_cast<const Vec*>(row + at.head);
    const int v0 = (int)((int64_t)at.n_vec * slice / sl.n), v1 = (int)((int64_t)at.n_vec * (slice + 1) / sl.n);
    // the row's ends, a class a lane: the head with the first slice (its classes come first), the tail with the last (last)
    const bool head = slice == 0 && lane < at.head, tail = slice == sl.n - 1 && lane < at.tail;
    const int tail_c = at.head + at.n_vec * W + lane;
    const float z_head = head ? (float)row[lane] : -INFINITY, z_tail = tail ? (float)row[tail_c] : -INFINITY;
    Vec raw[kVectors];
    auto fetch = [&](int v) {
#pragma unroll
      for (int q = 0; q < kVectors; ++q)
        raw[q] = v + q * 64 + lane < v1 ? vecs[v + q * 64 + lane] : Vec((T)-INFINITY);
    };
    fetch(v0);
    Running r{-INFINITY, 0.0f, 0.0f};
    auto take = [&](float z) {  // a class of the row's ends
      const bool any = z != -INFINITY;
      r = merged(r, Running{z, any ? (z - z == 0.0f ? 1.0f : __builtin_nanf("")) : 0.0f, 0.0f});
    };
    take(z_head);
    take(z_tail);
    Candidates best;
    if constexpr (TOP) {
      best.start(lds[wave], n_top);
    }
    for (int v = v0; v < v1; v += 64 * kVectors) {
      float z[kVectors][W];
#pragma unroll
      for (int q = 0; q < kVectors; ++q) {
#pragma unroll
        for (int w = 0; w < W; ++w) z[q][w] = (float)raw[q][w];
      }
      if (v + 64 * kVectors < v1) fetch(v + 64 * kVectors);
      float pm = z[0][0];
#pragma unroll
      for (int q = 0; q < kVectors; ++q)
#pragma unroll
        for (int w = 0; w < W; ++w) pm = __builtin_fmaxf(pm, z[q][w]);
      if (!(pm <= r.m)) {  // the lane's maximum moves
        r = moved(r, __builtin_fmaxf(pm, r.m));
      }
      const float ref = r.m == -INFINITY ? 0.0f : r.m;
#pragma unroll
      for (int q = 0; q < kVectors; ++q) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float d = (z[q][w] - ref) * kLog2e, e = fast_exp2(d);
          r.s += e;
          r.u = __builtin_fmaf(e, __builtin_fmaxf(d, -200.0f), r.u);
        }
      }
      if constexpr (TOP) {
        if (v == v0) {
          best.bound = first_bound(pm, n_top);
          best.add(head, candidate(z_head, lane));
        }
#pragma unroll
        for (int q = 0; q < kVectors; ++q) {
          const bool in = v + q * 64 + lane < v1;
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const bool may = !(z[q][w] < best.bound);
            if (__ballot(may)) best.add(may && in, candidate(z[q][w], at.head + (v + q * 64 + lane) * W + w));
          }
        }
        if (v == v0) best.rank();
      }
    }
    if constexpr (TOP) {
      if (v0 >= v1) best.add(head, candidate(z_head, lane));
      best.add(tail, candidate(z_tail, tail_c));
      best.rank();
    }
    r = wave_merged(r);
    if (sl.n == 1) {
      write_row(out, i, row, n, t, tok.p != nullptr, finish(r), TOP ? n_top : 0, lds[wave]);
    } else {
      if (lane == 0) {
        float* p = sl.running + unit * 3;
        p[0] = r.m, p[1] = r.s, p[2] = r.u;
      }
      if constexpr (TOP) {
        if (lane < n_top) sl.best[unit * n_top + lane] = lane < best.n ? best.list[lane] : 0;
      }
    }
    wave_meets();
  }
}

// The slices of a row, by one wavefront: a lane holds a slice's sums.
template <typename T>
__global__ __launch_bounds__(64) void join_slices_kernel(const T* __restrict__ logits, int64_t n_rows, int32_t n, int64_t ld, Tokens tok, int32_t n_top,
                                                         Slices sl, ManyOut out) {
  __shared__ uint64_t lds[128];
  const int lane = threadIdx.x;
  for (int64_t i = blockIdx.x; i < n_rows; i += gridDim.x) {
    const int64_t t = tok.p ? token_at(tok, i) : 0;
    if (tok.p && t == tok.ignore) {
      write_skipped(out, i, n_top);
      continue;
    }
    Running r{-INFINITY, 0.0f, 0.0f};
    if (lane < sl.n) {
      const float* p = sl.running + (i * sl.n + lane) * 3;
      r = {p[0], p[1], p[2]};
    }
    r = wave_merged(r);
    Candidates best;
    if (n_top > 0) {
      best.start(lds, n_top);
      // a lane holds a slice: its candidates come in order, so it is done at the first one below the bound
      const uint64_t* from = sl.best + (i * sl.n + (lane < sl.n ? lane : 0)) * n_top;
      uint64_t cand = lane < sl.n ? from[0] : 0;  // (0: no candidate)
      best.bound = first_bound(cand ? key_value((uint32_t)(cand >> 32)) : -INFINITY, n_top);
      for (int q = 0; q < n_top; ++q) {
        const bool may = cand != 0 && !(key_value((uint32_t)(cand >> 32)) < best.bound);
        if (!__ballot(may)) break;
        best.add(may, cand);
        cand = may && q + 1 < n_top ? from[q + 1] : 0;
      }
      best.rank();
    }
    write_row(out, i, logits + i * ld, n, t, tok.p != nullptr, finish(r), n_top, lds);
    wave_meets();
  }
}

// A workgroup per kVectors x 256 vectors of a row; the first one also takes the row's head, the last its tail.
template <typename T>
__global__ __launch_bounds__(256) void many_classes_backward_kernel(const T* logits, int64_t n_rows, int32_t n, int64_t ld, Tokens tok,
                                                                    const float* __restrict__ stats, const float* __restrict__ g_logprob,
                                                                    const float* __restrict__ g_entropy, T* out, int64_t ld_out, int32_t n_blocks) {
  constexpr int W = 16 / sizeof(T);
  using Vec = vec_t<T, W>;
  for (int64_t unit = blockIdx.x; unit < n_rows * n_blocks; unit += gridDim.x) {
    const int64_t i = unit / n_blocks;
    const int b = (int)(unit - i * n_blocks);
    const T* row = logits + i * ld;
    T* o = out + i * ld_out;
    const Layout<T> at(row, n);
    const Vec* vecs = reinterpret_cast<const Vec*>(row + at.head);
    const int v0 = b * kVectors * 256 + threadIdx.x;
    Vec raw[kVectors];
    const int64_t t = tok.p ? token_at(tok, i) : -1;
    const bool skip = tok.p && t == tok.ignore;
    if (!skip) {
#pragma unroll
      for (int q = 0; q < kVectors; ++q)
        if (v0 + q * 256 < at.n_vec) raw[q] = vecs[v0 + q * 256];
    }
    const RowStats r{stats[3 * i], stats[3 * i + 1], stats[3 * i + 2]};
    const float g = g_logprob ? g_logprob[i] : 0.0f, h = g_entropy ? g_entropy[i] : 0.0f;
    const RowGrad what = row_grad(skip, r, g_logprob && !(t >= 0 && t < n));
    const float flat = what == kNans ? __builtin_nanf("") : 0.0f;
#pragma unroll
    for (int q = 0; q < kVectors; ++q) {
      const int v = v0 + q * 256;
      if (v >= at.n_vec) continue;
      const int c = at.head + v * W;
      float d[W];
#pragma unroll
      for (int w = 0; w < W; ++w) d[w] = flat;
      if (what == kFormula) {
#pragma unroll
        for (int w = 0; w < W; ++w) d[w] = grad_at(r, (float)raw[q][w], g, h);
        if (t >= c && t < c + W) {
          float given = 0.0f;
#pragma unroll
          for (int w = 0; w < W; ++w) given = c + w == t ? (float)raw[q][w] : given;
          given = grad_of_given(r, given, g, h);
#pragma unroll
          for (int w = 0; w < W; ++w) d[w] = c + w == t ? given : d[w];
        }
      }
      store_vec<W>(o + c, d);
    }
    const int tail_at = at.head + at.n_vec * W;
    const bool first = b == 0 && (int)threadIdx.x < at.head, last = b == n_blocks - 1 && (int)threadIdx.x < at.tail;
    for (int e = 0; e < 2; ++e) {
      if (!(e ? last : first)) continue;
      const int c = (e ? tail_at : 0) + threadIdx.x;
      o[c] = (T)(what != kFormula ? flat : c == t ? grad_of_given(r, (float)row[c], g, h) : grad_at(r, (float)row[c], g, h));
    }
  }
}

// How a forward call is divided beyond DC_STATS_FROM classes: about four wavefronts a SIMD, slices of at least 1 024 classes, none from 2 048
// rows on.  Calls in bf16, a wavefront a row against slices: 512 x 100 003 53 / 27 us, 1 024 x 100 003 54 / 42 us, 2 047 x 100 003 81 / 84 us,
// 2 048 x 100 003 81 / 84 us, 512 x 32 768 17 / 14 us; up to 8 192 classes the second launch is what counts (512 x 8 192 10.4 / 14.6 us).
int slices_of(int64_t n_rows, int32_t n_classes) {
  if (n_rows <= 0 || n_rows >= 2048 || n_classes < DC_STATS_FROM) return 1;
  int64_t s = (4096 + n_rows - 1) / n_rows;
  if (s > n_classes / 1024) s = n_classes / 1024;
  return (int)(s > kMaxSlices ? kMaxSlices : s < 1 ? 1 : s);
}

// Up to 512 classes: classes a lane and lanes a row, as a power of two.  4 neighbouring classes a lane and up to 16 lanes; then more of
// them a lane, so that four (two) rows share a wavefront's reductions.  4, 8 and 16 a lane, fp32, forward + backward: 524 352 x 16
// 13.6 + 17.1, 10.7 + 15.6 and 10.6 + 20.2 us; 400 000 x 64 34 + 43, 24 + 34 and 22 + 41 us; 300 000 x 128 51 + 76, 35 + 58 and 30 + 68 us: 8
// from 5 classes on are faster than the 4 taken here.
int few_classes_a_lane(int32_t n_classes) { return n_classes <= 2 ? 2 : n_classes <= 64 ? 4 : n_classes <= 128 ? 8 : 16; }
int lane_bits_of(int32_t n_classes) {
  int bits = 0;
  while (n_classes > few_classes_a_lane(n_classes) << bits) ++bits;
  return bits;
}

// calls f with the element type and the classes a lane
template <typename F>
int with_few(int32_t dtype, int32_t n_classes, F&& f) {
  return with_dtype(dtype, [&](auto t) {
    if (n_classes <= 2) return f(t, std::integral_constant<int, 2>{}, std::true_type{});
    if (n_classes <= 4) return f(t, std::integral_constant<int, 4>{}, std::true_type{});
    switch (few_classes_a_lane(n_classes)) {
      case 4: return f(t, std::integral_constant<int, 4>{}, std::false_type{});
      case 8: return f(t, std::integral_constant<int, 8>{}, std::false_type{});
      default: return f(t, std::integral_constant<int, 16>{}, std::false_type{});
    }
  });
}

int check_logits(const void* logits, int32_t dtype, int64_t n_rows, int32_t n_classes, int64_t row_stride, const void* tokens, int32_t token_type) {
  DC_REQUIRE(dtype_ok(dtype), "unknown element type");
  DC_REQUIRE(n_rows >= 0 && n_classes >= 1, "negative size");
  DC_REQUIRE(n_classes <= 1 << 30, "more than 2^30 classes");
  DC_REQUIRE(n_rows == 0 || logits, "null pointer");
  DC_REQUIRE(row_stride >= 0, "negative stride");
  DC_REQUIRE(token_type >= DC_TOKENS_I8 && token_type <= DC_TOKENS_I64, "unknown token type");
  DC_REQUIRE(aligned(logits, dtype_size(dtype)), "misaligned pointer");
  DC_REQUIRE(aligned(tokens, token_type == DC_TOKENS_I64 ? 8 : token_type == DC_TOKENS_I32 ? 4 : 1), "misaligned pointer");
  return DC_OK;
}

unsigned grid_of(int64_t blocks) { return (unsigned)(blocks < (1 << 22) ? blocks : 1 << 22); }

}  // namespace
}  // namespace dc

extern "C" int64_t dc_token_logprobs_workspace(int64_t n_rows, int32_t n_classes, int32_t n_top) {
  const int64_t s = dc::slices_of(n_rows, n_classes);
  return s > 1 ? n_rows * s * ((n_top > 0 ? n_top : 0) * 8 + 12) : 0;
}

extern "C" int dc_token_logprobs(void* stream, const void* d_logits, int32_t dtype, int64_t n_rows, int32_t n_classes, int64_t row_stride,
                                 const void* d_tokens, int32_t token_type, int64_t ignore_token, int32_t n_top, float* d_logprob, float* d_entropy,
                                 float* d_stats, int32_t* d_top_ids, float* d_top_logprob, void* d_workspace, int64_t workspace_bytes) {
  using namespace dc;
  if (int rc = check_logits(d_logits, dtype, n_rows, n_classes, row_stride, d_tokens, token_type)) return rc;
  DC_REQUIRE(n_top >= 0 && n_top <= n_classes && n_top <= DC_MAX_TOP, "n_top must be in [0, min(n_classes, 32)]");
  DC_REQUIRE(n_rows == 0 || n_top == 0 || (d_top_ids && d_top_logprob), "null pointer");
  const int64_t need = dc_token_logprobs_workspace(n_rows, n_classes, n_top);
  DC_REQUIRE(workspace_bytes >= need && (need == 0 || d_workspace) && aligned(d_workspace, 16), "workspace too small");
  if (n_rows == 0) return DC_OK;
  const Tokens tok{d_tokens, token_type, ignore_token};
  if (n_classes < DC_STATS_FROM) {
    const int bits = lane_bits_of(n_classes);
    return with_few(dtype, n_classes, [&](auto t, auto e, auto one) {
      using T = decltype(t);
      auto kernel = n_top > 0 ? few_classes_kernel<T, decltype(e)::value, decltype(one)::value, true> : few_classes_kernel<T, decltype(e)::value, decltype(one)::value, false>;
      kernel<<<dim3(grid_of((n_rows + (256 >> bits) - 1) / (256 >> bits))), dim3(256), 0, as_stream(stream)>>>(
          (const T*)d_logits, n_rows, n_classes, row_stride, bits, tok, n_top, d_logprob, d_entropy, d_stats, d_top_ids, d_top_logprob);
      DC_LAUNCH_CHECK();
      return DC_OK;
    });
  }
  const int s = slices_of(n_rows, n_classes);
  uint64_t* best = (uint64_t*)d_workspace;
  const Slices sl{s, (float*)(best + (s > 1 ? n_rows * s * n_top : 0)), best};
  const ManyOut out{d_logprob, d_entropy, d_stats, d_top_ids, d_top_logprob};
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 grid(grid_of((n_rows * s + 3) / 4));
    if (n_top > 0) many_classes_kernel<T, true><<<grid, dim3(256), 0, as_stream(stream)>>>((const T*)d_logits, n_rows, n_classes, row_stride, tok, n_top, sl, out);
    else many_classes_kernel<T, false><<<grid, dim3(256), 0, as_stream(stream)>>>((const T*)d_logits, n_rows, n_classes, row_stride, tok, n_top, sl, out);
    DC_LAUNCH_CHECK();
    if (s > 1) {
      join_slices_kernel<T><<<dim3(grid_of(n_rows)), dim3(64), 0, as_stream(stream)>>>((const T*)d_logits, n_rows, n_classes, row_stride, tok, n_top, sl, out);
      DC_LAUNCH_CHECK();
    }
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
  const Tokens tok{d_tokens, token_type, ignore_token};
  if (n_classes < DC_STATS_FROM) {
    const int bits = lane_bits_of(n_classes);
    return with_few(dtype, n_classes, [&](auto t, auto e, auto one) {
      using T = decltype(t);
      few_classes_backward_kernel<T, decltype(e)::value, decltype(one)::value><<<dim3(grid_of((n_rows + (256 >> bits) - 1) / (256 >> bits))), dim3(256), 0, as_stream(stream)>>>(
          (const T*)d_logits, n_rows, n_classes, row_stride, bits, tok, d_grad_logprob, d_grad_entropy, (T*)d_grad_logits, grad_stride);
      DC_LAUNCH_CHECK();
      return DC_OK;
    });
  }
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int per_block = kVectors * 256 * (16 / (int)sizeof(T)), n_blocks = (n_classes + per_block - 1) / per_block;
    many_classes_backward_kernel<T><<<dim3(grid_of(n_rows * n_blocks)), dim3(256), 0, as_stream(stream)>>>(
        (const T*)d_logits, n_rows, n_classes, row_stride, tok, d_stats, d_grad_logprob, d_grad_entropy, (T*)d_grad_logits, grad_stride, n_blocks);
    DC_LAUNCH_CHECK();
    return DC_OK;
  });
}
