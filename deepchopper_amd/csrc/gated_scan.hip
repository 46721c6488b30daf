// dc_gated_scan: h_t = a_t h_(t-1) + (1 - a_t) x_t with a = sigmoid(f), per channel of every sequence, and its backward pass.
//
// Arithmetic.  A gate has two weights, a and 1 - a, and fp32 holds only the smaller of them to full relative accuracy:
// p = min(a, 1 - a) = 1 / (1 + exp(|f|)).  Each step is a move by p from one operand towards the other,
//   f > 0: h' = h + p (x - h)        f <= 0: h' = x - p (x - h)
// so a gate that keeps 99.99 % for thousands of tokens loses no more than one that forgets at once (with a rounded, a h would
// drift by 2^-25 a step).  A span of steps is the map h -> H + A h; it carries both A and G = 1 - A and is applied with the
// smaller of them, for the same reason.  Weights below 2^-126 are 0.
// x - h can be beyond fp32 where a h + (1 - a) x is not, and is NaN for an infinite state.  A state (or gradient) that is not finite stays
// so to the end of a group's 8 tokens, a span's passes to the groups behind: the last one of every 8 tells, and at the end a thread walks
// such a channel once more, token after token, with the sure_ forms (100 001 x 256 fp32 with gradients: 229 us without that, 233 us with;
// 1 024 sequences of 500 - 1 500 x 256 bf16: 341 us both).
//
// Form.  HBM-bound: 3 elements of traffic per element forward, 5 backward, about 35 and 50 vector operations.  Lanes run along the
// channels (a row of 64 lanes is 256 contiguous bytes), time is divided: a workgroup's 8 wavefronts take 8 consecutive tokens each of
// a 64-token tile (narrow batches: 16 or 32 lanes a row and 32 or 16 such groups), keep them in registers, pass each other their
// maps through LDS and run the steps again from the state they then know.  Where sequences and channels alone do not fill the chip,
// a sequence is divided into chunks: a first kernel reads each chunk for its map alone, the second starts from the composed maps.
// Measured (a large copy: 4.7 TB/s): 1 024 sequences of 500 - 1 500 x 256 bf16 342 us = 4.6 TB/s; 255 of 20 - 4 001 x 768 fp16 forward 571 us =
// 4.2 TB/s, backward 965 us = 4.1 TB/s (vector work, 81 % busy both); one of 100 001 x 256 fp32 43 + 55 us and 37 + 94 us backward.  Channels
// that do not fill the lanes cost their idle ones and a check a row: 255 of 20 - 4 001 x 129 fp16 445 + 651 us, x 128 220 + 302 us.  Up to 16
// tokens: 16 384 x 16 x 256 bf16 forward 87 us = 4.6 TB/s, backward 225 us = 3.0 TB/s.
#include <initializer_list>
#include <type_traits>

#include "elem_io.h"

namespace dc {
namespace {

constexpr int kTile = 64;      // tokens between two states of d_saved
constexpr int kThreads = 512;  // a workgroup
constexpr int kSteps = 8;      // consecutive tokens of one group of lanes: their inputs live in registers
constexpr int kShort = 16;     // sequences up to here: a thread per channel, token after token

struct ScanArgs {
  const int64_t* begin;  // or null: dense sequences of max_len tokens
  const int64_t* end;
  int64_t n_tokens, max_len;
  int32_t n_seqs, n_channels, reverse;
  int32_t lane_bits;  // log2 of the lanes along the channels
  int32_t n_chunks;   // chunks of a sequence ...
  int64_t chunk;      // ... of so many tokens each (a multiple of the workgroup's tile)
  int32_t n_blocks;   // workgroups of the recurrence; those behind them are fill_rest's
  int32_t whole;      // every lane has channels and all strides are at most 2^20: tiles inside a sequence need no checks
};

// a value that is the same in all lanes, into scalar registers
__device__ __forceinline__ int64_t scalar(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// whether [b, e) is a sequence of this call; one that is not is refused
__device__ __forceinline__ bool fits(const ScanArgs& a, int64_t b, int64_t e) { return b >= 0 && e >= b && e <= a.n_tokens && e - b <= a.max_len; }

// A sequence in the order of the recurrence: its token j is row base + dir * j.
struct Seq {
  int64_t base, len;
  int32_t dir;
  bool ok;
  __device__ __forceinline__ Seq(const ScanArgs& a, int s) {
    const int64_t b = scalar(a.begin ? a.begin[s] : s * a.max_len), e = scalar(a.end ? a.end[s] : b + a.max_len);
    ok = fits(a, b, e);
    len = ok ? e - b : 0;
    base = a.reverse ? e - 1 : b;
    dir = a.reverse ? -1 : 1;
  }
  __device__ __forceinline__ int64_t row(int64_t j) const { return dir < 0 ? base - j : base + j; }
};

// The gate's smaller weight, with the gate's sign: non-negative where the state is what is moved, negative where x is.
__device__ __forceinline__ float signed_gate(float f) { return __builtin_copysignf(gate_minor(f), f); }
__device__ __forceinline__ bool keeps(float ps) { return __float_as_int(ps) >= 0; }
__device__ __forceinline__ float step(float h, float x, float ps) { return __builtin_fmaf(ps, x - h, keeps(ps) ? h : x); }
// a * v
__device__ __forceinline__ float decay(float v, float ps) { return keeps(ps) ? __builtin_fmaf(-ps, v, v) : -ps * v; }

__device__ __forceinline__ bool finite(float v) { return __builtin_fabsf(v) < INFINITY; }
template <int V>
__device__ __forceinline__ bool all_finite(const float (&h)[V]) {
  bool ok = true;
#pragma unroll
  for (int v = 0; v < V; ++v) ok = ok && finite(h[v]);
  return ok;
}
constexpr float kLeast = 1.17549435e-38f, kMost = 3.40282347e+38f;  // normal fp32 numbers

// The factor a of a state or gradient v: an infinite one stays infinite however small a is (where a is 0 in fp32 too).
__device__ __forceinline__ float weight_of(float a, float v) { return __builtin_fabsf(v) == INFINITY ? __builtin_fmaxf(a, kLeast) : a; }

// step and decay; where those leave fp32, from the two products (a step between finite operands does not leave them)
__device__ __forceinline__ float sure_step(float h, float x, float ps) {
  float r = step(h, x, ps);
  if (__builtin_expect(!finite(r), 0)) {
    const float p = __builtin_fabsf(ps), q = 1.0f - p;
    r = __builtin_fmaf(weight_of(keeps(ps) ? q : p, h), h, (keeps(ps) ? p : q) * x);
    if (finite(h) && finite(x)) r = __builtin_amdgcn_fmed3f(r, h, x);
  }
  return r;
}
__device__ __forceinline__ float sure_decay(float v, float ps) {
  const float r = decay(v, ps), p = __builtin_fabsf(ps);
  return finite(r) ? r : weight_of(keeps(ps) ? 1.0f - p : p, v) * v;
}

// One token's gradients from half of h_(t-1) - x_t (the whole may be beyond fp32) and g_t; g_t becomes a_t g_t.
__device__ __forceinline__ void sure_back(float& g, float ps, float half, float& dx, float& df) {
  const float p = __builtin_fabsf(ps), part = p * g, rest = finite(g) ? __builtin_fmaf(-p, g, g) : (1.0f - p) * g;
  dx = keeps(ps) ? part : rest;
  df = p * rest * half * 2.0f;
  g = sure_decay(g, ps);
}

// Comparisons made of ps so far are not kept (in scalar registers that spill) but made again.
template <int V>
__device__ __forceinline__ void forget(float (&ps)[kSteps][V]) {
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v) asm volatile("" : "+v"(ps[i][v]));
}

// x where it counts: a gate of +inf (or one whose other weight is 0 in fp32) does not look at it
__device__ __forceinline__ float seen(float x, float ps) { return __float_as_int(ps) == 0 ? 0.0f : x; }

// A span of steps: h -> H + A h, G = 1 - A
struct Span {
  float A, G, H;
};
__device__ __forceinline__ Span identity_span() { return {1.0f, 0.0f, 0.0f}; }
__device__ __forceinline__ float apply(float A, float G, float H, float h) {
  return A > 0.5f ? h + __builtin_fmaf(-G, h, H) : __builtin_fmaf(A, h, H);
}
__device__ __forceinline__ void extend(float& A, float& G, float ps) {  // by one step; G is what an input of 1 makes of a state of 0
  const float t = __builtin_fabsf(ps) * A;
  A = keeps(ps) ? A - t : t;
  G = step(G, 1.0f, ps);
}
__device__ __forceinline__ Span then(const Span& a, const Span& b) {  // a, then b
  return {a.A * b.A, __builtin_fmaf(b.G, 1.0f - a.G, a.G), apply(b.A, b.G, b.H, a.H)};
}
// apply where that leaves fp32: a state, between finite H and h, by rounding alone; a gradient (BACK) on the way
template <bool BACK>
__device__ __forceinline__ float sure_apply(float A, float G, float H, float h) {
  const float r = apply(A, G, H, h);
  if (finite(r)) return r;
  if (!BACK && finite(h) && finite(H)) return __builtin_amdgcn_fmed3f(r, -kMost, kMost);
  return __builtin_fmaf(weight_of(A, h), h, H);
}

__device__ __forceinline__ int64_t inside(const ScanArgs& a, int64_t t) { return t < 0 ? 0 : t > a.n_tokens ? a.n_tokens : t; }

// zero_rest, by the workgroups behind the recurrence's: the rows in front of the first and behind the last sequence to zero, and those of a
// refused sequence to NaN.  Every lane looks at a sequence; the wavefront writes the rows of those that are refused, one after the other.
template <typename T>
__device__ void fill_rest(const ScanArgs& a, T* y, int64_t ldy, T* y2, int64_t ldy2) {
  const int block = blockIdx.x - a.n_blocks, n_blocks = gridDim.x - a.n_blocks;
  int64_t b = a.n_tokens, e = a.n_tokens;
  if (a.n_seqs > 0) {
    b = inside(a, a.begin ? a.begin[0] : 0);
    e = inside(a, a.end ? a.end[a.n_seqs - 1] : a.n_seqs * a.max_len);
    e = e < b ? b : e;
  }
  for (int64_t i = block; i < b + a.n_tokens - e; i += n_blocks) {
    const int64_t t = i < b ? i : i - b + e;
    for (int c = threadIdx.x; c < a.n_channels; c += blockDim.x) {
      y[t * ldy + c] = (T)0.0f;
      if (y2) y2[t * ldy2 + c] = (T)0.0f;
    }
  }
  if (!a.begin) return;  // (dense sequences are checked on the host)
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  for (int64_t first = (int64_t)(block * waves + (int)(threadIdx.x >> 6)) * 64; first < a.n_seqs; first += (int64_t)n_blocks * waves * 64) {
    const int64_t s = first + lane;
    bool refused = false;
    if (s < a.n_seqs) b = a.begin[s], e = a.end[s], refused = !fits(a, b, e);
    for (uint64_t left = __ballot(refused); left; left &= left - 1) {
      const int64_t r = first + __builtin_ctzll(left), rb = inside(a, a.begin[r]), re = inside(a, a.end[r]);
      for (int64_t t = rb; t < re; ++t) {
        for (int c = lane; c < a.n_channels; c += 64) {
          y[t * ldy + c] = (T)__builtin_nanf("");
          if (y2) y2[t * ldy2 + c] = (T)__builtin_nanf("");
        }
      }
    }
  }
}

// workgroups of fill_rest (as small as 64 threads): a wavefront looks at no more than a few times 64 sequences
int rest_blocks(int64_t n_tokens, int32_t n_seqs, int32_t zero_rest) { return zero_rest && n_tokens > 0 ? 32 + n_seqs / 256 : 0; }

// Of an odd number of channels the last lane takes the last two and writes only the second: the first is its neighbour's.
template <int V, typename T>
__device__ __forceinline__ void store_channels(T* p, const float (&v)[V], bool second) {
  if (V == 2 && second) p[V - 1] = (T)v[V - 1];
  else store_vec<V>(p, v);
}

// ---- sequences of at most kShort tokens: a thread per V channels ---------------------------------------------------------------
constexpr int kWalkThreads = 64;

template <typename T, int V>
__global__ __launch_bounds__(kWalkThreads) void scan_walk_kernel(ScanArgs a, const T* __restrict__ x, int64_t ldx, const T* __restrict__ f, int64_t ldf,
                                                                 const float* h0, T* __restrict__ y, int64_t ldy, float* h_last) {
  if ((int)blockIdx.x >= a.n_blocks) return fill_rest<T>(a, y, ldy, nullptr, 0);
  const int per_seq = (a.n_channels + kWalkThreads * V - 1) / (kWalkThreads * V);
  const int s = blockIdx.x / per_seq;
  int c = (blockIdx.x % per_seq * kWalkThreads + threadIdx.x) * V;
  if (c >= a.n_channels) return;
  const bool second = c + V > a.n_channels;
  if (second) --c;
  const Seq q(a, s);
  const int64_t sc = (int64_t)s * a.n_channels + c;
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = h0 ? h0[sc + v] : 0.0f;
#pragma unroll 4
  for (int64_t j = 0; j < q.len; ++j) {
    const int64_t t = q.row(j);
    float xv[V], fv[V];
    load_vec<V>(x + t * ldx + c, xv);
    load_vec<V>(f + t * ldf + c, fv);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float ps = signed_gate(fv[v]);
      h[v] = sure_step(h[v], seen(xv[v], ps), ps);
    }
    store_channels<V>(y + t * ldy + c, h, second);
  }
  if (h_last) {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = q.ok ? h[v] : __builtin_nanf("");
    store_channels<V>(h_last + sc, h, second);
  }
}

// The states again from h0, kept in LDS, then the gradients from the last token back.
template <typename T, int V>
__global__ __launch_bounds__(kWalkThreads) void scan_walk_backward_kernel(ScanArgs a, const T* __restrict__ x, int64_t ldx, const T* __restrict__ f, int64_t ldf,
                                                                          const float* __restrict__ h0, const T* __restrict__ gy, int64_t ldgy,
                                                                          const float* g_last, T* __restrict__ gx, int64_t ldgx, T* __restrict__ gf,
                                                                          int64_t ldgf, float* g_h0) {
  if ((int)blockIdx.x >= a.n_blocks) return fill_rest<T>(a, gx, ldgx, gf, ldgf);
  __shared__ float half[kShort][kWalkThreads * V];  // of h_(t-1) - x_t
  const int per_seq = (a.n_channels + kWalkThreads * V - 1) / (kWalkThreads * V);
  const int s = blockIdx.x / per_seq;
  int c = (blockIdx.x % per_seq * kWalkThreads + threadIdx.x) * V;
  if (c >= a.n_channels) return;
  const bool second = c + V > a.n_channels;
  if (second) --c;
  const Seq q(a, s);
  const int64_t sc = (int64_t)s * a.n_channels + c;
  const int n = (int)q.len;
  float h[V], g[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = h0 ? h0[sc + v] : 0.0f, g[v] = g_last ? g_last[sc + v] : 0.0f;
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const int64_t t = q.row(j);
    float xv[V], fv[V];
    load_vec<V>(x + t * ldx + c, xv);
    load_vec<V>(f + t * ldf + c, fv);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float ps = signed_gate(fv[v]), xs = seen(xv[v], ps);
      half[j][threadIdx.x * V + v] = __builtin_fmaf(-0.5f, xs, 0.5f * h[v]);
      h[v] = sure_step(h[v], xs, ps);
    }
  }
#pragma unroll 4
  for (int j = n - 1; j >= 0; --j) {
    const int64_t t = q.row(j);
    float fv[V], yv[V], ox[V], of[V];
    load_vec<V>(f + t * ldf + c, fv);
    load_vec<V>(gy + t * ldgy + c, yv);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      g[v] += yv[v];
      sure_back(g[v], signed_gate(fv[v]), half[j][threadIdx.x * V + v], ox[v], of[v]);
    }
    store_channels<V>(gx + t * ldgx + c, ox, second);
    store_channels<V>(gf + t * ldgf + c, of, second);
  }
  if (g_h0) {
#pragma unroll
    for (int v = 0; v < V; ++v) g[v] = q.ok ? g[v] : __builtin_nanf("");
    store_channels<V>(g_h0 + sc, g, second);
  }
}

// ---- longer sequences: tiles of (kThreads >> lane_bits) groups of kSteps tokens --------------------------------------------------
// Which sequence, chunk, channels and group of tokens a thread works on.
template <int V>
struct Place {
  int s, chunk, group, n_groups, channel, slot;  // slot: of this thread's channels in a group's row of LDS
  bool active, second;                           // second: see store_channels
  __device__ __forceinline__ Place(const ScanArgs& a) {
    const int lanes = 1 << a.lane_bits, per_row = (a.n_channels + lanes * V - 1) / (lanes * V);
    const int lane = threadIdx.x & (lanes - 1);
    group = threadIdx.x >> a.lane_bits;
    n_groups = kThreads >> a.lane_bits;
    channel = ((int)blockIdx.x % per_row * lanes + lane) * V;
    chunk = (int)blockIdx.x / per_row % a.n_chunks;
    s = (int)blockIdx.x / per_row / a.n_chunks;
    slot = lane * V;
    active = channel < a.n_channels;
    second = active && channel + V > a.n_channels;
    if (second) --channel;
  }
  __device__ __forceinline__ int at(int grp, int lanes_v) const { return grp * lanes_v + slot; }
};

// kSteps rows of V channels, raw; rows from n on are not read
template <typename T, int V>
struct Rows {
  vec_t<T, V> r[kSteps];
  __device__ __forceinline__ void load(const T* p, int64_t ld, int n) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (i < n) {
        if constexpr (V == 1) r[i][0] = p[i * ld];
        else r[i] = *reinterpret_cast<const typename loose_vec<T, V>::type*>(p + i * ld);
      } else {
        r[i] = vec_t<T, V>(0);
      }
    }
  }
};

// The rows of a whole tile: a scalar base a row of a group and one 32-bit byte offset a lane (strides up to 2^20: ScanArgs.whole).
template <typename T, int V>
struct TileRows {
  int64_t first, per_step;  // elements from the row of a tile's first token to the lowest row of a group's step 0; from step to step
  uint32_t lane;            // bytes
  __device__ __forceinline__ TileRows(const Place<V>& at, const Seq& q, int64_t ld) {
    const int group = q.dir < 0 ? at.n_groups - 1 - at.group : at.group;
    first = q.dir < 0 ? -(int64_t)(at.n_groups - 1) * kSteps * ld : 0;
    per_step = q.dir * ld;
    lane = ((uint32_t)(group * kSteps) * (uint32_t)ld + (uint32_t)at.channel) * (uint32_t)sizeof(T);
  }
  // `tile`: the row of the tile's first token
  __device__ __forceinline__ void load(const T* tile, Rows<T, V>& to) const {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const char* p = reinterpret_cast<const char*>(tile + first + i * per_step) + lane;
      if constexpr (V == 1) to.r[i][0] = *reinterpret_cast<const T*>(p);
      else to.r[i] = *reinterpret_cast<const typename loose_vec<T, V>::type*>(p);
    }
  }
  __device__ __forceinline__ void store(T* tile, int i, const float (&v)[V]) const {
    store_vec<V>(reinterpret_cast<T*>(reinterpret_cast<char*>(tile + first + i * per_step) + lane), v);
  }
};

// Chunk maps in the workspace: [sequence][chunk][A, G, H][channel], and behind them the states the sequences start from.
__device__ __forceinline__ int64_t map_at(const ScanArgs& a, int s, int chunk, int k, int channel) {
  return (((int64_t)s * a.n_chunks + chunk) * 3 + k) * a.n_channels + channel;
}
__device__ __forceinline__ int64_t start_at(const ScanArgs& a, int s, int channel) {
  return ((int64_t)a.n_seqs * a.n_chunks * 3 + s) * a.n_channels + channel;
}

// The map of every chunk, forward (x is the third input) or backward (c -> Q + A c against the recurrence; gy is).  Every group of lanes
// walks its own part of the chunk; one exchange at the end.  `start` (h0 or the gradient of h_last, or null) is copied behind the maps:
// the second kernel may then write where it came from.
template <typename T, int V, bool BACK>
__global__ __launch_bounds__(kThreads) void scan_map_kernel(ScanArgs a, const T* __restrict__ f, int64_t ldf, const T* __restrict__ x, int64_t ldx,
                                                            const float* start, float* __restrict__ maps) {
  __shared__ float lds[3][kThreads * V];
  const Place<V> at(a);
  const Seq q(a, at.s);
  const int lanes_v = V << a.lane_bits;
  const int64_t j0 = at.chunk * a.chunk, part = a.chunk / at.n_groups;
  if (at.chunk == 0 && at.active && at.group == 0) {
    for (int v = at.second ? 1 : 0; v < V; ++v)
      maps[start_at(a, at.s, at.channel + v)] = start ? start[(int64_t)at.s * a.n_channels + at.channel + v] : 0.0f;
  }
  if (j0 >= q.len) return;
  const int64_t p0 = j0 + at.group * part, p1 = p0 + part < q.len ? p0 + part : q.len;
  Span m[V];
#pragma unroll
  for (int v = 0; v < V; ++v) m[v] = identity_span();
  if (at.active) {
    const int64_t sf = q.dir * ldf, sx = q.dir * ldx;
    const int n_blocks = p1 > p0 ? (int)((p1 - p0 + kSteps - 1) / kSteps) : 0;
    for (int b = 0; b < n_blocks; ++b) {
      const int64_t j = p0 + (int64_t)(BACK ? n_blocks - 1 - b : b) * kSteps;
      const int n = p1 - j < kSteps ? (int)(p1 - j) : kSteps;
      Rows<T, V> rf, rx;
      rf.load(f + q.row(j) * ldf + at.channel, sf, n);
      rx.load(x + q.row(j) * ldx + at.channel, sx, n);
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const int i = BACK ? kSteps - 1 - k : k;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float ps = i < n ? signed_gate((float)rf.r[i][v]) : 0.0f, xv = (float)rx.r[i][v];
          extend(m[v].A, m[v].G, ps);
          m[v].H = BACK ? decay(m[v].H + xv, ps) : step(m[v].H, seen(xv, ps), ps);
        }
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (__builtin_expect(!finite(m[v].H), 0)) {
      m[v].H = 0.0f;
      for (int64_t k = p0; k < p1; ++k) {
        const int64_t t = q.row(BACK ? p1 - 1 - (k - p0) : k);
        const float ps = signed_gate((float)f[t * ldf + at.channel + v]), xv = (float)x[t * ldx + at.channel + v];
        m[v].H = BACK ? sure_decay(m[v].H + xv, ps) : sure_step(m[v].H, seen(xv, ps), ps);
      }
    }
    const int i = at.at(at.group, lanes_v) + v;
    lds[0][i] = m[v].A, lds[1][i] = m[v].G, lds[2][i] = m[v].H;
  }
  __syncthreads();
  if (at.group != 0 || !at.active) return;
  for (int v = at.second ? 1 : 0; v < V; ++v) {
    Span all = identity_span();
    for (int k = 0; k < at.n_groups; ++k) {
      const int i = at.at(BACK ? at.n_groups - 1 - k : k, lanes_v) + v;
      const float H = sure_apply<BACK>(lds[0][i], lds[1][i], lds[2][i], all.H);
      all = then(all, Span{lds[0][i], lds[1][i], lds[2][i]});
      all.H = H;
    }
    maps[map_at(a, at.s, at.chunk, 0, at.channel + v)] = all.A;
    maps[map_at(a, at.s, at.chunk, 1, at.channel + v)] = all.G;
    maps[map_at(a, at.s, at.chunk, 2, at.channel + v)] = all.H;
  }
}

// What a chunk starts from: the sequence's start through the maps of chunks [from, from + n) (dir 1) or (from, from - n] downwards
// (dir -1); the groups of lanes compose a part each.  Ends with a barrier behind the last use of `lds`.
template <int V>
__device__ void compose_chunks(const ScanArgs& a, const Place<V>& at, const float* __restrict__ maps, int from, int dir, int n, float (*lds)[kThreads * V],
                               float (&h)[V]) {
  const int lanes_v = V << a.lane_bits;
  Span m[V];
#pragma unroll
  for (int v = 0; v < V; ++v) m[v] = identity_span();
  if (at.active) {
    const int lo = (int)((int64_t)n * at.group / at.n_groups), hi = (int)((int64_t)n * (at.group + 1) / at.n_groups);
#pragma unroll 4
    for (int k = lo; k < hi; ++k) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int64_t i = map_at(a, at.s, from + dir * k, 0, at.channel + v);
        m[v] = then(m[v], Span{maps[i], maps[i + a.n_channels], maps[i + 2 * (int64_t)a.n_channels]});
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = at.at(at.group, lanes_v) + v;
    lds[0][i] = m[v].A, lds[1][i] = m[v].G, lds[2][i] = m[v].H;
    h[v] = at.active ? maps[start_at(a, at.s, at.channel + v)] : 0.0f;
  }
  __syncthreads();
  for (int k = 0; k < at.n_groups; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = at.at(k, lanes_v) + v;
      h[v] = apply(lds[0][i], lds[1][i], lds[2][i], h[v]);
    }
  }
  __syncthreads();
}

// What a chunk starts from, by one thread with the sure forms: `start` (h0 or the gradient of h_last, or null) where there are no maps.
template <bool BACK, int V>
__device__ __forceinline__ void sure_start(const ScanArgs& a, const Place<V>& at, const float* maps, const float* start, int from, int dir, int n, float (&h)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    h[v] = maps ? maps[start_at(a, at.s, at.channel + v)] : start ? start[(int64_t)at.s * a.n_channels + at.channel + v] : 0.0f;
    for (int k = 0; maps && k < n; ++k) {
      const int64_t i = map_at(a, at.s, from + dir * k, 0, at.channel + v);
      h[v] = sure_apply<BACK>(maps[i], maps[i + a.n_channels], maps[i + 2 * (int64_t)a.n_channels], h[v]);
    }
  }
}

// A kernel's own arguments, loaded (again) where this stands: what only the second walk looks at is not kept in (spilling) scalar registers
// through the loops in front of it (3 300 sequences of 29 - 38 x 43 fp32: 24.2 us kept, 22.9 us loaded).  Arguments lie one after the
// other, each at its alignment; these structs name them in the kernels' order.
template <typename Args>
__device__ __forceinline__ const Args& own_arguments() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const Args*)p;
}

// scan_tile_kernel's
template <typename T>
struct TileArgs {
  ScanArgs a;
  const T* x;
  int64_t ldx;
  const T* f;
  int64_t ldf;
  const float* h0;
  T* y;
  int64_t ldy;
  float *h_last, *saved;
  const float* maps;
};
// scan_tile_backward_kernel's
template <typename T>
struct TileBackArgs {
  ScanArgs a;
  const T* x;
  int64_t ldx;
  const T* f;
  int64_t ldf;
  const float *h0, *saved;
  const T* gy;
  int64_t ldgy;
  const float* g_last;
  T* gx;
  int64_t ldgx;
  T* gf;
  int64_t ldgf;
  float* g_h0;
  const float* maps;
};

// A chunk's tokens for a thread's channels, one after the other, with the sure forms: the states written again; h: the last one.
template <typename T, int V>
__device__ __forceinline__ void sure_walk(const TileArgs<T>& k, float (&h)[V]) {
  const Place<V> at(k.a);
  const Seq q(k.a, at.s);
  const int64_t j0 = at.chunk * k.a.chunk, j1 = j0 + k.a.chunk < q.len ? j0 + k.a.chunk : q.len;
  sure_start<false, V>(k.a, at, k.maps, k.h0, 0, 1, at.chunk, h);
#pragma unroll 1
  for (int64_t j = j0; j < j1; ++j) {
    const int64_t t = q.row(j);
    if (k.saved && j % kTile == 0 && j > 0) store_channels<V>(k.saved + (t / kTile * k.a.n_channels + at.channel), h, at.second);
    float xv[V], fv[V];
    load_vec<V>(k.x + t * k.ldx + at.channel, xv);
    load_vec<V>(k.f + t * k.ldf + at.channel, fv);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float ps = signed_gate(fv[v]);
      h[v] = sure_step(h[v], seen(xv[v], ps), ps);
    }
    store_channels<V>(k.y + t * k.ldy + at.channel, h, at.second);
  }
}

// ... and their gradients, from the last token back, kTile tokens from each state of `saved`; c: what comes out of the first one.  `lds`:
// half of h_(t-1) - x_t for kTile tokens.
template <typename T, int V>
__device__ __forceinline__ void sure_walk_back(const TileBackArgs<T>& k, float* lds, float (&c)[V]) {
  const Place<V> at(k.a);
  const Seq q(k.a, at.s);
  const int64_t j0 = at.chunk * k.a.chunk, j1 = j0 + k.a.chunk < q.len ? j0 + k.a.chunk : q.len;
  const int last = q.len > 0 ? (int)((q.len - 1) / k.a.chunk) : 0, lanes_v = V << k.a.lane_bits;
  float* half = lds + at.slot;
  sure_start<true, V>(k.a, at, k.maps, k.g_last, last, -1, last - at.chunk, c);
#pragma unroll 1
  for (int64_t jt = j0 + (j1 - j0 - 1) / kTile * kTile; j1 > j0 && jt >= j0; jt -= kTile) {
    const int n = j1 - jt < kTile ? (int)(j1 - jt) : kTile;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
      h[v] = jt > 0 ? k.saved[q.row(jt) / kTile * k.a.n_channels + at.channel + v] : k.h0 ? k.h0[(int64_t)at.s * k.a.n_channels + at.channel + v] : 0.0f;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int64_t t = q.row(jt + i);
      float xv[V], fv[V];
      load_vec<V>(k.x + t * k.ldx + at.channel, xv);
      load_vec<V>(k.f + t * k.ldf + at.channel, fv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float ps = signed_gate(fv[v]), xs = seen(xv[v], ps);
        half[i * lanes_v + v] = __builtin_fmaf(-0.5f, xs, 0.5f * h[v]);
        h[v] = sure_step(h[v], xs, ps);
      }
    }
#pragma unroll 1
    for (int i = n - 1; i >= 0; --i) {
      const int64_t t = q.row(jt + i);
      float fv[V], yv[V], dx[V], df[V];
      load_vec<V>(k.f + t * k.ldf + at.channel, fv);
      load_vec<V>(k.gy + t * k.ldgy + at.channel, yv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        c[v] += yv[v];
        sure_back(c[v], signed_gate(fv[v]), half[i * lanes_v + v], dx[v], df[v]);
      }
      store_channels<V>(k.gx + t * k.ldgx + at.channel, dx, at.second);
      store_channels<V>(k.gf + t * k.ldgf + at.channel, df, at.second);
    }
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads, 4) void scan_tile_kernel(ScanArgs a, const T* __restrict__ x, int64_t ldx, const T* __restrict__ f, int64_t ldf,
                                                                const float* h0, T* __restrict__ y, int64_t ldy, float* h_last,
                                                                float* __restrict__ saved, const float* __restrict__ maps) {
  __shared__ float lds[2][3][kThreads * V], ends[2][64 * V];
  __shared__ int lost[64];  // a lane's states left the finite numbers somewhere
  if ((int)blockIdx.x >= a.n_blocks) return fill_rest<T>(a, y, ldy, nullptr, 0);
  const Place<V> at(a);
  const Seq q(a, at.s);
  const int lanes_v = V << a.lane_bits, tile = at.n_groups * kSteps;
  const int64_t sc = (int64_t)at.s * a.n_channels + at.channel;
  const int64_t j0 = at.chunk * a.chunk, j1 = j0 + a.chunk < q.len ? j0 + a.chunk : q.len;
  if (j0 >= q.len && at.chunk > 0) return;
  if (threadIdx.x < 64) lost[threadIdx.x] = 0;  // (set behind the chunks' barriers or the last tile's; with neither there is nothing to walk)
  float carry[V];
  if (maps) {
    compose_chunks<V>(a, at, maps, 0, 1, at.chunk, lds[0], carry);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = h0 && at.active ? h0[sc + v] : 0.0f;
  }
  float trace = 0.0f;  // NaN once something is not finite
#pragma unroll
  for (int v = 0; v < V; ++v) trace = __builtin_fmaf(carry[v], 0.0f, trace);
  const TileRows<T, V> tx(at, q, ldx), tf(at, q, ldf), ty(at, q, ldy);
  const int64_t sx = q.dir * ldx, sf = q.dir * ldf, sy = q.dir * ldy;
  const bool last_group = at.group == at.n_groups - 1;
  int turn = 0;
  auto one_tile = [&](auto whole, int64_t jt) {
    constexpr bool WHOLE = decltype(whole)::value;
    const int64_t j = jt + at.group * kSteps, left = j1 - j;
    const int n = WHOLE ? kSteps : !at.active || left <= 0 ? 0 : left < kSteps ? (int)left : kSteps;
    Rows<T, V> rx, rf;
    if constexpr (WHOLE) {
      const int64_t row = q.row(jt);
      tx.load(x + row * ldx, rx);
      tf.load(f + row * ldf, rf);
    } else {
      rx.load(x + q.row(j) * ldx + at.channel, sx, n);
      rf.load(f + q.row(j) * ldf + at.channel, sf, n);
    }
    float xs[kSteps][V], ps[kSteps][V];
    Span m[V];
#pragma unroll
    for (int v = 0; v < V; ++v) m[v] = identity_span();
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        ps[i][v] = WHOLE || i < n ? signed_gate((float)rf.r[i][v]) : 0.0f;
        xs[i][v] = seen((float)rx.r[i][v], ps[i][v]);
        extend(m[v].A, m[v].G, ps[i][v]);
        m[v].H = step(m[v].H, xs[i][v], ps[i][v]);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = at.at(at.group, lanes_v) + v;
      lds[turn][0][i] = m[v].A, lds[turn][1][i] = m[v].G, lds[turn][2][i] = m[v].H;
    }
    __syncthreads();  // (one a tile: the next tile writes the other halves)
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = jt == j0 ? carry[v] : ends[turn ^ 1][at.slot + v];
    for (int k = 0; k < at.group; ++k) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = at.at(k, lanes_v) + v;
        h[v] = apply(lds[turn][0][i], lds[turn][1][i], lds[turn][2][i], h[v]);
      }
    }
    if (WHOLE || n > 0) {
      forget<V>(ps);
      if (saved && j % kTile == 0 && j > 0) {
        store_channels<V>(saved + (q.row(j) / kTile * a.n_channels + at.channel), h, at.second);
      }
      T* out = y + q.row(j) * ldy + at.channel;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = step(h[v], xs[i][v], ps[i][v]);
        if constexpr (WHOLE) ty.store(y + q.row(jt) * ldy, i, h);
        else if (i < n) store_channels<V>(out + i * sy, h, at.second);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) trace = __builtin_fmaf(h[v], 0.0f, trace);
    if (last_group) {  // the state behind the tile, for the next one
#pragma unroll
      for (int v = 0; v < V; ++v) ends[turn][at.slot + v] = carry[v] = h[v];
    }
    turn ^= 1;
  };
  int64_t jt = j0;
  if (a.whole)
    for (; jt + tile <= j1; jt += tile) one_tile(std::true_type{}, jt);
  for (; jt < j1; jt += tile) one_tile(std::false_type{}, jt);
  if (__builtin_expect(trace != 0.0f, 0)) lost[at.slot / V] = 1;
  __syncthreads();  // (what the other groups have stored is written again behind them)
  if (__builtin_expect(last_group && at.active && lost[at.slot / V], 0)) {
    float h[V];
    sure_walk<T, V>(own_arguments<TileArgs<T>>(), h);
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = h[v];
  }
  if (h_last && last_group && at.active && j1 == q.len) {
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = q.ok ? carry[v] : __builtin_nanf("");
    store_channels<V>(h_last + sc, carry, at.second);
  }
}

// Tiles from the last one back.  The state a tile was entered with comes from `saved`; maps of the states and of what comes back go
// through the same exchange.
template <typename T, int V>
__global__ __launch_bounds__(kThreads, 4) void scan_tile_backward_kernel(ScanArgs a, const T* __restrict__ x, int64_t ldx, const T* __restrict__ f,
                                                                         int64_t ldf, const float* __restrict__ h0, const float* __restrict__ saved,
                                                                         const T* __restrict__ gy, int64_t ldgy, const float* g_last,
                                                                         T* __restrict__ gx, int64_t ldgx, T* __restrict__ gf, int64_t ldgf, float* g_h0,
                                                                         const float* __restrict__ maps) {
  __shared__ float lds[2][4][kThreads * V], ends[2][64 * V];
  __shared__ int lost[64];  // a lane's states or gradients left the finite numbers somewhere
  if ((int)blockIdx.x >= a.n_blocks) return fill_rest<T>(a, gx, ldgx, gf, ldgf);
  const Place<V> at(a);
  const Seq q(a, at.s);
  const int lanes_v = V << a.lane_bits, tile = at.n_groups * kSteps;
  const int64_t sc = (int64_t)at.s * a.n_channels + at.channel;
  const int64_t j0 = at.chunk * a.chunk, j1 = j0 + a.chunk < q.len ? j0 + a.chunk : q.len;
  if (j0 >= q.len && at.chunk > 0) return;
  if (threadIdx.x < 64) lost[threadIdx.x] = 0;  // (set behind the chunks' barriers or the last tile's; with neither there is nothing to walk)
  float carry[V];  // a_t g_t of the token behind
  if (maps) {
    const int last = q.len > 0 ? (int)((q.len - 1) / a.chunk) : 0;
    compose_chunks<V>(a, at, maps, last, -1, last - at.chunk, lds[0], carry);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = g_last && at.active ? g_last[sc + v] : 0.0f;
  }
  float trace = 0.0f;  // NaN once something is not finite
#pragma unroll
  for (int v = 0; v < V; ++v) trace = __builtin_fmaf(carry[v], 0.0f, trace);
  const int64_t sx = q.dir * ldx, sf = q.dir * ldf, sy = q.dir * ldgy;
  const TileRows<T, V> tx(at, q, ldx), tf(at, q, ldf), ty(at, q, ldgy), tgx(at, q, ldgx), tgf(at, q, ldgf);
  const int64_t last_tile = j1 > j0 ? j0 + (j1 - j0 - 1) / tile * tile : j0 - tile;
  int turn = 0;
  auto one_tile = [&](auto whole, int64_t jt) {
    constexpr bool WHOLE = decltype(whole)::value;
    const int64_t j = jt + at.group * kSteps, left = j1 - j;
    const int n = WHOLE ? kSteps : !at.active || left <= 0 ? 0 : left < kSteps ? (int)left : kSteps;
    Rows<T, V> rx, rf, ry;
    if constexpr (WHOLE) {
      const int64_t row = q.row(jt);
      tx.load(x + row * ldx, rx);
      tf.load(f + row * ldf, rf);
      ty.load(gy + row * ldgy, ry);
    } else {
      rx.load(x + q.row(j) * ldx + at.channel, sx, n);
      rf.load(f + q.row(j) * ldf + at.channel, sf, n);
      ry.load(gy + q.row(j) * ldgy + at.channel, sy, n);
    }
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
      h[v] = !at.active ? 0.0f : jt > 0 ? saved[q.row(jt) / kTile * a.n_channels + at.channel + v] : h0 ? h0[sc + v] : 0.0f;
    float xs[kSteps][V], ps[kSteps][V], Q[V];
    Span m[V];
#pragma unroll
    for (int v = 0; v < V; ++v) m[v] = identity_span(), Q[v] = 0.0f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        ps[i][v] = WHOLE || i < n ? signed_gate((float)rf.r[i][v]) : 0.0f;
        xs[i][v] = seen((float)rx.r[i][v], ps[i][v]);
        extend(m[v].A, m[v].G, ps[i][v]);
        m[v].H = step(m[v].H, xs[i][v], ps[i][v]);
      }
    }
    forget<V>(ps);
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) {
#pragma unroll
      for (int v = 0; v < V; ++v) Q[v] = decay(Q[v] + (float)ry.r[i][v], ps[i][v]);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = at.at(at.group, lanes_v) + v;
      lds[turn][0][i] = m[v].A, lds[turn][1][i] = m[v].G, lds[turn][2][i] = m[v].H, lds[turn][3][i] = Q[v];
    }
    __syncthreads();
    float c[V];
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = jt == last_tile ? carry[v] : ends[turn ^ 1][at.slot + v];
    for (int k = 0; k < at.group; ++k) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = at.at(k, lanes_v) + v;
        h[v] = apply(lds[turn][0][i], lds[turn][1][i], lds[turn][2][i], h[v]);
      }
    }
    for (int k = at.n_groups - 1; k > at.group; --k) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = at.at(k, lanes_v) + v;
        c[v] = apply(lds[turn][0][i], lds[turn][1][i], lds[turn][3][i], c[v]);
      }
    }
    if (WHOLE || n > 0) {
      forget<V>(ps);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float above = h[v] - xs[i][v];
          h[v] = step(h[v], xs[i][v], ps[i][v]);
          xs[i][v] = above;
        }
      }
      forget<V>(ps);
      T *ox = gx + q.row(j) * ldgx + at.channel, *of = gf + q.row(j) * ldgf + at.channel;
#pragma unroll
      for (int i = kSteps - 1; i >= 0; --i) {
        float dx[V], df[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float p = __builtin_fabsf(ps[i][v]), total = c[v] + (float)ry.r[i][v];
          const float part = p * total, rest = __builtin_fmaf(-p, total, total);
          const bool k = keeps(ps[i][v]);
          dx[v] = k ? part : rest;
          c[v] = k ? rest : part;
          df[v] = p * rest * xs[i][v];
        }
        if constexpr (WHOLE) {
          tgx.store(gx + q.row(jt) * ldgx, i, dx);
          tgf.store(gf + q.row(jt) * ldgf, i, df);
        } else if (i < n) {
          store_channels<V>(ox + i * (q.dir * ldgx), dx, at.second);
          store_channels<V>(of + i * (q.dir * ldgf), df, at.second);
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) trace = __builtin_fmaf(h[v], 0.0f, __builtin_fmaf(c[v], 0.0f, trace));
    if (at.group == 0) {  // what goes back into the tile in front
#pragma unroll
      for (int v = 0; v < V; ++v) ends[turn][at.slot + v] = carry[v] = c[v];
    }
    turn ^= 1;
  };
  for (int64_t jt = last_tile; jt >= j0; jt -= tile) {
    if (a.whole && jt + tile <= j1) one_tile(std::true_type{}, jt);
    else one_tile(std::false_type{}, jt);
  }
  if (__builtin_expect(trace != 0.0f, 0)) lost[at.slot / V] = 1;
  __syncthreads();
  if (__builtin_expect(at.group == 0 && at.active && lost[at.slot / V], 0)) {
    float back[V];
    sure_walk_back<T, V>(own_arguments<TileBackArgs<T>>(), &lds[0][0][0], back);
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = back[v];
  }
  if (g_h0 && at.chunk == 0 && at.group == 0 && at.active) {
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = q.ok ? carry[v] : __builtin_nanf("");
    store_channels<V>(g_h0 + sc, carry, at.second);
  }
}

// How a call is divided.  A workgroup walks a whole sequence at 64 channels a go, unless that leaves the 256 CUs without two workgroups
// each, or one long sequence would still be walked when the others are done: then sequences are cut into chunks.
struct Plan {
  int v, lane_bits, n_chunks, per_row;
  int64_t chunk;
};

Plan scan_plan(int64_t n_tokens, int32_t n_channels, int32_t n_seqs, int64_t max_len, int v) {
  Plan p;
  p.v = v;
  if (max_len > n_tokens) max_len = n_tokens;  // (a longer sequence does not fit)
  const int lanes_needed = (n_channels + v - 1) / v;
  p.lane_bits = lanes_needed > 32 ? 6 : lanes_needed > 16 ? 5 : 4;
  p.per_row = (lanes_needed + (1 << p.lane_bits) - 1) >> p.lane_bits;
  const int64_t tile = (int64_t)(kThreads >> p.lane_bits) * kSteps, tiles = max_len > 0 ? (max_len + tile - 1) / tile : 1;
  const int64_t rows = (int64_t)n_seqs * p.per_row;
  int64_t all = (n_tokens + tile - 1) / tile * p.per_row;  // tiles of the whole call, if its sequences fill them
  if (all > rows * tiles) all = rows * tiles;
  // A workgroup's fair share of tiles: of sequences as long as the longest, over the two workgroups a CU that run at once (one of 100 001 x
  // 256 bf16 64 + 89 us against 77 + 105 us with twice as many); of unequal ones over four (8 of 8 - 19 k x 274 109 + 157 us against
  // 123 + 178 us with half as many).
  const int64_t target = 10 * all >= 9 * rows * tiles ? 512 : 1024;
  const int64_t share = all > target ? (all + target - 1) / target : 1;
  p.n_chunks = 1;
  int64_t each = tiles;  // tiles of a chunk
  if (n_tokens > 0 && tiles > 2 * share && tiles > 6) {  // (a second kernel takes as long as a few tiles)
    int64_t c = (tiles + share - 1) / share;
    const int64_t most = rows > 0 ? (1 << 18) / rows : 1;  // short sequences have as many chunks as the longest: mostly empty workgroups
    if (c > 1024) c = 1024;
    if (c > most) c = most > 1 ? most : 1;
    each = (tiles + c - 1) / c;
    p.n_chunks = (int)((tiles + each - 1) / each);
  }
  p.chunk = each * tile;
  return p;
}

// Channels per lane: two of 16 bits.
inline int channels_per_lane(int32_t dtype, int32_t n_channels) { return dtype == DC_DTYPE_F32 || n_channels == 1 ? 1 : 2; }

int32_t whole_tiles(const Plan& p, int32_t n_channels, std::initializer_list<int64_t> strides) {
  for (int64_t s : strides)
    if (s > (1 << 20)) return 0;
  return n_channels == p.per_row * (p.v << p.lane_bits);
}

// calls f with the element type and the channels per lane
template <typename F>
int with_lanes(int32_t dtype, int v, F&& f) {
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) {
      if (v == 2) return f(t, std::integral_constant<int, 2>{});
    }
    return f(t, std::integral_constant<int, 1>{});
  });
}

int check_scan(int32_t dtype, const void* x, int64_t x_stride, const void* f, int64_t f_stride, int64_t n_tokens, int32_t n_channels,
               const int64_t* begin, const int64_t* end, int32_t n_seqs, int64_t max_len, const void* workspace, int64_t workspace_bytes) {
  DC_REQUIRE(dtype_ok(dtype), "unknown element type");
  DC_REQUIRE(n_tokens >= 0 && n_channels > 0 && n_seqs >= 0 && max_len >= 0, "negative size");
  DC_REQUIRE((begin == nullptr) == (end == nullptr), "begin and end come together");
  DC_REQUIRE(begin || max_len == 0 || n_seqs <= n_tokens / max_len, "dense sequences exceed the tokens");
  DC_REQUIRE(n_tokens == 0 || (x && f), "null pointer");
  DC_REQUIRE(x_stride >= 0 && f_stride >= 0, "negative stride");
  DC_REQUIRE(n_channels <= (1 << 24) && (int64_t)n_seqs * ((n_channels + 63) / 64) < ((int64_t)1 << 20), "more than 2^20 blocks of 64 channels");
  DC_REQUIRE(aligned(x, dtype_size(dtype)) && aligned(f, dtype_size(dtype)), "misaligned pointer");
  const int64_t need = dc_gated_scan_workspace(n_tokens, n_channels, n_seqs, max_len);
  DC_REQUIRE(workspace_bytes >= need && (need == 0 || workspace) && aligned(workspace, 16), "workspace too small");
  return DC_OK;
}

}  // namespace
}  // namespace dc

extern "C" int64_t dc_gated_scan_saved(int64_t n_tokens, int32_t n_channels) {
  return n_tokens > 0 && n_channels > 0 ? (n_tokens + dc::kTile - 1) / dc::kTile * n_channels : 0;
}

extern "C" int64_t dc_gated_scan_workspace(int64_t n_tokens, int32_t n_channels, int32_t n_seqs, int64_t max_len) {
  if (n_tokens <= 0 || n_channels <= 0 || n_seqs <= 0 || max_len <= dc::kShort) return 0;
  // maps and starts of either division: with one or with two channels a lane (by the element type, which is not said here)
  int64_t most = 0;
  for (int v = 1; v <= 2; ++v) {
    const dc::Plan p = dc::scan_plan(n_tokens, n_channels, n_seqs, max_len, v);
    if (p.n_chunks > 1 && p.n_chunks > most) most = p.n_chunks;
  }
  return most ? (int64_t)n_seqs * (3 * most + 1) * n_channels * 4 : 0;
}

extern "C" int dc_gated_scan(void* stream, int32_t dtype, const void* d_x, int64_t x_stride, const void* d_f, int64_t f_stride,
                             int64_t n_tokens, int32_t n_channels, const int64_t* d_begin, const int64_t* d_end, int32_t n_seqs,
                             int64_t max_len, int32_t reverse, const float* d_h0, void* d_y, int64_t y_stride, int32_t zero_rest,
                             float* d_h_last, float* d_saved, void* d_workspace, int64_t workspace_bytes) {
  using namespace dc;
  if (int rc = check_scan(dtype, d_x, x_stride, d_f, f_stride, n_tokens, n_channels, d_begin, d_end, n_seqs, max_len, d_workspace, workspace_bytes)) return rc;
  DC_REQUIRE(n_tokens == 0 || d_y, "null pointer");
  DC_REQUIRE(y_stride >= n_channels, "rows of the output overlap");
  DC_REQUIRE(aligned(d_y, dtype_size(dtype)), "misaligned pointer");
  const int v = channels_per_lane(dtype, n_channels);
  const Plan p = scan_plan(n_tokens, n_channels, n_seqs, max_len, v);
  ScanArgs a{d_begin, d_end, n_tokens, max_len, n_seqs, n_channels, reverse, p.lane_bits, p.n_chunks, p.chunk, 0, whole_tiles(p, n_channels, {x_stride, f_stride, y_stride})};
  const int rest = rest_blocks(n_tokens, n_seqs, zero_rest);
  return with_lanes(dtype, v, [&](auto t, auto lanes) {
    using T = decltype(t);
    constexpr int V = decltype(lanes)::value;
    const T *x = (const T*)d_x, *f = (const T*)d_f;
    if (max_len <= kShort) {
      a.n_blocks = n_seqs * ((n_channels + kWalkThreads * V - 1) / (kWalkThreads * V));
      if (a.n_blocks + rest == 0) return DC_OK;
      scan_walk_kernel<T, V><<<dim3(a.n_blocks + rest), dim3(kWalkThreads), 0, as_stream(stream)>>>(a, x, x_stride, f, f_stride, d_h0, (T*)d_y, y_stride, d_h_last);
      DC_LAUNCH_CHECK();
      return DC_OK;
    }
    a.n_blocks = n_seqs * p.per_row * p.n_chunks;
    if (a.n_blocks + rest == 0) return DC_OK;
    float* maps = p.n_chunks > 1 ? (float*)d_workspace : nullptr;
    if (maps) {
      scan_map_kernel<T, V, false><<<dim3(a.n_blocks), dim3(kThreads), 0, as_stream(stream)>>>(a, f, f_stride, x, x_stride, d_h0, maps);
      DC_LAUNCH_CHECK();
    }
    scan_tile_kernel<T, V><<<dim3(a.n_blocks + rest), dim3(kThreads), 0, as_stream(stream)>>>(a, x, x_stride, f, f_stride, d_h0, (T*)d_y, y_stride, d_h_last,
                                                                                               d_saved, maps);
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
  if (int rc = check_scan(dtype, d_x, x_stride, d_f, f_stride, n_tokens, n_channels, d_begin, d_end, n_seqs, max_len, d_workspace, workspace_bytes)) return rc;
  DC_REQUIRE(n_tokens == 0 || (d_saved && d_grad_y && d_grad_x && d_grad_f), "null pointer");
  DC_REQUIRE(grad_y_stride >= 0, "negative stride");
  DC_REQUIRE(grad_x_stride >= n_channels && grad_f_stride >= n_channels, "rows of an output overlap");
  DC_REQUIRE(aligned(d_grad_y, dtype_size(dtype)) && aligned(d_grad_x, dtype_size(dtype)) && aligned(d_grad_f, dtype_size(dtype)), "misaligned pointer");
  const int v = channels_per_lane(dtype, n_channels);
  const Plan p = scan_plan(n_tokens, n_channels, n_seqs, max_len, v);
  ScanArgs a{d_begin, d_end, n_tokens, max_len, n_seqs, n_channels, reverse, p.lane_bits, p.n_chunks, p.chunk, 0, whole_tiles(p, n_channels, {x_stride, f_stride, grad_y_stride, grad_x_stride, grad_f_stride})};
  const int rest = rest_blocks(n_tokens, n_seqs, zero_rest);
  return with_lanes(dtype, v, [&](auto t, auto lanes) {
    using T = decltype(t);
    constexpr int V = decltype(lanes)::value;
    const T *x = (const T*)d_x, *f = (const T*)d_f, *gy = (const T*)d_grad_y;
    T *gx = (T*)d_grad_x, *gf = (T*)d_grad_f;
    if (max_len <= kShort) {
      a.n_blocks = n_seqs * ((n_channels + kWalkThreads * V - 1) / (kWalkThreads * V));
      if (a.n_blocks + rest == 0) return DC_OK;
      scan_walk_backward_kernel<T, V><<<dim3(a.n_blocks + rest), dim3(kWalkThreads), 0, as_stream(stream)>>>(
          a, x, x_stride, f, f_stride, d_h0, gy, grad_y_stride, d_grad_h_last, gx, grad_x_stride, gf, grad_f_stride, d_grad_h0);
      DC_LAUNCH_CHECK();
      return DC_OK;
    }
    a.n_blocks = n_seqs * p.per_row * p.n_chunks;
    if (a.n_blocks + rest == 0) return DC_OK;
    float* maps = p.n_chunks > 1 ? (float*)d_workspace : nullptr;
    if (maps) {
      scan_map_kernel<T, V, true><<<dim3(a.n_blocks), dim3(kThreads), 0, as_stream(stream)>>>(a, f, f_stride, gy, grad_y_stride, d_grad_h_last, maps);
      DC_LAUNCH_CHECK();
    }
    scan_tile_backward_kernel<T, V><<<dim3(a.n_blocks + rest), dim3(kThreads), 0, as_stream(stream)>>>(
        a, x, x_stride, f, f_stride, d_h0, d_saved, gy, grad_y_stride, d_grad_h_last, gx, grad_x_stride, gf, grad_f_stride, d_grad_h0, maps);
    DC_LAUNCH_CHECK();
    return DC_OK;
  });
}
