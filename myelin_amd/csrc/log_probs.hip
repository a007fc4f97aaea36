// Log probabilities of given tokens, with the entropy of the distribution and
// its top alternatives, and the gradient of both.
//
//   lse = log sum_i e^x_i     log_prob = x[target] - lse
//   entropy = lse - sum_i p_i x_i,  p_i = e^(x_i - lse)
//   top: the n largest x_i - lse, equal ones by the lower index
//   dx_i = g_lp (1[i = target] - p_i) - g_ent p_i (log p_i + entropy)
//
// The rows are read past the caches (nontemporal) and a large gradient written
// so: 8192 x 32768 bf16, forward and backward, 290 -> 263 us (1.55 GB, 5.9 TB/s).
//
// One pass: a lane keeps the running maximum m of its elements, s = sum
// e^(x - m) and u = sum e^(x - m) (x - m); a larger maximum m' rescales them by
// f = e^(m - m') as s' = f s, u' = f (u + (m - m') s).  Then log p = (x - m) -
// log s and entropy = log s - u / s, which lose nothing to a large |m| (a row
// of nothing but a type's lowest value is uniform); m and log s are kept apart
// for the backward pass for the same reason.  All of it is fp32, whatever the
// logits' type.
//
// Masked logits: -inf (and anything so low that e^(x - m) is 0) adds nothing to
// either sum, its 0 * (x - m) included.  A row of nothing but -inf has no
// distribution: log_prob -inf, entropy 0, gradient 0.  NaN and +inf make the
// row's results NaN.  A row whose target is ignore_index is not read: log_prob
// and entropy 0, no alternatives (-inf, token -1), gradient 0.  Any other
// target outside [0, V) gives NaN.

#include "common.h"

namespace {

using myelin::kWave;

constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr int kMaxTop = 64;  // one alternative a lane

// e^d to fp32 accuracy: 2^t with t = d log2(e) rounded, and its rounding error
// put back to first order.  d = -inf gives 0, NaN stays NaN.
__device__ __forceinline__ float exp_f32(float d) {
  const float t = d * kLog2e;
  const float e = __builtin_amdgcn_exp2f(t);
  const float r = __builtin_fmaf(d, kLog2e, -t);
  // (past |t| = 2^24 r may be inf - inf; the exponential is 0 there)
  return t > -200.0f ? __builtin_fmaf(e, r * kLn2, e) : e;
}

struct F32 {
  using T = float;
  static constexpr int VEC = 4;
  __device__ static float get(T v) { return v; }
  __device__ static T put(float v) { return v; }
};
struct BF16 {
  using T = __bf16;
  static constexpr int VEC = 8;
  __device__ static float get(T v) { return static_cast<float>(v); }
  __device__ static T put(float v) { return static_cast<__bf16>(v); }
};

struct Stats {
  float m, s, u;
  __device__ static Stats none() { return {kLowest, 0.0f, 0.0f}; }
  // m is finite or +inf and never NaN (a NaN element makes s NaN); the clamps
  // keep 0 * inf out of the rescaling
  __device__ void rescale(float to) {
    const float d = fmaxf(m - to, -1000.0f), f = exp_f32(d);
    u = f * __builtin_fmaf(d, s, u);
    s = f * s;
    m = to;
  }
  __device__ void merge(Stats o) {
    const float to = fmaxf(m, o.m);
    rescale(to);
    o.rescale(to);
    s += o.s;
    u += o.u;
  }
  // (the rounding of d log2(e), |d| 2^-24 of e, is left: it is small where e is
  // large and of random sign over the sum.  At 2 bytes an element the sum is
  // bound by these instructions, not by memory: 8192 x 32768 133 -> 127 us
  // without the correction.)
  __device__ void add(float x) {
    const float d = x - m;
    const float e = __builtin_amdgcn_exp2f(d * kLog2e);
    s += e;
    u = __builtin_fmaf(e, fmaxf(d, -1000.0f), u);
  }
};

__device__ __forceinline__ Stats across(Stats a, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    Stats b = {__shfl_xor(a.m, o), __shfl_xor(a.s, o), __shfl_xor(a.u, o)};
    a.merge(b);
  }
  return a;
}

struct Args {
  const void *x;
  int64_t ld;
  const int64_t *targets;  // null: no given tokens
  int64_t ignore;
  float *log_probs, *entropy;
  float *stats;  // [2, R]: m, then log s (-inf: nothing allowed)
  float *top_lp;
  int64_t *top_tok;
  int64_t R, V;
  int top;
  int parts;
  int64_t part;  // elements of a part
  int64_t rows;  // of a launch in x
  Stats *part_stats;
  uint64_t *part_keys;
};

struct Row {
  float m, log_s, entropy, log_prob;
  __device__ float log_p(float x) const { return log_s == -__builtin_huge_valf() ? log_s : (x - m) - log_s; }
};

template <class E>
__device__ __forceinline__ Row finish(const Args &a, int64_t row, Stats t) {
  Row r;
  if (t.s == 0.0f) {  // nothing allowed
    r = {0.0f, -__builtin_huge_valf(), 0.0f, -__builtin_huge_valf()};
    if (a.targets) {
      const int64_t tok = a.targets[row];
      if (tok < 0 || tok >= a.V) r.log_prob = __builtin_nanf("");
    }
    return r;
  }
  r.m = t.m;
  r.log_s = logf(t.s);
  r.entropy = r.log_s - t.u / t.s;
  r.log_prob = 0.0f;
  if (a.targets) {
    const int64_t tok = a.targets[row];
    if (tok >= 0 && tok < a.V)
      r.log_prob = r.log_p(E::get(static_cast<const typename E::T *>(a.x)[row * a.ld + tok]));
    else
      r.log_prob = __builtin_nanf("");
  }
  return r;
}

__device__ __forceinline__ void store_row(const Args &a, int64_t row, Row r) {
  if (a.log_probs) a.log_probs[row] = r.log_prob;
  a.entropy[row] = r.entropy;
  a.stats[row] = r.m;
  a.stats[a.R + row] = r.log_s;
}

__device__ __forceinline__ bool ignored(const Args &a, int64_t row) {
  return a.targets && a.targets[row] == a.ignore;
}

// ---- few classes: a row to LANES lanes ---------------------------------
// 8 lanes for up to 32 classes, so that a wave has 8 rows, a wave for up to
// kNarrow.  12800 rows of 10: 3.8 us, a launch's latency.
template <class E, int LANES>
__global__ __launch_bounds__(256) void narrow_rows(Args a) {
  const int64_t row = (myelin::block_id() * 256 + threadIdx.x) / LANES;
  const int l = threadIdx.x % LANES;
  if (row >= a.R) return;  // whole groups of lanes
  if (ignored(a, row)) {
    if (l == 0) store_row(a, row, {0.0f, 0.0f, 0.0f, 0.0f});
    return;
  }
  const typename E::T *x = static_cast<const typename E::T *>(a.x) + row * a.ld;
  Stats t = Stats::none();
  for (int64_t i = l; i < a.V; i += LANES) {
    const float v = E::get(x[i]);
    if (v > t.m) t.rescale(v);
    t.add(v);
  }
  t = across(t, LANES);
  const Row r = finish<E>(a, row, t);
  if (l == 0) store_row(a, row, r);
}

// ---- wide rows: a workgroup to a row, or to one of its parts -----------
// Order of the alternatives: by value, equal ones by the lower index, as one
// unsigned comparison.  -0 is made +0, NaN sorts above everything; 0 is no
// element.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) {
  uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
  b = (v != v) ? 0xffffffffu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<uint64_t>(b) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t b = static_cast<uint32_t>(key >> 32);
  if (b == 0xffffffffu) return __builtin_nanf("");
  return __builtin_bit_cast(float, (b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}
__device__ __forceinline__ int64_t index_of(uint64_t key) {
  return static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key));
}

__device__ __forceinline__ uint64_t key_of_lane(uint64_t k, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(k)), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(k >> 32)), lane);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// The lane's place among the wave's keys, which are distinct or 0.
__device__ __forceinline__ int rank_in_wave(uint64_t mine) {
  int rank = 0;
#pragma unroll
  for (int o = 0; o < kWave; ++o) rank += key_of_lane(mine, o) > mine;
  return rank;
}

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kPerThread = 16;               // elements of a tile a thread holds
constexpr int kTile = kThreads * kPerThread;  // 4096

// The n best of `count` distinct keys, sorted, by counting for each how many
// are larger (16 reads of LDS in flight: a loop of one waits for each).
__device__ __forceinline__ void select(const uint64_t *from, int count, uint64_t *to, int n) {
  for (int c = threadIdx.x; c < count; c += kThreads) {
    const uint64_t k = from[c];
    int rank = 0, j = 0;
    for (; j + 16 <= count && rank < n; j += 16) {
      uint64_t other[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) other[i] = from[j + i];
#pragma unroll
      for (int i = 0; i < 16; ++i) rank += other[i] > k;
    }
    for (; j < count; ++j) rank += from[j] > k;
    if (rank < n) to[rank] = k;
  }
}

// A tile of 4096 elements is 16 a thread in registers, two or four 16-byte loads
// in flight.  8192 x 32768 bf16, a tenth ignored: about 100 us, 4.8 TB/s, by
// memory and by the exponentials alike; 8 x 100003 with 20 alternatives 14 us,
// latency.
//
// TOP: the alternatives too.  A tile's elements sit in registers.  Candidates
// are those over a bound that at least n elements reach: before there are n,
// the n-th largest of a wave's 64 lane maxima (the best of the waves'), after
// that the n-th best so far.  Their number is near n for all but contrived
// rows; the buffer holds the whole tile.
template <class E, bool TOP>
__global__ __launch_bounds__(kThreads) void wide_rows(Args a) {
  using T = typename E::T;
  constexpr int VEC = E::VEC, NV = kPerThread / VEC;
  __shared__ Stats red[kWaves];
  __shared__ uint64_t cand[TOP ? kTile + kMaxTop : 1];
  __shared__ uint64_t best[TOP ? kMaxTop : 1];
  __shared__ uint64_t bound_of[kWaves];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = tid >> 6;
  const int64_t row = blockIdx.x / a.parts + blockIdx.y * a.rows;
  if (row >= a.R) return;  // the whole workgroup
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int64_t begin = part * a.part;
  const int64_t end = begin + a.part < a.V ? begin + a.part : a.V;
  if (ignored(a, row)) {
    if (part == 0) {
      if (tid == 0) store_row(a, row, {0.0f, 0.0f, 0.0f, 0.0f});
      if (TOP && tid < a.top) {
        a.top_lp[row * a.top + tid] = -__builtin_huge_valf();
        a.top_tok[row * a.top + tid] = -1;
      }
    }
    return;
  }
  const T *x = static_cast<const T *>(a.x) + row * a.ld;
  // whole vectors start where the address is a multiple of 16: `lead`
  // elements before `begin` belong to the first one
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(x + begin) % 16) / sizeof(T));
  typedef T vec __attribute__((ext_vector_type(VEC)));
  Stats t = Stats::none();
  int have = 0;
  for (int64_t at = begin - lead; at < end; at += kTile) {
    float v[kPerThread];
    bool in[kPerThread];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t i = at + (static_cast<int64_t>(j) * kThreads + tid) * VEC;
      if (i >= begin && i + VEC <= end) {
        const vec p = __builtin_nontemporal_load(reinterpret_cast<const vec *>(x + i));
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          v[j * VEC + q] = E::get(p[q]);
          in[j * VEC + q] = true;
        }
      } else {
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          const bool ok = i + q >= begin && i + q < end;
          in[j * VEC + q] = ok;
          v[j * VEC + q] = ok ? E::get(x[i + q]) : -__builtin_huge_valf();
        }
      }
    }
    float top = t.m;
#pragma unroll
    for (int q = 0; q < kPerThread; ++q) top = fmaxf(top, v[q]);
    if (top > t.m) t.rescale(top);
#pragma unroll
    for (int q = 0; q < kPerThread; ++q) t.add(v[q]);
    if constexpr (TOP) {
      uint64_t key[kPerThread];
      uint64_t mine = 0;
#pragma unroll
      for (int q = 0; q < kPerThread; ++q) {
        const int64_t i = at + (static_cast<int64_t>(q / VEC) * kThreads + tid) * VEC + q % VEC;
        key[q] = in[q] ? key_of(v[q], static_cast<uint32_t>(i)) : 0;
        mine = key[q] > mine ? key[q] : mine;
      }
      uint64_t bound;
      if (have < a.top) {
        // (lanes without an element share a rank, and the bound 0)
        if (lane == 0) bound_of[w] = 0;
        if (rank_in_wave(mine) == a.top - 1) bound_of[w] = mine;
        if (tid == 0) count = have;
        if (tid < have) cand[tid] = best[tid];
        __syncthreads();
        bound = 1;
        for (int o = 0; o < kWaves; ++o) bound = bound_of[o] > bound ? bound_of[o] : bound;
      } else {
        if (tid == 0) count = have;
        if (tid < have) cand[tid] = best[tid];
        __syncthreads();
        bound = best[a.top - 1];
      }
#pragma unroll
      for (int q = 0; q < kPerThread; ++q)
        if (key[q] >= bound) cand[atomicAdd(&count, 1)] = key[q];
      __syncthreads();
      const int n = count;
      if (n > have) select(cand, n, best, a.top);
      have = n < a.top ? n : a.top;
      __syncthreads();
    }
  }
  t = across(t, kWave);
  if (lane == 0) red[w] = t;
  __syncthreads();
  t = red[0];
  for (int o = 1; o < kWaves; ++o) t.merge(red[o]);
  if (a.parts > 1) {
    if (tid == 0) a.part_stats[row * a.parts + part] = t;
    if (TOP && tid < a.top) a.part_keys[(row * a.parts + part) * a.top + tid] = tid < have ? best[tid] : 0;
    return;
  }
  const Row r = finish<E>(a, row, t);
  if (tid == 0) store_row(a, row, r);
  if (TOP && tid < a.top) {
    const uint64_t k = best[tid];
    a.top_lp[row * a.top + tid] = r.log_p(value_of(k));
    a.top_tok[row * a.top + tid] = index_of(k);
  }
}

// Joins a row's parts: a workgroup a row (25 parts, 20 alternatives: 5.6 us, of
// reads that wait for each other).
template <class E, bool TOP>
__global__ __launch_bounds__(kThreads) void join_parts(Args a) {
  __shared__ Stats red[kWaves];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  if (ignored(a, row)) return;
  Stats t = Stats::none();
  for (int p = tid; p < a.parts; p += kThreads) t.merge(a.part_stats[row * a.parts + p]);
  t = across(t, kWave);
  if ((tid & (kWave - 1)) == 0) red[tid >> 6] = t;
  __syncthreads();
  t = red[0];
  for (int o = 1; o < kWaves; ++o) t.merge(red[o]);
  const Row r = finish<E>(a, row, t);
  if (tid == 0) store_row(a, row, r);
  if constexpr (TOP) {
    // Each part's keys are sorted.  Of ceil(top / l) parts whose l-th key reaches
    // a bound, top keys reach it: wave w takes l = 2^w, a lane a part (or the
    // best of several), and the largest bound holds.  A tile of keys at a time,
    // as wide_rows takes elements.
    __shared__ uint64_t cand[kTile + kMaxTop], best[kMaxTop], bound_of[kWaves];
    __shared__ int count;
    const uint64_t *keys = a.part_keys + row * a.parts * a.top;
    const int lane = tid & (kWave - 1), w = tid >> 6, l = 1 << w;
    uint64_t bound = 0;
    if (l <= a.top)
      for (int p = lane; p < a.parts; p += kWave) {
        const uint64_t k = keys[p * a.top + l - 1];
        bound = k > bound ? k : bound;
      }
    if (lane == 0) bound_of[w] = 0;
    if (rank_in_wave(bound) == (a.top + l - 1) / l - 1) bound_of[w] = bound;
    bound = 1;
    int have = 0;
    for (int at = 0; at < a.parts * a.top; at += kTile) {
      if (tid == 0) count = have;
      if (tid < have) cand[tid] = best[tid];
      __syncthreads();
      for (int o = 0; o < kWaves; ++o) bound = bound_of[o] > bound ? bound_of[o] : bound;
      const int end = at + kTile < a.parts * a.top ? at + kTile : a.parts * a.top;
      for (int c = at + tid; c < end; c += kThreads) {
        const uint64_t k = keys[c];
        if (k >= bound) cand[atomicAdd(&count, 1)] = k;
      }
      __syncthreads();
      select(cand, count, best, a.top);
      have = count < a.top ? count : a.top;
      __syncthreads();
      if (have == a.top && best[a.top - 1] > bound) bound = best[a.top - 1] + 1;
    }
    if (tid < a.top) {
      a.top_lp[row * a.top + tid] = r.log_p(value_of(best[tid]));
      a.top_tok[row * a.top + tid] = index_of(best[tid]);
    }
  }
}

// ---- gradient ------------------------------------------------------------
struct BwdArgs {
  const void *x;
  int64_t ld;
  const int64_t *targets;
  int64_t ignore;
  const float *stats, *entropy, *g_lp, *g_ent;
  void *dx;  // [R, V] contiguous
  int64_t R, V;
  int64_t per_row;  // workgroups of a row
  int64_t rows;     // of a launch in x
};

struct RowGrad {
  float m, log_s, entropy, g_lp, g_ent;
  int64_t target;
  bool zero;
};

__device__ __forceinline__ RowGrad row_grad(const BwdArgs &a, int64_t row) {
  RowGrad g;
  g.target = a.targets ? a.targets[row] : -1;
  g.m = a.stats[row];
  g.log_s = a.stats[a.R + row];
  g.entropy = a.entropy[row];
  g.g_lp = a.g_lp ? a.g_lp[row] : 0.0f;
  g.g_ent = a.g_ent ? a.g_ent[row] : 0.0f;
  g.zero = (a.targets && g.target == a.ignore) || g.log_s == -__builtin_huge_valf();
  if (a.targets && (g.target < 0 || g.target >= a.V)) g.g_lp = a.g_lp ? __builtin_nanf("") : 0.0f;
  return g;
}

__device__ __forceinline__ float grad_of(const RowGrad &g, float x, int64_t i) {
  const float d = (x - g.m) - g.log_s;
  const float p = exp_f32(d);
  // p (log p + H), 0 where p is 0
  const float ent = p == 0.0f ? 0.0f : p * (d + g.entropy);
  const float hit = i == g.target ? g.g_lp : 0.0f;
  return __builtin_fmaf(-g.g_ent, ent, __builtin_fmaf(-g.g_lp, p, hit));
}

template <class E>
__global__ __launch_bounds__(256) void grad_flat(BwdArgs a) {
  const int64_t at = myelin::block_id() * 256 + threadIdx.x;
  if (at >= a.R * a.V) return;
  const int64_t row = at / a.V, i = at - row * a.V;
  const RowGrad g = row_grad(a, row);
  const typename E::T *x = static_cast<const typename E::T *>(a.x);
  static_cast<typename E::T *>(a.dx)[at] = g.zero ? E::put(0.0f) : E::put(grad_of(g, E::get(x[row * a.ld + i]), i));
}

template <class E, bool VECTOR, bool STREAM>
__global__ __launch_bounds__(256) void grad_wide(BwdArgs a) {
  using T = typename E::T;
  constexpr int VEC = VECTOR ? E::VEC : 1, NV = kPerThread / VEC;
  typedef T vec __attribute__((ext_vector_type(VEC)));
  const int64_t row = blockIdx.x / a.per_row + blockIdx.y * a.rows;
  if (row >= a.R) return;
  const int64_t at = (blockIdx.x % a.per_row) * kTile;
  const RowGrad g = row_grad(a, row);
  const T *x = static_cast<const T *>(a.x) + row * a.ld;
  T *dx = static_cast<T *>(a.dx) + row * a.V;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t i = at + (static_cast<int64_t>(j) * 256 + threadIdx.x) * VEC;
    if (i >= a.V) continue;
    if constexpr (VECTOR) {  // V is a multiple of VEC
      vec o;
      if (g.zero) {
#pragma unroll
        for (int q = 0; q < VEC; ++q) o[q] = E::put(0.0f);
      } else {
        const vec p = __builtin_nontemporal_load(reinterpret_cast<const vec *>(x + i));
#pragma unroll
        for (int q = 0; q < VEC; ++q) o[q] = E::put(grad_of(g, E::get(p[q]), i + q));
      }
      myelin::store<STREAM>(o, reinterpret_cast<vec *>(dx + i));
    } else {
      dx[i] = g.zero ? E::put(0.0f) : E::put(grad_of(g, E::get(x[i]), i));
    }
  }
}

// Parts of a row: enough workgroups to fill the chip where rows are few, of
// whole tiles.
void split(int64_t R, int64_t V, int64_t *parts, int64_t *part) {
  const int64_t tiles = (V + kTile - 1) / kTile;
  int64_t n = R > 0 ? 512 / R : 1;
  if (n < 1) n = 1;
  if (n > tiles) n = tiles;
  const int64_t per = (tiles + n - 1) / n;
  *part = per * kTile;
  *parts = (tiles + per - 1) / per;
}

constexpr int64_t kNarrow = 1024;  // widest row of narrow_rows: 16 elements a lane, as wide_rows

bool narrow(int64_t V, int top) { return V <= kNarrow && top == 0; }

int check(const char *what, const void *x, int dtype, int64_t ld, int64_t R, int64_t V) {
  if (dtype != 0 && dtype != 2) return myelin::invalid("%s: unsupported dtype %d", what, dtype);
  if (R < 0 || V < 1) return myelin::invalid("%s: rows must be non-negative and V positive", what);
  if (V > 0x7fffffff) return myelin::invalid("%s: V must be below 2^31", what);
  if (R > 1 && ld < V) return myelin::invalid("%s: row stride below V", what);
  if (R > 0 && !x) return myelin::invalid("%s: null pointer", what);
  return MYELIN_OK;
}

// `per_row` workgroups for each of R rows, whole rows in x.
dim3 row_grid(int64_t R, int64_t per_row, int64_t *rows) {
  *rows = R < myelin::kGridX / per_row ? R : myelin::kGridX / per_row;
  return dim3(static_cast<unsigned>(*rows * per_row), static_cast<unsigned>((R + *rows - 1) / *rows));
}

template <class E>
void launch_fwd(Args &a, hipStream_t s) {
  if (narrow(a.V, a.top)) {
    if (a.V <= 32)
      narrow_rows<E, 8><<<myelin::grid_of((a.R * 8 + 255) / 256), 256, 0, s>>>(a);
    else
      narrow_rows<E, 64><<<myelin::grid_of((a.R * 64 + 255) / 256), 256, 0, s>>>(a);
    return;
  }
  const dim3 grid = row_grid(a.R, a.parts, &a.rows);
  if (a.top)
    wide_rows<E, true><<<grid, kThreads, 0, s>>>(a);
  else
    wide_rows<E, false><<<grid, kThreads, 0, s>>>(a);
  if (a.parts > 1) {
    if (a.top)
      join_parts<E, true><<<static_cast<unsigned>(a.R), kThreads, 0, s>>>(a);
    else
      join_parts<E, false><<<static_cast<unsigned>(a.R), kThreads, 0, s>>>(a);
  }
}

template <class E>
void launch_bwd(BwdArgs &a, hipStream_t s) {
  const int64_t total = a.R * a.V;
  if (a.V < 256) {
    grad_flat<E><<<myelin::grid_of((total + 255) / 256), 256, 0, s>>>(a);
    return;
  }
  const bool vector = a.V % E::VEC == 0 && (a.ld * sizeof(typename E::T)) % 16 == 0 && myelin::aligned(a.x, 16) &&
                      myelin::aligned(a.dx, 16);
  a.per_row = (a.V + kTile - 1) / kTile;
  const dim3 grid = row_grid(a.R, a.per_row, &a.rows);
  if (!vector)
    grad_wide<E, false, false><<<grid, 256, 0, s>>>(a);
  else if (total * static_cast<int64_t>(sizeof(typename E::T)) >= myelin::kStreamBytes)
    grad_wide<E, true, true><<<grid, 256, 0, s>>>(a);
  else
    grad_wide<E, true, false><<<grid, 256, 0, s>>>(a);
}

}  // namespace

extern "C" int64_t myelin_token_log_probs_workspace_bytes(int64_t R, int64_t V, int top) {
  if (R < 1 || V < 1 || top < 0 || narrow(V, top)) return 0;
  int64_t parts, part;
  split(R, V, &parts, &part);
  if (parts == 1) return 0;
  return R * parts * (16 + 8 * static_cast<int64_t>(top));
}

extern "C" int myelin_token_log_probs(const void *logits, int dtype, int64_t ld, const int64_t *targets,
                                      int64_t ignore_index, float *log_probs, float *entropy, float *stats,
                                      float *top_log_probs, int64_t *top_tokens, int64_t R, int64_t V, int top,
                                      void *workspace, int64_t workspace_bytes, myelin_stream_t stream) {
  const char *what = "token_log_probs";
  if (int rc = check(what, logits, dtype, ld, R, V)) return rc;
  if (top < 0 || top > kMaxTop || top > V) return myelin::invalid("%s: top must be in [0, min(%d, V)]", what, kMaxTop);
  if (R == 0) return MYELIN_OK;
  if (!entropy || !stats || (top && (!top_log_probs || !top_tokens)) || (targets && !log_probs))
    return myelin::invalid("%s: null pointer", what);
  Args a{logits, ld, targets, ignore_index, targets ? log_probs : nullptr, entropy, stats, top_log_probs, top_tokens,
         R, V, top, 1, V, R, nullptr, nullptr};
  if (!narrow(V, top)) {
    int64_t parts;
    split(R, V, &parts, &a.part);
    a.parts = static_cast<int>(parts);
    if (a.parts > 1) {
      const int64_t need = myelin_token_log_probs_workspace_bytes(R, V, top);
      if (!workspace || workspace_bytes < need)
        return myelin::invalid("%s: workspace of %lld bytes needed", what, static_cast<long long>(need));
      if (!myelin::aligned(workspace, 16)) return myelin::invalid("%s: workspace must be 16-byte aligned", what);
      a.part_keys = static_cast<uint64_t *>(workspace);
      a.part_stats = reinterpret_cast<Stats *>(a.part_keys + R * parts * top);
    }
  }
  if (R * (a.parts > 64 ? a.parts : 64) / 4 > 0x7fffffff) return myelin::invalid("%s: too many rows", what);
  if (dtype == 0)
    launch_fwd<F32>(a, myelin::as_hip(stream));
  else
    launch_fwd<BF16>(a, myelin::as_hip(stream));
  return myelin::launched(what);
}

extern "C" int myelin_token_log_probs_bwd(const void *logits, int dtype, int64_t ld, const int64_t *targets,
                                          int64_t ignore_index, const float *stats, const float *entropy,
                                          const float *grad_log_probs, const float *grad_entropy, void *grad_logits,
                                          int64_t R, int64_t V, myelin_stream_t stream) {
  const char *what = "token_log_probs_bwd";
  if (int rc = check(what, logits, dtype, ld, R, V)) return rc;
  if (R == 0) return MYELIN_OK;
  if (!stats || !entropy || !grad_logits) return myelin::invalid("%s: null pointer", what);
  if (R * ((V + kTile - 1) / kTile) > 0x7fffffff || (V < 256 && R * V / 256 >= 0x7fffffff))
    return myelin::invalid("%s: too many rows", what);
  BwdArgs a{logits, ld, targets, ignore_index, stats, entropy, targets ? grad_log_probs : nullptr, grad_entropy,
            grad_logits, R, V, 1, R};
  if (dtype == 0)
    launch_bwd<F32>(a, myelin::as_hip(stream));
  else
    launch_bwd<BF16>(a, myelin::as_hip(stream));
  return myelin::launched(what);
}
