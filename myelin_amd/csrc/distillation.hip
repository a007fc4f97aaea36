// Distillation from a teacher's top logits: with the teacher's K values z and
// their tokens, the student's logits x and a temperature,
//
//   p = softmax(z / temperature) over the K    q = softmax(x / temperature) over V
//   loss = sum_k p_k (log p_k - log q[token_k])
//   dx_i = g / temperature (q_i - sum_{k: token_k = i} p_k)
//
// A place of token -1 or value -inf is empty.  A row whose places are all empty is
// not read: loss 0, gradient 0.  A row of logits of nothing but -inf has no
// distribution: loss +inf, gradient 0.  Any other token outside [0, V) makes the
// row NaN (nothing is read out of range), as do NaN and +inf.
//
// One pass: a lane keeps the running maximum m of its elements and s = sum
// e^((x - m) / temperature); all of it is fp32, whatever the logits' type.
//
// The forward pass writes p for the backward pass with tokens that are named twice
// put together at the first of their places (0 at the others): each token then has
// one place, and the backward pass can put p where its element looks for it.

#include "elements.h"

namespace {

using myelin::BF16;
using myelin::F32;
using myelin::kLog2e;
using myelin::kWave;

constexpr float kLowest = -3.402823466e38f;
constexpr float kInf = __builtin_huge_valf();
constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kNarrow = 1024;  // widest row of a single wave

// e^((x - m) rate), rate = 1 / temperature
struct Stats {
  float m, s;
  __device__ static Stats none() { return {kLowest, 0.0f}; }
  __device__ void rescale(float to, float rate) {
    s *= myelin::exp_f32(fmaxf(m - to, kLowest) * rate);
    m = to;
  }
  __device__ void merge(Stats o, float rate) {
    const float to = fmaxf(m, o.m);
    rescale(to, rate);
    o.rescale(to, rate);
    s += o.s;
  }
};

__device__ __forceinline__ Stats across(Stats a, float rate) {
  for (int o = kWave >> 1; o > 0; o >>= 1) {
    Stats b = {__shfl_xor(a.m, o), __shfl_xor(a.s, o)};
    a.merge(b, rate);
  }
  return a;
}

__device__ __forceinline__ float wave_sum(float v) {
  for (int o = kWave >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// The rounding of d rate log2(e), |d| rate 2^-24 of an exponential, is left: it is
// small where the exponential is large and of random sign over the sum.
struct Rate {
  float rate, log2;  // 1 / temperature, and times log2(e)
  __device__ explicit Rate(float r) : rate(r), log2(r * kLog2e) {}
  __device__ float exp(float d) const { return __builtin_amdgcn_exp2f(d * log2); }
};

struct Args {
  const void *x;
  int64_t ld;
  const float *values;
  const int64_t *tokens;
  float rate;
  float *loss, *probs;  // probs [R, K] or null
  float *stats;         // [2, R]: m, then log s (-inf: no gradient)
  int64_t R, V;
  int K;
  int parts;
  int64_t part;  // elements of a part
  int64_t rows;  // of a launch in x
  Stats *part_stats;
};

__device__ __forceinline__ bool empty(int64_t token, float value) { return token == -1 || value == -kInf; }

__device__ __forceinline__ bool nothing(const Args &a, int64_t row, int lane) {
  bool some = false;
  for (int k = lane; k < a.K; k += kWave) some |= !empty(a.tokens[row * a.K + k], a.values[row * a.K + k]);
  return !__any(some);
}

// a row with nothing to learn from
__device__ __forceinline__ void store_nothing(const Args &a, int64_t row, int lane) {
  if (a.probs)
    for (int k = lane; k < a.K; k += kWave) a.probs[row * a.K + k] = 0.0f;
  if (lane == 0) {
    a.loss[row] = 0.0f;
    a.stats[row] = 0.0f;
    a.stats[a.R + row] = -kInf;
  }
}

// Bits of the tokens seen, by their number modulo BITS, and of those where two have
// met: a wave's, cleared.  Only for the latter is it looked at which are the same.
constexpr int kSeen = 1 << 15;

template <int BITS>
struct Seen {
  uint32_t once[BITS / 32], twice[BITS / 32];
  __device__ void clear(int lane) {
    for (int o = lane; o < BITS / 32; o += kWave) once[o] = twice[o] = 0;
  }
  __device__ void add(int64_t token) {
    const uint32_t at = static_cast<uint32_t>(token) % BITS, bit = 1u << (at % 32);
    if (atomicOr(&once[at / 32], bit) & bit) atomicOr(&twice[at / 32], bit);
  }
  __device__ bool met(int64_t token) const {
    const uint32_t at = static_cast<uint32_t>(token) % BITS;
    return twice[at / 32] >> (at % 32) & 1;
  }
};

// What the places of this lane's token have, added up in their order, where place k is
// the first of them, and 0 elsewhere; a lane without such a token has -1.  The places of
// tokens that have met (among the 64 of each bit of `met`) come past all lanes one at a
// time, at most K^2 / 64 of them for a row, until each lane knows of a place before its
// own.  Each place looked for and added up by itself took K^2: 4 rows of 1024 places of
// one token 50 ms -> 0.12, of two places to a token 2.9 ms -> 0.66; 2048 rows of 40000 and 64
// places of one token 302 us -> 60, 56 of different ones.
template <int BITS>
__device__ __forceinline__ float together(const Args &a, int64_t first, uint32_t met, int token, int k, float peak,
                                          float total, const Seen<BITS> &seen) {
  constexpr int kSome = 28;  // of 64: 60 ns each; past that all of them, 2 us
  const int lane = threadIdx.x & (kWave - 1);
  bool later = token < 0;
  float sum = 0.0f;
  for (uint32_t m = met; m && __any(!later); m &= m - 1) {
    const int from = __builtin_ctz(m) * kWave, o = from + lane, before = k - from;
    const int64_t other = o < a.K ? a.tokens[first + o] : -1;
    const float value = o < a.K ? a.values[first + o] : 0.0f;
    const bool there = !empty(other, value) && seen.met(other);
    const int name = there ? static_cast<int>(other) : -2;
    const int v = __builtin_bit_cast(int, there ? myelin::exp_f32((value - peak) * a.rate) / total : 0.0f);
    const auto pass = [&](int i) {
      const bool same = __builtin_amdgcn_readlane(name, i) == token;
      later |= same && i < before;
      sum += same ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(v, i)) : 0.0f;
    };
    uint64_t s = __ballot(there);
    if (__builtin_popcountll(s) > kSome) {
#pragma unroll 16  // (whole, it takes 100 registers, and 8 waves a SIMD have 64)
      for (int i = 0; i < kWave; ++i) pass(i);
    } else {
      for (; s; s &= s - 1) pass(__builtin_ctzll(s));
    }
  }
  return later ? 0.0f : sum;
}

// The row's loss from its logits' statistics, by one wave.
template <class E, int BITS>
__device__ __forceinline__ void finish(const Args &a, int64_t row, Stats t, int lane, Seen<BITS> &seen) {
  const int64_t first = row * a.K;
  const typename E::T *x = static_cast<const typename E::T *>(a.x) + row * a.ld;
  float peak = kLowest;
  bool bad = false;
  for (int k = lane; k < a.K; k += kWave) {
    const int64_t token = a.tokens[first + k];
    const float v = a.values[first + k];
    if (empty(token, v)) continue;
    peak = fmaxf(peak, v);
    bad |= token < 0 || token >= a.V;
    if (a.probs) seen.add(token);
  }
  for (int o = kWave >> 1; o > 0; o >>= 1) peak = fmaxf(peak, __shfl_xor(peak, o));
  bad = __any(bad);
  float total = 0.0f;
  uint32_t met = 0;  // the 64 places with tokens that have met
  for (int at = 0; at < a.K; at += kWave) {
    const int k = at + lane;
    const int64_t token = k < a.K ? a.tokens[first + k] : -1;
    const float value = k < a.K ? a.values[first + k] : 0.0f;
    const bool there = !empty(token, value);
    if (there) total += myelin::exp_f32((value - peak) * a.rate);
    if (a.probs && !bad && __any(there && seen.met(token))) met |= 1u << (at / kWave);
  }
  total = wave_sum(total);
  const float log_total = logf(total), log_s = t.s == 0.0f ? -kInf : logf(t.s);
  float loss = 0.0f;
  for (int at = 0; at < a.K; at += kWave) {
    const int k = at + lane;
    const int64_t token = k < a.K ? a.tokens[first + k] : -1;
    const float value = k < a.K ? a.values[first + k] : 0.0f;
    const bool there = !empty(token, value);
    float p = 0.0f;
    if (there) {
      const float d = (value - peak) * a.rate;
      p = myelin::exp_f32(d) / total;
      if (p != 0.0f && !bad) {
        // nothing allowed: log q is -inf for every token
        const float log_q = t.s == 0.0f ? -kInf : (E::get(x[token]) - t.m) * a.rate - log_s;
        loss += p * ((d - log_total) - log_q);
      }
    }
    if (!a.probs) continue;
    if (met >> (at / kWave) & 1) {
      const bool mine = there && seen.met(token);
      const float sum = together(a, first, met, mine ? static_cast<int>(token) : -1, k, peak, total, seen);
      if (mine) p = sum;
    }
    if (k < a.K) a.probs[first + k] = p;
  }
  loss = wave_sum(loss);
  if (lane == 0) {
    a.loss[row] = bad ? __builtin_nanf("") : loss;
    a.stats[row] = bad ? __builtin_nanf("") : t.m;
    a.stats[a.R + row] = bad ? 0.0f : log_s;
  }
}

// ---- few classes: a wave to a row ---------------------------------------
// All of the row in registers: 2048 rows of 1000 fp32 6.5 us (8 MB), latency.
template <class E>
__global__ __launch_bounds__(kThreads) void narrow_rows(Args a) {
  __shared__ Seen<kNarrow> seen[kWaves];
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x >> 6;
  const int64_t row = myelin::block_id() * kWaves + w;
  if (row >= a.R) return;  // whole waves
  const typename E::T *x = static_cast<const typename E::T *>(a.x) + row * a.ld;
  // (in LDS a wave's own writes and atomics are done in its order)
  if (a.probs) seen[w].clear(lane);
  if (nothing(a, row, lane)) {
    store_nothing(a, row, lane);
    return;
  }
  const Rate r(a.rate);
  Stats t = Stats::none();
  constexpr int kEach = kNarrow / kWave;
  float v[kEach];
#pragma unroll
  for (int o = 0; o < kEach; ++o) v[o] = o * kWave + lane < a.V ? E::get(x[o * kWave + lane]) : -kInf;
#pragma unroll
  for (int o = 0; o < kEach; ++o) t.m = fmaxf(t.m, v[o]);
#pragma unroll
  for (int o = 0; o < kEach; ++o) t.s += r.exp(v[o] - t.m);
  t = across(t, a.rate);
  finish<E>(a, row, t, lane, seen[w]);
}

// ---- wide rows: a workgroup to a row, or to one of its parts -------------
constexpr int kPerThread = 16;                // elements of a tile a thread holds
constexpr int kTile = kThreads * kPerThread;  // 4096

// 16 elements a thread in registers, in 16-byte loads past the caches: 8192 rows of
// 32768 bf16, a tenth of them empty, 95 us (483 MB, 5.1 TB/s), bound by memory and the
// exponentials alike.
template <class E>
__global__ __launch_bounds__(kThreads) void wide_rows(Args a) {
  using T = typename E::T;
  constexpr int VEC = E::VEC, NV = kPerThread / VEC;
  __shared__ Stats red[kWaves];
  __shared__ Seen<kSeen> seen;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = tid >> 6;
  const int64_t row = blockIdx.x / a.parts + blockIdx.y * a.rows;
  if (row >= a.R) return;  // the whole workgroup
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int64_t begin = part * a.part;
  const int64_t end = begin + a.part < a.V ? begin + a.part : a.V;
  if (nothing(a, row, lane)) {
    if (part == 0 && w == 0) store_nothing(a, row, lane);
    return;
  }
  if (a.probs && w == 0 && a.parts == 1) seen.clear(lane);
  const Rate r(a.rate);
  const T *x = static_cast<const T *>(a.x) + row * a.ld;
  // whole vectors start where the address is a multiple of 16: `lead` elements
  // before `begin` belong to the first one
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(x + begin) % 16) / sizeof(T));
  typedef T vec __attribute__((ext_vector_type(VEC)));
  Stats t = Stats::none();
  for (int64_t at = begin - lead; at < end; at += kTile) {
    float v[kPerThread];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t i = at + (static_cast<int64_t>(j) * kThreads + tid) * VEC;
      if (i >= begin && i + VEC <= end) {
        const vec p = __builtin_nontemporal_load(reinterpret_cast<const vec *>(x + i));
#pragma unroll
        for (int q = 0; q < VEC; ++q) v[j * VEC + q] = E::get(p[q]);
      } else {
#pragma unroll
        for (int q = 0; q < VEC; ++q) v[j * VEC + q] = i + q >= begin && i + q < end ? E::get(x[i + q]) : -kInf;
      }
    }
    float top = t.m;
#pragma unroll
    for (int q = 0; q < kPerThread; ++q) top = fmaxf(top, v[q]);
    if (top > t.m) t.rescale(top, a.rate);
#pragma unroll
    for (int q = 0; q < kPerThread; ++q) t.s += r.exp(v[q] - t.m);
  }
  t = across(t, a.rate);
  if (lane == 0) red[w] = t;
  __syncthreads();
  if (w != 0) return;
  t = red[0];
  for (int o = 1; o < kWaves; ++o) t.merge(red[o], a.rate);
  if (a.parts > 1) {
    if (lane == 0) a.part_stats[row * a.parts + part] = t;
    return;
  }
  finish<E>(a, row, t, lane, seen);
}

// joins a row's parts: a wave a row
template <class E>
__global__ __launch_bounds__(kWave) void join_parts(Args a) {
  __shared__ Seen<kSeen> seen;
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  if (a.probs) seen.clear(lane);
  if (nothing(a, row, lane)) return;
  Stats t = Stats::none();
  for (int p = lane; p < a.parts; p += kWave) t.merge(a.part_stats[row * a.parts + p], a.rate);
  finish<E>(a, row, across(t, a.rate), lane, seen);
}

// ---- gradient ------------------------------------------------------------
struct BwdArgs {
  const void *x;
  int64_t ld;
  const int64_t *tokens;
  const float *probs, *stats, *g;
  float rate;
  void *dx;  // [R, V] contiguous
  int64_t R, V;
  int K;
  int64_t per_row;  // groups of a row
};

// GROUP threads have a tile of a row, 16 elements each.  The tile's tokens put
// their p into LDS, at their element's place, and a bit that says that it is there:
// an element looks at a bit, not at the tokens.  8192 x 32768 bf16 with 64 tokens: 176
// us (1.02 GB, 5.8 TB/s), bound by memory.
//
// kSkewed: logits and gradients of a row start equally far from a multiple of 16
// bytes.  Tiles start at the multiple before the row, and only what sticks out at its
// ends goes element by element (2048 x 100003 bf16: 354 us element by element, 160
// so).  kWhole: they start there and end there, which spares 2 % of the time.
enum Rows { kSingly, kWhole, kSkewed };

template <class E, int GROUP, Rows ROWS, bool STREAM>
__global__ __launch_bounds__(kThreads) void gradient(BwdArgs a) {
  using T = typename E::T;
  constexpr bool VECTOR = ROWS != kSingly;
  constexpr int VEC = VECTOR ? E::VEC : 1, NV = kPerThread / VEC, TILE = GROUP * kPerThread;
  typedef T vec __attribute__((ext_vector_type(VEC)));
  __shared__ float put[kThreads / GROUP][TILE];
  __shared__ uint32_t bits[kThreads / GROUP][TILE / 32];
  const int tid = threadIdx.x % GROUP, group = threadIdx.x / GROUP;
  const int64_t unit = myelin::block_id() * (kThreads / GROUP) + group, row = unit / a.per_row;
  const bool in = row < a.R;
  const T *x = static_cast<const T *>(a.x) + (in ? row : 0) * a.ld;
  T *dx = static_cast<T *>(a.dx) + row * a.V;
  const int lead = ROWS == kSkewed ? static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)) : 0;
  const int64_t at = (unit - row * a.per_row) * TILE - lead;
  const float m = in ? a.stats[row] : 0.0f, log_s = in ? a.stats[a.R + row] : -kInf;
  const bool zero = log_s == -kInf;
  float v[kPerThread];
  if (!zero) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t i = at + (static_cast<int64_t>(j) * GROUP + tid) * VEC;
      if (ROWS == kWhole && i >= a.V) continue;
      if (ROWS == kWhole || (i >= 0 && i + VEC <= a.V)) {
        if constexpr (VECTOR) {
          const vec p = __builtin_nontemporal_load(reinterpret_cast<const vec *>(x + i));
#pragma unroll
          for (int q = 0; q < VEC; ++q) v[j * VEC + q] = E::get(p[q]);
        } else {
          v[j] = E::get(x[i]);
        }
      } else {
#pragma unroll
        for (int q = 0; q < VEC; ++q) v[j * VEC + q] = i + q >= 0 && i + q < a.V ? E::get(x[i + q]) : 0.0f;
      }
    }
  }
  if (tid < TILE / 32) bits[group][tid] = 0;
  __syncthreads();
  if (!zero)
    for (int k = tid; k < a.K; k += GROUP) {
      const int64_t o = a.tokens[row * a.K + k] - at;
      const float p = a.probs[row * a.K + k];
      if (p != 0.0f && o >= 0 && o < TILE) {
        put[group][o] = p;
        atomicOr(&bits[group][o / 32], 1u << (o % 32));
      }
    }
  __syncthreads();
  if (!in) return;
  const float rate = a.rate * kLog2e, less = log_s * kLog2e, g = zero ? 0.0f : a.g[row] * a.rate;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int o = (j * GROUP + tid) * VEC;
    const int64_t i = at + o;
    if (i >= a.V || i + VEC <= 0) continue;
    T out[VEC];
    if (zero) {
#pragma unroll
      for (int q = 0; q < VEC; ++q) out[q] = E::put(0.0f);
    } else {
      const uint32_t here = bits[group][o / 32] >> (o % 32);
      float d[VEC];
#pragma unroll
      for (int q = 0; q < VEC; ++q) d[q] = __builtin_amdgcn_exp2f(__builtin_fmaf(v[j * VEC + q] - m, rate, -less));
      if (here & ((1u << VEC) - 1)) {
#pragma unroll
        for (int q = 0; q < VEC; ++q)
          if (here >> q & 1) d[q] -= put[group][o + q];
      }
#pragma unroll
      for (int q = 0; q < VEC; ++q) out[q] = E::put(g * d[q]);
    }
    if (ROWS == kWhole || (VECTOR && i >= 0 && i + VEC <= a.V)) {
      vec w;
#pragma unroll
      for (int q = 0; q < VEC; ++q) w[q] = out[q];
      myelin::store<STREAM>(w, reinterpret_cast<vec *>(dx + i));
    } else {
#pragma unroll
      for (int q = 0; q < VEC; ++q)
        if (i + q >= 0 && i + q < a.V) dx[i + q] = out[q];
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

template <class E>
void launch_fwd(Args &a, hipStream_t s) {
  if (a.V <= kNarrow) {
    narrow_rows<E><<<myelin::grid_of((a.R + kWaves - 1) / kWaves), kThreads, 0, s>>>(a);
    return;
  }
  a.rows = a.R < myelin::kGridX / a.parts ? a.R : myelin::kGridX / a.parts;
  const dim3 grid(static_cast<unsigned>(a.rows * a.parts), static_cast<unsigned>((a.R + a.rows - 1) / a.rows));
  wide_rows<E><<<grid, kThreads, 0, s>>>(a);
  if (a.parts > 1) join_parts<E><<<static_cast<unsigned>(a.R), kWave, 0, s>>>(a);
}

template <class E, int GROUP>
void launch_gradient(BwdArgs &a, hipStream_t s) {
  const int64_t size = sizeof(typename E::T);
  const bool vector = (reinterpret_cast<uintptr_t>(a.x) - reinterpret_cast<uintptr_t>(a.dx)) % 16 == 0 &&
                      (a.R == 1 || (a.ld - a.V) * size % 16 == 0);
  const bool whole = myelin::aligned(a.x, 16) && a.V * size % 16 == 0;
  a.per_row = (a.V + (vector && !whole ? E::VEC - 1 : 0) + GROUP * kPerThread - 1) / (GROUP * kPerThread);
  const int64_t units = a.R * a.per_row, each = kThreads / GROUP;
  const dim3 grid = myelin::grid_of((units + each - 1) / each);
  const bool stream = a.R * a.V * size >= myelin::kStreamBytes;
  if (!vector)
    gradient<E, GROUP, kSingly, false><<<grid, kThreads, 0, s>>>(a);
  else if (whole)
    stream ? gradient<E, GROUP, kWhole, true><<<grid, kThreads, 0, s>>>(a)
           : gradient<E, GROUP, kWhole, false><<<grid, kThreads, 0, s>>>(a);
  else
    stream ? gradient<E, GROUP, kSkewed, true><<<grid, kThreads, 0, s>>>(a)
           : gradient<E, GROUP, kSkewed, false><<<grid, kThreads, 0, s>>>(a);
}

template <class E>
void launch_bwd(BwdArgs &a, hipStream_t s) {
  if (a.V <= kNarrow)
    launch_gradient<E, kWave>(a, s);
  else
    launch_gradient<E, kThreads>(a, s);
}

constexpr int kMaxTop = 1024;

int check(const char *what, const void *x, int dtype, int64_t ld, int64_t R, int64_t V, int64_t K, float temperature) {
  if (dtype != 0 && dtype != 2) return myelin::invalid("%s: unsupported dtype %d", what, dtype);
  if (R < 0 || V < 1) return myelin::invalid("%s: rows must be non-negative and V positive", what);
  if (V > 0x7fffffff || R > 0x7fffffff) return myelin::invalid("%s: R and V must be below 2^31", what);
  if (K < 1 || K > kMaxTop) return myelin::invalid("%s: K must be in [1, %d]", what, kMaxTop);
  if (R > 1 && ld < V) return myelin::invalid("%s: row stride below V", what);
  if (!(temperature > 0.0f && temperature <= 3.402823466e38f && 1.0f / temperature <= 3.402823466e38f))
    return myelin::invalid("%s: temperature must be positive and finite", what);
  if (R > 0 && !x) return myelin::invalid("%s: null pointer", what);
  return MYELIN_OK;
}

}  // namespace

extern "C" int64_t myelin_distillation_loss_workspace_bytes(int64_t R, int64_t V) {
  if (R < 1 || V <= kNarrow) return 0;
  int64_t parts, part;
  split(R, V, &parts, &part);
  return parts == 1 ? 0 : R * parts * static_cast<int64_t>(sizeof(Stats));
}

extern "C" int myelin_distillation_loss(const void *logits, int dtype, int64_t ld, const float *teacher_logits,
                                        const int64_t *teacher_tokens, float temperature, float *loss, float *probs,
                                        float *stats, int64_t R, int64_t V, int K, void *workspace,
                                        int64_t workspace_bytes, myelin_stream_t stream) {
  const char *what = "distillation_loss";
  if (int rc = check(what, logits, dtype, ld, R, V, K, temperature)) return rc;
  if (R == 0) return MYELIN_OK;
  if (!teacher_logits || !teacher_tokens || !loss || !stats) return myelin::invalid("%s: null pointer", what);
  Args a{logits, ld, teacher_logits, teacher_tokens, 1.0f / temperature, loss, probs, stats, R, V, K, 1, V, R, nullptr};
  if (const int64_t need = myelin_distillation_loss_workspace_bytes(R, V)) {
    if (!workspace || workspace_bytes < need)
      return myelin::invalid("%s: workspace of %lld bytes needed", what, static_cast<long long>(need));
    if (!myelin::aligned(workspace, 16)) return myelin::invalid("%s: workspace must be 16-byte aligned", what);
    int64_t parts;
    split(R, V, &parts, &a.part);
    a.parts = static_cast<int>(parts);
    a.part_stats = static_cast<Stats *>(workspace);
  }
  if (dtype == 0)
    launch_fwd<F32>(a, myelin::as_hip(stream));
  else
    launch_fwd<BF16>(a, myelin::as_hip(stream));
  return myelin::launched(what);
}

extern "C" int myelin_distillation_loss_bwd(const void *logits, int dtype, int64_t ld, const int64_t *teacher_tokens,
                                            const float *probs, const float *stats, const float *grad_loss,
                                            float temperature, void *grad_logits, int64_t R, int64_t V, int K,
                                            myelin_stream_t stream) {
  const char *what = "distillation_loss_bwd";
  if (int rc = check(what, logits, dtype, ld, R, V, K, temperature)) return rc;
  if (R == 0) return MYELIN_OK;
  if (!teacher_tokens || !probs || !stats || !grad_loss || !grad_logits)
    return myelin::invalid("%s: null pointer", what);
  BwdArgs a{logits, ld, teacher_tokens, probs, stats, grad_loss, 1.0f / temperature, grad_logits, R, V, K, 1};
  if (dtype == 0)
    launch_bwd<F32>(a, myelin::as_hip(stream));
  else
    launch_bwd<BF16>(a, myelin::as_hip(stream));
  return myelin::launched(what);
}
