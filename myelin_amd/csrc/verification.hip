// Verification of drafted tokens (speculative sampling): with the target's
// probabilities p, the draft's q, the drafted tokens x and uniform numbers u,
//
//   x_i is taken while  u_i q_i(x_i) < p_i(x_i)
//   the first that is not is replaced by a draw from  w = max(p_i - q_i, 0);
//   after n taken ones the next token is a draw from  w = p_{n+1}
//   a draw: the lowest token whose  w_0 + ... + w_token > u_last (w_0 + ... + w_{V-1})
//
// so that the tokens have the target's distribution.  Without q the draft was a
// choice (q is 1 at x_i).  All of it is computed in 64 bits: a token at the border
// of two must not depend on the order of a sum.  What is not positive and finite
// counts as w = 0; where w has nothing (p <= q everywhere, by rounding) the draw is
// from p, and where that has nothing either the token is -1.

#include "elements.h"

namespace {

using myelin::BF16;
using myelin::F32;
using myelin::kWave;

constexpr int kThreads = 256, kWaves = kThreads / kWave;

struct Args {
  const void *p, *q;  // q null: a choice
  int64_t pn, pb, qn, qb;
  const int64_t *tokens;  // [n, B]
  const float *uniforms;  // [n + 1, B]
  const int32_t *lengths;
  int64_t *accepted, *out;
  int64_t n, B, V;
};

// How many tokens of a sequence are taken, by one wave.
template <class E>
__device__ __forceinline__ int64_t taken(const Args &a, int64_t b, int64_t drafted, int lane) {
  using T = typename E::T;
  for (int64_t at = 0; at < drafted; at += kWave) {
    const int64_t i = at + lane;
    bool good = true;
    if (i < drafted) {
      const int64_t x = a.tokens[i * a.B + b];
      good = false;
      if (x >= 0 && x < a.V) {
        const double p = E::get(static_cast<const T *>(a.p)[i * a.pn + b * a.pb + x]);
        const double q = a.q ? E::get(static_cast<const T *>(a.q)[i * a.qn + b * a.qb + x]) : 1.0;
        good = static_cast<double>(a.uniforms[i * a.B + b]) * q < p;
      }
    }
    const uint64_t refused = ~__ballot(good);
    if (refused) return at + __builtin_ctzll(refused);
  }
  return drafted;
}

__device__ __forceinline__ double positive(double w) { return w > 0.0 && w < __builtin_huge_val() ? w : 0.0; }

// What a draw is made from.
template <class E>
struct Weights {
  using T = typename E::T;
  const T *p, *q;  // q null: p alone, less `without`
  int64_t without;
  __device__ double of_p(int64_t i) const { return positive(E::get(p[i])); }
  __device__ double operator()(int64_t i) const {
    const double w = E::get(p[i]);
    if (q) return positive(w - static_cast<double>(E::get(q[i])));
    return i == without ? 0.0 : positive(w);
  }
};

__device__ __forceinline__ int64_t drafted_of(const Args &a, int64_t b) {
  if (!a.lengths) return a.n;
  const int64_t l = a.lengths[b];
  return l < 0 ? 0 : l < a.n ? l : a.n;
}

template <class E>
__device__ __forceinline__ Weights<E> weights_of(const Args &a, int64_t b, int64_t accepted, bool refused) {
  using T = typename E::T;
  Weights<E> w{static_cast<const T *>(a.p) + accepted * a.pn + b * a.pb, nullptr, -1};
  if (refused && a.q) w.q = static_cast<const T *>(a.q) + accepted * a.qn + b * a.qb;
  if (refused && !a.q) w.without = a.tokens[accepted * a.B + b];
  return w;
}

__device__ __forceinline__ double wave_sum(double v) {
  for (int o = kWave >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// What each part of a row holds: the sum of w, and that of p alone.
struct Sums {
  double rest, all;
};

// Tiles of a part: enough workgroups to fill the chip where sequences are few.
constexpr int kPer = 16, kTile = kThreads * kPer, kMaxParts = 512;

void split(int64_t B, int64_t V, int64_t *parts, int64_t *part) {
  const int64_t tiles = (V + kTile - 1) / kTile;
  int64_t n = B > 0 ? 1024 / B : 1;
  n = n < 1 ? 1 : n > kMaxParts ? kMaxParts : n;
  if (n > tiles) n = tiles;
  const int64_t per = (tiles + n - 1) / n;
  *part = per * kTile;
  *parts = (tiles + per - 1) / per;
}

// A workgroup to a part of a sequence's row: each finds out by itself how many
// tokens are taken, so that none waits for another.
template <class E>
__global__ __launch_bounds__(kThreads) void sum_parts(Args a, int parts, int64_t part, Sums *sums) {
  __shared__ Sums red[kWaves];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6;
  const int64_t b = blockIdx.x / parts, at = blockIdx.x % parts;
  const int64_t drafted = drafted_of(a, b), accepted = taken<E>(a, b, drafted, lane);
  const bool refused = accepted < drafted;
  const Weights<E> w = weights_of<E>(a, b, accepted, refused);
  const int64_t begin = at * part, end = begin + part < a.V ? begin + part : a.V;
  Sums s{0.0, 0.0};
  for (int64_t i = begin + tid; i < end; i += kThreads) {
    s.rest += w(i);
    s.all += w.of_p(i);
  }
  s = {wave_sum(s.rest), wave_sum(s.all)};
  if (lane == 0) red[wave] = s;
  if (at == 0) {
    for (int64_t i = tid; i <= a.n; i += kThreads)
      if (i != accepted) a.out[i * a.B + b] = i < accepted ? a.tokens[i * a.B + b] : -1;
    if (tid == 0) a.accepted[b] = accepted;
  }
  __syncthreads();
  if (tid == 0) {
    for (int o = 1; o < kWaves; ++o) {
      s.rest += red[o].rest;
      s.all += red[o].all;
    }
    sums[blockIdx.x] = s;
  }
}

// The sum of v over the threads before this one, and over all.
__device__ __forceinline__ double before(double v, double *red, double *total) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  double run = v;
  for (int o = 1; o < kWave; o <<= 1) {
    const double up = __shfl_up(run, o);
    if (lane >= o) run += up;
  }
  __syncthreads();  // (the last call's values are read)
  if (lane == kWave - 1) red[wave] = run;
  __syncthreads();
  double base = 0.0, sum = 0.0;
  for (int o = 0; o < kWaves; ++o) {
    if (o < wave) base += red[o];
    sum += red[o];
  }
  *total = sum;
  const double up = __shfl_up(run, 1);
  return base + (lane ? up : 0.0);
}

// A workgroup to a sequence: the part of its row that the draw falls into, then
// the token.  Sums in another order than the parts' may differ in their last bits:
// a draw that is not found in its part is looked for in the next ones, and the last
// token with a weight takes what is left.
template <class E>
__global__ __launch_bounds__(kThreads) void locate(Args a, int parts, int64_t part, const Sums *sums) {
  __shared__ double red[kWaves];
  __shared__ int first, last;
  __shared__ double run_at;
  __shared__ int64_t found, some;
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x, accepted = a.accepted[b];
  const bool refused = accepted < drafted_of(a, b);
  Weights<E> w = weights_of<E>(a, b, accepted, refused);
  sums += b * parts;
  // each thread two parts
  double s[2], total, ignored;
  for (int o = 0; o < 2; ++o) s[o] = 2 * tid + o < parts ? sums[2 * tid + o].rest : 0.0;
  double base = before(s[0] + s[1], red, &total);
  if (!(total > 0.0)) {
    w.q = nullptr;
    w.without = -1;
    for (int o = 0; o < 2; ++o) s[o] = 2 * tid + o < parts ? sums[2 * tid + o].all : 0.0;
    base = before(s[0] + s[1], red, &total);
  }
  if (!(total > 0.0)) {
    if (tid == 0) a.out[accepted * a.B + b] = -1;
    return;
  }
  const double bound = static_cast<double>(a.uniforms[a.n * a.B + b]) * total;
  if (tid == 0) {
    first = kMaxParts;
    last = 0;
    found = a.V;
    some = -1;
  }
  __syncthreads();
  const double from_here[2] = {base, base + s[0]};
  for (int o = 0; o < 2; ++o)
    if (s[o] > 0.0) {
      atomicMax(&last, 2 * tid + o);
      if (from_here[o] + s[o] > bound) atomicMin(&first, 2 * tid + o);
    }
  __syncthreads();
  const int from = first < kMaxParts ? first : last;
  for (int o = 0; o < 2; ++o)
    if (2 * tid + o == from) run_at = from_here[o];
  __syncthreads();
  double run = run_at;
  for (int64_t at = from * part; at < a.V; at += kTile) {
    const int64_t mine = at + tid * kPer;
    double v[kPer], sum = 0.0;
    for (int o = 0; o < kPer; ++o) {
      v[o] = mine + o < a.V ? w(mine + o) : 0.0;
      sum += v[o];
    }
    double here = run + before(sum, red, &ignored);
    int64_t hit = a.V, kept = -1;
    for (int o = 0; o < kPer; ++o) {
      here += v[o];
      if (v[o] > 0.0) {
        kept = mine + o;
        if (hit == a.V && here > bound) hit = mine + o;
      }
    }
    if (hit < a.V) atomicMin(reinterpret_cast<unsigned long long *>(&found), static_cast<unsigned long long>(hit));
    if (kept >= 0) atomicMax(reinterpret_cast<long long *>(&some), static_cast<long long>(kept));
    __syncthreads();
    if (found < a.V) break;  // (the same for all threads)
    run += ignored;
  }
  if (tid == 0) a.out[accepted * a.B + b] = found < a.V ? found : some;
}

template <class E>
void launch(const Args &a, int64_t parts, int64_t part, Sums *sums, hipStream_t s) {
  sum_parts<E><<<static_cast<unsigned>(a.B * parts), kThreads, 0, s>>>(a, static_cast<int>(parts), part, sums);
  locate<E><<<static_cast<unsigned>(a.B), kThreads, 0, s>>>(a, static_cast<int>(parts), part, sums);
}

}  // namespace

extern "C" int64_t myelin_verify_draft_workspace_bytes(int64_t B, int64_t V) {
  if (B < 1 || V < 1) return 0;
  int64_t parts, part;
  split(B, V, &parts, &part);
  return B * parts * static_cast<int64_t>(sizeof(Sums));
}

extern "C" int myelin_verify_draft(const void *target, const void *draft, int dtype, const int64_t *strides,
                                   const int64_t *tokens, const float *uniforms, const int32_t *lengths,
                                   int64_t *accepted, int64_t *out_tokens, int64_t n, int64_t B, int64_t V,
                                   void *workspace, int64_t workspace_bytes, myelin_stream_t stream) {
  const char *what = "verify_draft";
  if (dtype != 0 && dtype != 2) return myelin::invalid("%s: unsupported dtype %d", what, dtype);
  if (n < 0 || B < 0 || V < 1) return myelin::invalid("%s: V must be positive, n and B not negative", what);
  if (n >= int64_t{1} << 31 || B >= int64_t{1} << 24 || V >= int64_t{1} << 31)
    return myelin::invalid("%s: too many tokens or sequences", what);
  if (B == 0) return MYELIN_OK;
  if (!target || !strides || !uniforms || !accepted || !out_tokens || (n > 0 && !tokens))
    return myelin::invalid("%s: null pointer", what);
  int64_t parts, part;
  split(B, V, &parts, &part);
  const int64_t need = myelin_verify_draft_workspace_bytes(B, V);
  if (!workspace || workspace_bytes < need)
    return myelin::invalid("%s: workspace of %lld bytes needed", what, static_cast<long long>(need));
  if (!myelin::aligned(workspace, 16)) return myelin::invalid("%s: workspace must be 16-byte aligned", what);
  Args a{target, draft, strides[0], strides[1], draft ? strides[2] : 0, draft ? strides[3] : 0, tokens, uniforms,
         lengths, accepted, out_tokens, n, B, V};
  if (dtype == 0)
    launch<F32>(a, parts, part, static_cast<Sums *>(workspace), myelin::as_hip(stream));
  else
    launch<BF16>(a, parts, part, static_cast<Sums *>(workspace), myelin::as_hip(stream));
  return myelin::launched(what);
}
