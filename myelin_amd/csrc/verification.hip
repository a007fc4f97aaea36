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
  int64_t n, B, V, pieces;
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

// A row in pieces of 1024 tokens, a wave each: what a piece's weights add up to, and
// what p alone does.
constexpr int kEach = 16, kPiece = kEach * kWave;

struct Sums {
  double rest, all;
};

// Each wave finds out by itself how many tokens are taken, so that none waits for
// another: 64 sequences of 8 tokens and 100003 fp32 probabilities 12.7 us (51 MB, 4
// TB/s, after two reads that wait for each other), one of 32768 5 us.
template <class E>
__global__ __launch_bounds__(kThreads) void sum_pieces(Args a, Sums *sums) {
  using T = typename E::T;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t unit = myelin::block_id() * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t b = unit / a.pieces, piece = unit - b * a.pieces;
  if (b >= a.B) return;  // the whole wave
  const int64_t drafted = drafted_of(a, b), accepted = taken<E>(a, b, drafted, lane);
  const Weights<E> w = weights_of<E>(a, b, accepted, accepted < drafted);
  if (piece == 0) {
    for (int64_t i = lane; i <= a.n; i += kWave)
      if (i != accepted) a.out[i * a.B + b] = i < accepted ? a.tokens[i * a.B + b] : -1;
    if (lane == 0) a.accepted[b] = accepted;
  }
  // (loads under conditions wait for each other: past the end it is the last token's)
  const int64_t at = piece * kPiece + lane;
  T p[kEach], q[kEach];
#pragma unroll
  for (int o = 0; o < kEach; ++o) p[o] = w.p[at + o * kWave < a.V ? at + o * kWave : a.V - 1];
  if (w.q) {
#pragma unroll
    for (int o = 0; o < kEach; ++o) q[o] = w.q[at + o * kWave < a.V ? at + o * kWave : a.V - 1];
  }
  Sums s{0.0, 0.0};
#pragma unroll
  for (int o = 0; o < kEach; ++o) {
    const bool in = at + o * kWave < a.V;
    const double v = E::get(p[o]);
    s.all += in ? positive(v) : 0.0;
    if (w.q)
      s.rest += in ? positive(v - static_cast<double>(E::get(q[o]))) : 0.0;
    else
      s.rest += in && at + o * kWave != w.without ? positive(v) : 0.0;
  }
  s = {wave_sum(s.rest), wave_sum(s.all)};
  if (lane == 0) sums[unit] = s;
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

// Of values that grow from thread to thread: the smallest and the largest of the
// workgroup's, by one atomic of each wave (by one of each lane: locate 17 us, not 5).
__device__ __forceinline__ void take_first(unsigned long long *to, unsigned long long v, bool have) {
  const uint64_t m = __ballot(have);
  if (m && (threadIdx.x & (kWave - 1)) == __builtin_ctzll(m)) atomicMin(to, v);
}
__device__ __forceinline__ void take_last(long long *to, long long v, bool have) {
  const uint64_t m = __ballot(have);
  if (m && (threadIdx.x & (kWave - 1)) == 63 - __builtin_clzll(m)) atomicMax(to, v);
}

// A workgroup to a sequence: the piece of its row that the draw falls into, then the
// token.  Sums in another order than the pieces' may differ in their last bits: a
// draw that is not found in its piece is looked for in the next ones, and the last
// token with a weight takes what is left.  5 us: latency of reads that follow from each
// other.
template <class E>
__global__ __launch_bounds__(kThreads) void locate(Args a, const Sums *sums) {
  constexpr int FEW = kPiece / kThreads;
  __shared__ double red[kWaves];
  __shared__ unsigned long long first, found;
  __shared__ long long last, some;
  __shared__ double run_at;
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x, accepted = a.accepted[b];
  Weights<E> w = weights_of<E>(a, b, accepted, accepted < drafted_of(a, b));
  sums += b * a.pieces;
  // each thread has some pieces in a row
  const int64_t each = (a.pieces + kThreads - 1) / kThreads, from = tid * each;
  const int64_t to = from + each < a.pieces ? from + each : a.pieces;
  const double u = a.uniforms[a.n * a.B + b];
  const Sums own = from < to ? sums[from] : Sums{0.0, 0.0};  // (all there are below 2^18 tokens)
  double rest = own.rest, all = own.all, total, ignored;
  for (int64_t o = from + 1; o < to; ++o) {
    rest += sums[o].rest;
    all += sums[o].all;
  }
  double base = before(rest, red, &total);
  const bool refilled = !(total > 0.0);
  if (refilled) {
    w.q = nullptr;
    w.without = -1;
    base = before(all, red, &total);
  }
  if (!(total > 0.0)) {
    if (tid == 0) a.out[accepted * a.B + b] = -1;
    return;  // the whole workgroup
  }
  const double bound = u * total;
  if (tid == 0) {
    first = found = ~0ull;
    last = some = -1;
  }
  __syncthreads();
  long long mine = -1;
  unsigned long long hit = ~0ull;
  double run = base, at_hit = 0.0, at_last = 0.0;
  for (int64_t o = from; o < to; ++o) {
    const Sums here = o == from ? own : sums[o];
    const double v = refilled ? here.all : here.rest;
    if (v > 0.0) {
      mine = o;
      at_last = run;
      if (hit == ~0ull && run + v > bound) {
        hit = static_cast<unsigned long long>(o);
        at_hit = run;
      }
    }
    run += v;
  }
  take_first(&first, hit, hit != ~0ull);
  take_last(&last, mine, mine >= 0);
  __syncthreads();
  const int64_t start = first != ~0ull ? static_cast<int64_t>(first) : last;
  if (start >= from && start < to) run_at = first != ~0ull ? at_hit : at_last;
  __syncthreads();
  run = run_at;
  for (int64_t at = start * kPiece; at < a.V; at += kPiece) {
    double v[FEW], sum = 0.0;
    const int64_t here = at + tid * FEW;
#pragma unroll
    for (int o = 0; o < FEW; ++o) {
      const double weight = w(here + o < a.V ? here + o : a.V - 1);
      v[o] = here + o < a.V ? weight : 0.0;
      sum += v[o];
    }
    double upto = run + before(sum, red, &ignored);
    unsigned long long at_bound = ~0ull;
    long long kept = -1;
#pragma unroll
    for (int o = 0; o < FEW; ++o) {
      upto += v[o];
      if (v[o] > 0.0) {
        kept = here + o;
        if (at_bound == ~0ull && upto > bound) at_bound = static_cast<unsigned long long>(here + o);
      }
    }
    take_first(&found, at_bound, at_bound != ~0ull);
    take_last(&some, kept, kept >= 0);
    __syncthreads();
    if (found != ~0ull) break;  // (the same for all threads)
    run += ignored;
  }
  if (tid == 0) a.out[accepted * a.B + b] = found != ~0ull ? static_cast<int64_t>(found) : some;
}

template <class E>
void launch(const Args &a, Sums *sums, hipStream_t s) {
  sum_pieces<E><<<myelin::grid_of((a.B * a.pieces + kWaves - 1) / kWaves), kThreads, 0, s>>>(a, sums);
  locate<E><<<static_cast<unsigned>(a.B), kThreads, 0, s>>>(a, sums);
}

}  // namespace

extern "C" int64_t myelin_verify_draft_workspace_bytes(int64_t B, int64_t V) {
  return B < 1 || V < 1 ? 0 : B * ((V + kPiece - 1) / kPiece) * static_cast<int64_t>(sizeof(Sums));
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
  const int64_t need = myelin_verify_draft_workspace_bytes(B, V);
  if (!workspace || workspace_bytes < need)
    return myelin::invalid("%s: workspace of %lld bytes needed", what, static_cast<long long>(need));
  if (!myelin::aligned(workspace, 16)) return myelin::invalid("%s: workspace must be 16-byte aligned", what);
  Args a{target, draft, strides[0], strides[1], draft ? strides[2] : 0, draft ? strides[3] : 0, tokens, uniforms,
         lengths, accepted, out_tokens, n, B, V, (V + kPiece - 1) / kPiece};
  if (dtype == 0)
    launch<F32>(a, static_cast<Sums *>(workspace), myelin::as_hip(stream));
  else
    launch<BF16>(a, static_cast<Sums *>(workspace), myelin::as_hip(stream));
  return myelin::launched(what);
}
