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

#include "elements.h"

namespace {

using myelin::BF16;
using myelin::F32;
using myelin::kLog2e;
using myelin::kWave;

constexpr float kLowest = -3.402823466e38f;
constexpr float kInf = __builtin_huge_valf();
constexpr int kThreads = 256, kWaves = kThreads / kWave;

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
};

__device__ __forceinline__ bool empty(const Args &a, int64_t at) { return a.tokens[at] == -1 || a.values[at] == -kInf; }

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

// The row's loss from its logits' statistics, by one wave.
template <class E>
__device__ __forceinline__ void finish(const Args &a, int64_t row, Stats t, int lane) {
  const int64_t first = row * a.K;
  const typename E::T *x = static_cast<const typename E::T *>(a.x) + row * a.ld;
  float peak = kLowest;
  bool bad = false;
  for (int k = lane; k < a.K; k += kWave)
    if (!empty(a, first + k)) {
      peak = fmaxf(peak, a.values[first + k]);
      bad |= a.tokens[first + k] < 0 || a.tokens[first + k] >= a.V;
    }
  for (int o = kWave >> 1; o > 0; o >>= 1) peak = fmaxf(peak, __shfl_xor(peak, o));
  float total = 0.0f;
  for (int k = lane; k < a.K; k += kWave)
    if (!empty(a, first + k)) total += myelin::exp_f32((a.values[first + k] - peak) * a.rate);
  total = wave_sum(total);
  bad = __any(bad);
  const float log_total = logf(total), log_s = t.s == 0.0f ? -kInf : logf(t.s);
  float loss = 0.0f;
  for (int k = lane; k < a.K; k += kWave) {
    float p = 0.0f;
    if (!empty(a, first + k)) {
      const float d = (a.values[first + k] - peak) * a.rate;
      p = myelin::exp_f32(d) / total;
      const int64_t token = a.tokens[first + k];
      if (p != 0.0f && !bad) {
        // nothing allowed: log q is -inf for every token
        const float log_q = t.s == 0.0f ? -kInf : (E::get(x[token]) - t.m) * a.rate - log_s;
        loss += p * ((d - log_total) - log_q);
      }
    }
    if (a.probs) a.probs[first + k] = p;
  }
  loss = wave_sum(loss);
  if (lane == 0) {
    a.loss[row] = bad ? __builtin_nanf("") : loss;
    a.stats[row] = bad ? __builtin_nanf("") : t.m;
    a.stats[a.R + row] = bad ? 0.0f : log_s;
  }
}

__device__ __forceinline__ bool nothing(const Args &a, int64_t row) {
  bool some = false;
  for (int k = threadIdx.x & (kWave - 1); k < a.K; k += kWave) some |= !empty(a, row * a.K + k);
  return !__any(some);
}

// a workgroup to a row
template <class E>
__global__ __launch_bounds__(kThreads) void rows(Args a) {
  __shared__ Stats red[kWaves];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = tid >> 6;
  const int64_t row = myelin::block_id();
  if (row >= a.R) return;
  if (nothing(a, row)) {
    if (w == 0) store_nothing(a, row, lane);
    return;
  }
  const typename E::T *x = static_cast<const typename E::T *>(a.x) + row * a.ld;
  Stats t = Stats::none();
  for (int64_t i = tid; i < a.V; i += kThreads) {
    const float v = E::get(x[i]);
    if (v > t.m) t.rescale(v, a.rate);
    t.s += myelin::exp_f32((v - t.m) * a.rate);
  }
  t = across(t, a.rate);
  if (lane == 0) red[w] = t;
  __syncthreads();
  t = red[0];
  for (int o = 1; o < kWaves; ++o) t.merge(red[o], a.rate);
  if (w == 0) finish<E>(a, row, t, lane);
}

struct BwdArgs {
  const void *x;
  int64_t ld;
  const int64_t *tokens;
  const float *probs, *stats, *g;
  float rate;
  void *dx;  // [R, V] contiguous
  int64_t R, V;
  int K;
};

template <class E>
__global__ __launch_bounds__(kThreads) void gradient(BwdArgs a) {
  const int64_t at = myelin::block_id() * kThreads + threadIdx.x;
  if (at >= a.R * a.V) return;
  const int64_t row = at / a.V, i = at - row * a.V;
  const float m = a.stats[row], log_s = a.stats[a.R + row];
  float d = 0.0f;
  if (log_s != -kInf) {
    const float x = E::get(static_cast<const typename E::T *>(a.x)[row * a.ld + i]);
    d = myelin::exp_f32((x - m) * a.rate - log_s);
    for (int k = 0; k < a.K; ++k)
      if (a.tokens[row * a.K + k] == i) d -= a.probs[row * a.K + k];
    d *= a.g[row] * a.rate;
  }
  static_cast<typename E::T *>(a.dx)[at] = E::put(d);
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

extern "C" int64_t myelin_distillation_loss_workspace_bytes(int64_t R, int64_t V) { return 0; }

extern "C" int myelin_distillation_loss(const void *logits, int dtype, int64_t ld, const float *teacher_logits,
                                        const int64_t *teacher_tokens, float temperature, float *loss, float *probs,
                                        float *stats, int64_t R, int64_t V, int K, void *workspace,
                                        int64_t workspace_bytes, myelin_stream_t stream) {
  const char *what = "distillation_loss";
  if (int rc = check(what, logits, dtype, ld, R, V, K, temperature)) return rc;
  if (R == 0) return MYELIN_OK;
  if (!teacher_logits || !teacher_tokens || !loss || !stats) return myelin::invalid("%s: null pointer", what);
  Args a{logits, ld, teacher_logits, teacher_tokens, 1.0f / temperature, loss, probs, stats, R, V, K};
  const dim3 grid = myelin::grid_of(R);
  if (dtype == 0)
    rows<F32><<<grid, kThreads, 0, myelin::as_hip(stream)>>>(a);
  else
    rows<BF16><<<grid, kThreads, 0, myelin::as_hip(stream)>>>(a);
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
  BwdArgs a{logits, ld, teacher_tokens, probs, stats, grad_loss, 1.0f / temperature, grad_logits, R, V, K};
  const dim3 grid = myelin::grid_of((R * V + kThreads - 1) / kThreads);
  if (dtype == 0)
    gradient<F32><<<grid, kThreads, 0, myelin::as_hip(stream)>>>(a);
  else
    gradient<BF16><<<grid, kThreads, 0, myelin::as_hip(stream)>>>(a);
  return myelin::launched(what);
}
