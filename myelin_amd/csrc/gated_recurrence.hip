// A linear recurrence with a gate for every step and channel:
//
//   a_t = sigmoid(gate_t)      h_t = a_t h_{t-1} + (1 - a_t) x_t
//
// a leaky integrator whose time constant 1 / (1 - a_t) is an input.  Its adjoint,
// with g_t the gradient of h_t (of the output and of all later steps):
//
//   g_t = dh_t + a_{t+1} g_{t+1}
//   dx_t = (1 - a_t) g_t      dgate_t = g_t (h_{t-1} - x_t) a_t (1 - a_t)
//   dh_0 = a_1 g_1
//
// The backward pass takes h_{t-1} from the states that the forward pass kept
// before every kSteps-th step, in fp32, and the steps from there again: 4 / kSteps
// bytes an element, where the output's bf16 would cost h_{t-1} - x_t its accuracy.

#include "elements.h"

namespace {

using myelin::BF16;
using myelin::F32;

constexpr int kSteps = 16;  // steps between two kept states

struct Args {
  const void *x, *gate, *g_out;
  int64_t xt, xb, gt, gb, ot, ob;  // element strides of time and batch
  const int32_t *lengths;
  const float *state;  // [B, N] or null: of the first step; backward: gradient of the last
  void *out, *gx, *gg;
  float *state_out;  // [B, N] or null: the last; backward: gradient of the first
  float *kept;       // [ceil(T / kSteps), B, N] or null
  int64_t T, B, N;
};

// sigmoid and 1 - sigmoid, each to its own accuracy
struct Gate {
  float a, b;
  __device__ explicit Gate(float g) {
    const float e = myelin::exp_f32(-__builtin_fabsf(g));
    const float r = 1.0f / (1.0f + e), s = e * r;
    a = g >= 0.0f ? r : s;
    b = g >= 0.0f ? s : r;
    if (g != g) a = b = g;
  }
};

__device__ __forceinline__ int64_t steps_of(const Args &a, int64_t b) {
  if (!a.lengths) return a.T;
  const int64_t n = a.lengths[b];
  return n < 0 ? 0 : n < a.T ? n : a.T;
}

// a thread to a channel
template <class E>
__global__ __launch_bounds__(256) void forward(Args a) {
  using T = typename E::T;
  const int64_t c = myelin::block_id() * 256 + threadIdx.x;
  if (c >= a.B * a.N) return;
  const int64_t b = c / a.N, n = c - b * a.N, live = steps_of(a, b);
  const T *x = static_cast<const T *>(a.x) + b * a.xb + n, *gate = static_cast<const T *>(a.gate) + b * a.gb + n;
  T *out = static_cast<T *>(a.out) + c;
  float h = a.state ? a.state[c] : 0.0f;
  for (int64_t t = 0; t < a.T; ++t) {
    if (a.kept && t % kSteps == 0) a.kept[(t / kSteps) * a.B * a.N + c] = h;
    float o = 0.0f;
    if (t < live) {
      const Gate g(E::get(gate[t * a.gt]));
      o = h = __builtin_fmaf(g.a, h, g.b * E::get(x[t * a.xt]));
    }
    out[t * a.B * a.N] = E::put(o);
  }
  a.state_out[c] = h;
}

template <class E>
__global__ __launch_bounds__(256) void backward(Args a) {
  using T = typename E::T;
  const int64_t BN = a.B * a.N, c = myelin::block_id() * 256 + threadIdx.x;
  if (c >= BN) return;
  const int64_t b = c / a.N, n = c - b * a.N, live = steps_of(a, b);
  const T *x = static_cast<const T *>(a.x) + b * a.xb + n, *gate = static_cast<const T *>(a.gate) + b * a.gb + n;
  const T *go = a.g_out ? static_cast<const T *>(a.g_out) + b * a.ob + n : nullptr;
  T *gx = a.gx ? static_cast<T *>(a.gx) + c : nullptr, *gg = a.gg ? static_cast<T *>(a.gg) + c : nullptr;
  float g = a.state ? a.state[c] : 0.0f;
  for (int64_t t0 = (a.T - 1) / kSteps * kSteps; t0 >= 0; t0 -= kSteps) {
    float h[kSteps];
    float s = a.kept[(t0 / kSteps) * BN + c];
    for (int i = 0; i < kSteps; ++i) {
      h[i] = s;
      if (t0 + i < live) {
        const Gate k(E::get(gate[(t0 + i) * a.gt]));
        s = __builtin_fmaf(k.a, s, k.b * E::get(x[(t0 + i) * a.xt]));
      }
    }
    for (int i = kSteps - 1; i >= 0; --i) {
      const int64_t t = t0 + i;
      if (t >= a.T) continue;
      float dx = 0.0f, dg = 0.0f;
      if (t < live) {
        const Gate k(E::get(gate[t * a.gt]));
        if (go) g += E::get(go[t * a.ot]);
        dx = k.b * g;
        dg = dx * (h[i] - E::get(x[t * a.xt])) * k.a;
        g = k.a * g;
      }
      if (gx) gx[t * BN] = E::put(dx);
      if (gg) gg[t * BN] = E::put(dg);
    }
  }
  if (a.state_out) a.state_out[c] = g;
}

template <class E>
__global__ __launch_bounds__(256) void step(Args a) {
  using T = typename E::T;
  const int64_t c = myelin::block_id() * 256 + threadIdx.x;
  if (c >= a.B * a.N) return;
  const int64_t b = c / a.N, n = c - b * a.N;
  const Gate g(E::get(static_cast<const T *>(a.gate)[b * a.gb + n]));
  const float h = __builtin_fmaf(g.a, a.state[c], g.b * E::get(static_cast<const T *>(a.x)[b * a.xb + n]));
  a.state_out[c] = h;
  static_cast<T *>(a.out)[c] = E::put(h);
}

int check(const char *what, int dtype, int64_t T, int64_t B, int64_t N) {
  if (dtype != 0 && dtype != 2) return myelin::invalid("%s: unsupported dtype %d", what, dtype);
  if (T < 1 || B < 0 || N < 0) return myelin::invalid("%s: T must be positive, B and N not negative", what);
  if (T >= int64_t{1} << 31 || B >= int64_t{1} << 31 || N >= int64_t{1} << 31 || B * N >= int64_t{1} << 36)
    return myelin::invalid("%s: too many steps or channels", what);
  return MYELIN_OK;
}

}  // namespace

extern "C" int64_t myelin_gated_recurrence_kept_elems(int64_t T, int64_t B, int64_t N) {
  return (T + kSteps - 1) / kSteps * B * N;
}

extern "C" int64_t myelin_gated_recurrence_workspace_elems(int dtype, int64_t T, int64_t B, int64_t N, int backward) {
  return 0;
}

extern "C" int myelin_gated_recurrence_fwd(const void *x, const void *gate, int dtype, const int64_t *strides,
                                           const float *state, const int32_t *lengths, void *out, float *state_out,
                                           float *kept, int64_t T, int64_t B, int64_t N, float *workspace,
                                           int64_t workspace_elems, myelin_stream_t stream) {
  const char *what = "gated_recurrence_fwd";
  if (int rc = check(what, dtype, T, B, N)) return rc;
  if (B == 0 || N == 0) return MYELIN_OK;
  if (!x || !gate || !strides || !out || !state_out) return myelin::invalid("%s: null pointer", what);
  Args a{x, gate, nullptr, strides[0], strides[1], strides[2], strides[3], 0, 0, lengths, state, out, nullptr, nullptr,
         state_out, kept, T, B, N};
  const dim3 grid = myelin::grid_of((B * N + 255) / 256);
  if (dtype == 0)
    forward<F32><<<grid, 256, 0, myelin::as_hip(stream)>>>(a);
  else
    forward<BF16><<<grid, 256, 0, myelin::as_hip(stream)>>>(a);
  return myelin::launched(what);
}

extern "C" int myelin_gated_recurrence_bwd(const void *x, const void *gate, const void *grad_out, int dtype,
                                           const int64_t *strides, const int32_t *lengths, const float *kept,
                                           const float *grad_state_out, void *grad_x, void *grad_gate,
                                           float *grad_state, int64_t T, int64_t B, int64_t N, float *workspace,
                                           int64_t workspace_elems, myelin_stream_t stream) {
  const char *what = "gated_recurrence_bwd";
  if (int rc = check(what, dtype, T, B, N)) return rc;
  if (B == 0 || N == 0) return MYELIN_OK;
  if (!x || !gate || !strides || !kept) return myelin::invalid("%s: null pointer", what);
  Args a{x, gate, grad_out, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], lengths,
         grad_state_out, nullptr, grad_x, grad_gate, grad_state, const_cast<float *>(kept), T, B, N};
  const dim3 grid = myelin::grid_of((B * N + 255) / 256);
  if (dtype == 0)
    backward<F32><<<grid, 256, 0, myelin::as_hip(stream)>>>(a);
  else
    backward<BF16><<<grid, 256, 0, myelin::as_hip(stream)>>>(a);
  return myelin::launched(what);
}

extern "C" int myelin_gated_recurrence_step(const void *x, const void *gate, int dtype, const int64_t *strides,
                                            const float *state, void *out, float *state_out, int64_t B, int64_t N,
                                            myelin_stream_t stream) {
  const char *what = "gated_recurrence_step";
  if (int rc = check(what, dtype, 1, B, N)) return rc;
  if (B == 0 || N == 0) return MYELIN_OK;
  if (!x || !gate || !strides || !state || !out || !state_out) return myelin::invalid("%s: null pointer", what);
  Args a{x, gate, nullptr, 0, strides[0], 0, strides[1], 0, 0, nullptr, state, out, nullptr, nullptr, state_out,
         nullptr, 1, B, N};
  const dim3 grid = myelin::grid_of((B * N + 255) / 256);
  if (dtype == 0)
    step<F32><<<grid, 256, 0, myelin::as_hip(stream)>>>(a);
  else
    step<BF16><<<grid, 256, 0, myelin::as_hip(stream)>>>(a);
  return myelin::launched(what);
}
