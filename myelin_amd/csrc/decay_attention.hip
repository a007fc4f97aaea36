// Linear attention with a decay for each head.
//
//   S_t = d_h S_{t-1} + k_t v_t^T        o_t = scale S_t^T q_t
//
// [Dk, Dv] states in fp32 for every batch row and head; a row b has lengths[b]
// steps, later ones leave its state as it is and give o_t = 0.
//
// The backward pass, with G_t = dL/dS_t = d_h G_{t+1} + scale q_t do_t^T (and
// dL/dS_T added at the last step):
//   dq_t = scale S_t do_t    dk_t = G_t v_t    dv_t = G_t^T k_t    dS_0 = d_h G_0
// These are the forward's form again, with the roles changed and for dk and dv
// with time reversed: dq = LA(do, v, k), dk = RLA(v, do, q), dv = RLA(k, q, do)
// for LA(a, b, c): X = d X + b c^T, o = a X, and RLA: X = X + b c^T, o = a X,
// X = d X.  One kernel computes all four (Problem).

#include "common.h"

namespace {

using myelin::kWave;

constexpr int kMaxDim = 128;

struct F32 {
  using T = float;
};
struct BF16 {
  using T = __bf16;
};

// One recurrence over [T, B, H] rows; a, b of KD elements and c, o of VD, each
// with unit stride and strides of t, b and h.  The state of (b, h) is KD x VD
// with element strides sk and sv, those of one (b, h) KD * VD apart.
struct Problem {
  const void *a, *b, *c;
  void *o;
  int64_t at, ab, ah, bt, bb, bh, ct, cb, ch, ot, ob, oh;
  const float *s_in;
  float *s_out;
  int64_t sk, sv;
  int KD, VD;
  int ga, gb, gc;  // query heads to a head of a, b, c
  float in_scale, out_scale, o_scale;
  int reverse, o_f32;
};

struct Args {
  Problem p[3];
  const float *decay;
  const int32_t *lengths;
  int64_t T, B, H;
};

// The recurrence step by step: a lane has a column of the state.
template <class E, int KDP>
__global__ __launch_bounds__(64) void recurrent(Args args) {
  using T = typename E::T;
  const Problem &p = args.p[blockIdx.z];
  __shared__ float sa[KDP], sb[KDP];
  const int lane = threadIdx.x;
  const int64_t b = blockIdx.x / args.H, h = blockIdx.x % args.H;
  const int v = blockIdx.y * 64 + lane;
  if (static_cast<int>(blockIdx.y) * 64 >= p.VD) return;
  const bool on = v < p.VD;
  const float d = args.decay[h];
  int64_t n = args.T;
  if (args.lengths) {
    n = args.lengths[b];
    n = n < 0 ? 0 : n > args.T ? args.T : n;
  }
  const T *pa = static_cast<const T *>(p.a) + b * p.ab + (h / p.ga) * p.ah;
  const T *pb = static_cast<const T *>(p.b) + b * p.bb + (h / p.gb) * p.bh;
  const T *pc = static_cast<const T *>(p.c) + b * p.cb + (h / p.gc) * p.ch;
  const int64_t state = (b * args.H + h) * p.KD * p.VD;
  float X[KDP];
#pragma unroll
  for (int k = 0; k < KDP; ++k)
    X[k] = (p.s_in && on && k < p.KD) ? p.s_in[state + k * p.sk + v * p.sv] * p.in_scale : 0.0f;
  for (int64_t r = 0; r < args.T; ++r) {
    const int64_t t = (p.reverse && r < n) ? n - 1 - r : r;
    const int64_t o = t * p.ot + b * p.ob + h * p.oh + v;
    float out = 0.0f;
    if (r < n) {
      __syncthreads();
      for (int k = lane; k < KDP; k += 64) {
        sa[k] = k < p.KD ? static_cast<float>(pa[t * p.at + k]) : 0.0f;
        sb[k] = k < p.KD ? static_cast<float>(pb[t * p.bt + k]) : 0.0f;
      }
      __syncthreads();
      const float c = on ? static_cast<float>(pc[t * p.ct + v]) : 0.0f;
#pragma unroll
      for (int k = 0; k < KDP; ++k) {
        X[k] = __builtin_fmaf(sb[k], c, p.reverse ? X[k] : d * X[k]);
        out = __builtin_fmaf(sa[k], X[k], out);
        if (p.reverse) X[k] *= d;
      }
    }
    if (on) {
      if (p.o_f32)
        static_cast<float *>(p.o)[o] = out * p.o_scale;
      else
        static_cast<T *>(p.o)[o] = static_cast<T>(out * p.o_scale);
    }
  }
  if (p.s_out && on) {
#pragma unroll
    for (int k = 0; k < KDP; ++k)
      if (k < p.KD) p.s_out[state + k * p.sk + v * p.sv] = X[k] * p.out_scale;
  }
}

// Sums the fp32 gradients of the query heads that share a key/value head, in
// their order: from [rows, Hk, group, D] to [rows, Hk, D].
template <class E>
__global__ __launch_bounds__(256) void sum_groups(const float *__restrict__ from, void *__restrict__ to, int64_t n,
                                                  int group, int D) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t head = i / D;
  const float *f = from + head * group * D + (i - head * D);
  float s = 0.0f;
  for (int g = 0; g < group; ++g) s += f[static_cast<int64_t>(g) * D];
  static_cast<typename E::T *>(to)[i] = static_cast<typename E::T>(s);
}

// ---- one step --------------------------------------------------------------
struct StepArgs {
  const void *q, *k, *v;
  int64_t qb, qh, kb, kh, vb, vh;
  const float *decay, *state;
  float *state_out;
  void *o;
  int64_t H;
  int group, Dk, Dv;
  float scale;
};

// A workgroup has a (b, h); LX lanes to a row of the state, VEC columns a lane,
// the other 256 / LX threads the next rows.  It reads the state once and writes
// it once, which is nearly all that a step moves.
template <class E, int VEC, int LX>
__global__ __launch_bounds__(256) void step_kernel(StepArgs a) {
  using T = typename E::T;
  constexpr int RY = 256 / LX;
  typedef float vec __attribute__((ext_vector_type(VEC)));
  __shared__ float part[RY][LX * VEC];
  __shared__ float sq[kMaxDim], sk[kMaxDim];
  const int64_t b = blockIdx.x / a.H, h = blockIdx.x % a.H;
  const int lx = threadIdx.x % LX, ry = threadIdx.x / LX;
  const T *q = static_cast<const T *>(a.q) + b * a.qb + h * a.qh;
  const T *k = static_cast<const T *>(a.k) + b * a.kb + (h / a.group) * a.kh;
  const T *v = static_cast<const T *>(a.v) + b * a.vb + (h / a.group) * a.vh;
  if (static_cast<int>(threadIdx.x) < a.Dk) {
    sq[threadIdx.x] = static_cast<float>(q[threadIdx.x]);
    sk[threadIdx.x] = static_cast<float>(k[threadIdx.x]);
  }
  const float d = a.decay[h];
  const int col = lx * VEC;
  const bool on = col < a.Dv;  // Dv is a multiple of VEC
  vec c, out;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    c[i] = on ? static_cast<float>(v[col + i]) : 0.0f;
    out[i] = 0.0f;
  }
  __syncthreads();
  const int64_t base = (b * a.H + h) * a.Dk * a.Dv + col;
  if (on) {
#pragma unroll 8
    for (int r = ry; r < a.Dk; r += RY) {
      vec s = *reinterpret_cast<const vec *>(a.state + base + static_cast<int64_t>(r) * a.Dv);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        s[i] = __builtin_fmaf(sk[r], c[i], d * s[i]);
        out[i] = __builtin_fmaf(sq[r], s[i], out[i]);
      }
      *reinterpret_cast<vec *>(a.state_out + base + static_cast<int64_t>(r) * a.Dv) = s;
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) part[ry][col + i] = out[i];
  __syncthreads();
  for (int j = threadIdx.x; j < a.Dv; j += 256) {
    float s = 0.0f;
    for (int y = 0; y < RY; ++y) s += part[y][j];
    static_cast<T *>(a.o)[(b * a.H + h) * a.Dv + j] = static_cast<T>(s * a.scale);
  }
}

template <class E>
void launch_step(const StepArgs &a, unsigned grid, hipStream_t s) {
  const bool vector = a.Dv % 4 == 0 && myelin::aligned(a.state, 16) && myelin::aligned(a.state_out, 16);
  if (vector) {
    if (a.Dv <= 32)
      step_kernel<E, 4, 8><<<grid, 256, 0, s>>>(a);
    else if (a.Dv <= 64)
      step_kernel<E, 4, 16><<<grid, 256, 0, s>>>(a);
    else
      step_kernel<E, 4, 32><<<grid, 256, 0, s>>>(a);
  } else {
    if (a.Dv <= 32)
      step_kernel<E, 1, 32><<<grid, 256, 0, s>>>(a);
    else
      step_kernel<E, 1, 128><<<grid, 256, 0, s>>>(a);
  }
}

template <class E>
void launch_recurrent(const Args &a, int problems, hipStream_t s) {
  int kd = 0, vd = 0;
  for (int i = 0; i < problems; ++i) {
    kd = a.p[i].KD > kd ? a.p[i].KD : kd;
    vd = a.p[i].VD > vd ? a.p[i].VD : vd;
  }
  const dim3 grid(static_cast<unsigned>(a.B * a.H), (vd + 63) / 64, problems);
  if (kd <= 64)
    recurrent<E, 64><<<grid, 64, 0, s>>>(a);
  else
    recurrent<E, 128><<<grid, 64, 0, s>>>(a);
}

int check(const char *what, int dtype, int64_t T, int64_t B, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv,
          float scale) {
  if (dtype != 0 && dtype != 2) return myelin::invalid("%s: unsupported dtype %d", what, dtype);
  if (T < 1 || B < 0 || H < 1 || Hk < 1) return myelin::invalid("%s: sizes must be positive", what);
  if (H % Hk) return myelin::invalid("%s: H must be a multiple of Hk", what);
  if (Dk < 1 || Dk > kMaxDim || Dv < 1 || Dv > kMaxDim)
    return myelin::invalid("%s: Dk and Dv must be in [1, %d]", what, kMaxDim);
  if (T > 0x7fffffff || B * H > 0x7fffffff) return myelin::invalid("%s: too many rows", what);
  if (!(scale > 0.0f) && !(scale < 0.0f)) return myelin::invalid("%s: scale must not be zero", what);
  if (scale - scale != 0.0f) return myelin::invalid("%s: scale must be finite", what);
  return MYELIN_OK;
}

// A problem's rows: t, b and h strides of a, b, c from the callers' arrays and
// a contiguous [T, B, heads, VD] result.
Problem problem(const void *a, const int64_t *as, const void *b, const int64_t *bs, const void *c, const int64_t *cs,
                void *o, int64_t B, int64_t H, int KD, int VD) {
  Problem p{};
  p.a = a, p.b = b, p.c = c, p.o = o;
  p.at = as[0], p.ab = as[1], p.ah = as[2];
  p.bt = bs[0], p.bb = bs[1], p.bh = bs[2];
  p.ct = cs[0], p.cb = cs[1], p.ch = cs[2];
  p.ot = B * H * VD, p.ob = H * VD, p.oh = VD;
  p.KD = KD, p.VD = VD;
  p.ga = p.gb = p.gc = 1;
  p.in_scale = p.out_scale = p.o_scale = 1.0f;
  return p;
}

}  // namespace

extern "C" int64_t myelin_decay_attention_workspace_elems(int64_t T, int64_t B, int64_t H, int64_t Hk, int64_t Dk,
                                                          int64_t Dv, int backward) {
  if (T < 1 || B < 1 || H < 1 || Hk < 1 || Dk < 1 || Dv < 1) return 0;
  return backward && H != Hk ? T * B * H * (Dk + Dv) : 0;
}

extern "C" int myelin_decay_attention_fwd(const void *q, const void *k, const void *v, int dtype,
                                          const int64_t *strides, const float *decay, const float *state,
                                          const int32_t *lengths, void *out, float *state_out, int64_t T, int64_t B,
                                          int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, float scale, float *workspace,
                                          int64_t workspace_elems, myelin_stream_t stream) {
  const char *what = "decay_attention_fwd";
  if (int rc = check(what, dtype, T, B, H, Hk, Dk, Dv, scale)) return rc;
  if (B == 0) return MYELIN_OK;
  if (!q || !k || !v || !strides || !decay || !out || !state_out) return myelin::invalid("%s: null pointer", what);
  Args a{};
  a.decay = decay, a.lengths = lengths, a.T = T, a.B = B, a.H = H;
  Problem &p = a.p[0];
  p = problem(q, strides, k, strides + 3, v, strides + 6, out, B, H, static_cast<int>(Dk), static_cast<int>(Dv));
  p.gb = p.gc = static_cast<int>(H / Hk);
  p.s_in = state, p.s_out = state_out, p.sk = Dv, p.sv = 1;
  p.o_scale = scale;
  if (dtype == 0)
    launch_recurrent<F32>(a, 1, myelin::as_hip(stream));
  else
    launch_recurrent<BF16>(a, 1, myelin::as_hip(stream));
  return myelin::launched(what);
}

extern "C" int myelin_decay_attention_bwd(const void *q, const void *k, const void *v, const void *grad_out, int dtype,
                                          const int64_t *strides, const float *decay, const float *state,
                                          const int32_t *lengths, const float *grad_state_out, void *grad_q,
                                          void *grad_k, void *grad_v, float *grad_state, int64_t T, int64_t B,
                                          int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, float scale, float *workspace,
                                          int64_t workspace_elems, myelin_stream_t stream) {
  const char *what = "decay_attention_bwd";
  if (int rc = check(what, dtype, T, B, H, Hk, Dk, Dv, scale)) return rc;
  if (B == 0) return MYELIN_OK;
  if (!q || !k || !v || !grad_out || !strides || !decay || !grad_q || !grad_k || !grad_v)
    return myelin::invalid("%s: null pointer", what);
  const int64_t need = myelin_decay_attention_workspace_elems(T, B, H, Hk, Dk, Dv, 1);
  if (need && (!workspace || workspace_elems < need))
    return myelin::invalid("%s: workspace of %lld floats needed", what, static_cast<long long>(need));
  const int group = static_cast<int>(H / Hk), dk = static_cast<int>(Dk), dv = static_cast<int>(Dv);
  const int64_t *qs = strides, *ks = strides + 3, *vs = strides + 6, *gs = strides + 9;
  Args a{};
  a.decay = decay, a.lengths = lengths, a.T = T, a.B = B, a.H = H;
  // dq = scale LA(do, v, k), from S_0 transposed
  Problem &pq = a.p[0], &pk = a.p[1], &pv = a.p[2];
  pq = problem(grad_out, gs, v, vs, k, ks, grad_q, B, H, dv, dk);
  pq.gb = pq.gc = group;
  pq.s_in = state, pq.sk = 1, pq.sv = Dv;
  // dk = RLA(v, do, scale q), dv = RLA(k, scale q, do), both from dS_T: with
  // the scale taken out of the whole, its share of dS_T is divided by it
  void *to_k = group > 1 ? static_cast<void *>(workspace) : grad_k;
  void *to_v = group > 1 ? static_cast<void *>(workspace + T * B * H * Dk) : grad_v;
  pk = problem(v, vs, grad_out, gs, q, qs, to_k, B, H, dv, dk);
  pk.ga = group;
  pk.s_in = grad_state_out, pk.sk = 1, pk.sv = Dv;
  pv = problem(k, ks, q, qs, grad_out, gs, to_v, B, H, dk, dv);
  pv.ga = group;
  pv.s_in = grad_state_out, pv.s_out = grad_state, pv.sk = Dv, pv.sv = 1;
  pq.o_scale = pk.o_scale = pv.o_scale = scale;
  pk.in_scale = pv.in_scale = 1.0f / scale;
  pv.out_scale = scale;
  pk.reverse = pv.reverse = 1;
  pk.o_f32 = pv.o_f32 = group > 1;
  const hipStream_t s = myelin::as_hip(stream);
  if (dtype == 0)
    launch_recurrent<F32>(a, 3, s);
  else
    launch_recurrent<BF16>(a, 3, s);
  if (group > 1) {
    for (int i = 0; i < 2; ++i) {
      const int D = i ? dv : dk;
      const int64_t n = T * B * Hk * D;
      const unsigned grid = static_cast<unsigned>((n + 255) / 256);
      const float *from = static_cast<const float *>(i ? to_v : to_k);
      void *to = i ? grad_v : grad_k;
      if (dtype == 0)
        sum_groups<F32><<<grid, 256, 0, s>>>(from, to, n, group, D);
      else
        sum_groups<BF16><<<grid, 256, 0, s>>>(from, to, n, group, D);
    }
  }
  return myelin::launched(what);
}

extern "C" int myelin_decay_attention_step(const void *q, const void *k, const void *v, int dtype,
                                           const int64_t *strides, const float *decay, const float *state, void *out,
                                           float *state_out, int64_t B, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv,
                                           float scale, myelin_stream_t stream) {
  const char *what = "decay_attention_step";
  if (int rc = check(what, dtype, 1, B, H, Hk, Dk, Dv, scale)) return rc;
  if (B == 0) return MYELIN_OK;
  if (!q || !k || !v || !strides || !decay || !state || !out || !state_out)
    return myelin::invalid("%s: null pointer", what);
  const StepArgs a{q, k, v, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], decay, state,
                   state_out, out, H, static_cast<int>(H / Hk), static_cast<int>(Dk), static_cast<int>(Dv), scale};
  const unsigned grid = static_cast<unsigned>(B * H);
  if (dtype == 0)
    launch_step<F32>(a, grid, myelin::as_hip(stream));
  else
    launch_step<BF16>(a, grid, myelin::as_hip(stream));
  return myelin::launched(what);
}
