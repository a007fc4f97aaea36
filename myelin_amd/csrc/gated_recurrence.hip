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
// before every 8th step, in fp32, and the steps from there again: half a byte, for
// bytes an element, where the output's bf16 would cost h_{t-1} - x_t its accuracy.

#include "elements.h"

namespace {

using myelin::BF16;
using myelin::F32;

constexpr int kSteps = 16;     // steps of a wave at a time
constexpr int kBackSteps = 8;  // and in the backward pass; and steps between two kept states
constexpr int kMaxWaves = 16;

struct Affine;

struct Args {
  const void *x, *gate, *g_out;
  int64_t xt, xb, gt, gb, ot, ob;  // element strides of time and batch
  const int32_t *lengths;
  const float *state;  // [B, N] or null: of the first step; backward: gradient of the last
  void *out, *gx, *gg;
  float *state_out;  // [B, N] or null: the last; backward: gradient of the first
  float *kept;       // [ceil(T / kBackSteps), B, N] or null
  int64_t T, B, N;
  int64_t blocks, segments, seg_steps, seg;  // seg: a workgroup's own
  Affine *joins;                             // [segments, B, N]
};

// sigmoid and 1 - sigmoid, each to its own accuracy
struct Gate {
  float a, b;
  __device__ explicit Gate(float g) {
    const float e = myelin::exp_f32(-__builtin_fabsf(g));
    const float r = myelin::recip_rn(1.0f + e), s = e * r;
    a = g >= 0.0f ? r : s;
    b = g >= 0.0f ? s : r;
  }
};

constexpr float kInf = __builtin_huge_valf();

// A workgroup has 64 channels, a lane each, and walks over time in tiles: each of
// its waves takes the next kSteps steps, into registers.  A run of steps maps the
// state before it to the one after it as h -> A h + H; the waves exchange A and H
// in LDS, join those before them to their own first state and only then run their
// steps again.  x and gate are read once.
struct Affine {
  float A, H;
};

// A lane's channel.  Rows are addressed from bases that the workgroup shares, with
// 32-bit byte offsets of the lanes: a load takes no address registers of its own.
struct Place {
  int64_t first;  // the workgroup's first channel, of B * N
  int lane, wave, waves;
  bool in;
  int64_t live;                   // its steps
  const char *x, *gate, *out;     // of the first channel's batch row
  uint32_t at_x, at_gate, at_out;  // bytes from there
  __device__ int64_t c() const { return first + lane; }
};

template <class T>
__device__ __forceinline__ Place place_of(const Args &a, int64_t block) {
  Place p;
  p.lane = threadIdx.x & (myelin::kWave - 1);
  p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x / myelin::kWave);
  p.waves = blockDim.x / myelin::kWave;
  p.first = block * myelin::kWave;
  p.in = p.c() < a.B * a.N;
  const int64_t b0 = p.first / a.N, b = (p.in ? p.c() : p.first) / a.N, n = (p.in ? p.c() : p.first) - b * a.N;
  p.x = reinterpret_cast<const char *>(static_cast<const T *>(a.x) + b0 * a.xb);
  p.gate = reinterpret_cast<const char *>(static_cast<const T *>(a.gate) + b0 * a.gb);
  p.out = reinterpret_cast<const char *>(static_cast<const T *>(a.g_out) + b0 * a.ob);
  p.at_x = static_cast<uint32_t>(((b - b0) * a.xb + n) * sizeof(T));
  p.at_gate = static_cast<uint32_t>(((b - b0) * a.gb + n) * sizeof(T));
  p.at_out = static_cast<uint32_t>(((b - b0) * a.ob + n) * sizeof(T));
  int64_t live = a.T;
  if (a.lengths) {
    live = a.lengths[b];
    live = live < 0 ? 0 : live < a.T ? live : a.T;
  }
  p.live = p.in ? live : 0;
  return p;
}

// STEPS values from step t0 on.  Rows past the last are the last; what a lane has
// no step for is masked below.
template <int STEPS, class T>
__device__ __forceinline__ void load(T *v, const char *from, uint32_t at, int64_t stride, int64_t t0, int64_t steps) {
  const char *p = from + t0 * stride * static_cast<int64_t>(sizeof(T));
  const int64_t row = stride * static_cast<int64_t>(sizeof(T));
  if (t0 + STEPS <= steps) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) v[i] = *reinterpret_cast<const T *>(p + i * row + at);
  } else {
    const int last = static_cast<int>(steps - 1 - t0);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) v[i] = *reinterpret_cast<const T *>(p + (i < last ? i : last) * row + at);
  }
}

template <int STEPS, class T>
__device__ __forceinline__ void mask(T *v, int n, T past) {
#pragma unroll
  for (int i = 0; i < STEPS; ++i) v[i] = i < n ? v[i] : past;
}

template <int STEPS>
__device__ __forceinline__ int steps_from(const Place &p, int64_t t0) {
  const int64_t n = p.live - t0;
  return n < 0 ? 0 : n < STEPS ? static_cast<int>(n) : STEPS;
}

// The state before segment `seg` of a sequence, from the one before the first.
__device__ __forceinline__ float join_before(const Args &a, const Place &p, float s) {
  for (int64_t o = 0; o < a.seg; ++o) {
    const Affine m = a.joins[o * a.B * a.N + p.c()];
    s = __builtin_fmaf(m.A, s, m.H);
  }
  return s;
}
__device__ __forceinline__ float join_after(const Args &a, const Place &p, float s) {
  for (int64_t o = a.segments - 1; o > a.seg; --o) {
    const Affine m = a.joins[o * a.B * a.N + p.c()];
    s = __builtin_fmaf(m.A, s, m.H);
  }
  return s;
}

// A block's channels and segment.
__device__ __forceinline__ int64_t locate(Args &a) {
  const int64_t block = myelin::block_id();
  a.seg = block / a.blocks;
  return block - a.seg * a.blocks;
}

template <class E>
__global__ __launch_bounds__(kMaxWaves * myelin::kWave) void forward(Args a) {
  using T = typename E::T;
  __shared__ Affine maps[2][kMaxWaves][myelin::kWave];
  const int64_t block = locate(a);
  if (a.seg >= a.segments) return;  // the whole workgroup
  const Place p = place_of<T>(a, block);
  const int lane = p.lane, wave = p.wave, waves = p.waves;
  const int64_t BN = a.B * a.N, first = a.seg * a.seg_steps;
  const int64_t end = first + a.seg_steps < a.T ? first + a.seg_steps : a.T;
  float s = p.in && a.state ? a.state[p.c()] : 0.0f;
  if (p.in) s = join_before(a, p, s);
  T x[kSteps], gate[kSteps];
  int64_t t0 = first + wave * kSteps;
  int n = steps_from<kSteps>(p, t0);
  const auto fetch = [&]() {
    if (!__any(n > 0)) return;
    load<kSteps>(x, p.x, p.at_x, a.xt, t0, a.T);
    load<kSteps>(gate, p.gate, p.at_gate, a.gt, t0, a.T);
  };
  fetch();
  for (int64_t tile = first, turn = 0; tile < end; tile += waves * kSteps, ++turn) {
    const bool all = __all(n == kSteps);
    if (!all) {
      mask<kSteps>(x, n, E::put(0.0f));
      mask<kSteps>(gate, n, E::put(kInf));
    }
    float ra[kSteps], ru[kSteps];
    Affine m{1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const Gate g(E::get(gate[i]));
      ra[i] = g.a;
      ru[i] = g.b * E::get(x[i]);
      m = {m.A * g.a, __builtin_fmaf(g.a, m.H, ru[i])};
    }
    maps[turn & 1][wave][lane] = m;
    const int64_t here = t0;
    const int mine = n;
    t0 += waves * kSteps;
    if (tile + waves * kSteps < end) {
      n = steps_from<kSteps>(p, t0);
      fetch();
    }
    __syncthreads();
    float h = s;
#pragma unroll 4
    for (int o = 0; o < waves; ++o) {
      if (o == wave) h = s;
      const Affine q = maps[turn & 1][o][lane];
      s = __builtin_fmaf(q.A, s, q.H);
    }
    float *kept = a.kept && p.in ? a.kept + here / kBackSteps * BN + p.first : nullptr;
    T *out = static_cast<T *>(a.out) + here * BN + p.first;
    if (all) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (kept && i % kBackSteps == 0) (kept + i / kBackSteps * BN)[lane] = h;
        h = __builtin_fmaf(ra[i], h, ru[i]);
        (out + i * BN)[lane] = E::put(h);
      }
    } else if (p.in) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (kept && i % kBackSteps == 0 && here + i < end) (kept + i / kBackSteps * BN)[lane] = h;
        h = __builtin_fmaf(ra[i], h, ru[i]);
        if (here + i < end) (out + i * BN)[lane] = E::put(i < mine ? h : 0.0f);
      }
    }
  }
  if (p.in && wave == 0 && a.seg == a.segments - 1) a.state_out[p.c()] = s;
}

template <class E>
__global__ __launch_bounds__(kMaxWaves * myelin::kWave) void backward(Args a) {
  using T = typename E::T;
  __shared__ Affine maps[2][kMaxWaves][myelin::kWave];
  const int64_t block = locate(a);
  if (a.seg >= a.segments) return;  // the whole workgroup
  const Place p = place_of<T>(a, block);
  const int lane = p.lane, wave = p.wave, waves = p.waves;
  const int64_t BN = a.B * a.N, first = a.seg * a.seg_steps, tile_steps = waves * kBackSteps;
  const int64_t end = first + a.seg_steps < a.T ? first + a.seg_steps : a.T;
  float s = p.in && a.state ? a.state[p.c()] : 0.0f;
  if (p.in) s = join_after(a, p, s);
  T x[kBackSteps], gate[kBackSteps], go[kBackSteps];
  float start = 0.0f;
  int64_t tile = first + (end - first - 1) / tile_steps * tile_steps;
  int64_t t0 = tile + wave * kBackSteps;
  int n = steps_from<kBackSteps>(p, t0);
  const auto fetch = [&]() {
    start = 0.0f;
    if (!__any(n > 0)) return;
    load<kBackSteps>(x, p.x, p.at_x, a.xt, t0, a.T);
    load<kBackSteps>(gate, p.gate, p.at_gate, a.gt, t0, a.T);
    if (a.g_out) load<kBackSteps>(go, p.out, p.at_out, a.ot, t0, a.T);
    if (p.in) start = (a.kept + t0 / kBackSteps * BN + p.first)[lane];
  };
  fetch();
  for (int64_t turn = 0; tile >= first; tile -= tile_steps, ++turn) {
    const bool all = __all(n == kBackSteps);
    if (!all) {
      mask<kBackSteps>(x, n, E::put(0.0f));
      mask<kBackSteps>(gate, n, E::put(kInf));
    }
    if (!all || !a.g_out) mask<kBackSteps>(go, a.g_out ? n : 0, E::put(0.0f));
    float ra[kBackSteps], rb[kBackSteps], rd[kBackSteps], rg[kBackSteps];
    Affine m{1.0f, 0.0f};
    float h = start;
#pragma unroll
    for (int i = 0; i < kBackSteps; ++i) {
      const Gate g(E::get(gate[i]));
      ra[i] = g.a;
      rb[i] = g.b;
      const float v = E::get(x[i]);
      rd[i] = h - v;
      h = __builtin_fmaf(g.a, h, g.b * v);
      rg[i] = E::get(go[i]);
    }
#pragma unroll
    for (int i = kBackSteps - 1; i >= 0; --i) m = {m.A * ra[i], ra[i] * (rg[i] + m.H)};
    maps[turn & 1][wave][lane] = m;
    const int64_t here = t0;
    const int mine = n;
    t0 -= tile_steps;
    if (tile > first) {
      n = steps_from<kBackSteps>(p, t0);
      fetch();
    }
    __syncthreads();
    float c = s;
#pragma unroll 4
    for (int o = waves - 1; o >= 0; --o) {
      if (o == wave) c = s;
      const Affine q = maps[turn & 1][o][lane];
      s = __builtin_fmaf(q.A, s, q.H);
    }
    T *gx = static_cast<T *>(a.gx) + here * BN + p.first, *gg = static_cast<T *>(a.gg) + here * BN + p.first;
#pragma unroll
    for (int i = kBackSteps - 1; i >= 0; --i) {
      const float g = rg[i] + c, dx = rb[i] * g, dg = dx * rd[i] * ra[i];
      c = ra[i] * g;
      if (all) {
        if (a.gx) (gx + i * BN)[lane] = E::put(dx);
        if (a.gg) (gg + i * BN)[lane] = E::put(dg);
      } else if (p.in && here + i < end) {
        if (a.gx) (gx + i * BN)[lane] = E::put(i < mine ? dx : 0.0f);
        if (a.gg) (gg + i * BN)[lane] = E::put(i < mine ? dg : 0.0f);
      }
    }
  }
  if (p.in && wave == 0 && a.seg == 0 && a.state_out) a.state_out[p.c()] = s;
}

// What a segment does to the state before it (BACK: to the gradient of the state
// after it): each wave runs over a stretch of its own, then they are joined.
template <class E, bool BACK>
__global__ __launch_bounds__(kMaxWaves * myelin::kWave) void summarise(Args a) {
  using T = typename E::T;
  __shared__ Affine maps[kMaxWaves][myelin::kWave];
  const int64_t block = locate(a);
  if (BACK) ++a.seg;  // the first needs none, as the last forward
  if (a.seg >= a.segments - !BACK) return;
  const Place p = place_of<T>(a, block);
  const int lane = p.lane, wave = p.wave, waves = p.waves;
  const int64_t first = a.seg * a.seg_steps;
  const int64_t end = first + a.seg_steps < a.T ? first + a.seg_steps : a.T;
  // (whole chunks: a segment is a multiple of waves * kSteps steps)
  const int64_t each = a.seg_steps / waves, from = first + wave * each;
  const int64_t to = from + each < end ? from + each : end;
  Affine m{1.0f, 0.0f};
  const int chunks = to > from ? static_cast<int>((to - from + kSteps - 1) / kSteps) : 0;
  for (int k = 0; k < chunks; ++k) {
    const int64_t t0 = from + (BACK ? chunks - 1 - k : k) * kSteps;
    const int n = steps_from<kSteps>(p, t0);
    if (!__any(n > 0)) continue;
    T v[kSteps], gate[kSteps];
    load<kSteps>(gate, p.gate, p.at_gate, a.gt, t0, a.T);
    if (!BACK)
      load<kSteps>(v, p.x, p.at_x, a.xt, t0, a.T);
    else if (a.g_out)
      load<kSteps>(v, p.out, p.at_out, a.ot, t0, a.T);
    if (!__all(n == kSteps)) mask<kSteps>(gate, n, E::put(kInf));
    if (!__all(n == kSteps) || (BACK && !a.g_out)) mask<kSteps>(v, BACK && !a.g_out ? 0 : n, E::put(0.0f));
#pragma unroll
    for (int o = 0; o < kSteps; ++o) {
      const int i = BACK ? kSteps - 1 - o : o;
      const Gate g(E::get(gate[i]));
      if (BACK)
        m = {m.A * g.a, g.a * (E::get(v[i]) + m.H)};
      else
        m = {m.A * g.a, __builtin_fmaf(g.a, m.H, g.b * E::get(v[i]))};
    }
  }
  maps[wave][lane] = m;
  __syncthreads();
  if (wave == 0 && p.in) {
    m = {1.0f, 0.0f};
    for (int o = 0; o < waves; ++o) {
      const Affine q = maps[BACK ? waves - 1 - o : o][lane];
      m = {m.A * q.A, __builtin_fmaf(q.A, m.H, q.H)};
    }
    a.joins[a.seg * a.B * a.N + p.c()] = m;
  }
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

// A workgroup's lanes reach over this many batch rows; their offsets have 32 bits.
bool reachable(int64_t stride, int64_t B, int64_t N) {
  return B == 1 || (stride < int64_t{1} << 30 && (64 / N + 1) * stride + N < int64_t{1} << 30);
}

int check(const char *what, int dtype, int64_t T, int64_t B, int64_t N) {
  if (dtype != 0 && dtype != 2) return myelin::invalid("%s: unsupported dtype %d", what, dtype);
  if (T < 1 || B < 0 || N < 0) return myelin::invalid("%s: T must be positive, B and N not negative", what);
  if (T >= int64_t{1} << 31 || B >= int64_t{1} << 31 || N >= int64_t{1} << 29 || B * N >= int64_t{1} << 36)
    return myelin::invalid("%s: too many steps or channels", what);
  return MYELIN_OK;
}

struct Plan {
  int64_t blocks, segments, seg_steps;
  int waves;
};

// Time is split where the channels leave CUs without a workgroup.
Plan plan_of(int64_t T, int64_t B, int64_t N, bool back) {
  Plan p;
  p.blocks = (B * N + myelin::kWave - 1) / myelin::kWave;
  // (segments are whole chunks of kSteps to each wave for summarise)
  const int64_t chunks = (T + kSteps - 1) / kSteps;
  p.waves = static_cast<int>(chunks < kMaxWaves ? chunks : kMaxWaves);
  const int64_t tile = p.waves * kSteps, tiles = (T + tile - 1) / tile;
  (void)back;
  int64_t n = p.blocks >= 128 ? 1 : 256 / p.blocks;
  if (n > tiles) n = tiles;
  const int64_t each = (tiles + n - 1) / n;
  p.seg_steps = each * tile;
  p.segments = (tiles + each - 1) / each;
  return p;
}

// Workgroups of up to 1024 threads, fewer than 2^32 in x.
dim3 grid_for(int64_t blocks) {
  const int64_t x = int64_t{1} << 21, y = (blocks + x - 1) / x;
  return dim3(static_cast<unsigned>(y > 1 ? x : blocks), static_cast<unsigned>(y));
}

int64_t workspace_of(int64_t T, int64_t B, int64_t N, bool back) {
  const Plan p = plan_of(T, B, N, back);
  return p.segments == 1 ? 0 : 2 * p.segments * B * N;
}

int prepare(const char *what, Args &a, Plan &p, float *workspace, int64_t elems, bool back) {
  p = plan_of(a.T, a.B, a.N, back);
  const int64_t need = workspace_of(a.T, a.B, a.N, back);
  if (need) {
    if (!workspace || elems < need)
      return myelin::invalid("%s: workspace of %lld floats needed", what, static_cast<long long>(need));
    if (!myelin::aligned(workspace, 16)) return myelin::invalid("%s: workspace must be 16-byte aligned", what);
  }
  a.blocks = p.blocks;
  a.segments = p.segments;
  a.seg_steps = p.seg_steps;
  a.joins = reinterpret_cast<Affine *>(workspace);
  return MYELIN_OK;
}

template <class E, bool BACK>
void launch(const Args &a, const Plan &p, hipStream_t s) {
  const int threads = p.waves * myelin::kWave;
  if (p.segments > 1) summarise<E, BACK><<<grid_for(p.blocks * (p.segments - 1)), threads, 0, s>>>(a);
  if (BACK)
    backward<E><<<grid_for(p.blocks * p.segments), threads, 0, s>>>(a);
  else
    forward<E><<<grid_for(p.blocks * p.segments), threads, 0, s>>>(a);
}

}  // namespace

extern "C" int64_t myelin_gated_recurrence_kept_elems(int64_t T, int64_t B, int64_t N) {
  return (T + kBackSteps - 1) / kBackSteps * B * N;
}

extern "C" int64_t myelin_gated_recurrence_workspace_elems(int dtype, int64_t T, int64_t B, int64_t N, int backward) {
  (void)dtype;
  return T < 1 || B < 1 || N < 1 ? 0 : workspace_of(T, B, N, backward);
}

extern "C" int myelin_gated_recurrence_fwd(const void *x, const void *gate, int dtype, const int64_t *strides,
                                           const float *state, const int32_t *lengths, void *out, float *state_out,
                                           float *kept, int64_t T, int64_t B, int64_t N, float *workspace,
                                           int64_t workspace_elems, myelin_stream_t stream) {
  const char *what = "gated_recurrence_fwd";
  if (int rc = check(what, dtype, T, B, N)) return rc;
  if (B == 0 || N == 0) return MYELIN_OK;
  if (!x || !gate || !strides || !out || !state_out) return myelin::invalid("%s: null pointer", what);
  for (int o = 1; o < 4; o += 2)
    if (!reachable(strides[o], B, N)) return myelin::invalid("%s: batch stride too large", what);
  Args a{};
  a.T = T, a.B = B, a.N = N;
  Plan p;
  if (int rc = prepare(what, a, p, workspace, workspace_elems, false)) return rc;
  a.x = x, a.gate = gate, a.lengths = lengths, a.state = state;
  a.xt = strides[0], a.xb = strides[1], a.gt = strides[2], a.gb = strides[3];
  a.out = out, a.state_out = state_out, a.kept = kept;
  if (dtype == 0)
    launch<F32, false>(a, p, myelin::as_hip(stream));
  else
    launch<BF16, false>(a, p, myelin::as_hip(stream));
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
  for (int o = 1; o < (grad_out ? 6 : 4); o += 2)
    if (!reachable(strides[o], B, N)) return myelin::invalid("%s: batch stride too large", what);
  Args a{};
  a.T = T, a.B = B, a.N = N;
  Plan p;
  if (int rc = prepare(what, a, p, workspace, workspace_elems, true)) return rc;
  a.x = x, a.gate = gate, a.g_out = grad_out, a.lengths = lengths, a.state = grad_state_out;
  a.xt = strides[0], a.xb = strides[1], a.gt = strides[2], a.gb = strides[3], a.ot = strides[4], a.ob = strides[5];
  a.gx = grad_x, a.gg = grad_gate, a.state_out = grad_state, a.kept = const_cast<float *>(kept);
  if (dtype == 0)
    launch<F32, true>(a, p, myelin::as_hip(stream));
  else
    launch<BF16, true>(a, p, myelin::as_hip(stream));
  return myelin::launched(what);
}

extern "C" int myelin_gated_recurrence_step(const void *x, const void *gate, int dtype, const int64_t *strides,
                                            const float *state, void *out, float *state_out, int64_t B, int64_t N,
                                            myelin_stream_t stream) {
  const char *what = "gated_recurrence_step";
  if (int rc = check(what, dtype, 1, B, N)) return rc;
  if (B == 0 || N == 0) return MYELIN_OK;
  if (!x || !gate || !strides || !state || !out || !state_out) return myelin::invalid("%s: null pointer", what);
  Args a{};
  a.x = x, a.gate = gate, a.xb = strides[0], a.gb = strides[1], a.state = state, a.out = out, a.state_out = state_out;
  a.B = B, a.N = N;
  const dim3 grid = myelin::grid_of((B * N + 255) / 256);
  if (dtype == 0)
    step<F32><<<grid, 256, 0, myelin::as_hip(stream)>>>(a);
  else
    step<BF16><<<grid, 256, 0, myelin::as_hip(stream)>>>(a);
  return myelin::launched(what);
}
