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
constexpr int kApart = 4;      // waves of a workgroup whose waves have channels of their own
constexpr int kWave = myelin::kWave;

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

// sigmoid and 1 - sigmoid, each to its own accuracy: the smaller of the two from the
// exponential, the larger as what it leaves of 1 (a time constant of 1000 steps adds
// up a thousand of its roundings; a reciprocal's would be twice as large).  fp32 puts
// the rounding of the exponential's argument back, |g| 2^-24 of the smaller.  A bf16
// gate is itself only known to |g| 2^-9.
template <class E>
struct Gate {
  float a, b;
  __device__ explicit Gate(float g) {
    const float d = -__builtin_fabsf(g);
    const float e = sizeof(typename E::T) == 4 ? myelin::exp_f32(d) : __builtin_amdgcn_exp2f(d * myelin::kLog2e);
    const float s = e * __builtin_amdgcn_rcpf(1.0f + e), r = 1.0f - s;
    a = g >= 0.0f ? r : s;
    b = g >= 0.0f ? s : r;
  }
};

constexpr float kInf = __builtin_huge_valf();

// A run of steps maps the state before it to the one after it as h -> A h + H.
struct Affine {
  float A, H;
};

// A workgroup has 64 channels, a lane each, and walks over time in tiles: each of its
// waves takes the next STEPS steps, into registers; the waves exchange A and H of
// their steps in LDS, join those before them to their own first state and only then
// run their steps again.  x and gate are read once.  (Two groups of 32 channels to a
// wave, for twice the workgroups, read rows in pieces of 64 bytes: [2048, 8, 2048]
// bf16 48 -> 62 us forward, 88 -> 105 us backward.)
//
// Rows are addressed from bases that the wave shares, with 32-bit byte offsets of
// the lanes: a load takes no address registers of its own.
template <int STEPS>
struct Place {
  int64_t first;  // the workgroup's first channel, of B * N
  int lane, wave, waves;
  int base = 0;                    // the first wave's
  int64_t live;                    // the channel's steps
  bool in;
  const char *x, *gate, *out;      // of the first channel's batch row
  uint32_t at_x, at_gate, at_out;  // bytes from there
  __device__ int64_t c() const { return first + lane; }
  __device__ int64_t tile_steps() const { return waves * STEPS; }
  // the wave's first step of a tile, and how many the lane has from there
  __device__ int64_t step(int64_t tile) const { return tile + wave * STEPS; }
  __device__ int steps(int64_t tile) const {
    const int64_t n = live - step(tile);
    return n < 0 ? 0 : n < STEPS ? static_cast<int>(n) : STEPS;
  }

  template <class T, bool APART>
  __device__ void set(const Args &a, int64_t block) {
    lane = threadIdx.x % kWave;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    // (one where they are apart; known to the compiler, it takes more addresses into
    // scalar registers than there are)
    waves = blockDim.x / (APART ? kApart * kWave : kWave);
    if (APART) {
      block = block * kApart + wave;
      base = wave;
      wave = 0;
    }
    // (behind the last block: the last one, with nothing to do)
    first = (!APART || block < a.blocks ? block : a.blocks - 1) * kWave;
    in = (!APART || block < a.blocks) && c() < a.B * a.N;
    const int64_t mine = in ? c() : first;
    const int64_t b0 = first / a.N, b = mine / a.N, n = mine - b * a.N;
    x = reinterpret_cast<const char *>(static_cast<const T *>(a.x) + b0 * a.xb);
    gate = reinterpret_cast<const char *>(static_cast<const T *>(a.gate) + b0 * a.gb);
    out = reinterpret_cast<const char *>(static_cast<const T *>(a.g_out) + b0 * a.ob);
    at_x = static_cast<uint32_t>(((b - b0) * a.xb + n) * sizeof(T));
    at_gate = static_cast<uint32_t>(((b - b0) * a.gb + n) * sizeof(T));
    at_out = static_cast<uint32_t>(((b - b0) * a.ob + n) * sizeof(T));
    live = a.T;
    if (a.lengths) {
      live = a.lengths[b];
      live = live < 0 ? 0 : live < a.T ? live : a.T;
    }
    if (!in) live = 0;
  }

  // The lane's STEPS values of a tile.  Rows past the last are the last; what a lane
  // has no step for is masked afterwards (loads under conditions wait for each other).
  template <class T>
  __device__ void load(T *v, const char *from, uint32_t at, int64_t stride, int64_t tile, int64_t steps) const {
    const int64_t t0 = step(tile), row = stride * static_cast<int64_t>(sizeof(T));
    const char *p = from + t0 * row;
    if (t0 + STEPS <= steps) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) v[i] = *reinterpret_cast<const T *>(p + i * row + at);
    } else {
      const int last = static_cast<int>(steps - 1 - t0);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) v[i] = *reinterpret_cast<const T *>(p + (i < last ? i : last) * row + at);
    }
  }
};

template <int STEPS, class T>
__device__ __forceinline__ void mask(T *v, int n, T past) {
#pragma unroll
  for (int i = 0; i < STEPS; ++i) v[i] = i < n ? v[i] : past;
}

// The state in front of a channel's segments joined in order, `step` apart from the
// first of them: eight at a time, so that their loads do not wait for each other.
__device__ __forceinline__ float join(const Args &a, int64_t c, float s, int64_t from, int64_t count, int64_t step) {
  const int64_t BN = a.B * a.N;
  const Affine *m = a.joins + from * BN + c;
  int64_t o = 0;
  for (; o + 8 <= count; o += 8) {
    Affine q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = m[(o + i) * step * BN];
#pragma unroll
    for (int i = 0; i < 8; ++i) s = __builtin_fmaf(q[i].A, s, q[i].H);
  }
  for (; o < count; ++o) {
    const Affine q = m[o * step * BN];
    s = __builtin_fmaf(q.A, s, q.H);
  }
  return s;
}

// A workgroup's segment and block of channels, or -1.  Consecutive workgroups run on
// XCDs in turn; each XCD takes a stretch of the (segment, channels), so that blocks
// that share lines of 128 bytes share an L2.
template <bool APART>
__device__ __forceinline__ int64_t locate(Args &a, int64_t segments) {
  constexpr int kXcds = 8;
  const int64_t blocks = APART ? (a.blocks + kApart - 1) / kApart : a.blocks, units = blocks * segments;
  const int64_t id = myelin::block_id(), each = (units + kXcds - 1) / kXcds;
  const int64_t unit = id % kXcds * each + id / kXcds;
  if (id >= each * kXcds || unit >= units) return -1;
  a.seg = unit / blocks;
  return unit - a.seg * blocks;
}

// Bound by memory, with the gates' instructions half of the time beside it: [2048, 8,
// 2048] bf16 48 us with the kept states (218 MB, 4.5 TB/s), 256 workgroups of 16
// waves, one to a CU.  The next tile's rows are on their way while the waves join.
template <class E, bool APART>
__global__ __launch_bounds__(kMaxWaves * kWave) void forward(Args a) {
  using T = typename E::T;
  using P = Place<kSteps>;
  __shared__ Affine maps[2][kMaxWaves][kWave];
  const int64_t block = locate<APART>(a, a.segments);
  if (block < 0) return;  // the whole workgroup
  P p;
  p.template set<T, APART>(a, block);
  const int64_t BN = a.B * a.N, first = a.seg * a.seg_steps;
  const int64_t end = first + a.seg_steps < a.T ? first + a.seg_steps : a.T;
  float s = p.in && a.state ? a.state[p.c()] : 0.0f;
  if (p.in) s = join(a, p.c(), s, 0, a.seg, 1);
  T x[kSteps], gate[kSteps];
  int n = 0;
  const auto fetch = [&](int64_t tile) {
    n = p.steps(tile);
    if (!__any(n > 0)) return;
    p.load(x, p.x, p.at_x, a.xt, tile, a.T);
    p.load(gate, p.gate, p.at_gate, a.gt, tile, a.T);
  };
  fetch(first);
  for (int64_t tile = first, turn = 0; tile < end; tile += p.tile_steps(), ++turn) {
    const bool all = __all(n == kSteps);
    if (!all) {
      mask<kSteps>(x, n, E::put(0.0f));
      mask<kSteps>(gate, n, E::put(kInf));
    }
    float ra[kSteps], ru[kSteps];
    Affine m{1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const Gate<E> g(E::get(gate[i]));
      ra[i] = g.a;
      ru[i] = g.b * E::get(x[i]);
      m = {m.A * g.a, __builtin_fmaf(g.a, m.H, ru[i])};
    }
    Affine(*const map)[kWave] = &maps[turn & 1][p.base];
    map[p.wave][p.lane] = m;
    const int mine = n;
    if (tile + p.tile_steps() < end) fetch(tile + p.tile_steps());
    if (!APART) __syncthreads();
    float h = s;
#pragma unroll 4
    for (int o = 0; o < p.waves; ++o) {
      if (o == p.wave) h = s;
      const Affine q = map[o][p.lane];
      s = __builtin_fmaf(q.A, s, q.H);
    }
    const int64_t here = p.step(tile);
    const int left = p.in ? static_cast<int>(end - p.step(tile) < kSteps ? end - p.step(tile) : kSteps) : 0;
    T *out = static_cast<T *>(a.out) + here * BN + p.first;
    float *kept = a.kept ? a.kept + here / kBackSteps * BN + p.first : nullptr;
    if (all) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (kept && i % kBackSteps == 0) (kept + i / kBackSteps * BN)[p.lane] = h;
        h = __builtin_fmaf(ra[i], h, ru[i]);
        (out + i * BN)[p.lane] = E::put(h);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (kept && i % kBackSteps == 0 && i < left) (kept + i / kBackSteps * BN)[p.lane] = h;
        h = __builtin_fmaf(ra[i], h, ru[i]);
        if (i < left) (out + i * BN)[p.lane] = E::put(i < mine ? h : 0.0f);
      }
    }
  }
  if (p.in && p.wave == 0 && a.seg == a.segments - 1) a.state_out[p.c()] = s;
}

// As forward, from the last tile, with three rows in and two out: 84 us (352 MB, 4.2
// TB/s) for the same.  8 steps of a wave: 16 do not fit 128 registers, and 16 waves of
// them are a CU's.
template <class E, bool APART>
__global__ __launch_bounds__(kMaxWaves * kWave) void backward(Args a) {
  using T = typename E::T;
  using P = Place<kBackSteps>;
  __shared__ Affine maps[2][kMaxWaves][kWave];
  const int64_t block = locate<APART>(a, a.segments);
  if (block < 0) return;  // the whole workgroup
  P p;
  p.template set<T, APART>(a, block);
  const int64_t BN = a.B * a.N, first = a.seg * a.seg_steps;
  const int64_t end = first + a.seg_steps < a.T ? first + a.seg_steps : a.T;
  float s = p.in && a.state ? a.state[p.c()] : 0.0f;
  if (p.in) s = join(a, p.c(), s, a.segments - 1, a.segments - 1 - a.seg, -1);
  T x[kBackSteps], gate[kBackSteps], go[kBackSteps];
  float start = 0.0f;
  int n = 0;
  const auto fetch = [&](int64_t tile) {
    n = p.steps(tile);
    start = 0.0f;
    if (!__any(n > 0)) return;
    p.load(x, p.x, p.at_x, a.xt, tile, a.T);
    p.load(gate, p.gate, p.at_gate, a.gt, tile, a.T);
    if (a.g_out) p.load(go, p.out, p.at_out, a.ot, tile, a.T);
    if (n > 0) start = (a.kept + p.step(tile) / kBackSteps * BN + p.first)[p.lane];
  };
  int64_t tile = first + (end - first - 1) / p.tile_steps() * p.tile_steps();
  fetch(tile);
  for (int64_t turn = 0; tile >= first; tile -= p.tile_steps(), ++turn) {
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
      const Gate<E> g(E::get(gate[i]));
      ra[i] = g.a;
      rb[i] = g.b;
      const float v = E::get(x[i]);
      rd[i] = h - v;
      h = __builtin_fmaf(g.a, h, g.b * v);
      rg[i] = E::get(go[i]);
    }
#pragma unroll
    for (int i = kBackSteps - 1; i >= 0; --i) m = {m.A * ra[i], ra[i] * (rg[i] + m.H)};
    Affine(*const map)[kWave] = &maps[turn & 1][p.base];
    map[p.wave][p.lane] = m;
    const int mine = n;
    if (tile > first) fetch(tile - p.tile_steps());
    if (!APART) __syncthreads();
    float c = s;
#pragma unroll 4
    for (int o = p.waves - 1; o >= 0; --o) {
      if (o == p.wave) c = s;
      const Affine q = map[o][p.lane];
      s = __builtin_fmaf(q.A, s, q.H);
    }
    const int64_t here = p.step(tile);
    const int left = p.in ? static_cast<int>(end - p.step(tile) < kBackSteps ? end - p.step(tile) : kBackSteps) : 0;
    T *gx = static_cast<T *>(a.gx) + here * BN + p.first, *gg = static_cast<T *>(a.gg) + here * BN + p.first;
#pragma unroll
    for (int i = kBackSteps - 1; i >= 0; --i) {
      const float g = rg[i] + c, dx = rb[i] * g, dg = dx * rd[i] * ra[i];
      c = ra[i] * g;
      if (all) {
        if (a.gx) (gx + i * BN)[p.lane] = E::put(dx);
        if (a.gg) (gg + i * BN)[p.lane] = E::put(dg);
      } else if (i < left) {
        if (a.gx) (gx + i * BN)[p.lane] = E::put(i < mine ? dx : 0.0f);
        if (a.gg) (gg + i * BN)[p.lane] = E::put(i < mine ? dg : 0.0f);
      }
    }
  }
  if (p.in && p.wave == 0 && a.seg == 0 && a.state_out) a.state_out[p.c()] = s;
}

// What a segment does to the state before it (BACK: to the gradient of the state
// after it).  The waves take their steps of a tile as in the main pass and leave
// what these do in LDS, for kTiles tiles at once.  [32768, 1, 2048] bf16: 73 us for 235
// MB, beside 76 us of the main pass; stretches of time to the waves, two rows of tiles
// on their way or twice the waves change nothing.
constexpr int kTiles = 4;

template <class E, bool BACK>
__global__ __launch_bounds__(kMaxWaves * kWave) void summarise(Args a) {
  using T = typename E::T;
  constexpr int STEPS = BACK ? kBackSteps : kSteps;  // (16 do not fit the registers)
  using P = Place<STEPS>;
  __shared__ Affine maps[kTiles][kMaxWaves][kWave];
  __shared__ Affine whole[kTiles][kWave];
  const int64_t block = locate<false>(a, a.segments - 1);
  if (block < 0) return;  // the whole workgroup
  if (BACK) ++a.seg;      // the first needs none, as the last forward
  P p;
  p.template set<T, false>(a, block);
  const int64_t first = a.seg * a.seg_steps;
  const int64_t end = first + a.seg_steps < a.T ? first + a.seg_steps : a.T;
  const int tiles = static_cast<int>((end - first + p.tile_steps() - 1) / p.tile_steps());
  T v[STEPS], gate[STEPS];
  int n = 0;
  const auto fetch = [&](int o) {
    const int64_t tile = first + (BACK ? tiles - 1 - o : o) * p.tile_steps();
    n = p.steps(tile);
    if (!__any(n > 0)) return;
    p.load(gate, p.gate, p.at_gate, a.gt, tile, a.T);
    if (!BACK)
      p.load(v, p.x, p.at_x, a.xt, tile, a.T);
    else if (a.g_out)
      p.load(v, p.out, p.at_out, a.ot, tile, a.T);
  };
  fetch(0);
  Affine all{1.0f, 0.0f};
  for (int o = 0; o < tiles; ++o) {
    if (!__all(n == STEPS)) mask<STEPS>(gate, n, E::put(kInf));
    if (!__all(n == STEPS) || (BACK && !a.g_out)) mask<STEPS>(v, BACK && !a.g_out ? 0 : n, E::put(0.0f));
    float ra[STEPS], ru[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const Gate<E> g(E::get(gate[i]));
      ra[i] = g.a;
      ru[i] = BACK ? E::get(v[i]) : g.b * E::get(v[i]);
    }
    if (o + 1 < tiles) fetch(o + 1);
    Affine m{1.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      const int i = BACK ? STEPS - 1 - k : k;
      m = {m.A * ra[i], BACK ? ra[i] * (ru[i] + m.H) : __builtin_fmaf(ra[i], m.H, ru[i])};
    }
    const int slot = o % kTiles;
    maps[slot][p.wave][p.lane] = m;
    if (slot + 1 < kTiles && o + 1 < tiles) continue;
    __syncthreads();
    // a wave to a tile, then the first one over the tiles
    for (int t = p.wave; t <= slot; t += p.waves) {
      m = {1.0f, 0.0f};
      for (int g = 0; g < p.waves; ++g) {
        const Affine q = maps[t][BACK ? p.waves - 1 - g : g][p.lane];
        m = {m.A * q.A, __builtin_fmaf(q.A, m.H, q.H)};
      }
      whole[t][p.lane] = m;
    }
    __syncthreads();
    if (p.wave == 0)
      for (int t = 0; t <= slot; ++t) {
        const Affine q = whole[t][p.lane];
        all = {all.A * q.A, __builtin_fmaf(q.A, all.H, q.H)};
      }
  }
  if (p.wave == 0 && p.in) a.joins[a.seg * a.B * a.N + p.c()] = all;
}

// A launch's latency for one sequence (2.2 us); 256 of 4096 channels, bf16: 4.8 us (15
// MB, 3.1 TB/s).
template <class E>
__global__ __launch_bounds__(256) void step(Args a) {
  using T = typename E::T;
  const int64_t c = myelin::block_id() * 256 + threadIdx.x;
  if (c >= a.B * a.N) return;
  const int64_t b = c / a.N, n = c - b * a.N;
  const Gate<E> g(E::get(static_cast<const T *>(a.gate)[b * a.gb + n]));
  const float h = __builtin_fmaf(g.a, a.state[c], g.b * E::get(static_cast<const T *>(a.x)[b * a.xb + n]));
  a.state_out[c] = h;
  static_cast<T *>(a.out)[c] = E::put(h);
}

// A workgroup's lanes reach over this many batch rows; their offsets have 32 bits.
bool reachable(int64_t stride, int64_t B, int64_t N) {
  return B == 1 || (stride >= 0 && stride < int64_t{1} << 29 && (64 / N + 1) * stride + N < int64_t{1} << 29);
}

int check(const char *what, int dtype, int64_t T, int64_t B, int64_t N) {
  if (dtype != 0 && dtype != 2) return myelin::invalid("%s: unsupported dtype %d", what, dtype);
  if (T < 1 || B < 0 || N < 0) return myelin::invalid("%s: T must be positive, B and N not negative", what);
  if (T >= int64_t{1} << 31 || B >= int64_t{1} << 31 || N >= int64_t{1} << 28 || B * N >= int64_t{1} << 36)
    return myelin::invalid("%s: too many steps or channels", what);
  return MYELIN_OK;
}

struct Plan {
  int64_t blocks, segments, seg_steps;
  int waves;
  bool apart;
};

// A CU holds 16 waves of these registers: its workgroups share them, so that none waits
// for others to end and each runs over several tiles, whose loads and sums overlap.
// bf16, forward and backward, against 16 waves to each: [512, 32, 2048] 60 -> 50 us and
// 97 -> 83, [67, 38, 6917] 45 -> 34 and 73 -> 56, [256, 66, 1000] 33 -> 26 and 59 -> 44.
// (Powers of two: 5 waves fall on the SIMDs so that three workgroups do not fit a CU.
// One wave to a workgroup of many: [200, 150, 2048] backward 151 -> 167.  LDS of the
// waves' own size, so that two have 2 KB of it: 2 % slower everywhere.)
//
// Up to 64 steps of many channels, a wave goes over all of a block's time, beside three of
// other blocks in its workgroup (APART): nothing is exchanged, and a CU does not run out of
// LDS for workgroups of one.  [24, 700, 2048] bf16, forward and backward: 63 -> 56 us and
// 92 -> 80, [8, 1024, 4096] 135 -> 92 and 122 -> 82; of 67 steps the backward pass is slower
// so, 55 -> 61.
//
// Time is split where the channels leave half of the CUs without a workgroup: 128
// blocks in two segments, [8192, 4, 2048] bf16: forward 142 us either way, backward
// 276 -> 210; 175 blocks are faster whole (70 and 140 us, against 101 and 172).
Plan plan_of(int64_t T, int64_t B, int64_t N) {
  Plan p;
  p.blocks = (B * N + kWave - 1) / kWave;
  const int64_t needed = (T + kSteps - 1) / kSteps;
  int waves = kMaxWaves;
  const int least = needed > kApart ? 2 : 1;
  while (waves > least && p.blocks * waves > 256 * kMaxWaves) waves /= 2;
  p.waves = static_cast<int>(needed < waves ? needed : waves);
  p.apart = p.waves == 1 && p.blocks > 2048;
  const int64_t tile = p.waves * kSteps, tiles = (T + tile - 1) / tile;
  int64_t n = p.blocks > 128 ? 1 : 256 / p.blocks;
  if (n > tiles) n = tiles;
  const int64_t some = (tiles + n - 1) / n;
  p.seg_steps = some * tile;
  p.segments = (tiles + some - 1) / some;
  return p;
}

// Workgroups of up to 1024 threads, fewer than 2^32 in x.
dim3 grid_for(int64_t blocks) {
  blocks = (blocks + 7) / 8 * 8;  // as many to each XCD
  const int64_t x = int64_t{1} << 21, y = (blocks + x - 1) / x;
  return dim3(static_cast<unsigned>(y > 1 ? x : blocks), static_cast<unsigned>(y));
}

int64_t workspace_of(const Plan &p, int64_t B, int64_t N) { return p.segments == 1 ? 0 : 2 * p.segments * B * N; }

int prepare(const char *what, Args &a, Plan &p, float *workspace, int64_t elems) {
  p = plan_of(a.T, a.B, a.N);
  const int64_t need = workspace_of(p, a.B, a.N);
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
  const int threads = p.waves * kWave;
  if (p.segments > 1) summarise<E, BACK><<<grid_for(p.blocks * (p.segments - 1)), threads, 0, s>>>(a);
  if (p.apart) {
    const dim3 grid = grid_for((p.blocks + kApart - 1) / kApart);
    BACK ? backward<E, true><<<grid, kApart * kWave, 0, s>>>(a) : forward<E, true><<<grid, kApart * kWave, 0, s>>>(a);
  } else {
    const dim3 grid = grid_for(p.blocks * p.segments);
    BACK ? backward<E, false><<<grid, threads, 0, s>>>(a) : forward<E, false><<<grid, threads, 0, s>>>(a);
  }
}

}  // namespace

extern "C" int64_t myelin_gated_recurrence_kept_elems(int64_t T, int64_t B, int64_t N) {
  return (T + kBackSteps - 1) / kBackSteps * B * N;
}

extern "C" int64_t myelin_gated_recurrence_workspace_elems(int dtype, int64_t T, int64_t B, int64_t N, int backward) {
  (void)dtype;
  (void)backward;
  if (T < 1 || B < 1 || N < 1) return 0;
  return workspace_of(plan_of(T, B, N), B, N);
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
    if (!reachable(strides[o], B, N)) return myelin::invalid("%s: batch stride negative or too large", what);
  Args a{};
  a.T = T, a.B = B, a.N = N;
  Plan p;
  if (int rc = prepare(what, a, p, workspace, workspace_elems)) return rc;
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
    if (!reachable(strides[o], B, N)) return myelin::invalid("%s: batch stride negative or too large", what);
  Args a{};
  a.T = T, a.B = B, a.N = N;
  Plan p;
  if (int rc = prepare(what, a, p, workspace, workspace_elems)) return rc;
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
