// The embeddings of tokens, scaled, and the gradient of their table:
//
//   y_i = scale w[token_i]      dw[v] = scale sum_{i: token_i = v} dy_i
//
// A padding token's row is 0 and has no gradient; a token outside [0, V) gives a
// row of NaN and has none either: nothing is read out of range.  The sums are
// fp32, of groups of a token's positions that the positions alone decide, and of those
// groups in their order: the same bits on every run.
//
// The gradient takes the positions in the order of their tokens (a stable sort), so
// that each row of the table is written once, by the threads that sum it, and nothing
// in memory is atomic (the sort's whole numbers are counted with atomics in LDS, whose
// order does not show).  A token may have a tenth of all positions: a run of equal
// tokens is cut at multiples of 32 sorted positions, whole pieces are summed by
// workgroups of their own, and the row's threads add up what is left.

#include "elements.h"

namespace {

using myelin::BF16;
using myelin::F32;
using myelin::kWave;

constexpr int kThreads = 256;
constexpr int64_t kNoPadding = INT64_MIN;  // no token is padding, this one neither

struct Args {
  const int64_t *tokens;
  const void *from;  // the table; backward: dy [M, D]
  void *to;          // y [M, D]; backward: dw [V, D]
  int64_t ld, M, V, D, padding;
  float scale;
  int64_t units;        // vectors of a row, the last shifted back to end with it
  int64_t slices;       // pieces of a row that a group of threads takes at a time
  const int32_t *keys, *places, *starts;
  float *pieces, *pieces2;
};

// The first element of a row's vector.  (Where D is not a multiple of VEC the last two
// share elements, and their threads find the same values for them.  16384 tokens of
// [32000, 1001] bf16, against an element to a thread: lookup 24 -> 10 us, gradient 74 ->
// 46.)
template <int VEC>
__device__ __forceinline__ int64_t column(const Args &a, int64_t u) {
  return u < a.units - 1 ? u * VEC : a.D - VEC;
}

// A row's threads: a power of two of them, each with a vector of VEC elements.
int threads_of(int64_t units, int most) {
  int t = 1;
  while (t < most && t < units) t *= 2;
  return t;
}

template <class E, int VEC>
struct Vector {
  using T = typename E::T;
  // (at any element: the memory takes vectors that are not aligned)
  typedef T vec __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  float v[VEC];
  __device__ void zero() {
#pragma unroll
    for (int q = 0; q < VEC; ++q) v[q] = 0.0f;
  }
  __device__ void load(const T *p) {
    if constexpr (VEC == 1) {
      v[0] = E::get(*p);
    } else {
      const vec r = *reinterpret_cast<const vec *>(p);
#pragma unroll
      for (int q = 0; q < VEC; ++q) v[q] = E::get(r[q]);
    }
  }
  __device__ void add(const Vector &o) {
#pragma unroll
    for (int q = 0; q < VEC; ++q) v[q] += o.v[q];
  }
  template <bool STREAM>
  __device__ void store(T *p, float scale) const {
    if constexpr (VEC == 1) {
      *p = E::put(v[0] * scale);
    } else {
      vec r;
#pragma unroll
      for (int q = 0; q < VEC; ++q) r[q] = E::put(v[q] * scale);
      if constexpr (STREAM)
        __builtin_nontemporal_store(r, reinterpret_cast<vec *>(p));
      else
        *reinterpret_cast<vec *>(p) = r;
    }
  }
};

// ---- lookup ----------------------------------------------------------------
constexpr int kRows = 4;  // rows of a thread, loaded together

// PER threads to a row (or a slice of it).  16384 tokens of [32768, 2048] bf16: 17 us,
// bound by memory (67 MB written past the caches, rows of frequent tokens read from
// them).
template <class E, int VEC, bool STREAM>
__global__ __launch_bounds__(kThreads) void lookup(Args a, int per) {
  using T = typename E::T;
  const int groups = kThreads / per, group = threadIdx.x / per;
  const int64_t block = myelin::block_id(), rows = block / a.slices, slice = block - rows * a.slices;
  const int64_t u = slice * per + threadIdx.x % per;
  if (u >= a.units) return;
  // (what is not there is loaded from the last position and the first row: loads
  // under conditions wait for each other)
  Vector<E, VEC> r[kRows];
  int64_t i[kRows], token[kRows];
#pragma unroll
  for (int o = 0; o < kRows; ++o) {
    i[o] = (rows * kRows + o) * groups + group;
    token[o] = a.tokens[i[o] < a.M ? i[o] : a.M - 1];
  }
#pragma unroll
  for (int o = 0; o < kRows; ++o) {
    const bool inside = token[o] >= 0 && token[o] < a.V;
    r[o].load(static_cast<const T *>(a.from) + (inside ? token[o] : 0) * a.ld + column<VEC>(a, u));
  }
#pragma unroll
  for (int o = 0; o < kRows; ++o) {
    if (i[o] >= a.M) continue;
    const bool hole = a.padding != kNoPadding && token[o] == a.padding, outside = token[o] < 0 || token[o] >= a.V;
#pragma unroll
    for (int q = 0; q < VEC; ++q) r[o].v[q] = hole ? 0.0f : outside ? __builtin_nanf("") : r[o].v[q];
    r[o].template store<STREAM>(static_cast<T *>(a.to) + i[o] * a.D + column<VEC>(a, u), a.scale);
  }
}

// ---- gradient: the positions in the order of their tokens -------------------
// A stable sort by digits of the key, the lowest first.  Padding and tokens outside
// the table have the key V, behind all others.
constexpr int kDigit = 9, kBins = 1 << kDigit;

__device__ __forceinline__ int32_t key_of(const Args &a, int64_t i) {
  const int64_t t = a.tokens[i < a.M ? i : a.M - 1];
  return static_cast<int32_t>(t < 0 || t >= a.V || t == a.padding ? a.V : t);
}

// The lanes whose digit is this lane's, of those that have one.  (BITS: 2 passes
// of 8 bits rather than 9 where they will do: these ballots are what a sort takes.)
template <int BITS>
__device__ __forceinline__ uint64_t alike(int digit, bool in) {
  const uint64_t m = __ballot(in);
  uint32_t lo = static_cast<uint32_t>(m), hi = static_cast<uint32_t>(m >> 32);
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const int one = digit << (31 - b) >> 31;  // all ones where the bit is set
    const uint64_t set = __ballot(one != 0);
    lo &= ~(static_cast<uint32_t>(set) ^ one);
    hi &= ~(static_cast<uint32_t>(set >> 32) ^ one);
  }
  return static_cast<uint64_t>(hi) << 32 | lo;
}

__device__ __forceinline__ int lower(uint64_t m) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(m >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(m), 0));
}

// An item's place among those of its digit that its wave has had, in `count`, which
// it goes into.  (One lane of those alike writes it: as atomics, equal digits would
// wait for each other.  In LDS a wave's accesses are done in its order.)
template <int BITS>
__device__ __forceinline__ int32_t place_in_wave(int32_t *count, int digit, bool in) {
  const uint64_t m = alike<BITS>(digit, in);
  const int rank = lower(m);
  const int32_t had = in ? count[digit] : 0;
  if (in && rank == 0) count[digit] = had + __popcll(m);
  return had + rank;
}

// Each workgroup has a stretch of the positions, in turns of kTurn.  A pass over a
// digit: its counts of the bins, the offsets of all counts, and each position to its
// place.  (16 waves of a turn of 64 each: the ballots are what takes the time.  Waves of 4
// turns: 131072 positions of [2000, 256] bf16 49 -> 59 us.  Up to 16384 positions in one
// workgroup's LDS, in one launch: [10000, 256] 32 -> 40.)
constexpr int kSortWaves = 16, kTurn = kSortWaves * kWave, kSortThreads = kTurn;

// Up to kAlone workgroups count all positions themselves: no launch before that (8192
// positions 28 us either way, 16384 6 us more).  Up to kDirect add up all workgroups'
// counts; more have it done for them (128 of them, [2000, 256] bf16: 49 us, 52 with the
// launch that does it).
constexpr int kAlone = 8, kDirect = 128, kMostBlocks = 512;
enum Counts { kOwn, kOthers, kSums };

struct Sort {
  Args a;
  const int32_t *from_keys, *from_places;  // null: the tokens
  int32_t *to_keys, *to_places;
  int32_t *counts;  // kOthers: [blocks, bins]; kSums: [bins, blocks] and the bins' sums
  int blocks, shift;
  Counts which;
  int64_t stretch;  // a multiple of kTurn
  __device__ int32_t key(int64_t i) const { return from_keys ? from_keys[i < a.M ? i : a.M - 1] : key_of(a, i); }
  __device__ int32_t place(int64_t i) const { return from_keys ? from_places[i] : static_cast<int32_t>(i); }
};

template <int BITS>
__global__ __launch_bounds__(kSortThreads) void sort_count(Sort s) {
  constexpr int BINS = 1 << BITS;
  __shared__ int32_t count[kSortWaves][BINS];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  for (int b = lane; b < BINS; b += kWave) count[wave][b] = 0;
  const int64_t begin = blockIdx.x * s.stretch, end = begin + s.stretch < s.a.M ? begin + s.stretch : s.a.M;
  for (int64_t i = begin + tid; i - tid < end; i += kTurn)
    place_in_wave<BITS>(count[wave], s.key(i) >> s.shift & (BINS - 1), i < end);
  __syncthreads();
  for (int b = tid; b < BINS; b += kSortThreads) {
    int32_t sum = 0;
    for (int w = 0; w < kSortWaves; ++w) sum += count[w][b];
    s.counts[s.which == kOthers ? blockIdx.x * BINS + b : static_cast<int64_t>(b) * s.blocks + blockIdx.x] = sum;
  }
}

// A wave to a bin: what each workgroup's positions of it come after, and behind all
// of these the bins' sums.
template <int BITS>
__global__ __launch_bounds__(kThreads) void sort_offsets(int32_t *counts, int blocks) {
  constexpr int BINS = 1 << BITS, EACH = kMostBlocks / kWave;
  const int lane = threadIdx.x & (kWave - 1), bin = blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave;
  const int each = (blocks + kWave - 1) / kWave, first = lane * each;
  int32_t *const of = counts + static_cast<int64_t>(bin) * blocks;
  int32_t v[EACH], sum = 0;
#pragma unroll
  for (int o = 0; o < EACH; ++o) v[o] = of[first + o < blocks ? first + o : blocks - 1];
#pragma unroll
  for (int o = 0; o < EACH; ++o) sum += o < each && first + o < blocks ? v[o] : 0;
  int32_t run = sum;
  for (int o = 1; o < kWave; o <<= 1) {
    const int32_t up = __shfl_up(run, o);
    if (lane >= o) run += up;
  }
  if (lane == kWave - 1) counts[static_cast<int64_t>(BINS) * blocks + bin] = run;
  run -= sum;
#pragma unroll
  for (int o = 0; o < EACH; ++o) {
    if (o < each && first + o < blocks) of[first + o] = run;
    run += v[o];
  }
}

template <int BITS>
__global__ __launch_bounds__(kSortThreads) void sort_place(Sort s) {
  constexpr int BINS = 1 << BITS;
  __shared__ int32_t count[kSortWaves][BINS], next[BINS];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  // what comes before this workgroup's: all smaller digits, and equal ones of earlier
  // workgroups
  if (s.which == kOwn) {  // (whole numbers: the order of the atomics does not show)
    for (int b = tid; b < 2 * BINS; b += kSortThreads) count[b / BINS][b % BINS] = 0;
    __syncthreads();
    constexpr int MANY = 8;
    for (int turn = 0; turn < s.blocks; turn += MANY) {
      int digit[MANY];
#pragma unroll
      for (int o = 0; o < MANY; ++o)
        digit[o] = s.key(static_cast<int64_t>(turn + o) * kTurn + tid) >> s.shift & (BINS - 1);
#pragma unroll
      for (int o = 0; o < MANY; ++o) {
        int32_t *const to = count[turn + o < static_cast<int>(blockIdx.x)];
        const bool in = static_cast<int64_t>(turn + o) * kTurn + tid < s.a.M;
        // (one token in all lanes: they would wait for each other)
        const int first = __builtin_amdgcn_readfirstlane(digit[o]);
        if (__all(in && digit[o] == first)) {
          if (lane == 0) atomicAdd(to + first, kWave);
        } else if (in) {
          atomicAdd(to + digit[o], 1);
        }
      }
    }
    __syncthreads();
    if (tid < BINS) {
      next[tid] = count[1][tid];
      count[0][tid] += count[1][tid];
    }
  } else if (s.which == kOthers) {
    constexpr int GROUPS = kSortThreads / BINS < kSortWaves / 2 ? kSortThreads / BINS : kSortWaves / 2;
    const int b = tid % BINS, group = tid / BINS, each = (s.blocks + GROUPS - 1) / GROUPS;
    const int last = (group + 1) * each < s.blocks ? (group + 1) * each : s.blocks;
    if (group < GROUPS) {
      int32_t all = 0, earlier = 0;
#pragma unroll 8
      for (int o = group * each; o < last; ++o) {
        const int32_t c = s.counts[o * BINS + b];
        all += c;
        earlier += o < static_cast<int>(blockIdx.x) ? c : 0;
      }
      count[2 * group][b] = all;
      count[2 * group + 1][b] = earlier;
    }
    __syncthreads();
    if (tid < BINS) {
      int32_t total = 0, before = 0;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        total += count[2 * g][tid];
        before += count[2 * g + 1][tid];
      }
      count[0][tid] = total;
      next[tid] = before;
    }
  } else if (tid < BINS) {
    next[tid] = s.counts[static_cast<int64_t>(tid) * s.blocks + blockIdx.x];
    count[0][tid] = s.counts[static_cast<int64_t>(BINS) * s.blocks + tid];
  }
  __syncthreads();
  if (wave == 0) {
    constexpr int EACH = BINS / kWave;
    int32_t v[EACH], sum = 0;
    for (int o = 0; o < EACH; ++o) {
      v[o] = count[0][lane * EACH + o];
      sum += v[o];
    }
    int32_t run = sum;
    for (int o = 1; o < kWave; o <<= 1) {
      const int32_t up = __shfl_up(run, o);
      if (lane >= o) run += up;
    }
    run -= sum;
    for (int o = 0; o < EACH; ++o) {
      next[lane * EACH + o] += run;
      run += v[o];
    }
  }
  __syncthreads();
  const int64_t begin = blockIdx.x * s.stretch, end = begin + s.stretch < s.a.M ? begin + s.stretch : s.a.M;
  for (int64_t turn = begin; turn < end; turn += kTurn) {
    const int64_t i = turn + tid;
    const int32_t k = s.key(i);
    const int digit = k >> s.shift & (BINS - 1);
    for (int b = lane; b < BINS; b += kWave) count[wave][b] = 0;
    const int32_t local = place_in_wave<BITS>(count[wave], digit, i < end);
    __syncthreads();
    for (int b = tid; b < BINS; b += kSortThreads) {
      int32_t run = next[b];
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {
        const int32_t c = count[w][b];
        count[w][b] = run;
        run += c;
      }
      next[b] = run;
    }
    __syncthreads();
    if (i < end) {
      const int32_t to = count[wave][digit] + local;
      s.to_keys[to] = k;
      s.to_places[to] = s.place(i);
    }
    __syncthreads();
  }
}

// ---- gradient: sums ---------------------------------------------------------
constexpr int kPiece = 32;  // sorted positions of a piece, pieces of a larger one

// Sums n rows (of the list places[0, n)) into r, in order, some loads at a time.
template <class E, int VEC>
__device__ __forceinline__ void sum_rows(const Args &a, const int32_t *places, int n, int64_t u, Vector<E, VEC> &r) {
  using T = typename E::T;
  const T *from = static_cast<const T *>(a.from) + column<VEC>(a, u);
  constexpr int MANY = 8;
  int i = 0;
  for (; i + MANY <= n; i += MANY) {
    Vector<E, VEC> v[MANY];
#pragma unroll
    for (int o = 0; o < MANY; ++o) v[o].load(from + places[i + o] * a.D);
#pragma unroll
    for (int o = 0; o < MANY; ++o) r.add(v[o]);
  }
  for (; i < n; ++i) {
    Vector<E, VEC> v;
    v.load(from + places[i] * a.D);
    r.add(v);
  }
}

// fp32 rows [n, D] in a row
template <class E, int VEC>
__device__ __forceinline__ void sum_pieces(const float *from, int64_t n, int64_t D, Vector<E, VEC> &r) {
  constexpr int MANY = 8;
  int64_t i = 0;
  for (; i + MANY <= n; i += MANY) {
    float v[MANY][VEC];
#pragma unroll
    for (int o = 0; o < MANY; ++o)
#pragma unroll
      for (int q = 0; q < VEC; ++q) v[o][q] = from[(i + o) * D + q];
#pragma unroll
    for (int o = 0; o < MANY; ++o)
#pragma unroll
      for (int q = 0; q < VEC; ++q) r.v[q] += v[o][q];
  }
  for (; i < n; ++i)
#pragma unroll
    for (int q = 0; q < VEC; ++q) r.v[q] += from[i * D + q];
}

// Adds up the groups' vectors, in their order, into the first group's.
template <class E, int VEC>
__device__ __forceinline__ void join(float *red, int groups, int group, int per, int at, Vector<E, VEC> &r) {
#pragma unroll
  for (int q = 0; q < VEC; ++q) red[(group * per + at) * VEC + q] = r.v[q];
  __syncthreads();
  if (group == 0)
    for (int o = 1; o < groups; ++o)
#pragma unroll
      for (int q = 0; q < VEC; ++q) r.v[q] += red[(o * per + at) * VEC + q];
}

// The pieces of the sorted positions that one token has, a workgroup each (and
// slice); the workgroups after them find where each token's positions start.  7 us:
// of latency.  (A search among keys in LDS first changes nothing.)
template <class E, int VEC>
__global__ __launch_bounds__(kThreads) void sum_whole_pieces(Args a, int per, int64_t blocks, int32_t *starts) {
  __shared__ float red[kThreads * VEC];
  const int64_t block = myelin::block_id();
  if (block >= blocks) {
    const int64_t v = (block - blocks) * kThreads + threadIdx.x;
    if (v > a.V) return;
    int64_t lo = 0, hi = a.M;  // the first whose key is at least v
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (a.keys[mid] < v)
        lo = mid + 1;
      else
        hi = mid;
    }
    starts[v] = static_cast<int32_t>(lo);
    return;
  }
  const int64_t piece = block / a.slices, slice = block - piece * a.slices, at = piece * kPiece;
  if (a.keys[at] != a.keys[at + kPiece - 1] || a.keys[at] == a.V) return;  // the whole workgroup
  const int groups = kThreads / per, group = threadIdx.x / per, lane = threadIdx.x % per;
  const int64_t u = slice * per + lane;
  Vector<E, VEC> r;
  r.zero();
  const int each = kPiece / groups > 0 ? kPiece / groups : 1, used = kPiece / each;
  if (u < a.units && group < used) sum_rows<E, VEC>(a, a.places + at + group * each, each, u, r);
  join<E, VEC>(red, used < groups ? used : groups, group, per, lane, r);
  if (group == 0 && u < a.units)
#pragma unroll
    for (int q = 0; q < VEC; ++q) a.pieces[piece * a.D + column<VEC>(a, u) + q] = r.v[q];
}

// and 32 of those that one token has
template <class E, int VEC>
__global__ __launch_bounds__(kThreads) void sum_larger_pieces(Args a, int per) {
  __shared__ float red[kThreads * VEC];
  const int64_t block = myelin::block_id();
  const int64_t piece = block / a.slices, slice = block - piece * a.slices, at = piece * kPiece * kPiece;
  if (at + kPiece * kPiece > a.M || a.keys[at] != a.keys[at + kPiece * kPiece - 1] || a.keys[at] == a.V) return;
  const int groups = kThreads / per, group = threadIdx.x / per, lane = threadIdx.x % per;
  const int64_t u = slice * per + lane;
  Vector<E, VEC> r;
  r.zero();
  const int each = kPiece / groups > 0 ? kPiece / groups : 1, used = kPiece / each;
  if (u < a.units && group < used)
    sum_pieces<E, VEC>(a.pieces + (piece * kPiece + group * each) * a.D + column<VEC>(a, u), each, a.D, r);
  join<E, VEC>(red, used < groups ? used : groups, group, per, lane, r);
  if (group == 0 && u < a.units)
#pragma unroll
    for (int q = 0; q < VEC; ++q) a.pieces2[piece * a.D + column<VEC>(a, u) + q] = r.v[q];
}

// Each row of the table: what of its run is before the first whole piece, the whole
// pieces (the larger ones among them), what is behind them.  ROWS of a group of threads:
// 1 where the table is small, so that its rows with many positions do not wait for each
// other.  16384 positions of [32768, 2048] bf16: 35 us (201 MB, 5.7 TB/s).  (Zeros that the
// sort's launches write on CUs that it leaves free, and only rows with positions here: 5
// us more in all.)
constexpr int kTableRows = 4;

template <class E, int VEC, int ROWS, bool STREAM>
__global__ __launch_bounds__(kThreads) void sum_runs(Args a, int per) {
  using T = typename E::T;
  const int groups = kThreads / per, group = threadIdx.x / per;
  const int64_t block = myelin::block_id(), rows = block / a.slices, slice = block - rows * a.slices;
  const int64_t first = (rows * groups + group) * ROWS, u = slice * per + threadIdx.x % per;
  if (first >= a.V || u >= a.units) return;
  int32_t start[ROWS + 1];
#pragma unroll
  for (int o = 0; o <= ROWS; ++o) start[o] = a.starts[first + o < a.V ? first + o : a.V];
#pragma unroll
  for (int o = 0; o < ROWS; ++o) {
    const int64_t v = first + o, lo = start[o], hi = start[o + 1];
    if (v >= a.V) return;
    Vector<E, VEC> r;
    r.zero();
    const int64_t p0 = (lo + kPiece - 1) / kPiece, p1 = hi / kPiece;
    if (p0 >= p1) {
      sum_rows<E, VEC>(a, a.places + lo, static_cast<int>(hi - lo), u, r);
    } else {
      sum_rows<E, VEC>(a, a.places + lo, static_cast<int>(p0 * kPiece - lo), u, r);
      const float *pieces = a.pieces + column<VEC>(a, u);
      const int64_t l0 = (p0 + kPiece - 1) / kPiece, l1 = p1 / kPiece;
      if (!a.pieces2 || l0 >= l1) {
        sum_pieces<E, VEC>(pieces + p0 * a.D, p1 - p0, a.D, r);
      } else {
        sum_pieces<E, VEC>(pieces + p0 * a.D, l0 * kPiece - p0, a.D, r);
        sum_pieces<E, VEC>(a.pieces2 + column<VEC>(a, u) + l0 * a.D, l1 - l0, a.D, r);
        sum_pieces<E, VEC>(pieces + l1 * kPiece * a.D, p1 - l1 * kPiece, a.D, r);
      }
      sum_rows<E, VEC>(a, a.places + p1 * kPiece, static_cast<int>(hi - p1 * kPiece), u, r);
    }
    r.template store<STREAM>(static_cast<T *>(a.to) + v * a.D + column<VEC>(a, u), a.scale);
  }
}

// ---- gradient: few tokens, small tables -------------------------------------
// A workgroup to a row (and slice): it goes through all tokens itself, keeps the
// positions of its own in order, and sums their rows.  No sort, one launch: 2048
// tokens of [50, 128] fp32 6.6 us, latency.  Tables of more rows are zeros first, and a
// workgroup has a position, and its token's row if no earlier position has.
constexpr int kFewThreads = 512, kFew = 4096;  // (kFewPositions is less)

template <class E, int VEC, bool POSITIONS>
__global__ __launch_bounds__(kFewThreads) void sum_few(Args a, int per) {
  using T = typename E::T;
  __shared__ int32_t list[kFew];
  __shared__ int found[kFew / kFewThreads][kFewThreads / kWave];
  __shared__ float red[kFewThreads * VEC];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int64_t block = myelin::block_id(), unit = block / a.slices, slice = block - unit * a.slices;
  const int64_t v = POSITIONS ? key_of(a, unit) : unit;
  if (POSITIONS && (unit >= a.M || v == a.V)) return;  // the whole workgroup
  constexpr int ROUNDS = kFew / kFewThreads, WAVES = kFewThreads / kWave;
  uint64_t hit[ROUNDS];
#pragma unroll
  for (int o = 0; o < ROUNDS; ++o) {
    const int i = o * kFewThreads + tid;
    hit[o] = __ballot(i < a.M && key_of(a, i) == v);
    if (lane == 0) found[o][wave] = __popcll(hit[o]);
  }
  __syncthreads();
  int before = 0, n = 0;
#pragma unroll
  for (int o = 0; o < ROUNDS; ++o) {
    for (int w = 0; w < WAVES; ++w) {
      if (w == wave) before = n;
      n += found[o][w];
    }
    if (hit[o] >> lane & 1) list[before + lower(hit[o])] = o * kFewThreads + tid;
  }
  __syncthreads();
  if (POSITIONS && list[0] != unit) return;
  const int groups = kFewThreads / per, group = tid / per, at = tid % per;
  const int64_t u = slice * per + at;
  const int each = (n + groups - 1) / groups, from = group * each < n ? group * each : n,
            to = from + each < n ? from + each : n;
  Vector<E, VEC> r;
  r.zero();
  if (u < a.units) sum_rows<E, VEC>(a, list + from, to - from, u, r);
  join<E, VEC>(red, groups, group, per, at, r);
  if (group == 0 && u < a.units)
    r.template store<false>(static_cast<T *>(a.to) + v * a.D + column<VEC>(a, u), a.scale);
}

// no tokens at all
template <class E, int VEC>
__global__ __launch_bounds__(kThreads) void zeros(Args a) {
  using T = typename E::T;
  const int64_t i = (myelin::block_id() * kThreads + threadIdx.x) * VEC, all = a.V * a.D;
  if (i >= all) return;
  Vector<E, VEC> r;
  r.zero();
  r.template store<false>(static_cast<T *>(a.to) + (i + VEC < all ? i : all - VEC), 1.0f);
}

// ---- launches ---------------------------------------------------------------
struct Layout {  // of the workspace, in bytes
  bool few, positions;  // a workgroup to a row, to a position: none
  int passes, bits, blocks;
  int64_t stretch, keys[2], places[2], counts, starts, pieces, pieces2, size;
};

// Rows of the table, times D / 64 where they are wider, that sum_few is taken for: each
// goes through all tokens.
constexpr int64_t kFewRows = 2048;

// Positions times slices of 128 threads (so that a group of threads has at most 512 rows,
// if all are one token's) that it is taken for elsewhere, against the sort: 60 of [5407, 26]
// bf16 16 -> 6 us, 1024 of [32000, 512] 27 -> 16, 2048 30 -> 23, 4096 32 -> 42.
constexpr int64_t kFewPositions = 2048;

// vec: elements of a thread's vector
Layout layout_of(int64_t M, int64_t V, int64_t D, int vec) {
  Layout l{};
  l.few = M <= kFew && V * ((D + 63) / 64) <= kFewRows;
  const int64_t units = (D + vec - 1) / vec, some = threads_of(units, 2 * kWave);
  l.positions = !l.few && M * ((units + some - 1) / some) <= kFewPositions;
  if (l.few || l.positions || M == 0) return l;
  int bits = 1;
  while (V >> bits) ++bits;
  l.passes = (bits + kDigit - 1) / kDigit;
  l.bits = (bits + l.passes - 1) / l.passes;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 15) / 16 * 16;
    return here;
  };
  for (int o = 0; o < 2; ++o) {
    l.keys[o] = take(4 * M);
    l.places[o] = take(4 * M);
  }
  // workgroups of whole turns
  const int64_t turns = (M + kTurn - 1) / kTurn, each = (turns + kMostBlocks - 1) / kMostBlocks;
  l.stretch = each * kTurn;
  l.blocks = static_cast<int>((M + l.stretch - 1) / l.stretch);
  l.counts = take(4 * static_cast<int64_t>(kBins) * (l.blocks + 1));
  l.starts = take(4 * (V + 1));
  l.pieces = take(4 * (M / kPiece) * D);
  // (a run of 16384 has 512 pieces: few enough to add up at once)
  l.pieces2 = M <= 16384 ? -1 : take(4 * (M / (kPiece * kPiece)) * D);
  l.size = at;
  return l;
}

template <class E, int VEC>
void launch_lookup(Args &a, hipStream_t s) {
  a.units = (a.D + VEC - 1) / VEC;
  const int per = threads_of(a.units, kThreads);
  a.slices = (a.units + per - 1) / per;
  const int64_t rows = static_cast<int64_t>(kThreads / per) * kRows;
  const dim3 grid = myelin::grid_of((a.M + rows - 1) / rows * a.slices);
  if (a.M * a.D * static_cast<int64_t>(sizeof(typename E::T)) >= myelin::kStreamBytes)
    lookup<E, VEC, true><<<grid, kThreads, 0, s>>>(a, per);
  else
    lookup<E, VEC, false><<<grid, kThreads, 0, s>>>(a, per);
}

template <int BITS>
void launch_sort(const Sort &t, hipStream_t s) {
  if (t.which != kOwn) sort_count<BITS><<<t.blocks, kSortThreads, 0, s>>>(t);
  if (t.which == kSums) sort_offsets<BITS><<<(1 << BITS) / (kThreads / kWave), kThreads, 0, s>>>(t.counts, t.blocks);
  sort_place<BITS><<<t.blocks, kSortThreads, 0, s>>>(t);
}

template <class E, int VEC>
void launch_gradient(Args &a, const Layout &l, char *ws, hipStream_t s) {
  a.units = (a.D + VEC - 1) / VEC;
  const auto zero = [&] {
    const int64_t each = kThreads * VEC;
    zeros<E, VEC><<<myelin::grid_of((a.V * a.D + each - 1) / each), kThreads, 0, s>>>(a);
  };
  if (a.M == 0) return zero();
  const int some = threads_of(a.units, l.few ? kWave : 2 * kWave);
  a.slices = (a.units + some - 1) / some;
  if (l.few) {
    sum_few<E, VEC, false><<<myelin::grid_of(a.V * a.slices), kFewThreads, 0, s>>>(a, some);
    return;
  }
  if (l.positions) {
    zero();
    sum_few<E, VEC, true><<<myelin::grid_of(a.M * a.slices), kFewThreads, 0, s>>>(a, some);
    return;
  }
  a.starts = reinterpret_cast<int32_t *>(ws + l.starts);
  a.pieces = reinterpret_cast<float *>(ws + l.pieces);
  a.pieces2 = l.pieces2 < 0 ? nullptr : reinterpret_cast<float *>(ws + l.pieces2);
  const auto words = [&](int64_t at) { return reinterpret_cast<int32_t *>(ws + at); };
  const int64_t bytes = a.V * a.D * static_cast<int64_t>(sizeof(typename E::T));
  const int digit = l.bits <= 6 ? 6 : l.bits <= 8 ? 8 : 9;
  const Counts which = l.blocks <= kAlone ? kOwn : l.blocks <= kDirect ? kOthers : kSums;
  for (int pass = 0; pass < l.passes; ++pass) {
    const Sort t{a,
                 pass ? a.keys : nullptr,
                 pass ? a.places : nullptr,
                 words(l.keys[pass & 1]),
                 words(l.places[pass & 1]),
                 words(l.counts),
                 l.blocks,
                 pass * digit,
                 which,
                 l.stretch};
    if (digit == 6)
      launch_sort<6>(t, s);
    else if (digit == 8)
      launch_sort<8>(t, s);
    else
      launch_sort<9>(t, s);
    a.keys = t.to_keys;
    a.places = t.to_places;
  }
  int per = threads_of(a.units, kWave);
  a.slices = (a.units + per - 1) / per;
  const int64_t blocks = a.M / kPiece * a.slices;
  sum_whole_pieces<E, VEC><<<myelin::grid_of(blocks + a.V / kThreads + 1), kThreads, 0, s>>>(a, per, blocks,
                                                                                        words(l.starts));
  if (a.pieces2 && a.M >= kPiece * kPiece)
    sum_larger_pieces<E, VEC><<<myelin::grid_of(a.M / (kPiece * kPiece) * a.slices), kThreads, 0, s>>>(a, per);
  per = threads_of(a.units, kThreads);
  a.slices = (a.units + per - 1) / per;
  const int64_t groups = kThreads / per;
  const auto grid = [&](int64_t rows) { return myelin::grid_of((a.V + rows - 1) / rows * a.slices); };
  const bool stream = bytes >= myelin::kStreamBytes;
  // with 4 rows a group: 131072 positions of [2000, 256] bf16 49 -> 72 us, 2^20 of
  // [32000, 32] 111 -> 150; with 1: 57049 rows of 73 66 -> 98, of [32768, 2048] 54 -> 64
  if (!stream && a.V / groups * a.slices < 4096)
    sum_runs<E, VEC, 1, false><<<grid(groups), kThreads, 0, s>>>(a, per);
  else if (stream)
    sum_runs<E, VEC, kTableRows, true><<<grid(groups * kTableRows), kThreads, 0, s>>>(a, per);
  else
    sum_runs<E, VEC, kTableRows, false><<<grid(groups * kTableRows), kThreads, 0, s>>>(a, per);
}

int vector_of(int dtype, int64_t D) {
  const int vec = dtype == 0 ? F32::VEC : BF16::VEC;
  return D >= vec ? vec : 1;
}

int check(const char *what, int dtype, int64_t M, int64_t V, int64_t D, float scale) {
  if (dtype != 0 && dtype != 2) return myelin::invalid("%s: unsupported dtype %d", what, dtype);
  if (M < 0 || V < 1 || D < 1) return myelin::invalid("%s: V and D must be positive, M not negative", what);
  if (M >= int64_t{1} << 30 || V >= int64_t{1} << 31 || D >= int64_t{1} << 31 || M * D >= int64_t{1} << 40 ||
      V * D >= int64_t{1} << 40)
    return myelin::invalid("%s: too many tokens or elements", what);
  if (!(__builtin_fabsf(scale) <= 3.402823466e38f)) return myelin::invalid("%s: scale must be finite", what);
  return MYELIN_OK;
}

}  // namespace

extern "C" int myelin_token_embedding(const int64_t *tokens, const void *weight, int dtype, int64_t ld, void *out,
                                      int64_t M, int64_t V, int64_t D, float scale, int64_t padding,
                                      myelin_stream_t stream) {
  const char *what = "token_embedding";
  if (int rc = check(what, dtype, M, V, D, scale)) return rc;
  if (V > 1 && ld < D) return myelin::invalid("%s: row stride below D", what);
  if (M == 0) return MYELIN_OK;
  if (!tokens || !weight || !out) return myelin::invalid("%s: null pointer", what);
  Args a{};
  a.tokens = tokens, a.from = weight, a.to = out, a.ld = ld, a.M = M, a.V = V, a.D = D;
  a.padding = padding, a.scale = scale;
  hipStream_t s = myelin::as_hip(stream);
  const bool vector = vector_of(dtype, D) > 1;
  if (dtype == 0)
    vector ? launch_lookup<F32, F32::VEC>(a, s) : launch_lookup<F32, 1>(a, s);
  else
    vector ? launch_lookup<BF16, BF16::VEC>(a, s) : launch_lookup<BF16, 1>(a, s);
  return myelin::launched(what);
}

extern "C" int64_t myelin_token_embedding_bwd_workspace_bytes(int64_t M, int64_t V, int64_t D) {
  if (M < 1 || V < 1 || D < 1) return 0;
  const int64_t f32 = layout_of(M, V, D, vector_of(0, D)).size, bf16 = layout_of(M, V, D, vector_of(2, D)).size;
  return f32 > bf16 ? f32 : bf16;
}

extern "C" int myelin_token_embedding_bwd(const int64_t *tokens, const void *grad_out, int dtype, void *grad_weight,
                                          int64_t M, int64_t V, int64_t D, float scale, int64_t padding,
                                          void *workspace, int64_t workspace_bytes, myelin_stream_t stream) {
  const char *what = "token_embedding_bwd";
  if (int rc = check(what, dtype, M, V, D, scale)) return rc;
  if (!grad_weight || (M > 0 && (!tokens || !grad_out))) return myelin::invalid("%s: null pointer", what);
  const Layout l = layout_of(M, V, D, vector_of(dtype, D));
  if (l.size) {
    if (!workspace || workspace_bytes < l.size)
      return myelin::invalid("%s: workspace of %lld bytes needed", what, static_cast<long long>(l.size));
    if (!myelin::aligned(workspace, 16)) return myelin::invalid("%s: workspace must be 16-byte aligned", what);
  }
  Args a{};
  a.tokens = tokens, a.from = grad_out, a.to = grad_weight, a.ld = D, a.M = M, a.V = V, a.D = D;
  a.padding = padding, a.scale = scale;
  hipStream_t s = myelin::as_hip(stream);
  const bool vector = vector_of(dtype, D) > 1;
  char *ws = static_cast<char *>(workspace);
  if (dtype == 0)
    vector ? launch_gradient<F32, F32::VEC>(a, l, ws, s) : launch_gradient<F32, 1>(a, l, ws, s);
  else
    vector ? launch_gradient<BF16, BF16::VEC>(a, l, ws, s) : launch_gradient<BF16, 1>(a, l, ws, s);
  return myelin::launched(what);
}
