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

#include <type_traits>

#include "common.h"

namespace {

using myelin::kWave;

constexpr int kMaxDim = 128;

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

// Operand fragments of 16 x 16 products reduced over 32 indices: a lane l has
// row (or column) l % 16 and, with g = l / 16, the indices 4 g .. 4 g + 3 of
// each half.  A product's result has column l % 16 and rows 4 g .. 4 g + 3, so
// two results are a fragment of the transposed product as they are.
struct F32 {
  using T = float;
  using Frag = f32x8;
  static constexpr int VEC = 4;    // elements of 16 bytes
  static constexpr int C = 32;     // steps of a chunk
  static constexpr int PARTS = 1;   // fragments that hold an fp32 value
  static constexpr int HALVES = 1;  // that hold 16 bits of one
  // LDS rows 16 bytes past a multiple of 64 banks: 16 rows' 16-byte pieces are
  // on distinct banks, and 4 rows 4 apart
  static constexpr int PAD = 4;
  __device__ static int at(int row, int col, int ld) { return row * ld + col; }
  template <int N>
  __device__ static void parts(Frag (&part)[N], f32x4 a, f32x4 b) {
    part[0] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
  __device__ static void mma(f32x4 &acc, const Frag &a, const Frag &b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
  }
  __device__ static Frag row(const T *p) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 16);
    return {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
  // 0 if all are finite, else NaN
  __device__ static float zero_of(const Frag &a, float s) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s = __builtin_fmaf(a[i], 0.0f, s);
    return s;
  }
  // a lane's first row and column of a column block of 32 rows
  __device__ static int column_row(int lane) { return (lane >> 4) * 4; }
  __device__ static int column_at(int lane, int ld) { return lane & 15; }
  __device__ static Frag column(const T *p, int ld) {
    return {p[0], p[ld], p[2 * ld], p[3 * ld], p[16 * ld], p[17 * ld], p[18 * ld], p[19 * ld]};
  }
};
struct BF16 {
  using T = __bf16;
  using Frag = bf16x8;
  static constexpr int VEC = 8;
  static constexpr int C = 64;
  static constexpr int PARTS = 3;
  static constexpr int HALVES = 2;
  // LDS rows an odd multiple of 32 bytes long, which puts the transposing read's
  // 4 rows of 32 bytes on distinct banks (16 lanes take 128 bytes a cycle).  Of
  // 16 rows' 8-byte pieces two share a bank; exchanging the halves of each 32
  // bytes in rows 8 .. 15 keeps it at two.  (A permutation of 8-byte slots by
  // the row's low four bits has no conflicts either way, but its addresses cost
  // the registers that hold two workgroups to a CU: 2048 steps of 8 x 16 heads of
  // 128, training, 380 -> 625 us.)
  static constexpr int PAD = 16;
  __device__ static int at(int row, int col, int ld) { return row * ld + (col ^ (row & 8)); }
  // a and b in N parts, each the rounded rest of those before
  template <int N>
  __device__ static void parts(Frag (&part)[N], f32x4 a, f32x4 b) {
    float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
    for (int k = 0; k < N; ++k) {
      uint32_t bits[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2 x = {v[2 * i], v[2 * i + 1]};
        bits[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
        if (k + 1 < N) {
          v[2 * i] -= __builtin_bit_cast(float, bits[i] << 16);
          v[2 * i + 1] -= __builtin_bit_cast(float, bits[i] & 0xffff0000u);
        }
      }
      const u32x4 all = {bits[0], bits[1], bits[2], bits[3]};
      part[k] = __builtin_bit_cast(Frag, all);
    }
  }
  __device__ static void mma(f32x4 &acc, const Frag &a, const Frag &b) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
  }
  __device__ static Frag row(const T *p) {
    const bf16x4 a = *reinterpret_cast<const bf16x4 *>(p), b = *reinterpret_cast<const bf16x4 *>(p + 16);
    return {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
  __device__ static float zero_of(const Frag &a, float s) {
    const bf16x2 zero = {__bf16(0.0f), __bf16(0.0f)};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const bf16x2 two = {a[i], a[i + 1]};
      s = __builtin_amdgcn_fdot2_f32_bf16(two, zero, s, false);
    }
    return s;
  }
  // the transposing read: lane r of a group of 16 points at row r / 4 and
  // columns 4 (r % 4) .. + 3 of a 4 x 16 block, lane i receives column i
  __device__ static int column_row(int lane) { return (lane >> 4) * 4 + ((lane & 15) >> 2); }
  __device__ static int column_at(int lane, int ld) { return at(column_row(lane), (lane & 3) * 4, ld); }
  __device__ static Frag column(const T *p, int ld) {
    const bf16x4 a = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)((lds_void *)p)));
    const bf16x4 b =
        __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)((lds_void *)(p + 16 * ld))));
    return {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
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
  float s_scale, x_scale, c_scale;  // of a b^T, of a X, of the c that are added to X
  int reverse, o_f32;
};

struct Args {
  Problem p[3];
  int problems, slices;  // slices of the widest problem's columns
  const float *decay;
  const int32_t *lengths;
  int64_t T, B, H;
  int64_t segments, segment;  // of steps, whole chunks
  // [problems, slices, B * H, segments - 1] states, as the lanes hold them: what each
  // segment adds, or (joined) the states at their ends
  float *ends;
  int joined;
};

__device__ __forceinline__ int64_t steps_of(const Args &a, int64_t b) {
  if (!a.lengths) return a.T;
  const int64_t n = a.lengths[b];
  return n < 0 ? 0 : n > a.T ? a.T : n;
}

// d^n, by squaring in double: 0^0 = 1
__device__ __forceinline__ float power(float d, int64_t n) {
  double p = 1.0, s = d;
  for (; n > 0; n >>= 1) {
    if (n & 1) p *= s;
    s *= s;
  }
  return static_cast<float>(p);
}

// The recurrence by chunks of C steps.  With X the state before a chunk (after
// it, reversed), rows i, j of the chunk in the order of the recurrence and e =
// 1 - reverse:
//   o_i = x d^(i + e) a_i X + s sum_{j <= i} d^(i - j) (a_i . b_j) c_j
//   X'  = d^C X + c sum_j d^(C - j - e) b_j c_j^T
// with the scales (s, x, c) = (scale, scale, 1) where X is the state and (scale, 1,
// scale) where it is the state's gradient.
// A workgroup has one (problem, b, h), a slice of 16 columns of X for each of
// its NW waves and a segment of the steps; wave w has columns 16 w .. 16 w + 15
// of the slice in the accumulators of its products, which are
// also, rounded, the operand of the next chunk's a X.  The waves share out the
// 16 x 16 blocks of a b^T, scale them and put them into LDS.  Everything that
// reads a chunk's a, b and c comes before the barrier that ends those blocks,
// so the next chunk's rows, fetched meanwhile, are staged behind it: two
// barriers a chunk.  C is 64 for bf16 and 32 for fp32.
//
// Roundings to bf16: the scaled a b^T, multiplied by the bf16 c, and X where it is
// an operand to two parts each, 16 bits, so that the result has no error but its own
// rounding's (1.66e-3 of its norm; with one part of a b^T 1.85e-3, for 3 to 6 % less
// time); the scaled c of the state's sum to three, which are
// fp32's 24 bits, in the forward pass and in the gradients of a call with an
// initial state, and to two in the others, whose sums are only operands (2048
// steps of 8 x 16 heads of 128, training, 389 -> 363 us).  Which it is does not
// depend on the gradients that are asked for: nor do their bits.
//
// What bounds it: the waits between LDS reads, products and the two barriers of
// a chunk, at 16 waves to a CU.  32768 steps of 16 heads of 128, bf16: the main
// launch moves its 538 MB at about 3.4 TB/s (matrix cores busy 0.29 of the time,
// VALU 0.44, LDS 0.57, two fifths of that in conflicts), the one that forms the
// segments' states k and v at 3.9; 501 steps of 16 x 8 heads of 50 and 75, fp32,
// backward 126 us; 1024 of 4 x 16 heads of 128, fp32, training 317 us.
//
// WHOLE: all rows are whole 16-byte pieces.

template <class E>
constexpr int lds_bytes(int kt, int waves) {
  return E::C * (2 * (16 * kt + E::PAD) + 16 * waves + E::PAD + E::HALVES * (E::C + E::PAD) + 2) *
         static_cast<int>(sizeof(typename E::T));
}

// Registers bound how many waves a CU holds: with whole rows 8 waves to a
// workgroup fit 128, so that two of them share it, and 4 fit 168, for three where
// LDS holds them.
constexpr int waves_per_simd(int waves, int lds, bool whole) {
  return !whole ? 2 : waves == 8 ? 4 : 160 * 1024 / lds < 3 ? 2 : 3;
}

// EXACT: the sum of the state with all 24 bits.
template <class E, int KT, int NW, bool WHOLE, bool STATE_ONLY, bool EXACT>
__global__ __launch_bounds__(64 * NW)
__attribute__((amdgpu_waves_per_eu(waves_per_simd(NW, lds_bytes<E>(KT, NW), WHOLE)))) void chunked(Args args) {
  using T = typename E::T;
  using Frag = typename E::Frag;
  constexpr int C = E::C, VEC = E::VEC, CT = C / 16, CF = C / 32, KF = KT / 2;
  constexpr int NT = 64 * NW, KD = 16 * KT, VD = 16 * NW;             // threads, padded widths
  constexpr int LK = KD + E::PAD, LV = VD + E::PAD, LP = C + E::PAD;  // row lengths in LDS
  constexpr int PK = KD / VEC, PV = VD / VEC;                         // pieces of a row
  constexpr int NK = C * PK / NT, NV = C * PV / NT;                   // pieces of a thread
  static_assert(C * PK % NT == 0 && C * PV % NT == 0, "whole pieces");
  typedef T piece __attribute__((ext_vector_type(VEC)));
  typedef T four __attribute__((ext_vector_type(4)));
  __shared__ __attribute__((aligned(16))) T sa[STATE_ONLY ? 1 : C * LK];
  __shared__ __attribute__((aligned(16))) T sb[C * LK];
  __shared__ __attribute__((aligned(16))) T sc[C * LV];
  __shared__ __attribute__((aligned(16))) T sp[STATE_ONLY ? 1 : E::HALVES * C * LP];  // scaled a b^T
  __shared__ __attribute__((aligned(16))) float pw[C + 4];                // d^n
  __shared__ __attribute__((aligned(16))) float weight[C];                // of c_j in a whole chunk: c d^(C - j - e)

  // Workgroups go to the 8 XCDs in turn.  Those of one (b, h) and segment run on one
  // of them, whose L2 the problems and slices share; (b, h) and segments together
  // are dealt out evenly (32768 steps of 128, bf16, 1 head 57 us, 12 heads 193; by
  // (b, h) alone 127 and 267).
  const uint32_t id = blockIdx.x, rest = id >> 3;
  const int which = static_cast<int>(rest % args.problems);
  const Problem &p = args.p[which];
  const uint32_t heads = static_cast<uint32_t>(args.B * args.H), r1 = rest / args.problems;
  const int slice = static_cast<int>(r1 % args.slices), first = slice * VD;  // its first column
  const uint32_t unit = r1 / args.slices * 8 + (id & 7);
  const int64_t bh = __builtin_amdgcn_readfirstlane(unit % heads), seg = __builtin_amdgcn_readfirstlane(unit / heads);
  if (first >= p.VD) return;
  if (seg >= args.segments - (STATE_ONLY ? 1 : 0)) return;
  const int64_t b = bh / args.H, h = bh % args.H;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, l16 = lane & 15;
  const float d = args.decay[h];
  const int64_t n = steps_of(args, b);
  // (held in registers: arguments read in the loop cost it a scalar load each)
  const T *pa = static_cast<const T *>(p.a) + b * p.ab + (h / p.ga) * p.ah;
  const T *pb = static_cast<const T *>(p.b) + b * p.bb + (h / p.gb) * p.bh;
  const T *pc = static_cast<const T *>(p.c) + b * p.cb + (h / p.gc) * p.ch + first;
  const int64_t at = p.at, bt = p.bt, ct = p.ct, ot = p.ot;
  const int kd = p.KD, vd = p.VD - first < VD ? p.VD - first : VD;
  const bool o_f32 = p.o_f32;
  const float s_scale = p.s_scale, x_scale = p.x_scale;
  char *po = static_cast<char *>(p.o) + (b * p.ob + h * p.oh + first) * (o_f32 ? 4 : sizeof(T));
  const int64_t begin = seg * args.segment;
  const int64_t end = begin + args.segment < args.T ? begin + args.segment : args.T;
  const int64_t last = n < end ? n : end;  // the segment's steps end here
  const bool reverse = p.reverse;
  const bool active = 16 * w < vd;  // this wave has columns
  const int e = reverse ? 0 : 1;

  if (tid <= C) pw[tid] = power(d, tid);
  if (tid < C) weight[tid] = power(d, C - tid - e) * p.c_scale;
  if constexpr (!STATE_ONLY && E::HALVES == 1)  // blocks right of the diagonal stay zero
    for (int i = tid; i < C * LP; i += NT) sp[i] = T(0.0f);

  // Rows r0 .. r0 + C - 1 (in the recurrence's order) of one operand, `per`
  // pieces a row, in pieces or (not WHOLE) element by element, a row's to
  // consecutive lanes.  Rows past the last step and columns past the width are
  // zero; their loads go to the nearest element that there is (r0 < last, width
  // > 0).
  auto fetch = [&](auto per, auto &to, const T *from, int64_t stride, int width, int64_t r0) {
    constexpr int PER = decltype(per)::value;
    const int c = last - r0 < C ? static_cast<int>(last - r0) : C;
    if constexpr (WHOLE) {
      // a uniform address and 32-bit offsets, of rows back from the chunk's
      // last one if reversed
      constexpr int N = C * PER / NT;
      const int row0 = tid / PER, col = (tid % PER) * VEC;
      const T *base = from + (reverse ? n - r0 - c : r0) * stride;
      const int at = col < width ? col : 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        int row = i * (NT / PER) + row0;
        row = reverse ? c - 1 - row : row;
        row = row < 0 ? 0 : row >= c ? c - 1 : row;
        const uint32_t off = (static_cast<uint32_t>(row) * static_cast<uint32_t>(stride) + at) * sizeof(T);
        to[i] = *reinterpret_cast<const piece *>(reinterpret_cast<const char *>(base) + off);
      }
      if (c < C || width < PER * VEC) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int q = 0; q < VEC; ++q)
            to[i][q] = (col < width && i * (NT / PER) + row0 < c) ? to[i][q] : T(0.0f);
      }
    } else {
      // a lane's first address, the others whole rows on
      constexpr int ROW = PER * VEC, N = C * ROW / NT;
      const int row0 = tid / ROW, col = tid % ROW;
      const bool in = col < width;
      const int64_t step = reverse ? -stride : stride;
      const T *base = from + (reverse ? n - 1 - r0 : r0) * stride;
      const int at = in ? col : width - 1;
      if (c == C) {
        const int64_t mine = row0 * step + at;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const T v = base[i * (NT / ROW) * step + mine];
          to[i / VEC][i % VEC] = in ? v : T(0.0f);
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int row = i * (NT / ROW) + row0;
          const T v = base[(row < c ? row : c - 1) * step + at];
          to[i / VEC][i % VEC] = (in && row < c) ? v : T(0.0f);
        }
      }
    }
  };
  // The lane, counted where it is asked for: what is kept over the loop is spilled
  // in the 8-wave kernels, and its load back waits for the rows that are on their
  // way (2048 steps of 8 x 16 heads of 128, training, 372 us for 337).
  const auto lane_anew = []() {
    uint32_t all = ~0u;
    asm volatile("" : "+v"(all));
    return static_cast<int>(__builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0)));
  };
  auto stage = [&](auto per, T *to, const auto &from, int ld, int t) {
    constexpr int PER = decltype(per)::value, N = C * PER / NT;
    if constexpr (WHOLE) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        *reinterpret_cast<piece *>(to + E::at(i * (NT / PER) + t / PER, (t % PER) * VEC, ld)) = from[i];
    } else {
#pragma unroll
      for (int i = 0; i < N * VEC; ++i)
        to[E::at((i * NT + t) / (PER * VEC), t % (PER * VEC), ld)] = from[i / VEC][i % VEC];
    }
  };
  const std::integral_constant<int, PK> wide{};
  const std::integral_constant<int, PV> narrow{};
  piece na[STATE_ONLY ? 1 : NK], nb[NK], nc[NV];
  auto fetch_a = [&](int64_t r0) {
    if constexpr (!STATE_ONLY) fetch(wide, na, pa, at, kd, r0);
  };
  auto fetch_bc = [&](int64_t r0) {
    fetch(wide, nb, pb, bt, kd, r0);
    fetch(narrow, nc, pc, ct, vd, r0);
  };
  auto stage_all = [&]() {
    const int t = WHOLE ? 64 * w + lane_anew() : tid;
    if constexpr (!STATE_ONLY) stage(wide, sa, na, LK, t);
    stage(wide, sb, nb, LK, t);
    stage(narrow, sc, nc, LV, t);
  };
  if (begin < last) {
    fetch_a(begin);
    fetch_bc(begin);
  }

  // X: rows 16 t + 4 g + r, column 16 w + l16 of the slice
  f32x4 X[KT];
  const int col = first + 16 * w + l16;
  const int64_t state = bh * p.KD * p.VD;
  float *ends =
      args.ends + (((which * args.slices + slice) * args.B * args.H + bh) * (args.segments - 1)) * (KD * VD);
  const auto at_end = [&](int t) { return ((w * KT + t) * 64 + lane) * 4; };
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    X[t] = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (!STATE_ONLY) {
      if (seg > 0 && args.joined) {
        X[t] = *reinterpret_cast<const f32x4 *>(ends + (seg - 1) * (KD * VD) + at_end(t));
      } else if (p.s_in) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int k = 16 * t + 4 * g + r;
          if (k < p.KD && col < p.VD) X[t][r] = p.s_in[state + k * p.sk + col * p.sv];
        }
      }
    }
  }

  if constexpr (!STATE_ONLY) {
    if (!args.joined) {
      const float whole = power(d, args.segment);
      for (int64_t q = 0; q < seg; ++q) {
        const int64_t left = n - q * args.segment;
        const float f = left >= args.segment ? whole : left > 0 ? power(d, left) : 1.0f;
#pragma unroll
        for (int t = 0; t < KT; ++t)
          X[t] = f * X[t] + *reinterpret_cast<const f32x4 *>(ends + q * (KD * VD) + at_end(t));
      }
    }
  }

  // Blocks of 32 rows of X past the width.  fp32's products take long enough for
  // this to pay (100 steps of 4 x 4 heads of 32: 19.2 -> 17.0 us; 501 of 16 x 8
  // heads of 50 and 75, training, 351 -> 296 us); in the bf16 kernels the branches
  // cost more than the products, and in fp32's of whole rows past 64 they cost 114
  // spilled registers (1024 steps of 4 x 16 heads of 128, training, 317 -> 488 us).
  const auto past = [&](int f) { return E::PARTS == 1 && (KT == 4 || !WHOLE) && 32 * f >= kd; };

  // where a lane's fragments start: of row l16, and of a column block
  const int at_row = E::at(l16, 4 * g, 0), at_col = E::column_at(lane, 0);
  const int row_k = l16 * LK + at_row, col_k = E::column_row(lane) * LK + at_col;
  const int row_p = l16 * LP + at_row, col_v = E::column_row(lane) * LV + at_col;

  if (begin < last) stage_all();
  for (int64_t r0 = begin; r0 < last; r0 += C) {
    const int c = last - r0 < C ? static_cast<int>(last - r0) : C;  // steps of this chunk
    __syncthreads();
    if (r0 + C < last) fetch_bc(r0 + C);
    if constexpr (!STATE_ONLY) {
      // blocks (it, jt), jt <= it, of a b^T, transposed: rows j, column i
      for (int q = w; q < CT * (CT + 1) / 2; q += NW) {
        int it = 0, jt = q;
        while (jt > it) jt -= ++it;
        Frag x[KF], y[KF];
#pragma unroll
        for (int f = 0; f < KF; ++f) {
          if (past(f)) continue;
          x[f] = E::row(sb + 16 * jt * LK + 32 * f + row_k);
          y[f] = E::row(sa + 16 * it * LK + 32 * f + row_k);
        }
        f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f}, s1 = s;
#pragma unroll
        for (int f = 0; f < KF; f += 2) {
          if (!past(f)) E::mma(s, x[f], y[f]);
          if (!past(f + 1)) E::mma(s1, x[f + 1], y[f + 1]);
        }
        s = (s + s1) * s_scale;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int ij = 16 * (it - jt) + l16 - 4 * g - r;
          s[r] = ij >= 0 ? s[r] * pw[ij >= 0 ? ij : 0] : 0.0f;
        }
        const four z = __builtin_convertvector(s, four);
        T *to = sp + 16 * it * LP + 16 * jt + row_p;
        *reinterpret_cast<four *>(to) = z;
        if constexpr (E::HALVES == 2) {
          // the lower halves in a matrix of their own, but those of a diagonal block
          // that begins 32 steps in the block to its right, which is past the diagonal
          to += it == jt && it % 2 == 0 ? 16 : C * LP;
          *reinterpret_cast<four *>(to) = __builtin_convertvector(s - __builtin_convertvector(z, f32x4), four);
        }
      }
    }
    // (of two workgroups of 8 waves the one in its products goes first: 2048 steps
    // of 8 x 16 heads of 128, training, 369 -> 361 us)
    if constexpr (NW == 8) __builtin_amdgcn_s_setprio(1);
    Frag vf[CF];
    f32x4 o[CT];
    bool strange = false;  // c holds an infinity or a NaN
    if (active) {
#pragma unroll
      for (int f = 0; f < CF; ++f) vf[f] = E::column(sc + 32 * f * LV + 16 * w + col_v, LV);
      if constexpr (!STATE_ONLY) {
        // a X, transposed: rows are columns of the result, the column its row
        constexpr int XP = E::HALVES;
#pragma unroll
        for (int it = 0; it < CT; ++it) o[it] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int f = 0; f < KF; ++f) {
          if (past(f)) continue;
          Frag xf[XP];
          E::parts(xf, X[2 * f], X[2 * f + 1]);
          Frag af[CT];
#pragma unroll
          for (int it = 0; it < CT; ++it) af[it] = E::row(sa + 16 * it * LK + 32 * f + row_k);
#pragma unroll
          for (int k = 0; k < XP; ++k)
#pragma unroll
            for (int it = 0; it < CT; ++it) E::mma(o[it], xf[k], af[it]);
        }
#pragma unroll
        for (int it = 0; it < CT; ++it) o[it] *= pw[16 * it + l16 + e] * x_scale;
        float zero = 0.0f;
#pragma unroll
        for (int f = 0; f < CF; ++f) zero = E::zero_of(vf[f], zero);
        strange = __any(zero != 0.0f);
      }
      // (a's rows later than the others: the registers of a X are free here)
      if (r0 + C < last) fetch_a(r0 + C);
      // the state: c scaled by d^(c - j - e)
      const float fade = pw[c];
#pragma unroll
      for (int t = 0; t < KT; ++t) X[t] *= fade;
#pragma unroll
      for (int f = 0; f < CF; ++f) {
        f32x4 wt[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int j0 = 32 * f + 16 * half + 4 * g;
          if (c == C) {
            wt[half] = *reinterpret_cast<const f32x4 *>(weight + j0);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int x = C - c + j0 + r;  // (rows past the last step are zero)
              wt[half][r] = weight[x < C ? x : C - 1];
            }
          }
        }
        // (16 bits of X where it is only an operand)
        constexpr int VP = EXACT ? E::PARTS : E::HALVES;
        Frag vs[VP];
        f32x4 lo, hi;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          lo[r] = static_cast<float>(vf[f][r]) * wt[0][r];
          hi[r] = static_cast<float>(vf[f][4 + r]) * wt[1][r];
        }
        E::parts(vs, lo, hi);
        // (two blocks at a time, so that a product does not wait for the one before)
#pragma unroll
        for (int t0 = 0; t0 < KT; t0 += 2) {
          if (past(t0 / 2)) continue;
          Frag kf[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) kf[t] = E::column(sb + 32 * f * LK + 16 * (t0 + t) + col_k, LK);
#pragma unroll
          for (int k = 0; k < VP; ++k)
#pragma unroll
            for (int t = 0; t < 2; ++t) E::mma(X[t0 + t], kf[t], vs[k]);
        }
      }
    } else if (r0 + C < last) {
      fetch_a(r0 + C);
    }
    if constexpr (NW == 8) __builtin_amdgcn_s_setprio(0);
    __syncthreads();
    if (r0 + C < last) stage_all();
    if (!STATE_ONLY && active) {
      // A product takes 0 for the steps after its row: an infinity or a NaN in one of
      // them would reach the row as 0 * inf.  Where c has any they leave the product,
      // and rows from their step on become NaN.  (Told by the dot products
      // beside those of the state: behind the barrier 2048 steps of 8 x 16 heads of 128,
      // training, took 395 us for 362.)
      if (__builtin_expect(strange, 0)) {
        int ahead = l16 - 4 * g;  // (computed here: its operands would be kept over the loop)
        asm volatile("" : "+v"(ahead));
#pragma unroll
        for (int f = 0; f < CF; ++f) {
          Frag bad;
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const bool is = static_cast<float>(vf[f][x]) * 0.0f != 0.0f;
            bad[x] = T(is ? 1.0f : 0.0f);
            vf[f][x] = is ? T(0.0f) : vf[f][x];
          }
#pragma unroll
          for (int it = 2 * f; it < CT; ++it) {
            Frag upto;  // of the steps, those that row i sums
#pragma unroll
            for (int x = 0; x < 8; ++x)
              upto[x] = T(32 * f + 16 * (x / 4) + x % 4 - 16 * it <= ahead ? 1.0f : 0.0f);
            f32x4 found = {0.0f, 0.0f, 0.0f, 0.0f};
            E::mma(found, bad, upto);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[it][r] = found[r] > 0.0f ? __builtin_nanf("") : o[it][r];
          }
        }
      }
#pragma unroll
      for (int f = 0; f < CF; ++f)
#pragma unroll
        for (int it = 2 * f; it < CT; ++it) {
          const T *z = sp + 16 * it * LP + 32 * f + row_p;
          if constexpr (E::HALVES == 2) {
            if (it == 2 * f) {
              Frag twice = vf[f];
#pragma unroll
              for (int x = 0; x < 4; ++x) twice[4 + x] = twice[x];
              E::mma(o[it], twice, E::row(z));
              continue;
            }
            E::mma(o[it], vf[f], E::row(z + C * LP));
          }
          E::mma(o[it], vf[f], E::row(z));
        }
      // row i of the chunk, columns 16 w + 4 g .. + 3
      char *out = po + (reverse ? n - r0 - c : r0) * ot * (o_f32 ? 4 : sizeof(T));
      const int oc = 16 * w + 4 * (lane_anew() >> 4);
#pragma unroll
      for (int it = 0; it < CT; ++it) {
        const int i = 16 * it + l16;
        if (i >= c) continue;
        if constexpr (WHOLE) {
          // a uniform address and a 32-bit offset
          const uint32_t at = static_cast<uint32_t>(reverse ? c - 1 - i : i) * static_cast<uint32_t>(ot) + oc;
          if (oc >= vd) continue;
          if (o_f32)
            *reinterpret_cast<f32x4 *>(out + at * 4) = o[it];
          else
            *reinterpret_cast<four *>(out + at * sizeof(T)) = __builtin_convertvector(o[it], four);
        } else {
          const int64_t at = static_cast<int64_t>(reverse ? c - 1 - i : i) * ot + oc;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (oc + q >= vd) continue;
            if (o_f32)
              reinterpret_cast<float *>(out)[at + q] = o[it][q];
            else
              reinterpret_cast<T *>(out)[at + q] = static_cast<T>(o[it][q]);
          }
        }
      }
    }
  }
  if constexpr (STATE_ONLY) {
#pragma unroll
    for (int t = 0; t < KT; ++t) *reinterpret_cast<f32x4 *>(ends + seg * (KD * VD) + at_end(t)) = X[t];
  } else {
    // steps past the length give zeros
    for (int64_t r = last > begin ? last : begin; r < end; ++r) {
      for (int i = tid; i < vd; i += NT) {
        if (o_f32)
          reinterpret_cast<float *>(po)[r * ot + i] = 0.0f;
        else
          reinterpret_cast<T *>(po)[r * ot + i] = T(0.0f);
      }
    }
    if (p.s_out && seg == args.segments - 1 && col < p.VD) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int k = 16 * t + 4 * g + r;
          if (k < p.KD) p.s_out[state + k * p.sk + col * p.sv] = X[t][r];
        }
    }
  }
}

// Turns the segments' own contributions into the states at their ends: a thread
// an element of one (problem, b, h), segments read ahead of the chain.  Bound by
// memory: 31 segments of 16 heads of 128 x 128, 65 MB, 13 us (5 TB/s).
template <int KT, int NW>
__global__ __launch_bounds__(256) void join_segments(Args args) {
  constexpr int VD = 16 * NW, SIZE = 16 * KT * VD, AHEAD = 8;
  const int at = static_cast<int>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t bh = blockIdx.y;
  const Problem &p = args.p[blockIdx.z / args.slices];
  const int first = static_cast<int>(blockIdx.z % args.slices) * VD;
  const int r = at & 3, lane = (at >> 2) & 63, t = (at >> 8) % KT, block = (at >> 8) / KT;
  const int k = 16 * t + 4 * (lane >> 4) + r, col = first + 16 * block + (lane & 15);
  float *x = args.ends + ((blockIdx.z * args.B * args.H + bh) * (args.segments - 1)) * SIZE + at;
  const float d = args.decay[bh % args.H];
  const int64_t n = steps_of(args, bh / args.H);
  float s = (p.s_in && k < p.KD && col < p.VD) ? p.s_in[bh * p.KD * p.VD + k * p.sk + col * p.sv] : 0.0f;
  const float whole = power(d, args.segment);
  for (int64_t seg = 0; seg + 1 < args.segments; seg += AHEAD, x += AHEAD * SIZE) {
    const int m = args.segments - 1 - seg < AHEAD ? static_cast<int>(args.segments - 1 - seg) : AHEAD;
    float y[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) y[i] = i < m ? x[static_cast<int64_t>(i) * SIZE] : 0.0f;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int64_t left = n - (seg + i) * args.segment;
      const float f = left >= args.segment ? whole : left > 0 ? power(d, left) : 1.0f;
      s = __builtin_fmaf(f, s, y[i]);
      if (i < m) x[static_cast<int64_t>(i) * SIZE] = s;
    }
  }
}

// Sums the fp32 gradients of the query heads that share a key/value head, in
// their order (no atomics: the same bits on every run; 19 MB in 6.6 us): from [rows, Hk, group, D] to [rows, Hk, D].
template <class E>
__global__ __launch_bounds__(256) void sum_groups(const float *__restrict__ from, void *__restrict__ to, int64_t n,
                                                  int group, int D) {
  const int64_t i = myelin::block_id() * 256 + threadIdx.x;
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
// it once, which is nearly all that a step moves, both past the caches where the
// states are large: 256 x 16 states of 128 x 128 109 -> 99 us (5.5 TB/s).
template <class E, int VEC, int LX, bool STREAM>
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
      vec s = __builtin_nontemporal_load(reinterpret_cast<const vec *>(a.state + base + static_cast<int64_t>(r) * a.Dv));
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        s[i] = __builtin_fmaf(sk[r], c[i], d * s[i]);
        out[i] = __builtin_fmaf(sq[r], s[i], out[i]);
      }
      myelin::store<STREAM>(s, reinterpret_cast<vec *>(a.state_out + base + static_cast<int64_t>(r) * a.Dv));
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
  if (!vector) {
    if (a.Dv <= 32)
      step_kernel<E, 1, 32, false><<<grid, 256, 0, s>>>(a);
    else
      step_kernel<E, 1, 128, false><<<grid, 256, 0, s>>>(a);
    return;
  }
  const auto go = [&](auto stream) {
    constexpr bool STREAM = decltype(stream)::value;
    if (a.Dv <= 32)
      step_kernel<E, 4, 8, STREAM><<<grid, 256, 0, s>>>(a);
    else if (a.Dv <= 64)
      step_kernel<E, 4, 16, STREAM><<<grid, 256, 0, s>>>(a);
    else
      step_kernel<E, 4, 32, STREAM><<<grid, 256, 0, s>>>(a);
  };
  if (static_cast<int64_t>(grid) * a.Dk * a.Dv * 4 >= myelin::kStreamBytes)
    go(std::true_type{});
  else
    go(std::false_type{});
}

// How a call is cut, by its widest problem: the padded KD (16 kt), slices of 16
// nw columns, and the workgroups that the chip holds of it.  For bf16 of both
// widths past 64 one workgroup of 8 waves has all columns, since each forms the
// whole of a b^T; the others' smaller workgroups fill the chip more evenly (501
// steps of 16 x 8 heads of 50 and 75, fp32, training: 258 -> 220 us; 1021 of 8 x
// 16 heads of 64 and 96, bf16: 59 -> 56 us; but 2048 of 8 x 16 heads of 128, bf16,
// training: 380 -> 390 us), three to a CU where its LDS holds them, else two.
// (Element-wise kernels are counted as the others, though their registers hold
// two: whether rows are whole is not known where the workspace is asked for.)
struct Shape {
  int kt, nw, slices, places;
};
Shape shape_of(int dtype, int kd, int vd) {
  const bool all = dtype != 0 && kd > 64 && vd > 64;
  const int kt = kd <= 64 ? 4 : 8, nw = all ? 8 : 4;
  const int lds = dtype == 0 ? lds_bytes<F32>(kt, nw) : lds_bytes<BF16>(kt, nw);
  return {kt, nw, all ? 1 : (vd + 63) / 64, 256 * 4 * waves_per_simd(nw, lds, true) / nw};
}

// Segments of the time axis: as many as fill the workgroups' places,
// of 4 chunks at least.
void split(int64_t T, int64_t workgroups, int places, int C, int64_t *segments, int64_t *segment) {
  const int64_t chunks = (T + C - 1) / C;
  int64_t n = places / workgroups;
  if (n > chunks / 4) n = chunks / 4;
  if (n < 1) n = 1;
  const int64_t per = (chunks + n - 1) / n;
  *segment = per * C;
  *segments = (chunks + per - 1) / per;
}

int chunk_of(int dtype) { return dtype == 0 ? F32::C : BF16::C; }

// Floats of the segments' states.
int64_t ends_elems(int dtype, int64_t T, int64_t BH, int problems, Shape sh) {
  int64_t segments, segment;
  split(T, BH * problems * sh.slices, sh.places, chunk_of(dtype), &segments, &segment);
  return (segments - 1) * BH * problems * sh.slices * (16 * sh.kt) * (16 * sh.nw);
}

template <class E, int KT, int NW, bool WHOLE>
void launch_shape(const Args &a, bool exact, hipStream_t s) {
  const auto groups = [&](int64_t segments) {
    return static_cast<unsigned>((a.B * a.H * segments + 7) / 8 * 8 * a.problems * a.slices);
  };
  if (a.segments > 1) {
    // (the last segment's end is nobody's start)
    chunked<E, KT, NW, WHOLE, true, true><<<groups(a.segments - 1), 64 * NW, 0, s>>>(a);
    if (a.joined) {
      const dim3 grid(KT * NW, static_cast<unsigned>(a.B * a.H), a.problems * a.slices);
      join_segments<KT, NW><<<grid, 256, 0, s>>>(a);
    }
  }
  const unsigned grid = groups(a.segments);
  if constexpr (E::PARTS == 3) {
    if (!exact) {
      chunked<E, KT, NW, WHOLE, false, false><<<grid, 64 * NW, 0, s>>>(a);
      return;
    }
  }
  chunked<E, KT, NW, WHOLE, false, true><<<grid, 64 * NW, 0, s>>>(a);
}

template <class E>
void launch(Args &a, int problems, bool exact, float *ends, hipStream_t s) {
  int kd = 0, vd = 0;
  a.problems = problems;
  a.ends = ends;
  // rows of whole 16-byte pieces everywhere, and a chunk of them within 2^31 bytes
  bool whole = true;
  for (int i = 0; i < problems; ++i) {
    const Problem &p = a.p[i];
    kd = p.KD > kd ? p.KD : kd;
    vd = p.VD > vd ? p.VD : vd;
    const auto rows = [](const void *x, int64_t t, int64_t b, int64_t h, int width) {
      return width % E::VEC == 0 && t % E::VEC == 0 && b % E::VEC == 0 && h % E::VEC == 0 && myelin::aligned(x, 16) &&
             t >= 0 && t < (1 << 23);
    };
    whole = whole && rows(p.a, p.at, p.ab, p.ah, p.KD) && rows(p.b, p.bt, p.bb, p.bh, p.KD) &&
            rows(p.c, p.ct, p.cb, p.ch, p.VD) && rows(p.o, p.ot, p.ob, p.oh, p.VD);
  }
  const Shape sh = shape_of(sizeof(typename E::T) == 4 ? 0 : 2, kd, vd);
  a.slices = sh.slices;
  split(a.T, a.B * a.H * problems * a.slices, sh.places, E::C, &a.segments, &a.segment);
  // Where they are few each segment adds up those before it (2048 steps of 8 x 16
  // heads of 128, 4 segments: training 396 -> 381 us); where they are many that
  // reads more than joining them does (32768 steps of 16 heads, 32 segments: 253
  // against 242 us).
  a.joined = a.segments > 8;
  const auto go = [&](auto kt, auto waves) {
    constexpr int KT = decltype(kt)::value, NW = decltype(waves)::value;
    if (whole)
      launch_shape<E, KT, NW, true>(a, exact, s);
    else
      launch_shape<E, KT, NW, false>(a, exact, s);
  };
  const std::integral_constant<int, 4> four{};
  const std::integral_constant<int, 8> eight{};
  if (sh.kt == 4)
    go(four, four);
  else if (sh.nw == 4)
    go(eight, four);
  else if constexpr (sizeof(typename E::T) == 2)
    go(eight, eight);
}

int check(const char *what, int dtype, int64_t T, int64_t B, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv,
          float scale) {
  if (dtype != 0 && dtype != 2) return myelin::invalid("%s: unsupported dtype %d", what, dtype);
  if (T < 1 || B < 0 || H < 1 || Hk < 1) return myelin::invalid("%s: sizes must be positive", what);
  if (H % Hk) return myelin::invalid("%s: H must be a multiple of Hk", what);
  if (Dk < 1 || Dk > kMaxDim || Dv < 1 || Dv > kMaxDim)
    return myelin::invalid("%s: Dk and Dv must be in [1, %d]", what, kMaxDim);
  // (six workgroups of 256 threads for a head, fewer than 2^32 threads in all)
  if (T > 0x7fffffff || B > (1 << 21) / H) return myelin::invalid("%s: too many rows", what);
  if (!(scale > 0.0f) && !(scale < 0.0f)) return myelin::invalid("%s: scale must not be zero", what);
  if (scale - scale != 0.0f) return myelin::invalid("%s: scale must be finite", what);
  return MYELIN_OK;
}

int check_workspace(const char *what, const float *workspace, int64_t elems, int64_t need) {
  if (need && (!workspace || elems < need))
    return myelin::invalid("%s: workspace of %lld floats needed", what, static_cast<long long>(need));
  if (need && !myelin::aligned(workspace, 16)) return myelin::invalid("%s: workspace must be 16-byte aligned", what);
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
  p.s_scale = p.x_scale = p.c_scale = 1.0f;
  return p;
}

}  // namespace

extern "C" int64_t myelin_decay_attention_workspace_elems(int dtype, int64_t T, int64_t B, int64_t H, int64_t Hk,
                                                          int64_t Dk, int64_t Dv, int backward) {
  if (T < 1 || B < 1 || H < 1 || Hk < 1 || Dk < 1 || Dv < 1 || Dk > kMaxDim || Dv > kMaxDim) return 0;
  const int dk = static_cast<int>(Dk), dv = static_cast<int>(Dv);
  if (!backward) return ends_elems(dtype, T, B * H, 1, shape_of(dtype, dk, dv));
  // one launch for the three problems, of the wider shape (a launch for each
  // shape would need more segments to fill the chip: 501 steps of 16 x 8 heads
  // of 50 and 75, fp32, 290 against 263 us)
  const int widest = dk > dv ? dk : dv;
  return ends_elems(dtype, T, B * H, 3, shape_of(dtype, widest, widest)) + (H != Hk ? T * B * H * (Dk + Dv) : 0);
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
  p.s_scale = p.x_scale = scale;
  const int64_t need = myelin_decay_attention_workspace_elems(dtype, T, B, H, Hk, Dk, Dv, 0);
  if (int rc = check_workspace(what, workspace, workspace_elems, need)) return rc;
  if (dtype == 0)
    launch<F32>(a, 1, true, workspace, myelin::as_hip(stream));
  else
    launch<BF16>(a, 1, true, workspace, myelin::as_hip(stream));
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
  const int64_t need = myelin_decay_attention_workspace_elems(dtype, T, B, H, Hk, Dk, Dv, 1);
  if (int rc = check_workspace(what, workspace, workspace_elems, need)) return rc;
  const int group = static_cast<int>(H / Hk), dk = static_cast<int>(Dk), dv = static_cast<int>(Dv);
  const int64_t *qs = strides, *ks = strides + 3, *vs = strides + 6, *gs = strides + 9;
  Args a{};
  a.decay = decay, a.lengths = lengths, a.T = T, a.B = B, a.H = H;
  // dq = scale LA(do, v, k), from S_0 transposed
  Problem &pq = a.p[0], &pk = a.p[1], &pv = a.p[2];
  pq = problem(grad_out, gs, v, vs, k, ks, grad_q, B, H, dv, dk);
  pq.gb = pq.gc = group;
  pq.s_in = state, pq.sk = 1, pq.sv = Dv;
  // dk = RLA(v, do, scale q), dv = RLA(k, scale q, do), both from dS_T
  // (in the workspace the segments' states come first: they are read 16 bytes at a time)
  float *per_head = group > 1 ? workspace + need - T * B * H * (Dk + Dv) : nullptr;
  void *to_k = group > 1 ? static_cast<void *>(per_head) : grad_k;
  void *to_v = group > 1 ? static_cast<void *>(per_head + T * B * H * Dk) : grad_v;
  pk = problem(v, vs, grad_out, gs, q, qs, to_k, B, H, dv, dk);
  pk.ga = group;
  pk.s_in = grad_state_out, pk.sk = 1, pk.sv = Dv;
  pv = problem(k, ks, q, qs, grad_out, gs, to_v, B, H, dk, dv);
  pv.ga = group;
  pv.s_in = grad_state_out, pv.s_out = grad_state, pv.sk = Dv, pv.sv = 1;
  pq.s_scale = pk.s_scale = pv.s_scale = scale;
  pq.x_scale = pk.c_scale = pv.c_scale = scale;
  pk.reverse = pv.reverse = 1;
  pk.o_f32 = pv.o_f32 = group > 1;
  const hipStream_t s = myelin::as_hip(stream);
  if (dtype == 0)
    launch<F32>(a, 3, true, workspace, s);
  else
    launch<BF16>(a, 3, state || grad_state, workspace, s);
  if (group > 1) {
    for (int i = 0; i < 2; ++i) {
      const int D = i ? dv : dk;
      const int64_t n = T * B * Hk * D;
      const dim3 grid = myelin::grid_of((n + 255) / 256);
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
