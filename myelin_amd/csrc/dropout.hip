// Dropout from a counter-based generator: the mask is a function of (seed,
// offset, element), so the backward pass computes it again and nothing of it is
// stored.
//
// Element i of the mask uses word i % 4 of Philox 4x32 with 10 rounds (Salmon,
// Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC11)
// at the counter (i / 4, offset), each 64 bits, low word first, and the key
// seed.  The element is kept where the word is >= threshold = floor(p 2^32).
//   y = x * scale (+ residual) where kept, 0 (+ residual) elsewhere
// in fp32, rounded once; a dropped NaN or infinity is dropped.
//
// Bound by memory: x and the residual are read past the caches (nontemporal),
// and large results written so: forward and backward of 26 M fp32 with a shared
// mask 83 -> 76 us (5.5 TB/s), of 38 M bf16 with a residual 74 -> 71.
//
// x is [steps, n]: one mask of n elements for all steps (a spiking layer keeps
// its mask over time), or steps = 1 and a mask element for each of x.

#include "common.h"

namespace {

struct F32 {
  using T = float;
  static constexpr int VEC = 4;
};
struct BF16 {
  using T = __bf16;
  static constexpr int VEC = 8;
};

struct Args {
  const void *x, *residual;
  void *y;
  int64_t steps, n;
  uint64_t threshold;
  uint32_t k0, k1;
  uint64_t offset;
  const int64_t *offset_at;  // added to offset, if given
  float scale;
  int64_t per;  // steps of a workgroup
};

// the four words of one counter
__device__ __forceinline__ void philox(uint64_t group, uint64_t offset, uint32_t k0, uint32_t k1, uint32_t out[4]) {
  uint32_t c0 = static_cast<uint32_t>(group), c1 = static_cast<uint32_t>(group >> 32);
  uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  out[0] = c0, out[1] = c1, out[2] = c2, out[3] = c3;
}

// A thread has VEC mask elements, for `per` steps of them.  VECTOR: rows start
// on multiples of 16 bytes and hold whole vectors.
template <class E, bool VECTOR, bool STREAM>
__global__ __launch_bounds__(256) void dropout_kernel(Args a) {
  using T = typename E::T;
  constexpr int VEC = E::VEC;
  typedef T vec __attribute__((ext_vector_type(VEC)));
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * VEC;
  if (i >= a.n) return;
  const uint64_t offset = a.offset + (a.offset_at ? static_cast<uint64_t>(*a.offset_at) : 0);
  uint32_t word[VEC];
#pragma unroll
  for (int g = 0; g < VEC / 4; ++g) philox(static_cast<uint64_t>(i) / 4 + g, offset, a.k0, a.k1, word + 4 * g);
  bool keep[VEC];
#pragma unroll
  for (int q = 0; q < VEC; ++q) keep[q] = word[q] >= a.threshold;
  const int64_t t0 = blockIdx.y * a.per, t1 = t0 + a.per < a.steps ? t0 + a.per : a.steps;
  const int m = a.n - i < VEC ? static_cast<int>(a.n - i) : VEC;
  for (int64_t t = t0; t < t1; ++t) {
    const T *x = static_cast<const T *>(a.x) + t * a.n + i;
    const T *r = a.residual ? static_cast<const T *>(a.residual) + t * a.n + i : nullptr;
    T *y = static_cast<T *>(a.y) + t * a.n + i;
    if (VECTOR || m == VEC) {
      vec v, b, o;
      if constexpr (VECTOR) {
        v = __builtin_nontemporal_load(reinterpret_cast<const vec *>(x));
        if (r) b = __builtin_nontemporal_load(reinterpret_cast<const vec *>(r));
      } else {
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          v[q] = x[q];
          if (r) b[q] = r[q];
        }
      }
#pragma unroll
      for (int q = 0; q < VEC; ++q) {
        float f = keep[q] ? static_cast<float>(v[q]) * a.scale : 0.0f;
        if (r) f += static_cast<float>(b[q]);
        o[q] = static_cast<T>(f);
      }
      if constexpr (VECTOR) {
        myelin::store<STREAM>(o, reinterpret_cast<vec *>(y));
      } else {
#pragma unroll
        for (int q = 0; q < VEC; ++q) y[q] = o[q];
      }
    } else {
#pragma unroll
      for (int q = 0; q < VEC; ++q) {
        if (q >= m) break;
        float f = keep[q] ? static_cast<float>(x[q]) * a.scale : 0.0f;
        if (r) f += static_cast<float>(r[q]);
        y[q] = static_cast<T>(f);
      }
    }
  }
}

template <class E>
int launch(Args &a, hipStream_t s) {
  // (fewer than 2^32 threads in x)
  const int64_t threads = (a.n + E::VEC - 1) / E::VEC, bx = (threads + 255) / 256;
  if (bx > 0xffffff) return myelin::invalid("counter_dropout: too many elements");
  // steps to a workgroup: as many as leave 2048 workgroups
  int64_t by = bx >= 2048 ? 1 : (2048 + bx - 1) / bx;
  if (by > a.steps) by = a.steps;
  a.per = (a.steps + by - 1) / by;
  by = (a.steps + a.per - 1) / a.per;
  const bool vector = a.n % E::VEC == 0 && myelin::aligned(a.x, 16) && myelin::aligned(a.y, 16) &&
                      myelin::aligned(a.residual, 16);
  const dim3 grid(static_cast<unsigned>(bx), static_cast<unsigned>(by));
  if (!vector)
    dropout_kernel<E, false, false><<<grid, 256, 0, s>>>(a);
  else if (a.steps * a.n * static_cast<int64_t>(sizeof(typename E::T)) >= myelin::kStreamBytes)
    dropout_kernel<E, true, true><<<grid, 256, 0, s>>>(a);
  else
    dropout_kernel<E, true, false><<<grid, 256, 0, s>>>(a);
  return myelin::launched("counter_dropout");
}

}  // namespace

extern "C" int myelin_counter_dropout(const void *x, int dtype, const void *residual, void *y, int64_t steps, int64_t n,
                                      int64_t threshold, float scale, int64_t seed, int64_t offset,
                                      const int64_t *offset_at, myelin_stream_t stream) {
  if (dtype != 0 && dtype != 2) return myelin::invalid("counter_dropout: unsupported dtype %d", dtype);
  if (steps < 0 || n < 0) return myelin::invalid("counter_dropout: negative size");
  if (threshold < 0 || threshold > (int64_t{1} << 32))
    return myelin::invalid("counter_dropout: threshold must be in [0, 2^32]");
  if (steps == 0 || n == 0) return MYELIN_OK;
  if (!x || !y) return myelin::invalid("counter_dropout: null pointer");
  Args a{x, residual, y, steps, n, static_cast<uint64_t>(threshold), static_cast<uint32_t>(seed),
         static_cast<uint32_t>(static_cast<uint64_t>(seed) >> 32), static_cast<uint64_t>(offset), offset_at, scale, 1};
  return dtype == 0 ? launch<F32>(a, myelin::as_hip(stream)) : launch<BF16>(a, myelin::as_hip(stream));
}
