// The embeddings of tokens, scaled, and the gradient of their table:
//
//   y_i = scale w[token_i]      dw[v] = scale sum_{i: token_i = v} dy_i
//
// A padding token's row is 0 and has no gradient; a token outside [0, V) gives a
// row of NaN and has none either: nothing is read out of range.  The sums are
// fp32, over the positions in order: the same bits on every run.

#include "elements.h"

namespace {

using myelin::BF16;
using myelin::F32;

struct Args {
  const int64_t *tokens;
  const void *from;  // the table; backward: dy [M, D]
  void *to;          // y [M, D]; backward: dw [V, D]
  int64_t ld, M, V, D, padding;
  float scale;
};

template <class E>
__global__ __launch_bounds__(256) void lookup(Args a) {
  using T = typename E::T;
  const int64_t at = myelin::block_id() * 256 + threadIdx.x;
  if (at >= a.M * a.D) return;
  const int64_t i = at / a.D, d = at - i * a.D, token = a.tokens[i];
  float v = 0.0f;
  if (token != a.padding)
    v = token < 0 || token >= a.V ? __builtin_nanf("")
                                  : E::get(static_cast<const T *>(a.from)[token * a.ld + d]) * a.scale;
  static_cast<T *>(a.to)[at] = E::put(v);
}

// a thread to an element of the table, over all positions
template <class E>
__global__ __launch_bounds__(256) void gradient(Args a) {
  using T = typename E::T;
  const int64_t at = myelin::block_id() * 256 + threadIdx.x;
  if (at >= a.V * a.D) return;
  const int64_t v = at / a.D, d = at - v * a.D;
  float sum = 0.0f;
  if (v != a.padding)
    for (int64_t i = 0; i < a.M; ++i)
      if (a.tokens[i] == v) sum += E::get(static_cast<const T *>(a.from)[i * a.D + d]);
  static_cast<T *>(a.to)[at] = E::put(sum * a.scale);
}

int check(const char *what, int dtype, int64_t M, int64_t V, int64_t D, float scale) {
  if (dtype != 0 && dtype != 2) return myelin::invalid("%s: unsupported dtype %d", what, dtype);
  if (M < 0 || V < 1 || D < 1) return myelin::invalid("%s: V and D must be positive, M not negative", what);
  if (M >= int64_t{1} << 31 || V >= int64_t{1} << 31 || D >= int64_t{1} << 31 || M * D >= int64_t{1} << 40 ||
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
  Args a{tokens, weight, out, ld, M, V, D, padding, scale};
  const dim3 grid = myelin::grid_of((M * D + 255) / 256);
  if (dtype == 0)
    lookup<F32><<<grid, 256, 0, myelin::as_hip(stream)>>>(a);
  else
    lookup<BF16><<<grid, 256, 0, myelin::as_hip(stream)>>>(a);
  return myelin::launched(what);
}

extern "C" int64_t myelin_token_embedding_bwd_workspace_bytes(int64_t M, int64_t V, int64_t D) { return 0; }

extern "C" int myelin_token_embedding_bwd(const int64_t *tokens, const void *grad_out, int dtype, void *grad_weight,
                                          int64_t M, int64_t V, int64_t D, float scale, int64_t padding,
                                          void *workspace, int64_t workspace_bytes, myelin_stream_t stream) {
  const char *what = "token_embedding_bwd";
  if (int rc = check(what, dtype, M, V, D, scale)) return rc;
  if (!grad_weight || (M > 0 && (!tokens || !grad_out))) return myelin::invalid("%s: null pointer", what);
  Args a{tokens, grad_out, grad_weight, D, M, V, D, padding, scale};
  const dim3 grid = myelin::grid_of((V * D + 255) / 256);
  if (dtype == 0)
    gradient<F32><<<grid, 256, 0, myelin::as_hip(stream)>>>(a);
  else
    gradient<BF16><<<grid, 256, 0, myelin::as_hip(stream)>>>(a);
  return myelin::launched(what);
}
