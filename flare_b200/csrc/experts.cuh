// Host interface of the routed-expert kernels (experts.cu, grouped_gemm.cu).
#pragma once

#include "common.cuh"

namespace flare {

constexpr int kRouteMaxExperts = 512;  // per slot
constexpr int kRouteMaxTopK = 32;
constexpr int kRouteMaxGroups = 65536;  // every block of the last pass reads all groups' sizes

struct RouteParams {
  const void* logits;  // [S][B][E], inner stride 1
  int64_t stride_slot, stride_token;
  int dtype;
  int S, B, E, k;
  int* experts;    // [S*B, k]
  float* weights;  // [S*B, k]
  int* offsets;    // [S*E + 1]
  int* rows;       // [S*B*k]
  int* row_of;     // [S*B, k]
  int* work;       // route_work_ints() ints of scratch
};

struct RouteBwdParams {
  const int* experts;
  const float* weights;
  const float* dweights;
  int64_t T;
  int E, k;
  void* dlogits;  // [T, E] contiguous
  int dtype;
};

int64_t route_work_ints(int S, int B, int E);
void route_topk(const RouteParams& p, cudaStream_t s);
void route_topk_backward(const RouteBwdParams& p, cudaStream_t s);

struct SwigluParams {
  const void* x;  // [R, 2h], row pitch ldx
  int64_t ldx;
  void* y;  // [R, h] contiguous
  int64_t R, h;
  int dtype;
  uint8_t* q;      // [R, 2h] e4m3 (null: keep nothing)
  uint8_t* scale;  // [R, 2 * ceil(h / 32)] biased power-of-two exponents
  const void* dy;  // backward: [R, h], row pitch lddy
  int64_t lddy;
  void* dx;  // backward: [R, 2h] contiguous
};

void swiglu_forward(const SwigluParams& p, cudaStream_t s);
void swiglu_backward(const SwigluParams& p, cudaStream_t s);

struct CombineParams {
  const void* z;  // [R, N], row pitch ldz
  int64_t ldz;
  const int* row_of;     // [T, k]
  const float* weights;  // [T, k] or null (plain sum)
  int64_t T, R;
  int N, k;
  int dtype;
  int out_dtype;    // forward: of y; z's, or a 16-bit type when z is fp32
  void* y;          // [T, N] contiguous
  const void* dy;   // backward: [T, N], row pitch lddy
  int64_t lddy;
  void* dz;         // backward: [R, N] contiguous
  float* dw;        // backward: [T, k]
  const int* total;  // rows in use (the last offset)
};

void combine_forward(const CombineParams& p, cudaStream_t s);
void combine_backward(const CombineParams& p, cudaStream_t s);

// ------------------------------------------------------------ grouped products
enum GroupedMode : int { kGroupedFwd = 0, kGroupedDgrad = 1, kGroupedWgrad = 2 };
constexpr int kGroupedMaxGroups = 2048;

struct GroupedArgs {
  int mode;
  int dtype;  // kBF16 or kF16: x, w, dy and (fwd, dgrad) out
  const void* x;  // fwd, wgrad: [R, K] in group order; [x_rows, K] tokens when rows is set
  int64_t ldx, x_rows;
  const int* rows;  // [R] token of each row, or null (set for few rows only)
  const void* w;    // fwd, dgrad: [G, K, N]
  const void* dy;   // dgrad, wgrad: [R, N]
  int64_t lddy;
  const int* offsets;  // [G + 1]
  int G;
  int64_t R;
  int K, N;
  const void* bias;  // fwd: [G, N] of bias_dtype or null
  int bias_dtype;
  void* out;  // fwd [R, N], dgrad [R, K], wgrad [G, K, N]
  int out_dtype;  // fwd: dtype; dgrad: dtype or fp32; wgrad: any
  int accumulate;  // wgrad: fp32 out += result
  float* work;     // wgrad: grouped_work_floats() floats of scratch
  int* status;
  uint64_t timeout_ns;
};

void grouped_gemm(const GroupedArgs& a, cudaStream_t s);
int64_t grouped_work_floats(int G, int64_t R, int K, int N);
// Forward products of this many rows stream the weights with plain loads, and gather x themselves.
bool grouped_few_rows(int64_t rows);

struct GroupSumArgs {  // out[g, n] = sum over the group's rows of y[r, n]
  const void* y;
  int64_t ldy, R;
  int dtype;
  const int* offsets;
  int G, N;
  void* out;
  int out_dtype;
  int accumulate;
  float* work;  // group_sum_work_floats() floats of scratch
};
int64_t group_sum_work_floats(int G, int64_t R, int N);
void group_colsum(const GroupSumArgs& a, cudaStream_t s);

}  // namespace flare
