// Routed experts around the grouped products: top-k routing with a stable
// counting sort, SwiGLU with an 8-bit checkpoint, and the combination of the
// experts' rows.  Everything here is bound by memory or, for a handful of
// tokens, by the launch; the products are in grouped_gemm.cu.
//
// Routing (tokens t = slot * B + b, groups slot * E + e):
//   chosen experts = the k largest logits, ties to the lowest expert, an expert
//   at -inf never; w_j = exp(l_j - l_0) / sum_i exp(l_i - l_0) in fp32.
//   Rows are the (token, choice) pairs sorted by group, within a group by token.
//   Every count is an integer, so the order does not depend on the schedule.
// SwiGLU: y = up * gate * sigmoid(gate).  The checkpoint holds up and gate in
//   e4m3 with one power-of-two scale per 32 columns of a row: dividing by a
//   power of two is exact, so the only rounding is the one to e4m3.
// Combination: y_t = sum_j w_tj z[row_of[t, j]], summed in order of j in fp32.
#include "experts.cuh"

#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

namespace flare {
namespace {

// ------------------------------------------------------------------ routing
constexpr int kSub = 256;  // tokens that are ranked together (one bit each)

// An unsigned key in the order of the logits: NaN above all, -0 equal to +0, -inf at kDeadKey.
// Adding +0 turns -0 into +0 and every NaN into the positive one, whose key is the largest.
constexpr uint32_t kDeadKey = 0x007FFFFFu;
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.f));
  return b ^ (static_cast<uint32_t>(static_cast<int>(b) >> 31) | 0x80000000u);
}

__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}

// LANES lanes share a token, each with NV of its experts (expert = v * LANES + lane).
template <typename T, int LANES, int NV>
__device__ __forceinline__ void route_load(const RouteParams& p, int slot, int b, bool live, T (&raw)[NV]) {
  const int sub = threadIdx.x % LANES;
  const T* row = static_cast<const T*>(p.logits) + slot * p.stride_slot + b * p.stride_token + sub;
#pragma unroll
  for (int v = 0; v < NV; ++v)
    if (live && v * LANES + sub < p.E) raw[v] = row[v * LANES];
}

template <typename T, int LANES, int NV>
__device__ __forceinline__ void route_pick(const RouteParams& p, int slot, int b, bool live_token, const T (&raw)[NV],
                                           int* hist) {
  const int sub = threadIdx.x % LANES;
  uint32_t key[NV];  // 0 is below every logit's key
#pragma unroll
  for (int v = 0; v < NV; ++v) key[v] = live_token && v * LANES + sub < p.E ? order_key(to_f32(raw[v])) : 0u;
  int my_e = -1;  // lane j of the token keeps choice j
  uint32_t my_k = kDeadKey;
  for (int j = 0; j < p.k; ++j) {
    uint32_t best = 0;
    int at = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v)  // the first of equal keys has the lowest expert
      if (key[v] > best) best = key[v], at = v * LANES + sub;
    if constexpr (LANES == 32) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, best);
      at = __reduce_min_sync(0xffffffffu, best == top ? at : 0x7fffffff);
      best = top;
    } else {
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) {
        const uint32_t ob = __shfl_xor_sync(0xffffffffu, best, o);
        const int oa = __shfl_xor_sync(0xffffffffu, at, o);
        if (ob > best || (ob == best && oa < at)) best = ob, at = oa;
      }
    }
    if (sub == j && best > kDeadKey) my_e = at, my_k = best;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (v * LANES + sub == at) key[v] = 0u;
  }
  const float my_v = key_value(my_k);
  const float top = __shfl_sync(0xffffffffu, my_v, 0, LANES);
  const float mine = my_e >= 0 ? expf(my_v - top) : 0.f;
  float sum = 0.f;
  for (int j = 0; j < p.k; ++j) sum += __shfl_sync(0xffffffffu, mine, j, LANES);
  if (live_token && sub < p.k) {
    const int64_t i = (static_cast<int64_t>(slot) * p.B + b) * p.k + sub;
    p.experts[i] = my_e;
    p.weights[i] = my_e >= 0 ? mine / sum : 0.f;
    if (my_e >= 0) atomicAdd(hist + my_e, 1);
  }
}

// The experts of tokens [b0, b1) of one slot; counts in hist[E] (shared memory, zeroed here).  The
// next token's logits are on their way while a token is picked.
template <typename T, int LANES, int NV>
__device__ __forceinline__ void route_pick_chunk(const RouteParams& p, int slot, int b0, int b1, int* hist) {
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  const int per = blockDim.x / LANES, mine = b0 + threadIdx.x / LANES;
  T raw[NV], next[NV];
  route_load<T, LANES, NV>(p, slot, mine, mine < b1, raw);
  for (int b = b0; b < b1; b += per) {  // block-uniform: the picks shuffle across whole warps
    const int at = mine + b - b0;
    route_load<T, LANES, NV>(p, slot, at + per, at + per < b1, next);
    route_pick<T, LANES, NV>(p, slot, at, at < b1, raw, hist);
#pragma unroll
    for (int v = 0; v < NV; ++v) raw[v] = next[v];
  }
  __syncthreads();
}

// Gives every chosen pair of tokens [b0, b1) its row: base[e] (shared) is the next free row of
// expert e.  The tokens of a sub-block that chose e are bits of mask[e], so a pair's rank is a
// population count: the order is that of the tokens whatever the threads do.
__device__ __forceinline__ void route_place_chunk(const RouteParams& p, int slot, int b0, int b1, int* base,
                                                  uint32_t* mask) {
  constexpr int W = kSub / 32;
  for (int s0 = b0; s0 < b1; s0 += kSub) {
    const int n = min(kSub, b1 - s0) * p.k;
    const int64_t t0 = static_cast<int64_t>(slot) * p.B + s0;
    for (int i = threadIdx.x; i < p.E * W; i += blockDim.x) mask[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int e = p.experts[t0 * p.k + i], b = i / p.k;
      if (e >= 0) atomicOr(&mask[e * W + (b >> 5)], 1u << (b & 31));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int e = p.experts[t0 * p.k + i], b = i / p.k;
      int row = -1;
      if (e >= 0) {
        row = base[e] + __popc(mask[e * W + (b >> 5)] & ((1u << (b & 31)) - 1u));
        for (int w = 0; w < (b >> 5); ++w) row += __popc(mask[e * W + w]);
        p.rows[row] = static_cast<int>(t0 + b);
      }
      p.row_of[t0 * p.k + i] = row;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
      int c = 0;
      for (int w = 0; w < W; ++w) c += __popc(mask[e * W + w]);
      base[e] += c;
    }
    __syncthreads();
  }
}

// Exclusive prefix of tot[E] in place by one warp; returns the total to every lane.
__device__ __forceinline__ int warp_exclusive(int* tot, int E) {
  const int lane = lane_id();
  int carry = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int c = e0 + lane < E ? tot[e0 + lane] : 0;
    int inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (e0 + lane < E) tot[e0 + lane] = carry + inc - c;
    carry += __shfl_sync(0xffffffffu, inc, 31);
  }
  return carry;
}

// Many tokens take three passes (131071 tokens of 128 fp32 logits, four choices: 41 + 5 + 8 us for 67
// MB read, 10 us at the measured copy; the gradient 13 us for 67 MB written).  The picks, four tokens
// to a warp, are bound by their instructions where they run (ncu: stalls are "not selected" and the
// math pipe, memory waits a tenth of these; 60 % of issue slots, since 512 blocks are three or four
// to an SM).  With the prefix over all blocks' counts in every block of a second pass instead of a
// pass of its own, the placing alone took 42 us.
// Pass 1: experts and weights of every token of a sub-block (block = slot * chunks + chunk), and
// its counts: work[slot][chunk][E].
template <typename T, int LANES, int NV>
__global__ void __launch_bounds__(256) route_pick_kernel(RouteParams p, int chunks) {
  __shared__ int hist[kRouteMaxExperts];
  const int slot = blockIdx.x / chunks, c = blockIdx.x % chunks;
  route_pick_chunk<T, LANES, NV>(p, slot, c * kSub, min(p.B, (c + 1) * kSub), hist);
  int* out = p.work + static_cast<int64_t>(blockIdx.x) * p.E;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) out[e] = hist[e];
}

// Pass 2: along the chunks of a slot, counts become the rows of the same expert before the chunk;
// their sum goes to work[S * chunks * E + group].  Block = 32 experts of a slot; thread y takes a
// 32nd of the chunks.
__global__ void __launch_bounds__(1024) route_scan_kernel(RouteParams p, int chunks) {
  __shared__ int part[32][33];
  const int e = blockIdx.y * 32 + threadIdx.x, slot = blockIdx.x;
  const int per = (chunks + 31) / 32, q0 = min(chunks, static_cast<int>(threadIdx.y) * per), q1 = min(chunks, q0 + per);
  int* col = p.work + static_cast<int64_t>(slot) * chunks * p.E + e;
  int mine = 0;
  if (e < p.E) {
#pragma unroll 4
    for (int q = q0; q < q1; ++q) mine += col[static_cast<int64_t>(q) * p.E];
  }
  part[threadIdx.y][threadIdx.x] = mine;
  __syncthreads();
  int run = 0;
  for (int y = 0; y < static_cast<int>(threadIdx.y); ++y) run += part[y][threadIdx.x];
  if (e >= p.E) return;
#pragma unroll 4
  for (int q = q0; q < q1; ++q) {
    const int64_t i = static_cast<int64_t>(q) * p.E;
    const int v = col[i];
    col[i] = run;
    run += v;
  }
  if (threadIdx.y == 31) p.work[(static_cast<int64_t>(p.S) * chunks + slot) * p.E + e] = run;
}

// Pass 3: a sub-block's first row of each expert = rows of the groups before + of the chunks
// before; then its pairs' rows.
__global__ void __launch_bounds__(256) route_place_kernel(RouteParams p, int chunks) {
  __shared__ int base[kRouteMaxExperts];
  __shared__ uint32_t mask[kRouteMaxExperts * (kSub / 32)];
  __shared__ int before, total;
  const int slot = blockIdx.x / chunks, c = blockIdx.x % chunks;
  const int* counts = p.work + static_cast<int64_t>(p.S) * chunks * p.E;
  if (threadIdx.x == 0) before = total = 0;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) base[e] = counts[slot * p.E + e];
  __syncthreads();
  int bsum = 0, tsum = 0;
  for (int i = threadIdx.x; i < p.S * p.E; i += blockDim.x) {
    const int v = counts[i];
    tsum += v;
    if (i < slot * p.E) bsum += v;
  }
  if (bsum) atomicAdd(&before, bsum);
  if (tsum) atomicAdd(&total, tsum);
  if (threadIdx.x < 32) warp_exclusive(base, p.E);
  __syncthreads();
  const int* mine = p.work + static_cast<int64_t>(blockIdx.x) * p.E;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    const int first = before + base[e];
    if (c == 0) p.offsets[slot * p.E + e] = first;
    base[e] = first + mine[e];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.offsets[p.S * p.E] = total;
  const int64_t R = static_cast<int64_t>(p.S) * p.B * p.k;
  for (int64_t i = total + static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < R;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x)
    p.rows[i] = -1;
  __syncthreads();
  route_place_chunk(p, slot, c * kSub, min(p.B, (c + 1) * kSub), base, mask);
}

// Both passes in one block: one slot of at most kRouteOneBlock tokens.
constexpr int kRouteOneBlock = 512;
template <typename T, int LANES, int NV>
__global__ void __launch_bounds__(512) route_one_kernel(RouteParams p) {
  __shared__ int hist[kRouteMaxExperts];
  __shared__ uint32_t mask[kRouteMaxExperts * (kSub / 32)];
  __shared__ int total;
  route_pick_chunk<T, LANES, NV>(p, 0, 0, p.B, hist);
  if (threadIdx.x < 32) {
    const int t = warp_exclusive(hist, p.E);
    if (threadIdx.x == 0) total = t;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) p.offsets[e] = hist[e];
  if (threadIdx.x == 0) p.offsets[p.E] = total;
  for (int i = total + threadIdx.x; i < p.B * p.k; i += blockDim.x) p.rows[i] = -1;
  __syncthreads();
  route_place_chunk(p, 0, 0, p.B, hist, mask);
}

template <typename T, int LANES, int NV>
void route_launch(const RouteParams& p, cudaStream_t s) {
  if (p.S == 1 && p.B <= kRouteOneBlock) {
    // enough threads for every token at once, 512 at most
    const int threads = std::min(512, std::max(64, ceil_div(static_cast<int64_t>(p.B) * LANES, 32) * 32));
    route_one_kernel<T, LANES, NV><<<1, threads, 0, s>>>(p);
    FLARE_CUDA_CHECK(cudaGetLastError());
    count_launch();
    return;
  }
  const int chunks = ceil_div(p.B, kSub);
  route_pick_kernel<T, LANES, NV><<<p.S * chunks, 256, 0, s>>>(p, chunks);
  FLARE_CUDA_CHECK(cudaGetLastError());
  route_scan_kernel<<<dim3(p.S, ceil_div(p.E, 32)), dim3(32, 32), 0, s>>>(p, chunks);
  FLARE_CUDA_CHECK(cudaGetLastError());
  route_place_kernel<<<p.S * chunks, 256, 0, s>>>(p, chunks);
  FLARE_CUDA_CHECK(cudaGetLastError());
  count_launch(3);
}

template <typename T>
void route_typed(const RouteParams& p, cudaStream_t s) {
  // Eight lanes a token where they can hold its choices: four tokens share each instruction
  // (131071 x 128 fp32, k = 4: 97 us with 32 lanes a token).
  if (p.k <= 8 && p.E <= 256) {
    if (p.E <= 8) route_launch<T, 8, 1>(p, s);
    else if (p.E <= 16) route_launch<T, 8, 2>(p, s);
    else if (p.E <= 32) route_launch<T, 8, 4>(p, s);
    else if (p.E <= 64) route_launch<T, 8, 8>(p, s);
    else if (p.E <= 128) route_launch<T, 8, 16>(p, s);
    else route_launch<T, 8, 32>(p, s);
  } else if (p.E <= 64) {
    route_launch<T, 32, 2>(p, s);
  } else if (p.E <= 256) {
    route_launch<T, 32, 8>(p, s);
  } else {
    route_launch<T, 32, 16>(p, s);
  }
}

// ----------------------------------------------------------------- vectors
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_f(const T* p, float (&f)[N]) {
  const Vec<T, N> u = *reinterpret_cast<const Vec<T, N>*>(p);
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {  // in pairs
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        f[i] = __uint_as_float(w[i / 2] << 16);
        f[i + 1] = __uint_as_float(w[i / 2] & 0xFFFF0000u);
      } else {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(w + i / 2));
        f[i] = t.x;
        f[i + 1] = t.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_f32(u.v[i]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_f(T* p, const float (&f)[N]) {
  Vec<T, N> u;
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(f[i], f[i + 1]);
        w[i / 2] = *reinterpret_cast<const uint32_t*>(&t);
      } else {
        const __half2 t = __floats2half2_rn(f[i], f[i + 1]);
        w[i / 2] = *reinterpret_cast<const uint32_t*>(&t);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) u.v[i] = from_f32<T>(f[i]);
  }
  *reinterpret_cast<Vec<T, N>*>(p) = u;
}

// d logits[t, e] = w_j (dw_j - sum_i w_i dw_i) where choice j of t is e, else 0.  A block takes
// kBwdTokens tokens: it writes zeros over their rows in 16-byte stores, then a thread works out
// one token's k values and puts them in place (the barrier orders the two).
constexpr int kBwdTokens = 128;
template <typename T>
__global__ void __launch_bounds__(kBwdTokens) route_bwd_kernel(RouteBwdParams p) {
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kBwdTokens;
  const int n = static_cast<int>(min(static_cast<long long>(kBwdTokens), static_cast<long long>(p.T - t0)));
  T* out = static_cast<T*>(p.dlogits) + t0 * p.E;  // 16-byte aligned: kBwdTokens is a multiple of 8
  constexpr int per = 16 / sizeof(T);
  const int total = n * p.E, whole = total / per;
  for (int i = threadIdx.x; i < whole; i += kBwdTokens) reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
  for (int i = whole * per + threadIdx.x; i < total; i += kBwdTokens) out[i] = from_f32<T>(0.f);
  __syncthreads();
  if (static_cast<int>(threadIdx.x) >= n) return;
  const int64_t i0 = (t0 + threadIdx.x) * p.k;
  float dot = 0.f;
  for (int j = 0; j < p.k; ++j) dot += p.experts[i0 + j] >= 0 ? p.weights[i0 + j] * p.dweights[i0 + j] : 0.f;
  for (int j = 0; j < p.k; ++j) {
    const int e = p.experts[i0 + j];
    if (e >= 0) out[threadIdx.x * p.E + e] = from_f32<T>(p.weights[i0 + j] * (p.dweights[i0 + j] - dot));
  }
}

template <typename T>
void route_bwd_launch(const RouteBwdParams& p, cudaStream_t s) {
  route_bwd_kernel<T><<<static_cast<int>((p.T + kBwdTokens - 1) / kBwdTokens), kBwdTokens, 0, s>>>(p);
  FLARE_CUDA_CHECK(cudaGetLastError());
  count_launch();
}

// ------------------------------------------------------------------ SwiGLU
constexpr int kGroupCols = 32;

// sigmoid of gates from kTailGate up: outputs of 16 bits lose nothing to the fast exponential (2 ulp
// of fp32 and more for large arguments) and division; fp32 outputs take the accurate ones.
template <bool kFast>
__device__ __forceinline__ float sigmoid_f(float g) {
  if constexpr (kFast) return __fdividef(1.f, 1.f + __expf(-g));
  return 1.f / (1.f + expf(-g));
}

// Below about -87, exp(-gate) passes fp32's range (and the fast division gives 0 for divisors above
// 2^126), but up and dy can be as large as the sigmoid is small: with up = 1e36 and a gate of -89 the
// result is -0.2.  Such gates are rare; their products are taken in 64 bits, value by value from
// memory and over what the vector store wrote (with the operands kept in registers for it, the
// backward kernel took 72 of them instead of 48, and a pass of 131072 x 2 x 2048 bf16 844 us instead
// of 737).  sigmoid(g) is exp(g) there (1 + exp(g) rounds to 1), and exp(g) the eighth power of
// expf(g / 8), which is a normal number down to -698: off by 8 ulp of fp32 at most.
constexpr float kTailGate = -80.f;
__device__ __forceinline__ double tail_sigmoid(float g) {
  const double e = expf(0.125f * g), e2 = e * e, e4 = e2 * e2;
  return e4 * e4;
}
template <int N>
__device__ __forceinline__ bool has_tail(const float (&gate)[N]) {
  float low = gate[0];
#pragma unroll
  for (int i = 1; i < N; ++i) low = fminf(low, gate[i]);  // fminf passes over NaN
  return low < kTailGate;
}

// The scale exponent of a group whose largest finite magnitude is `top`: the largest value lands
// in (224, 448], 448 being e4m3's largest.  -126 keeps the scale's inverse finite.
__device__ __forceinline__ int scale_exponent(float top) {
  const uint32_t b = __float_as_uint(top);
  const int x = static_cast<int>(b >> 23) - 127;  // floor(log2(top)), or -127 below 2^-126
  return max((b & 0x007FFFFFu) <= 0x00600000u ? x - 8 : x - 7, -126);
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Largest finite magnitude of N values (NaN and infinities say nothing about the others); inf is
// set where there is an infinity.
template <int N>
__device__ __forceinline__ float finite_top(const float (&v)[N], bool& inf) {
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) t = fmaxf(t, fabsf(v[i]));  // fmaxf passes over NaN
  inf = t == INFINITY;
  if (inf) {
    t = 0.f;
    for (int i = 0; i < N; ++i) t = fmaxf(t, fabsf(v[i]) < INFINITY ? fabsf(v[i]) : 0.f);
  }
  return t;
}

// e4m3 of v * inv; infinities become NaN (e4m3 has no infinity), NaN stays.
template <int N>
__device__ __forceinline__ void pack_e4m3(const float (&v)[N], float inv, bool inf, uint8_t* out) {
  Vec<uint8_t, N> u;
  if constexpr (N == 1) {
    u.v[0] = static_cast<uint8_t>(__nv_cvt_float_to_fp8(v[0] * inv, __NV_SATFINITE, __NV_E4M3));
  } else {
    uint16_t* w = reinterpret_cast<uint16_t*>(&u);
#pragma unroll
    for (int i = 0; i < N; i += 2)
      w[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(v[i] * inv, v[i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
  }
  if (inf) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (fabsf(v[i]) == INFINITY) u.v[i] = 0x7F;
  }
  *reinterpret_cast<Vec<uint8_t, N>*>(out) = u;
}
template <int N>
__device__ __forceinline__ void unpack_e4m3(const uint8_t* in, float scale, float (&v)[N]) {
  const Vec<uint8_t, N> u = *reinterpret_cast<const Vec<uint8_t, N>*>(in);
  if constexpr (N == 1) {
    v[0] = __half2float(__half(__nv_cvt_fp8_to_halfraw(u.v[0], __NV_E4M3))) * scale;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint16_t two = reinterpret_cast<const uint16_t*>(&u)[i / 2];
      const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
      v[i] = f.x * scale;
      v[i + 1] = f.y * scale;
    }
  }
}

// Bound by memory and, nearly as much, by the instructions of the sigmoid and the rounding, although
// conversions go in pairs (ncu, 32768 rows: 77 and 73 % of issue slots, DRAM at 65 %, stalls waiting
// for memory first).  131072 rows of 2 x 2048 bf16 with the checkpoint: forward 358 to 380 us, backward
// 370 to 390 us, 2.16 GB each (5.5 to 6.0 TB/s, 0.85 to 0.92 of the measured copy); without it 243
// (1.61 GB) and 433 us (2.68 GB).  Rows that do not start on 16 bytes go element by element: 131072
// rows of 2 x 2047 take 1129 and 972 us with the checkpoint, 631 and 955 us without.
// A thread owns N consecutive columns of up and the same of gate; kGroupCols / N lanes share a
// scale.  A row's columns are padded to whole scale groups (`cols` chunks of N), short rows share
// a block.  One pass: x is read once, y and the checkpoint are written once.
struct RowTiling {
  int cols;  // chunks per row, padded to whole scale groups
  int rows;  // rows of one block step (1 where a row fills the block)
};

template <typename T, int N, bool kKeep>
__global__ void __launch_bounds__(256) swiglu_fwd_kernel(SwigluParams p, RowTiling t) {
  constexpr int GL = kGroupCols / N;
  const int r0 = t.rows > 1 ? threadIdx.x / t.cols : 0;
  const int c0 = t.rows > 1 ? threadIdx.x % t.cols : threadIdx.x;
  const int64_t groups = (p.h + kGroupCols - 1) / kGroupCols;
  for (int64_t rb = static_cast<int64_t>(blockIdx.x) * t.rows; rb < p.R; rb += static_cast<int64_t>(gridDim.x) * t.rows) {
    const int64_t r = rb + r0;
    const bool row_in = r0 < t.rows && r < p.R;
    for (int cb = 0; cb < t.cols; cb += 256) {  // block-uniform: the scales are shared by shuffles
      const int c = c0 + cb;
      const int64_t col = static_cast<int64_t>(c) * N;
      const bool in = row_in && col < p.h;
      float up[N], gate[N];
#pragma unroll
      for (int i = 0; i < N; ++i) up[i] = gate[i] = 0.f;
      if (in) {
        const T* x = static_cast<const T*>(p.x) + r * p.ldx + col;
        load_f<T, N>(x, up);
        load_f<T, N>(x + p.h, gate);
        float y[N];
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = up[i] * (gate[i] * sigmoid_f<sizeof(T) == 2>(gate[i]));
        T* out = static_cast<T*>(p.y) + r * p.h + col;
        store_f<T, N>(out, y);
        if (has_tail(gate)) {
#pragma unroll 1
          for (int i = 0; i < N; ++i) {
            const float g = to_f32(x[p.h + i]);
            if (g < kTailGate) out[i] = from_f32<T>(static_cast<float>(to_f32(x[i]) * (g * tail_sigmoid(g))));
          }
        }
      }
      if constexpr (kKeep) {
        bool iu, ig;
        float tu = finite_top<N>(up, iu), tg = finite_top<N>(gate, ig);
#pragma unroll
        for (int o = GL / 2; o > 0; o >>= 1) {
          tu = fmaxf(tu, __shfl_xor_sync(0xffffffffu, tu, o));
          tg = fmaxf(tg, __shfl_xor_sync(0xffffffffu, tg, o));
        }
        if (in) {
          const int eu = scale_exponent(tu), eg = scale_exponent(tg);
          uint8_t* q = p.q + r * 2 * p.h + col;
          pack_e4m3<N>(up, exp2_int(-eu), iu, q);
          pack_e4m3<N>(gate, exp2_int(-eg), ig, q + p.h);
          if (c % GL == 0) {
            uint8_t* sc = p.scale + r * 2 * groups + c / GL;
            sc[0] = static_cast<uint8_t>(eu + 127);
            sc[groups] = static_cast<uint8_t>(eg + 127);
          }
        }
      }
    }
  }
}

// d up = dy * gate * s, d gate = dy * up * s * (1 + gate * (1 - s)), s = sigmoid(gate), from x
// itself or from the values that the checkpoint stands for.  The factors of s come first: a large
// negative gate makes them 0 before the others can overflow.  Five blocks an SM: 48 registers.
template <typename T, int N, bool kKeep>
__global__ void __launch_bounds__(256, 5) swiglu_bwd_kernel(SwigluParams p, RowTiling t) {
  constexpr int GL = kGroupCols / N;
  const int r0 = t.rows > 1 ? threadIdx.x / t.cols : 0;
  const int c0 = t.rows > 1 ? threadIdx.x % t.cols : threadIdx.x;
  const int64_t groups = (p.h + kGroupCols - 1) / kGroupCols;
  for (int64_t rb = static_cast<int64_t>(blockIdx.x) * t.rows; rb < p.R; rb += static_cast<int64_t>(gridDim.x) * t.rows) {
    const int64_t r = rb + r0;
    if (r0 >= t.rows || r >= p.R) continue;
    for (int c = c0; c < t.cols; c += 256) {
      const int64_t col = static_cast<int64_t>(c) * N;
      if (col >= p.h) continue;
      float up[N], gate[N], dy[N], du[N], dg[N];
      if constexpr (kKeep) {
        const uint8_t* q = p.q + r * 2 * p.h + col;
        const uint8_t* sc = p.scale + r * 2 * groups + c / GL;
        unpack_e4m3<N>(q, exp2_int(static_cast<int>(sc[0]) - 127), up);
        unpack_e4m3<N>(q + p.h, exp2_int(static_cast<int>(sc[groups]) - 127), gate);
      } else {
        const T* x = static_cast<const T*>(p.x) + r * p.ldx + col;
        load_f<T, N>(x, up);
        load_f<T, N>(x + p.h, gate);
      }
      load_f<T, N>(static_cast<const T*>(p.dy) + r * p.lddy + col, dy);
      const bool tail = has_tail(gate);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float s = sigmoid_f<sizeof(T) == 2>(gate[i]);
        du[i] = dy[i] * (gate[i] * s);
        dg[i] = dy[i] * (up[i] * (s * (1.f + gate[i] * (1.f - s))));
      }
      T* dx = static_cast<T*>(p.dx) + r * 2 * p.h + col;
      store_f<T, N>(dx, du);
      store_f<T, N>(dx + p.h, dg);
      if (tail) {
#pragma unroll 1
        for (int i = 0; i < N; ++i) {
          float u[1], g[1];
          if constexpr (kKeep) {
            const uint8_t* q = p.q + r * 2 * p.h + col + i;
            const uint8_t* sc = p.scale + r * 2 * groups + c / GL;
            unpack_e4m3<1>(q, exp2_int(static_cast<int>(sc[0]) - 127), u);
            unpack_e4m3<1>(q + p.h, exp2_int(static_cast<int>(sc[groups]) - 127), g);
          } else {
            const T* x = static_cast<const T*>(p.x) + r * p.ldx + col + i;
            load_f<T, 1>(x, u);
            load_f<T, 1>(x + p.h, g);
          }
          if (g[0] < kTailGate) {
            const double d = to_f32(static_cast<const T*>(p.dy)[r * p.lddy + col + i]), s = tail_sigmoid(g[0]);
            dx[i] = from_f32<T>(static_cast<float>(d * (g[0] * s)));
            dx[p.h + i] = from_f32<T>(static_cast<float>(d * (u[0] * (s * (1.0 + g[0])))));
          }
        }
      }
    }
  }
}

template <typename T, int N>
void swiglu_launch(const SwigluParams& p, bool backward, cudaStream_t s) {
  constexpr int GL = kGroupCols / N;
  RowTiling t;
  t.cols = static_cast<int>((p.h + kGroupCols - 1) / kGroupCols) * GL;
  t.rows = t.cols <= 128 ? 256 / t.cols : 1;
  const int grid = static_cast<int>(std::min<int64_t>((p.R + t.rows - 1) / t.rows, 148 * 64));
  if (!backward) {
    if (p.q != nullptr) swiglu_fwd_kernel<T, N, true><<<grid, 256, 0, s>>>(p, t);
    else swiglu_fwd_kernel<T, N, false><<<grid, 256, 0, s>>>(p, t);
  } else {
    if (p.q != nullptr) swiglu_bwd_kernel<T, N, true><<<grid, 256, 0, s>>>(p, t);
    else swiglu_bwd_kernel<T, N, false><<<grid, 256, 0, s>>>(p, t);
  }
  FLARE_CUDA_CHECK(cudaGetLastError());
  count_launch();
}

bool vec_ok(const void* p, int64_t ld, int dtype) {
  const int es = dtype == kF32 ? 4 : 2;
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * es) % 16 == 0);
}

void swiglu_dispatch(const SwigluParams& p, bool backward, cudaStream_t s) {
  if (p.R == 0 || p.h == 0) return;
  // 16-byte vectors where rows and halves start on 16 bytes, single elements elsewhere
  const int64_t per = p.dtype == kF32 ? 4 : 8;
  const bool vec = p.h % per == 0 && vec_ok(p.x, p.ldx, p.dtype) && (!backward || vec_ok(p.dy, p.lddy, p.dtype));
  switch (p.dtype) {
    case kF32: vec ? swiglu_launch<float, 4>(p, backward, s) : swiglu_launch<float, 1>(p, backward, s); break;
    case kBF16: vec ? swiglu_launch<__nv_bfloat16, 8>(p, backward, s) : swiglu_launch<__nv_bfloat16, 1>(p, backward, s); break;
    default: vec ? swiglu_launch<__half, 8>(p, backward, s) : swiglu_launch<__half, 1>(p, backward, s); break;
  }
}

// ------------------------------------------------------------- combination
// Bound by memory: 65536 tokens of 512 bf16, two rows each: forward 50 us for 201 MB (0.62 of the
// measured copy; rows of 1 KB in the order of the groups), backward 56 us for 336 MB (0.92).  Rows
// that do not start on 16 bytes go element by element: 511 columns take 123 and 145 us.
// A thread owns N columns of two tokens at a time (of one where z is fp32: its registers are full)
// and reads their rows, KU of each in flight.
template <typename T, int N, typename O, int KU>
__global__ void __launch_bounds__(256) combine_fwd_kernel(CombineParams p, RowTiling t) {
  constexpr int U = sizeof(T) == 2 ? 2 : 1;
  const int r0 = t.rows > 1 ? threadIdx.x / t.cols : 0;
  const int c0 = t.rows > 1 ? threadIdx.x % t.cols : threadIdx.x;
  if (r0 >= t.rows) return;
  const int64_t step = static_cast<int64_t>(gridDim.x) * t.rows;
  for (int64_t tok = static_cast<int64_t>(blockIdx.x) * t.rows + r0; tok < p.T; tok += U * step) {
    const int live = U == 2 && tok + step < p.T ? 2 : 1;
    for (int c = c0; c < t.cols; c += 256) {
      const T* z = static_cast<const T*>(p.z) + static_cast<int64_t>(c) * N;
      float acc[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[u][i] = 0.f;
      for (int j0 = 0; j0 < p.k; j0 += KU) {
        int row[U][KU];
        float w[U][KU], f[U][KU][N];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int q = 0; q < KU; ++q) {
            const int64_t at = (tok + u * step) * p.k + j0 + q;
            const bool in = u < live && j0 + q < p.k;
            row[u][q] = in ? p.row_of[at] : -1;
            w[u][q] = in && p.weights != nullptr ? p.weights[at] : 1.f;
          }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int q = 0; q < KU; ++q) {
            if (row[u][q] >= 0 && row[u][q] < p.R) {
              load_f<T, N>(z + row[u][q] * p.ldz, f[u][q]);
            } else {
              w[u][q] = 0.f;
#pragma unroll
              for (int i = 0; i < N; ++i) f[u][q][i] = 0.f;
            }
          }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int q = 0; q < KU; ++q)
#pragma unroll
            for (int i = 0; i < N; ++i) acc[u][i] = fmaf(w[u][q], f[u][q][i], acc[u][i]);
      }
      O* y = static_cast<O*>(p.y) + static_cast<int64_t>(c) * N;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < live) store_f<O, N>(y + (tok + u * step) * p.N, acc[u]);
    }
  }
}

// A warp per (token, choice): dz[row] = w * dy[t], dw = <z[row], dy[t]>; a token's choices are
// neighbours, so its dy comes from the caches.  Rows behind the last group get zeros.  kWeighted
// off: dz[row] = dy[t], and z is not read.
template <typename T, int N, bool kWeighted>
__global__ void __launch_bounds__(256) combine_bwd_kernel(CombineParams p) {
  const int lane = lane_id();
  const int64_t warps = static_cast<int64_t>(gridDim.x) * 8, pairs = p.T * p.k;
  int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + warp_id();
  int next = i < pairs ? p.row_of[i] : -1;  // a pair ahead
  for (; i < pairs; i += warps) {
    const int row = next;
    if (i + warps < pairs) next = p.row_of[i + warps];
    if (row < 0 || row >= p.R) {
      if (kWeighted && lane == 0) p.dw[i] = 0.f;
      continue;
    }
    const float w = kWeighted ? p.weights[i] : 1.f;
    const T* dy = static_cast<const T*>(p.dy) + (i / p.k) * p.lddy;
    const T* z = kWeighted ? static_cast<const T*>(p.z) + row * p.ldz : nullptr;
    T* dz = static_cast<T*>(p.dz) + static_cast<int64_t>(row) * p.N;
    float dot = 0.f;
    for (int c = lane * N; c < p.N; c += 64 * N) {  // both halves' loads before either store
      const bool second = c + 32 * N < p.N;
      float a[2][N], b[2][N];
      load_f<T, N>(dy + c, a[0]);
      if (second) load_f<T, N>(dy + c + 32 * N, a[1]);
      if constexpr (kWeighted) {
        load_f<T, N>(z + c, b[0]);
        if (second) load_f<T, N>(z + c + 32 * N, b[1]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1 && !second) break;
        float o[N];
#pragma unroll
        for (int q = 0; q < N; ++q) {
          if constexpr (kWeighted) dot = fmaf(a[h][q], b[h][q], dot);
          o[q] = w * a[h][q];
        }
        store_f<T, N>(dz + c + h * 32 * N, o);
      }
    }
    if constexpr (kWeighted) {
      dot = warp_sum(dot);
      if (lane == 0) p.dw[i] = dot;
    }
  }
  const int64_t total = max(0, *p.total);
  for (int64_t r = total + static_cast<int64_t>(blockIdx.x) * 8 + warp_id(); r < p.R; r += warps) {
    float zero[N];
#pragma unroll
    for (int q = 0; q < N; ++q) zero[q] = 0.f;
    for (int c = lane * N; c < p.N; c += 32 * N) store_f<T, N>(static_cast<T*>(p.dz) + r * p.N + c, zero);
  }
}

template <typename T, int N>
void combine_launch(const CombineParams& p, bool backward, cudaStream_t s) {
  if (!backward) {
    RowTiling t;
    t.cols = p.N / N;
    t.rows = t.cols <= 128 ? 256 / t.cols : 1;
    const int grid = static_cast<int>(std::min<int64_t>((p.T + t.rows - 1) / t.rows, 148 * 16));
    auto go = [&](auto out) {
      using O = decltype(out);
      if (p.k == 1) combine_fwd_kernel<T, N, O, 1><<<grid, 256, 0, s>>>(p, t);
      else if (p.k == 2) combine_fwd_kernel<T, N, O, 2><<<grid, 256, 0, s>>>(p, t);
      else combine_fwd_kernel<T, N, O, 4><<<grid, 256, 0, s>>>(p, t);
    };
    if constexpr (sizeof(T) == 4) {
      if (p.out_dtype == kBF16) go(__nv_bfloat16());
      else if (p.out_dtype == kF16) go(__half());
      else go(T());
    } else {
      go(T());
    }
  } else {
    const int grid = static_cast<int>(std::min<int64_t>((std::max(p.T * p.k, p.R) + 7) / 8, 148 * 16));
    if (p.weights != nullptr) combine_bwd_kernel<T, N, true><<<grid, 256, 0, s>>>(p);
    else combine_bwd_kernel<T, N, false><<<grid, 256, 0, s>>>(p);
  }
  FLARE_CUDA_CHECK(cudaGetLastError());
  count_launch();
}

void combine_dispatch(const CombineParams& p, bool backward, cudaStream_t s) {
  if (p.N == 0 || (p.T == 0 && !(backward && p.R > 0))) return;
  const int per = p.dtype == kF32 ? 4 : 8;
  const bool vec = p.N % per == 0 && vec_ok(p.z, p.ldz, p.dtype) && (!backward || vec_ok(p.dy, p.lddy, p.dtype));
  switch (p.dtype) {
    case kF32: vec ? combine_launch<float, 4>(p, backward, s) : combine_launch<float, 1>(p, backward, s); break;
    case kBF16: vec ? combine_launch<__nv_bfloat16, 8>(p, backward, s) : combine_launch<__nv_bfloat16, 1>(p, backward, s); break;
    default: vec ? combine_launch<__half, 8>(p, backward, s) : combine_launch<__half, 1>(p, backward, s); break;
  }
}

}  // namespace

int64_t route_work_ints(int S, int B, int E) {
  if (S == 1 && B <= kRouteOneBlock) return 0;
  return static_cast<int64_t>(S) * (ceil_div(B, kSub) + 1) * E;
}

void route_topk(const RouteParams& p, cudaStream_t s) {
  FLARE_CHECK(p.S > 0 && p.B > 0, "route_topk: no tokens");
  FLARE_CHECK(p.E > 0 && p.E <= kRouteMaxExperts, "route_topk: 1 to 512 experts");
  FLARE_CHECK(p.k > 0 && p.k <= p.E && p.k <= kRouteMaxTopK, "route_topk: top_k is at most the experts, and 32");
  switch (p.dtype) {
    case kF32: route_typed<float>(p, s); break;
    case kBF16: route_typed<__nv_bfloat16>(p, s); break;
    default: route_typed<__half>(p, s); break;
  }
}

void route_topk_backward(const RouteBwdParams& p, cudaStream_t s) {
  if (p.T == 0) return;
  switch (p.dtype) {
    case kF32: route_bwd_launch<float>(p, s); break;
    case kBF16: route_bwd_launch<__nv_bfloat16>(p, s); break;
    default: route_bwd_launch<__half>(p, s); break;
  }
}

void swiglu_forward(const SwigluParams& p, cudaStream_t s) { swiglu_dispatch(p, false, s); }
void swiglu_backward(const SwigluParams& p, cudaStream_t s) { swiglu_dispatch(p, true, s); }
void combine_forward(const CombineParams& p, cudaStream_t s) { combine_dispatch(p, false, s); }
void combine_backward(const CombineParams& p, cudaStream_t s) { combine_dispatch(p, true, s); }

}  // namespace flare
