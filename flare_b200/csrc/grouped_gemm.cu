// Grouped matrix products with ragged groups on tcgen05 (sm_100a).
//
// Rows 0 .. R are sorted by group; group g owns rows [offsets[g], offsets[g+1])
// and the weight W_g [K, N] of w [G, K, N].  The offsets stay on the device.
//   forward   Y[r, :]  = X[r or rows[r], :] W_g + b_g        (contraction K)
//   input     dX[r, :] = dY[r, :] W_g^T                      (contraction N)
//   weight    dW_g     = X_g^T dY_g                          (contraction: the group's rows)
// Operands are read as they are stored: W is the MN-major operand of the forward
// product and the K-major one of the input gradient; the weight gradient reads X
// and dY MN-major.  W's tensor map has three dimensions, so a tile that reaches
// past K or N of one group reads zeros and never the next group's weights.
//
// A persistent grid walks output tiles (n fastest: the tiles in flight share a
// group's weights in L2 and the rows of a few tiles).  Per CTA: warp 0 loads
// (TMA, a STAGES-deep ring of 128-byte-swizzled tiles), warp 1 issues the MMAs
// into one of two TMEM accumulators, warps 2..5 drain the other: the epilogue of
// a tile overlaps the mainloop of the next.  Rows gathered by index, and rows of
// the weight gradient's last, partial step, are fetched four at a time by index
// (a row outside the tensor reads as zeros: the next group's rows, and whatever
// infinities are in them, never enter a product).
// Variants: CTA pairs on 256 x 256 tiles (each CTA stages half of B, which halves
// its operand traffic), one CTA on 128 x 128 or 128 x 64 tiles.
// Every sum is held in fp32 and rounded once.  Every wait is bounded.
#include "experts.cuh"
#include "gemm.cuh"
#include "sm100.cuh"

#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace flare {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn();  // gemm_tcgen05.cu

namespace {

constexpr int kBK = 64;          // contraction step: one 128-byte swizzle atom of 16-bit values
constexpr int kThreads = 192;    // producer, MMA issuer, four epilogue warps
constexpr int kEpiWarps = 4;
constexpr int kTileA = 128 * kBK * 2;

struct GP {
  const int* offsets;
  int G, R;
  const int* rows;
  int x_rows;    // rows of x (an index of this value reads zeros)
  int dy_rows;
  int Mo;        // weight gradient: output rows of a group
  int No;        // output columns
  int Kc;        // forward, input gradient: contraction length
  int mt, nt;    // tiles of a group's output rows (weight gradient) and columns
  void* out;
  int64_t ldo;
  int out_dtype, accumulate;
  const void* bias;
  int bias_dtype;
  uint32_t idesc;
  int* status;
  uint64_t timeout_ns;
};

template <bool PAIR, int BN, int STAGES>
struct Smem {
  static constexpr int kBNh = PAIR ? BN / 2 : BN;  // B rows that one CTA stages
  static constexpr int kTileB = kBNh * kBK * 2;
  static constexpr int kStage = kTileA + kTileB;
  static constexpr int kOffB = STAGES * kTileA;
  static constexpr int kOffEpi = kOffB + STAGES * kTileB;       // 4 KiB per epilogue warp
  static constexpr int kOffBias = kOffEpi + kEpiWarps * 4096;   // 64 floats per epilogue warp
  static constexpr int kOffPre = kOffBias + kEpiWarps * 256;    // tile prefix of the groups
  static constexpr int kOffBar = kOffPre + (kGroupedMaxGroups + 2) * 4;
  static constexpr int kBytes = kOffBar + (2 * STAGES + 4) * 8 + 16;
  static constexpr int kAlloc = kBytes + 1024;
  static_assert(kOffBar % 8 == 0, "barriers are 8-byte aligned");
  static_assert(kAlloc <= 227 * 1024, "shared memory of one CTA");
};

__device__ __forceinline__ int2 group_range(const GP& p, int g) {
  const int lo = min(max(p.offsets[g], 0), p.R);
  return make_int2(lo, min(max(p.offsets[g + 1], lo), p.R));
}

struct Tile {
  int g, m0, n0, lo, hi, steps;
};

// Walks this CTA's (or pair's) tiles in order.
template <int MODE, int BM, int BN>
struct Walk {
  const GP& p;
  const int* pre;
  int u, step, total, g;
  __device__ Walk(const GP& p_, const int* pre_, int first, int step_)
      : p(p_), pre(pre_), u(first), step(step_), total(MODE == kGroupedWgrad ? p_.G * p_.mt * p_.nt : pre_[p_.G] * p_.nt), g(0) {}
  __device__ bool next(Tile& t) {
    if (u >= total) return false;
    const int n = u % p.nt;
    int m = u / p.nt;
    if constexpr (MODE == kGroupedWgrad) {
      g = m / p.mt;
      m -= g * p.mt;
    } else {
      while (pre[g + 1] <= m) ++g;
      m -= pre[g];
    }
    const int2 r = group_range(p, g);
    t.g = g;
    t.lo = r.x;
    t.hi = r.y;
    t.n0 = n * BN;
    if constexpr (MODE == kGroupedWgrad) {
      t.m0 = m * BM;
      t.steps = (r.y - r.x + kBK - 1) / kBK;
    } else {
      t.m0 = r.x + m * BM;
      t.steps = (p.Kc + kBK - 1) / kBK;
    }
    u += step;
    return true;
  }
};

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
  if (dtype == kF32) return static_cast<const float*>(p)[i];
  if (dtype == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ uint32_t pack2(float a, float b, bool bf16) {
  if (bf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 64 columns of 32 rows (lane = row) to out, through 4 KiB of shared memory: eight lanes write one
// row's 128 bytes (64 values of 16 bits, or 32 of fp32 at a time) instead of every lane 16 bytes of
// its own row.  16-byte pieces lie at piece ^ (row % 8): no bank is hit twice on either side.
__device__ __forceinline__ void store_chunk(const GP& p, float (&v)[64], int64_t row0, int rows, int col, int64_t base,
                                            uint8_t* stage) {
  const int lane = lane_id(), q = lane & 7;
  if (p.out_dtype == kF32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int j = h * 32 + c * 4;
        *reinterpret_cast<float4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
      }
      __syncwarp();
      float* o = static_cast<float*>(p.out) + base + row0 * p.ldo + col + h * 32 + q * 4;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + (lane >> 3);
        float4 u = *reinterpret_cast<const float4*>(stage + r * 128 + ((q ^ (r & 7)) << 4));
        if (r < rows && col + h * 32 + q * 4 < p.No) {
          if (p.accumulate) u = f4_add(u, *reinterpret_cast<const float4*>(o + r * p.ldo));
          *reinterpret_cast<float4*>(o + r * p.ldo) = u;
        }
      }
      __syncwarp();
    }
    return;
  }
  const bool bf = p.out_dtype == kBF16;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint4 u;
    u.x = pack2(v[8 * c], v[8 * c + 1], bf);
    u.y = pack2(v[8 * c + 2], v[8 * c + 3], bf);
    u.z = pack2(v[8 * c + 4], v[8 * c + 5], bf);
    u.w = pack2(v[8 * c + 6], v[8 * c + 7], bf);
    *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) = u;
  }
  __syncwarp();
  uint16_t* o = static_cast<uint16_t*>(p.out) + base + row0 * p.ldo + col + q * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + (lane >> 3);
    const uint4 u = *reinterpret_cast<const uint4*>(stage + r * 128 + ((q ^ (r & 7)) << 4));
    if (r < rows && col + q * 8 < p.No) *reinterpret_cast<uint4*>(o + r * p.ldo) = u;
  }
  __syncwarp();
}

// Rows outside every group (before the first, behind the last) become zeros.
__device__ __forceinline__ void zero_outside(const GP& p, int warp, int warps) {
  const int lane = lane_id();
  const int first = group_range(p, 0).x, last = group_range(p, p.G - 1).y;
  const int64_t n = static_cast<int64_t>(first) + (p.R - last);
  for (int64_t i = warp; i < n; i += warps) {
    const int64_t r = i < first ? i : last + (i - first);
    const int es = p.out_dtype == kF32 ? 4 : 2, per = 16 / es;
    uint8_t* o = static_cast<uint8_t*>(p.out) + r * p.ldo * es;
    for (int c = lane * per; c < p.No; c += 32 * per) *reinterpret_cast<uint4*>(o + c * es) = make_uint4(0, 0, 0, 0);
  }
}

// ta / tb: tiles of A and B; ga / gb: the same tensors with boxes of one row (gathered rows).
template <int MODE, bool PAIR, int BN, int STAGES, bool GATHER>
__device__ __forceinline__ void grouped_body(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& ga,
                                             const CUtensorMap& gb, const GP& p) {
  using L = Smem<PAIR, BN, STAGES>;
  constexpr int BM = PAIR ? 256 : 128;
  constexpr bool A_MN = MODE == kGroupedWgrad, B_MN = MODE != kGroupedDgrad;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  int* pre = reinterpret_cast<int*>(sm + L::kOffPre);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::kOffBar);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  const int warp = warp_id(), lane = lane_id();
  const int rank = PAIR ? static_cast<int>(sm100::cluster_ctarank()) : 0;
  const int first = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;

  if (threadIdx.x == 0) {
    sm100::tma_prefetch_desc(&ta);
    sm100::tma_prefetch_desc(&tb);
    for (int s = 0; s < STAGES; ++s) {
      sm100::mbar_init(&full[s], 1);
      sm100::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      sm100::mbar_init(&acc_full[b], 1);
      sm100::mbar_init(&acc_empty[b], kEpiWarps * (PAIR ? 2 : 1));
    }
    sm100::fence_mbar_init();
  }
  if (warp == 0) {
    if constexpr (PAIR) {
      sm100::tmem_alloc_pair(slot, 2 * BN);
      sm100::tmem_relinquish_pair();
    } else {
      sm100::tmem_alloc(slot, 2 * BN);
      sm100::tmem_relinquish();
    }
  }
  if constexpr (MODE != kGroupedWgrad) {
    for (int g = threadIdx.x; g < p.G; g += kThreads) {
      const int2 r = group_range(p, g);
      pre[g + 1] = (r.y - r.x + BM - 1) / BM;
    }
    if (threadIdx.x == 0) pre[0] = 0;
    __syncthreads();
    if (warp == 1) {
      int carry = 0;
      for (int g0 = 0; g0 < p.G; g0 += 32) {
        int v = g0 + lane < p.G ? pre[g0 + lane + 1] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += up;
        }
        if (g0 + lane < p.G) pre[g0 + lane + 1] = carry + v;
        carry += __shfl_sync(0xffffffffu, v, 31);
      }
    }
  }
  if (blockIdx.x == 0) {  // a group that ends before it starts, or outside the rows, is reported
    for (int g = threadIdx.x; g < p.G; g += kThreads)
      if (p.offsets[g] < 0 || p.offsets[g + 1] < p.offsets[g] || p.offsets[g + 1] > p.R)
        report_error(p.status, kIndexOutOfRange, g);
  }
  sm100::tc_fence_before();
  if constexpr (PAIR) sm100::cluster_sync();  // both CTAs' barriers and TMEM exist before any cross-CTA use
  else __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *slot;
  Tile t;
  Walk<MODE, BM, BN> walk(p, pre, first, step);

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    uint32_t it = 0;
    bool ok = true;
    auto load2 = [&](void* dst, const CUtensorMap& m, int s, int x, int y) {
      if constexpr (PAIR) sm100::tma_load_2d_pair(dst, &m, sm100::mapa_shared(&full[s], 0), x, y);
      else sm100::tma_load_2d(dst, &m, &full[s], x, y);
    };
    auto load3 = [&](void* dst, const CUtensorMap& m, int s, int x, int y, int z) {
      if constexpr (PAIR) sm100::tma_load_3d_pair(dst, &m, sm100::mapa_shared(&full[s], 0), x, y, z);
      else sm100::tma_load_3d(dst, &m, &full[s], x, y, z);
    };
    auto gather = [&](void* dst, const CUtensorMap& m, int s, int x, int4 r) {
      if constexpr (PAIR) sm100::tma_gather4_pair(dst, &m, sm100::mapa_shared(&full[s], 0), x, r);
      else sm100::tma_gather4(dst, &m, &full[s], x, r);
    };
    // rows r .. r + 3 of x: their tokens, or the rows themselves; outside [.., hi): a row of zeros
    auto row4 = [&](int r, int hi, const int* rows, int none) {
      int v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int x = r + i < hi ? (rows != nullptr ? rows[r + i] : r + i) : none;
        v[i] = static_cast<unsigned>(x) < static_cast<unsigned>(none) ? x : none;
      }
      return make_int4(v[0], v[1], v[2], v[3]);
    };
    while (ok && walk.next(t)) {
      int4 ar = make_int4(0, 0, 0, 0);
      if constexpr (MODE == kGroupedFwd && GATHER) ar = row4(t.m0 + rank * 128 + 4 * lane, t.hi, p.rows, p.x_rows);
      for (int k = 0; k < t.steps; ++k, ++it) {
        const int s = it % STAGES;
        int4 xr = make_int4(0, 0, 0, 0);
        const int r0 = t.lo + k * kBK;
        if constexpr (MODE == kGroupedWgrad && GATHER) xr = row4(r0 + 4 * (lane & 15), t.hi, p.rows, p.x_rows);
        if (it >= STAGES && !sm100::mbar_wait(&empty[s], ((it / STAGES) - 1) & 1, p.timeout_ns, p.status, 400 + s)) ok = false;
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        uint8_t* sa = sm + s * kTileA;
        uint8_t* sb = sm + L::kOffB + s * L::kTileB;
        if (lane == 0 && rank == 0) sm100::mbar_arrive_expect_tx(&full[s], (PAIR ? 2 : 1) * L::kStage);
        if constexpr (MODE != kGroupedWgrad) {
          const int k0 = k * kBK;
          if constexpr (GATHER) gather(sa + lane * 512, ga, s, k0, ar);
          if (lane == 0) {
            if constexpr (!GATHER) load2(sa, ta, s, k0, t.m0 + rank * 128);
            if constexpr (B_MN) {
#pragma unroll
              for (int j = 0; j < L::kBNh / 64; ++j) load3(sb + j * 8192, tb, s, t.n0 + rank * L::kBNh + 64 * j, k0, t.g);
            } else {
              load3(sb, tb, s, k0, t.n0 + rank * L::kBNh, t.g);
            }
          }
        } else {
          const int ma = t.m0 + rank * 128, nb = t.n0 + rank * L::kBNh, sub = lane & 15, half = lane >> 4;
          const bool whole = r0 + kBK <= t.hi;
          if constexpr (GATHER) {
            gather(sa + half * 8192 + sub * 512, ga, s, ma + 64 * half, xr);
          } else if (!whole) {
            gather(sa + half * 8192 + sub * 512, ga, s, ma + 64 * half, row4(r0 + 4 * sub, t.hi, nullptr, p.x_rows));
          }
          if (!whole) {
            const int4 br = row4(r0 + 4 * sub, t.hi, nullptr, p.dy_rows);
#pragma unroll
            for (int j = 0; j < L::kBNh / 64; j += 2)
              if (j + half < L::kBNh / 64) gather(sb + (j + half) * 8192 + sub * 512, gb, s, nb + 64 * (j + half), br);
          }
          if (lane == 0 && whole) {
            if constexpr (!GATHER) {
              load2(sa, ta, s, ma, r0);
              load2(sa + 8192, ta, s, ma + 64, r0);
            }
#pragma unroll
            for (int j = 0; j < L::kBNh / 64; ++j) load2(sb + j * 8192, tb, s, nb + 64 * j, r0);
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (lane == 0 && rank == 0) {
      uint32_t it = 0, i = 0;
      bool ok = true;
      while (ok && walk.next(t)) {
        if (t.steps == 0) continue;
        const int buf = i & 1;
        const uint32_t d = tmem + buf * BN;
        if (i >= 2 && !sm100::mbar_wait_cluster(&acc_empty[buf], ((i >> 1) - 1) & 1, p.timeout_ns, p.status, 420 + buf)) break;
        sm100::tc_fence_after();
        for (int k = 0; k < t.steps; ++k, ++it) {
          const int s = it % STAGES;
          if (!sm100::mbar_wait(&full[s], (it / STAGES) & 1, p.timeout_ns, p.status, 440 + s)) {
            ok = false;
            break;
          }
          sm100::tc_fence_after();
          const uint32_t sa = smem_u32(sm + s * kTileA), sb = smem_u32(sm + L::kOffB + s * L::kTileB);
#pragma unroll
          for (int q = 0; q < kBK / 16; ++q) {
            const uint64_t da = A_MN ? sm100::make_smem_desc(sa + q * 2048, 8192, 1024) : sm100::make_smem_desc(sa + q * 32, 16, 1024);
            const uint64_t db = B_MN ? sm100::make_smem_desc(sb + q * 2048, 8192, 1024) : sm100::make_smem_desc(sb + q * 32, 16, 1024);
            if constexpr (PAIR) sm100::mma_f16_ss_pair(d, da, db, p.idesc, (k | q) != 0);
            else sm100::mma_f16_ss(d, da, db, p.idesc, (k | q) != 0);
          }
          if constexpr (PAIR) {
            sm100::mma_commit_pair(sm100::mapa_shared(&empty[s], 0));
            sm100::mma_commit_pair(sm100::mapa_shared(&empty[s], 1));
          } else {
            sm100::mma_commit(&empty[s]);
          }
        }
        if (!ok) break;
        if constexpr (PAIR) {
          sm100::mma_commit_pair(sm100::mapa_shared(&acc_full[buf], 0));
          sm100::mma_commit_pair(sm100::mapa_shared(&acc_full[buf], 1));
        } else {
          sm100::mma_commit(&acc_full[buf]);
        }
        ++i;
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;  // the TMEM lanes that this warp may read
    uint8_t* stage = sm + L::kOffEpi + (warp - 2) * 4096;
    float* bias = reinterpret_cast<float*>(sm + L::kOffBias + (warp - 2) * 256);
    if constexpr (MODE != kGroupedWgrad) zero_outside(p, blockIdx.x * kEpiWarps + warp - 2, gridDim.x * kEpiWarps);
    uint32_t i = 0;
    while (walk.next(t)) {
      const int buf = i & 1;
      const bool any = t.steps > 0;
      if (any) {
        bool ok = sm100::mbar_wait(&acc_full[buf], (i >> 1) & 1, p.timeout_ns, p.status, 460 + buf);
        if (!__all_sync(0xffffffffu, ok)) break;
        sm100::tc_fence_after();
      }
      const int64_t row0 = t.m0 + rank * 128 + quarter * 32;
      const int rows = min(32, (MODE == kGroupedWgrad ? p.Mo : t.hi) - static_cast<int>(row0));
      const int64_t base = MODE == kGroupedWgrad ? static_cast<int64_t>(t.g) * p.Mo * p.ldo : 0;
      for (int c = 0; c < BN; c += 64) {
        const int col = t.n0 + c;
        if (col >= p.No || rows <= 0) break;  // warp-uniform
        float v[64];
        if (any) {
          uint32_t r[2][32];
          const uint32_t at = tmem + buf * BN + c + (static_cast<uint32_t>(quarter * 32) << 16);
          sm100::tmem_ld_32x32b_x32(at, r[0]);
          sm100::tmem_ld_32x32b_x32(at + 32, r[1]);
          if (MODE == kGroupedFwd && p.bias != nullptr) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              bias[h * 32 + lane] = col + h * 32 + lane < p.No ? load_any(p.bias, static_cast<int64_t>(t.g) * p.No + col + h * 32 + lane, p.bias_dtype) : 0.f;
            __syncwarp();
          }
          sm100::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 64; ++j) {
            asm volatile("" : "+r"(r[j >> 5][j & 31]));
            v[j] = __uint_as_float(r[j >> 5][j & 31]);
          }
          if (MODE == kGroupedFwd && p.bias != nullptr) {
#pragma unroll
            for (int j = 0; j < 64; j += 4) {
              const float4 b = *reinterpret_cast<const float4*>(bias + j);
              v[j] += b.x, v[j + 1] += b.y, v[j + 2] += b.z, v[j + 3] += b.w;
            }
            __syncwarp();
          }
        } else {
          if (p.accumulate) break;
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = 0.f;
        }
        store_chunk(p, v, row0, rows, col, base, stage);
      }
      if (any) {
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) sm100::mbar_arrive_cluster(sm100::mapa_shared(&acc_empty[buf], 0));
          else sm100::mbar_arrive(&acc_empty[buf]);
        }
        ++i;
      }
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) sm100::cluster_sync();  // neither CTA leaves while the other may signal it or read its TMEM
  if (warp == 0) {
    if constexpr (PAIR) sm100::tmem_dealloc_pair(tmem, 2 * BN);
    else sm100::tmem_dealloc(tmem, 2 * BN);
  }
}

template <int MODE, int BN, int STAGES, bool GATHER>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                   const __grid_constant__ CUtensorMap ga, const __grid_constant__ CUtensorMap gb, const __grid_constant__ GP p) {
  grouped_body<MODE, false, BN, STAGES, GATHER>(ta, tb, ga, gb, p);
}
template <int MODE, int BN, int STAGES, bool GATHER>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    grouped_pair_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                        const __grid_constant__ CUtensorMap ga, const __grid_constant__ CUtensorMap gb,
                        const __grid_constant__ GP p) {
  grouped_body<MODE, true, BN, STAGES, GATHER>(ta, tb, ga, gb, p);
}

// ------------------------------------------------------------------- host
CUtensorMap make_map(const void* base, int dtype, int rank, const int64_t* dims, const int64_t* pitch, const int* box) {
  FLARE_CHECK((reinterpret_cast<uintptr_t>(base) & 15) == 0, "grouped products: operands must be 16-byte aligned");
  CUtensorMap m;
  cuuint64_t d[3], st[2];
  cuuint32_t b[3], es[3] = {1u, 1u, 1u};
  for (int i = 0; i < rank; ++i) {
    d[i] = static_cast<cuuint64_t>(dims[i]);
    b[i] = static_cast<cuuint32_t>(box[i]);
    if (i > 0) {
      FLARE_CHECK((pitch[i - 1] * 2) % 16 == 0, "grouped products: row pitches must be multiples of 8 elements");
      st[i - 1] = static_cast<cuuint64_t>(pitch[i - 1] * 2);
    }
  }
  const CUresult r = encode_fn()(&m, dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                                 const_cast<void*>(base), d, st, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  FLARE_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (code " + std::to_string(static_cast<int>(r)) + ")");
  return m;
}
CUtensorMap map2(const void* base, int dtype, int64_t inner, int64_t rows, int64_t ld, int box_rows) {
  const int64_t d[2] = {inner, rows}, pt[1] = {ld};
  const int b[2] = {64, box_rows};
  return make_map(base, dtype, 2, d, pt, b);
}

constexpr int kMaxDevices = 64;

// Sets a kernel's shared-memory limit once per device and returns how many CTAs (or pairs) of it
// the current device runs at once.
int resident(const void* kern, int smem, bool pair, int (&cache)[kMaxDevices]) {
  static std::mutex mu;
  int dev = 0;
  FLARE_CUDA_CHECK(cudaGetDevice(&dev));
  FLARE_CHECK(dev >= 0 && dev < kMaxDevices, "device index");
  std::lock_guard<std::mutex> lock(mu);
  if (cache[dev] == 0) {
    FLARE_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    int n = 0;
    if (pair) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(2);
      cfg.blockDim = dim3(kThreads);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = 2;
      at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      FLARE_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
    } else {
      FLARE_CUDA_CHECK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    }
    cache[dev] = std::max(1, n);
  }
  return cache[dev];
}

template <int MODE, bool PAIR, int BN, int STAGES, bool GATHER>
void launch(const GroupedArgs& a, cudaStream_t s) {
  using L = Smem<PAIR, BN, STAGES>;
  constexpr int BM = PAIR ? 256 : 128;
  GP p{};
  p.offsets = a.offsets;
  p.G = a.G;
  p.R = static_cast<int>(a.R);
  p.rows = a.rows;
  p.x_rows = static_cast<int>(a.x_rows);
  p.dy_rows = p.R;
  p.Mo = a.K;
  p.No = MODE == kGroupedDgrad ? a.K : a.N;
  p.Kc = MODE == kGroupedDgrad ? a.N : a.K;
  p.mt = ceil_div(a.K, BM);
  p.nt = ceil_div(p.No, BN);
  p.out = a.out;
  p.ldo = p.No;
  p.out_dtype = a.out_dtype;
  p.accumulate = a.accumulate;
  p.bias = MODE == kGroupedFwd ? a.bias : nullptr;
  p.bias_dtype = a.bias_dtype;
  p.idesc = sm100::make_idesc_16bit(BM, BN, MODE == kGroupedWgrad, MODE != kGroupedDgrad, a.dtype == kBF16);
  p.status = a.status;
  p.timeout_ns = a.timeout_ns;
  CUtensorMap ta, tb, ga, gb;
  if (MODE == kGroupedWgrad) {
    ta = map2(a.x, a.dtype, a.K, a.x_rows, a.ldx, kBK);
    ga = map2(a.x, a.dtype, a.K, a.x_rows, a.ldx, 1);
    tb = map2(a.dy, a.dtype, a.N, a.R, a.lddy, kBK);
    gb = map2(a.dy, a.dtype, a.N, a.R, a.lddy, 1);
  } else {
    const int64_t wd[3] = {a.N, a.K, a.G}, wp[2] = {a.N, static_cast<int64_t>(a.K) * a.N};
    const int box_fwd[3] = {64, kBK, 1}, box_bwd[3] = {64, L::kBNh, 1};
    tb = make_map(a.w, a.dtype, 3, wd, wp, MODE == kGroupedFwd ? box_fwd : box_bwd);
    if (MODE == kGroupedFwd) ta = map2(a.x, a.dtype, a.K, a.x_rows, a.ldx, GATHER ? 1 : 128);
    else ta = map2(a.dy, a.dtype, a.N, a.R, a.lddy, 128);
    ga = ta;
    gb = tb;
  }
  // as many tiles as there can be: the groups' sizes are on the device
  const int64_t tiles = MODE == kGroupedWgrad
                            ? static_cast<int64_t>(a.G) * p.mt * p.nt
                            : (a.R / BM + std::min<int64_t>(a.G, a.R)) * p.nt;
  FLARE_CHECK(tiles < (1ll << 31), "grouped products: too many tiles");
  static int cache[kMaxDevices];
  if constexpr (PAIR) {
    auto kern = grouped_pair_kernel<MODE, BN, STAGES, GATHER>;
    const int n = static_cast<int>(std::min<int64_t>(std::max<int64_t>(1, tiles), resident(reinterpret_cast<const void*>(kern), L::kAlloc, true, cache)));
    kern<<<2 * n, kThreads, L::kAlloc, s>>>(ta, tb, ga, gb, p);
  } else {
    auto kern = grouped_kernel<MODE, BN, STAGES, GATHER>;
    const int n = static_cast<int>(std::min<int64_t>(std::max<int64_t>(1, tiles), resident(reinterpret_cast<const void*>(kern), L::kAlloc, false, cache)));
    kern<<<n, kThreads, L::kAlloc, s>>>(ta, tb, ga, gb, p);
  }
  FLARE_CUDA_CHECK(cudaGetLastError());
  count_launch();
}

template <int MODE, bool GATHER>
void pick(const GroupedArgs& a, cudaStream_t s) {
  const int no = MODE == kGroupedDgrad ? a.K : a.N;
  // rows of an average group fill a pair's 256 at least once, and both sides of the tile are used
  const bool tall = MODE == kGroupedWgrad ? a.K > 128 : a.R >= 256ll * a.G;
  if (tall && no > 128) launch<MODE, true, 256, 6, GATHER>(a, s);
  else if (no > 64) launch<MODE, false, 128, 6, GATHER>(a, s);
  else launch<MODE, false, 64, 8, GATHER>(a, s);
}

// ------------------------------------------------------- per-group column sums
// Block = 64 columns (eight lanes x 8) of one slice of one group; 32 rows at a time.  The slices'
// sums are added in order by the second kernel: nothing depends on the schedule.
template <typename T>
__global__ void __launch_bounds__(256) group_sum_kernel(GroupSumArgs a, float* part, int slices) {
  const int g = blockIdx.y, sl = blockIdx.z;
  const int lo = min(max(a.offsets[g], 0), static_cast<int>(a.R)), hi = min(max(a.offsets[g + 1], lo), static_cast<int>(a.R));
  const int per = (hi - lo + slices - 1) / slices;
  const int r0 = lo + sl * per, r1 = min(hi, r0 + per);
  const int c = blockIdx.x * 64 + (threadIdx.x & 7) * 8, rr = threadIdx.x >> 3;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (c < a.N) {
#pragma unroll 4
    for (int r = r0 + rr; r < r1; r += 32) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.y) + r * a.ldy + c));
      const T* v = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += to_f32(v[i]);
    }
  }
  __shared__ float red[32][65];
#pragma unroll
  for (int i = 0; i < 8; ++i) red[rr][(threadIdx.x & 7) * 8 + i] = acc[i];
  __syncthreads();
  if (threadIdx.x < 64) {
    const int col = blockIdx.x * 64 + threadIdx.x;
    if (col >= a.N) return;
    float sum = 0.f;
    for (int i = 0; i < 32; ++i) sum += red[i][threadIdx.x];
    if (part != nullptr) {
      part[(static_cast<int64_t>(g) * slices + sl) * a.N + col] = sum;
      return;
    }
    const int64_t o = static_cast<int64_t>(g) * a.N + col;
    if (a.out_dtype == kF32) static_cast<float*>(a.out)[o] = a.accumulate ? static_cast<float*>(a.out)[o] + sum : sum;
    else if (a.out_dtype == kBF16) static_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16_rn(sum);
    else static_cast<__half*>(a.out)[o] = __float2half_rn(sum);
  }
}

}  // namespace

void grouped_gemm(const GroupedArgs& a, cudaStream_t s) {
  FLARE_CHECK(a.dtype == kBF16 || a.dtype == kF16, "grouped products take bf16 or fp16");
  FLARE_CHECK(a.G > 0 && a.G <= kGroupedMaxGroups, "grouped products: 1 to 2048 groups");
  FLARE_CHECK(a.K > 0 && a.N > 0 && a.K % 8 == 0 && a.N % 8 == 0, "grouped products: widths must be multiples of 8");
  FLARE_CHECK(a.R >= 0 && a.R < (1ll << 31) - 512 && a.x_rows < (1ll << 31) - 512, "grouped products: too many rows");
  // a thread of the autograd engine may not have the device's context yet, and encoding a tensor map needs one
  int dev = 0;
  FLARE_CUDA_CHECK(cudaGetDevice(&dev));
  FLARE_CUDA_CHECK(cudaSetDevice(dev));
  switch (a.mode) {
    case kGroupedFwd:
      if (a.R == 0) return;
      a.rows != nullptr ? pick<kGroupedFwd, true>(a, s) : pick<kGroupedFwd, false>(a, s);
      break;
    case kGroupedDgrad:
      if (a.R == 0) return;
      pick<kGroupedDgrad, false>(a, s);
      break;
    default:
      a.rows != nullptr ? pick<kGroupedWgrad, true>(a, s) : pick<kGroupedWgrad, false>(a, s);
      break;
  }
}

void group_colsum(const GroupSumArgs& a, cudaStream_t s) {
  const dim3 grid(ceil_div(a.N, 64), a.G, 1);
  if (a.dtype == kBF16) group_sum_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a, nullptr, 1);
  else group_sum_kernel<__half><<<grid, 256, 0, s>>>(a, nullptr, 1);
  FLARE_CUDA_CHECK(cudaGetLastError());
  count_launch();
}

}  // namespace flare
