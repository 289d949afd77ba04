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
// into one of two TMEM accumulators, warps 2..9 drain the other: the epilogue of
// a tile overlaps the mainloop of the next (4096 cycles with K = 512).  The weight
// gradient's last, partial step of a group multiplies whole sixteens of rows: a warp
// overwrites the rows of the next group among them with zeros (whatever infinities
// are in them never enter a product).
//
// Rows are gathered from the tokens by a kernel of their own before the product:
// fetched by index inside it (four rows a load), they cost 45 ns of a CTA's load unit
// each time, 1293 us against 432 us for 131072 x 512 x 4096.  Tiles are 128 x 256,
// 128 x 128 or 128 x 64; CTA pairs on 256 x 256 tiles were no faster (554 / 446 us against
// 529 / 436 us for the forward product and the input gradient of that size in 32
// groups, 177 us against 155 us for 200000 x 256 x 1024 in 64).  A tile that reaches
// past its group loads only the sixteens of rows that the group has.
//
// Measured on B200s, 131072 rows, 512 -> 4096, 32 groups of unequal size, bf16 (550 GFLOP
// a direction), in a training pass: forward 480 to 500 us, input gradient 455 to 472 us,
// weight gradient 485 to 511 us (1.08 to 1.21 PFLOP/s, 0.66 to 0.74 of the measured burst);
// each back to back for seconds 605, 516 and 601 us (0.66, 0.78 and 0.67 of the measured
// sustained rate).  cuBLAS on one product of the same size, without groups: 448, 368 and 404
// us, back to back 580, 461 and 509 us.  The power limit bounds both: 965 to 1000 W, SM
// clocks at 1.3 to 1.5 GHz of 1.97.  96 groups of 341 rows on average, 2048 -> 512, fp16:
// 90, 82 and 103 us for 369 MB each, 57 us at the measured copy bandwidth.
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

constexpr int kBM = 128;         // rows of a tile
constexpr int kBK = 64;          // contraction step: one 128-byte swizzle atom of 16-bit values
constexpr int kEpiWarps = 8;     // two for each quarter of the TMEM lanes, half of the columns each
// the producer and MMA issuer warps, these, and one that zeroes the weight gradient's partial steps
constexpr int threads_of(int mode) { return 64 + 32 * kEpiWarps + (mode == kGroupedWgrad ? 32 : 0); }
constexpr int kTileA = kBM * kBK * 2;

struct GP {
  const int* offsets;
  int G, R;
  int Mo;        // weight gradient: output rows of a group
  int No;        // output columns
  int Kc;        // forward, input gradient: contraction length
  int mt, nt;    // tiles of a group's output rows (weight gradient) and columns
  int slices;    // weight gradient: parts of a group's rows, each with an output of its own
  void* out;
  int64_t ldo;
  int out_dtype, accumulate;
  const void* bias;
  int bias_dtype;
  uint32_t idesc;
  int* status;
  uint64_t timeout_ns;
};

template <int BN, int STAGES>
struct Smem {
  static constexpr int kTileB = BN * kBK * 2;
  static constexpr int kStage = kTileA + kTileB;
  static constexpr int kOffB = STAGES * kTileA;
  static constexpr int kOffEpi = kOffB + STAGES * kTileB;       // 2 KiB per epilogue warp
  static constexpr int kOffBias = kOffEpi + kEpiWarps * 2048;   // 32 floats per epilogue warp
  static constexpr int kOffPre = kOffBias + kEpiWarps * 128;    // tile prefix of the groups, or their order
  static constexpr int kOffOff = kOffPre + (kGroupedMaxGroups + 2) * 4;  // offsets
  static constexpr int kOffBar = kOffOff + (kGroupedMaxGroups + 2) * 4;
  static constexpr int kBytes = kOffBar + (3 * STAGES + 4) * 8 + 16;
  static constexpr int kAlloc = kBytes + 1024;
  static_assert(kOffBar % 8 == 0, "barriers are 8-byte aligned");
  static_assert(kAlloc <= 227 * 1024, "shared memory of one CTA");
};

// Offsets are clamped to the rows, and a group starts at the largest offset up to its own, so that no
// two groups share a row whatever the offsets are (a row that two had would be written by two CTAs).
__device__ __forceinline__ int clamped(const GP& p, int g) { return min(max(p.offsets[g], 0), p.R); }

// The same rising offsets off[0 .. G] in shared memory, by a whole block of n threads.  Whether there
// were any that fell.
__device__ __forceinline__ bool load_offsets(const GP& p, int* off, int n) {
  bool fall = false;
  for (int g = threadIdx.x; g <= p.G; g += n) {
    const int a = p.offsets[g];
    off[g] = min(max(a, 0), p.R);
    fall |= p.offsets[min(g + 1, p.G)] < a;
  }
  fall = __syncthreads_or(fall);
  if (fall) {
    if (threadIdx.x == 0)
      for (int g = 1; g <= p.G; ++g) off[g] = max(off[g], off[g - 1]);
    __syncthreads();
  }
  return fall;
}

// The rows of one group by a whole warp, straight from the offsets: all of its loads at once.
__device__ __forceinline__ int2 group_range_warp(const GP& p, int g) {
  int lo = clamped(p, g);
  const int hi = clamped(p, g + 1);
  int top = lane_id() < g ? clamped(p, lane_id()) : 0;
  for (int o = lane_id() + 32; o < g; o += 32) top = max(top, clamped(p, o));
  if (__any_sync(0xffffffffu, top > lo)) lo = max(lo, __reduce_max_sync(0xffffffffu, top));
  return make_int2(lo, max(lo, hi));
}

struct Tile {
  int g, m0, n0;
  int lo, hi;    // rows: of the group, or of the weight gradient's slice
  int steps, slice;
};

constexpr int kSortGroups = 512;

// Walks this CTA's tiles in order.  The weight gradient's tiles differ in length: they
// come by falling size of their group, dealt out back and forth, so that every CTA gets about the
// same number of steps.
template <int MODE, int BN>
struct Walk {
  const GP& p;
  const int *off, *pre;
  int turn, me, step, total, g;
  __device__ Walk(const GP& p_, const int* off_, const int* pre_, int first, int step_)
      : p(p_), off(off_), pre(pre_), turn(0), me(first), step(step_),
        total(MODE == kGroupedWgrad ? p_.G * p_.mt * p_.nt * p_.slices : pre_[p_.G] * p_.nt), g(0) {}
  __device__ bool next(Tile& t) {
    int u = turn * step + me;
    if (MODE == kGroupedWgrad && (turn & 1)) u = turn * step + (step - 1 - me);
    if (u >= total) return false;  // so is every later one
    ++turn;
    const int n = u % p.nt;
    int m = u / p.nt;
    t.n0 = n * BN;
    t.slice = 0;
    if constexpr (MODE == kGroupedWgrad) {
      const int per = p.mt * p.slices, at = m / per;
      m -= at * per;
      t.slice = m / p.mt;
      m -= t.slice * p.mt;
      t.g = p.G <= kSortGroups ? pre[at] : at;
      const int2 r = make_int2(off[t.g], off[t.g + 1]);
      t.m0 = m * kBM;
      const int steps = (r.y - r.x + kBK - 1) / kBK;
      const int s0 = static_cast<int>(static_cast<int64_t>(steps) * t.slice / p.slices);
      const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (t.slice + 1) / p.slices);
      t.lo = r.x + s0 * kBK;
      t.hi = min(r.y, r.x + s1 * kBK);
      t.steps = s1 - s0;
    } else {
      while (pre[g + 1] <= m) ++g;
      m -= pre[g];
      const int2 r = make_int2(off[g], off[g + 1]);
      t.g = g;
      t.lo = r.x;
      t.hi = r.y;
      t.m0 = r.x + m * kBM;
      t.steps = (p.Kc + kBK - 1) / kBK;
    }
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

// 32 columns of 32 rows (lane = row) to out, through 2 KiB of shared memory: four lanes write 64
// bytes of one row (32 values of 16 bits, or 16 of fp32 at a time) instead of every lane 16 bytes
// of its own row.  16-byte pieces lie at piece ^ (row / 2 % 4): no bank is hit twice on either side.
__device__ __forceinline__ void store_chunk(const GP& p, const float (&v)[32], int64_t row0, int rows, int col, int64_t base,
                                            uint8_t* stage) {
  const int lane = lane_id(), q = lane & 3, key = (lane >> 1) & 3;
  if (p.out_dtype == kF32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = h * 16 + c * 4;
        *reinterpret_cast<float4*>(stage + lane * 64 + ((c ^ key) << 4)) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
      }
      __syncwarp();
      float* o = static_cast<float*>(p.out) + base + row0 * p.ldo + col + h * 16 + q * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 2);
        float4 u = *reinterpret_cast<const float4*>(stage + r * 64 + ((q ^ ((r >> 1) & 3)) << 4));
        if (r < rows && col + h * 16 + q * 4 < p.No) {
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
  for (int c = 0; c < 4; ++c) {
    uint4 u;
    u.x = pack2(v[8 * c], v[8 * c + 1], bf);
    u.y = pack2(v[8 * c + 2], v[8 * c + 3], bf);
    u.z = pack2(v[8 * c + 4], v[8 * c + 5], bf);
    u.w = pack2(v[8 * c + 6], v[8 * c + 7], bf);
    *reinterpret_cast<uint4*>(stage + lane * 64 + ((c ^ key) << 4)) = u;
  }
  __syncwarp();
  uint16_t* o = static_cast<uint16_t*>(p.out) + base + row0 * p.ldo + col + q * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2);
    const uint4 u = *reinterpret_cast<const uint4*>(stage + r * 64 + ((q ^ ((r >> 1) & 3)) << 4));
    if (r < rows && col + q * 8 < p.No) *reinterpret_cast<uint4*>(o + r * p.ldo) = u;
  }
  __syncwarp();
}

// Bytes of A that a CTA loads for the rows from row0 on: one box of 128 rows, or up to four of 16.
__device__ __forceinline__ int a_boxes(int rows) { return (max(rows, 0) + 15) >> 4; }
__device__ __forceinline__ uint32_t a_bytes(int rows) { return rows > 64 ? kTileA : a_boxes(rows) * 2048; }

// Keeps uses of a TMEM load's registers behind the wait for it.
__device__ __forceinline__ void regs_ready(uint32_t (&r)[32]) {
#pragma unroll
  for (int j = 0; j < 32; ++j) asm volatile("" : "+r"(r[j]));
}

// Rows outside every group (before the first, behind the last) become zeros.
__device__ __forceinline__ void zero_outside(const GP& p, const int* off, int warp, int warps) {
  const int lane = lane_id();
  const int first = off[0], last = off[p.G];
  const int64_t n = static_cast<int64_t>(first) + (p.R - last);
  for (int64_t i = warp; i < n; i += warps) {
    const int64_t r = i < first ? i : last + (i - first);
    const int es = p.out_dtype == kF32 ? 4 : 2, per = 16 / es;
    uint8_t* o = static_cast<uint8_t*>(p.out) + r * p.ldo * es;
    for (int c = lane * per; c < p.No; c += 32 * per) *reinterpret_cast<uint4*>(o + c * es) = make_uint4(0, 0, 0, 0);
  }
}

// Zeros in rows [r, r rounded up to 16) of `boxes` MN-major boxes (64 rows of 128 bytes) by one warp.
__device__ __forceinline__ void zero_rows(uint8_t* tile, int boxes, int r) {
  const int n = ((r + 15) & ~15) - r;
  for (int i = lane_id(); i < boxes * n * 8; i += 32) {
    const int box = i / (n * 8), j = i - box * n * 8;
    *reinterpret_cast<uint4*>(tile + box * 8192 + r * 128 + j * 16) = make_uint4(0, 0, 0, 0);
  }
}

// ta / tb: tiles of A and B; ta16: A in boxes of 16 rows (forward, input gradient).
template <int MODE, int BN, int STAGES>
__global__ void __launch_bounds__(threads_of(MODE), 1)
    grouped_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap ta16,
                   const __grid_constant__ CUtensorMap tb, const __grid_constant__ GP p) {
  using L = Smem<BN, STAGES>;
  constexpr bool A_MN = MODE == kGroupedWgrad, B_MN = MODE != kGroupedDgrad;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  int* pre = reinterpret_cast<int*>(sm + L::kOffPre);
  int* off = reinterpret_cast<int*>(sm + L::kOffOff);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::kOffBar);
  uint64_t* empty = full + STAGES;
  uint64_t* tail = empty + STAGES;  // a partial step has landed in this CTA
  uint64_t* acc_full = tail + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  const int warp = warp_id(), lane = lane_id();

  if (threadIdx.x == 0) {
    sm100::tma_prefetch_desc(&ta);
    sm100::tma_prefetch_desc(&tb);
    for (int s = 0; s < STAGES; ++s) {
      sm100::mbar_init(&full[s], 1);
      sm100::mbar_init(&empty[s], 1);
      sm100::mbar_init(&tail[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      sm100::mbar_init(&acc_full[b], 1);
      sm100::mbar_init(&acc_empty[b], kEpiWarps);
    }
    sm100::fence_mbar_init();
  }
  if (warp == 0) {
    sm100::tmem_alloc(slot, 2 * BN);
    sm100::tmem_relinquish();
  }
  load_offsets(p, off, threads_of(MODE));
  if constexpr (MODE != kGroupedWgrad) {
    if (warp == 1) {
      if (lane == 0) pre[0] = 0;
      int carry = 0;
      for (int g0 = 0; g0 < p.G; g0 += 32) {
        int v = g0 + lane < p.G ? (off[g0 + lane + 1] - off[g0 + lane] + kBM - 1) / kBM : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += up;
        }
        if (g0 + lane < p.G) pre[g0 + lane + 1] = carry + v;
        carry += __shfl_sync(0xffffffffu, v, 31);
      }
    }
  } else if (p.G <= kSortGroups) {  // by falling size, equal ones in order
    for (int g = threadIdx.x; g < p.G; g += threads_of(MODE)) {
      const int mine = off[g + 1] - off[g];
      int at = 0;
      for (int o = 0, from = off[0]; o < p.G; ++o) {
        const int to = off[o + 1], size = to - from;
        at += size > mine || (size == mine && o < g);
        from = to;
      }
      pre[at] = g;
    }
  }
  // A group that ends before it starts, or outside the rows, is reported.  (In load_offsets, in front
  // of everything else, this cost the forward product of 96 short groups 5 us of 90.)
  if (blockIdx.x == 0) {
    for (int g = threadIdx.x; g < p.G; g += threads_of(MODE))
      if (p.offsets[g] < 0 || p.offsets[g + 1] < p.offsets[g] || p.offsets[g + 1] > p.R)
        report_error(p.status, kIndexOutOfRange, g);
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *slot;
  Tile t;
  Walk<MODE, BN> walk(p, off, pre, blockIdx.x, gridDim.x);

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      while (ok && walk.next(t)) {
        for (int k = 0; k < t.steps; ++k, ++it) {
          const int s = it % STAGES;
          if (it >= STAGES && !sm100::mbar_wait(&empty[s], ((it / STAGES) - 1) & 1, p.timeout_ns, p.status, 400 + s)) {
            ok = false;
            break;
          }
          uint8_t* sa = sm + s * kTileA;
          uint8_t* sb = sm + L::kOffB + s * L::kTileB;
          if constexpr (MODE != kGroupedWgrad) {
            const int k0 = k * kBK, rows = t.hi - t.m0;
            sm100::mbar_arrive_expect_tx(&full[s], a_bytes(rows) + L::kTileB);
            if (rows > 64) {
              sm100::tma_load_2d(sa, &ta, &full[s], k0, t.m0);
            } else {
              for (int j = 0; j < a_boxes(rows); ++j) sm100::tma_load_2d(sa + j * 2048, &ta16, &full[s], k0, t.m0 + j * 16);
            }
            if constexpr (B_MN) {
#pragma unroll
              for (int j = 0; j < BN / 64; ++j) sm100::tma_load_3d(sb + j * 8192, &tb, &full[s], t.n0 + 64 * j, k0, t.g);
            } else {
              sm100::tma_load_3d(sb, &tb, &full[s], k0, t.n0, t.g);
            }
          } else {
            const int r0 = t.lo + k * kBK;
            uint64_t* bar = r0 + kBK <= t.hi ? &full[s] : &tail[s];
            sm100::mbar_arrive_expect_tx(bar, L::kStage);
            sm100::tma_load_2d(sa, &ta, bar, t.m0, r0);
            sm100::tma_load_2d(sa + 8192, &ta, bar, t.m0 + 64, r0);
#pragma unroll
            for (int j = 0; j < BN / 64; ++j) sm100::tma_load_2d(sb + j * 8192, &tb, bar, t.n0 + 64 * j, r0);
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    // One thread.  What it does between two steps' products is what the tensor
    // cores may wait for, so the next step's barrier is tried while this one's products are queued,
    // and descriptors are an addition each.
    if (lane == 0) {
      // 16 columns of a K-major row are 32 bytes, 16 rows of an MN-major box 2048
      constexpr int kStepA = (A_MN ? 2048 : 32) >> 4, kStepB = (B_MN ? 2048 : 32) >> 4;
      const uint64_t da0 = sm100::make_smem_desc(smem_u32(sm), A_MN ? 8192 : 16, 1024);
      const uint64_t db0 = sm100::make_smem_desc(smem_u32(sm + L::kOffB), B_MN ? 8192 : 16, 1024);
      uint32_t it = 0, i = 0;
      bool ok = true, ready = false;
      while (ok && walk.next(t)) {
        if (t.steps == 0) continue;
        const int buf = i & 1;
        const uint32_t d = tmem + buf * BN;
        const int last = MODE == kGroupedWgrad ? (t.hi - t.lo) - (t.steps - 1) * kBK : kBK;  // rows of the last step
        if (i >= 2 && !sm100::mbar_wait(&acc_empty[buf], ((i >> 1) - 1) & 1, p.timeout_ns, p.status, 420 + buf)) break;
        sm100::tc_fence_after();
        for (int k = 0; k < t.steps; ++k) {
          const int s = it % STAGES;
          if (!ready && !sm100::mbar_wait(&full[s], (it / STAGES) & 1, p.timeout_ns, p.status, 440 + s)) {
            ok = false;
            break;
          }
          sm100::tc_fence_after();
          const uint64_t da = da0 + static_cast<uint32_t>(s) * (kTileA >> 4), db = db0 + static_cast<uint32_t>(s) * (L::kTileB >> 4);
          if (MODE == kGroupedWgrad && k == t.steps - 1 && last <= kBK - 16) {
            for (int q = 0; q < (last + 15) / 16; ++q) sm100::mma_f16_ss(d, da + q * kStepA, db + q * kStepB, p.idesc, (k | q) != 0);
          } else {
#pragma unroll
            for (int q = 0; q < kBK / 16; ++q) sm100::mma_f16_ss(d, da + q * kStepA, db + q * kStepB, p.idesc, (k | q) != 0);
          }
          sm100::mma_commit(&empty[s]);
          ++it;
          ready = sm100::mbar_test_wait(&full[it % STAGES], (it / STAGES) & 1);
        }
        if (!ok) break;
        sm100::mma_commit(&acc_full[buf]);
        ++i;
      }
    }
    __syncwarp();
  } else if (MODE == kGroupedWgrad && warp == 2 + kEpiWarps) {
    // -------------------------------------------------------- partial steps
    // A stage's partial steps are waited for one after another: this warp completes each one (the
    // MMAs and the next load wait for it), so it is never a phase behind, nor ahead.
    uint32_t it = 0, tails = 0;
    while (MODE == kGroupedWgrad && walk.next(t)) {
      it += t.steps;
      const int last = (t.hi - t.lo) - (t.steps - 1) * kBK;
      if (t.steps == 0 || last == kBK) continue;
      const int s = (it - 1) % STAGES;
      if (!__all_sync(0xffffffffu, sm100::mbar_wait(&tail[s], (tails >> s) & 1, p.timeout_ns, p.status, 480 + s))) break;
      tails ^= 1u << s;
      zero_rows(sm + s * kTileA, 2, last);
      zero_rows(sm + L::kOffB + s * L::kTileB, BN / 64, last);
      sm100::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&full[s]);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;  // the TMEM lanes that this warp may read
    const int c0 = ((warp - 2) >> 2) * (BN / 2);
    uint8_t* stage = sm + L::kOffEpi + (warp - 2) * 2048;
    float* bias = reinterpret_cast<float*>(sm + L::kOffBias + (warp - 2) * 128);
    if constexpr (MODE != kGroupedWgrad) zero_outside(p, off, blockIdx.x * kEpiWarps + warp - 2, gridDim.x * kEpiWarps);
    uint32_t i = 0;
    while (walk.next(t)) {
      const int buf = i & 1;
      const bool any = t.steps > 0;
      const int row0 = t.m0 + quarter * 32;
      const int rows = min(32, (MODE == kGroupedWgrad ? p.Mo : t.hi) - row0);
      const int chunks = rows > 0 ? min(BN / 64, (p.No - t.n0 - c0 + 31) / 32) : 0;  // of 32 columns, with some inside
      const int64_t base = MODE == kGroupedWgrad ? (static_cast<int64_t>(t.slice) * p.G + t.g) * p.Mo * p.ldo : 0;
      float ahead[BN / 64];  // this lane's column of each chunk: asked for before the products are done
      if (MODE == kGroupedFwd && p.bias != nullptr) {
#pragma unroll
        for (int c = 0; c < BN / 64; ++c) {
          const int col = t.n0 + c0 + c * 32 + lane;
          ahead[c] = col < p.No ? load_any(p.bias, static_cast<int64_t>(t.g) * p.No + col, p.bias_dtype) : 0.f;
        }
      }
      auto finish = [&](uint32_t (&r)[32], int c, float b0) {
        const int col = t.n0 + c0 + c * 32;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
        if (MODE == kGroupedFwd && p.bias != nullptr) {
          bias[lane] = b0;
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 b = *reinterpret_cast<const float4*>(bias + j);
            v[j] += b.x, v[j + 1] += b.y, v[j + 2] += b.z, v[j + 3] += b.w;
          }
        }
        store_chunk(p, v, row0, rows, col, base, stage);
      };
      if (any) {
        const bool ok = sm100::mbar_wait(&acc_full[buf], (i >> 1) & 1, p.timeout_ns, p.status, 460 + buf);
        if (!__all_sync(0xffffffffu, ok)) break;
        sm100::tc_fence_after();
        const uint32_t at = tmem + buf * BN + c0 + (static_cast<uint32_t>(quarter * 32) << 16);
        uint32_t ra[32], rb[32];  // the next chunk is on its way while one is written
        if (chunks > 0) sm100::tmem_ld_32x32b_x32(at, ra);
#pragma unroll
        for (int c = 0; c < BN / 64; c += 2) {
          if (c >= chunks) break;
          sm100::tmem_ld_wait();
          regs_ready(ra);
          if (c + 1 < chunks) sm100::tmem_ld_32x32b_x32(at + (c + 1) * 32, rb);
          finish(ra, c, ahead[c]);
          if (c + 1 < BN / 64 && c + 1 < chunks) {
            sm100::tmem_ld_wait();
            regs_ready(rb);
            if (c + 2 < chunks) sm100::tmem_ld_32x32b_x32(at + (c + 2) * 32, ra);
            finish(rb, c + 1, ahead[c + 1 < BN / 64 ? c + 1 : c]);
          }
        }
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&acc_empty[buf]);
        ++i;
      } else if (!p.accumulate) {  // a group without rows has a gradient of zeros
        uint32_t zero[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) zero[j] = 0u;
        for (int c = 0; c < chunks; ++c) finish(zero, c, 0.f);
      }
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 0) sm100::tmem_dealloc(tmem, 2 * BN);
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

// Sets a kernel's shared-memory limit once per device; returns the current device's SMs (one CTA each).
int prepare(const void* kern, int smem, int (&sms)[kMaxDevices]) {
  static std::mutex mu;
  int dev = 0;
  FLARE_CUDA_CHECK(cudaGetDevice(&dev));
  FLARE_CHECK(dev >= 0 && dev < kMaxDevices, "device index");
  std::lock_guard<std::mutex> lock(mu);
  if (sms[dev] == 0) {
    FLARE_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    FLARE_CUDA_CHECK(cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev));
  }
  return sms[dev];
}

template <int MODE, int BN, int STAGES>
void launch(const GroupedArgs& a, cudaStream_t s, int slices = 1) {
  using L = Smem<BN, STAGES>;
  GP p{};
  p.offsets = a.offsets;
  p.G = a.G;
  p.R = static_cast<int>(a.R);
  p.Mo = a.K;
  p.No = MODE == kGroupedDgrad ? a.K : a.N;
  p.Kc = MODE == kGroupedDgrad ? a.N : a.K;
  p.mt = ceil_div(a.K, kBM);
  p.nt = ceil_div(p.No, BN);
  p.slices = slices;
  p.out = slices > 1 ? a.work : a.out;
  p.ldo = p.No;
  p.out_dtype = slices > 1 ? kF32 : a.out_dtype;
  p.accumulate = slices > 1 ? 0 : a.accumulate;
  p.bias = MODE == kGroupedFwd ? a.bias : nullptr;
  p.bias_dtype = a.bias_dtype;
  p.idesc = sm100::make_idesc_16bit(kBM, BN, MODE == kGroupedWgrad, MODE != kGroupedDgrad, a.dtype == kBF16);
  p.status = a.status;
  p.timeout_ns = a.timeout_ns;
  CUtensorMap ta, ta16, tb;
  if (MODE == kGroupedWgrad) {
    ta = map2(a.x, a.dtype, a.K, a.R, a.ldx, kBK);
    tb = map2(a.dy, a.dtype, a.N, a.R, a.lddy, kBK);
    ta16 = ta;
  } else {
    const int64_t wd[3] = {a.N, a.K, a.G}, wp[2] = {a.N, static_cast<int64_t>(a.K) * a.N};
    const int box_fwd[3] = {64, kBK, 1}, box_bwd[3] = {64, BN, 1};
    tb = make_map(a.w, a.dtype, 3, wd, wp, MODE == kGroupedFwd ? box_fwd : box_bwd);
    const void* rows = MODE == kGroupedFwd ? a.x : a.dy;
    const int64_t ld = MODE == kGroupedFwd ? a.ldx : a.lddy;
    ta = map2(rows, a.dtype, p.Kc, a.R, ld, 128);
    ta16 = map2(rows, a.dtype, p.Kc, a.R, ld, 16);
  }
  // as many tiles as there can be: the groups' sizes are on the device
  const int64_t tiles = MODE == kGroupedWgrad
                            ? static_cast<int64_t>(a.G) * p.mt * p.nt * slices
                            : (a.R / kBM + std::min<int64_t>(a.G, a.R)) * p.nt;
  FLARE_CHECK(tiles < (1ll << 31) - 65536, "grouped products: too many tiles");
  static int sms[kMaxDevices];
  auto kern = grouped_kernel<MODE, BN, STAGES>;
  const int64_t grid = std::min<int64_t>(std::max<int64_t>(1, tiles), prepare(reinterpret_cast<const void*>(kern), L::kAlloc, sms));
  kern<<<static_cast<int>(grid), threads_of(MODE), L::kAlloc, s>>>(ta, ta16, tb, p);
  FLARE_CUDA_CHECK(cudaGetLastError());
  count_launch();
}

// The weight gradient's tiles are as wide as N allows.  A few groups of a small weight and many
// rows leave most of the machine idle: their rows are cut into slices of at least 512 rows of an
// average group, about two tiles for each SM (33 us against 630 us for 131072 x 64 x 128 in 2 groups).
// And whatever the groups, a slice has 2^25 rows at most: one group may have nearly all of them, and
// the waits for a tile's end are bounded by time.
constexpr int64_t kMaxSliceRows = 1 << 25;
struct WgradShape {
  int bn, slices;
};
WgradShape wgrad_shape(int G, int64_t R, int K, int N) {
  WgradShape w;
  w.bn = N > 128 ? 256 : N > 64 ? 128 : 64;
  const int64_t tiles = static_cast<int64_t>(G) * ceil_div(K, 128) * ceil_div(N, w.bn);
  w.slices = static_cast<int>(std::max<int64_t>({1, ceil_div(R, kMaxSliceRows), std::min<int64_t>({64, R / G / 512, 296 / tiles})}));
  return w;
}

__global__ void __launch_bounds__(256) add_slices_kernel(const float* part, int64_t n, int slices, void* out, int dtype, int accumulate) {
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4; i < n; i += static_cast<int64_t>(gridDim.x) * 1024) {
    float4 v = *reinterpret_cast<const float4*>(part + i);
#pragma unroll 4
    for (int s = 1; s < slices; ++s) v = f4_add(v, *reinterpret_cast<const float4*>(part + s * n + i));
    if (dtype == kF32) {
      float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + i);
      *o = accumulate ? f4_add(*o, v) : v;
    } else {
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i) = make_uint2(pack2(v.x, v.y, dtype == kBF16), pack2(v.z, v.w, dtype == kBF16));
    }
  }
}

// The widest tile that still gives half of the SMs one (3003 rows of 200 x 328 in 7 groups: 10.4 us
// at 256 columns, 8.4 us at 128; 400 rows of 2048 x 512 in 8: 21 us at 256, 17 us at 64).
template <int MODE>
void pick(const GroupedArgs& a, cudaStream_t s) {
  const int no = MODE == kGroupedDgrad ? a.K : a.N;
  const int64_t mt = a.R / kBM + std::min<int64_t>(a.G, a.R);
  int bn = 256;
  while (bn > 64 && (no <= bn / 2 || mt * ceil_div(no, bn) < 74)) bn /= 2;
  if (bn == 256) launch<MODE, 256, 4>(a, s);
  else if (bn == 128) launch<MODE, 128, 6>(a, s);
  else launch<MODE, 64, 8>(a, s);
}

void wgrad(const GroupedArgs& a, cudaStream_t s) {
  const WgradShape w = wgrad_shape(a.G, a.R, a.K, a.N);
  if (w.bn == 256) launch<kGroupedWgrad, 256, 4>(a, s, w.slices);
  else if (w.bn == 128) launch<kGroupedWgrad, 128, 6>(a, s, w.slices);
  else launch<kGroupedWgrad, 64, 8>(a, s, w.slices);
  if (w.slices > 1) {
    const int64_t n = static_cast<int64_t>(a.G) * a.K * a.N;
    add_slices_kernel<<<static_cast<int>(std::min<int64_t>((n + 1023) / 1024, 148 * 8)), 256, 0, s>>>(
        static_cast<const float*>(a.work), n, w.slices, a.out, a.out_dtype, a.accumulate);
    FLARE_CUDA_CHECK(cudaGetLastError());
    count_launch();
  }
}

// ------------------------------------------------------------- cluster sums
// The CTAs of a cluster hold partial sums in shared memory; rank 0 adds them in order of rank.
__device__ __forceinline__ float cluster_value(const float* local, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(sm100::mapa_shared(local, rank)) : "memory");
  return v;
}

template <typename... Args>
void launch_cluster(void (*kern)(Args...), dim3 grid, int threads, int cluster_z, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = cluster_z;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  FLARE_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, args...));
  count_launch();
}

__device__ __forceinline__ void store_any(void* p, int64_t i, int dtype, float v) {
  if (dtype == kF32) static_cast<float*>(p)[i] = v;
  else if (dtype == kBF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// ---------------------------------------------------------------- few rows
// A serving step has a row or two in each chosen group: what counts is to stream those groups'
// weights with every SM at work, and the tensor cores would multiply tiles of nothing.
// Block = 64 columns of one chosen group (blockIdx.y-th of those that have rows), one slice of K
// (a cluster's CTAs share the columns and K).  A thread owns 8 columns (one 16-byte load of a
// weight row) of every 32nd row of the slice and up to MR rows of x; its partial sums meet by
// shuffles, then through shared memory, then across the cluster, always in the same order.
// Eight rows in as many groups of 16, 512 -> 4096: 7.2 us for 34 MB of weights (5.2 us at the
// measured copy bandwidth; the launch is about 2); 2048 -> 512: 7.1 us for 17 MB.  Both with the
// weights in L2, one launch after another.
constexpr int kFewK = 512;  // a chunk of K whose x values are in shared memory
constexpr int kFewRows = 4; // of a group at a time: 32 sums a thread, three blocks on an SM
template <typename T, int MR>
__device__ __forceinline__ void few_rows(const GroupedArgs& a, int g, int r0, int nr, int k0, int k1, float (*xs)[kFewRows],
                                         float (*part)[kFewRows][64]) {
  const int c8 = threadIdx.x & 7, kl = threadIdx.x >> 3, warp = warp_id(), lane = lane_id();
  const int col = blockIdx.x * 64 + c8 * 8;
  const bool in = col < a.N;
  const T* w = static_cast<const T*>(a.w) + (static_cast<int64_t>(g) * a.K) * a.N + col;
  float acc[MR][8];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[m][i] = 0.f;
  auto fetch = [&](uint4 (&u)[4], int kc, int kk, int kn) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      u[q] = in && kk + 32 * q < kn ? __ldg(reinterpret_cast<const uint4*>(w + static_cast<int64_t>(kc + kk + 32 * q) * a.N))
                                    : make_uint4(0, 0, 0, 0);
  };
  for (int kc = k0; kc < k1; kc += kFewK) {
    const int kn = min(kFewK, k1 - kc);
    uint4 u[4];
    fetch(u, kc, kl, kn);  // the first weights are on their way while x is fetched
    __syncthreads();
    const int m = threadIdx.x >> 6;  // a quarter of the block for each row
    if (m < nr) {
      const int row = a.rows != nullptr ? a.rows[r0 + m] : r0 + m;
      const bool live = row >= 0 && row < a.x_rows;
      const T* x = static_cast<const T*>(a.x) + row * a.ldx + kc;
      for (int k = (threadIdx.x & 63); k < kn; k += 64) xs[k][m] = live ? to_f32(x[k]) : 0.f;
    }
    __syncthreads();
    for (int kk = kl; kk < kn; kk += 128) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (kk + 32 * q < kn) {
          const T* wv = reinterpret_cast<const T*>(&u[q]);
          float x[MR];
#pragma unroll
          for (int j = 0; j < MR; ++j) x[j] = xs[kk + 32 * q][j];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float f = to_f32(wv[i]);
#pragma unroll
            for (int j = 0; j < MR; ++j) acc[j][i] = fmaf(x[j], f, acc[j][i]);
          }
        }
      }
      if (kk + 128 < kn) fetch(u, kc, kk + 128, kn);
    }
  }
#pragma unroll
  for (int j = 0; j < MR; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = acc[j][i];
      v += __shfl_xor_sync(0xffffffffu, v, 8);
      v += __shfl_xor_sync(0xffffffffu, v, 16);
      if (lane < 8) part[warp][j][c8 * 8 + i] = v;
    }
}

template <typename T>
__global__ void __launch_bounds__(256, 3) few_rows_kernel(GroupedArgs a, int slices) {
  __shared__ float xs[kFewK][kFewRows];
  __shared__ float part[8][kFewRows][64];
  __shared__ float sum[kFewRows][64];
  __shared__ int found, found_lo, found_hi, top[8];
  const int lane = lane_id();
  const uint32_t rank = blockIdx.z;
  const int R = static_cast<int>(a.R);
  const GP p{a.offsets, a.G, R};
  if (threadIdx.x < 32) {  // the blockIdx.y-th group with rows, and those rows
    int seen = 0, g = -1, run = 0;  // run: the largest offset so far, where the next group starts at least
    for (int g0 = 0; g0 < a.G && g < 0; g0 += 32) {
      int lo = clamped(p, min(g0 + lane, a.G));
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, lo, o);
        if (lane >= o) lo = max(lo, up);
      }
      lo = max(lo, run);
      run = __shfl_sync(0xffffffffu, lo, 31);
      const int hi = max(lo, clamped(p, min(g0 + lane + 1, a.G)));
      const unsigned m = __ballot_sync(0xffffffffu, hi > lo);
      const int n = __popc(m), want = static_cast<int>(blockIdx.y) - seen;
      if (want < n) {  // the want-th set bit: the lane with that many below it
        const bool mine = hi > lo && __popc(m & ((1u << lane) - 1u)) == want;
        g = g0 + __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
        if (mine) found_lo = lo, found_hi = hi;
      }
      seen += n;
    }
    if (lane == 0) found = g;
  }
  const bool lead = blockIdx.y == 0 && rank == 0;
  if (lead) {
    int last = 0;
    for (int g = threadIdx.x; g <= a.G; g += 256) last = max(last, clamped(p, g));
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0) top[warp_id()] = last;
    if (blockIdx.x == 0) {
      for (int g = threadIdx.x; g < a.G; g += 256)
        if (a.offsets[g] < 0 || a.offsets[g + 1] < a.offsets[g] || a.offsets[g + 1] > R) report_error(a.status, kIndexOutOfRange, g);
    }
  }
  __syncthreads();
  if (lead) {  // rows of no group
    int first = clamped(p, 0), last = 0;
#pragma unroll
    for (int q = 0; q < 8; ++q) last = max(last, top[q]);
    if (first > 0 || last < R) {
      for (int i = threadIdx.x; i < R * 64; i += 256) {
        const int r = i >> 6, c = blockIdx.x * 64 + (i & 63);
        if ((r < first || r >= last) && c < a.N) store_any(a.out, static_cast<int64_t>(r) * a.N + c, a.out_dtype, 0.f);
      }
    }
  }
  const int g = found;
  if (g < 0) return;  // every CTA of the cluster
  const int2 rg = make_int2(found_lo, found_hi);
  const int per = (a.K + slices - 1) / slices, k0 = min(a.K, static_cast<int>(rank) * per), k1 = min(a.K, k0 + per);
  for (int r0 = rg.x; r0 < rg.y; r0 += kFewRows) {
    const int nr = min(kFewRows, rg.y - r0);
    if (nr == 1) few_rows<T, 1>(a, g, r0, nr, k0, k1, xs, part);
    else if (nr == 2) few_rows<T, 2>(a, g, r0, nr, k0, k1, xs, part);
    else few_rows<T, 4>(a, g, r0, nr, k0, k1, xs, part);
    __syncthreads();
    for (int i = threadIdx.x; i < nr * 64; i += 256) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) v += part[q][i >> 6][i & 63];
      sum[i >> 6][i & 63] = v;
    }
    if (slices > 1) sm100::cluster_sync();
    else __syncthreads();
    if (rank == 0) {
      for (int i = threadIdx.x; i < nr * 64; i += 256) {
        const int c = blockIdx.x * 64 + (i & 63);
        if (c >= a.N) continue;
        float v = sum[i >> 6][i & 63];
        for (int q = 1; q < slices; ++q) v += cluster_value(&sum[i >> 6][i & 63], q);
        if (a.bias != nullptr) v += load_any(a.bias, static_cast<int64_t>(g) * a.N + c, a.bias_dtype);
        store_any(a.out, static_cast<int64_t>(r0 + (i >> 6)) * a.N + c, a.out_dtype, v);
      }
    }
    if (slices > 1) sm100::cluster_sync();  // the sums are read before they are overwritten, or their CTA leaves
    else __syncthreads();
  }
}

// Column slices that fill the machine about twice over: K is cut where groups and columns are few.
int slices_for(int64_t blocks, int64_t length, int64_t least) {
  int n = 1;
  while (n < 8 && blocks * n < 296 && length >= 2 * n * least) n *= 2;
  return n;
}

void few_rows_launch(const GroupedArgs& a, cudaStream_t s) {
  const int groups = static_cast<int>(std::min<int64_t>(a.G, a.R)), cols = ceil_div(a.N, 64);
  const int slices = slices_for(static_cast<int64_t>(groups) * cols, a.K, 128);
  const dim3 grid(cols, groups, slices);
  if (a.dtype == kBF16) launch_cluster(few_rows_kernel<__nv_bfloat16>, grid, 256, slices, s, a, slices);
  else launch_cluster(few_rows_kernel<__half>, grid, 256, slices, s, a, slices);
}

// ------------------------------------------------------- per-group column sums
// Many rows: rows are cut into chunks of equal length whatever the groups' sizes (by group, the
// fullest one holds up the others: 517 us against 173 us for 131072 x 4096 in 32 groups).  Block =
// 256 columns (a warp reads 512 bytes of a row) of one chunk; each group's part of the chunk is a
// segment of its own, number chunk + group: one of the two grows from a segment to the next.  A
// second kernel adds a group's segments in order.
// Up to kSumOneLaunch rows: one kernel, block = 64 columns of a slice of one group, slices of a
// group a cluster, added in order (3003 x 328: 4.8 us against 12 us for the two kernels).
// 131072 x 4096: 173 + 9 us, 1.07 GB at 5.9 TB/s.  Added up by warps of the weight gradient from its
// stages instead, the columns cost that kernel 120 to 150 us: its four stages could not spare them.
constexpr int64_t kSumOneLaunch = 8192;
int sum_rows(int64_t R, int cols) {  // about eight blocks for each SM
  return static_cast<int>(std::max<int64_t>(32, std::min<int64_t>(512, R * cols / 1184 / 32 * 32)));
}

template <typename T>
__global__ void __launch_bounds__(256) group_sum_small_kernel(GroupSumArgs a, int slices) {
  __shared__ float red[8][64];
  __shared__ float sum[64];
  const int g = blockIdx.y, lane = lane_id(), warp = warp_id(), c8 = threadIdx.x & 7;
  const uint32_t rank = blockIdx.z;
  const GP p{a.offsets, a.G, static_cast<int>(a.R)};
  const int c = blockIdx.x * 64 + c8 * 8;
  float acc[8];
  auto add = [&](int2 rg) {
    const int per = (rg.y - rg.x + slices - 1) / slices;
    const int r0 = min(rg.y, rg.x + static_cast<int>(rank) * per), r1 = min(rg.y, r0 + per);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    if (c < a.N) {
#pragma unroll 8
      for (int r = r0 + (threadIdx.x >> 3); r < r1; r += 32) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.y) + r * a.ldy + c));
        const T* v = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += to_f32(v[i]);
      }
    }
  };
  // the group's own offsets, and once more where an earlier one is larger (in one, 6.2 us instead of 5.0)
  const int2 own = make_int2(clamped(p, g), max(clamped(p, g), clamped(p, g + 1)));
  add(own);
  const int2 rg = group_range_warp(p, g);
  if (rg.x != own.x) add(rg);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 8);
    acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 16);
    if (lane < 8) red[warp][c8 * 8 + i] = acc[i];
  }
  __syncthreads();
  float v = 0.f;
  if (threadIdx.x < 64) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v += red[i][threadIdx.x];
    sum[threadIdx.x] = v;
  }
  if (slices > 1) sm100::cluster_sync();
  const int col = blockIdx.x * 64 + threadIdx.x;
  if (rank == 0 && threadIdx.x < 64 && col < a.N) {
    for (int q = 1; q < slices; ++q) v += cluster_value(&sum[threadIdx.x], q);
    const int64_t o = static_cast<int64_t>(g) * a.N + col;
    if (a.accumulate) v += static_cast<const float*>(a.out)[o];
    store_any(a.out, o, a.out_dtype, v);
  }
  if (slices > 1) sm100::cluster_sync();
}

template <typename T>
__global__ void __launch_bounds__(256) group_part_kernel(GroupSumArgs a, int rows) {
  __shared__ float red[8][256];
  extern __shared__ int off[];  // [G + 1]
  const GP p{a.offsets, a.G, static_cast<int>(a.R)};
  const int lane = lane_id(), warp = warp_id(), chunk = blockIdx.x;
  const int c0 = chunk * rows, c1 = min(p.R, c0 + rows), c = blockIdx.y * 256 + lane * 8;
  const bool falls = load_offsets(p, off, 256);
  auto sums = [&](auto range) {
    int lo = 0, hi = a.G;  // the first group that ends behind c0
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (off[mid + 1] > c0) hi = mid;
      else lo = mid + 1;
    }
    for (int g = lo; g < a.G; ++g) {
      const int2 rg = range(g);
      if (rg.x >= c1) break;
      const int r0 = max(rg.x, c0), r1 = min(rg.y, c1);
      if (r0 >= r1) continue;
      float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (c < a.N) {
#pragma unroll 8
        for (int r = r0 + warp; r < r1; r += 8) {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.y) + r * a.ldy + c));
          const T* v = reinterpret_cast<const T*>(&u);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] += to_f32(v[i]);
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) red[warp][lane * 8 + i] = acc[i];
      __syncthreads();
      const int col = blockIdx.y * 256 + threadIdx.x;
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v += red[i][threadIdx.x];
      if (col < a.N) a.work[static_cast<int64_t>(chunk + g) * a.N + col] = v;
    }
  };
  // The rows of a group are read from the offsets themselves where these rise: with the ones in shared
  // memory as bounds of the loop, 131072 x 4096 took 190 us instead of 170.
  if (falls) sums([&](int g) { return make_int2(off[g], off[g + 1]); });
  else sums([&](int g) { return make_int2(clamped(p, g), clamped(p, g + 1)); });
}

__global__ void __launch_bounds__(256) group_sum_kernel(GroupSumArgs a, int rows) {
  const int g = blockIdx.x, col = blockIdx.y * 256 + threadIdx.x;
  const int2 rg = group_range_warp(GP{a.offsets, a.G, static_cast<int>(a.R)}, g);
  if (col >= a.N) return;
  float v = 0.f;
  if (rg.y > rg.x) {
#pragma unroll 4
    for (int c = rg.x / rows; c <= (rg.y - 1) / rows; ++c) v += a.work[static_cast<int64_t>(c + g) * a.N + col];
  }
  const int64_t o = static_cast<int64_t>(g) * a.N + col;
  if (a.accumulate) v += static_cast<const float*>(a.out)[o];
  store_any(a.out, o, a.out_dtype, v);
}

}  // namespace

void grouped_gemm(const GroupedArgs& a, cudaStream_t s) {
  FLARE_CHECK(a.dtype == kBF16 || a.dtype == kF16, "grouped products take bf16 or fp16");
  FLARE_CHECK(a.G > 0 && a.G <= kGroupedMaxGroups, "grouped products: 1 to 2048 groups");
  FLARE_CHECK(a.K > 0 && a.N > 0 && a.K % 8 == 0 && a.N % 8 == 0, "grouped products: widths must be multiples of 8");
  FLARE_CHECK(a.R >= 0 && a.R < (1ll << 31) - 512 && a.x_rows < (1ll << 31) - 512, "grouped products: too many rows");
  FLARE_CHECK(a.rows == nullptr || (a.mode == kGroupedFwd && grouped_few_rows(a.R)), "grouped products: rows are gathered beforehand");
  // a thread of the autograd engine may not have the device's context yet, and encoding a tensor map needs one
  int dev = 0;
  FLARE_CUDA_CHECK(cudaGetDevice(&dev));
  FLARE_CUDA_CHECK(cudaSetDevice(dev));
  switch (a.mode) {
    case kGroupedFwd:
      if (a.R == 0) return;
      if (grouped_few_rows(a.R)) few_rows_launch(a, s);
      else pick<kGroupedFwd>(a, s);
      break;
    case kGroupedDgrad:
      if (a.R == 0) return;
      pick<kGroupedDgrad>(a, s);
      break;
    default:
      wgrad(a, s);
      break;
  }
}

int64_t grouped_work_floats(int G, int64_t R, int K, int N) {
  const int slices = wgrad_shape(G, R, K, N).slices;
  return slices > 1 ? static_cast<int64_t>(slices) * G * K * N : 0;
}

// 12 us against 16 us for 16 rows of 2048 x 512 in 16 groups, 18 us against 16 us for 32.
bool grouped_few_rows(int64_t rows) { return rows <= 16; }

int64_t group_sum_work_floats(int G, int64_t R, int N) {
  return R <= kSumOneLaunch ? 0 : (ceil_div(R, sum_rows(R, ceil_div(N, 256))) + static_cast<int64_t>(G)) * N;
}

void group_colsum(const GroupSumArgs& a, cudaStream_t s) {
  FLARE_CHECK(a.G > 0 && a.G <= kGroupedMaxGroups, "grouped products: 1 to 2048 groups");
  if (a.R <= kSumOneLaunch) {
    const int cols = ceil_div(a.N, 64), slices = slices_for(static_cast<int64_t>(a.G) * cols, a.R / a.G, 128);
    const dim3 grid(cols, a.G, slices);
    if (a.dtype == kBF16) launch_cluster(group_sum_small_kernel<__nv_bfloat16>, grid, 256, slices, s, a, slices);
    else launch_cluster(group_sum_small_kernel<__half>, grid, 256, slices, s, a, slices);
    return;
  }
  const int cols = ceil_div(a.N, 256), rows = sum_rows(a.R, cols);
  const dim3 grid(ceil_div(a.R, rows), cols);
  const int smem = (a.G + 1) * 4;
  if (a.dtype == kBF16) group_part_kernel<__nv_bfloat16><<<grid, 256, smem, s>>>(a, rows);
  else group_part_kernel<__half><<<grid, 256, smem, s>>>(a, rows);
  FLARE_CUDA_CHECK(cudaGetLastError());
  group_sum_kernel<<<dim3(a.G, cols), 256, 0, s>>>(a, rows);
  FLARE_CUDA_CHECK(cudaGetLastError());
  count_launch(2);
}

}  // namespace flare
