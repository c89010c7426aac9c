// pkt_fp8_gemm: out = sum over blocks kb of 128 along K of
//   scale_a[kb, m] scale_b[kb, n] * sum over k in kb of a[m, k] b[n, k],
// e4m3 / e5m2 operands on tcgen05 (kind::f8f6f4), fp32 throughout.
//
// The scales change every 128 values of K, so a tensor-core accumulator holds one
// block of K only: the MMA issuer writes each block's product to the next of
// several TMEM buffers (4 MMAs of K = 32) and the epilogue warps read it back,
// multiply by the block's scales and add to accumulators in their registers, while
// the MMAs of the next blocks run. One fp32 FMA per output value and block of 128.
//
// Roles of a CTA: warps 0..3 (0..7) epilogue, one per 32 TMEM lanes (and half of the
// columns); then one TMA producer warp and one MMA issuer warp. Operand tiles are
// 128-byte rows (128 values of K) in 128B-swizzled shared memory, in a ring of stages.
//
// "Rows" below are the operand whose 128 rows lie along the TMEM lanes, "cols" the one
// along the columns of a tile. For few output rows (M) the operands change places, so
// that the 128 lanes are filled by the weights and the columns by the few tokens.
// When there are few tiles, the CTAs of a cluster split K between them and add their
// accumulators through distributed shared memory in rank order.
//
// Every wait is bounded (2 s); one that runs out sets a status word that
// pkt_fp8_gemm_status reads, and the kernel drains its copies and returns.
#include <algorithm>
#include <atomic>

#include "ops_common.h"
#include "ops_device.cuh"

namespace pkb {
namespace {

constexpr int kRows = 128;    // TMEM lanes
constexpr int kKBytes = 128;  // one block of K: a 128-byte row of an operand tile
constexpr unsigned long long kWaitNs = 2000000000ull;

__device__ int g_fp8_status;

struct alignas(64) Fp8Args {
  CUtensorMap map_r, map_c;
  int rows, cols, num_kb;
  int tiles_r, tiles_c;
  const float *scale_r, *scale_c;
  long long ld_r, ld_c;
  int r_shift, c_shift;  // log2 of the rows that share a scale (0 or 7)
  void* out;
  long long ldo;
  int out_bf16, swap, wide;  // swap: out[col * ldo + row]; wide: 16-byte stores along out's rows
  uint32_t idesc;
};

template <int BN, int PAIR>
struct Shape {
  static constexpr int kHalves = BN > 128 ? 2 : 1;   // epilogue warps per 32 lanes
  static constexpr int kCols = BN / kHalves;         // columns of an epilogue warp
  static constexpr int kEpiWarps = 4 * kHalves;
  static constexpr int kThreads = 32 * (kEpiWarps + (kHalves == 2 ? 4 : 2));
  static constexpr int kRowBytes = kRows * kKBytes;
  static constexpr int kColBytes = BN / PAIR * kKBytes;
  static constexpr int kStageBytes = kRowBytes + kColBytes;
  static constexpr int kStages = kStageBytes >= 32768 ? 6 : 8;
  static constexpr int kBufs = BN > 128 ? 2 : 4;     // TMEM accumulators
  static constexpr int kTmemCols = kBufs * BN < 32 ? 32 : kBufs * BN;
  static constexpr int kChunk = kCols < 32 ? kCols : 32;  // columns per TMEM load
};

template <int BN, int PAIR>
struct Smem {
  using S = Shape<BN, PAIR>;
  uint8_t stages[S::kStages][S::kStageBytes];
  float col_scale[S::kEpiWarps][S::kCols];
  uint64_t full[S::kStages], empty[S::kStages];
  uint64_t tfull[S::kBufs], tempty[S::kBufs];
  uint64_t drain;
  uint32_t tmem;
  int abort;
};

template <bool CL>
__device__ __forceinline__ bool wait_once(uint64_t* bar, uint32_t parity) {
  return CL ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity);
}

// Waits until the phase of `parity` has completed; false when the time ran out here
// or somewhere else in the CTA.
template <bool CL>
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, int* abort) {
  if (wait_once<CL>(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  uint32_t it = 0;
  while (!wait_once<CL>(bar, parity)) {
    if ((++it & 31u) == 0) {
      if (*reinterpret_cast<volatile int*>(abort)) return false;
      if (globaltimer_ns() - t0 > kWaitNs) {
        *reinterpret_cast<volatile int*>(abort) = 1;
        atomicExch(&g_fp8_status, PKT_DEV_TIMEOUT_PIPE);
        return false;
      }
    }
  }
  return true;
}

template <int PAIR>
__device__ __forceinline__ void mma_fp8(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
  if (PAIR == 2)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) {
  tmem_ld32(taddr, r);
  tmem_ld_wait_regs(r);
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// Two fp32 lanes in one 64-bit register.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Tiles in groups of 8 tile rows swept column by column: what runs at the same time
// shares operand tiles in L2.
__device__ __forceinline__ void tile_at(int t, int tiles_r, int tiles_c, int* tr, int* tc) {
  constexpr int kGroup = 8;
  const int per = kGroup * tiles_c, g = t / per, r0 = g * kGroup, rows = min(kGroup, tiles_r - r0), in = t - g * per;
  *tr = r0 + in % rows;
  *tc = in / rows;
}

// One value to out at (row, col) of the tile's orientation.
__device__ __forceinline__ void store_one(const Fp8Args& a, int row, int col, float v) {
  const long long at = a.swap ? (long long)col * a.ldo + row : (long long)row * a.ldo + col;
  if (a.out_bf16)
    static_cast<uint16_t*>(a.out)[at] = f32_to_bf16_rn(v);
  else
    static_cast<float*>(a.out)[at] = v;
}

// Columns [col, col + 8) of one row per lane.
__device__ __forceinline__ void store_row8(const Fp8Args& a, int row, int col, const float (&v)[8]) {
  if (row >= a.rows) return;
  if (a.wide && col + 8 <= a.cols) {
    if (a.out_bf16) {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (long long)row * a.ldo + col) =
          make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    } else {
      float4* to = reinterpret_cast<float4*>(static_cast<float*>(a.out) + (long long)row * a.ldo + col);
      to[0] = make_float4(v[0], v[1], v[2], v[3]);
      to[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (col + i < a.cols) store_one(a, row, col + i, v[i]);
}

template <int BN, int PAIR, bool COLV>
__global__ void __launch_bounds__(Shape<BN, PAIR>::kThreads, 1) fp8_gemm_kernel(const __grid_constant__ Fp8Args a) {
  using S = Shape<BN, PAIR>;
  extern __shared__ uint8_t smem_raw[];
  Smem<BN, PAIR>& s = *reinterpret_cast<Smem<BN, PAIR>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t cluster_size;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cluster_size));
  const uint32_t rank = cluster_ctarank();
  const int split = PAIR == 2 ? 1 : int(cluster_size), part = PAIR == 2 ? 0 : int(rank);
  const uint32_t half = PAIR == 2 ? rank : 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(&s.full[i], 1), mbar_init(&s.empty[i], 1);
    for (int i = 0; i < S::kBufs; ++i) mbar_init(&s.tfull[i], 1), mbar_init(&s.tempty[i], S::kEpiWarps * PAIR);
    mbar_init(&s.drain, 1);
    s.abort = 0;
    fence_mbar_init();
  }
  if (warp == S::kEpiWarps + 1) {
    if (PAIR == 2)
      tmem_alloc_pair(&s.tmem, S::kTmemCols), tmem_relinquish_pair();
    else
      tmem_alloc(&s.tmem, S::kTmemCols), tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  if (cluster_size > 1) cluster_sync();  // the barriers of the whole cluster exist
  tc_fence_after();
  const uint32_t tmem = s.tmem;

  const int tiles = a.tiles_r * a.tiles_c;
  const int first = int(blockIdx.x / cluster_size), step = int(gridDim.x / cluster_size);
  const int kb0 = int((long long)a.num_kb * part / split), kb1 = int((long long)a.num_kb * (part + 1) / split);

  // With two column halves, 12 warps are launched with 168 registers each: the
  // epilogue warps, whose accumulators take 128, get 232 and the other four 40
  // (8 x 232 + 4 x 40 = 12 x 168)
  if (warp == S::kEpiWarps) {
    // ---- producer: one lane
    if (S::kHalves == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, issued = 0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += step) {
        int tr, tc;
        tile_at(t, a.tiles_r, a.tiles_c, &tr, &tc);
        const int r0 = (tr * PAIR + int(half)) * kRows, c0 = tc * BN + int(half) * (BN / PAIR);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = wait_phase<false>(&s.empty[stage], phase ^ 1, &s.abort))) break;
          if (half == 0) mbar_arrive_expect_tx(&s.full[stage], PAIR * S::kStageBytes);
          uint8_t* to = s.stages[stage];
          if (PAIR == 2) {
            const uint32_t bar = mapa_shared(smem_u32(&s.full[stage]), 0);  // both CTAs' bytes count on the leader's barrier
            tma_load_2d_pair(to, &a.map_r, bar, kb * kKBytes, r0);
            tma_load_2d_pair(to + S::kRowBytes, &a.map_c, bar, kb * kKBytes, c0);
          } else {
            tma_load_2d(to, &a.map_r, &s.full[stage], kb * kKBytes, r0);
            tma_load_2d(to + S::kRowBytes, &a.map_c, &s.full[stage], kb * kKBytes, c0);
          }
          ++issued;
          if (++stage == S::kStages) stage = 0, phase ^= 1;
        }
      }
      // every issued copy lands before the CTA may exit (the leader's barriers count
      // the other CTA's bytes too, which the final cluster barrier waits for)
      const uint32_t last = half != 0 ? 0 : min(issued, uint32_t(S::kStages));
      for (uint32_t i = 0; i < last; ++i) {
        const uint32_t fill = issued - 1 - i;
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&s.full[fill % S::kStages], (fill / S::kStages) & 1))
          if (globaltimer_ns() - t0 > kWaitNs) break;
      }
    }
    __syncwarp();
  } else if (warp == S::kEpiWarps + 1) {
    // ---- MMA issuer: the leader's warp, one lane issues
    if (S::kHalves == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (half == 0) {
      uint32_t stage = 0, phase = 0, buf = 0, bphase = 0;
      bool ok = true, any = false;
      const uint64_t hi = smem_desc(0, 16, 1024, 2);
      for (int t = first; ok && t < tiles; t += step) {
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = wait_phase<(PAIR == 2)>(&s.tempty[buf], bphase ^ 1, &s.abort);
          ok = ok && wait_phase<false>(&s.full[stage], phase, &s.abort);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          if (lane == 0) {
            const uint32_t sr = smem_u32(s.stages[stage]), sc = sr + S::kRowBytes;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_fp8<PAIR>(tmem + buf * BN, hi | uint64_t((sr + 32 * k) >> 4), hi | uint64_t((sc + 32 * k) >> 4), a.idesc, k > 0);
            if (PAIR == 2)
              mma_commit_pair_both(&s.empty[stage]), mma_commit_pair_both(&s.tfull[buf]);
            else
              mma_commit(&s.empty[stage]), mma_commit(&s.tfull[buf]);
          }
          __syncwarp();
          any = true;
          if (++stage == S::kStages) stage = 0, phase ^= 1;
          if (++buf == S::kBufs) buf = 0, bphase ^= 1;
        }
      }
      if (any) {  // no MMA is in flight when TMEM is released
        if (lane == 0) {
          if (PAIR == 2)
            mma_commit_pair_local(&s.drain);
          else
            mma_commit(&s.drain);
        }
        __syncwarp();
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&s.drain, 0))
          if (globaltimer_ns() - t0 > kWaitNs) break;
      }
    }
    __syncwarp();
  } else if (warp < S::kEpiWarps) {
    // ---- epilogue
    if (S::kHalves == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int quad = warp & 3, side = warp >> 2;
    uint32_t buf = 0, bphase = 0;
    bool ok = true;
    for (int t = first; ok && t < tiles; t += step) {
      int tr, tc;
      tile_at(t, a.tiles_r, a.tiles_c, &tr, &tc);
      const int row = (tr * PAIR + int(half)) * kRows + quad * 32 + lane, col0 = tc * BN + side * S::kCols;
      const float* pr = a.scale_r + (min(row, a.rows - 1) >> a.r_shift);
      // the scale of a column (COLV: 4 columns per lane) or of all columns of the warp
      const float* pc = a.scale_c + (min(col0, a.cols - 1) >> a.c_shift);
      uint64_t acc[S::kCols / 2];
#pragma unroll
      for (int i = 0; i < S::kCols / 2; ++i) acc[i] = 0;
      constexpr int kPer = (S::kCols + 31) / 32;
      float rs = 0.f, cs[kPer];
      auto fetch = [&](int kb) {
        rs = pr[kb * a.ld_r];
        if (COLV) {
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int c = col0 + lane + 32 * i;
            cs[i] = c < a.cols && lane + 32 * i < S::kCols ? a.scale_c[kb * a.ld_c + c] : 0.f;
          }
        } else {
          cs[0] = pc[kb * a.ld_c];
        }
      };
      if (kb0 < kb1) fetch(kb0);
      for (int kb = kb0; kb < kb1; ++kb) {
        const float r = rs, c = cs[0];
        if (COLV) {
          __syncwarp();  // the last block's scales have been read
#pragma unroll
          for (int i = 0; i < kPer; ++i)
            if (lane + 32 * i < S::kCols) s.col_scale[warp][lane + 32 * i] = cs[i];
          __syncwarp();
        }
        if (kb + 1 < kb1) fetch(kb + 1);
        ok = __all_sync(0xffffffffu, wait_phase<(PAIR == 2)>(&s.tfull[buf], bphase, &s.abort));
        if (!ok) break;
        tc_fence_after();
        const uint64_t both = COLV ? pair_of(r, r) : pair_of(r * c, r * c);
        const uint32_t from = tmem + buf * BN + side * S::kCols + (uint32_t(quad * 32) << 16);
#pragma unroll
        for (int j = 0; j < S::kCols / S::kChunk; ++j) {
          uint32_t v[S::kChunk];
          tmem_load(from + j * S::kChunk, v);
          if (j == S::kCols / S::kChunk - 1) {  // all of the buffer is in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (PAIR == 2 && half != 0)
                mbar_arrive_remote(mapa_shared(smem_u32(&s.tempty[buf]), 0));
              else
                mbar_arrive(&s.tempty[buf]);
            }
          }
#pragma unroll
          for (int i = 0; i < S::kChunk; i += 2) {
            const int at = (j * S::kChunk + i) / 2;
            const uint64_t p = pair_of(__uint_as_float(v[i]), __uint_as_float(v[i + 1]));
            if (COLV) {
              const float2 c2 = *reinterpret_cast<const float2*>(&s.col_scale[warp][j * S::kChunk + i]);
              acc[at] = fma2(p, mul2(pair_of(c2.x, c2.y), both), acc[at]);
            } else {
              acc[at] = fma2(p, both, acc[at]);
            }
          }
        }
        if (++buf == S::kBufs) buf = 0, bphase ^= 1;
      }
      if (!ok) break;
      if (PAIR == 1 && split > 1) {
        // this CTA's sums over its part of K, column by column (the operand stages
        // have all been consumed: the last block's product has been read)
        float* sums = reinterpret_cast<float*>(s.stages);
#pragma unroll
        for (int i = 0; i < S::kCols / 2; ++i) {
          const float2 v = unpair(acc[i]);
          sums[(side * S::kCols + 2 * i) * kRows + quad * 32 + lane] = v.x;
          sums[(side * S::kCols + 2 * i + 1) * kRows + quad * 32 + lane] = v.y;
        }
      } else if (a.swap) {
#pragma unroll
        for (int i = 0; i < S::kCols / 2; ++i) {
          const float2 v = unpair(acc[i]);
          if (row < a.rows && col0 + 2 * i < a.cols) store_one(a, row, col0 + 2 * i, v.x);
          if (row < a.rows && col0 + 2 * i + 1 < a.cols) store_one(a, row, col0 + 2 * i + 1, v.y);
        }
      } else {
#pragma unroll
        for (int i = 0; i < S::kCols / 2; i += 4) {
          const float2 v0 = unpair(acc[i]), v1 = unpair(acc[i + 1]), v2 = unpair(acc[i + 2]), v3 = unpair(acc[i + 3]);
          const float v[8] = {v0.x, v0.y, v1.x, v1.y, v2.x, v2.y, v3.x, v3.y};
          store_row8(a, row, col0 + 2 * i, v);
        }
      }
    }
  } else if constexpr (S::kHalves == 2) {  // two warps that only complete the register exchange
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
  }

  __syncthreads();
  if (PAIR == 1 && split > 1) {
    cluster_sync();  // the sums of every CTA of the cluster are in its shared memory
    if (warp < 4 && first < tiles && !*reinterpret_cast<volatile int*>(&s.abort)) {
      int tr, tc;
      tile_at(first, a.tiles_r, a.tiles_c, &tr, &tc);
      const int per = BN / split, at = warp * 32 + lane, row = tr * kRows + at;
      for (int c = part * per; c < (part + 1) * per; ++c) {
        const int col = tc * BN + c;
        if (row >= a.rows || col >= a.cols) continue;
        const uint32_t from = smem_u32(reinterpret_cast<float*>(s.stages) + c * kRows + at);
        float v = 0.f;
        for (int q = 0; q < split; ++q) v += ld_cluster(mapa_shared(from, q));
        store_one(a, row, col, v);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (cluster_size > 1) cluster_sync();  // no CTA leaves while another reads its memory or uses its TMEM
  if (warp == S::kEpiWarps + 1) {
    tc_fence_after();
    if (PAIR == 2)
      tmem_dealloc_pair(tmem, S::kTmemCols);
    else
      tmem_dealloc(tmem, S::kTmemCols);
  }
}

// ---------------------------------------------------------------- host side
int operand_map(CUtensorMap* map, const void* base, int k, int rows, long long ld, int box_rows) {
  const EncodeTiled enc = op_encode_tiled();
  if (!enc) return fail(PKT_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {cuuint64_t(k), cuuint64_t(rows)};
  cuuint64_t strides[1] = {cuuint64_t(ld)};
  cuuint32_t box[2] = {cuuint32_t(kKBytes), cuuint32_t(box_rows)};
  cuuint32_t ones[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? PKT_OK : fail(PKT_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", int(r));
}

template <int BN, int PAIR, bool COLV>
cudaError_t fp8_launch(const Fp8Args& a, int dev, int clusters, int cluster_size, cudaStream_t st) {
  using S = Shape<BN, PAIR>;
  constexpr int smem = int(sizeof(Smem<BN, PAIR>)) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of one CTA");
  static std::atomic<bool> ready[64];
  if (!ready[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(fp8_gemm_kernel<BN, PAIR, COLV>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    ready[dev].store(true, std::memory_order_release);
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(cluster_size);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(clusters) * unsigned(cluster_size));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<BN, PAIR, COLV>, a);
}

template <int BN, int PAIR>
cudaError_t fp8_launch(const Fp8Args& a, int dev, int clusters, int cluster_size, cudaStream_t st) {
  return a.c_shift == 0 ? fp8_launch<BN, PAIR, true>(a, dev, clusters, cluster_size, st)
                        : fp8_launch<BN, PAIR, false>(a, dev, clusters, cluster_size, st);
}

int check_operand(const char* name, const void* p, long long ld, const float* scale, long long ld_scale, int rows, int k, int block_rows, int dtype) {
  if (dtype != PKT_DTYPE_E4M3 && dtype != PKT_DTYPE_E5M2) return fail(PKT_ERR_ARGS, "%s_dtype must be e4m3 or e5m2", name);
  if (block_rows != 1 && block_rows != 128) return fail(PKT_ERR_ARGS, "%s_block_rows must be 1 or 128", name);
  if (!p || !aligned_to(p, 16) || ld % 16 != 0) return fail(PKT_ERR_ARGS, "%s must be 16-byte aligned with a row stride that is a multiple of 16", name);
  if (ld < k) return fail(PKT_ERR_ARGS, "row stride %lld of %s is below K = %d", ld, name, k);
  if (!scale || !aligned_to(scale, 4)) return fail(PKT_ERR_ARGS, "%s needs its scales, aligned to 4 bytes", name);
  if (ld_scale < (rows - 1) / block_rows + 1)
    return fail(PKT_ERR_ARGS, "row stride %lld of scale_%s is below its %d columns", ld_scale, name, (rows - 1) / block_rows + 1);
  return PKT_OK;
}

}  // namespace
}  // namespace pkb

extern "C" {

int pkt_fp8_gemm(const pkt_fp8_gemm_desc* d, void* stream) {
  using namespace pkb;
  if (!d) return fail(PKT_ERR_ARGS, "null fp8 gemm descriptor");
  if (d->M < 0 || d->N < 0 || d->K < 0) return fail(PKT_ERR_ARGS, "fp8 gemm of M=%d N=%d K=%d", d->M, d->N, d->K);
  if (d->out_dtype != PKT_DTYPE_BF16 && d->out_dtype != PKT_DTYPE_F32) return fail(PKT_ERR_ARGS, "fp8 gemm out_dtype must be bf16 or f32");
  if (d->M == 0 || d->N == 0) return PKT_OK;
  int dev = 0, sms = 0, rc;
  const int es = d->out_dtype == PKT_DTYPE_BF16 ? 2 : 4;
  if (!d->out || !aligned_to(d->out, es)) return fail(PKT_ERR_ARGS, "fp8 gemm needs out, aligned to its type");
  if (d->ldo < d->N) return fail(PKT_ERR_ARGS, "row stride %lld of out is below N = %d", d->ldo, d->N);
  if (d->K > 0 && ((rc = check_operand("a", d->a, d->lda, d->scale_a, d->ld_scale_a, d->M, d->K, d->a_block_rows, d->a_dtype)) ||
                   (rc = check_operand("b", d->b, d->ldb, d->scale_b, d->ld_scale_b, d->N, d->K, d->b_block_rows, d->b_dtype))))
    return rc;
  if ((rc = op_device(&dev, &sms)) || (rc = op_check_memory(d->out, "out", dev))) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->K == 0) {
    const cudaError_t e = cudaMemset2DAsync(d->out, size_t(d->ldo) * es, 0, size_t(d->N) * es, size_t(d->M), st);
    return e == cudaSuccess ? PKT_OK : cuda_fail(e, "clear out");
  }
  if ((rc = op_check_memory(d->a, "a", dev)) || (rc = op_check_memory(d->scale_a, "scale_a", dev)) || (rc = op_check_memory(d->b, "b", dev)) ||
      (rc = op_check_memory(d->scale_b, "scale_b", dev)))
    return rc;
  const int num_kb = (d->K - 1) / kKBytes + 1;
  // few output rows: the weights fill the lanes
  const bool swap = d->M <= 64;
  int bn = 128, pair = 1, split = 1;
  if (swap) {
    bn = d->M <= 16 ? 16 : d->M <= 32 ? 32 : 64;
  } else if ((long long)((d->M + 255) / 256) * ((d->N + 255) / 256) * 2 > sms / 2) {
    bn = 256, pair = 2;
  }
  Fp8Args a{};
  a.rows = swap ? d->N : d->M, a.cols = swap ? d->M : d->N, a.num_kb = num_kb;
  a.tiles_r = (a.rows - 1) / (kRows * pair) + 1, a.tiles_c = (a.cols - 1) / bn + 1;
  const long long tiles = (long long)a.tiles_r * a.tiles_c;
  if (tiles > 0x7fffffffLL) return fail(PKT_ERR_UNSUPPORTED, "fp8 gemm of M=%d N=%d has too many tiles", d->M, d->N);
  if (pair == 1)
    while (split < 8 && tiles * split * 2 <= sms && num_kb >= split * 4) split *= 2;
  const void *pr = swap ? d->b : d->a, *pc = swap ? d->a : d->b;
  if ((rc = operand_map(&a.map_r, pr, d->K, a.rows, swap ? d->ldb : d->lda, kRows)) ||
      (rc = operand_map(&a.map_c, pc, d->K, a.cols, swap ? d->lda : d->ldb, bn / pair)))
    return rc;
  a.scale_r = swap ? d->scale_b : d->scale_a, a.ld_r = swap ? d->ld_scale_b : d->ld_scale_a;
  a.scale_c = swap ? d->scale_a : d->scale_b, a.ld_c = swap ? d->ld_scale_a : d->ld_scale_b;
  a.r_shift = (swap ? d->b_block_rows : d->a_block_rows) == 1 ? 0 : 7;
  a.c_shift = (swap ? d->a_block_rows : d->b_block_rows) == 1 ? 0 : 7;
  a.out = d->out, a.ldo = d->ldo, a.out_bf16 = es == 2, a.swap = swap;
  a.wide = !swap && aligned_to(d->out, 16) && d->ldo * es % 16 == 0;
  const uint32_t fr = (swap ? d->b_dtype : d->a_dtype) == PKT_DTYPE_E5M2, fc = (swap ? d->a_dtype : d->b_dtype) == PKT_DTYPE_E5M2;
  a.idesc = (1u << 4) | (fr << 7) | (fc << 10) | (uint32_t(bn >> 3) << 17) | (uint32_t((kRows * pair) >> 4) << 24);
  // a cluster per tile when K is split, else a persistent grid
  const int clusters = split > 1 ? int(tiles) : int(std::min<long long>(tiles, sms / pair));
  const int cs = pair == 2 ? 2 : split;
  const cudaError_t e = pair == 2 ? fp8_launch<256, 2>(a, dev, clusters, cs, st)
                        : bn == 128 ? fp8_launch<128, 1>(a, dev, clusters, cs, st)
                        : bn == 64 ? fp8_launch<64, 1>(a, dev, clusters, cs, st)
                        : bn == 32 ? fp8_launch<32, 1>(a, dev, clusters, cs, st)
                                   : fp8_launch<16, 1>(a, dev, clusters, cs, st);
  return e == cudaSuccess ? PKT_OK : cuda_fail(e, "launch fp8 gemm");
}

int pkt_fp8_gemm_status(int* code) {
  using namespace pkb;
  if (!code) return fail(PKT_ERR_ARGS, "null argument");
  int dev = 0, sms = 0, rc;
  if ((rc = op_device(&dev, &sms))) return rc;
  cudaError_t e = cudaDeviceSynchronize();
  const int zero = 0;
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(code, g_fp8_status, sizeof(int));
  if (e == cudaSuccess && *code) e = cudaMemcpyToSymbol(g_fp8_status, &zero, sizeof(int));
  return e == cudaSuccess ? PKT_OK : cuda_fail(e, "read the fp8 gemm status");
}

}  // extern "C"
