// pkt_fp8_gemm: out = sum over blocks kb of 128 along K of
//   scale_a[kb, m] scale_b[kb, n] * sum over k in kb of a[m, k] b[n, k],
// e4m3 / e5m2 operands on tcgen05 (kind::f8f6f4), fp32 throughout.
//
// The scales change every 128 values of K, so a tensor-core accumulator holds one
// block of K only: the MMA issuer writes each block's product to the next of
// several TMEM buffers (4 MMAs of K = 32) and the epilogue warps read it back,
// multiply by the block's scales and add to accumulators in their registers, while
// the MMAs of the next blocks run. One fp32 FMA per output value and block of 128, or a
// product more where the columns have a scale each.
//
// A lane holds a row and all the warp's columns when the columns share a scale. When
// they do not, it holds 4 rows and a quarter of the columns (TMEM loads of 16 lanes x
// 256 bits): each lane then needs a quarter of the columns' scales, and it is their
// delivery from shared memory, 128 bytes a cycle for all warps, that bounds this case
// (8192 x 4096 x 4096: 180 us where a row per lane took 215 us, at the same clock).
//
// Roles of a CTA: warps 0..3 (0..7) epilogue, one per 32 TMEM lanes (and half of the
// columns); then one TMA producer warp, one MMA issuer warp and one that copies the
// scales of the coming blocks into shared memory (a load from L2 takes longer than a
// block). Operand tiles are 128-byte rows (128 values of K) in 128B-swizzled shared
// memory, in a ring of stages.
//
// "Rows" below are the operand whose 128 rows lie along the TMEM lanes, "cols" the one
// along the columns of a tile. For few output rows (M) the operands change places, so
// that the 128 lanes are filled by the weights and the columns by the few tokens.
// When there are few tiles, the CTAs of a cluster split K between them and add their
// accumulators through distributed shared memory in rank order.
//
// What bounds it. 8192 x 4096 x 4096 with 128 x 128 blocks of b takes 154 us call after
// call (1.78 PFLOP/s; the power limit lowers the clock) and 131 to 149 us in short runs, with
// a scale per column 195 to 208 us; the tensor pipe is busy 48 % of the time. A block of K
// (512 MMA cycles) is bounded by its turn through one of the two TMEM accumulators that
// fit: the MMAs, the epilogue's reads, and a release and an acquire through shared memory
// of 150 to 250 cycles each while MMAs run. That is why one issuer hands over all 256
// columns at once. In runs at the clock of 134 us two issuers with 128 columns each took
// 139 us, parts that every epilogue warp shares 170 us, 256 x 128 tiles with four
// accumulators 186 us, and the same pipeline without the promotion 104 us.
//
// Only M asks for narrow tiles: 65536 x 16 x 4096 runs in 256-wide pair tiles and takes 77
// us, 1.8 times the reading of its operands.
//
// Every wait is bounded (2 s); one that runs out sets a status word that
// pkt_ops_status reads, and the kernel drains its copies and returns.
#include <algorithm>
#include <atomic>

#include "ops_common.h"
#include "ops_device.cuh"

namespace pkb {
namespace {

constexpr int kRows = 128;    // TMEM lanes
constexpr int kKBytes = 128;  // one block of K: a 128-byte row of an operand tile

struct alignas(64) Fp8Args {
  CUtensorMap map_r, map_c, map_out;
  int rows, cols, num_kb;
  int tiles_r, tiles_c;
  const float *scale_r, *scale_c;
  long long ld_r, ld_c;
  int r_shift, c_shift;  // log2 of the rows that share a scale (0 or 7)
  void* out;
  long long ldo;
  int out_bf16, swap;  // swap: out[col * ldo + row]
  int wide, tma_out;   // 4 values of out in one store; map_out is valid
  int tma_cols;        // columns that map_out covers
  uint32_t idesc;
  int* status;
};

template <int BN, int PAIR>
struct Shape {
  static constexpr int kSides = BN > 64 ? 2 : 1;     // epilogue warps per 32 lanes
  static constexpr int kCols = BN / kSides;          // columns of an epilogue warp
  static constexpr int kEpiWarps = 4 * kSides;
  static constexpr int kThreads = 32 * (kEpiWarps + 4);
  static constexpr int kRowBytes = kRows * kKBytes;
  static constexpr int kColBytes = BN / PAIR * kKBytes;
  static constexpr int kStageBytes = kRowBytes + kColBytes;
  static constexpr int kStages = kStageBytes >= 32768 ? 5 : 8;
  static constexpr int kBufs = BN > 128 ? 2 : 4;     // TMEM accumulators
  static constexpr int kTmemCols = kBufs * BN < 32 ? 32 : kBufs * BN;
  static constexpr int kChunk = kCols < 32 ? kCols : 32;  // columns per TMEM load, two in flight
  static constexpr bool kStore = BN >= 128;          // the result leaves by TMA stores
  static constexpr int kGroup = 4;                   // blocks of K whose scales are handed over together
  static constexpr int kScales = 2;                  // such groups held
};

template <int BN, int PAIR>
struct Smem {
  using S = Shape<BN, PAIR>;
  uint8_t stages[S::kStages][S::kStageBytes];
  uint8_t staging[S::kStore ? S::kEpiWarps : 1][S::kStore ? 4096 : 16];  // 32 rows x 128 bytes of the result
  float row_scale[S::kScales][S::kGroup][kRows];
  float col_scale[S::kScales][S::kGroup][BN];  // of every column, or of every 128
  uint64_t sfull[S::kScales], sempty[S::kScales];
  uint64_t full[S::kStages], empty[S::kStages];
  uint64_t tfull[S::kBufs], tempty[S::kBufs];
  uint64_t drain;
  uint32_t tmem;
  int abort;
};

// One look without waiting. While MMAs run, a shared-memory access of any kind takes
// 150 to 250 cycles, so the loops ask for the next block's barrier early and use the
// answer late.
__device__ __forceinline__ uint32_t peek_phase(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok;
}
// A warp's bounded wait; a timeout is recorded for the CTA too.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, int* status, int* abort) {
  if (pkb::wait_phase(bar, parity, status)) return true;
  *reinterpret_cast<volatile int*>(abort) = 1;
  return false;
}

// One lane of a converged warp; known to the compiler as one, which lets the
// descriptors of tcgen05 instructions stay in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred P;\n elect.sync _|P, 0xffffffff;\n selp.u32 %0, 1, 0, P;\n}\n" : "=r"(p));
  return p != 0;
}

// One word global -> shared without waiting for it; zero where !in.
__device__ __forceinline__ void copy_word_async(float* to, const float* from, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(in ? 4 : 0) : "memory");
}
// Arrives on `bar` once this thread's copies so far have landed.
__device__ __forceinline__ void copy_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Arrives on a barrier of another CTA of the cluster. Only the order of TMEM reads
// matters here (tcgen05.wait::ld and the fence come before it), no memory is handed
// over: a release at cluster scope would wait for this thread's global stores, which
// measured 2000 cycles per block of K.
__device__ __forceinline__ void arrive_peer(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
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

// Columns of this warp's 32 lanes to registers; they hold the values after tmem_wait.
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld32(taddr, r); }
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) { tmem_ld_wait_regs(r); }
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

// 16 lanes x 8 N columns: a thread gets, for each 8 columns, those at 2 (lane % 4) and
// the next one, of rows lane / 4 and lane / 4 + 8.
__device__ __forceinline__ void tmem_load16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
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

// 4 consecutive values along out's rows: of one row, or (swap) of one column.
__device__ __forceinline__ void store_four(const Fp8Args& a, int row, int col, float4 v) {
  const int at = a.swap ? row : col, end = a.swap ? a.rows : a.cols;
  if (a.swap ? col >= a.cols : row >= a.rows) return;
  const long long off = (long long)(a.swap ? col : row) * a.ldo + at;
  if (a.wide && at + 4 <= end) {
    if (a.out_bf16)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + off) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    else
      *reinterpret_cast<float4*>(static_cast<float*>(a.out) + off) = v;
    return;
  }
  const float u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i < end) store_one(a, a.swap ? row + i : row, a.swap ? col : col + i, u[i]);
}

template <int BN, int PAIR, bool COLV>
__global__ void __launch_bounds__(Shape<BN, PAIR>::kThreads, 1) fp8_gemm_kernel(const __grid_constant__ Fp8Args a) {
  using S = Shape<BN, PAIR>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];  // the swizzle pattern's alignment
  Smem<BN, PAIR>& s = *reinterpret_cast<Smem<BN, PAIR>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t cluster_size;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cluster_size));
  const uint32_t rank = cluster_ctarank();
  const int split = PAIR == 2 ? 1 : int(cluster_size), part = PAIR == 2 ? 0 : int(rank);
  const uint32_t half = PAIR == 2 ? rank : 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(&s.full[i], 1), mbar_init(&s.empty[i], 1);
    for (int i = 0; i < S::kScales; ++i) mbar_init(&s.sfull[i], 32), mbar_init(&s.sempty[i], S::kEpiWarps);
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
  grid_dependents_launch();  // a product behind this one may set up as far as here on the SMs left over
  grid_dependency_wait();    // nothing of global memory has been touched yet

  const int tiles = a.tiles_r * a.tiles_c;
  const int first = int(blockIdx.x / cluster_size), step = int(gridDim.x / cluster_size);
  const int kb0 = int((long long)a.num_kb * part / split), kb1 = int((long long)a.num_kb * (part + 1) / split);

  // In 256-wide tiles 12 warps are launched with 168 registers each: the
  // epilogue warps, whose accumulators take 128, get 232 and the other four 40
  // (8 x 232 + 4 x 40 = 12 x 168)
  if (warp == S::kEpiWarps) {
    // ---- producer: one lane
    if (BN > 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    uint32_t stage = 0, phase = 0, issued = 0;
    bool ok = true;
    for (int t = first; ok && t < tiles; t += step) {
      int tr, tc;
      tile_at(t, a.tiles_r, a.tiles_c, &tr, &tc);
      const int r0 = (tr * PAIR + int(half)) * kRows, c0 = tc * BN + int(half) * (BN / PAIR);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = wait_phase(&s.empty[stage], phase ^ 1, a.status, &s.abort))) break;
        if (elect_one()) {
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
        }
        __syncwarp();
        ++issued;
        if (++stage == S::kStages) stage = 0, phase ^= 1;
      }
    }
    // every issued copy lands before the CTA may exit (the leader's barriers count
    // the other CTA's bytes too, which the final cluster barrier waits for)
    const uint32_t last = half != 0 ? 0 : min(issued, uint32_t(S::kStages));
    for (uint32_t i = 0; i < last; ++i) {
      const uint32_t fill = issued - 1 - i;
      try_phase(&s.full[fill % S::kStages], (fill / S::kStages) & 1);
    }
    __syncwarp();
  } else if (warp == S::kEpiWarps + 1) {
    // ---- MMA issuer, in the leader CTA; one lane issues
    if (BN > 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (half == 0) {
      uint32_t stage = 0, phase = 0, buf = 0, bphase = 0;
      uint32_t loaded = 0, drained = 0;  // the next block's barriers were found complete
      bool ok = true, any = false;
      const uint64_t hi = smem_desc(0, 16, 1024, 2);
      for (int t = first; ok && t < tiles; t += step) {
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!__all_sync(0xffffffffu, loaded)) ok = wait_phase(&s.full[stage], phase, a.status, &s.abort);
          if (ok && !__all_sync(0xffffffffu, drained)) ok = wait_phase(&s.tempty[buf], bphase ^ 1, a.status, &s.abort);
          if (!ok) break;
          const uint32_t sr = smem_u32(s.stages[stage]), sc = sr + S::kRowBytes;
          const uint32_t to = tmem + buf * BN;
          const uint32_t now = stage, nbuf = buf;
          if (++stage == S::kStages) stage = 0, phase ^= 1;
          if (++buf == S::kBufs) buf = 0, bphase ^= 1;
          loaded = peek_phase(&s.full[stage], phase);
          drained = peek_phase(&s.tempty[buf], bphase ^ 1);
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_fp8<PAIR>(to, hi | uint64_t((sr + 32 * k) >> 4), hi | uint64_t((sc + 32 * k) >> 4), a.idesc, k > 0);
            if (PAIR == 2)
              mma_commit_pair_both(&s.tfull[nbuf]), mma_commit_pair_both(&s.empty[now]);
            else
              mma_commit(&s.tfull[nbuf]), mma_commit(&s.empty[now]);
          }
          __syncwarp();
          any = true;
        }
      }
      if (any) {  // no MMA is in flight when TMEM is released
        if (elect_one()) {
          if (PAIR == 2)
            mma_commit_pair_local(&s.drain);
          else
            mma_commit(&s.drain);
        }
        __syncwarp();
        try_phase(&s.drain, 0);
      }
    }
    __syncwarp();
  } else if (warp < S::kEpiWarps) {
    // ---- epilogue
    if (BN > 128) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int quad = warp & 3, side = warp >> 2;
    // where this lane's values lie in the warp's 32 rows: value v of chunk j
    auto row_of = [&](int v) { return COLV ? v / (S::kChunk / 2) * 16 + (v >> 1 & 1) * 8 + (lane >> 2) : lane; };
    auto col_of = [&](int j, int v) {
      return j * S::kChunk + (COLV ? v % (S::kChunk / 2) / 4 * 8 + 2 * (lane & 3) + (v & 1) : v);
    };
    constexpr int R = COLV ? 4 : 1;  // rows of a lane
    uint32_t buf = 0, bphase = 0, slot = 0, sphase = 0;
    bool ok = true;
    for (int t = first; ok && t < tiles; t += step) {
      int tr, tc;
      tile_at(t, a.tiles_r, a.tiles_c, &tr, &tc);
      const int row0 = (tr * PAIR + int(half)) * kRows + quad * 32, col0 = tc * BN + side * S::kCols;
      uint64_t acc[S::kCols / 2];  // values 2 i and 2 i + 1
#pragma unroll
      for (int i = 0; i < S::kCols / 2; ++i) acc[i] = 0;
      // the scales of a block are fetched while the block before it is added, and its
      // barrier is asked for
      float next_r[R], next_c = 1.f;
      auto fetch = [&](int kb, uint32_t at, uint32_t ph) {
        const int in = (kb - kb0) % S::kGroup;
        if (in == 0 && !wait_phase(&s.sfull[at], ph, a.status, &s.abort)) return false;
#pragma unroll
        for (int i = 0; i < R; ++i) next_r[i] = s.row_scale[at][in][quad * 32 + (COLV ? 8 * i + (lane >> 2) : lane)];
        if (!COLV) next_c = s.col_scale[at][in][side * S::kCols / kScaleBlock];
        return true;
      };
      uint32_t ready = 0;
      if (kb0 < kb1) ok = fetch(kb0, slot, sphase);
      for (int kb = kb0; ok && kb < kb1; ++kb) {
        const int in = (kb - kb0) % S::kGroup;
        const bool last = in == S::kGroup - 1 || kb == kb1 - 1;
        float scale[R];
#pragma unroll
        for (int i = 0; i < R; ++i) scale[i] = next_r[i] * next_c;
        const float* cs = &s.col_scale[slot][in][side * S::kCols + 2 * (lane & 3)];
        if (!__all_sync(0xffffffffu, ready)) ok = wait_phase(&s.tfull[buf], bphase, a.status, &s.abort);
        if (!ok) break;
        tc_fence_after();
        const uint32_t from = tmem + buf * BN + side * S::kCols + (uint32_t(quad * 32) << 16);
        constexpr int kLoads = S::kCols / S::kChunk, kSplit = COLV ? 2 : 1, kRegs = S::kChunk / kSplit;
        uint32_t v[2][kSplit][kRegs];  // the next load is in flight while one chunk is added
        auto load = [&](int j) {
          if constexpr (COLV) {
            tmem_load16(from + j * S::kChunk, v[j & 1][0]);
            tmem_load16(from + j * S::kChunk + (16u << 16), v[j & 1][kSplit - 1]);
          } else {
            tmem_load(from + j * S::kChunk, v[j & 1][0]);
          }
        };
        load(0);
        if (kb + 1 < kb1) {
          const bool wrap = slot + 1 == S::kScales;
          ok = fetch(kb + 1, last ? (wrap ? 0 : slot + 1) : slot, last && wrap ? sphase ^ 1 : sphase);
        }
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          float2 c[COLV ? S::kChunk / 8 : 1];
          if constexpr (COLV) {
#pragma unroll
            for (int i = 0; i < S::kChunk / 8; ++i) c[i] = *reinterpret_cast<const float2*>(cs + j * S::kChunk + 8 * i);
          }
#pragma unroll
          for (int h = 0; h < kSplit; ++h) tmem_wait(v[j & 1][h]);
          if (j + 1 == kLoads) {  // all of the buffer is in registers
            ready = peek_phase(&s.tfull[buf + 1 == S::kBufs ? 0 : buf + 1], buf + 1 == S::kBufs ? bphase ^ 1 : bphase);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (PAIR == 2 && half != 0)
                arrive_peer(mapa_shared(smem_u32(&s.tempty[buf]), 0));
              else
                mbar_arrive(&s.tempty[buf]);
            }
          } else {
            load(j + 1);
          }
#pragma unroll
          for (int i = 0; i < S::kChunk; i += 2) {
            const float p0 = __uint_as_float(v[j & 1][i / kRegs][i % kRegs]), p1 = __uint_as_float(v[j & 1][i / kRegs][i % kRegs + 1]);
            uint64_t& to = acc[(j * S::kChunk + i) / 2];
            if constexpr (COLV) {
              const float2 q = c[i % kRegs / 4];
              const float r = scale[i / kRegs * 2 + (i >> 1 & 1)];
              to = fma2(mul2(pair_of(p0, p1), pair_of(q.x, q.y)), pair_of(r, r), to);
            } else {
              const float2 f = unpair(to);
              to = pair_of(fmaf(p0, scale[0], f.x), fmaf(p1, scale[0], f.y));
            }
          }
        }
        if (last) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.sempty[slot]);
          if (++slot == S::kScales) slot = 0, sphase ^= 1;
        }
        if (++buf == S::kBufs) buf = 0, bphase ^= 1;
      }
      if (!ok) break;
      if (PAIR == 1 && split > 1) {
        // this CTA's sums over its part of K, 4 consecutive values of the result to 16
        // bytes (the operand stages have all been consumed: the last block's product
        // has been read)
        float* sums = reinterpret_cast<float*>(s.stages);
#pragma unroll
        for (int i = 0; i < S::kCols; i += 2) {
          const int v = i % S::kChunk, r = quad * 32 + row_of(v), c = side * S::kCols + col_of(i / S::kChunk, v);
          const float2 f = unpair(acc[i / 2]);
          if (a.swap) {
            sums[c * kRows + r] = f.x;
            sums[(c + 1) * kRows + r] = f.y;
          } else {
            *reinterpret_cast<float2*>(sums + r * (BN + 4) + c) = f;
          }
        }
      } else if constexpr (S::kStore) {
        // 32 rows x 128 bytes at a time through swizzled shared memory, then a TMA store, or
        // (rows that do not start on 16 bytes) row by row, 32 neighbouring values at once: a
        // lane's own values of a row, stored one by one, made 1500x1500x2048 take 34 us instead
        // of 12.2 us; 8 rows are read before they are stored (26675x4397x919: 365 -> 254 us)
        uint8_t* to = s.staging[S::kStore ? warp : 0];
        const int per = a.out_bf16 ? 64 : 32;
#pragma unroll
        for (int j = 0; j < S::kCols / 32; ++j) {
          if (!a.out_bf16 || (j & 1) == 0) {
            if (lane == 0) bulk_wait_read_all();  // the last TMA store has left the staging
            __syncwarp();
          }
          if constexpr (COLV) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const int r = row_of(i), c = col_of(0, i);
              const float2 f = unpair(acc[j * 16 + i / 2]);
              if (a.out_bf16) {
                const int at = (j & 1) * 64 + c * 2;
                *reinterpret_cast<uint32_t*>(to + r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15)) = pack_bf16x2(f.x, f.y);
              } else {
                *reinterpret_cast<float2*>(to + r * 128 + (((c >> 2) ^ (r & 7)) << 4) + (c & 3) * 4) = f;
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              const uint64_t* v = acc + j * 16 + i / 2;
              const float2 f0 = unpair(v[0]), f1 = unpair(v[1]), f2 = unpair(v[2]), f3 = unpair(v[3]);
              if (a.out_bf16) {
                *reinterpret_cast<uint4*>(to + lane * 128 + ((((j & 1) * 4 + i / 8) ^ (lane & 7)) << 4)) =
                    make_uint4(pack_bf16x2(f0.x, f0.y), pack_bf16x2(f1.x, f1.y), pack_bf16x2(f2.x, f2.y), pack_bf16x2(f3.x, f3.y));
              } else {
                *reinterpret_cast<float4*>(to + lane * 128 + (((i / 4) ^ (lane & 7)) << 4)) = make_float4(f0.x, f0.y, f1.x, f1.y);
                *reinterpret_cast<float4*>(to + lane * 128 + (((i / 4 + 1) ^ (lane & 7)) << 4)) = make_float4(f2.x, f2.y, f3.x, f3.y);
              }
            }
          }
          if (!a.out_bf16 || (j & 1) == 1) {
            const int col = col0 + j * 32 + 32 - per;
            if (a.tma_out) {
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0 && row0 < a.rows && col < a.tma_cols) {
                tma_store_2d(&a.map_out, to, col, row0);
                bulk_commit();
              }
              if (a.tma_cols < col + per && row0 + lane < a.rows) {  // the columns left behind it, a row per lane
                for (int c = max(a.tma_cols, col); c < a.cols; ++c) {
                  const long long at = (long long)(row0 + lane) * a.ldo + c;
                  const int in = (c - col) * (a.out_bf16 ? 2 : 4);
                  const uint8_t* from = to + lane * 128 + (((in >> 4) ^ (lane & 7)) << 4) + (in & 15);
                  if (a.out_bf16)
                    static_cast<uint16_t*>(a.out)[at] = *reinterpret_cast<const uint16_t*>(from);
                  else
                    static_cast<float*>(a.out)[at] = *reinterpret_cast<const float*>(from);
                }
              }
            } else {
              __syncwarp();
              const int rows = min(32, a.rows - row0);
              const long long off = (long long)row0 * a.ldo + col + lane;
              const bool in0 = col + lane < a.cols, in1 = col + lane + 32 < a.cols;
              uint16_t* out16 = static_cast<uint16_t*>(a.out) + off;
              float* out32 = static_cast<float*>(a.out) + off;
#pragma unroll 1
              for (int r0 = 0; r0 < rows; r0 += 8) {
                const uint8_t* from = to + r0 * 128;
                if (a.out_bf16) {
                  uint16_t v[8][2];
#pragma unroll
                  for (int r = 0; r < 8; ++r)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                      v[r][i] = *reinterpret_cast<const uint16_t*>(from + r * 128 + ((((lane >> 3) + 4 * i) ^ r) << 4) + (lane & 7) * 2);
#pragma unroll
                  for (int r = 0; r < 8; ++r, out16 += a.ldo) {
                    if (r0 + r >= rows) break;
                    if (in0) out16[0] = v[r][0];
                    if (in1) out16[32] = v[r][1];
                  }
                } else {
                  float v[8];
#pragma unroll
                  for (int r = 0; r < 8; ++r) v[r] = *reinterpret_cast<const float*>(from + r * 128 + (((lane >> 2) ^ r) << 4) + (lane & 3) * 4);
#pragma unroll
                  for (int r = 0; r < 8; ++r, out32 += a.ldo) {
                    if (r0 + r >= rows) break;
                    if (in0) out32[0] = v[r];
                  }
                }
              }
            }
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < S::kCols; i += 2) {
          const int v = i % S::kChunk, r = row0 + row_of(v), c = col0 + col_of(i / S::kChunk, v);
          const float2 f = unpair(acc[i / 2]);
          if (r < a.rows && c < a.cols) store_one(a, r, c, f.x);
          if (r < a.rows && c + 1 < a.cols) store_one(a, r, c + 1, f.y);
        }
      }
    }
    if (S::kStore && a.tma_out && lane == 0) bulk_wait_all();
  } else {
    // ---- scales: a warp copies those of the tile's rows and columns, blocks ahead
    if (BN > 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == S::kEpiWarps + 2) {
      uint32_t slot = 0, phase = 0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += step) {
        int tr, tc;
        tile_at(t, a.tiles_r, a.tiles_c, &tr, &tc);
        const int row0 = (tr * PAIR + int(half)) * kRows, col0 = tc * BN;
        for (int kb = kb0; kb < kb1; ++kb) {
          if ((kb - kb0) % S::kGroup == 0) {
            ok = (wait_phase(&s.sempty[slot], phase ^ 1, a.status, &s.abort));
            if (!ok) break;
          }
          const int in = (kb - kb0) % S::kGroup;
          const float *pr = a.scale_r + kb * a.ld_r, *pc = a.scale_c + kb * a.ld_c;
#pragma unroll
          for (int i = 0; i < kRows; i += 32) {
            const int row = row0 + lane + i;
            copy_word_async(&s.row_scale[slot][in][lane + i], pr + (min(row, a.rows - 1) >> a.r_shift), row < a.rows);
          }
          if (COLV) {
#pragma unroll
            for (int i = 0; i < BN; i += 32) {
              const int col = col0 + lane + i;
              if (BN >= 32 || lane < BN) copy_word_async(&s.col_scale[slot][in][lane + i], pc + min(col, a.cols - 1), col < a.cols);
            }
          } else if (lane < (BN + 127) / 128) {
            const int col = col0 + lane * kScaleBlock;
            copy_word_async(&s.col_scale[slot][in][lane], pc + (min(col, a.cols - 1) >> 7), col < a.cols);
          }
          if (in == S::kGroup - 1 || kb == kb1 - 1) {
            copy_arrive(&s.sfull[slot]);
            if (++slot == S::kScales) slot = 0, phase ^= 1;
          }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    __syncwarp();
  }

  __syncthreads();
  if (PAIR == 1 && split > 1) {
    cluster_sync();  // the sums of every CTA of the cluster are in its shared memory
    if (first < tiles && !*reinterpret_cast<volatile int*>(&s.abort)) {
      int tr, tc;
      tile_at(first, a.tiles_r, a.tiles_c, &tr, &tc);
      const uint32_t sums = smem_u32(s.stages);
      uint32_t peer[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) peer[q] = mapa_shared(sums, min(q, split - 1));
      // a part of the tile's groups of 4 values for each CTA, added in rank order
      constexpr int kItems = kRows * BN / 4;
      for (int i = part * kItems / split + int(threadIdx.x); i < (part + 1) * kItems / split; i += S::kThreads) {
        const int r = a.swap ? i % (kRows / 4) * 4 : i / (BN / 4), c = a.swap ? i / (kRows / 4) : i % (BN / 4) * 4;
        const uint32_t at = 4 * (a.swap ? c * kRows + r : r * (BN + 4) + c);
        float4 v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = q < split ? ld_cluster(peer[q] + at) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int q = 1; q < 8; ++q) v[0].x += v[q].x, v[0].y += v[q].y, v[0].z += v[q].z, v[0].w += v[q].w;
        store_four(a, tr * kRows + r, tc * BN + c, v[0]);
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

// The result in boxes of 32 rows x 128 bytes (one epilogue warp's staging).
int result_map(CUtensorMap* map, void* base, int dtype, int cols, int rows, long long ld) {
  const EncodeTiled enc = op_encode_tiled();
  if (!enc) return fail(PKT_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const bool bf = dtype == PKT_DTYPE_BF16;
  cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
  cuuint64_t strides[1] = {cuuint64_t(ld) * (bf ? 2 : 4)};
  cuuint32_t box[2] = {bf ? 64u : 32u, 32};
  cuuint32_t ones[2] = {1, 1};
  const CUresult r = enc(map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, base, dims, strides, box, ones,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? PKT_OK : fail(PKT_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", int(r));
}

template <int BN, int PAIR, bool COLV>
int fp8_launch(const Fp8Args& a, int dev, int clusters, int cluster_size, cudaStream_t st) {
  using S = Shape<BN, PAIR>;
  constexpr int smem = int(sizeof(Smem<BN, PAIR>));
  static_assert(smem <= 227 * 1024, "shared memory of one CTA");
  static std::atomic<uint64_t> done;
  const int rc = op_shared_memory(reinterpret_cast<const void*>(fp8_gemm_kernel<BN, PAIR, COLV>), &done, dev, smem);
  if (rc) return rc;
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // as in op_launch
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(cluster_size);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(clusters) * unsigned(cluster_size));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<BN, PAIR, COLV>, a);
  return e == cudaSuccess ? PKT_OK : cuda_fail(e, "launch fp8 gemm");
}

template <int BN, int PAIR>
int fp8_launch(const Fp8Args& a, int dev, int clusters, int cluster_size, cudaStream_t st) {
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
  constexpr int kMost = 0x7fffffff - 255;  // the last tile's rows and columns are counted in 32 bits
  if (d->M > kMost || d->N > kMost) return fail(PKT_ERR_UNSUPPORTED, "fp8 gemm of M=%d N=%d", d->M, d->N);
  if (d->out_dtype != PKT_DTYPE_BF16 && d->out_dtype != PKT_DTYPE_F32) return fail(PKT_ERR_ARGS, "fp8 gemm out_dtype must be bf16 or f32");
  if (d->M == 0 || d->N == 0) return PKT_OK;
  int dev = 0, sms = 0, rc;
  const int es = d->out_dtype == PKT_DTYPE_BF16 ? 2 : 4;
  if (!d->out || !aligned_to(d->out, es)) return fail(PKT_ERR_ARGS, "fp8 gemm needs out, aligned to its type");
  if (d->ldo < d->N) return fail(PKT_ERR_ARGS, "row stride %lld of out is below N = %d", d->ldo, d->N);
  if (d->K > 0 && ((rc = check_operand("a", d->a, d->lda, d->scale_a, d->ld_scale_a, d->M, d->K, d->a_block_rows, d->a_dtype)) ||
                   (rc = check_operand("b", d->b, d->ldb, d->scale_b, d->ld_scale_b, d->N, d->K, d->b_block_rows, d->b_dtype))))
    return rc;
  int* status = nullptr;
  if ((rc = op_device(&dev, &sms, &status)) || (rc = op_check_memory(d->out, "out", dev))) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->K == 0) {
    const cudaError_t e = cudaMemset2DAsync(d->out, size_t(d->ldo) * es, 0, size_t(d->N) * es, size_t(d->M), st);
    return e == cudaSuccess ? PKT_OK : cuda_fail(e, "clear out");
  }
  if ((rc = op_check_memory(d->a, "a", dev)) || (rc = op_check_memory(d->scale_a, "scale_a", dev)) || (rc = op_check_memory(d->b, "b", dev)) ||
      (rc = op_check_memory(d->scale_b, "scale_b", dev)))
    return rc;
  const int num_kb = (d->K - 1) / kKBytes + 1;
  // Few output rows: the weights fill the lanes (64x4096x4096 10.4 us, 12.1 us with 128 x
  // 128 tiles; 8 rows 8.6 and 12.6 us). Pairs with 256 x 256 tiles once 128 x 128 tiles
  // would be more than one per SM (1536x1792x4096 21.9 us, 30.0 us with single CTAs;
  // 1280x1536x4096, 120 single tiles, 17.9 us, in pairs 21.1 us).
  const bool swap = d->M <= 64;
  int bn = 128, pair = 1, split = 1;
  if (swap) {
    bn = d->M <= 16 ? 16 : d->M <= 32 ? 32 : 64;
  } else if (((d->M - 1) / 256 + 1LL) * ((d->N - 1) / 256 + 1) * 2 > sms / 2) {
    bn = 256, pair = 2;
  }
  Fp8Args a{};
  a.status = status;
  a.rows = swap ? d->N : d->M, a.cols = swap ? d->M : d->N, a.num_kb = num_kb;
  a.tiles_r = (a.rows - 1) / (kRows * pair) + 1, a.tiles_c = (a.cols - 1) / bn + 1;
  const long long tiles = (long long)a.tiles_r * a.tiles_c;
  if (tiles > 0x7fffffffLL) return fail(PKT_ERR_UNSUPPORTED, "fp8 gemm of M=%d N=%d has too many tiles", d->M, d->N);
  // K over the CTAs of a cluster while all of them run at once, 2 blocks of K each at least
  // (128x4096x4096: 17.8 us whole, 15.4 us in 2 parts, 13.1 us in 4; 512x4096x4096, 128
  // tiles, 18.8 us whole and 29.8 us in 2).
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
  a.wide = aligned_to(d->out, 4 * es) && d->ldo % 4 == 0;
  // TMA stores need 16-byte aligned rows; else value by value. They write 16 bytes whole,
  // zeros past a map's last column, and behind column N there may be the next columns of a
  // wider matrix: the map ends at the last whole 16 bytes, what is left of a row is stored
  // value by value (8192x777x4096 into rows of 784 bf16 39.0 us, all value by value 42.3 us).
  a.tma_cols = d->N & -(16 / es);
  if (!swap && a.tma_cols > 0 && aligned_to(d->out, 16) && d->ldo * es % 16 == 0) {
    if ((rc = result_map(&a.map_out, d->out, d->out_dtype, a.tma_cols, d->M, d->ldo))) return rc;
    a.tma_out = 1;
  }
  const uint32_t fr = (swap ? d->b_dtype : d->a_dtype) == PKT_DTYPE_E5M2, fc = (swap ? d->a_dtype : d->b_dtype) == PKT_DTYPE_E5M2;
  a.idesc = (1u << 4) | (fr << 7) | (fc << 10) | (uint32_t(bn >> 3) << 17) | (uint32_t((kRows * pair) >> 4) << 24);
  // a cluster per tile when K is split, else a persistent grid
  const int clusters = split > 1 ? int(tiles) : int(std::min<long long>(tiles, sms / pair));
  const int cs = pair == 2 ? 2 : split;
  return pair == 2 ? fp8_launch<256, 2>(a, dev, clusters, cs, st)
         : bn == 128 ? fp8_launch<128, 1>(a, dev, clusters, cs, st)
         : bn == 64 ? fp8_launch<64, 1>(a, dev, clusters, cs, st)
         : bn == 32 ? fp8_launch<32, 1>(a, dev, clusters, cs, st)
                    : fp8_launch<16, 1>(a, dev, clusters, cs, st);
}

}  // extern "C"
