// pkt_layernorm_forward / pkt_layernorm_backward.
//
//   forward   mean = sum x / C,  rstd = 1 / sqrt(sum (x - mean)^2 / C + eps),
//             y = (x - mean) rstd gamma + beta
//   backward  h = (x - mean) rstd,  w = dy gamma,
//             dx = rstd (w - mean(w) - h mean(w h)),
//             dgamma = sum over rows of dy h,  dbeta = sum over rows of dy
//
// Both are bound by memory: 2 and 3 passes over the rows. A row is read once and stays
// in registers between the statistics and the result (the variance is the mean square
// of the centred values, not E x^2 - mean^2, which cancels). Rows belong to groups of
// 32..512 threads, several groups to a block where rows are short.
//
// Where there are many 16-byte aligned rows, each group runs its own ring of row
// buffers in shared memory, filled by bulk copies several rows ahead: the bytes in
// flight do not depend on the registers left over. Few rows, or unaligned ones, are
// loaded directly. Rows of more than 8192 values take two passes in the backward
// direction: the row sums first, then slabs of columns that need no reduction.
//
// The column sums dgamma / dbeta are kept in the registers of the threads that own the
// columns, across the rows of a block; every block writes one partial row to the
// workspace and a second kernel (launched with programmatic dependency) adds the
// partial rows in a fixed order, so results do not depend on timing. All sums are fp32.
#include <algorithm>
#include <type_traits>

#include "ops_common.h"
#include "ops_device.cuh"

namespace pkb {
namespace {

struct LnArgs {
  long long rows;
  int cols;
  float eps, inv_cols;
  const void *x, *gamma, *beta, *dy;
  void *y, *dx;
  long long ldx, ldy, lddy, lddx;
  float *mean, *rstd;
  float *dgamma, *dbeta;
  float* part;    // backward: [parts][2][cols]
  float4* stats;  // backward, long rows: [rows] mean, rstd and the two row sums
  int parts, size, slots;
  int* status;
};

constexpr int kWarpsPerBlock = 4;   // rows per block where a warp has a row (direct loads)
constexpr int kRingThreads = 512;
constexpr int kMaxSlots = 8;

// The sums of `v` over the threads of a row group (a power of two of warps); `red`
// holds one word per warp of the block. One barrier: callers alternate between two
// arrays, so that the barrier of one reduction protects the other's words.
__device__ __forceinline__ float add_to(float a, float b) { return a + b; }
__device__ __forceinline__ float2 add_to(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }
__device__ __forceinline__ float shuffled(float v, int off) { return __shfl_xor_sync(0xffffffffu, v, off); }
__device__ __forceinline__ float2 shuffled(float2 v, int off) { return make_float2(shuffled(v.x, off), shuffled(v.y, off)); }
__device__ __forceinline__ float4 add_to(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
__device__ __forceinline__ float4 shuffled(float4 v, int off) {
  return make_float4(shuffled(v.x, off), shuffled(v.y, off), shuffled(v.z, off), shuffled(v.w, off));
}

template <typename V>
__device__ __forceinline__ V group_sum(V v, V* red, int size, int group) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v = add_to(v, shuffled(v, off));
  if (size == 32) return v;
  const int lane = threadIdx.x & 31, nw = size >> 5;
  if (lane == 0) red[threadIdx.x >> 5] = v;
  named_barrier_sync(1 + group, size);
  v = red[group * nw + (lane & (nw - 1))];
  for (int off = nw >> 1; off >= 1; off >>= 1) v = add_to(v, shuffled(v, off));
  return v;
}

// VEC parameters at col (whole vectors: a row's columns are a multiple of VEC).
template <typename P, int VEC>
__device__ __forceinline__ void load_param(const void* base, int col, bool in, float other, float (&v)[VEC]) {
  Raw<P, VEC> r;
  r.load(static_cast<const P*>(base) + col, in && base != nullptr);
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = base != nullptr ? r.get(i) : in ? other : 0.f;
}

// ---------------------------------------------------------------- forward
// Statistics of a row that a group holds as K vectors per thread.
template <typename T, int VEC, int K>
__device__ __forceinline__ float2 row_stats(const Raw<T, VEC> (&raw)[K], const LnArgs& a, int tid, int size, int group, float (*red)[32]) {
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum += raw[k].get(i);
  const float mean = group_sum(sum, red[0], size, group) * a.inv_cols;
  float sq = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if ((k * size + tid) * VEC < a.cols) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = raw[k].get(i) - mean;
        sq = fmaf(d, d, sq);
      }
    }
  }
  return make_float2(mean, 1.f / sqrtf(group_sum(sq, red[1], size, group) * a.inv_cols + a.eps));
}

__device__ __forceinline__ void put_stats(const LnArgs& a, long long row, float2 st) {
  if (a.mean) a.mean[row] = st.x;
  if (a.rstd) a.rstd[row] = st.y;
}

template <typename T, typename P, int VEC, int K>
__global__ void __launch_bounds__(1024) ln_forward(const LnArgs a) {
  __shared__ float red[2][32];
  const int size = a.size, groups = blockDim.x / size, group = threadIdx.x / size, tid = threadIdx.x - group * size;
  for (long long row = (long long)blockIdx.x * groups + group; row < a.rows; row += (long long)gridDim.x * groups) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    Raw<T, VEC> raw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * size + tid) * VEC;
      raw[k].load(x + col, col < a.cols);
    }
    const float2 st = row_stats<T, VEC, K>(raw, a, tid, size, group, red);
    if (tid == 0) put_stats(a, row, st);
    T* y = static_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * size + tid) * VEC;
      if (col >= a.cols) continue;
      float g[VEC], b[VEC], out[VEC];
      load_param<P, VEC>(a.gamma, col, true, 1.f, g);
      load_param<P, VEC>(a.beta, col, true, 0.f, b);
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = fmaf((raw[k].get(i) - st.x) * st.y, g[i], b[i]);
      store_vec<T, VEC>(y + col, out);
    }
  }
}

// One ring of row buffers per group.
struct Ring {
  uint8_t* buf;     // [slots][bytes]
  uint64_t* full;   // [slots]
  uint32_t bytes;
  int slots, slot;
  uint32_t phase;
  bool dead;        // a wait ran out: go on without waiting (the results are not valid)

  __device__ __forceinline__ void wait(int* status) {
    if (!dead) dead = !wait_phase(&full[slot], phase, status);
  }
  __device__ __forceinline__ const uint8_t* at() const { return buf + slot * bytes; }
  __device__ __forceinline__ void next() {
    if (++slot == slots) slot = 0, phase ^= 1;
  }
  // no copy is in flight when the block exits, not even after a timeout
  __device__ __forceinline__ void drain(long long filled) {
    if (!dead) return;
    for (long long f = filled > slots ? filled - slots : 0; f < filled; ++f) try_phase(&full[f % slots], (f / slots) & 1);
  }
};

__device__ __forceinline__ Ring make_ring(uint8_t* smem, uint64_t (*full)[kMaxSlots], const LnArgs& a, int groups, int group, uint32_t bytes) {
  if (threadIdx.x == 0) {
    for (int g = 0; g < groups; ++g)
      for (int i = 0; i < a.slots; ++i) mbar_init(&full[g][i], 1);
    fence_mbar_init();
  }
  __syncthreads();
  return Ring{smem + (size_t)group * a.slots * bytes, full[group], bytes, a.slots, 0, 0, false};
}

// Two rows at a time, so that their reductions overlap, up to 32 values of each per
// thread in pairs, the parameters as fp32 in shared memory. The kernel was bound by its
// instructions: 30 per value with 8 values per thread (the fixed work of a row is two
// thirds of that), 19 with 16, 12 like this (8192 x 4096 bf16: 43, 33 and 27 us).
// EXACT: the group's threads cover the row without a rest.
template <typename T, typename P, int VEC, int K, bool EXACT>
__global__ void __launch_bounds__(kRingThreads) ln_forward_ring(const LnArgs a) {
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ uint64_t full[kRingThreads / 32][kMaxSlots];
  __shared__ float2 red[2][32];
  constexpr int H = VEC / 2;
  const int size = a.size, groups = kRingThreads / size, group = threadIdx.x / size, tid = threadIdx.x - group * size;
  const long long first = (long long)blockIdx.x * groups + group, step = (long long)gridDim.x * groups;
  const uint32_t bytes = uint32_t(a.cols) * sizeof(T);
  float* params = reinterpret_cast<float*>(ring_smem);  // [2][cols]
  for (int c = threadIdx.x; c < a.cols; c += kRingThreads) {
    params[c] = a.gamma ? to_f32(static_cast<const P*>(a.gamma)[c]) : 1.f;
    params[a.cols + c] = a.beta ? to_f32(static_cast<const P*>(a.beta)[c]) : 0.f;
  }
  Ring ring = make_ring(ring_smem + 8 * (size_t)a.cols, full, a, groups, group, bytes);
  const T* x = static_cast<const T*>(a.x);
  long long fill = first;  // the next row to copy
  auto copy = [&](int slot) {
    mbar_arrive_expect_tx(&ring.full[slot], bytes);
    bulk_load(ring.buf + slot * bytes, x + fill * a.ldx, bytes, &ring.full[slot]);
  };
  for (int i = 0; i < a.slots && fill < a.rows; ++i, fill += step)
    if (tid == 0) copy(i);
  bool in[K];
#pragma unroll
  for (int k = 0; k < K; ++k) in[k] = EXACT || (k * size + tid) * VEC < a.cols;
  params += tid * VEC;
  T* y = static_cast<T*>(a.y) + first * a.ldy + tid * VEC;
  const long long next_y = step * a.ldy;
  for (long long row = first; row < a.rows; row += 2 * step, y += 2 * next_y) {
    const bool two = row + step < a.rows;
    Raw<T, VEC> raw[2][K];
    int slot[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {  // a missing second row is zeros
      slot[r] = ring.slot;
      if (r == 0 || two) ring.wait(a.status);
      const T* from = reinterpret_cast<const T*>(ring.at()) + tid * VEC;
#pragma unroll
      for (int k = 0; k < K; ++k) raw[r][k].load(from + k * size * VEC, in[k] && (r == 0 || two));
      if (r == 0 || two) ring.next();
    }
    uint64_t s0 = 0, s1 = 0;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < H; ++i) s0 = add2(s0, raw[0][k].get2(i)), s1 = add2(s1, raw[1][k].get2(i));
    const float2 sum = group_sum(make_float2(sum_of(s0), sum_of(s1)), red[0], size, group);
    const float2 mean = make_float2(sum.x * a.inv_cols, sum.y * a.inv_cols);
    const uint64_t m0 = pair_of(-mean.x, -mean.x), m1 = pair_of(-mean.y, -mean.y);
    s0 = s1 = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!in[k]) continue;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const uint64_t d0 = add2(raw[0][k].get2(i), m0), d1 = add2(raw[1][k].get2(i), m1);
        s0 = fma2(d0, d0, s0);
        s1 = fma2(d1, d1, s1);
      }
    }
    const float2 sq = group_sum(make_float2(sum_of(s0), sum_of(s1)), red[1], size, group);
    const float2 rstd = make_float2(1.f / sqrtf(sq.x * a.inv_cols + a.eps), 1.f / sqrtf(sq.y * a.inv_cols + a.eps));
    // the reductions are behind every thread's reads of the buffers
    if (tid == 0) {
      if (fill < a.rows) copy(slot[0]);
      fill += step;
      if (two && fill < a.rows) copy(slot[1]);
      fill += step;
      put_stats(a, row, make_float2(mean.x, rstd.x));
      if (two) put_stats(a, row + step, make_float2(mean.y, rstd.y));
    }
    const uint64_t r0 = pair_of(rstd.x, rstd.x), r1 = pair_of(rstd.y, rstd.y);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!in[k]) continue;
      Raw<float, VEC> g, b;
      g.load(params + k * size * VEC, true);
      b.load(params + a.cols + k * size * VEC, true);
      uint64_t out[H];
#pragma unroll
      for (int i = 0; i < H; ++i) out[i] = fma2(mul2(add2(raw[0][k].get2(i), m0), r0), g.get2(i), b.get2(i));
      store_pairs<T, VEC>(y + k * size * VEC, out);
      if (!two) continue;
#pragma unroll
      for (int i = 0; i < H; ++i) out[i] = fma2(mul2(add2(raw[1][k].get2(i), m1), r1), g.get2(i), b.get2(i));
      store_pairs<T, VEC>(y + next_y + k * size * VEC, out);
    }
  }
  if (tid == 0) ring.drain((min(fill, a.rows + step - 1) - first) / step);
}

// Rows longer than a block's registers: a block per row that reads it three times
// (the second and third time from L2).
template <typename T, typename P, int VEC>
__global__ void __launch_bounds__(1024) ln_forward_long(const LnArgs a) {
  __shared__ float red[2][32];
  const int step = blockDim.x * VEC, begin = threadIdx.x * VEC;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    float sum = 0.f;
    for (int col = begin; col < a.cols; col += step) {
      Raw<T, VEC> r;
      r.load(x + col, true);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += r.get(i);
    }
    const float mean = group_sum(sum, red[0], blockDim.x, 0) * a.inv_cols;
    float sq = 0.f;
    for (int col = begin; col < a.cols; col += step) {
      Raw<T, VEC> r;
      r.load(x + col, true);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = r.get(i) - mean;
        sq = fmaf(d, d, sq);
      }
    }
    const float rstd = 1.f / sqrtf(group_sum(sq, red[1], blockDim.x, 0) * a.inv_cols + a.eps);
    if (threadIdx.x == 0) put_stats(a, row, make_float2(mean, rstd));
    T* y = static_cast<T*>(a.y) + row * a.ldy;
    for (int col = begin; col < a.cols; col += step) {
      Raw<T, VEC> r;
      r.load(x + col, true);
      float g[VEC], b[VEC], out[VEC];
      load_param<P, VEC>(a.gamma, col, true, 1.f, g);
      load_param<P, VEC>(a.beta, col, true, 0.f, b);
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = fmaf((r.get(i) - mean) * rstd, g[i], b[i]);
      store_vec<T, VEC>(y + col, out);
    }
  }
}

// ---------------------------------------------------------------- backward
// A thread's columns across the rows of its group, in pairs where it has vectors.
template <typename T, typename P, int VEC, int K>
struct Columns {
  static constexpr int kPair = VEC > 1 ? 2 : 1, H = VEC / kPair;
  using V = std::conditional_t<VEC == 1, float, uint64_t>;
  V gamma[K][H], dg[K][H], db[K][H];

  static __device__ __forceinline__ float both(float v, float) { return v; }
  static __device__ __forceinline__ uint64_t both(float v, uint64_t) { return pair_of(v, v); }
  static __device__ __forceinline__ float add(float a, float b) { return a + b; }
  static __device__ __forceinline__ uint64_t add(uint64_t a, uint64_t b) { return add2(a, b); }
  static __device__ __forceinline__ float mul(float a, float b) { return a * b; }
  static __device__ __forceinline__ uint64_t mul(uint64_t a, uint64_t b) { return mul2(a, b); }
  static __device__ __forceinline__ float fma(float a, float b, float c) { return fmaf(a, b, c); }
  static __device__ __forceinline__ uint64_t fma(uint64_t a, uint64_t b, uint64_t c) { return fma2(a, b, c); }
  static __device__ __forceinline__ float total(float v) { return v; }
  static __device__ __forceinline__ float total(uint64_t v) { return sum_of(v); }
  static __device__ __forceinline__ V value(const Raw<T, VEC>& r, int i) {
    if constexpr (VEC > 1)
      return r.get2(i);
    else
      return r.get(0);
  }

  __device__ __forceinline__ void init(const LnArgs& a, int col0, int size) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = col0 + k * size * VEC;
      float g[VEC];
      load_param<P, VEC>(a.gamma, col, col < a.cols, 1.f, g);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        if constexpr (VEC > 1)
          gamma[k][i] = pair_of(g[2 * i], g[2 * i + 1]);
        else
          gamma[k][i] = g[0];
        dg[k][i] = db[k][i] = V(0);
      }
    }
  }
  // Adds a row and returns its sums of w and w h. Beyond the row's end dy and gamma
  // are zero, and so is what they add.
  __device__ __forceinline__ float2 add(const Raw<T, VEC> (&rx)[K], const Raw<T, VEC> (&ry)[K], float mean, float rstd) {
    V s1 = V(0), s2 = V(0);
    const V m = both(-mean, V(0)), r = both(rstd, V(0));
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const V dy = value(ry[k], i), h = mul(add(value(rx[k], i), m), r), w = mul(dy, gamma[k][i]);
        dg[k][i] = fma(dy, h, dg[k][i]);
        db[k][i] = add(db[k][i], dy);
        s1 = add(s1, w);
        s2 = fma(w, h, s2);
      }
    return make_float2(total(s1), total(s2));
  }
  // dx = rstd (w - c1 - h c2); `dx`: this thread's first column of the row
  __device__ __forceinline__ void write(const Raw<T, VEC> (&rx)[K], const Raw<T, VEC> (&ry)[K], const bool (&in)[K], T* dx, int size, float mean,
                                        float rstd, float c1, float c2) {
    const V m = both(-mean, V(0)), r = both(rstd, V(0)), r1 = both(-rstd * c1, V(0)), r2 = both(-rstd * c2 * rstd, V(0));
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!in[k]) continue;
      V out[H];
#pragma unroll
      for (int i = 0; i < H; ++i) out[i] = fma(mul(value(ry[k], i), gamma[k][i]), r, fma(add(value(rx[k], i), m), r2, r1));
      if constexpr (VEC > 1)
        store_pairs<T, VEC>(dx + k * size * VEC, out);
      else
        from_f32(out[0], dx + k * size);
    }
  }
  // The block's partial row: its groups' column sums, added in group order. `sums`:
  // shared memory, [groups][2 K VEC][size].
  __device__ __forceinline__ void finish(const LnArgs& a, int tid, int size, int group, int groups, float* sums) {
    constexpr int kHalf = K * VEC;
    float* part = a.part + (long long)blockIdx.x * 2 * a.cols;
    float* mine = sums + group * 2 * kHalf * size + tid;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < H; ++i) {
        if constexpr (VEC > 1) {
          const float2 g = unpair(dg[k][i]), b = unpair(db[k][i]);
          mine[(k * VEC + 2 * i) * size] = g.x, mine[(k * VEC + 2 * i + 1) * size] = g.y;
          mine[(kHalf + k * VEC + 2 * i) * size] = b.x, mine[(kHalf + k * VEC + 2 * i + 1) * size] = b.y;
        } else {
          mine[k * size] = dg[k][i], mine[(kHalf + k) * size] = db[k][i];
        }
      }
    __syncthreads();
    const int shift = 31 - __clz(size);
    for (int j = threadIdx.x; j < 2 * kHalf * size; j += blockDim.x) {
      float t = sums[j];
      for (int g = 1; g < groups; ++g) t += sums[g * 2 * kHalf * size + j];
      const int v = j >> shift, which = v >= kHalf, u = which ? v - kHalf : v;
      const int col = (u / VEC * size + (j & (size - 1))) * VEC + u % VEC;
      if (col < a.cols) part[which * a.cols + col] = t;
    }
  }
};

// Direct loads; the next row's are issued before this row's reduction.
template <typename T, typename P, int VEC, int K>
__global__ void __launch_bounds__(512) ln_backward(const LnArgs a) {
  __shared__ float2 red[2][32];
  extern __shared__ __align__(128) uint8_t ring_smem[];
  const int size = a.size, groups = blockDim.x / size, group = threadIdx.x / size, tid = threadIdx.x - group * size;
  const long long first = (long long)blockIdx.x * groups + group, step = (long long)gridDim.x * groups;
  Columns<T, P, VEC, K> c;
  c.init(a, tid * VEC, size);
  Raw<T, VEC> rx[K], ry[K], nx[K], ny[K];
  bool in[K];
#pragma unroll
  for (int k = 0; k < K; ++k) in[k] = (k * size + tid) * VEC < a.cols;
  float next_mean = 0.f, next_rstd = 0.f;
  auto fetch = [&](long long row) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * size + tid) * VEC;
      nx[k].load(x + col, col < a.cols);
      ny[k].load(dy + col, col < a.cols);
    }
    next_mean = a.mean[row], next_rstd = a.rstd[row];
  };
  if (first < a.rows) fetch(first);
  int flip = 0;
  for (long long row = first; row < a.rows; row += step, flip ^= 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) rx[k] = nx[k], ry[k] = ny[k];
    const float mean = next_mean, rstd = next_rstd;
    if (row + step < a.rows) fetch(row + step);
    const float2 s = group_sum(c.add(rx, ry, mean, rstd), red[flip], size, group);
    if (a.dx)
      c.write(rx, ry, in, static_cast<T*>(a.dx) + row * a.lddx + tid * VEC, size, mean, rstd, s.x * a.inv_cols, s.y * a.inv_cols);
  }
  grid_dependents_launch();
  c.finish(a, tid, size, group, groups, reinterpret_cast<float*>(ring_smem));
}

template <typename T, typename P, int VEC, int K, bool EXACT>
__global__ void __launch_bounds__(kRingThreads) ln_backward_ring(const LnArgs a) {
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ uint64_t full[kRingThreads / 32][kMaxSlots];
  __shared__ float4 red[2][kRingThreads / 32];
  const int size = a.size, groups = kRingThreads / size, group = threadIdx.x / size, tid = threadIdx.x - group * size;
  const long long first = (long long)blockIdx.x * groups + group, step = (long long)gridDim.x * groups;
  const uint32_t bytes = uint32_t(a.cols) * sizeof(T);
  Ring ring = make_ring(ring_smem, full, a, groups, group, 2 * bytes);
  const T *x = static_cast<const T*>(a.x), *dy = static_cast<const T*>(a.dy);
  long long fill = first;
  auto copy = [&](int slot) {
    mbar_arrive_expect_tx(&ring.full[slot], 2 * bytes);
    bulk_load(ring.buf + slot * 2 * bytes, x + fill * a.ldx, bytes, &ring.full[slot]);
    bulk_load(ring.buf + slot * 2 * bytes + bytes, dy + fill * a.lddy, bytes, &ring.full[slot]);
  };
  for (int i = 0; i < a.slots && fill < a.rows; ++i, fill += step)
    if (tid == 0) copy(i);
  Columns<T, P, VEC, K> c;
  c.init(a, tid * VEC, size);
  bool in[K];
#pragma unroll
  for (int k = 0; k < K; ++k) in[k] = EXACT || (k * size + tid) * VEC < a.cols;
  // the rows of an iteration overlap their reductions; a missing row is zeros
  constexpr int R = 1;
  float next_mean[R], next_rstd[R];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool here = row + r * step < a.rows;
      next_mean[r] = here ? a.mean[row + r * step] : 0.f;
      next_rstd[r] = here ? a.rstd[row + r * step] : 0.f;
    }
  };
  fetch(first);
  T* dx = static_cast<T*>(a.dx) + (a.dx ? first * a.lddx + tid * VEC : 0);
  const long long next_dx = step * a.lddx;
  int flip = 0;
  for (long long row = first; row < a.rows; row += R * step, flip ^= 1, dx += R * next_dx) {
    float mean[R], rstd[R];
    Raw<T, VEC> rx[R][K], ry[R][K];
    int slot[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool here = r == 0 || row + r * step < a.rows;
      mean[r] = next_mean[r], rstd[r] = next_rstd[r];
      slot[r] = ring.slot;
      if (here) ring.wait(a.status);
      const T* from = reinterpret_cast<const T*>(ring.at()) + tid * VEC;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        rx[r][k].load(from + k * size * VEC, here && in[k]);
        ry[r][k].load(from + a.cols + k * size * VEC, here && in[k]);
      }
      if (here) ring.next();
    }
    fetch(row + R * step);
    float2 s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = c.add(rx[r], ry[r], mean[r], rstd[r]);
    if constexpr (R == 2) {
      const float4 t = group_sum(make_float4(s[0].x, s[0].y, s[R - 1].x, s[R - 1].y), red[flip], size, group);
      s[0] = make_float2(t.x, t.y), s[R - 1] = make_float2(t.z, t.w);
    } else {
      const float4 t = group_sum(make_float4(s[0].x, s[0].y, 0.f, 0.f), red[flip], size, group);
      s[0] = make_float2(t.x, t.y);
    }
    // the reduction is behind every thread's reads of the buffers
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (fill < a.rows && (r == 0 || row + r * step < a.rows)) {
        if (tid == 0) copy(slot[r]);
        fill += step;
      }
    if (a.dx) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r == 0 || row + r * step < a.rows)
          c.write(rx[r], ry[r], in, dx + r * next_dx, size, mean[r], rstd[r], s[r].x * a.inv_cols, s[r].y * a.inv_cols);
    }
  }
  if (tid == 0) ring.drain((fill - first) / step);
  grid_dependents_launch();
  __syncthreads();  // the buffers are free: they take the groups' sums
  c.finish(a, tid, size, group, groups, reinterpret_cast<float*>(ring_smem));
}

// Long rows, first pass: a block per row, its mean, rstd and two sums to `stats`.
template <typename T, typename P, int VEC>
__global__ void __launch_bounds__(1024) ln_row_sums(const LnArgs a) {
  __shared__ float2 red[2][32];
  int flip = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll 2
    for (int col = threadIdx.x * VEC; col < a.cols; col += 1024 * VEC) {
      Raw<T, VEC> rx, ry;
      rx.load(x + col, true);
      ry.load(dy + col, true);
      float g[VEC];
      load_param<P, VEC>(a.gamma, col, true, 1.f, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float w = ry.get(i) * g[i];
        s.x += w;
        s.y = fmaf(w, (rx.get(i) - mean) * rstd, s.y);
      }
    }
    s = group_sum(s, red[flip], 1024, 0);
    if (threadIdx.x == 0) a.stats[row] = make_float4(mean, rstd, s.x * a.inv_cols, s.y * a.inv_cols);
  }
}

// Long rows, second pass: blockIdx.y is a slab of columns, blockIdx.x a part of the
// rows; the row sums are known, so threads own their columns without a reduction.
constexpr int kSlabThreads = 256, kSlabRows = 4;
template <typename T, typename P, int VEC>
__global__ void __launch_bounds__(kSlabThreads) ln_backward_slab(const LnArgs a) {
  const int col0 = blockIdx.y * kSlabThreads * VEC, col = col0 + threadIdx.x * VEC;
  const bool in = col < a.cols, mine[1] = {in};
  Columns<T, P, VEC, 1> c;
  c.init(a, col, kSlabThreads);
  for (long long row0 = (long long)blockIdx.x * kSlabRows; row0 < a.rows; row0 += (long long)gridDim.x * kSlabRows) {
    Raw<T, VEC> rx[kSlabRows][1], ry[kSlabRows][1];
    float4 st[kSlabRows];
#pragma unroll
    for (int r = 0; r < kSlabRows; ++r) {
      const long long row = row0 + r;
      const bool here = row < a.rows;
      rx[r][0].load(static_cast<const T*>(a.x) + row * a.ldx + col, in && here);
      ry[r][0].load(static_cast<const T*>(a.dy) + row * a.lddy + col, in && here);
      st[r] = here ? a.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int r = 0; r < kSlabRows; ++r) {
      if (row0 + r >= a.rows) break;
      c.add(rx[r], ry[r], st[r].x, st[r].y);
      if (a.dx) c.write(rx[r], ry[r], mine, static_cast<T*>(a.dx) + (row0 + r) * a.lddx + col, kSlabThreads, st[r].x, st[r].y, st[r].z, st[r].w);
    }
  }
  if (!in) return;
  float* part = a.part + (long long)blockIdx.x * 2 * a.cols + col;
#pragma unroll
  for (int i = 0; i < c.H; ++i) {
    if constexpr (VEC > 1) {
      const float2 g = unpair(c.dg[0][i]), b = unpair(c.db[0][i]);
      part[2 * i] = g.x, part[2 * i + 1] = g.y, part[a.cols + 2 * i] = b.x, part[a.cols + 2 * i + 1] = b.y;
    } else {
      part[0] = c.dg[0][i], part[a.cols] = c.db[0][i];
    }
  }
}

// dgamma / dbeta = the partial rows added in order: 32 columns per block, the
// partial rows dealt to 32 warps, their sums added in warp order.
__global__ void __launch_bounds__(1024) ln_column_sums(const float* part, int parts, int cols, float* dgamma, float* dbeta) {
  __shared__ float2 sums[32][33];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float2 s = make_float2(0.f, 0.f);
  if (col < cols) {
#pragma unroll 4
    for (int p = warp; p < parts; p += 32) {
      s.x += part[(long long)p * 2 * cols + col];
      s.y += part[(long long)p * 2 * cols + cols + col];
    }
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && col < cols) {
    s = sums[0][lane];
#pragma unroll
    for (int w = 1; w < 32; ++w) s.x += sums[w][lane].x, s.y += sums[w][lane].y;
    if (dgamma) dgamma[col] = s.x;
    if (dbeta) dbeta[col] = s.y;
  }
}

// ---------------------------------------------------------------- host side
struct LnPlan {
  int vec;      // elements per access: 16 bytes of the row's type, or 1
  int k;        // vectors per thread; 0: the long-row kernels
  int size;     // threads per row
  int threads;  // per block
  bool ring;    // rows through shared memory
  int slots;    // row buffers per group
  size_t smem;
};

constexpr int kHeld = 8192;  // values of a row that the backward kernels hold at once

// 16-byte accesses need every row of every tensor to start on a 16-byte boundary and
// to end on one; other rows go element by element.
LnPlan ln_plan(const pkt_layernorm_desc& d, bool backward, int sms) {
  const int es = d.dtype == PKT_DTYPE_BF16 ? 2 : 4;
  auto rows_ok = [&](const void* p, long long ld) { return aligned_to(p, 16) && ld * es % 16 == 0; };
  bool wide = (long long)d.cols * es % 16 == 0 && rows_ok(d.x, d.ldx) && aligned_to(d.gamma, 16);
  if (backward)
    wide = wide && rows_ok(d.dy, d.lddy) && (!d.dx || rows_ok(d.dx, d.lddx));
  else
    wide = wide && rows_ok(d.y, d.ldy) && aligned_to(d.beta, 16);
  LnPlan p{};
  p.vec = wide ? 16 / es : 1;
  const int nvec = d.cols / p.vec;
  auto sums_bytes = [](const LnPlan& q) { return size_t(512) * 2 * q.k * q.vec * sizeof(float); };
  auto threads_for = [&](int k, int most) {
    int t = 32;
    while (t < most && (long long)t * k < nvec) t *= 2;
    return t;
  };
  auto choose = [&](const int* ks, int count, int most) {  // the fewest vectors per thread that fit
    for (int i = 0; i < count; ++i) {
      p.k = ks[i], p.size = threads_for(ks[i], most);
      if ((long long)p.size * p.k >= nvec) return true;
    }
    p.k = 0, p.size = p.threads = 1024;
    return false;
  };
  if (!wide) {
    const int few[3] = {1, 8, 16}, many[2] = {8, 16};
    const bool lots = d.rows >= 2LL * sms;
    if (backward ? choose(many, 2, 512) : lots ? choose(many, 2, 1024) : choose(few, 3, 1024)) {
      p.threads = backward ? 512 : std::max(p.size, 32 * kWarpsPerBlock);
      if (backward) p.smem = sums_bytes(p);
    }
    return p;
  }
  // The ring pays from a few rows per group on; up to 32 values per thread in the forward
  // pass, 16 in the backward pass (three more registers each), in as few threads as hold
  // the row.
  const int ks[3] = {1, 2, 16 / p.vec};
  p.k = (backward ? 16 : 32) / p.vec;
  while (p.k > 1 && 32 * (p.k / 2) >= nvec) p.k /= 2;
  p.size = threads_for(p.k, kRingThreads);
  if ((long long)p.size * p.k >= nvec) {
    const long long groups = (long long)sms * (kRingThreads / p.size);
    const size_t stage = size_t(kRingThreads / p.size) * d.cols * es * (backward ? 2 : 1);
    const size_t params = backward ? 0 : 8 * size_t(d.cols);
    p.slots = int(std::min<size_t>(kMaxSlots, (200 * 1024 - params) / stage));
    if (d.rows >= 2 * groups && p.slots >= 3) {
      p.ring = true;
      p.threads = kRingThreads;
      p.smem = std::max(p.slots * stage + params, backward ? sums_bytes(p) : size_t(0));
      return p;
    }
  }
  if (backward) {
    if (choose(ks, 3, 512)) p.threads = 512, p.smem = sums_bytes(p);
  } else {
    const int direct[3] = {1, 2, 4};
    if (choose(direct, 3, 1024)) p.threads = std::max(p.size, 32 * kWarpsPerBlock);
  }
  return p;
}

// Blocks along the rows in the backward pass, each with one partial row of column
// sums: two per SM. (From the sizes alone: the workspace is asked for before the
// pointers are known.)
int ln_parts(long long rows, int sms) { return int(std::max(1LL, std::min(rows, 2LL * sms))); }
// The partial rows, then (long rows) 4 values per row.
size_t ln_part_floats(const pkt_layernorm_desc* d, int sms) { return (size_t(ln_parts(d->rows, sms)) * 2 * d->cols + 3) / 4 * 4; }
size_t ln_workspace(const pkt_layernorm_desc* d, int sms) {
  return (ln_part_floats(d, sms) + (d->cols > kHeld ? size_t(d->rows) * 4 : 0)) * sizeof(float);
}

template <typename... KArgs>
int ln_launch_shared(void (*kernel)(KArgs...), std::atomic<uint64_t>* done, int dev, const LnArgs& a, const LnPlan& p, int blocks, cudaStream_t st) {
  const int rc = op_shared_memory(reinterpret_cast<const void*>(kernel), done, dev, 200 * 1024);
  if (rc) return rc;
  const cudaError_t e = op_launch(kernel, dim3(blocks), dim3(p.threads), p.smem, st, false, a);
  return e == cudaSuccess ? PKT_OK : cuda_fail(e, "launch layer norm");
}

// The partial rows that a backward kernel wrote (as a positive result).
template <typename T, typename P, int VEC, int K, bool EXACT>
int ln_run_ring(LnArgs a, const LnPlan& p, bool backward, int dev, int sms, cudaStream_t st) {
  static std::atomic<uint64_t> done[2];
  if (!backward) return ln_launch_shared(ln_forward_ring<T, P, VEC, K, EXACT>, &done[1], dev, a, p, sms, st);
  if constexpr (K * VEC <= 16) {
    const int blocks = std::min(a.parts, sms), rc = ln_launch_shared(ln_backward_ring<T, P, VEC, K, EXACT>, &done[0], dev, a, p, blocks, st);
    return rc ? rc : blocks;
  }
  return fail(PKT_ERR_UNSUPPORTED, "layer norm of %d columns", a.cols);
}

template <typename T, typename P, int VEC, int K>
int ln_run(LnArgs a, const LnPlan& p, bool backward, int dev, int sms, cudaStream_t st) {
  if constexpr (VEC > 1) {
    if (p.ring)
      return a.cols == p.size * K * VEC ? ln_run_ring<T, P, VEC, K, true>(a, p, backward, dev, sms, st)
                                        : ln_run_ring<T, P, VEC, K, false>(a, p, backward, dev, sms, st);
  }
  if constexpr (VEC == 1 || K <= 4) {
    if (!backward) {
      const long long blocks = (a.rows - 1) / (p.threads / p.size) + 1;
      const cudaError_t e = op_launch(ln_forward<T, P, VEC, K>, dim3(unsigned(std::min(blocks, 1LL << 30))), dim3(p.threads), 0, st, false, a);
      return e == cudaSuccess ? PKT_OK : cuda_fail(e, "launch layer norm");
    }
  }
  if constexpr (K * VEC <= 16 && !(VEC == 1 && K < 8)) {
    static std::atomic<uint64_t> done;
    const int rc = ln_launch_shared(ln_backward<T, P, VEC, K>, &done, dev, a, p, a.parts, st);
    return rc ? rc : a.parts;
  }
  return fail(PKT_ERR_UNSUPPORTED, "layer norm of %d columns", a.cols);
}

template <typename T, typename P, int VEC>
int ln_pick(LnArgs a, const LnPlan& p, bool backward, int dev, int sms, cudaStream_t st) {
  switch (p.k) {
    case 0: {
      if (!backward) {
        const cudaError_t e = op_launch(ln_forward_long<T, P, VEC>, dim3(unsigned(std::min(a.rows, 1LL << 30))), dim3(1024), 0, st, false, a);
        return e == cudaSuccess ? PKT_OK : cuda_fail(e, "launch layer norm");
      }
      const int slabs = (a.cols - 1) / (kSlabThreads * VEC) + 1;
      const long long want = std::max(1LL, 8LL * sms / slabs);  // about 8 blocks of 256 threads per SM
      const int rows = int(std::min<long long>({want, a.parts, (a.rows - 1) / kSlabRows + 1}));
      cudaError_t e = op_launch(ln_row_sums<T, P, VEC>, dim3(unsigned(std::min(a.rows, 1LL << 30))), dim3(1024), 0, st, false, a);
      if (e == cudaSuccess) e = op_launch(ln_backward_slab<T, P, VEC>, dim3(rows, slabs), dim3(kSlabThreads), 0, st, false, a);
      return e == cudaSuccess ? rows : cuda_fail(e, "launch layer norm");
    }
    case 1: return ln_run<T, P, VEC, 1>(a, p, backward, dev, sms, st);
    case 2: if constexpr (VEC > 1) return ln_run<T, P, VEC, 2>(a, p, backward, dev, sms, st); break;
    case 4: if constexpr (VEC > 1) return ln_run<T, P, VEC, 4>(a, p, backward, dev, sms, st); break;
    case 8: if constexpr (VEC != 8) return ln_run<T, P, VEC, 8>(a, p, backward, dev, sms, st); break;
    case 16: if constexpr (VEC == 1) return ln_run<T, P, 1, 16>(a, p, backward, dev, sms, st); break;
  }
  return fail(PKT_ERR_UNSUPPORTED, "layer norm of %d columns", a.cols);
}

template <typename T>
int ln_dispatch(const LnArgs& a, const LnPlan& p, int param_dtype, bool backward, int dev, int sms, cudaStream_t st) {
  constexpr int W = 16 / int(sizeof(T));
  if (param_dtype == PKT_DTYPE_F32)
    return p.vec > 1 ? ln_pick<T, float, W>(a, p, backward, dev, sms, st) : ln_pick<T, float, 1>(a, p, backward, dev, sms, st);
  return p.vec > 1 ? ln_pick<T, bf16_t, W>(a, p, backward, dev, sms, st) : ln_pick<T, bf16_t, 1>(a, p, backward, dev, sms, st);
}

int ln_check_common(const pkt_layernorm_desc* d) {
  if (!d) return fail(PKT_ERR_ARGS, "null layer norm descriptor");
  if (d->rows < 0 || d->cols <= 0) return fail(PKT_ERR_ARGS, "layer norm of %lld rows x %d columns", d->rows, d->cols);
  if (d->dtype != PKT_DTYPE_BF16 && d->dtype != PKT_DTYPE_F32) return fail(PKT_ERR_ARGS, "layer norm dtype must be bf16 or f32");
  if (d->param_dtype != PKT_DTYPE_BF16 && d->param_dtype != PKT_DTYPE_F32)
    return fail(PKT_ERR_ARGS, "layer norm param_dtype must be bf16 or f32");
  return PKT_OK;
}

int ln_check_rows(const void* p, long long ld, const char* what, const pkt_layernorm_desc* d) {
  if (!p) return fail(PKT_ERR_ARGS, "layer norm needs %s", what);
  if (ld < d->cols) return fail(PKT_ERR_ARGS, "row stride %lld of %s is below the %d columns", ld, what, d->cols);
  if (!aligned_to(p, d->dtype == PKT_DTYPE_BF16 ? 2 : 4)) return fail(PKT_ERR_ARGS, "%s is not aligned to its type", what);
  return PKT_OK;
}

int ln_check_param(const void* p, const char* what, int dtype) {
  if (!aligned_to(p, dtype == PKT_DTYPE_BF16 ? 2 : 4)) return fail(PKT_ERR_ARGS, "%s is not aligned to its type", what);
  return PKT_OK;
}

LnArgs ln_args(const pkt_layernorm_desc& d, const LnPlan& p, int* status) {
  LnArgs a{};
  a.size = p.size, a.slots = p.slots, a.status = status;
  a.rows = d.rows, a.cols = d.cols, a.eps = d.eps, a.inv_cols = 1.f / float(d.cols);
  a.x = d.x, a.gamma = d.gamma, a.beta = d.beta, a.dy = d.dy, a.y = d.y, a.dx = d.dx;
  a.ldx = d.ldx, a.ldy = d.ldy, a.lddy = d.lddy, a.lddx = d.lddx;
  a.mean = d.mean, a.rstd = d.rstd, a.dgamma = d.dgamma, a.dbeta = d.dbeta;
  return a;
}

}  // namespace
}  // namespace pkb

extern "C" {

int pkt_layernorm_forward(const pkt_layernorm_desc* d, void* stream) {
  using namespace pkb;
  int dev = 0, sms = 0, rc, *status = nullptr;
  if ((rc = ln_check_common(d))) return rc;
  if (!(d->eps >= 0.f)) return fail(PKT_ERR_ARGS, "layer norm eps must be >= 0");
  if (d->rows == 0) return PKT_OK;
  if ((rc = ln_check_rows(d->x, d->ldx, "x", d)) || (rc = ln_check_rows(d->y, d->ldy, "y", d)) ||
      (rc = ln_check_param(d->gamma, "gamma", d->param_dtype)) || (rc = ln_check_param(d->beta, "beta", d->param_dtype)) ||
      (rc = ln_check_param(d->mean, "mean", PKT_DTYPE_F32)) || (rc = ln_check_param(d->rstd, "rstd", PKT_DTYPE_F32)))
    return rc;
  if ((rc = op_device(&dev, &sms, &status)) || (rc = op_check_memory(d->x, "x", dev)) || (rc = op_check_memory(d->y, "y", dev)) ||
      (rc = op_check_memory(d->gamma, "gamma", dev)) || (rc = op_check_memory(d->beta, "beta", dev)) ||
      (rc = op_check_memory(d->mean, "mean", dev)) || (rc = op_check_memory(d->rstd, "rstd", dev)))
    return rc;
  const LnPlan p = ln_plan(*d, false, sms);
  const LnArgs a = ln_args(*d, p, status);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return d->dtype == PKT_DTYPE_BF16 ? ln_dispatch<bf16_t>(a, p, d->param_dtype, false, dev, sms, st)
                                    : ln_dispatch<float>(a, p, d->param_dtype, false, dev, sms, st);
}

int pkt_layernorm_backward_workspace(const pkt_layernorm_desc* d, size_t* bytes) {
  using namespace pkb;
  int dev = 0, sms = 0, rc;
  if (!bytes) return fail(PKT_ERR_ARGS, "null bytes");
  if ((rc = ln_check_common(d)) || (rc = op_device(&dev, &sms))) return rc;
  *bytes = ln_workspace(d, sms);
  return PKT_OK;
}

int pkt_layernorm_backward(const pkt_layernorm_desc* d, void* stream) {
  using namespace pkb;
  int dev = 0, sms = 0, rc, *status = nullptr;
  if ((rc = ln_check_common(d)) || (rc = ln_check_param(d->dgamma, "dgamma", PKT_DTYPE_F32)) ||
      (rc = ln_check_param(d->dbeta, "dbeta", PKT_DTYPE_F32)))
    return rc;
  if (d->rows > 0) {
    if ((rc = ln_check_rows(d->x, d->ldx, "x", d)) || (rc = ln_check_rows(d->dy, d->lddy, "dy", d)) ||
        (d->dx && (rc = ln_check_rows(d->dx, d->lddx, "dx", d))) || (rc = ln_check_param(d->gamma, "gamma", d->param_dtype)))
      return rc;
    if (!d->mean || !d->rstd) return fail(PKT_ERR_ARGS, "layer norm backward needs the forward pass's mean and rstd");
    if ((rc = ln_check_param(d->mean, "mean", PKT_DTYPE_F32)) || (rc = ln_check_param(d->rstd, "rstd", PKT_DTYPE_F32)) ||
        (rc = aligned_to(d->workspace, 16) ? PKT_OK : fail(PKT_ERR_ARGS, "workspace is not 16-byte aligned")))
      return rc;
  }
  if ((rc = op_device(&dev, &sms, &status)) || (rc = op_check_memory(d->dgamma, "dgamma", dev)) || (rc = op_check_memory(d->dbeta, "dbeta", dev)))
    return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->rows == 0) {  // no rows: the sums over them are zero
    for (float* p : {d->dgamma, d->dbeta}) {
      const cudaError_t e = p ? cudaMemsetAsync(p, 0, size_t(d->cols) * sizeof(float), st) : cudaSuccess;
      if (e != cudaSuccess) return cuda_fail(e, "clear the column sums");
    }
    return PKT_OK;
  }
  const size_t need = ln_workspace(d, sms);
  if (!d->workspace || d->workspace_bytes < need)
    return fail(PKT_ERR_ARGS, "layer norm backward needs a workspace of %zu bytes, got %zu", need, d->workspace ? d->workspace_bytes : size_t(0));
  if ((rc = op_check_memory(d->x, "x", dev)) || (rc = op_check_memory(d->dy, "dy", dev)) || (rc = op_check_memory(d->dx, "dx", dev)) ||
      (rc = op_check_memory(d->gamma, "gamma", dev)) || (rc = op_check_memory(d->mean, "mean", dev)) ||
      (rc = op_check_memory(d->rstd, "rstd", dev)) || (rc = op_check_memory(d->workspace, "workspace", dev)))
    return rc;
  const LnPlan p = ln_plan(*d, true, sms);
  LnArgs a = ln_args(*d, p, status);
  a.parts = ln_parts(d->rows, sms);
  a.part = static_cast<float*>(d->workspace);
  a.stats = reinterpret_cast<float4*>(a.part + ln_part_floats(d, sms));
  rc = d->dtype == PKT_DTYPE_BF16 ? ln_dispatch<bf16_t>(a, p, d->param_dtype, true, dev, sms, st)
                                  : ln_dispatch<float>(a, p, d->param_dtype, true, dev, sms, st);
  if (rc < 0) return rc;
  a.parts = rc;
  if (d->dgamma || d->dbeta) {
    const cudaError_t e = op_launch(ln_column_sums, dim3((d->cols - 1) / 32 + 1), dim3(1024), 0, st, true, static_cast<const float*>(a.part),
                                    a.parts, a.cols, d->dgamma, d->dbeta);
    if (e != cudaSuccess) return cuda_fail(e, "launch layer norm column sums");
  }
  return PKT_OK;
}

}  // extern "C"
