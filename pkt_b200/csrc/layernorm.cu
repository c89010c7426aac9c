// pkt_layernorm_forward / pkt_layernorm_backward.
//
//   forward   mean = sum x / C,  rstd = 1 / sqrt(sum (x - mean)^2 / C + eps),
//             y = (x - mean) rstd gamma + beta
//   backward  h = (x - mean) rstd,  w = dy gamma,
//             dx = rstd (w - mean(w) - h mean(w h)),
//             dgamma = sum over rows of dy h,  dbeta = sum over rows of dy
//
// Both are bound by memory: 2 and 3 passes over the rows. Measured (6.55 TB/s: a plain
// copy): forward 8192x4096 bf16 25.4 us, 5.28 TB/s, fp32 49.4 us, 5.43 TB/s; backward 38.0
// us, 5.30 TB/s, and 72 us, 5.58 TB/s, with 42 and 52 % of the issue slots used. Rows off 16
// bytes go value by value, and that, not memory, sets their time (4099x777 fp32: forward 8.9
// us, backward 13.0 us; 8192x4095 bf16 40 and 52 us). A row is read once and stays
// in registers between the statistics and the result (the variance is the mean square
// of the centred values, not E x^2 - mean^2, which cancels). Rows belong to groups of
// 32..512 threads, several groups to a block where rows are short; a thread computes on
// pairs of values (one instruction for two).
//
// Where there are many rows, each group runs its own ring of row buffers in shared
// memory, filled by bulk copies a few rows ahead, whatever the rows' alignment (a copy
// takes the 16-byte granules that hold the row). Few rows are loaded directly. Rows of
// more than 8192 values take two passes in the backward direction: the row sums first,
// then slabs of columns that need no reduction.
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
  float eps, num_cols, inv_cols;
  const void *x, *gamma, *beta, *dy;
  void *y, *dx;
  long long ldx, ldy, lddy, lddx;
  float *mean, *rstd;
  float *dgamma, *dbeta;
  float* part;    // backward: [parts][2][cols]
  float4* stats;  // backward, long rows: [rows] mean, rstd and the two row sums
  int parts, size, slots;
  uint32_t pitch;  // bytes of a row buffer
  int* status;
};

constexpr int kRingThreads = 512;
constexpr int kMaxSlots = 8;

// The sums of `v` over the threads of a row group (a power of two of warps); `red`
// holds one word per warp of the block. One barrier: callers alternate between two
// arrays, so that the barrier of one reduction protects the other's words.
__device__ __forceinline__ float2 add_to(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }
__device__ __forceinline__ float2 shuffled(float2 v, int off) {
  return make_float2(__shfl_xor_sync(0xffffffffu, v.x, off), __shfl_xor_sync(0xffffffffu, v.y, off));
}
__device__ __forceinline__ float2 group_sum(float2 v, float2* red, int size, int group) {
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

__device__ __forceinline__ uint64_t twice(float v) { return pair_of(v, v); }

// N values of a row in one thread, as raw words (as fp32 where they are loaded one by
// one): N / VEC vectors of VEC consecutive values; zeros past the row's end. A warp's
// columns are contiguous, vector k of lane l at (k * 32 + l) * VEC from its first one, so
// that all distances are constants. EXACT: the threads cover the row without a rest.
template <typename T, int VEC, int N>
struct Held {
  static constexpr int K = N / VEC;
  static constexpr int kWords = VEC == 1 ? N : N * int(sizeof(T)) / 4;
  uint32_t w[kWords];

  // the thread's first column
  static __device__ __forceinline__ int first(int tid) { return ((tid >> 5) * K * 32 + (tid & 31)) * VEC; }
  static __device__ __forceinline__ constexpr int at(int k) { return k * 32 * VEC; }
  static __device__ __forceinline__ bool whole(int tid, int cols) { return first(tid | 31) + at(K - 1) + VEC <= cols; }
  template <bool EXACT>
  __device__ __forceinline__ void load(const T* row, int c0, int cols) {
    row += c0;
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!EXACT && c0 + at(k) >= cols) continue;
      if constexpr (VEC > 1) {
        const uint4 v = *reinterpret_cast<const uint4*>(row + at(k));
        w[4 * k] = v.x, w[4 * k + 1] = v.y, w[4 * k + 2] = v.z, w[4 * k + 3] = v.w;
      } else {
        w[k] = __float_as_uint(to_f32(row[at(k)]));
      }
    }
  }
  // values 2 p and 2 p + 1 of the thread
  __device__ __forceinline__ uint64_t pair(int p) const {
    if constexpr (VEC == 1 || sizeof(T) == 4)
      return pair_of(__uint_as_float(w[2 * p]), __uint_as_float(w[2 * p + 1]));
    else
      return pair_of(bf16_lo(w[p]), bf16_hi(w[p]));
  }
  // -mean for the values inside the row, 0 for the zeros past its end
  template <bool EXACT>
  static __device__ __forceinline__ uint64_t minus(float mean, int p, int c0, int cols) {
    if constexpr (EXACT) return twice(-mean);
    return pair_of(c0 + at(2 * p / VEC) < cols ? -mean : 0.f, c0 + at((2 * p + 1) / VEC) < cols ? -mean : 0.f);
  }
};

// Runs f(true) where all of a warp's columns are inside the row, so that they need no
// comparisons (a third of the instructions where values go one by one), else f(false).
template <bool EXACT, typename F>
__device__ __forceinline__ void by_whole(bool whole, F f) {
  if (EXACT || whole)
    f(std::true_type{});
  else
    f(std::false_type{});
}

// The results of a row, rounded to its type once.
template <typename T, int VEC, int N, bool EXACT>
__device__ __forceinline__ void store_held(T* row, const uint64_t (&v)[N / 2], int c0, int cols) {
  using S = Held<T, VEC, N>;
  row += c0;
#pragma unroll
  for (int k = 0; k < S::K; ++k) {
    if (!EXACT && c0 + S::at(k) >= cols) continue;
    if constexpr (VEC > 1) {
      uint64_t q[VEC / 2];
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) q[i] = v[k * VEC / 2 + i];
      store_pairs<T, VEC>(row + S::at(k), q);
    } else {
      const float2 f = unpair(v[k / 2]);
      from_f32(k & 1 ? f.y : f.x, row + S::at(k));
    }
  }
}

// The thread's pairs of a parameter row (fp32 or bf16; `other` where there is none).
template <typename P, int VEC, int N>
__device__ __forceinline__ void load_params(const void* base, float other, int c0, int cols, uint64_t (&out)[N / 2]) {
  const P* from = static_cast<const P*>(base) + c0;
#pragma unroll
  for (int k = 0; k < N / (VEC > 1 ? VEC : 2); ++k) {
    if constexpr (VEC > 1) {
      const bool in = c0 + k * 32 * VEC < cols;
      Raw<P, VEC> r;
      r.load(from + k * 32 * VEC, base && in);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) out[k * VEC / 2 + i] = base ? r.get2(i) : twice(in ? other : 0.f);
    } else {
      float f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = (2 * k + i) * 32;
        f[i] = c0 + c >= cols ? 0.f : base ? to_f32(from[c]) : other;
      }
      out[k] = pair_of(f[0], f[1]);
    }
  }
}

// ---------------------------------------------------------------- rings of row buffers
// The rows of a group: first, first + step, ... A buffer takes the 16-byte granules
// that hold a row; shift() is where the row begins in it.
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
  __device__ __forceinline__ void next() {
    if (++slot == slots) slot = 0, phase ^= 1;
  }
  // no copy is in flight when the block exits, not even after a timeout
  __device__ __forceinline__ void drain(long long filled) {
    if (!dead) return;
    for (long long f = filled > slots ? filled - slots : 0; f < filled; ++f) try_phase(&full[f % slots], (f / slots) & 1);
  }
};

__device__ __forceinline__ uint32_t shift(const void* p) { return uint32_t(reinterpret_cast<uintptr_t>(p)) & 15u; }
__device__ __forceinline__ uint32_t granules(const void* p, uint32_t bytes) { return (shift(p) + bytes + 15u) & ~15u; }
__device__ __forceinline__ const void* granule(const void* p) {
  return reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15));
}

__device__ __forceinline__ Ring make_ring(uint8_t* smem, uint64_t (*full)[kMaxSlots], const LnArgs& a, int groups, int group, uint32_t bytes) {
  if (threadIdx.x == 0) {
    for (int g = 0; g < groups; ++g)
      for (int i = 0; i < a.slots; ++i) mbar_init(&full[g][i], 1);
    fence_mbar_init();
  }
  __syncthreads();
  return Ring{smem + (size_t)group * a.slots * bytes, full[group], bytes, a.slots, 0, 0, false};
}

// ---------------------------------------------------------------- forward
__device__ __forceinline__ void put_stats(const LnArgs& a, long long row, float mean, float rstd) {
  if (a.mean) a.mean[row] = mean;
  if (a.rstd) a.rstd[row] = rstd;
}

// sum / C: the product with 1 / C is off by up to 1.5 ulp, and the error of a mean comes
// back times rstd (a row of 1000 times 100.0 was off by 2.4e-3 gamma from y = beta). What
// it leaves of the sum, divided again, mends that: a quotient that is an fp32 value is
// exact, any other rounded once but for 2^-22 ulp. (bf16 8192x4096 25.5 us, 65536x256
// 25.6 us, as without it; a division by every thread 25.9 and 26.7 us.)
__device__ __forceinline__ float row_mean(const LnArgs& a, float sum) {
  const float q = sum * a.inv_cols;
  const float m = fmaf(fmaf(-a.num_cols, q, sum), a.inv_cols, q);
  return fabsf(q) < INFINITY ? m : q;
}

template <typename T, typename P, int VEC, int N>
__global__ void __launch_bounds__(1024) ln_forward(const LnArgs a) {
  grid_dependency_wait();
  __shared__ float2 red[2][32];
  const int size = a.size, groups = blockDim.x / size, group = threadIdx.x / size, tid = threadIdx.x - group * size;
  for (long long row = (long long)blockIdx.x * groups + group; row < a.rows; row += (long long)gridDim.x * groups) {
    const int c0 = Held<T, VEC, N>::first(tid);
    Held<T, VEC, N> x;
    x.template load<false>(static_cast<const T*>(a.x) + row * a.ldx, c0, a.cols);
    uint64_t s = 0;
#pragma unroll
    for (int p = 0; p < N / 2; ++p) s = add2(s, x.pair(p));
    const float mean = row_mean(a, group_sum(make_float2(sum_of(s), 0.f), red[0], size, group).x);
    s = 0;
#pragma unroll
    for (int p = 0; p < N / 2; ++p) {
      const uint64_t d = add2(x.pair(p), x.template minus<false>(mean, p, c0, a.cols));
      s = fma2(d, d, s);
    }
    const float rstd = 1.f / sqrtf(group_sum(make_float2(sum_of(s), 0.f), red[1], size, group).x * a.inv_cols + a.eps);
    if (tid == 0) put_stats(a, row, mean, rstd);
    uint64_t g[N / 2], b[N / 2], out[N / 2];
    load_params<P, VEC, N>(a.gamma, 1.f, c0, a.cols, g);
    load_params<P, VEC, N>(a.beta, 0.f, c0, a.cols, b);
#pragma unroll
    for (int p = 0; p < N / 2; ++p) out[p] = fma2(mul2(add2(x.pair(p), twice(-mean)), twice(rstd)), g[p], b[p]);
    store_held<T, VEC, N, false>(static_cast<T*>(a.y) + row * a.ldy, out, c0, a.cols);
  }
}

// Two rows at a time, so that their reductions overlap, up to 32 values of each per
// thread, the parameters as fp32 in shared memory. The kernel was bound by its
// instructions: 30 per value with 8 values per thread (the fixed work of a row is two
// thirds of that), 19 with 16, 12 like this (8192 x 4096 bf16: 43, 33 and 26 us).
template <typename T, typename P, int VEC, int N, bool EXACT>
__global__ void __launch_bounds__(kRingThreads) ln_forward_ring(const LnArgs a) {
  grid_dependency_wait();
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ uint64_t full[kRingThreads / 32][kMaxSlots];
  __shared__ float2 red[2][32];
  const int size = a.size, groups = kRingThreads / size, group = threadIdx.x / size, tid = threadIdx.x - group * size;
  const long long first = (long long)blockIdx.x * groups + group, step = (long long)gridDim.x * groups;
  const uint32_t bytes = uint32_t(a.cols) * sizeof(T);
  const int c0 = Held<T, VEC, N>::first(tid);
  const bool whole = Held<T, VEC, N>::whole(tid, a.cols);
  float* params = reinterpret_cast<float*>(ring_smem);  // [2][cols rounded up to 4]
  const int pcols = (a.cols + 3) & ~3;
  auto gamma_at = [&](int c) { return a.gamma ? to_f32(static_cast<const P*>(a.gamma)[c]) : 1.f; };
  auto beta_at = [&](int c) { return a.beta ? to_f32(static_cast<const P*>(a.beta)[c]) : 0.f; };
  // the loads of the parameters go out before the copies, which would hold them up, and
  // are waited for behind them
  constexpr int kFirst = 8;
  for (int c = threadIdx.x + kFirst * kRingThreads; c < a.cols; c += kRingThreads) params[c] = gamma_at(c), params[pcols + c] = beta_at(c);
  Ring ring = make_ring(ring_smem + 8 * (size_t)pcols, full, a, groups, group, a.pitch);
  float gammas[kFirst], betas[kFirst];
#pragma unroll
  for (int i = 0; i < kFirst; ++i) {
    const int c = threadIdx.x + i * kRingThreads;
    if (c < a.cols) gammas[i] = gamma_at(c), betas[i] = beta_at(c);
  }
  const T* x = static_cast<const T*>(a.x);
  long long fill = first;  // the next row to copy
  auto copy = [&](int slot, long long row) {
    const T* from = x + row * a.ldx;
    const uint32_t n = granules(from, bytes);
    mbar_arrive_expect_tx(&ring.full[slot], n);
    bulk_load(ring.buf + slot * ring.bytes, granule(from), n, &ring.full[slot]);
  };
  for (int i = 0; i < a.slots && fill < a.rows; ++i, fill += step)
    if (tid == 0) copy(i, fill);
#pragma unroll
  for (int i = 0; i < kFirst; ++i) {
    const int c = threadIdx.x + i * kRingThreads;
    if (c < a.cols) params[c] = gammas[i], params[pcols + c] = betas[i];
  }
  __syncthreads();
  T* y = static_cast<T*>(a.y) + first * a.ldy;
  const T* at = x + first * a.ldx;
  const long long next_y = step * a.ldy, next_x = step * a.ldx;
  for (long long row = first; row < a.rows; row += 2 * step, y += 2 * next_y, at += 2 * next_x) {
    const bool two = row + step < a.rows;
    Held<T, VEC, N> x0, x1;  // a missing second row: the first one again, not stored
    const int slot0 = ring.slot;
    const uint8_t* from0 = ring.buf + slot0 * ring.bytes + (VEC > 1 ? 0 : shift(at));
    ring.wait(a.status);
    if (two) ring.next(), ring.wait(a.status);
    const int slot1 = ring.slot;
    const uint8_t* from1 = VEC > 1 || !two ? ring.buf + slot1 * ring.bytes + (VEC > 1 ? 0 : shift(at)) : ring.buf + slot1 * ring.bytes + shift(at + next_x);
    ring.next();
    uint64_t s0 = 0, s1 = 0;
    by_whole<EXACT>(whole, [&](auto w) {
      x0.template load<decltype(w)::value>(reinterpret_cast<const T*>(from0), c0, a.cols);
      x1.template load<decltype(w)::value>(reinterpret_cast<const T*>(from1), c0, a.cols);
#pragma unroll
      for (int p = 0; p < N / 2; ++p) s0 = add2(s0, x0.pair(p)), s1 = add2(s1, x1.pair(p));
    });
    const float2 sum = group_sum(make_float2(sum_of(s0), sum_of(s1)), red[0], size, group);
    const float2 mean = make_float2(row_mean(a, sum.x), row_mean(a, sum.y));
    // the reduction is behind every thread's reads of the buffers
    if (tid == 0) {
      if (fill < a.rows) copy(slot0, fill);
      if (two && fill + step < a.rows) copy(slot1, fill + step);
    }
    fill += 2 * step;
    s0 = s1 = 0;
    by_whole<EXACT>(whole, [&](auto w) {
#pragma unroll
      for (int p = 0; p < N / 2; ++p) {
        const uint64_t d0 = add2(x0.pair(p), x0.template minus<decltype(w)::value>(mean.x, p, c0, a.cols));
        const uint64_t d1 = add2(x1.pair(p), x1.template minus<decltype(w)::value>(mean.y, p, c0, a.cols));
        s0 = fma2(d0, d0, s0);
        s1 = fma2(d1, d1, s1);
      }
    });
    const float2 sq = group_sum(make_float2(sum_of(s0), sum_of(s1)), red[1], size, group);
    const float2 rstd = make_float2(1.f / sqrtf(sq.x * a.inv_cols + a.eps), 1.f / sqrtf(sq.y * a.inv_cols + a.eps));
    if (tid == 0) {
      put_stats(a, row, mean.x, rstd.x);
      if (two) put_stats(a, row + step, mean.y, rstd.y);
    }
    const uint64_t m0 = twice(-mean.x), m1 = twice(-mean.y), r0 = twice(rstd.x), r1 = twice(rstd.y);
    constexpr int C = VEC > 1 ? VEC : 2;  // values stored together
    by_whole<EXACT>(whole, [&](auto w) {
#pragma unroll
      for (int q = 0; q < N / C; ++q) {
        const int ca = c0 + Held<T, VEC, N>::at(q * C / VEC), cb = VEC > 1 ? ca + 1 : ca + Held<T, VEC, N>::at(1);
        if (!decltype(w)::value && ca >= a.cols) continue;
        uint64_t g[C / 2], b[C / 2], out[C / 2];
        if constexpr (VEC > 1) {
#pragma unroll
          for (int i = 0; i < C / 4; ++i) {
            const float4 u = *reinterpret_cast<const float4*>(params + ca + 4 * i), v = *reinterpret_cast<const float4*>(params + pcols + ca + 4 * i);
            g[2 * i] = pair_of(u.x, u.y), g[2 * i + 1] = pair_of(u.z, u.w);
            b[2 * i] = pair_of(v.x, v.y), b[2 * i + 1] = pair_of(v.z, v.w);
          }
        } else {
          const bool in = decltype(w)::value || cb < a.cols;
          g[0] = pair_of(params[ca], in ? params[cb] : 0.f);
          b[0] = pair_of(params[pcols + ca], in ? params[pcols + cb] : 0.f);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (r == 1 && !two) break;
#pragma unroll
          for (int i = 0; i < C / 2; ++i)
            out[i] = fma2(mul2(add2((r ? x1 : x0).pair(q * C / 2 + i), r ? m1 : m0), r ? r1 : r0), g[i], b[i]);
          T* to = y + (r ? next_y : 0);
          if constexpr (VEC > 1) {
            store_pairs<T, VEC>(to + ca, out);
          } else {
            const float2 f = unpair(out[0]);
            from_f32(f.x, to + ca);
            if (decltype(w)::value || cb < a.cols) from_f32(f.y, to + cb);
          }
        }
      }
    });
  }
  if (tid == 0) ring.drain((min(fill, a.rows + step - 1) - first) / step);
}

// Rows longer than a block's registers: a block per row that reads it three times
// (the second and third time from L2).
template <typename T, typename P, int VEC>
__global__ void __launch_bounds__(1024) ln_forward_long(const LnArgs a) {
  grid_dependency_wait();
  constexpr int N = VEC > 1 ? VEC : 2;
  __shared__ float2 red[2][32];
  const int c0 = Held<T, VEC, N>::first(threadIdx.x);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    T* y = static_cast<T*>(a.y) + row * a.ldy;
    uint64_t s = 0;
#pragma unroll 4
    for (int c = 0; c < a.cols; c += 1024 * N) {
      Held<T, VEC, N> v;
      v.template load<false>(x + c, c0, a.cols - c);
#pragma unroll
      for (int p = 0; p < N / 2; ++p) s = add2(s, v.pair(p));
    }
    const float mean = row_mean(a, group_sum(make_float2(sum_of(s), 0.f), red[0], 1024, 0).x);
    s = 0;
#pragma unroll 4
    for (int c = 0; c < a.cols; c += 1024 * N) {
      Held<T, VEC, N> v;
      v.template load<false>(x + c, c0, a.cols - c);
#pragma unroll
      for (int p = 0; p < N / 2; ++p) {
        const uint64_t d = add2(v.pair(p), v.template minus<false>(mean, p, c0, a.cols - c));
        s = fma2(d, d, s);
      }
    }
    const float rstd = 1.f / sqrtf(group_sum(make_float2(sum_of(s), 0.f), red[1], 1024, 0).x * a.inv_cols + a.eps);
    if (threadIdx.x == 0) put_stats(a, row, mean, rstd);
#pragma unroll 2
    for (int c = 0; c < a.cols; c += 1024 * N) {
      Held<T, VEC, N> v;
      v.template load<false>(x + c, c0, a.cols - c);
      uint64_t g[N / 2], b[N / 2], out[N / 2];
      load_params<P, VEC, N>(a.gamma, 1.f, c + c0, a.cols, g);
      load_params<P, VEC, N>(a.beta, 0.f, c + c0, a.cols, b);
#pragma unroll
      for (int p = 0; p < N / 2; ++p) out[p] = fma2(mul2(add2(v.pair(p), twice(-mean)), twice(rstd)), g[p], b[p]);
      store_held<T, VEC, N, false>(y + c, out, c0, a.cols - c);
    }
  }
}

// ---------------------------------------------------------------- backward
// A thread's columns across the rows of its group.
template <typename T, typename P, int VEC, int N>
struct Columns {
  uint64_t gamma[N / 2], dg[N / 2], db[N / 2];

  __device__ __forceinline__ void init(const LnArgs& a, int c0) {
    load_params<P, VEC, N>(a.gamma, 1.f, c0, a.cols, gamma);
#pragma unroll
    for (int p = 0; p < N / 2; ++p) dg[p] = db[p] = 0;
  }
  // Adds a row and returns its sums of w and w h. Past the row's end dy and gamma are
  // zero, and so is what they add.
  __device__ __forceinline__ float2 add(const Held<T, VEC, N>& x, const Held<T, VEC, N>& y, float mean, float rstd) {
    uint64_t s1 = 0, s2 = 0;
    const uint64_t m = twice(-mean), r = twice(rstd);
#pragma unroll
    for (int p = 0; p < N / 2; ++p) {
      const uint64_t dy = y.pair(p), h = mul2(add2(x.pair(p), m), r), w = mul2(dy, gamma[p]);
      dg[p] = fma2(dy, h, dg[p]);
      db[p] = add2(db[p], dy);
      s1 = add2(s1, w);
      s2 = fma2(w, h, s2);
    }
    return make_float2(sum_of(s1), sum_of(s2));
  }
  // dx = rstd (w - c1 - h c2)
  template <bool EXACT>
  __device__ __forceinline__ void write(const Held<T, VEC, N>& x, const Held<T, VEC, N>& y, T* dx, int c0, int cols, float mean,
                                        float rstd, float c1, float c2) {
    const uint64_t m = twice(-mean), r = twice(rstd), r1 = twice(-rstd * c1), r2 = twice(-rstd * c2 * rstd);
    uint64_t out[N / 2];
#pragma unroll
    for (int p = 0; p < N / 2; ++p) out[p] = fma2(mul2(y.pair(p), gamma[p]), r, fma2(add2(x.pair(p), m), r2, r1));
    store_held<T, VEC, N, EXACT>(dx, out, c0, cols);
  }
  // 4 of the thread's column sums (its values 4 q..4 q + 3) to a partial row.
  static __device__ __forceinline__ void put4(float* part, int q, int c0, int cols, float4 v) {
    const int c = c0 + (4 * q / VEC) * 32 * VEC + 4 * q % VEC;
    if constexpr (VEC > 1) {
      if (c < cols) *reinterpret_cast<float4*>(part + c) = v;
    } else {
      const float u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + 32 * i < cols) part[c + 32 * i] = u[i];
    }
  }
  static __device__ __forceinline__ float4 four(const uint64_t (&v)[N / 2], int q) {
    const float2 a = unpair(v[2 * q]), b = unpair(v[2 * q + 1]);
    return make_float4(a.x, a.y, b.x, b.y);
  }
  // The block's partial row: its groups' column sums, added in group order. `sums`:
  // shared memory, [groups][2 N / 4][size] (one group needs none).
  __device__ __forceinline__ void finish(const LnArgs& a, int tid, int size, int group, int groups, float4* sums) {
    float* part = a.part + (long long)blockIdx.x * 2 * a.cols;
    const int c0 = Held<T, VEC, N>::first(tid);
    if (groups == 1) {
#pragma unroll
      for (int q = 0; q < N / 4; ++q) put4(part, q, c0, a.cols, four(dg, q)), put4(part + a.cols, q, c0, a.cols, four(db, q));
      return;
    }
    const int step = N / 2 * size;
    float4* mine = sums + group * step + tid;
#pragma unroll
    for (int q = 0; q < N / 4; ++q) mine[q * size] = four(dg, q), mine[(N / 4 + q) * size] = four(db, q);
    __syncthreads();
    for (int q = group; q < N / 2; q += groups) {
      float4 t = sums[q * size + tid];
      for (int g = 1; g < groups; ++g) {
        const float4 u = sums[g * step + q * size + tid];
        t.x += u.x, t.y += u.y, t.z += u.z, t.w += u.w;
      }
      put4(q < N / 4 ? part : part + a.cols, q < N / 4 ? q : q - N / 4, c0, a.cols, t);
    }
  }
};

// Few rows: direct loads, the next row's issued before this row's reduction.
template <typename T, typename P, int VEC, int N>
__global__ void __launch_bounds__(512) ln_backward(const LnArgs a) {
  grid_dependency_wait();
  __shared__ float2 red[2][32];
  extern __shared__ __align__(128) uint8_t ring_smem[];
  const int size = a.size, groups = blockDim.x / size, group = threadIdx.x / size, tid = threadIdx.x - group * size;
  const long long first = (long long)blockIdx.x * groups + group, step = (long long)gridDim.x * groups;
  const int c0 = Held<T, VEC, N>::first(tid);
  Held<T, VEC, N> nx, ny;
  float next_mean = 0.f, next_rstd = 0.f;
  auto fetch = [&](long long row) {
    nx.template load<false>(static_cast<const T*>(a.x) + row * a.ldx, c0, a.cols);
    ny.template load<false>(static_cast<const T*>(a.dy) + row * a.lddy, c0, a.cols);
    next_mean = a.mean[row], next_rstd = a.rstd[row];
  };
  if (first < a.rows) fetch(first);
  Columns<T, P, VEC, N> c;
  c.init(a, c0);
  int flip = 0;
  for (long long row = first; row < a.rows; row += step, flip ^= 1) {
    const Held<T, VEC, N> x = nx, y = ny;
    const float mean = next_mean, rstd = next_rstd;
    if (row + step < a.rows) fetch(row + step);
    const float2 s = group_sum(c.add(x, y, mean, rstd), red[flip], size, group);
    if (a.dx)
      c.template write<false>(x, y, static_cast<T*>(a.dx) + row * a.lddx, c0, a.cols, mean, rstd, s.x * a.inv_cols, s.y * a.inv_cols);
  }
  grid_dependents_launch();
  c.finish(a, tid, size, group, groups, reinterpret_cast<float4*>(ring_smem));
}

// x and dy through the ring, a row per turn. Narrow rows pay for a warp, a wait, two copies
// and a reduction each (65536x64 bf16 32 us, 4 us of reading and writing). The copies queued ahead of it make any other load slow
// (a mean loaded one row ahead measured 3400 cycles of waiting per row), so mean and
// rstd are loaded 32 rows at a time, one row per lane, 32 rows ahead.
template <typename T, typename P, int VEC, int N, bool EXACT>
__global__ void __launch_bounds__(kRingThreads) ln_backward_ring(const LnArgs a) {
  grid_dependency_wait();
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ uint64_t full[kRingThreads / 32][kMaxSlots];
  __shared__ float2 red[2][32];
  const int size = a.size, groups = kRingThreads / size, group = threadIdx.x / size, tid = threadIdx.x - group * size, lane = threadIdx.x & 31;
  const long long first = (long long)blockIdx.x * groups + group, step = (long long)gridDim.x * groups;
  const uint32_t bytes = uint32_t(a.cols) * sizeof(T);
  const int c0 = Held<T, VEC, N>::first(tid);
  const bool whole = Held<T, VEC, N>::whole(tid, a.cols);
  Columns<T, P, VEC, N> c;
  c.init(a, c0);
  float mean32, rstd32, next_mean32, next_rstd32;
  auto fetch = [&](long long row) {
    const bool here = row + lane * step < a.rows;
    next_mean32 = here ? a.mean[row + lane * step] : 0.f;
    next_rstd32 = here ? a.rstd[row + lane * step] : 0.f;
  };
  fetch(first);
  Ring ring = make_ring(ring_smem, full, a, groups, group, 2 * a.pitch);
  long long fill = first;
  const T *x = static_cast<const T*>(a.x), *dy = static_cast<const T*>(a.dy);
  const long long next_dx = step * a.lddx;
  uint32_t sx = shift(x + first * a.ldx), sy = shift(dy + first * a.lddy);  // of this row, modulo 16
  const uint32_t next_sx = uint32_t(step * a.ldx) * uint32_t(sizeof(T)), next_sy = uint32_t(step * a.lddy) * uint32_t(sizeof(T));
  T* dx = static_cast<T*>(a.dx) + (a.dx ? first * a.lddx : 0);
  auto copy = [&](int slot) {
    const T *fx = x + fill * a.ldx, *fy = dy + fill * a.lddy;
    const uint32_t nx = granules(fx, bytes), ny = granules(fy, bytes);
    uint8_t* to = ring.buf + slot * ring.bytes;
    mbar_arrive_expect_tx(&ring.full[slot], nx + ny);
    bulk_load(to, granule(fx), nx, &ring.full[slot]);
    bulk_load(to + a.pitch, granule(fy), ny, &ring.full[slot]);
  };
  for (int i = 0; i < a.slots && fill < a.rows; ++i, fill += step)
    if (tid == 0) copy(i);
  int flip = 0, at = 0;
  for (long long row = first; row < a.rows; row += step, flip ^= 1, at = (at + 1) & 31) {
    if (at == 0) {
      mean32 = next_mean32, rstd32 = next_rstd32;
      fetch(row + 32 * step);
    }
    const float mean = __shfl_sync(0xffffffffu, mean32, at), rstd = __shfl_sync(0xffffffffu, rstd32, at);
    ring.wait(a.status);
    const uint8_t* from = ring.buf + ring.slot * ring.bytes;
    const T *rx = reinterpret_cast<const T*>(from + (VEC > 1 ? 0 : sx & 15)), *ry = reinterpret_cast<const T*>(from + a.pitch + (VEC > 1 ? 0 : sy & 15));
    Held<T, VEC, N> hx, hy;
    by_whole<EXACT>(whole, [&](auto w) {
      hx.template load<decltype(w)::value>(rx, c0, a.cols);
      hy.template load<decltype(w)::value>(ry, c0, a.cols);
    });
    const float2 s = group_sum(c.add(hx, hy, mean, rstd), red[flip], size, group);
    // the reduction is behind every thread's reads of the buffer
    if (tid == 0 && fill < a.rows) copy(ring.slot);
    fill += step, sx += next_sx, sy += next_sy;
    ring.next();
    if (a.dx)
      by_whole<EXACT>(whole, [&](auto w) {
        c.template write<decltype(w)::value>(hx, hy, dx, c0, a.cols, mean, rstd, s.x * a.inv_cols, s.y * a.inv_cols);
      });
    dx += next_dx;
  }
  if (tid == 0) ring.drain((min(fill, a.rows + step - 1) - first) / step);
  grid_dependents_launch();
  __syncthreads();  // the buffers are free: they take the groups' sums
  c.finish(a, tid, size, group, groups, reinterpret_cast<float4*>(ring_smem));
}

// Long rows, first pass: a block per row, its mean, rstd and two sums to `stats`.
template <typename T, typename P, int VEC>
__global__ void __launch_bounds__(512) ln_row_sums(const LnArgs a) {
  grid_dependency_wait();
  constexpr int N = VEC > 1 ? VEC : 2;
  __shared__ float2 red[2][32];
  const int c0 = Held<T, VEC, N>::first(threadIdx.x);
  int flip = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    const float mean = a.mean[row], rstd = a.rstd[row];
    uint64_t s1 = 0, s2 = 0;
    const uint64_t m = twice(-mean), r = twice(rstd);
#pragma unroll 2
    for (int c = 0; c < a.cols; c += 512 * N) {
      Held<T, VEC, N> hx, hy;
      hx.template load<false>(x + c, c0, a.cols - c);
      hy.template load<false>(dy + c, c0, a.cols - c);
      uint64_t g[N / 2];
      load_params<P, VEC, N>(a.gamma, 1.f, c + c0, a.cols, g);
#pragma unroll
      for (int p = 0; p < N / 2; ++p) {
        const uint64_t w = mul2(hy.pair(p), g[p]);
        s1 = add2(s1, w);
        s2 = fma2(w, mul2(add2(hx.pair(p), m), r), s2);
      }
    }
    const float2 s = group_sum(make_float2(sum_of(s1), sum_of(s2)), red[flip], 512, 0);
    if (threadIdx.x == 0) a.stats[row] = make_float4(mean, rstd, s.x * a.inv_cols, s.y * a.inv_cols);
  }
}

// Long rows, second pass: blockIdx.x is a slab of columns, blockIdx.y a part of the
// rows; the row sums are known, so threads own their columns without a reduction.
constexpr int kSlabThreads = 256, kSlabRows = 4;
template <typename T, typename P, int VEC>
__global__ void __launch_bounds__(kSlabThreads) ln_backward_slab(const LnArgs a) {
  grid_dependency_wait();
  constexpr int N = VEC > 1 ? VEC : 2;
  const int c0 = blockIdx.x * kSlabThreads * N + Held<T, VEC, N>::first(threadIdx.x);
  Columns<T, P, VEC, N> c;
  c.init(a, c0);
  for (long long row0 = (long long)blockIdx.y * kSlabRows; row0 < a.rows; row0 += (long long)gridDim.y * kSlabRows) {
    Held<T, VEC, N> x[kSlabRows], y[kSlabRows];
    float4 st[kSlabRows];
#pragma unroll
    for (int r = 0; r < kSlabRows; ++r) {
      const long long row = row0 + r;
      const bool here = row < a.rows;
      const int cols = here ? a.cols : 0;
      x[r].template load<false>(static_cast<const T*>(a.x) + row * a.ldx, c0, cols);
      y[r].template load<false>(static_cast<const T*>(a.dy) + row * a.lddy, c0, cols);
      st[r] = here ? a.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int r = 0; r < kSlabRows; ++r) {
      if (row0 + r >= a.rows) break;
      c.add(x[r], y[r], st[r].x, st[r].y);
      if (a.dx)
        c.template write<false>(x[r], y[r], static_cast<T*>(a.dx) + (row0 + r) * a.lddx, c0, a.cols, st[r].x, st[r].y, st[r].z, st[r].w);
    }
  }
  float* part = a.part + (long long)blockIdx.y * 2 * a.cols;
#pragma unroll
  for (int v = 0; v < N; v += 2) {
    const float2 g = unpair(c.dg[v / 2]), b = unpair(c.db[v / 2]);
    const int ca = c0 + (v / VEC) * 32 * VEC + v % VEC, cb = VEC > 1 ? ca + 1 : ca + 32;
    if (ca < a.cols) part[ca] = g.x, part[a.cols + ca] = b.x;
    if (cb < a.cols) part[cb] = g.y, part[a.cols + cb] = b.y;
  }
}

// dgamma / dbeta = the partial rows added in order: 32 columns per block, the
// partial rows dealt to 32 warps, their sums added in warp order.
__global__ void __launch_bounds__(1024) ln_column_sums(const float* part, int parts, int cols, float* dgamma, float* dbeta) {
  grid_dependency_wait();
  __shared__ float2 sums[32][33];
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
  int vec;      // values per access: 16 bytes of the row's type, or 1
  int n;        // values per thread; 0: the long-row kernels
  int size;     // threads per row
  int threads;  // per block
  bool ring;    // rows through shared memory
  int slots;    // row buffers per group
  uint32_t pitch;
  size_t smem;
};

constexpr int kHeld = 8192;  // values of a row that the backward kernels hold at once
constexpr int kRingBytes = 128 * 1024;  // copies in flight per SM; more only lengthens the queue for all loads
constexpr int kSharedMax = 225 * 1024;

// 16-byte accesses need every row of every tensor to start on a 16-byte boundary and
// to end on one; other rows go value by value.
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
  auto fit = [&](int n, int most) {  // threads that hold a row with n values each
    p.n = n, p.size = 32;
    while (p.size < most && (long long)p.size * n < d.cols) p.size *= 2;
    return (long long)p.size * n >= d.cols;
  };
  // The ring pays from about one row per group of the GPU on (bf16, direct and ring:
  // forward 300x4096 5.2 and 5.5 us, 600x4096 7.0 and 6.0, 2400x1024, where it is one row,
  // 7.55 and 7.60; backward 150x4096, half a row, 8.2 and 8.2 us, 300x4096 11.7 and 9.5,
  // 600x777 7.4 and 7.8, 1200x1024 9.6 and 8.3): up to 32 values per thread in the
  // forward pass (16 one by one), 16 in the backward pass (three more registers each), in
  // as few threads as hold the row. One by one in the backward pass bf16 takes 16 (8192 x
  // 4095: 52 us, 65 us with 8) and fp32, whose two rows and sums then fill the registers,
  // 8 while they hold the row (65 us, 75 us with 16).
  const int most = wide && !backward ? 32 : backward && !wide && es == 4 && d.cols <= 8 * kRingThreads ? 8 : 16, least = 8;
  for (int n = most; n >= least; n /= 2) {
    if (!fit(n, kRingThreads)) break;
    if (p.size == 32 && 32 * (n / 2) >= d.cols && n / 2 >= least) continue;
    const int groups = kRingThreads / p.size;
    p.pitch = (uint32_t(d.cols) * es + (wide ? 15 : 30)) & ~15u;
    const size_t stage = size_t(groups) * p.pitch * (backward ? 2 : 1), params = backward ? 0 : 8 * size_t((d.cols + 3) & ~3);
    if (params + 3 * stage > kSharedMax) continue;  // fewer values per thread: fewer groups, fewer buffers
    p.slots = int(std::min({size_t(kMaxSlots), std::max<size_t>(kRingBytes / stage, 3), (kSharedMax - params) / stage}));
    p.smem = p.slots * stage + params;
    if (backward) p.smem = std::max(p.smem, size_t(kRingThreads) * 2 * p.n * sizeof(float));
    p.ring = 4 * d.rows >= (backward ? 3LL : 4LL) * sms * groups;
    p.threads = kRingThreads;
    if (p.ring) return p;
    break;
  }
  p.smem = 0;
  if (backward) {
    // few rows: threads first, then values per thread
    if (!(fit(8, 512) || fit(16, 512))) p.n = 0;
    p.threads = 512;
    p.smem = size_t(512) * 2 * p.n * sizeof(float);
  } else {
    const int few = wide ? p.vec : 2;
    if (!(fit(few, 1024) || fit(8, 1024) || fit(16, 1024))) p.n = 0;
    p.threads = std::max(p.size, 128);
  }
  return p;
}

// Blocks along the rows in the backward pass, each with one partial row of column
// sums: at most two per SM. (From the sizes alone: the workspace is asked for before
// the pointers are known.)
int ln_parts(long long rows, int sms) { return int(std::max(1LL, std::min(rows, 2LL * sms))); }
// The partial rows, then (long rows) 4 values per row.
size_t ln_part_floats(const pkt_layernorm_desc* d, int sms) { return (size_t(ln_parts(d->rows, sms)) * 2 * d->cols + 3) / 4 * 4; }
size_t ln_workspace(const pkt_layernorm_desc* d, int sms) {
  return (ln_part_floats(d, sms) + (d->cols > kHeld ? size_t(d->rows) * 4 : 0)) * sizeof(float);
}

unsigned ln_blocks(long long n) { return unsigned(std::min(n, 1LL << 30)); }

template <typename... KArgs>
int ln_launch(void (*kernel)(KArgs...), std::atomic<uint64_t>* done, int dev, const LnArgs& a, const LnPlan& p, unsigned blocks, cudaStream_t st) {
  const int rc = done ? op_shared_memory(reinterpret_cast<const void*>(kernel), done, dev, kSharedMax) : PKT_OK;
  if (rc) return rc;
  const cudaError_t e = op_launch(kernel, dim3(blocks), dim3(p.threads), p.smem, st, a);
  return e == cudaSuccess ? PKT_OK : cuda_fail(e, "launch layer norm");
}

// The launches of one plan. In the backward direction the result is the number of
// partial rows written.
template <typename T, typename P, int VEC, int N>
int ln_run(const LnArgs& a, const LnPlan& p, bool backward, int dev, int sms, cudaStream_t st) {
  static std::atomic<uint64_t> done[5];  // one per kernel
  const bool exact = a.cols == p.size * N;
  if (!backward) {
    if constexpr (N >= 8) {
      if (p.ring && VEC > 1 && exact) return ln_launch(ln_forward_ring<T, P, VEC, N, VEC != 1>, &done[0], dev, a, p, sms, st);
      if (p.ring) return ln_launch(ln_forward_ring<T, P, VEC, N, false>, &done[1], dev, a, p, sms, st);
    }
    if constexpr (N <= 16) return ln_launch(ln_forward<T, P, VEC, N>, nullptr, dev, a, p, ln_blocks((a.rows - 1) / (p.threads / p.size) + 1), st);
  } else if constexpr (N == 8 || N == 16) {
    int blocks = std::min(a.parts, sms), rc;
    if (p.ring && VEC > 1 && exact) {
      rc = ln_launch(ln_backward_ring<T, P, VEC, N, VEC != 1>, &done[2], dev, a, p, blocks, st);
    } else if (p.ring) {
      rc = ln_launch(ln_backward_ring<T, P, VEC, N, false>, &done[3], dev, a, p, blocks, st);
    } else {
      blocks = int(std::min<long long>(a.parts, (a.rows - 1) / (p.threads / p.size) + 1));
      rc = ln_launch(ln_backward<T, P, VEC, N>, &done[4], dev, a, p, blocks, st);
    }
    return rc ? rc : blocks;
  }
  return fail(PKT_ERR_UNSUPPORTED, "layer norm of %d columns", a.cols);
}

template <typename T, typename P, int VEC>
int ln_pick(const LnArgs& a, const LnPlan& p, bool backward, int dev, int sms, cudaStream_t st) {
  if (p.n == 0) {
    if (!backward) {
      const cudaError_t e = op_launch(ln_forward_long<T, P, VEC>, dim3(ln_blocks(a.rows)), dim3(1024), 0, st, a);
      return e == cudaSuccess ? PKT_OK : cuda_fail(e, "launch layer norm");
    }
    const int slabs = (a.cols - 1) / (kSlabThreads * (VEC > 1 ? VEC : 2)) + 1;
    const long long want = std::max(1LL, 8LL * sms / slabs);  // about 8 blocks of 256 threads per SM
    const int rows = int(std::min<long long>({want, a.parts, (a.rows - 1) / kSlabRows + 1}));
    cudaError_t e = op_launch(ln_row_sums<T, P, VEC>, dim3(ln_blocks(a.rows)), dim3(512), 0, st, a);
    if (e == cudaSuccess) e = op_launch(ln_backward_slab<T, P, VEC>, dim3(slabs, rows), dim3(kSlabThreads), 0, st, a);
    return e == cudaSuccess ? rows : cuda_fail(e, "launch layer norm");
  }
  switch (p.n) {
    case 2: if constexpr (VEC == 1) return ln_run<T, P, VEC, 2>(a, p, backward, dev, sms, st); break;
    case 4: if constexpr (VEC == 4) return ln_run<T, P, VEC, 4>(a, p, backward, dev, sms, st); break;
    case 8: return ln_run<T, P, VEC, 8>(a, p, backward, dev, sms, st);
    case 16: return ln_run<T, P, VEC, 16>(a, p, backward, dev, sms, st);
    case 32: if constexpr (VEC > 1) return ln_run<T, P, VEC, 32>(a, p, backward, dev, sms, st); break;
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
  if (d->cols > (1 << 29)) return fail(PKT_ERR_UNSUPPORTED, "layer norm of %d columns", d->cols);
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
  a.size = p.size, a.slots = p.slots, a.pitch = p.pitch, a.status = status;
  a.rows = d.rows, a.cols = d.cols, a.eps = d.eps, a.num_cols = float(d.cols), a.inv_cols = 1.f / a.num_cols;
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
  if (d->dgamma || d->dbeta) {
    const cudaError_t e = op_launch(ln_column_sums, dim3((d->cols - 1) / 32 + 1), dim3(1024), 0, st, static_cast<const float*>(a.part), rc,
                                    a.cols, d->dgamma, d->dbeta);
    if (e != cudaSuccess) return cuda_fail(e, "launch layer norm column sums");
  }
  return PKT_OK;
}

}  // extern "C"
