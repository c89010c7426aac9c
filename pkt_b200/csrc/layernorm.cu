// pkt_layernorm_forward / pkt_layernorm_backward.
//
//   forward   mean = sum x / C,  rstd = 1 / sqrt(sum (x - mean)^2 / C + eps),
//             y = (x - mean) rstd gamma + beta
//   backward  h = (x - mean) rstd,  w = dy gamma,
//             dx = rstd (w - mean(w) - h mean(w h)),
//             dgamma = sum over rows of dy h,  dbeta = sum over rows of dy
//
// Both are bound by memory. A row is read once and stays in registers between the
// statistics and the result (the variance is the mean square of the centred
// values, not E x^2 - mean^2, which cancels); short rows belong to one warp
// (shuffles only), longer ones to more threads, and rows beyond what 1024 threads
// hold are read again from L2. All sums are fp32.
//
// The column sums dgamma / dbeta of the backward pass are kept in the registers of
// the threads that own the columns, across the rows of a block; every block writes
// one partial row to the workspace and a second kernel (launched with programmatic
// dependency) adds the partial rows in a fixed order, so results do not depend on
// timing.
#include <algorithm>

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
  float* part;  // backward: [parts][2][cols]
  int parts;
};

constexpr int kWarpsPerBlock = 4;  // rows per block where a warp has a row

// The sum of `v` over the threads of a row: a warp, or the block with one barrier.
// `red` holds one word per warp; the callers alternate between two buffers, so the
// barrier of one reduction protects the other's words.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = warp_sum(v);
  if (WARP) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
  return warp_sum(lane < nw ? red[lane] : 0.f);
}
__device__ __forceinline__ float2 row_sum2(float2 v, float2* red) {
  v.x = warp_sum(v.x), v.y = warp_sum(v.y);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
  const float2 r = lane < nw ? red[lane] : make_float2(0.f, 0.f);
  return make_float2(warp_sum(r.x), warp_sum(r.y));
}

template <typename P, int VEC>
__device__ __forceinline__ void load_param(const void* base, int col, int valid, float other, float (&v)[VEC]) {
  if (base == nullptr) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = i < valid ? other : 0.f;
    return;
  }
  Raw<P, VEC> r;
  r.load(static_cast<const P*>(base) + col, valid);
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = r.get(i);
}

template <typename T, typename P, int VEC, int K, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 1024) ln_forward(const LnArgs a) {
  __shared__ float red[2][32];
  const int size = WARP ? 32 : blockDim.x, tid = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const long long first = WARP ? (long long)blockIdx.x * kWarpsPerBlock + (threadIdx.x >> 5) : blockIdx.x;
  const long long step = WARP ? (long long)gridDim.x * kWarpsPerBlock : gridDim.x;
  for (long long row = first; row < a.rows; row += step) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    Raw<T, VEC> raw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * size + tid) * VEC;
      raw[k].load(x + col, a.cols - col);
    }
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += raw[k].get(i);
    const float mean = row_sum<WARP>(sum, red[0]) * a.inv_cols;
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int valid = a.cols - (k * size + tid) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = i < valid ? raw[k].get(i) - mean : 0.f;
        sq = fmaf(d, d, sq);
      }
    }
    const float rstd = 1.f / sqrtf(row_sum<WARP>(sq, red[1]) * a.inv_cols + a.eps);
    if (tid == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * size + tid) * VEC, valid = a.cols - col;
      if (valid <= 0) continue;
      float g[VEC], b[VEC], out[VEC];
      load_param<P, VEC>(a.gamma, col, valid, 1.f, g);
      load_param<P, VEC>(a.beta, col, valid, 0.f, b);
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = fmaf((raw[k].get(i) - mean) * rstd, g[i], b[i]);
      store_vec<T, VEC>(y + col, out, valid);
    }
  }
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
      r.load(x + col, a.cols - col);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += r.get(i);
    }
    const float mean = row_sum<false>(sum, red[0]) * a.inv_cols;
    float sq = 0.f;
    for (int col = begin; col < a.cols; col += step) {
      Raw<T, VEC> r;
      r.load(x + col, a.cols - col);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = col + i < a.cols ? r.get(i) - mean : 0.f;
        sq = fmaf(d, d, sq);
      }
    }
    const float rstd = 1.f / sqrtf(row_sum<false>(sq, red[1]) * a.inv_cols + a.eps);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.ldy;
    for (int col = begin; col < a.cols; col += step) {
      const int valid = a.cols - col;
      Raw<T, VEC> r;
      r.load(x + col, valid);
      float g[VEC], b[VEC], out[VEC];
      load_param<P, VEC>(a.gamma, col, valid, 1.f, g);
      load_param<P, VEC>(a.beta, col, valid, 0.f, b);
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = fmaf((r.get(i) - mean) * rstd, g[i], b[i]);
      store_vec<T, VEC>(y + col, out, valid);
    }
  }
}

// A row belongs to a group of 32..1024 threads, and a block holds several groups
// where rows are short: enough loads are in flight with few blocks, and so few
// partial rows. The next row's loads are issued before the reduction of this one.
template <typename T, typename P, int VEC, int K>
__global__ void __launch_bounds__(K * VEC * int(sizeof(T)) <= 16 ? 1024 : 512) ln_backward(const LnArgs a, const int size) {
  __shared__ float2 red[2][32];
  extern __shared__ float col_sums[];  // [2][cols] when the block has several groups
  const int groups = blockDim.x / size, group = threadIdx.x / size, tid = threadIdx.x - group * size;
  const long long first = (long long)blockIdx.x * groups + group, step = (long long)gridDim.x * groups;
  const int lane = threadIdx.x & 31, warp0 = group * (size >> 5), warps = size >> 5;
  float gamma[K][VEC], dg[K][VEC], db[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int col = (k * size + tid) * VEC;
    load_param<P, VEC>(a.gamma, col, a.cols - col, 1.f, gamma[k]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) dg[k][i] = db[k][i] = 0.f;
  }
  Raw<T, VEC> rx[K], ry[K], nx[K], ny[K];
  float mean = 0.f, rstd = 0.f, next_mean = 0.f, next_rstd = 0.f;
  auto fetch = [&](long long row) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * size + tid) * VEC;
      nx[k].load(x + col, a.cols - col);
      ny[k].load(dy + col, a.cols - col);
    }
    next_mean = a.mean[row], next_rstd = a.rstd[row];
  };
  if (first < a.rows) fetch(first);
  int flip = 0;
  for (long long row = first; row < a.rows; row += step, flip ^= 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) rx[k] = nx[k], ry[k] = ny[k];
    mean = next_mean, rstd = next_rstd;
    if (row + step < a.rows) fetch(row + step);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        // beyond the row's end dy and gamma are zero, and so is what they add
        const float dy = ry[k].get(i), h = (rx[k].get(i) - mean) * rstd, w = dy * gamma[k][i];
        dg[k][i] = fmaf(dy, h, dg[k][i]);
        db[k][i] += dy;
        s.x += w;
        s.y = fmaf(w, h, s.y);
      }
    s.x = warp_sum(s.x), s.y = warp_sum(s.y);
    if (warps > 1) {
      if (lane == 0) red[flip][threadIdx.x >> 5] = s;
      named_barrier_sync(1 + group, size);
      s = lane < warps ? red[flip][warp0 + lane] : make_float2(0.f, 0.f);
      s.x = warp_sum(s.x), s.y = warp_sum(s.y);
    }
    const float c1 = s.x * a.inv_cols, c2 = s.y * a.inv_cols;
    if (a.dx) {
      T* dx = static_cast<T*>(a.dx) + row * a.lddx;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int col = (k * size + tid) * VEC, valid = a.cols - col;
        if (valid <= 0) continue;
        float out[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float h = (rx[k].get(i) - mean) * rstd;
          out[i] = rstd * (ry[k].get(i) * gamma[k][i] - c1 - h * c2);
        }
        store_vec<T, VEC>(dx + col, out, valid);
      }
    }
  }
  grid_dependents_launch();
  // the groups' column sums, added in group order
  float* part = a.part + (long long)blockIdx.x * 2 * a.cols;
  for (int g = 0; g < groups; ++g) {
    if (group == g) {
      const bool last = g == groups - 1;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int col = (k * size + tid) * VEC + i;
          if (col >= a.cols) continue;
          const float2 before = g == 0 ? make_float2(0.f, 0.f) : make_float2(col_sums[col], col_sums[a.cols + col]);
          float* to = last ? part : col_sums;
          to[col] = before.x + dg[k][i];
          to[a.cols + col] = before.y + db[k][i];
        }
    }
    __syncthreads();
  }
}

// Rows longer than a block's registers: x and dy are read twice (the second time
// from L2) and the column sums live in this block's partial row of the workspace.
template <typename T, typename P, int VEC>
__global__ void __launch_bounds__(1024) ln_backward_long(const LnArgs a) {
  __shared__ float2 red[2][32];
  const int step = blockDim.x * VEC, begin = threadIdx.x * VEC;
  float* part = a.part + (long long)blockIdx.x * 2 * a.cols;
  int flip = 0;
  bool fresh = true;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1, fresh = false) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dyp = static_cast<const T*>(a.dy) + row * a.lddy;
    T* dx = a.dx ? static_cast<T*>(a.dx) + row * a.lddx : nullptr;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float2 s = make_float2(0.f, 0.f);
    for (int col = begin; col < a.cols; col += step) {
      const int valid = a.cols - col;
      Raw<T, VEC> rx, ry;
      rx.load(x + col, valid);
      ry.load(dyp + col, valid);
      float g[VEC];
      load_param<P, VEC>(a.gamma, col, valid, 1.f, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float w = ry.get(i) * g[i];
        s.x += w;
        s.y = fmaf(w, (rx.get(i) - mean) * rstd, s.y);
      }
    }
    s = row_sum2(s, red[flip]);
    const float c1 = s.x * a.inv_cols, c2 = s.y * a.inv_cols;
    for (int col = begin; col < a.cols; col += step) {
      const int valid = a.cols - col;
      Raw<T, VEC> rx, ry;
      rx.load(x + col, valid);
      ry.load(dyp + col, valid);
      float g[VEC], out[VEC];
      load_param<P, VEC>(a.gamma, col, valid, 1.f, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float dy = ry.get(i), h = (rx.get(i) - mean) * rstd;
        out[i] = rstd * (dy * g[i] - c1 - h * c2);
        if (i < valid) {
          part[col + i] = fresh ? dy * h : fmaf(dy, h, part[col + i]);
          part[a.cols + col + i] = fresh ? dy : part[a.cols + col + i] + dy;
        }
      }
      if (dx) store_vec<T, VEC>(dx + col, out, valid);
    }
  }
  grid_dependents_launch();
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
  int k;        // vectors per thread; 0: the long-row kernel
  int size;     // threads per row
  int threads;  // per block
};

// 16-byte accesses need every row of every tensor to start on a 16-byte boundary;
// other rows go element by element.
LnPlan ln_plan(const pkt_layernorm_desc& d, bool backward, int sms) {
  const int es = d.dtype == PKT_DTYPE_BF16 ? 2 : 4;
  auto rows_ok = [&](const void* p, long long ld) { return aligned_to(p, 16) && ld * es % 16 == 0; };
  bool wide = rows_ok(d.x, d.ldx) && aligned_to(d.gamma, 16);
  if (backward)
    wide = wide && rows_ok(d.dy, d.lddy) && (!d.dx || rows_ok(d.dx, d.lddx));
  else
    wide = wide && rows_ok(d.y, d.ldy) && aligned_to(d.beta, 16);
  LnPlan p;
  p.vec = wide ? 16 / es : 1;
  const int nvec = (d.cols - 1) / p.vec + 1;
  auto threads_for = [&](int k) {
    int t = 32;
    while (t < 1024 && (long long)t * k < nvec) t *= 2;
    return t;
  };
  if (!backward) {
    // few rows: as many threads as the row has vectors; many rows: up to 4 vectors
    // (8 single elements) each
    const int ks[4] = {1, 2, wide ? 4 : 8, wide ? 4 : 16};
    int i = d.rows >= 2LL * sms ? 2 : 0;
    while (i > 0 && threads_for(ks[i - 1]) == threads_for(ks[i])) --i;
    while (i < 3 && (long long)threads_for(ks[i]) * ks[i] < nvec) ++i;
    p.k = ks[i];
    p.size = threads_for(p.k);
    p.threads = p.size > 32 ? p.size : 32 * kWarpsPerBlock;
  } else {
    // a block has 512 threads, or the 1024 of one row when 16 bytes per thread and
    // tensor do (the kernel's register bound)
    const int ks[3] = {wide ? 1 : 4, wide ? 2 : 8, wide ? 16 / p.vec : 16};
    int i = 0;
    auto fits = [&](int k) {
      const int most = k * p.vec * es <= 16 ? 1024 : 512;
      return threads_for(k) <= most && (long long)threads_for(k) * k >= nvec;
    };
    while (i < 3 && !fits(ks[i])) ++i;
    p.k = i < 3 ? ks[i] : 0;
    p.size = i < 3 ? threads_for(p.k) : 1024;
    p.threads = std::max(512, p.size);
  }
  if (p.k == 0 || (long long)p.size * p.k < nvec) p.k = 0, p.size = p.threads = 1024;
  return p;
}

// Blocks of the backward pass, each with one partial row of column sums: two per SM.
// (From the sizes alone: the workspace is asked for before the pointers are known.)
int ln_parts(long long rows, int sms) { return int(std::max(1LL, std::min(rows, 2LL * sms))); }

template <typename T, typename P, int VEC, int K>
cudaError_t ln_run(const LnArgs& a, const LnPlan& p, bool backward, cudaStream_t st) {
  if constexpr (K * VEC <= 16) if (backward) {
    const size_t smem = p.threads > p.size ? size_t(2) * a.cols * sizeof(float) : 0;
    return op_launch(ln_backward<T, P, VEC, K>, dim3(a.parts), dim3(p.threads), smem, st, false, a, p.size);
  }
  if constexpr (VEC == 1 ? K != 4 : true) {
  if (backward) return cudaErrorInvalidConfiguration;
  if (p.size == 32)
    return op_launch(ln_forward<T, P, VEC, K, true>, dim3(unsigned(std::min((a.rows - 1) / kWarpsPerBlock + 1, 1LL << 30))),
                     dim3(p.threads), 0, st, false, a);
  return op_launch(ln_forward<T, P, VEC, K, false>, dim3(unsigned(std::min(a.rows, 1LL << 30))), dim3(p.threads), 0, st, false, a);
  }
  return cudaErrorInvalidConfiguration;
}

template <typename T, typename P, int VEC>
cudaError_t ln_pick(const LnArgs& a, const LnPlan& p, bool backward, cudaStream_t st) {
  if (p.k == 0) {
    if (backward) return op_launch(ln_backward_long<T, P, VEC>, dim3(a.parts), dim3(1024), 0, st, false, a);
    return op_launch(ln_forward_long<T, P, VEC>, dim3(unsigned(std::min(a.rows, 1LL << 30))), dim3(1024), 0, st, false, a);
  }
  switch (p.k) {
    case 1: return ln_run<T, P, VEC, 1>(a, p, backward, st);
    case 2: return ln_run<T, P, VEC, 2>(a, p, backward, st);
    case 4: return ln_run<T, P, VEC, 4>(a, p, backward, st);
    case 8: if (VEC == 1) return ln_run<T, P, 1, 8>(a, p, backward, st); break;
    case 16: if (VEC == 1) return ln_run<T, P, 1, 16>(a, p, backward, st); break;
  }
  return cudaErrorInvalidConfiguration;
}

template <typename T>
cudaError_t ln_dispatch(const LnArgs& a, const LnPlan& p, int param_dtype, bool backward, cudaStream_t st) {
  constexpr int W = 16 / int(sizeof(T));
  if (param_dtype == PKT_DTYPE_F32)
    return p.vec > 1 ? ln_pick<T, float, W>(a, p, backward, st) : ln_pick<T, float, 1>(a, p, backward, st);
  return p.vec > 1 ? ln_pick<T, bf16_t, W>(a, p, backward, st) : ln_pick<T, bf16_t, 1>(a, p, backward, st);
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

size_t ln_workspace(const pkt_layernorm_desc* d, int sms) { return size_t(ln_parts(d->rows, sms)) * 2 * d->cols * sizeof(float); }

LnArgs ln_args(const pkt_layernorm_desc& d) {
  LnArgs a{};
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
  int dev = 0, sms = 0, rc;
  if ((rc = ln_check_common(d))) return rc;
  if (!(d->eps >= 0.f)) return fail(PKT_ERR_ARGS, "layer norm eps must be >= 0");
  if (d->rows == 0) return PKT_OK;
  if ((rc = ln_check_rows(d->x, d->ldx, "x", d)) || (rc = ln_check_rows(d->y, d->ldy, "y", d)) ||
      (rc = ln_check_param(d->gamma, "gamma", d->param_dtype)) || (rc = ln_check_param(d->beta, "beta", d->param_dtype)) ||
      (rc = ln_check_param(d->mean, "mean", PKT_DTYPE_F32)) || (rc = ln_check_param(d->rstd, "rstd", PKT_DTYPE_F32)))
    return rc;
  if ((rc = op_device(&dev, &sms)) || (rc = op_check_memory(d->x, "x", dev)) || (rc = op_check_memory(d->y, "y", dev)) ||
      (rc = op_check_memory(d->gamma, "gamma", dev)) || (rc = op_check_memory(d->beta, "beta", dev)) ||
      (rc = op_check_memory(d->mean, "mean", dev)) || (rc = op_check_memory(d->rstd, "rstd", dev)))
    return rc;
  const LnPlan p = ln_plan(*d, false, sms);
  const LnArgs a = ln_args(*d);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = d->dtype == PKT_DTYPE_BF16 ? ln_dispatch<bf16_t>(a, p, d->param_dtype, false, st)
                                                   : ln_dispatch<float>(a, p, d->param_dtype, false, st);
  return e == cudaSuccess ? PKT_OK : cuda_fail(e, "launch layer norm forward");
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
  int dev = 0, sms = 0, rc;
  if ((rc = ln_check_common(d)) || (rc = ln_check_param(d->dgamma, "dgamma", PKT_DTYPE_F32)) ||
      (rc = ln_check_param(d->dbeta, "dbeta", PKT_DTYPE_F32)))
    return rc;
  if (d->rows > 0) {
    if ((rc = ln_check_rows(d->x, d->ldx, "x", d)) || (rc = ln_check_rows(d->dy, d->lddy, "dy", d)) ||
        (d->dx && (rc = ln_check_rows(d->dx, d->lddx, "dx", d))) || (rc = ln_check_param(d->gamma, "gamma", d->param_dtype)))
      return rc;
    if (!d->mean || !d->rstd) return fail(PKT_ERR_ARGS, "layer norm backward needs the forward pass's mean and rstd");
    if ((rc = ln_check_param(d->mean, "mean", PKT_DTYPE_F32)) || (rc = ln_check_param(d->rstd, "rstd", PKT_DTYPE_F32)) ||
        (rc = ln_check_param(d->workspace, "workspace", PKT_DTYPE_F32)))
      return rc;
  }
  if ((rc = op_device(&dev, &sms)) || (rc = op_check_memory(d->dgamma, "dgamma", dev)) || (rc = op_check_memory(d->dbeta, "dbeta", dev)))
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
  LnArgs a = ln_args(*d);
  a.parts = ln_parts(d->rows, sms);
  a.part = static_cast<float*>(d->workspace);
  const LnPlan p = ln_plan(*d, true, sms);
  cudaError_t e = d->dtype == PKT_DTYPE_BF16 ? ln_dispatch<bf16_t>(a, p, d->param_dtype, true, st)
                                             : ln_dispatch<float>(a, p, d->param_dtype, true, st);
  if (e != cudaSuccess) return cuda_fail(e, "launch layer norm backward");
  if (d->dgamma || d->dbeta) {
    e = op_launch(ln_column_sums, dim3((d->cols - 1) / 32 + 1), dim3(1024), 0, st, true, static_cast<const float*>(a.part), a.parts, a.cols,
                  d->dgamma, d->dbeta);
    if (e != cudaSuccess) return cuda_fail(e, "launch layer norm column sums");
  }
  return PKT_OK;
}

}  // extern "C"
