// pkt_fp8_quantize: block-scaled 8-bit operands, plain and transposed, from one read.
//
// Bound by memory: a value is read once (2 or 4 bytes) and written once or twice as
// one byte, with one fp32 scale per 128 or 128 x 128 values. Measured at 8192x4096:
//   bf16, rows      17.1 us, 5.90 TB/s    bf16, both ways 24.0 us, 5.59 TB/s
//   fp32, rows      26.4 us, 6.35 TB/s    fp32, both ways 33.6 us, 6.00 TB/s
// (6.55 TB/s: a plain copy). What the bf16 forms lack is instruction issue: about 3 per
// value with both results.
//
// A warp holds 128 columns of a row, 4 consecutive ones per lane. Rows alone
// (block_rows 1, no transposed result) need nothing beyond a warp: the largest
// magnitude is one warp reduction, and a warp takes 4 or 16 rows: their loads overlap and
// their scales are computed at once, one per lane. Otherwise a block of 8 warps takes a
// 128 x 128 tile into registers (a lane has 4 columns x 16 rows, so a column's 16 values
// of a warp are 16 consecutive bytes of the transposed result); column maxima meet in
// shared memory, and the transposed bytes pass through it to leave as whole 128-byte rows.
#include <algorithm>

#include "ops_common.h"
#include "ops_device.cuh"

namespace pkb {
namespace {

struct QuantArgs {
  int rows, cols, block_rows;
  const void* x;
  long long ldx;
  uint8_t* q;
  long long ldq;
  float* scale;
  long long ld_scale;
  uint8_t* qt;
  long long ldqt;
  float* scale_t;
  long long ld_scale_t;
  float most;
};

// A lane's 4 consecutive values of a row as raw words.
template <typename T>
using Row4 = Raw<T, 4>;

// The largest magnitude of 4 values, as bits of |x| in fp32: packed pairs for bf16.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t row_big(const Row4<bf16_t>& r) {
  const uint32_t m = max_u16x2(r.w[0] & 0x7fff7fffu, r.w[1] & 0x7fff7fffu);
  return max(m << 16, m & 0xffff0000u);
}
__device__ __forceinline__ uint32_t row_big(const Row4<float>& r) {
  return max(max(r.w[0] & 0x7fffffffu, r.w[1] & 0x7fffffffu), max(r.w[2] & 0x7fffffffu, r.w[3] & 0x7fffffffu));
}
// The largest magnitude of each of 4 columns over N rows.
template <int N>
__device__ __forceinline__ void cols_big(const Row4<bf16_t> (&r)[N], uint32_t (&big)[4]) {
  uint32_t a = 0, b = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) a = max_u16x2(a, r[i].w[0] & 0x7fff7fffu), b = max_u16x2(b, r[i].w[1] & 0x7fff7fffu);
  big[0] = a << 16, big[1] = a & 0xffff0000u, big[2] = b << 16, big[3] = b & 0xffff0000u;
}
template <int N>
__device__ __forceinline__ void cols_big(const Row4<float> (&r)[N], uint32_t (&big)[4]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    big[c] = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) big[c] = max(big[c], r[i].w[c] & 0x7fffffffu);
  }
}

// 4 consecutive values that start s values into two neighbouring groups of 4.
__device__ __forceinline__ Row4<bf16_t> shifted(const Row4<bf16_t>& lo, const Row4<bf16_t>& hi, uint32_t s) {
  const uint32_t x0 = s & 2 ? lo.w[1] : lo.w[0], x1 = s & 2 ? hi.w[0] : lo.w[1], x2 = s & 2 ? hi.w[1] : hi.w[0], bits = 16 * (s & 1);
  Row4<bf16_t> r;
  r.w[0] = __funnelshift_r(x0, x1, bits), r.w[1] = __funnelshift_r(x1, x2, bits);
  return r;
}

// N rows of 4 columns: all loads before the first use. `whole`: every value is inside
// the matrix. bf16 rows that do not start on a boundary of 4 values (!WIDE) are read as
// the two aligned groups of 4 that hold a lane's values, a few rows at a time: a group
// with one value of the matrix in it is memory that may be read, and what else it holds
// goes (8192x4097 both ways 36 us, value by value 57 us; fp32 55 and 42 us).
template <typename T, bool WIDE, int N>
__device__ __forceinline__ void load_rows(const QuantArgs& a, long long row0, int col, bool whole, Row4<T> (&r)[N]) {
  const T* p = static_cast<const T*>(a.x) + row0 * a.ldx + col;
  if (WIDE && whole) {
#pragma unroll
    for (int i = 0; i < N; ++i, p += a.ldx) r[i].load(p, true);
    return;
  }
  const int left = a.cols - col;
  if constexpr (WIDE || sizeof(T) == 4) {
    const bool four = WIDE && left >= 4;
#pragma unroll
    for (int i = 0; i < N; ++i, p += a.ldx) {
#pragma unroll
      for (int k = 0; k < Row4<T>::kWords; ++k) r[i].w[k] = 0;
      if (row0 + i >= a.rows) continue;
      if (four) {
        r[i].load(p, true);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < left) r[i].set(k, p[k]);
      }
    }
  } else {
    uint32_t keep[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) keep[k] = 2 * k + 1 < left ? ~0u : 2 * k < left ? 0xffffu : 0u;
    constexpr int B = 4;
#pragma unroll
    for (int i0 = 0; i0 < N; i0 += B) {
      Row4<T> lo[B], hi[B];
      uint32_t s[B];
#pragma unroll
      for (int i = 0; i < B; ++i, p += a.ldx) {
        const bool in = row0 + i0 + i < a.rows;
        s[i] = uint32_t(reinterpret_cast<uintptr_t>(p) / sizeof(T)) & 3;
        const T* from = p - s[i];
        lo[i].load(from, in && left > 0);
        hi[i].load(from + 4, in && s[i] > 0 && left > 4 - int(s[i]));
      }
#pragma unroll
      for (int i = 0; i < B; ++i) {
        r[i0 + i] = shifted(lo[i], hi[i], s[i]);
#pragma unroll
        for (int k = 0; k < 2; ++k) r[i0 + i].w[k] &= keep[k];
      }
    }
  }
}

// 4 bytes of a row that starts on a 16-byte boundary, only those inside the matrix
__device__ __forceinline__ void store_cols4(uint8_t* row, int col, int cols, uint32_t q) {
  if (col + 4 <= cols) {
    *reinterpret_cast<uint32_t*>(row + col) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < cols) row[col + i] = uint8_t(q >> (8 * i));
  }
}

template <bool E5M2>
__device__ __forceinline__ uint32_t quantize4(uint64_t v01, uint64_t v23, uint64_t f) {
  const float2 a = unpair(mul2(v01, f)), b = unpair(mul2(v23, f));
  return pack_fp8x4<E5M2>(a.x, a.y, b.x, b.y);
}
template <typename T, bool E5M2>
__device__ __forceinline__ uint32_t quantize_row4(const Row4<T>& r, float f) {
  return quantize4<E5M2>(r.get2(0), r.get2(1), pair_of(f, f));
}

// N rows of 4 columns to q, row i with factor(i).
template <typename T, bool E5M2, int N, typename F>
__device__ __forceinline__ void store_rows(const QuantArgs& a, long long row0, int col, bool whole, const Row4<T> (&r)[N], F factor) {
  uint8_t* q = a.q + row0 * a.ldq;
  if (whole) {
    q += col;
#pragma unroll
    for (int i = 0; i < N; ++i, q += a.ldq) *reinterpret_cast<uint32_t*>(q) = quantize_row4<T, E5M2>(r[i], factor(i));
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i, q += a.ldq) {
    const uint32_t w = quantize_row4<T, E5M2>(r[i], factor(i));
    if (row0 + i < a.rows) store_cols4(q, col, a.cols, w);
  }
}

// Quantises N rows of a warp, each with its own scale: one reduction per row, then the
// N scales at once, one per lane.
template <typename T, bool E5M2, int N>
__device__ __forceinline__ void quantize_each_row(const QuantArgs& a, long long row0, int col, int kb, bool whole, const Row4<T> (&r)[N], int lane) {
  uint32_t big = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, row_big(r[i]));
    if (lane == i) big = m;
  }
  float f, s;
  block_scale(big, a.most, &f, &s);
  if (lane < N && row0 + lane < a.rows) a.scale[kb * a.ld_scale + row0 + lane] = s;
  store_rows<T, E5M2>(a, row0, col, whole, r, [&](int i) { return __shfl_sync(0xffffffffu, f, i); });
}

// Registers follow the blocks per SM that hide the most latency. 16 rows, 8192x4096 again
// and again: bf16 15.7 us with 8 blocks, 17.2 us with 6 and 18.2 us with 5; fp32 36.7 us with
// 8, 26.9 us with 6 (it spills 104 bytes) and 26.7 us with 5. bf16 rows off the boundary of 4
// values spill 188 bytes with 8 blocks (8192x4097 34.5 us; 31.2 us with 6).
template <typename T, bool WIDE, bool E5M2, int N>
__global__ void __launch_bounds__(128, N < 16 ? 1 : sizeof(T) == 2 ? 8 : 6) quantize_rows(const QuantArgs a) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, kb = blockIdx.x, col = kb * kScaleBlock + 4 * lane;
  const long long groups = ((long long)a.rows + N - 1) / N;
  for (long long g = (long long)blockIdx.y * 4 + (threadIdx.x >> 5); g < groups; g += (long long)gridDim.y * 4) {
    const long long row0 = g * N;
    const bool whole = row0 + N <= a.rows && (kb + 1LL) * kScaleBlock <= a.cols;
    Row4<T> r[N];
    load_rows<T, WIDE>(a, row0, col, whole, r);
    quantize_each_row<T, E5M2>(a, row0, col, kb, whole, r, lane);
  }
}

// Blocks per SM with both results, 8192x4096: bf16 31.5 us with 2, 26.7 us with 3 and
// 23.9 us with 4 (16 bytes spilled); fp32 49.0 us with 1, 33.6 us with 2 and with 3, but
// 4096x1024 in 128 x 128 blocks 4.6 us with 2 and 5.0 us with 3.
template <typename T, bool WIDE, bool E5M2>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2) quantize_tile(const QuantArgs a) {
  grid_dependency_wait();
  __shared__ __align__(16) uint32_t col_big[8][128];
  __shared__ __align__(16) float col_factor[128];
  __shared__ uint32_t tile_big[8];
  __shared__ __align__(16) uint8_t bytes[128 * 128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kb = blockIdx.x, col = kb * 128 + 4 * lane;
  const bool square = a.block_rows == 128;
  const int row_tiles = (a.rows - 1) / 128 + 1;
  for (int rt = blockIdx.y; rt < row_tiles; rt += gridDim.y) {
    const long long row0 = (long long)rt * 128 + warp * 16;
    const bool whole = (rt + 1LL) * 128 <= a.rows && (kb + 1LL) * 128 <= a.cols;
    Row4<T> r[16];
    load_rows<T, WIDE>(a, row0, col, whole, r);
    uint32_t cbig[4];
    float f = 0.f, s = 0.f;
    if (square || a.qt) cols_big(r, cbig);
    if (square) {
      const uint32_t big = __reduce_max_sync(0xffffffffu, max(max(cbig[0], cbig[1]), max(cbig[2], cbig[3])));
      if (lane == 0) tile_big[warp] = big;
      __syncthreads();
      uint32_t all = tile_big[0];
#pragma unroll
      for (int w = 1; w < 8; ++w) all = max(all, tile_big[w]);
      block_scale(all, a.most, &f, &s);
      if (threadIdx.x == 0) {
        if (a.q) a.scale[kb * a.ld_scale + rt] = s;
        if (a.qt) a.scale_t[rt * a.ld_scale_t + kb] = s;
      }
      if (a.q) store_rows<T, E5M2>(a, row0, col, whole, r, [&](int) { return f; });
    } else {
      *reinterpret_cast<uint4*>(&col_big[warp][4 * lane]) = make_uint4(cbig[0], cbig[1], cbig[2], cbig[3]);
      __syncthreads();
      if (threadIdx.x < 128) {
        uint32_t all = col_big[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < 8; ++w) all = max(all, col_big[w][threadIdx.x]);
        float cf, cs;
        block_scale(all, a.most, &cf, &cs);
        col_factor[threadIdx.x] = cf;
        if (kb * 128 + threadIdx.x < a.cols) a.scale_t[rt * a.ld_scale_t + kb * 128 + threadIdx.x] = cs;
      }
      if (a.q) quantize_each_row<T, E5M2>(a, row0, col, kb, whole, r, lane);
    }
    if (a.qt) {
      __syncthreads();  // col_factor is written; the tile before has left `bytes`
      const float4 cf = square ? make_float4(f, f, f, f) : *reinterpret_cast<const float4*>(&col_factor[4 * lane]);
      const float cfs[4] = {cf.x, cf.y, cf.z, cf.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = quantize4<E5M2>(pair_of(r[4 * k].get(i), r[4 * k + 1].get(i)), pair_of(r[4 * k + 2].get(i), r[4 * k + 3].get(i)),
                                 pair_of(cfs[i], cfs[i]));
        // 16-byte pieces of a row are permuted by its column group: 8 lanes, 8 banks
        *reinterpret_cast<uint4*>(bytes + (4 * lane + i) * 128 + ((warp ^ (lane & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      __syncthreads();
      const int piece = threadIdx.x & 7;
      const long long left = a.rows - (long long)rt * 128 - piece * 16;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = k * 32 + (threadIdx.x >> 3), out = kb * 128 + c;
        if (out >= a.cols || left <= 0) continue;
        const uint4 w = *reinterpret_cast<const uint4*>(bytes + c * 128 + ((piece ^ ((c >> 2) & 7)) * 16));
        uint8_t* to = a.qt + out * a.ldqt + (long long)rt * 128 + piece * 16;
        if (left >= 16) {
          *reinterpret_cast<uint4*>(to) = w;
        } else {
          const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (i < left) to[i] = uint8_t(ws[i >> 2] >> (8 * (i & 3)));
        }
      }
    }
    __syncthreads();  // the maxima and bytes are free for the next tile
  }
}

template <typename T, bool WIDE, bool E5M2>
cudaError_t quantize_run(const QuantArgs& a, int sms, cudaStream_t st) {
  const unsigned kbs = unsigned((a.cols - 1) / kScaleBlock + 1);
  if (a.block_rows == 1 && !a.qt) {
    // 16 rows per warp keep more bytes in flight, 4 start more warps: bf16 256x4096 (54
    // row blocks per SM) takes 2.4 us with 16 and 2.2 us with 4, 512x4096 2.8 and 3.1 us,
    // 8192x4096 17.5 and 34 us. Off the boundary of 4 values: bf16 4099x777 (194 row
    // blocks per SM) 8.8 us with 16 and 5.4 us with 4, 8192x4097 34 and 40 us; fp32, value
    // by value, takes 4.
    const bool many = (WIDE || sizeof(T) == 2) && (long long)kbs * a.rows >= (WIDE ? 110LL : 440LL) * sms;
    const int rows = many ? 64 : 16;
    const dim3 grid(kbs, unsigned(std::min((a.rows - 1) / rows + 1, 65535)));
    if constexpr (WIDE || sizeof(T) == 2)
      if (many) return op_launch(quantize_rows<T, WIDE, E5M2, 16>, grid, dim3(128), 0, st, a);
    return op_launch(quantize_rows<T, WIDE, E5M2, 4>, grid, dim3(128), 0, st, a);
  }
  const int tiles = (a.rows - 1) / 128 + 1;
  return op_launch(quantize_tile<T, WIDE, E5M2>, dim3(kbs, unsigned(std::min(tiles, 65535))), dim3(256), 0, st, a);
}

template <typename T>
cudaError_t quantize_dispatch(const QuantArgs& a, bool wide, bool e5m2, int sms, cudaStream_t st) {
  if (wide) return e5m2 ? quantize_run<T, true, true>(a, sms, st) : quantize_run<T, true, false>(a, sms, st);
  return e5m2 ? quantize_run<T, false, true>(a, sms, st) : quantize_run<T, false, false>(a, sms, st);
}

int check_result(const char* name, const void* q, long long ld, const float* scale, long long ld_scale, int cols, long long scales) {
  if (!aligned_to(q, 16) || ld % 16 != 0) return fail(PKT_ERR_ARGS, "%s must be 16-byte aligned with a row stride that is a multiple of 16", name);
  if (ld < cols) return fail(PKT_ERR_ARGS, "row stride %lld of %s is below its %d columns", ld, name, cols);
  if (!scale || !aligned_to(scale, 4)) return fail(PKT_ERR_ARGS, "%s needs its scales, aligned to 4 bytes", name);
  if (ld_scale < scales) return fail(PKT_ERR_ARGS, "row stride %lld of %s's scales is below their %lld columns", ld_scale, name, scales);
  return PKT_OK;
}

}  // namespace
}  // namespace pkb

extern "C" int pkt_fp8_quantize(const pkt_fp8_quantize_desc* d, void* stream) {
  using namespace pkb;
  if (!d) return fail(PKT_ERR_ARGS, "null quantize descriptor");
  if (d->rows < 0 || d->cols < 0) return fail(PKT_ERR_ARGS, "quantize of %d x %d values", d->rows, d->cols);
  constexpr int kMost = 0x7fffffff - 127;  // the last tile's columns are counted in 32 bits
  if (d->rows > kMost || d->cols > kMost) return fail(PKT_ERR_UNSUPPORTED, "quantize of %d x %d values", d->rows, d->cols);
  if (d->dtype != PKT_DTYPE_BF16 && d->dtype != PKT_DTYPE_F32) return fail(PKT_ERR_ARGS, "quantize dtype must be bf16 or f32");
  if (d->q_dtype != PKT_DTYPE_E4M3 && d->q_dtype != PKT_DTYPE_E5M2) return fail(PKT_ERR_ARGS, "quantize q_dtype must be e4m3 or e5m2");
  if (d->block_rows != 1 && d->block_rows != 128) return fail(PKT_ERR_ARGS, "block_rows must be 1 or 128");
  if (!d->q && !d->qt) return fail(PKT_ERR_ARGS, "quantize needs q or qt");
  if (d->rows == 0 || d->cols == 0) return PKT_OK;
  int dev = 0, sms = 0, rc;
  const int es = d->dtype == PKT_DTYPE_BF16 ? 2 : 4;
  if (!d->x || !aligned_to(d->x, es)) return fail(PKT_ERR_ARGS, "quantize needs x, aligned to its type");
  if (d->ldx < d->cols) return fail(PKT_ERR_ARGS, "row stride %lld of x is below the %d columns", d->ldx, d->cols);
  if (d->q && (rc = check_result("q", d->q, d->ldq, d->scale, d->ld_scale, d->cols, (d->rows - 1) / d->block_rows + 1))) return rc;
  if (d->qt && (rc = check_result("qt", d->qt, d->ldqt, d->scale_t, d->ld_scale_t, d->rows, (d->cols - 1) / d->block_rows + 1))) return rc;
  if ((rc = op_device(&dev, &sms)) || (rc = op_check_memory(d->x, "x", dev)) || (rc = op_check_memory(d->q, "q", dev)) ||
      (d->q && (rc = op_check_memory(d->scale, "scale", dev))) || (rc = op_check_memory(d->qt, "qt", dev)) ||
      (d->qt && (rc = op_check_memory(d->scale_t, "scale_t", dev))))
    return rc;
  QuantArgs a{};
  a.rows = d->rows, a.cols = d->cols, a.block_rows = d->block_rows, a.x = d->x, a.ldx = d->ldx;
  a.q = static_cast<uint8_t*>(d->q), a.ldq = d->ldq, a.scale = d->scale, a.ld_scale = d->ld_scale;
  a.qt = static_cast<uint8_t*>(d->qt), a.ldqt = d->ldqt, a.scale_t = d->scale_t, a.ld_scale_t = d->ld_scale_t;
  const bool e5m2 = d->q_dtype == PKT_DTYPE_E5M2;
  a.most = e5m2 ? 57344.f : 448.f;
  // 4 values in one access: every row of x starts on a boundary of 4 values
  const bool wide = aligned_to(d->x, 4 * es) && d->ldx % 4 == 0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = d->dtype == PKT_DTYPE_BF16 ? quantize_dispatch<bf16_t>(a, wide, e5m2, sms, st) : quantize_dispatch<float>(a, wide, e5m2, sms, st);
  return e == cudaSuccess ? PKT_OK : cuda_fail(e, "launch quantize");
}
