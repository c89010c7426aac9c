// pkt_adamw_*: one AdamW step over many tensors in one launch.
//
// Bound by memory: 28 bytes per parameter with fp32 states (parameter, m and v read
// and written, gradient read), 16 1/8 with 8-bit states, 2 more for a bf16 copy.
// Measured (6.55 TB/s: a plain copy): 41.9 million parameters, fp32 states and a bf16
// copy 200 us, 6.29 TB/s; 268 million, 8-bit states and a copy 790 us alone and 827 us
// among others, 5.9 TB/s; 5.3 million in 6 tensors, 8-bit states 21 us, 4.1 TB/s (a block
// has one or two chunks, each behind a chain of chunk record, tensor record and data; a
// block that fetches the records of 16 chunks ahead takes 21 and, on 268 million, 810 us).
// The tensors are cut into chunks of 4096 values, listed once in device memory; a
// block takes every gridDim-th chunk, and within it a warp owns blocks of 128 values,
// 4 per lane, so that a block of 8-bit states is quantised with one warp reduction.
// All loads of a warp's share are issued before the first is used, and the scales of
// its 8 state blocks are computed at once, one per lane.
//
// 8-bit states hold m and r = sqrt(v) as e4m3 with an fp32 scale per 128 values. The
// root, because its range is half of v's in octaves (e4m3 spans 18 octaves below the
// block's maximum, v would need 36) and because r is what the update divides by.
// The arithmetic of a step is fp32 with each operation rounded on its own where the
// result is quantised, so the stored 8-bit values do not depend on how a compiler
// contracts the expressions.
//
// The step count and the bias corrections live on the device: every block reads the
// corrections, and the last block to finish (an atomic ticket) advances them, in
// 64 bits, so a captured step can be replayed.
#include <algorithm>
#include <cmath>
#include <exception>
#include <utility>
#include <vector>

#include "ops_common.h"
#include "ops_device.cuh"

namespace pkb {
namespace {

constexpr int kChunk = 4096;
constexpr int kAdamThreads = 256;
constexpr int kBlocksPerWarp = kChunk / kScaleBlock / (kAdamThreads / 32);

struct AdamTensor {
  void* param;
  const void* grad;
  void *m, *v;
  float *m_scale, *v_scale;
  uint16_t* copy;
  long long n;
  float decay;
  int wide;  // every array starts on a boundary of 4 of its values
};

struct AdamState {
  double pow1, pow2;  // beta1^t, beta2^t of the steps taken
  long long step;
  float inv_bc1, inv_root_bc2;  // of the next step
  unsigned ticket;
};

struct AdamArgs {
  const AdamTensor* tensors;
  const int2* chunks;  // tensor, chunk within it
  int num_chunks;
  AdamState* state;
  const float* scales;
  float lr, grad_scale, b1, c1, b2, c2, eps;
  double beta1, beta2;
};

__device__ __forceinline__ void adam_advance(AdamState* s, double beta1, double beta2) {
  s->step += 1;
  s->pow1 *= beta1;
  s->pow2 *= beta2;
  s->inv_bc1 = float(1.0 / (1.0 - s->pow1 * beta1));
  s->inv_root_bc2 = float(1.0 / sqrt(1.0 - s->pow2 * beta2));
}

__global__ void adam_set_state(AdamState* s, double pow1, double pow2, long long step, double beta1, double beta2) {
  grid_dependency_wait();
  s->pow1 = pow1;
  s->pow2 = pow2;
  s->step = step;
  s->inv_bc1 = float(1.0 / (1.0 - pow1 * beta1));
  s->inv_root_bc2 = float(1.0 / sqrt(1.0 - pow2 * beta2));
}

// A lane's 4 values of a block of 128: consecutive, one access (FULL), or 32 apart and
// one by one, only those inside the tensor.
template <bool FULL, typename T>
__device__ __forceinline__ void load4(const T* p, int lane, int left, Raw<T, 4>* r) {
  if constexpr (FULL) {
    r->load(p + 4 * lane, true);
  } else {
#pragma unroll
    for (int i = 0; i < Raw<T, 4>::kWords; ++i) r->w[i] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < left) r->set(i, p[lane + 32 * i]);
  }
}
template <bool FULL, typename T>
__device__ __forceinline__ void store4(T* p, int lane, int left, const float (&v)[4]) {
  if constexpr (FULL) {
    store_vec<T, 4>(p + 4 * lane, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < left) from_f32(v[i], p + lane + 32 * i);
  }
}
template <bool FULL>
__device__ __forceinline__ uint32_t load_bytes4(const uint8_t* p, int lane, int left) {
  if constexpr (FULL) return *reinterpret_cast<const uint32_t*>(p + 4 * lane);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < left) w |= uint32_t(p[lane + 32 * i]) << (8 * i);
  return w;
}
template <bool FULL>
__device__ __forceinline__ void store_bytes4(uint8_t* p, int lane, int left, uint32_t w) {
  if constexpr (FULL) {
    *reinterpret_cast<uint32_t*>(p + 4 * lane) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < left) p[lane + 32 * i] = uint8_t(w >> (8 * i));
  }
}
__device__ __forceinline__ void unpack4(uint32_t w, float scale, float (&v)[4]) {
  const float2 lo = unpack_e4m3x2(uint16_t(w)), hi = unpack_e4m3x2(uint16_t(w >> 16));
  v[0] = __fmul_rn(lo.x, scale), v[1] = __fmul_rn(lo.y, scale), v[2] = __fmul_rn(hi.x, scale), v[3] = __fmul_rn(hi.y, scale);
}

// The factors of a step that all values share.
struct AdamStep {
  float gs, keep, step_size, inv_root;
};

// A warp's 4 blocks of 128 values from `base` on. FULL: all of them inside the tensor
// and every array aligned.
template <typename P, typename G, bool EIGHT, bool FULL>
__device__ __forceinline__ void adam_blocks(const AdamArgs& a, const AdamTensor& t, const AdamStep& u, long long base, int lane) {
  constexpr int B = kBlocksPerWarp;
  P* param = static_cast<P*>(t.param) + base;
  Raw<P, 4> rp[B];
  Raw<G, 4> rg[B];
  Raw<float, 4> rm[EIGHT ? 1 : B], rv[EIGHT ? 1 : B];
  uint32_t mq[EIGHT ? B : 1], vq[EIGHT ? B : 1];
  float ms[EIGHT ? B : 1], vs[EIGHT ? B : 1];
  const long long sb = base / kScaleBlock;
#pragma unroll
  for (int b = 0; b < B; ++b) {
    const int left = FULL ? kScaleBlock : int(min(t.n - base - b * kScaleBlock, (long long)kScaleBlock));
    load4<FULL>(param + b * kScaleBlock, lane, left, &rp[b]);
    load4<FULL>(static_cast<const G*>(t.grad) + base + b * kScaleBlock, lane, left, &rg[b]);
    if constexpr (EIGHT) {
      mq[b] = load_bytes4<FULL>(static_cast<const uint8_t*>(t.m) + base + b * kScaleBlock, lane, left);
      vq[b] = load_bytes4<FULL>(static_cast<const uint8_t*>(t.v) + base + b * kScaleBlock, lane, left);
      ms[b] = FULL || left > 0 ? t.m_scale[sb + b] : 0.f;
      vs[b] = FULL || left > 0 ? t.v_scale[sb + b] : 0.f;
    } else {
      load4<FULL>(static_cast<const float*>(t.m) + base + b * kScaleBlock, lane, left, &rm[b]);
      load4<FULL>(static_cast<const float*>(t.v) + base + b * kScaleBlock, lane, left, &rv[b]);
    }
  }
  float m[B][4], r[B][4];  // new m, new sqrt(v)
  uint32_t big = 0;        // lane b: the largest |m| of block b, lane B + b: of sqrt(v)
#pragma unroll
  for (int b = 0; b < B; ++b) {
    const int left = FULL ? kScaleBlock : int(min(t.n - base - b * kScaleBlock, (long long)kScaleBlock));
    float v[4], p[4];
    if constexpr (EIGHT) {
      unpack4(mq[b], ms[b], m[b]);
      unpack4(vq[b], vs[b], v);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __fmul_rn(v[i], v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) m[b][i] = rm[b].get(i), v[i] = rv[b].get(i);
    }
    uint32_t mbig = 0, rbig = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float g = rg[b].get(i) * u.gs;
      m[b][i] = __fadd_rn(__fmul_rn(m[b][i], a.b1), __fmul_rn(g, a.c1));
      v[i] = __fadd_rn(__fmul_rn(v[i], a.b2), __fmul_rn(__fmul_rn(g, g), a.c2));
      r[b][i] = __fsqrt_rn(v[i]);
      // the quotient's own error is 2 ulp of the step, like the rest of its arithmetic
      // (where p is near zero, of p too)
      p[i] = rp[b].get(i) * u.keep - __fdividef(u.step_size * m[b][i], fmaf(r[b][i], u.inv_root, a.eps));
      mbig = max(mbig, abs_bits(m[b][i]));
      rbig = max(rbig, abs_bits(r[b][i]));
    }
    store4<FULL>(param + b * kScaleBlock, lane, left, p);
    if (t.copy) store4<FULL>(reinterpret_cast<bf16_t*>(t.copy) + base + b * kScaleBlock, lane, left, p);
    if constexpr (EIGHT) {
      mbig = __reduce_max_sync(0xffffffffu, mbig);
      rbig = __reduce_max_sync(0xffffffffu, rbig);
      if (lane == b) big = mbig;
      if (lane == B + b) big = rbig;
    } else {
      store4<FULL>(static_cast<float*>(t.m) + base + b * kScaleBlock, lane, left, m[b]);
      store4<FULL>(static_cast<float*>(t.v) + base + b * kScaleBlock, lane, left, v);
    }
  }
  if constexpr (EIGHT) {
    float factor, scale;  // of 8 blocks at once, one per lane
    block_scale(big, 448.f, &factor, &scale);
    if (lane < 2 * B && (FULL || base + (lane & (B - 1)) * kScaleBlock < t.n)) (lane < B ? t.m_scale : t.v_scale)[sb + (lane & (B - 1))] = scale;
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int left = FULL ? kScaleBlock : int(min(t.n - base - b * kScaleBlock, (long long)kScaleBlock));
      const float mf = __shfl_sync(0xffffffffu, factor, b), rf = __shfl_sync(0xffffffffu, factor, B + b);
      store_bytes4<FULL>(static_cast<uint8_t*>(t.m) + base + b * kScaleBlock, lane, left,
                         pack_fp8x4<false>(__fmul_rn(m[b][0], mf), __fmul_rn(m[b][1], mf), __fmul_rn(m[b][2], mf), __fmul_rn(m[b][3], mf)));
      uint32_t q = pack_fp8x4<false>(__fmul_rn(r[b][0], rf), __fmul_rn(r[b][1], rf), __fmul_rn(r[b][2], rf), __fmul_rn(r[b][3], rf));
      // a root above zero stays above zero: the smallest 8-bit value is code 1
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r[b][i] > 0.f && rf > 0.f && ((q >> (8 * i)) & 0xffu) == 0) q |= 1u << (8 * i);
      store_bytes4<FULL>(static_cast<uint8_t*>(t.v) + base + b * kScaleBlock, lane, left, q);
    }
  }
}

// Three blocks per SM with 8-bit states leave 80 registers, and the form with fp32 gradients
// spills 84 bytes; it is faster all the same (5.3 million values: 25.6 us with two blocks and
// 22.5 us with three).
template <typename P, typename G, bool EIGHT>
__global__ void __launch_bounds__(kAdamThreads, EIGHT ? 3 : 2) adam_step(const AdamArgs a) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float lr = a.scales ? a.lr * a.scales[0] : a.lr;
  AdamStep u;
  u.gs = a.scales ? a.grad_scale * a.scales[1] : a.grad_scale;
  u.step_size = lr * a.state->inv_bc1;
  u.inv_root = a.state->inv_root_bc2;
  for (int c = blockIdx.x; c < a.num_chunks; c += gridDim.x) {
    const int2 where = a.chunks[c];
    const AdamTensor t = a.tensors[where.x];
    if (t.grad == nullptr) continue;
    u.keep = 1.f - lr * t.decay;
    const long long base = (long long)where.y * kChunk + warp * (kBlocksPerWarp * kScaleBlock);
    if (t.wide && base + kBlocksPerWarp * kScaleBlock <= t.n)
      adam_blocks<P, G, EIGHT, true>(a, t, u, base, lane);
    else if (base < t.n)
      adam_blocks<P, G, EIGHT, false>(a, t, u, base, lane);
  }
  __syncthreads();  // every thread of the block has read the state
  if (threadIdx.x == 0 && atomicAdd(&a.state->ticket, 1u) == gridDim.x - 1) {
    a.state->ticket = 0;
    adam_advance(a.state, a.beta1, a.beta2);
  }
}

struct AdamW {
  int device = 0, sms = 0;
  std::vector<AdamTensor> tensors;
  std::vector<std::pair<uintptr_t, uintptr_t>> written;  // begin and end of every array that a step writes, in order
  int num_chunks = 0;
  int param_dtype = 0, grad_dtype = 0, state_dtype = 0;
  double beta1 = 0, beta2 = 0, eps = 0;
  AdamTensor* d_tensors = nullptr;
  int2* d_chunks = nullptr;
  AdamState* d_state = nullptr;

  ~AdamW() {
    RelaxedCapture relaxed;  // a plan may be dropped while some stream is being captured
    int before = 0;
    const bool back = cudaGetDevice(&before) == cudaSuccess && before != device;
    cudaSetDevice(device);
    cudaFree(d_tensors);
    cudaFree(d_chunks);
    cudaFree(d_state);
    if (back) cudaSetDevice(before);
  }
  void set_wide(AdamTensor* t) const {
    const size_t p = param_dtype == PKT_DTYPE_F32 ? 16 : 8, g = grad_dtype == PKT_DTYPE_F32 ? 16 : 8,
                 s = state_dtype == PKT_DTYPE_F32 ? 16 : 4;
    t->wide = aligned_to(t->param, p) && aligned_to(t->grad, g) && aligned_to(t->m, s) && aligned_to(t->v, s) && aligned_to(t->copy, 8);
  }
  // Arrays that a step writes must not overlap (two chunks would race), nor a gradient
  // with one of them; gradients may be shared.
  void writes(const void* p, long long n, size_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    if (p) written.push_back({at, at + size_t(n) * bytes});
  }
  int sort_written() {
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i)
      if (written[i].first < written[i - 1].second) return fail(PKT_ERR_ARGS, "arrays that an AdamW step writes overlap");
    return PKT_OK;
  }
  int check_grad(const void* g, size_t i) const {
    const size_t bytes = grad_dtype == PKT_DTYPE_F32 ? 4 : 2;
    if (!g || tensors[i].n == 0) return PKT_OK;
    if (!aligned_to(g, bytes)) return fail(PKT_ERR_ARGS, "grad of tensor %zu is not aligned to its type", i);
    const uintptr_t at = reinterpret_cast<uintptr_t>(g), end = at + size_t(tensors[i].n) * bytes;
    const auto next = std::upper_bound(written.begin(), written.end(), at, [](uintptr_t v, const std::pair<uintptr_t, uintptr_t>& w) { return v < w.second; });
    if (next != written.end() && next->first < end) return fail(PKT_ERR_ARGS, "grad of tensor %zu overlaps an array that the step writes", i);
    return op_check_memory(g, "grad", device);
  }
  int set_step(long long step, cudaStream_t st) {
    const cudaError_t e = op_launch(adam_set_state, dim3(1), dim3(1), 0, st, d_state, std::pow(beta1, double(step)),
                                    std::pow(beta2, double(step)), step, beta1, beta2);
    return e == cudaSuccess ? PKT_OK : cuda_fail(e, "set the AdamW step");
  }
  int setup(const pkt_adamw_config& c);
  int run(float lr, float grad_scale, const float* scales, cudaStream_t st);
};

int AdamW::setup(const pkt_adamw_config& c) {
  if (c.num_tensors < 0 || (c.num_tensors > 0 && !c.tensors)) return fail(PKT_ERR_ARGS, "bad AdamW tensor list");
  if (c.param_dtype != PKT_DTYPE_F32 && c.param_dtype != PKT_DTYPE_BF16) return fail(PKT_ERR_ARGS, "AdamW param_dtype must be f32 or bf16");
  if (c.grad_dtype != PKT_DTYPE_F32 && c.grad_dtype != PKT_DTYPE_BF16) return fail(PKT_ERR_ARGS, "AdamW grad_dtype must be f32 or bf16");
  if (c.state_dtype != PKT_DTYPE_F32 && c.state_dtype != PKT_DTYPE_E4M3) return fail(PKT_ERR_ARGS, "AdamW state_dtype must be f32 or e4m3");
  if (!(c.beta1 >= 0 && c.beta1 < 1 && c.beta2 >= 0 && c.beta2 < 1)) return fail(PKT_ERR_ARGS, "AdamW betas must be in [0, 1)");
  if (!(c.eps >= 0) || !std::isfinite(c.eps)) return fail(PKT_ERR_ARGS, "AdamW eps must be >= 0");
  if (c.step < 0) return fail(PKT_ERR_ARGS, "AdamW step must be >= 0");
  param_dtype = c.param_dtype, grad_dtype = c.grad_dtype, state_dtype = c.state_dtype;
  beta1 = c.beta1, beta2 = c.beta2, eps = c.eps;
  const bool eight = state_dtype == PKT_DTYPE_E4M3;
  const size_t ps = param_dtype == PKT_DTYPE_F32 ? 4 : 2, ss = eight ? 1 : 4;
  std::vector<int2> chunks;
  int rc;
  for (int i = 0; i < c.num_tensors; ++i) {
    const pkt_adamw_tensor& s = c.tensors[i];
    if (s.n < 0) return fail(PKT_ERR_ARGS, "tensor %d has %lld values", i, s.n);
    if (s.n == 0) {  // it has no chunk: its pointers may be the next tensor's, or any
      tensors.push_back(AdamTensor{});
      continue;
    }
    if (!s.param || !s.m || !s.v) return fail(PKT_ERR_ARGS, "tensor %d needs param, m and v", i);
    if (eight && (!s.m_scale || !s.v_scale)) return fail(PKT_ERR_ARGS, "tensor %d needs m_scale and v_scale (8-bit states)", i);
    if (!aligned_to(s.param, ps) || !aligned_to(s.m, ss) || !aligned_to(s.v, ss) || !aligned_to(s.m_scale, 4) || !aligned_to(s.v_scale, 4) ||
        !aligned_to(s.copy_bf16, 2))
      return fail(PKT_ERR_ARGS, "an array of tensor %d is not aligned to its type", i);
    if ((rc = op_check_memory(s.param, "param", device)) || (rc = op_check_memory(s.m, "m", device)) || (rc = op_check_memory(s.v, "v", device)) ||
        (rc = op_check_memory(s.copy_bf16, "copy_bf16", device)))
      return rc;
    if (eight && ((rc = op_check_memory(s.m_scale, "m_scale", device)) || (rc = op_check_memory(s.v_scale, "v_scale", device)))) return rc;
    AdamTensor t{s.param, s.grad, s.m, s.v, s.m_scale, s.v_scale, static_cast<uint16_t*>(s.copy_bf16), s.n, s.weight_decay, 0};
    set_wide(&t);
    tensors.push_back(t);
    writes(s.param, s.n, ps), writes(s.m, s.n, ss), writes(s.v, s.n, ss), writes(s.copy_bf16, s.n, 2);
    if (eight) writes(s.m_scale, (s.n - 1) / kScaleBlock + 1, 4), writes(s.v_scale, (s.n - 1) / kScaleBlock + 1, 4);
    const long long count = (s.n - 1) / kChunk + 1;
    if (count + (long long)chunks.size() > 0x7fffffffLL) return fail(PKT_ERR_ARGS, "too many parameters for one AdamW plan");
    for (long long k = 0; k < count; ++k) chunks.push_back(make_int2(i, int(k)));
  }
  if ((rc = sort_written())) return rc;
  for (size_t i = 0; i < tensors.size(); ++i)
    if ((rc = check_grad(tensors[i].grad, i))) return rc;
  num_chunks = int(chunks.size());
  cudaError_t e = cudaMalloc(&d_tensors, sizeof(AdamTensor) * std::max<size_t>(1, tensors.size()));
  if (e == cudaSuccess) e = cudaMalloc(&d_chunks, sizeof(int2) * std::max<size_t>(1, chunks.size()));
  if (e == cudaSuccess) e = cudaMalloc(&d_state, sizeof(AdamState));
  if (e == cudaSuccess) e = cudaMemset(d_state, 0, sizeof(AdamState));
  if (e == cudaSuccess && !tensors.empty())
    e = cudaMemcpy(d_tensors, tensors.data(), sizeof(AdamTensor) * tensors.size(), cudaMemcpyHostToDevice);
  if (e == cudaSuccess && num_chunks) e = cudaMemcpy(d_chunks, chunks.data(), sizeof(int2) * chunks.size(), cudaMemcpyHostToDevice);
  if (e != cudaSuccess) return cuda_fail(e, "AdamW tables");
  if ((rc = set_step(c.step, nullptr))) return rc;
  e = cudaDeviceSynchronize();  // the state is set before a step on any stream
  return e == cudaSuccess ? PKT_OK : cuda_fail(e, "AdamW set-up");
}

template <typename P, typename G>
cudaError_t adam_launch(const AdamArgs& a, bool eight, int blocks, cudaStream_t st) {
  return eight ? op_launch(adam_step<P, G, true>, dim3(blocks), dim3(kAdamThreads), 0, st, a)
               : op_launch(adam_step<P, G, false>, dim3(blocks), dim3(kAdamThreads), 0, st, a);
}

int AdamW::run(float lr, float grad_scale, const float* scales, cudaStream_t st) {
  if (!aligned_to(scales, 4)) return fail(PKT_ERR_ARGS, "scales is not aligned to its type");
  int rc = op_check_memory(scales, "scales", device);
  if (rc) return rc;
  AdamArgs a{};
  a.tensors = d_tensors, a.chunks = d_chunks, a.num_chunks = num_chunks, a.state = d_state, a.scales = scales;
  a.lr = lr, a.grad_scale = grad_scale;
  a.b1 = float(beta1), a.c1 = float(1.0 - beta1), a.b2 = float(beta2), a.c2 = float(1.0 - beta2), a.eps = float(eps);
  a.beta1 = beta1, a.beta2 = beta2;
  // One block per chunk up to 8 per SM, more than the 3 (8-bit states, 80 registers) or 2
  // that an SM holds at once: a block that starts late fills the place of one that is done.
  // With 2, 3, 4, 8 and 16 per SM: 5.3 million values, 8-bit states 18.3, 17.2, 17.1, 16.9 and
  // 18.5 us in a graph, fp32 states 21, 24, 22, 24 and 25 us; 268 million 8-bit 867, 834, 929,
  // 811 and 789 us; 41.9 million fp32 208, 202, 206, 198 and 193 us. A plan without values
  // still counts the step.
  const int blocks = std::max(1, std::min(num_chunks, sms * 8));
  const bool eight = state_dtype == PKT_DTYPE_E4M3, pf = param_dtype == PKT_DTYPE_F32, gf = grad_dtype == PKT_DTYPE_F32;
  const cudaError_t e = pf ? (gf ? adam_launch<float, float>(a, eight, blocks, st) : adam_launch<float, bf16_t>(a, eight, blocks, st))
                           : (gf ? adam_launch<bf16_t, float>(a, eight, blocks, st) : adam_launch<bf16_t, bf16_t>(a, eight, blocks, st));
  return e == cudaSuccess ? PKT_OK : cuda_fail(e, "launch AdamW");
}

// The plan's device is current inside a call, the caller's afterwards.
struct OnDevice {
  int before = -1;
  explicit OnDevice(int device) {
    int cur = 0;
    if (cudaGetDevice(&cur) == cudaSuccess && cur != device) {
      before = cur;
      cudaSetDevice(device);
    }
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

// What a captured stream would refuse after it had spoilt the capture is refused before.
int outside_capture(cudaStream_t st, const char* what) {
  cudaStreamCaptureStatus capturing;
  const cudaError_t e = cudaStreamIsCapturing(st, &capturing);
  if (e != cudaSuccess) return cuda_fail(e, "cudaStreamIsCapturing");
  return capturing == cudaStreamCaptureStatusNone ? PKT_OK : fail(PKT_ERR_ARGS, "%s inside a stream capture", what);
}

}  // namespace
}  // namespace pkb

struct pkt_adamw {
  pkb::AdamW plan;
};

extern "C" {

int pkt_adamw_create(int device, const pkt_adamw_config* cfg, pkt_adamw** out) {
  using namespace pkb;
  if (!cfg || !out) return fail(PKT_ERR_ARGS, "null argument");
  int count = 0;
  const cudaError_t e = cudaGetDeviceCount(&count);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDeviceCount");
  if (device < 0 || device >= count) return fail(PKT_ERR_ARGS, "device %d out of range (%d devices)", device, count);
  OnDevice on(device);
  int dev = 0, sms = 0, rc;
  if ((rc = op_device(&dev, &sms))) return rc;
  pkt_adamw* h = nullptr;
  try {
    h = new pkt_adamw();
    h->plan.device = dev, h->plan.sms = sms;
    rc = h->plan.setup(*cfg);
  } catch (const std::exception&) {
    rc = fail(PKT_ERR_ARGS, "out of host memory");
  }
  if (rc) {
    delete h;
    return rc;
  }
  *out = h;
  return PKT_OK;
}

int pkt_adamw_destroy(pkt_adamw* h) {
  delete h;
  return PKT_OK;
}

int pkt_adamw_step(pkt_adamw* h, float lr, float grad_scale, const float* scales, void* stream) {
  if (!h) return pkb::fail(PKT_ERR_ARGS, "null AdamW plan");
  pkb::OnDevice on(h->plan.device);
  return h->plan.run(lr, grad_scale, scales, static_cast<cudaStream_t>(stream));
}

int pkt_adamw_set_grads(pkt_adamw* h, const void* const* grads, void* stream) {
  using namespace pkb;
  if (!h || (!grads && !h->plan.tensors.empty())) return fail(PKT_ERR_ARGS, "null argument");
  AdamW& p = h->plan;
  OnDevice on(p.device);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc = outside_capture(st, "AdamW gradients cannot be set");
  if (rc) return rc;
  for (size_t i = 0; i < p.tensors.size(); ++i)
    if ((rc = p.check_grad(grads[i], i))) return rc;
  for (size_t i = 0; i < p.tensors.size(); ++i) {
    p.tensors[i].grad = grads[i];
    p.set_wide(&p.tensors[i]);
  }
  if (p.tensors.empty()) return PKT_OK;
  const cudaError_t e = cudaMemcpyAsync(p.d_tensors, p.tensors.data(), sizeof(AdamTensor) * p.tensors.size(), cudaMemcpyHostToDevice, st);
  return e == cudaSuccess ? PKT_OK : cuda_fail(e, "copy AdamW gradients");
}

int pkt_adamw_set_step(pkt_adamw* h, long long step, void* stream) {
  if (!h || step < 0) return pkb::fail(PKT_ERR_ARGS, "bad AdamW step");
  pkb::OnDevice on(h->plan.device);
  return h->plan.set_step(step, static_cast<cudaStream_t>(stream));
}

int pkt_adamw_get_step(pkt_adamw* h, long long* step, void* stream) {
  using namespace pkb;
  if (!h || !step) return fail(PKT_ERR_ARGS, "null argument");
  OnDevice on(h->plan.device);
  AdamState s;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = outside_capture(st, "the AdamW step cannot be read");
  if (rc) return rc;
  cudaError_t e = cudaMemcpyAsync(&s, h->plan.d_state, sizeof(s), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return cuda_fail(e, "read the AdamW step");
  *step = s.step;
  return PKT_OK;
}

}  // extern "C"
