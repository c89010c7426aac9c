// Device helpers of the stand-alone operators: typed vector loads and stores, bulk
// copies and bounded waits, block-scaled 8-bit floats.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/pk/detail/ptx.cuh"
#include "../../include/pkt_b200.h"

namespace pkb {

struct bf16_t {
  uint16_t bits;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return __uint_as_float(uint32_t(v.bits) << 16); }
__device__ __forceinline__ void from_f32(float v, float* out) { *out = v; }
// results are rounded to the tensor's type once, at the store
__device__ __forceinline__ void from_f32(float v, bf16_t* out) { out->bits = f32_to_bf16_rn(v); }

// Two fp32 values in one 64-bit register: one instruction for two results, each
// rounded as by itself.
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
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float sum_of(uint64_t v) {
  const float2 f = unpair(v);
  return f.x + f.y;
}

// VEC consecutive elements as raw words: one load of up to 16 bytes each.
template <typename T, int VEC>
struct Raw {
  static constexpr int kBytes = VEC * int(sizeof(T));
  static constexpr int kWords = (kBytes + 3) / 4;
  uint32_t w[kWords];

  // One aligned access (the callers' rule), or zeros.
  __device__ __forceinline__ void load(const T* p, bool in) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
    if (!in) return;
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else {
      static_assert(kBytes == 8, "2, 4 or 8 words");
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    }
  }
  __device__ __forceinline__ void set(int i, float v) { w[i * int(sizeof(T)) / 4] = __float_as_uint(v); }
  __device__ __forceinline__ void set(int i, bf16_t v) { w[i >> 1] |= uint32_t(v.bits) << (16 * (i & 1)); }
  // elements 2 i and 2 i + 1
  __device__ __forceinline__ uint64_t get2(int i) const { return pair_of(get(2 * i), get(2 * i + 1)); }
  __device__ __forceinline__ float get(int i) const {
    if (sizeof(T) == 4) return __uint_as_float(w[i]);
    return (i & 1) ? bf16_hi(w[i >> 1]) : bf16_lo(w[i >> 1]);
  }
};

// Stores VEC values to p, as one aligned access.
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  constexpr int kBytes = VEC * int(sizeof(T));
  static_assert(kBytes == 8 || kBytes == 16, "one access");
  uint32_t w[kBytes / 4];
#pragma unroll
  for (int i = 0; i < kBytes / 4; ++i)
    w[i] = sizeof(T) == 4 ? __float_as_uint(v[i % VEC]) : pack_bf16x2(v[(2 * i) % VEC], v[(2 * i + 1) % VEC]);
  if constexpr (kBytes == 16)
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}

template <typename T, int VEC>
__device__ __forceinline__ void store_pairs(T* p, const uint64_t (&v)[VEC / 2]) {
  constexpr int kBytes = VEC * int(sizeof(T));
  static_assert(kBytes == 16, "one access");
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) {
    const float2 f = unpair(v[i]);
    if constexpr (sizeof(T) == 2)
      w[i] = pack_bf16x2(f.x, f.y);
    else
      w[2 * i] = __float_as_uint(f.x), w[2 * i + 1] = __float_as_uint(f.y);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// ---------------------------------------------------------------- bulk copies and bounded waits
// Waits until the phase of `parity` has completed; false when it has not after 2 s
// (the timer is only looked at every 1024 tries). One block of assembly: the
// compiler's own form of the loop kept the lanes apart (BSSY / BSYNC around each try)
// and cost hot loops a third of their instructions. No suspend-time hint: it turns a
// failed try into a sleep.
__device__ __forceinline__ bool try_phase(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .u32 n, m;\n .reg .u64 t, t0;\n"
      " mov.u32 n, 0;\n mov.u64 t0, 0;\n"
      "AGAIN:\n"
      " mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n"
      " @p bra DONE;\n"
      " add.u32 n, n, 1;\n"
      " and.b32 m, n, 1023;\n"
      " setp.ne.u32 q, m, 0;\n"
      " @q bra AGAIN;\n"
      " mov.u64 t, %%globaltimer;\n"
      " setp.eq.u64 q, t0, 0;\n"
      " @q mov.u64 t0, t;\n"
      " sub.u64 t, t, t0;\n"
      " setp.lt.u64 q, t, 2000000000;\n"
      " @q bra AGAIN;\n"
      "DONE:\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// The same for a converged warp (one answer for all lanes); a timeout is recorded.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, int* status) {
  if (__all_sync(0xffffffffu, try_phase(bar, parity))) return true;
  *reinterpret_cast<volatile int*>(status) = PKT_DEV_TIMEOUT_PIPE;
  return false;
}
// `bytes` (a multiple of 16, both addresses 16-byte aligned) global -> shared,
// counted on `bar`.
__device__ __forceinline__ void bulk_load(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(to)), "l"(from),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void grid_dependents_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---------------------------------------------------------------- block-scaled 8-bit floats
// Magnitudes are compared as unsigned bits of |x|: the order of finite values,
// infinities above them and NaN above those, so a block that holds one says so
// in its scale.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

constexpr int kScaleBlock = 128;  // values of one 8-bit block along the contiguous dimension
// A block whose largest magnitude is below 2^-100 is held as zeros with scale 0:
// from there on, largest value / magnitude stays far from fp32 overflow.
constexpr float kScaleTiny = 7.888609052210118e-31f;

// Factor and scale of a block from its largest magnitude: q = rn(x * factor), x ~ q * scale.
__device__ __forceinline__ void block_scale(uint32_t amax_bits, float most, float* factor, float* scale) {
  const float big = __uint_as_float(amax_bits);
  const bool none = big < kScaleTiny;
  *factor = none ? 0.f : __fdiv_rn(most, big);
  *scale = none ? 0.f : __fdiv_rn(big, most);
}

// Two values to e4m3 / e5m2 (round to nearest even, out of range to the largest
// finite value, NaN stays NaN); the first in the low byte.
template <bool E5M2>
__device__ __forceinline__ uint32_t pack_fp8x2(float lo, float hi) {
  uint16_t r;
  if (E5M2)
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool E5M2>
__device__ __forceinline__ uint32_t pack_fp8x4(float a, float b, float c, float d) {
  return pack_fp8x2<E5M2>(a, b) | (pack_fp8x2<E5M2>(c, d) << 16);
}
// Two e4m3 values to fp32 (exact).
__device__ __forceinline__ float2 unpack_e4m3x2(uint16_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(v));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

}  // namespace pkb
