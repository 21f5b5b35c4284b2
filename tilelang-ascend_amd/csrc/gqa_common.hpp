// Device helpers of the grouped-head attention kernels: LDS reads, waits, 16x16x32 products.
#pragma once
#include "common.hpp"

namespace dsa {

typedef __attribute__((address_space(3))) void gqa_lds_void;
typedef const __attribute__((address_space(1))) void gqa_gbl_void;

__device__ __forceinline__ uint32_t gqa_lds_u32(const void* p) {
  return (uint32_t)(uintptr_t)(const gqa_lds_void*)p;
}

// LDS reads as inline asm: through the builtins the compiler would wait for
// every outstanding DMA before each read.  Completion is waited for explicitly.
template <int kOff>
__device__ __forceinline__ void gqa_b128(u32x4& out, uint32_t addr) {
  __asm__ __volatile__("ds_read_b128 %0, %1 offset:%2" : "=v"(out) : "v"(addr), "i"(kOff));
}
template <int kOff>
__device__ __forceinline__ void gqa_tr(u32x2& out, uint32_t addr) {
  __asm__ __volatile__("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(out) : "v"(addr), "i"(kOff));
}
template <int N, typename V>
__device__ __forceinline__ void gqa_lgkm_wait(V (&v)[N]) {
  // All LDS operations retired; the values pass through the asm so that no use
  // is scheduled above the wait.
#pragma unroll
  for (int i = 0; i < N; ++i) __asm__ __volatile__("" : "+v"(v[i]));
  __asm__ __volatile__("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) __asm__ __volatile__("" : "+v"(v[i]));
}

// s_waitcnt with only vmcnt constrained.
template <int N>
__device__ __forceinline__ void gqa_wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

template <bool kF16>
__device__ __forceinline__ f32x4 gqa_mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                   0, 0, 0);
}

template <bool kF16>
__device__ __forceinline__ uint32_t gqa_pack(float lo, float hi) {
  if constexpr (kF16) {
    const _Float16 a = (_Float16)lo, b = (_Float16)hi;
    return (uint32_t)__builtin_bit_cast(uint16_t, a) | ((uint32_t)__builtin_bit_cast(uint16_t, b) << 16);
  } else {
    return pack_bf16x2(lo, hi);
  }
}

}  // namespace dsa
