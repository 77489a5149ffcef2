// Stored bytes to f16 pairs, exactly, in registers.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "gorgon_b200.h"

namespace gorgon {

// Byte e of a and byte f of b (numbered 4 .. 7, or 0 .. 3 for a again) as a
// pair of f16, exactly.
//   int8: 2^10 + (byte + 128) is the f16 0x6400 | (byte ^ 0x80); less 1152.
//   e4m3: the hardware's conversion.
template <int ST, int E, int F>
__device__ __forceinline__ uint32_t widen(uint32_t a, uint32_t b) {
  if constexpr (ST == GORGON_KV_INT8) {
    const uint32_t t = __byte_perm(a, b, E | (E << 4) | (F << 8) | (F << 12));
    const uint32_t x = (t & 0x00ff00ffu) ^ 0x64806480u;
    const uint32_t f = 0x64806480u;  // 1152
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&f));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const uint16_t t = static_cast<uint16_t>(__byte_perm(a, b, E | (F << 4)));
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(t));
    return r;
  }
}

// The four bytes of a word as two pairs.
template <int ST>
__device__ __forceinline__ void widen_word(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (ST == GORGON_KV_INT8) {
    const uint32_t u = w ^ 0x80808080u, f = 0x64806480u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&f));
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&f));
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(static_cast<uint16_t>(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(static_cast<uint16_t>(w >> 16)));
  }
}

// A stored byte's number.
template <int ST>
__device__ __forceinline__ float byte_value(uint8_t x) {
  if constexpr (ST == GORGON_KV_INT8) return static_cast<float>(static_cast<int8_t>(x));
  __nv_fp8_e4m3 f;
  f.__x = x;
  return static_cast<float>(f);
}

}  // namespace gorgon
