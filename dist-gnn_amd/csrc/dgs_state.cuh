// dgs_state.cuh -- device helpers of the 4-bit state cache (layout: dgs_ops.h StateView).
#pragma once

#include "context.h"
#include "dgs_common.h"
#include "dgs_guard.cuh"
#include "dgs_ops.h"

namespace dgs {

typedef unsigned int su32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float bf16_bits(uint32_t hi) { return __uint_as_float(hi); }
__device__ __forceinline__ float scale_of(uint32_t m) { return __uint_as_float(m << 16); }
__device__ __forceinline__ float base_of(uint32_t m) { return __uint_as_float(m & 0xffff0000u); }

// The eight codes of a word as floats, in channel order.  (Byte i of a word as a float is one
// instruction; written in C it becomes a field extraction and a conversion.)
__device__ __forceinline__ void codes8(uint32_t w, float (&c)[8]) {
  const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
  asm("v_cvt_f32_ubyte0_e32 %0, %1" : "=v"(c[0]) : "v"(lo));
  asm("v_cvt_f32_ubyte0_e32 %0, %1" : "=v"(c[1]) : "v"(hi));
  asm("v_cvt_f32_ubyte1_e32 %0, %1" : "=v"(c[2]) : "v"(lo));
  asm("v_cvt_f32_ubyte1_e32 %0, %1" : "=v"(c[3]) : "v"(hi));
  asm("v_cvt_f32_ubyte2_e32 %0, %1" : "=v"(c[4]) : "v"(lo));
  asm("v_cvt_f32_ubyte2_e32 %0, %1" : "=v"(c[5]) : "v"(hi));
  asm("v_cvt_f32_ubyte3_e32 %0, %1" : "=v"(c[6]) : "v"(lo));
  asm("v_cvt_f32_ubyte3_e32 %0, %1" : "=v"(c[7]) : "v"(hi));
}

// Eight consecutive values of a row (16-byte aligned) <-> floats.
template <int TYPE>
__device__ __forceinline__ void load8(const void *p, int64_t elem, float (&x)[8]) {
  if constexpr (TYPE == kStateF32) {
    const su32x4 a = ((const su32x4 *)((const float *)p + elem))[0];
    const su32x4 b = ((const su32x4 *)((const float *)p + elem))[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = __uint_as_float(a[i]);
      x[4 + i] = __uint_as_float(b[i]);
    }
  } else {
    const su32x4 a = *(const su32x4 *)((const uint16_t *)p + elem);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == kStateBF16) {
        x[2 * i] = __uint_as_float(a[i] << 16);
        x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
      } else {
        union {
          uint32_t u;
          _Float16 h[2];
        } v{a[i]};
        x[2 * i] = (float)v.h[0];
        x[2 * i + 1] = (float)v.h[1];
      }
    }
  }
}
template <int TYPE>
__device__ __forceinline__ void store8(void *p, int64_t elem, const float (&x)[8]) {
  if constexpr (TYPE == kStateF32) {
    su32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = __float_as_uint(x[i]);
      b[i] = __float_as_uint(x[4 + i]);
    }
    ((su32x4 *)((float *)p + elem))[0] = a;
    ((su32x4 *)((float *)p + elem))[1] = b;
  } else {
    su32x4 a;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == kStateBF16) {
        union {
          __bf16 h[2];
          uint32_t u;
        } v;
        v.h[0] = (__bf16)x[2 * i];  // round to nearest even
        v.h[1] = (__bf16)x[2 * i + 1];
        a[i] = v.u;
      } else {
        union {
          _Float16 h[2];
          uint32_t u;
        } v;
        v.h[0] = (_Float16)x[2 * i];
        v.h[1] = (_Float16)x[2 * i + 1];
        a[i] = v.u;
      }
    }
    *(su32x4 *)((uint16_t *)p + elem) = a;
  }
}

// Where a state-cache launch reports ids and lengths outside their bounds.
struct StateGuard {
  int64_t *err = nullptr;
  int64_t tag = 0;
};
inline StateGuard state_guard() {
  StateGuard g;
  g.err = async_err_dev();
  g.tag = (int64_t)async_err_next_state_tag();
  return g;
}

}  // namespace dgs
