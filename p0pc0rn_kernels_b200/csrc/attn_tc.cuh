// What the attention kernels on the 5th-generation tensor cores share: a wait without suspension, exponentials.
#pragma once
#include <stdint.h>

#include "sync.cuh"

namespace p0p {

constexpr uint32_t ATC_TILE = 32768u;      // bytes of a tile of 128 rows x 128 fp16

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_spin(uint32_t bar, uint32_t parity, int* status, int code) {
  if (mbar_test(bar, parity)) return true;
  const long long t0 = clock64();
  uint32_t n = 0;
  while (!mbar_test(bar, parity)) {
    if ((++n & 255u) == 0u && clock64() - t0 > WAIT_LIMIT_CYCLES) { if (status) atomicCAS(status, 0, code); return false; }
  }
  return true;
}
#ifndef ATC_EMU
#define ATC_EMU 6          // of every 16 pairs of scores, how many take their exponential on the FMA pipe instead of the MUFU
                           // (with two threads per query row, in long runs; 24 heads x 3600 x 3600 and 32:8 heads x 1000
                           // causal: 0 185.1, 20.95 us; 4 188.2, 20.50; 5 187.6, 20.41; 6 191.1, 20.71; 7 190.8, 20.75; 8 205.5, 22.72.
                           // 6 was the best with one thread per row: 0 193, 4 186, 6 183, 8 207)
#endif

__device__ __forceinline__ float atc_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// 2^t for a pair, without the special-function unit (16 results per clock per SM, the softmax's bound): t = n + f with
// n = floor(t); 2^f by a cubic (least-maximum relative error 8.6e-5, below the half-ulp of the fp16 the result is rounded
// to), then n is added into the exponent field.  (t + 1.5 * 2^23) rounded down holds n in its low mantissa bits; shifted
// left by 23 that is n in the exponent position (the constant's own bits shift out).  The cubic is >= 1, so n >= -126 keeps
// the sum a valid float.
__device__ __forceinline__ float2 atc_ex2_poly2(float2 t) {
  t.x = fmaxf(t.x, -126.0f); t.y = fmaxf(t.y, -126.0f);
  const float2 r = __fadd2_rd(t, make_float2(12582912.0f, 12582912.0f));
  const float2 fl = __fadd2_rn(r, make_float2(-12582912.0f, -12582912.0f));
  const float2 f = __ffma2_rn(fl, make_float2(-1.0f, -1.0f), t);
  float2 q = __ffma2_rn(f, make_float2(0.07706704f, 0.07706704f), make_float2(0.22764499f, 0.22764499f));
  q = __ffma2_rn(q, f, make_float2(0.69511679f, 0.69511679f));
  q = __ffma2_rn(q, f, make_float2(1.0f, 1.0f));
  return make_float2(__int_as_float(__float_as_int(q.x) + (__float_as_int(r.x) << 23)), __int_as_float(__float_as_int(q.y) + (__float_as_int(r.y) << 23)));
}

}  // namespace p0p
