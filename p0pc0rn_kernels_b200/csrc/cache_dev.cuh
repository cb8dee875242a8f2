// The 8-bit key/value cache as the kernels get it.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "cache_plan.h"
#include "sync.cuh"

namespace p0p {

struct CacheP {
  uint8_t* codes; float2* scales; __half* tail;
  const uint32_t* table; const uint32_t* lens; const uint32_t* rows;      // rows NULL: `each` rows per sequence
  uint32_t Hkv, pages, seqs, max_pages, M, each;
  int* status;
};

// two results as fp16: a mean of finite values stays finite, although a code of 127 times a scale that was rounded up, or weights that were, can pass the
// largest fp16.  NaN stays NaN
__device__ __forceinline__ uint32_t cache_result(float a, float b) { uint32_t r; asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a)); return r; }

__device__ __forceinline__ void cache_tell(int* status, int code) { if (code) atomicCAS(status, 0, code); }
// sequence b of the call; one whose numbers make no sense has n = 0 (every block that meets it says so)
__device__ __forceinline__ CacheSeq cache_seq(const CacheP& p, uint32_t b) {
  CacheSeq s;
  const uint32_t r0 = p.rows ? ld_now(p.rows + b) : b * p.each, r1 = p.rows ? ld_now(p.rows + b + 1u) : r0 + p.each;
  cache_tell(p.status, cache_seq_check(r0, r1, ld_now(p.lens + b), p.M, p.max_pages, s));
  return s;
}

}  // namespace p0p
