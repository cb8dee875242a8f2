// p0p_cache_attention: host entry.
#include <algorithm>
#include <cmath>

#include "cache_host.h"
#include "device_once.h"
#include "k_cache_attn.cuh"

using namespace p0p;

extern "C" int p0p_cache_attention(p0p_ctx* c, const p0p_cache_attn_args* a) {
  static const char* op = "cacheAttention";
  P0P_ALIVE(c);
  if (!a || a->struct_size < sizeof(p0p_cache_attn_args)) return fail(c, -1, "cacheAttention: bad argument block");
  CacheAttnP p{};
  if (int rc = cache_bind(c, op, a->cache, a->M, a->rows, a->rows_off, p.c)) return rc;
  const uint32_t M = a->M, Hq = a->Hq, ldq = a->ldq ? a->ldq : M, ldo = a->ldo ? a->ldo : Hq * 128u;
  if (!Hq || Hq > 65535u || Hq % p.c.Hkv) return fail(c, -3, "cacheAttention: Hq must be a multiple of Hkv, at most 65535");
  if (a->kernel != 0u && a->kernel != P0P_K_CACHE_SPLIT) return fail(c, -2, "cacheAttention: unknown kernel selector %u", a->kernel);
  if (std::isnan(a->scale) || std::isinf(a->scale)) return fail(c, -2, "cacheAttention: the scale must be finite");
  if (!M) return 0;
  __half* q;
  if (int rc = cache_heads(c, op, "q", a->q, a->q_off, Hq, M, ldq, q)) return rc;
  if (!cache_live(c, a->o)) return fail(c, -4, "cacheAttention: missing binding (o)");
  if ((a->o_off & 3u) || (ldo & 1u) || ldo < Hq * 128u) return fail(c, -5, "cacheAttention: o.off must be a multiple of 4 bytes and o.ld even and at least Hq * 128");
  const uint64_t os = ((uint64_t)(M - 1u) * ldo + (uint64_t)Hq * 128u) * 2u;
  if (cache_room(c, a->o, a->o_off) < os) return fail(c, -7, "cacheAttention: o needs %llu bytes", (unsigned long long)os);
  p.Q = q; p.O = cache_at<__half>(a->o, a->o_off);
  if (reinterpret_cast<uintptr_t>(p.O) & 3u) return fail(c, -5, "cacheAttention: o must lie at a multiple of 4 bytes");
  p.Hq = Hq; p.group = Hq / p.c.Hkv; p.ldq = ldq; p.ldo = ldo; p.window = a->window; p.sinks = a->window ? a->sinks : 0u;
  if ((uint64_t)M * p.group > 0x7fffffffu) return fail(c, -5, "cacheAttention: too many rows for one call");
  p.scale_log2 = (a->scale > 0.0f ? a->scale : 1.0f / std::sqrt(128.0f)) * 1.4426950408889634f;
  p.max_rows = 0xffffffffu;
  DeviceGuard g(c->device);
  const uint32_t G = std::min<uint32_t>((uint32_t)c->prop.multiProcessorCount, c->n_counters);
  static DeviceOnce once;
  int rc = once.run(c->device, [&] { return (int)cudaFuncSetAttribute(k_cache_attn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)CA_SMEM); });
  if (rc) return cuda_fail(c, (cudaError_t)rc, "cacheAttention kernel attribute");
  const uint64_t slabs = (uint64_t)G * 2u * 16u;
  if (int r = ensure_scratch(c, slabs * (512u + 8u))) return r;
  p.part = reinterpret_cast<float*>(c->scratch.ptr); p.part_ml = reinterpret_cast<float2*>((char*)c->scratch.ptr + slabs * 512u); p.count = c->counters;
  cudaError_t e = launch_chained(k_cache_attn, dim3(G), dim3(CA_WARPS * 32u), CA_SMEM, c->stream, p);
  if (e != cudaSuccess) return cuda_fail(c, e, "cacheAttention launch");
  c->launches += 1;
  c->last_kernel = P0P_K_CACHE_SPLIT;
  const uint32_t plan[8] = {G};
  std::copy(plan, plan + 8, c->last_plan);
  return 0;
}
