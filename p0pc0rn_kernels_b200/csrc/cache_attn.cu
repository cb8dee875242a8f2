// p0p_cache_attention: host entry.
#include <algorithm>
#include <cmath>

#include "cache_host.h"
#include "device_once.h"
#include "k_cache_attn.cuh"
#include "k_cache_attn_tc.cuh"
#include "tmap.h"

using namespace p0p;

namespace {

constexpr char OP[] = "cacheAttention";
// Query rows per kv head up to which a sequence is the split-key kernel's.  Its time grows with every 16 rows, the tensor-memory kernel's hardly up to
// 256, but that one has the longer pipeline.  Measured, split keys / tensor memory, us, 8 kv heads:
//   8 sequences of 16000:  32 rows 87 / 114, 48 rows 127 / 114, 64 rows 164 / 117      64 of 4000: 32 rows 176 / 221, 48 rows 253 / 251, 64 rows 331 / 246
//   1 sequence of 500:     96 rows 13 / 22, 128 rows 14 / 22      of 4000: 96 rows 18 / 25, 128 rows 21 / 24      of 32000: 48 rows 38 / 48, 64 rows 50 / 48, 96 rows 63 / 48
// With few sequences and heads, whose contexts hardly fill the machine, the border lies higher.  The host does not know the lengths, so both borders are a
// compromise: at 33 to 48 rows (three blocks of 16) the split-key kernel is the slower one over long contexts (above; with 4 heads 86 / 68) and the faster one
// over shorter ones (8 sequences of 4000: 41 / 43, with 4 heads 28 / 30; of 500 with 4 heads 11 / 19); one sequence of 32000 would be better off with the
// other kernel from 64 rows on, one of 500 at no size up to 256.
inline uint32_t split_rows(uint32_t seqs, uint32_t Hkv) { return (uint64_t)seqs * Hkv <= 16u ? 96u : 48u; }

int run_split(p0p_ctx* c, CacheAttnP& p, uint32_t G) {
  static DeviceOnce once;
  int rc = once.run(c->device, [&] { return (int)cudaFuncSetAttribute(k_cache_attn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)CA_SMEM); });
  if (rc) return cuda_fail(c, (cudaError_t)rc, "cacheAttention kernel attribute");
  const uint64_t slabs = (uint64_t)G * 2u * 16u;
  p.part = reinterpret_cast<float*>(c->scratch.ptr); p.part_ml = reinterpret_cast<float2*>((char*)c->scratch.ptr + slabs * 512u); p.count = c->counters;
  const cudaError_t e = launch_chained(k_cache_attn, dim3(G), dim3(CA_WARPS * 32u), CA_SMEM, c->stream, p);
  if (e != cudaSuccess) return cuda_fail(c, e, "cacheAttention launch");
  c->launches += 1;
  return 0;
}
constexpr uint64_t split_scratch(uint64_t G) { return G * 2u * 16u * (512u + 8u); }
constexpr uint64_t tc_scratch(uint64_t G) { return G * 2u * 256u * (512u + 2u * 8u) + G * sizeof(CacheTcDesc); }

int run_tc(p0p_ctx* c, const CacheAttnP& a, uint32_t G, uint32_t min_rows) {
  static DeviceOnce once;
  int rc = once.run(c->device, [&] {
    // the registers that the softmax threads take are those that the others give up: the kernel has to start with all of them
    cudaFuncAttributes at{};
    cudaError_t e = cudaFuncGetAttributes(&at, k_cache_attn_tc);
    if (e == cudaSuccess && at.numRegs * (int)(CTC_THREADS / 32u) < CTC_REGS) e = cudaErrorLaunchOutOfResources;
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_cache_attn_tc, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)CTC_SMEM);
    return (int)e;
  });
  if (rc) return cuda_fail(c, (cudaError_t)rc, "cacheAttention kernel attribute");
  tmap_encode_fn f = tmap_encoder();
  if (!f) return fail(c, -12, "cacheAttention: the driver offers no tensor-map encoder");
  CacheTcP p{};
  p.c = a.c; p.O = a.O; p.ldo = a.ldo; p.scale_log2 = a.scale_log2;
  p.geo = CacheTcGeo{a.c.Hkv, a.group, a.c.seqs, a.window, a.sinks, 128u / a.group, min_rows};
  p.part = reinterpret_cast<float4*>(c->scratch.ptr);
  p.part_ml = reinterpret_cast<float2*>((char*)c->scratch.ptr + (uint64_t)G * 2u * 256u * 512u);
  p.count = c->counters;
  // Few items are cut into many shares each, which a kernel of its own adds up faster than the block that arrives last with one; where there are none, that launch costs
  // 2 us.  Measured, within / by a second kernel, 8 kv heads: 1 sequence of 32000 (18 shares an item) 63 / 48 us, of 4000 29 / 24, of 500 (two shares)
  // 16 / 18; 8 sequences (two or three) of 16000 115 / 113, of 4000 42.5 / 41, of 500 16.7 / 18.8.  With row offsets this counts all sequences and all rows.
  const bool merge = (uint64_t)a.c.Hkv * std::max<uint64_t>(a.c.seqs, (a.c.M - 1u) / (2u * p.geo.qpt) + 1u) * 4u < G;
  p.desc = merge ? reinterpret_cast<CacheTcDesc*>((char*)c->scratch.ptr + (uint64_t)G * 2u * 256u * (512u + 2u * 8u)) : nullptr;
  // Q [Hq][ldq][128] as {64 of d, the heads of a group, qpt queries, a kv head}: a tile's rows query by query
  CUtensorMap mq;
  const cuuint64_t dims[4] = {128u, a.group, a.c.M, a.c.Hkv}, strides[3] = {(cuuint64_t)a.ldq * 256u, 256u, (cuuint64_t)a.ldq * a.group * 256u};
  const cuuint32_t box[4] = {64u, a.group, p.geo.qpt, 1u}, el[4] = {1u, 1u, 1u, 1u};
  if (f(&mq, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half*>(a.Q), dims, strides, box, el, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return fail(c, -12, "cacheAttention: a tensor map could not be encoded");
  cudaError_t e = launch_chained(k_cache_attn_tc, dim3(G), dim3(CTC_THREADS), CTC_SMEM, c->stream, p, mq);
  if (e == cudaSuccess && merge) e = launch_chained(k_cache_merge, dim3(G, 8u), dim3(256), 0, c->stream, CacheMergeP{p.part, p.part_ml, p.desc, p.O, p.ldo, a.group, p.geo.qpt});
  if (e != cudaSuccess) return cuda_fail(c, e, "cacheAttention launch");
  c->launches += merge ? 2 : 1;
  return 0;
}

}  // namespace

extern "C" int p0p_cache_attention(p0p_ctx* c, const p0p_cache_attn_args* a) {
  const char* op = OP;
  P0P_ALIVE(c);
  if (!a || a->struct_size < sizeof(p0p_cache_attn_args)) return fail(c, -1, "cacheAttention: bad argument block");
  CacheAttnP p{};
  if (int rc = cache_bind(c, op, a->cache, a->M, a->rows, a->rows_off, p.c)) return rc;
  const uint32_t M = a->M, Hq = a->Hq, ldq = a->ldq ? a->ldq : M, ldo = a->ldo ? a->ldo : Hq * 128u;
  if (!Hq || Hq > 65535u || Hq % p.c.Hkv) return fail(c, -3, "cacheAttention: Hq must be a multiple of Hkv, at most 65535");
  if (a->kernel != 0u && a->kernel != P0P_K_CACHE_SPLIT && a->kernel != P0P_K_CACHE_TMEM) return fail(c, -2, "cacheAttention: unknown kernel selector %u", a->kernel);
  if (!(a->scale >= 0.0f) || a->scale > 0x1p64f) return fail(c, -2, "cacheAttention: the scale must be finite and not negative, at most 2^64");
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
  // (a product of 128 pairs is below 2^39: scores stay finite, and a scale below 2^-80 leaves nothing of them.  It is kept above 0: a hidden key's -infinity times it)
  p.scale_log2 = std::max(a->scale > 0.0f ? a->scale : 1.0f / std::sqrt(128.0f), 0x1p-80f) * 1.4426950408889634f;
  DeviceGuard g(c->device);
  const uint32_t G = std::min<uint32_t>((uint32_t)c->prop.multiProcessorCount, c->n_counters / 16u);
  // Which kernel a sequence is for depends on its number of new tokens.  Without row offsets the host knows it; with them it knows the most any
  // sequence has, if the caller says so, and where that is many, both kernels run, each for its sequences.
  const uint64_t most = (uint64_t)p.group * (p.c.rows ? (a->max_new ? std::min(a->max_new, M) : M) : p.c.each);
  const uint32_t border = split_rows(p.c.seqs, p.c.Hkv);
  const bool fits = p.group <= 128u, forced = a->kernel != 0u;
  if (a->kernel == P0P_K_CACHE_TMEM && !fits) return fail(c, -2, "cacheAttention: more than 128 heads per kv head are not for the tensor-memory kernel");
  const bool tc = forced ? a->kernel == P0P_K_CACHE_TMEM : fits && most > border, split = forced ? !tc : !tc || p.c.rows;
  if (int rc = ensure_scratch(c, std::max(split ? split_scratch(G) : 0u, tc ? tc_scratch(G) : 0u))) return rc;
  if (split) {
    p.max_rows = tc ? border : 0xffffffffu;
    if (int rc = run_split(c, p, G)) return rc;
  }
  if (tc) {
    if (int rc = run_tc(c, p, G, split ? border : 0u)) return rc;
  }
  c->last_kernel = tc ? (split ? P0P_K_CACHE_BOTH : P0P_K_CACHE_TMEM) : P0P_K_CACHE_SPLIT;
  const uint32_t plan[8] = {G};
  std::copy(plan, plan + 8, c->last_plan);
  return 0;
}
