// Attention over the 8-bit cache for few new tokens per sequence (decoding steps): o = softmax(scale q K^T) V per query head, causal,
// with a sliding window and first tokens that stay visible.  K and V go from the cache's codes straight to the tensor cores:
//   a code byte u = code + 128 put into an fp16's low bits IS the subnormal u * 2^-24, one byte permute per pair, so
//   q . k = ks (2^24 (q . u 2^-24) - 128 sum q): the second term is the accumulator's starting value (a product with a constant operand)
//   sum p v = vs (2^24 (sum p u 2^-24) - 128 sum p): the page's scale joins the probability's exponent, w = 2^(score + log2 vs - m), and the
//   sum of the weights as rounded to fp16 comes from a product with ones: it serves the second term and, times 1 / vs, the softmax's sum.
//   The second term is taken off page by page: left to the end, the sums of u grow 128 times the number of keys and their rounding with
//   them (8000 keys in one accumulator: 2e-3 of the result; page by page 2.3e-4, of which 2.1e-4 is the result's own rounding).
// The running maximum m is that of score + log2 vs: weights are at most 1.  Statistics and sums are fp32; the weights' rounding to fp16 (2^-11 each,
// independent from key to key) is what tensor-core products of fp32 sums cost, as in k_attn.cuh.
//
// Work: a unit = one visible page of one kv head for up to 16 query rows (the rows of all heads that share the kv head, query-major; more
// rows are more row blocks).  All units of all sequences in one row are dealt out evenly: to blocks (one per SM), within a block to its 8 warps.  So
// contexts of any mix of lengths fill the machine, and the numbers on the device decide how: nothing but the launch is fixed on the host.
// A warp streams its pages through two 8-KB buffers of its own (K, V) by bulk copies, one page ahead.  An item (all pages of a
// sequence, kv head and row block) that lies within one warp's share is finished there; otherwise partial results (maximum, sum, O)
// are merged in the block, and across blocks by the one that arrives last (a counter per item that crosses blocks; it resets it), in
// order: deterministic, one launch.
// Bound: one pass over the visible codes (HBM).
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "cache_dev.cuh"
#include "k_attn.cuh"

namespace p0p {

struct CacheAttnP {
  CacheP c;
  const __half* Q; __half* O;
  uint32_t Hq, group, ldq, ldo, window, sinks;
  uint32_t max_rows;     // sequences with more query rows per kv head than this are another kernel's
  float scale_log2;      // scale * log2(e)
  float* part;           // [block][2][16][128] unnormalised O, then (maximum, sum) [block][2][16]
  float2* part_ml;
  uint32_t* count;       // [block] arrivals, zero between calls
};

constexpr uint32_t CA_WARPS = 8u, CA_LD = 132u, CA_RING = 2u * CACHE_BLOCK, CA_PART = 16u * CA_LD * 4u;
struct CaEntry { uint64_t i0, i1; uint32_t b, hk, rb, on; };              // a partial result of a warp: its item's units, the item
struct CaShared {
  uint64_t pre[CACHE_MAX_SEQS + 1];                                       // units before each sequence
  CacheSeq seq[CACHE_MAX_SEQS];
  float2 ml[CA_WARPS][2][16];
  CaEntry ent[CA_WARPS * 2];
  uint64_t bars[CA_WARPS][2];
  uint64_t warp_sum[CA_WARPS];
  uint32_t last[2], failed;
};
constexpr uint32_t CA_SMEM = CA_WARPS * (CA_RING + CA_PART) + (uint32_t)sizeof(CaShared) + 128u;
static_assert(CA_SMEM <= 232448u, "shared memory");
static_assert(CA_PART <= CA_RING, "a partial result fits a warp's buffers");

__device__ __forceinline__ uint4 ca_lds(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float ca_lg2(float x) { float y; asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

__global__ void __launch_bounds__(CA_WARPS * 32u, 1) k_cache_attn(const CacheAttnP p) {
  extern __shared__ __align__(128) unsigned char ca_raw[];
  const uint32_t base = (smem_u32(ca_raw) + 127u) & ~127u;
  unsigned char* gbase = ca_raw + (base - smem_u32(ca_raw));
  CaShared& sh = *reinterpret_cast<CaShared*>(gbase + CA_WARPS * (CA_RING + CA_PART));
  const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u, g = lane >> 2, t4 = lane & 3u;
  const uint32_t ring = base + warp * CA_RING;
  const CacheGeo geo{p.c.Hkv, p.group, p.c.seqs, p.window, p.sinks};
  float* const headp = reinterpret_cast<float*>(gbase + CA_WARPS * CA_RING + warp * CA_PART);
  float* const tailp = reinterpret_cast<float*>(gbase + warp * CA_RING);
  const uint32_t bar_k = smem_u32(&sh.bars[warp][0]), bar_v = smem_u32(&sh.bars[warp][1]);
  if (lane == 0u) { mbar_init(bar_k, 1u); mbar_init(bar_v, 1u); }
  if (tid < CA_WARPS * 2u) sh.ent[tid].on = 0u;
  if (tid == 0u) sh.failed = 0u;
  fence_mbar_init();
  grid_dependency_wait();
  grid_launch_dependents();
  // ---- how many units there are, sequence by sequence
  uint64_t U = 0u;
  for (uint32_t b0 = 0; b0 < p.c.seqs; b0 += CA_WARPS * 32u) {
    const uint32_t b = b0 + tid;
    uint64_t c = 0u;
    if (b < p.c.seqs) {
      const CacheSeq s = cache_seq(p.c, b);
      sh.seq[b] = s;
      if (s.n && (uint64_t)s.n * p.group <= p.max_rows) c = cache_units(s, geo);
    }
    uint64_t inc = c;
#pragma unroll
    for (uint32_t o = 1; o < 32u; o <<= 1) { const uint64_t v = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += v; }
    if (lane == 31u) sh.warp_sum[warp] = inc;
    __syncthreads();
    uint64_t before = U;
#pragma unroll
    for (uint32_t w = 0; w < CA_WARPS; w++) { if (w < warp) before += sh.warp_sum[w]; U += sh.warp_sum[w]; }
    if (b < p.c.seqs) { sh.pre[b + 1u] = before + inc; if (b == 0u) sh.pre[0] = 0u; }
    __syncthreads();
  }
  const uint64_t G = U < gridDim.x ? U : gridDim.x;
  if (blockIdx.x >= G) return;
  const uint64_t u0 = deal_first(blockIdx.x, U, G), u1 = deal_first(blockIdx.x + 1u, U, G), here = u1 - u0, W = here < CA_WARPS ? here : CA_WARPS;
  if (warp < W) {
    const uint64_t w0 = u0 + deal_first(warp, here, W), w1 = u0 + deal_first(warp + 1u, here, W);
    CacheCursor cur, nxt;
    cur.seek(geo, sh.pre, sh.seq, w0);
    nxt = cur;
    auto table_at = [&](const CacheCursor& c) { return c.tail() ? 0u : ld_now(p.c.table + (size_t)c.b * p.c.max_pages + c.page()); };
    auto checked = [&](uint32_t page) { if (page < p.c.pages) return page; if (lane == 0u) cache_tell(p.c.status, CACHE_BAD_PAGE); return 0u; };
    auto codes_at = [&](const CacheCursor& c, uint32_t page, uint32_t w) -> const void* {
      return c.tail() ? (const void*)(p.c.tail + (((size_t)c.b * p.c.Hkv + c.hk) * 2u + w) * CACHE_BLOCK) : (const void*)(p.c.codes + (((size_t)page * p.c.Hkv + c.hk) * 2u + w) * CACHE_BLOCK);
    };
    auto fetch = [&](const CacheCursor& c, uint32_t page, uint32_t w) {       // one lane: K (w 0) or V of a page; the tail's takes both buffers
      const uint32_t bytes = c.tail() ? 2u * CACHE_BLOCK : CACHE_BLOCK, bar = w ? bar_v : bar_k;
      mbar_expect_tx(bar, bytes);
      bulk_g2s(ring + (w && !c.tail() ? CACHE_BLOCK : 0u), codes_at(c, page, w), bytes, bar);
    };
    auto scales_at = [&](const CacheCursor& c, uint32_t page) { return c.tail() ? make_float2(1.0f, 1.0f) : ld_now(p.c.scales + (size_t)page * p.c.Hkv + c.hk); };
    uint32_t page = checked(table_at(cur)), nxt_raw = 0u;                  // this unit's page; the next one's as read
    float2 sc = scales_at(cur, page);
    if (lane == 0u) { fetch(cur, page, 0u); if (!cur.tail()) fetch(cur, page, 1u); }
    if (w0 + 1u < w1) { nxt.next(geo, sh.pre, sh.seq); nxt_raw = table_at(nxt); }
    uint32_t ph_k = 0u, ph_v = 0u;
    uint32_t qa[8][4];
    float bias[2] = {0.0f, 0.0f};
    uint32_t pos[2] = {0u, 0u};
    float o[16][4], m[2], l[2];
    bool fresh = true, ok = true;
    uint64_t i0 = 0u;                                                      // the item's first unit
    for (uint64_t u = w0; u < w1; u++) {
      const bool tail = cur.tail(), more = u + 1u < w1;
      const uint32_t kp = cur.page(), rows = cur.s.n * p.group;
      if (fresh) {
        // ---- a new item: this thread's two query rows (rows past the end repeat the last one; they are not stored)
        fresh = false;
        i0 = u - cur.t;
        const uint32_t first = cur.s.L - cur.s.n;
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++) {
          const uint32_t r = min(cur.rb * 16u + h * 8u + g, rows - 1u), i = r / p.group;
          pos[h] = first + i;
          const uint4* q = reinterpret_cast<const uint4*>(p.Q + ((size_t)(cur.hk * p.group + (r - i * p.group)) * p.ldq + cur.s.r0 + i) * 128u + t4 * 16u);
#pragma unroll
          for (uint32_t k = 0; k < 2u; k++) {
            const uint4 a = ld_now(q + k * 8u), c = ld_now(q + k * 8u + 1u);
            qa[k * 4u][h] = a.x; qa[k * 4u][2u + h] = a.y; qa[k * 4u + 1u][h] = a.z; qa[k * 4u + 1u][2u + h] = a.w;
            qa[k * 4u + 2u][h] = c.x; qa[k * 4u + 2u][2u + h] = c.y; qa[k * 4u + 3u][h] = c.z; qa[k * 4u + 3u][2u + h] = c.w;
          }
        }
        float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 8; k++) at_mma(s4, qa[k], 0x80808080u, 0x80808080u);      // -128 * 2^-24 each
        bias[0] = s4[0]; bias[1] = s4[2];
#pragma unroll
        for (int d = 0; d < 16; d++) { o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f; }
        m[0] = m[1] = -INFINITY; l[0] = l[1] = 0.0f;
      }
      // ---- scores of 64 keys
      float s[8][4];
      if (ok && !mbar_wait(bar_k, ph_k, p.c.status, 611)) ok = false;
      ph_k ^= 1u;
      if (!__all_sync(0xffffffffu, ok)) { sh.failed = 1u; break; }
      if (!tail) {
#pragma unroll
        for (uint32_t n = 0; n < 8u; n++) {
          s[n][0] = s[n][1] = bias[0]; s[n][2] = s[n][3] = bias[1];
#pragma unroll
          for (uint32_t k = 0; k < 2u; k++) {
            const uint4 w = ca_lds(ring + n * 1024u + k * 512u + lane * 16u);
            at_mma(s[n], qa[k * 4u], __byte_perm(w.x, 0u, 0x4140), __byte_perm(w.x, 0u, 0x4342));
            at_mma(s[n], qa[k * 4u + 1u], __byte_perm(w.y, 0u, 0x4140), __byte_perm(w.y, 0u, 0x4342));
            at_mma(s[n], qa[k * 4u + 2u], __byte_perm(w.z, 0u, 0x4140), __byte_perm(w.z, 0u, 0x4342));
            at_mma(s[n], qa[k * 4u + 3u], __byte_perm(w.w, 0u, 0x4140), __byte_perm(w.w, 0u, 0x4342));
          }
        }
      } else {
#pragma unroll
        for (uint32_t n = 0; n < 8u; n++) {
          s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
          for (uint32_t k = 0; k < 2u; k++) {
            const uint4 w = ca_lds(ring + n * 2048u + k * 1024u + lane * 32u), x = ca_lds(ring + n * 2048u + k * 1024u + lane * 32u + 16u);
            at_mma(s[n], qa[k * 4u], w.x, w.y);
            at_mma(s[n], qa[k * 4u + 1u], w.z, w.w);
            at_mma(s[n], qa[k * 4u + 2u], x.x, x.y);
            at_mma(s[n], qa[k * 4u + 3u], x.z, x.w);
          }
        }
      }
      __syncwarp();                                                        // the K buffer is read
      uint32_t nxt_page = 0u;
      float2 nxt_sc = make_float2(1.0f, 1.0f);
      if (tail) { if (lane == 0u) fetch(cur, 0u, 1u); }                    // the tail's V, into both buffers
      if (more) {
        nxt_page = checked(nxt_raw);
        if (lane == 0u && !tail && !nxt.tail()) fetch(nxt, nxt_page, 0u);
        nxt_sc = scales_at(nxt, nxt_page);
      }
      CacheCursor aft = nxt;                                                  // the unit after the next: its table entry is asked for now
      uint32_t aft_raw = 0u;
      if (u + 2u < w1) { aft.next(geo, sh.pre, sh.seq); aft_raw = table_at(aft); }
      // ---- masks, maximum, weights
      const float f = p.scale_log2 * sc.x * (tail ? 1.0f : 16777216.0f), lv = tail ? 0.0f : ca_lg2(sc.y), inv_v = tail ? 1.0f : __fdividef(1.0f, sc.y);
      const uint32_t p0 = cur.s.L - cur.s.n, p1 = cur.s.L - 1u;
      float mx[2] = {-INFINITY, -INFINITY};
      if (cache_page_masked(kp, p0, p1, p.window, p.sinks)) {
#pragma unroll
        for (uint32_t n = 0; n < 8u; n++)
#pragma unroll
          for (uint32_t e = 0; e < 4u; e++) {
            const uint32_t key = kp * CACHE_PAGE + 16u * (n >> 1) + 4u * t4 + 2u * (n & 1u) + (e & 1u);
            s[n][e] = cache_key_visible(key, pos[e >> 1], p.window, p.sinks) ? fmaf(s[n][e], f, lv) : -INFINITY;
            mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
          }
      } else {
#pragma unroll
        for (uint32_t n = 0; n < 8u; n++)
#pragma unroll
          for (uint32_t e = 0; e < 4u; e++) { s[n][e] = fmaf(s[n][e], f, lv); mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]); }
      }
#pragma unroll
      for (int h = 0; h < 2; h++) { mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1)); mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2)); }
      if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
        const float n0 = fmaxf(m[0], mx[0]), n1 = fmaxf(m[1], mx[1]);
        const float a0 = n0 == -INFINITY ? 1.0f : at_ex2(m[0] - n0), a1 = n1 == -INFINITY ? 1.0f : at_ex2(m[1] - n1);
        m[0] = n0; m[1] = n1; l[0] *= a0; l[1] *= a1;
#pragma unroll
        for (int d = 0; d < 16; d++) { o[d][0] *= a0; o[d][1] *= a0; o[d][2] *= a1; o[d][3] *= a1; }
      }
      const float e0 = m[0] == -INFINITY ? 0.0f : m[0], e1 = m[1] == -INFINITY ? 0.0f : m[1];
      uint32_t pa[4][4];
      float zp[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (uint32_t j = 0; j < 4u; j++) {
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++) {
          const float* x = s[2u * j + h];
          pa[j][2u * h] = at_pack(at_ex2(x[0] - e0), at_ex2(x[1] - e0));
          pa[j][2u * h + 1u] = at_pack(at_ex2(x[2] - e1), at_ex2(x[3] - e1));
        }
        at_mma(zp, pa[j], 0x3c003c00u, 0x3c003c00u);
      }
      l[0] = fmaf(zp[0], inv_v, l[0]); l[1] = fmaf(zp[2], inv_v, l[1]);
      // (the tail is the last page of its item: from there on O is in real units)
#pragma unroll
      for (int d = 0; d < 16; d++) {
        if (tail) { o[d][0] *= 16777216.0f; o[d][1] *= 16777216.0f; o[d][2] *= 16777216.0f; o[d][3] *= 16777216.0f; }
        else {
          const float c0 = -0x1p-17f * zp[0], c1 = -0x1p-17f * zp[2];      // -128 * 2^-24 each
          const float2 x = __fadd2_rn(make_float2(o[d][0], o[d][1]), make_float2(c0, c0)), y = __fadd2_rn(make_float2(o[d][2], o[d][3]), make_float2(c1, c1));
          o[d][0] = x.x; o[d][1] = x.y; o[d][2] = y.x; o[d][3] = y.y;
        }
      }
      // ---- weights times values
      if (ok && !mbar_wait(bar_v, ph_v, p.c.status, 612)) ok = false;
      ph_v ^= 1u;
      if (!__all_sync(0xffffffffu, ok)) { sh.failed = 1u; break; }
      if (!tail) {
#pragma unroll
        for (uint32_t d = 0; d < 16u; d++) {
          const uint4 w = ca_lds(ring + CACHE_BLOCK + d * 512u + lane * 16u);
          at_mma(o[d], pa[0], __byte_perm(w.x, 0u, 0x4140), __byte_perm(w.x, 0u, 0x4342));
          at_mma(o[d], pa[1], __byte_perm(w.y, 0u, 0x4140), __byte_perm(w.y, 0u, 0x4342));
          at_mma(o[d], pa[2], __byte_perm(w.z, 0u, 0x4140), __byte_perm(w.z, 0u, 0x4342));
          at_mma(o[d], pa[3], __byte_perm(w.w, 0u, 0x4140), __byte_perm(w.w, 0u, 0x4342));
        }
      } else {
        // (behind the sequence's end the tail may hold anything: those values weigh nothing, but 0 * NaN would count)
        const int have = (int)(cur.s.L - kp * CACHE_PAGE) - (int)(4u * t4);
        uint32_t keep[4][2];
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int h = 0; h < 2; h++) { const int r = have - 16 * j - 2 * h; keep[j][h] = r >= 2 ? 0xffffffffu : r == 1 ? 0xffffu : 0u; }
#pragma unroll
        for (uint32_t d = 0; d < 16u; d++) {
          const uint4 w = ca_lds(ring + d * 1024u + lane * 32u), x = ca_lds(ring + d * 1024u + lane * 32u + 16u);
          at_mma(o[d], pa[0], w.x & keep[0][0], w.y & keep[0][1]);
          at_mma(o[d], pa[1], w.z & keep[1][0], w.w & keep[1][1]);
          at_mma(o[d], pa[2], x.x & keep[2][0], x.y & keep[2][1]);
          at_mma(o[d], pa[3], x.z & keep[3][0], x.w & keep[3][1]);
        }
      }
      __syncwarp();                                                        // the V buffer is read
      if (more && lane == 0u) {
        if (tail || nxt.tail()) fetch(nxt, nxt_page, 0u);
        if (!nxt.tail()) fetch(nxt, nxt_page, 1u);
      }
      // ---- the end of the item, or of this warp's share
      const bool done = cur.t + 1u == cur.v.np;
      if (done || !more) {
        fresh = true;
        if (!tail) {
#pragma unroll
          for (int d = 0; d < 16; d++) { o[d][0] *= 16777216.0f; o[d][1] *= 16777216.0f; o[d][2] *= 16777216.0f; o[d][3] *= 16777216.0f; }
        }
        if (done && i0 >= w0) {
          const float inv[2] = {l[0] > 0.0f ? 1.0f / l[0] : l[0], l[1] > 0.0f ? 1.0f / l[1] : l[1]};      // (a row that saw only pages that do not exist: 0)
#pragma unroll
          for (uint32_t h = 0; h < 2u; h++) {
            const uint32_t r = cur.rb * 16u + h * 8u + g, i = r / p.group;
            if (r < rows) {
              __half2* dst = reinterpret_cast<__half2*>(p.O + (size_t)(cur.s.r0 + i) * p.ldo + (cur.hk * p.group + (r - i * p.group)) * 128u + 2u * t4);
#pragma unroll
              for (int d = 0; d < 16; d++) dst[4 * d] = __floats2half2_rn(o[d][2 * h] * inv[h], o[d][2 * h + 1] * inv[h]);
            }
          }
        } else {
          // a share of an item: the warp's first item goes to a place of its own, its last one over its buffers (nothing is in flight then)
          const uint32_t which = i0 < w0 ? 0u : 1u;
          float* dst = which ? tailp : headp;
#pragma unroll
          for (int d = 0; d < 16; d++) {
            *reinterpret_cast<float2*>(dst + g * CA_LD + d * 8 + 2 * t4) = make_float2(o[d][0], o[d][1]);
            *reinterpret_cast<float2*>(dst + (g + 8u) * CA_LD + d * 8 + 2 * t4) = make_float2(o[d][2], o[d][3]);
          }
          if (t4 == 0u) { sh.ml[warp][which][g] = make_float2(m[0], l[0]); sh.ml[warp][which][g + 8u] = make_float2(m[1], l[1]); }
          if (lane == 0u) { CaEntry& e = sh.ent[warp * 2u + which]; e.i0 = i0; e.i1 = i0 + cur.v.np; e.b = cur.b; e.hk = cur.hk; e.rb = cur.rb; e.on = 1u; }
        }
      }
      cur = nxt; nxt = aft; page = nxt_page; sc = nxt_sc; nxt_raw = aft_raw;
    }
    (void)page;
  }
  __syncthreads();
  // ---- the warps' shares of one item, merged in order; an item that is all here is finished, another one's partial result goes to memory
  auto store = [&](uint32_t b, uint32_t hk, uint32_t rb, uint32_t r, float4 v) {      // columns 4 lane .. of row r of the row block
    const CacheSeq q = sh.seq[b];
    const uint32_t x = rb * 16u + r, i = x / p.group;
    __half2* d = reinterpret_cast<__half2*>(p.O + (size_t)(q.r0 + i) * p.ldo + (hk * p.group + (x - i * p.group)) * 128u + 4u * lane);
    d[0] = __floats2half2_rn(v.x, v.y); d[1] = __floats2half2_rn(v.z, v.w);
  };
  auto rows_of = [&](const CaEntry& e) { return min(16u, sh.seq[e.b].n * p.group - e.rb * 16u); };
  CaEntry open[2];                                                         // items that other blocks share: the one that began before, the one that goes on
  open[0].on = open[1].on = 0u;
  for (uint32_t e0 = 0; e0 < CA_WARPS * 2u;) {
    if (!sh.ent[e0].on) { e0++; continue; }
    const CaEntry it = sh.ent[e0];
    uint32_t e1 = e0 + 1u;
    while (e1 < CA_WARPS * 2u && (!sh.ent[e1].on || sh.ent[e1].i0 == it.i0)) e1++;
    const bool whole = it.i0 >= u0 && it.i1 <= u1;
    const uint32_t slot = it.i0 < u0 ? 0u : 1u, n = rows_of(it);
    if (!whole) open[slot] = it;
    for (uint32_t r = warp; r < n; r += CA_WARPS) {
      float M = -INFINITY, L = 0.0f;
      for (uint32_t e = e0; e < e1; e++) if (sh.ent[e].on) M = fmaxf(M, sh.ml[e >> 1][e & 1u][r].x);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (uint32_t e = e0; e < e1; e++) {
        if (!sh.ent[e].on) continue;
        const float2 ml = sh.ml[e >> 1][e & 1u][r];
        const float f = ml.x == -INFINITY ? 0.0f : at_ex2(ml.x - M);
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(gbase + ((e & 1u) ? (e >> 1) * CA_RING : CA_WARPS * CA_RING + (e >> 1) * CA_PART)) + r * CA_LD + 4u * lane);
        L += f * ml.y;
        acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
      }
      if (whole) { const float inv = L > 0.0f ? 1.0f / L : L; store(it.b, it.hk, it.rb, r, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv)); }
      else {
        const size_t at = ((size_t)blockIdx.x * 2u + slot) * 16u + r;
        *reinterpret_cast<float4*>(p.part + at * 128u + 4u * lane) = acc;
        if (lane == 0u) p.part_ml[at] = make_float2(M, L);
      }
    }
    e0 = e1;
  }
  if (sh.failed) {                                                         // a wait ran out: the arrivals still have to be told, or the counters would not return to zero
    auto shared = [&](uint64_t u, uint32_t slot) {
      CacheCursor x;
      x.seek(geo, sh.pre, sh.seq, u);
      CaEntry e;
      e.i0 = u - x.t; e.i1 = e.i0 + x.v.np; e.b = x.b; e.hk = x.hk; e.rb = x.rb;
      e.on = (e.i0 < u0 || e.i1 > u1) && slot == (e.i0 < u0 ? 0u : 1u) ? 1u : 0u;
      open[slot] = e;
    };
    shared(u0, 0u); shared(u1 - 1u, 1u);
  }
  if (!open[0].on && !open[1].on) return;
  // ---- items that cross blocks: the last of their blocks merges them, in block order
  __threadfence();
  __syncthreads();
  if (tid < 2u) {
    uint32_t mine = 0u;
    const CaEntry it = open[tid];
    if (it.on) {
      const uint64_t c0 = deal_owner(it.i0, U, G), c1 = deal_owner(it.i1 - 1u, U, G);
      mine = atomicAdd(p.count + c0, 1u) == (uint32_t)(c1 - c0) ? 1u : 0u;
      if (mine) p.count[c0] = 0u;
    }
    sh.last[tid] = mine;
  }
  __syncthreads();
  __threadfence();
  for (uint32_t k = 0; k < 2u; k++) {
    if (!sh.last[k]) continue;
    const CaEntry it = open[k];
    const uint32_t c0 = (uint32_t)deal_owner(it.i0, U, G), c1 = (uint32_t)deal_owner(it.i1 - 1u, U, G), n = rows_of(it);
    auto at = [&](uint32_t c, uint32_t r) { return ((size_t)c * 2u + (c == c0 ? 1u : 0u)) * 16u + r; };      // (in the item's first block it is the item that goes on)
    for (uint32_t r = warp; r < n; r += CA_WARPS) {
      float M = -INFINITY;
      for (uint32_t c = c0 + lane; c <= c1; c += 32u) M = fmaxf(M, __ldcg(&p.part_ml[at(c, r)]).x);
#pragma unroll
      for (uint32_t x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float L = 0.0f;
      for (uint32_t b = c0; b <= c1; b += 8u) {
        float4 v[8]; float2 ml[8];
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) { const size_t x = at(min(b + i, c1), r); v[i] = __ldcg(reinterpret_cast<const float4*>(p.part + x * 128u) + lane); ml[i] = __ldcg(&p.part_ml[x]); }
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) {
          const float f = b + i <= c1 && ml[i].x != -INFINITY ? at_ex2(ml[i].x - M) : 0.0f;
          L += f * ml[i].y;
          acc.x += f * v[i].x; acc.y += f * v[i].y; acc.z += f * v[i].z; acc.w += f * v[i].w;
        }
      }
      const float inv = L > 0.0f ? 1.0f / L : L;
      store(it.b, it.hk, it.rb, r, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    }
  }
}

}  // namespace p0p
