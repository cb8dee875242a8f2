// Attention over the 8-bit cache for few new tokens per sequence (decoding steps): o = softmax(scale q K^T) V per query head, causal,
// with a sliding window and first tokens that stay visible.  K and V go from the cache's codes straight to the tensor cores:
//   a code byte u = code + 128 put into an fp16's low bits IS the subnormal u * 2^-24, one byte permute per pair, so
//   q . k = ks (2^24 (q . u 2^-24) - 128 sum q): the second term is the accumulator's starting value (a product with a constant operand)
//   sum p v = vs (2^24 (sum p u 2^-24) - 128 sum p): the page's scale joins the probability's exponent, w = 2^(score + log2 vs - m).  The second
//   term takes the weights as rounded to fp16, summed by a product with ones.  The softmax's sum adds up w / vs from the weights before their
//   rounding: where a page's scale is 2^20 times another's, the other's weights are subnormals or 0, which its own small values bear but the sum would not.
//   The second term is taken off page by page: left to the end, the sums of u grow 128 times the number of keys and their rounding with
//   them (8000 keys in one accumulator: 2e-3 of the result; page by page 2.3e-4, of which 2.1e-4 is the result's own rounding).
// The running maximum m is that of score + log2 vs, raised when it grew by more than 2^8: weights are at most 256.  Scores beyond 2^10 lose their page's largest
// first, so that no rounding of m comes into the exponent (cache_far).  Statistics and sums are fp32; the weights' rounding to fp16 (2^-11 each,
// independent from key to key) is what tensor-core products of fp32 sums cost, as in k_attn.cuh.
//
// Work: a unit = one visible page of one kv head for up to 16 query rows (the rows of all heads that share the kv head, query-major; more
// rows are more row blocks), and one unit before an item's pages for its fixed cost.  All units of all sequences in one row are dealt out evenly: to
// blocks (one per SM), within a block to its 8 warps.  So contexts of any mix of lengths fill the machine, and the numbers on the device decide how: nothing but the launch is fixed on the host.
// A warp streams its pages through two 8-KB buffers of its own by bulk copies, one page ahead.  An item (all pages of a
// sequence, kv head and row block) that lies within one warp's share is finished there; otherwise partial results (maximum, sum, O)
// are merged in the block, and across blocks by the warp that arrives last (a counter per row of an item that crosses blocks; it resets
// it), in order: deterministic, one launch.
// Bound: one pass over the visible codes (HBM).  32:8 heads, 64 sequences of up to 4096 tokens, 328 MB: 61 to 65 us = 5.0 to 5.4 TB/s, 0.77 to 0.82 of the measured copy (while
// all warps stream, at its rate; the rest is the launch, the first pages' latency and the end: shares of whole pages of 2.3 us, 3 us to
// merge).  One sequence of 32000, 66 MB: 20.0 us = 0.50 (three or four pages per warp).  One of 300: 7.2 us, all latency.  Tried and slower: K one more page
// ahead in a third buffer (66 -> 70 us: V then comes late), asking the L2 for pages 1, 2 or 4 ahead (63 -> 70, 80, 92).
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "cache_dev.cuh"
#include "k_attn.cuh"
#include "umma.cuh"

namespace p0p {

struct CacheAttnP {
  CacheP c;
  const __half* Q; __half* O;
  uint32_t Hq, group, ldq, ldo, window, sinks;
  uint32_t max_rows;     // sequences with more query rows per kv head than this are another kernel's
  float scale_log2;      // scale * log2(e)
  float* part;           // [block][2][16][128] unnormalised O, then (maximum, sum) [block][2][16]
  float2* part_ml;
  uint32_t* count;       // [block][16] arrivals, zero between calls
};

constexpr uint32_t CA_WARPS = 8u, CA_LD = 132u, CA_RING = 2u * CACHE_BLOCK, CA_PART = 16u * CA_LD * 4u;
struct CaEntry { uint64_t i0, i1; uint32_t b, hk, rb, on; };              // a partial result of a warp: the units of its item's pages, the item
struct CaShared {
  uint64_t pre[CACHE_MAX_SEQS + 1];                                       // units before each sequence
  CacheSeq seq[CACHE_MAX_SEQS];
  float2 ml[CA_WARPS][2][16];
  CaEntry ent[CA_WARPS * 2];
  uint64_t bars[CA_WARPS][2];
  uint64_t warp_sum[CA_WARPS];
  uint32_t items, failed;
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
  const uint32_t bars = smem_u32(&sh.bars[warp][0]);
  if (lane < 2u) mbar_init(bars + 8u * lane, 1u);
  if (tid < CA_WARPS * 2u) sh.ent[tid].on = 0u;
  if (tid == 0u) { sh.failed = 0u; sh.items = 0u; }
  __syncthreads();
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
      if (s.n && (uint64_t)s.n * p.group <= p.max_rows) { c = cache_units(s, geo); atomicAdd(&sh.items, (uint32_t)min((uint64_t)p.c.Hkv * ((s.n * p.group + 15u) >> 4), (uint64_t)1u << 20)); }
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
  const uint64_t G = cache_workers(U, sh.items, gridDim.x);
  if (blockIdx.x >= G) return;
  // (both ends by one division, in two lanes; eight shares by a shift)
  const uint64_t end = deal_first(blockIdx.x + (lane & 1u), U, G);
  const uint64_t u0 = __shfl_sync(0xffffffffu, end, 0), u1 = __shfl_sync(0xffffffffu, end, 1), here = u1 - u0;
  if (warp < here) {
    const uint64_t w0 = u0 + (here < CA_WARPS ? warp : warp * here / CA_WARPS), w1 = u0 + (here < CA_WARPS ? warp + 1u : (warp + 1u) * here / CA_WARPS);
    CacheCursor cur;
    cur.seek(geo, sh.pre, sh.seq, w0);
    // pages of a row's blocks of codes, by the lane's page of 32: as the table has them, then checked, as blocks (page * Hkv + kv head)
    auto raw_at = [&](const CacheCursor& c, uint32_t t) {
      return t >= c.v.np || cache_vis_page(c.v, t) == c.s.L / CACHE_PAGE ? 0u : ld_now(p.c.table + (size_t)c.b * p.c.max_pages + cache_vis_page(c.v, t));
    };
    auto block_of = [&](const CacheCursor& c, uint32_t raw) {
      if (raw >= p.c.pages) { cache_tell(p.c.status, CACHE_BAD_PAGE); raw = 0u; }
      return raw * p.c.Hkv + c.hk;
    };
    // Every load is 8 KB, into buffer 0 or 1: a page's K and V, or two quarters of the tail (fp16): its K's lower and upper 32 keys, then its V's lower and
    // upper 64 of d.  Each buffer is asked for again as soon as it is read.
    auto load = [&](const void* src, uint32_t buf) {
      if (elect_one()) {
        mbar_expect_tx(bars + 8u * buf, CACHE_BLOCK);
        bulk_g2s(ring + buf * CACHE_BLOCK, src, CACHE_BLOCK, bars + 8u * buf);
      }
    };
    auto code_at = [&](uint32_t block, uint32_t w) -> const void* { return p.c.codes + ((size_t)block * 2u + w) * CACHE_BLOCK; };
    auto tail_at = [&](const CacheCursor& c, uint32_t quarter) -> const void* {
      return reinterpret_cast<const uint8_t*>(p.c.tail) + (((size_t)c.b * p.c.Hkv + c.hk) * 4u + quarter) * CACHE_BLOCK;
    };
    auto first_at = [&](const CacheCursor& c, uint32_t block, uint32_t w) { return c.tail(c.t()) ? tail_at(c, w) : code_at(block, w); };
    uint32_t ph = 0u;                                                      // parities of the two buffers' barriers
    bool ok = true;
    auto wait = [&](uint32_t buf) { ok = __all_sync(0xffffffffu, mbar_wait(bars + 8u * buf, (ph >> buf) & 1u, p.c.status, 611 + (int)buf)); ph ^= 1u << buf; return ok; };
    uint32_t qa[8][4], pa[4][4], pos[2];
    float bias[2], o[16][4], m[2], l[2], s[8][4], zp[4];
    bool far = false;                                                      // the item's maximum is large
    // scores (scaled, log2) -> weights pa, their sums zp; the running maximum rises only when it grew by more than 2^8 (weights are at most 256 then)
    auto weigh = [&](uint32_t page, uint32_t p0, uint32_t p1, float f, float lv, float inv_v) {
      float mx[2] = {-INFINITY, -INFINITY};
      if (cache_page_masked(page, p0, p1, p.window, p.sinks)) {
#pragma unroll
        for (uint32_t n = 0; n < 8u; n++)
#pragma unroll
          for (uint32_t e = 0; e < 4u; e++) {
            const uint32_t key = page * CACHE_PAGE + 16u * (n >> 1) + 4u * t4 + 2u * (n & 1u) + (e & 1u);
            s[n][e] = cache_key_visible(key, pos[e >> 1], p.window, p.sinks) ? s[n][e] : -INFINITY;
          }
      }
#pragma unroll
      for (uint32_t n = 0; n < 8u; n++) { mx[0] = fmaxf(fmaxf(mx[0], s[n][0]), s[n][1]); mx[1] = fmaxf(fmaxf(mx[1], s[n][2]), s[n][3]); }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1)); mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
      }
      const float raw[2] = {mx[0], mx[1]};
#pragma unroll
      for (int h = 0; h < 2; h++) mx[h] = fmaf(raw[h], f, lv);
      // (the difference, not m + 8: where m is large that sum may be m, or 16 more.  Against a maximum of -infinity it is infinity, or no number where the page shows nothing either)
      if (__any_sync(0xffffffffu, mx[0] - m[0] > 8.0f || mx[1] - m[1] > 8.0f)) {
        const float n0 = fmaxf(m[0], mx[0]), n1 = fmaxf(m[1], mx[1]);
        const float a0 = n0 == -INFINITY ? 1.0f : at_ex2(m[0] - n0), a1 = n1 == -INFINITY ? 1.0f : at_ex2(m[1] - n1);
        m[0] = n0; m[1] = n1; l[0] *= a0; l[1] *= a1;
#pragma unroll
        for (int d = 0; d < 16; d++) { o[d][0] *= a0; o[d][1] *= a0; o[d][2] *= a1; o[d][3] *= a1; }
        far = __any_sync(0xffffffffu, cache_far(n0) || cache_far(n1));
      }
      float e0 = m[0] == -INFINITY ? 0.0f : lv - m[0], e1 = m[1] == -INFINITY ? 0.0f : lv - m[1];      // (a row that has seen no key yet: all its weights are 0)
      if (far) {                                                           // large scores: see cache_far
        const float r0 = raw[0] == -INFINITY ? 0.0f : raw[0], r1 = raw[1] == -INFINITY ? 0.0f : raw[1];
        e0 = raw[0] == -INFINITY ? 0.0f : mx[0] - m[0]; e1 = raw[1] == -INFINITY ? 0.0f : mx[1] - m[1];      // (at most 8)
#pragma unroll
        for (uint32_t n = 0; n < 8u; n++) { s[n][0] -= r0; s[n][1] -= r0; s[n][2] -= r1; s[n][3] -= r1; }
      }
      zp[0] = zp[1] = zp[2] = zp[3] = 0.0f;
      float2 z0 = make_float2(0.0f, 0.0f), z1 = z0;
#pragma unroll
      for (uint32_t j = 0; j < 4u; j++) {
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++) {
          const float* x = s[2u * j + h];
          const float2 u0 = __ffma2_rn(make_float2(x[0], x[1]), make_float2(f, f), make_float2(e0, e0)), u1 = __ffma2_rn(make_float2(x[2], x[3]), make_float2(f, f), make_float2(e1, e1));
          const float2 w0 = make_float2(at_ex2(u0.x), at_ex2(u0.y)), w1 = make_float2(at_ex2(u1.x), at_ex2(u1.y));
          z0 = __fadd2_rn(z0, w0); z1 = __fadd2_rn(z1, w1);
          pa[j][2u * h] = at_pack(w0.x, w0.y);
          pa[j][2u * h + 1u] = at_pack(w1.x, w1.y);
        }
        at_mma(zp, pa[j], 0x3c003c00u, 0x3c003c00u);
      }
      l[0] = fmaf(z0.x + z0.y, inv_v, l[0]); l[1] = fmaf(z1.x + z1.y, inv_v, l[1]);
    };
    // a thread's two query rows (rows past the end repeat the last one; they are not stored)
    auto queries = [&](const CacheCursor& c) {
#pragma unroll
      for (uint32_t h = 0; h < 2u; h++) {
        const uint32_t r = min(c.rb * 16u + h * 8u + g, c.s.n * p.group - 1u), i = r / p.group;
        const uint4* q = reinterpret_cast<const uint4*>(p.Q + ((size_t)(c.hk * p.group + (r - i * p.group)) * p.ldq + c.s.r0 + i) * 128u + t4 * 16u);
#pragma unroll
        for (uint32_t k = 0; k < 2u; k++) {
          const uint4 a = ld_now(q + k * 8u), z = ld_now(q + k * 8u + 1u);
          qa[k * 4u][h] = a.x; qa[k * 4u][2u + h] = a.y; qa[k * 4u + 1u][h] = a.z; qa[k * 4u + 1u][2u + h] = a.w;
          qa[k * 4u + 2u][h] = z.x; qa[k * 4u + 2u][2u + h] = z.y; qa[k * 4u + 3u][h] = z.z; qa[k * 4u + 3u][2u + h] = z.w;
        }
      }
    };
    // ---- the first page is on its way before anything else.  (What has to come from memory is asked for before any of it is looked at: one after the
    // other, an item's loads took 6000 cycles.)
    const bool any = cur.at != 0u || w1 - w0 > 1u;
    uint32_t raw = any ? raw_at(cur, cur.t() + lane) : 0u;
    if (any) queries(cur);
    uint32_t blk = block_of(cur, raw);                                     // this lane's page of the 32 at hand
    if (any) {
      const uint32_t first = __shfl_sync(0xffffffffu, blk, 0);
      load(first_at(cur, first, 0u), 0u); load(first_at(cur, first, 1u), 1u);
    }
    for (uint64_t u = w0; any;) {
      // ---- an item, or this warp's share of it: pages t .. t + cnt - 1, of which the last may be the tail
      const uint64_t i0 = u - cur.at, end = min(u + (cur.v.np + 1u - cur.at), w1);
      const uint32_t t = cur.t(), cnt = (uint32_t)(end - u) - (cur.at ? 0u : 1u), rows = cur.s.n * p.group, p0 = cur.s.L - cur.s.n, p1 = cur.s.L - 1u;
      const bool done = t + cnt == cur.v.np, has_tail = done && (cur.s.L & (CACHE_PAGE - 1u)) != 0u, more = end + 1u < w1;      // (a share may end behind the unit that stands before an item's pages)
      const uint32_t codes = cnt - (has_tail ? 1u : 0u);
      float2 sc = ld_now(p.c.scales + blk), sc2 = sc;
      CacheCursor nxt = cur;
      uint32_t nxt_raw = 0u, nxt_blk = 0u, blk2 = 0u, raw2 = 0u;
      if (more) { nxt.next_item(geo, sh.pre, sh.seq); nxt_raw = raw_at(nxt, lane); }
      uint32_t nxt_first = 0u;
      auto next_item = [&](uint32_t w) {                                   // the first loads of what comes after this item
        if (!more) return;
        if (w == 0u) { nxt_blk = block_of(nxt, nxt_raw); nxt_first = __shfl_sync(0xffffffffu, nxt_blk, 0); }
        load(first_at(nxt, nxt_first, w), w);
      };
#pragma unroll
      for (uint32_t h = 0; h < 2u; h++) pos[h] = p0 + min(cur.rb * 16u + h * 8u + g, rows - 1u) / p.group;
      {
        float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 8; k++) at_mma(s4, qa[k], 0x80808080u, 0x80808080u);      // -128 * 2^-24 each
        bias[0] = s4[0]; bias[1] = s4[2];
      }
#pragma unroll
      for (int d = 0; d < 16; d++) { o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f; }
      m[0] = m[1] = -INFINITY; l[0] = l[1] = 0.0f; far = false;
      for (uint32_t i = 0; i < codes && ok; i++) {
        const uint32_t at = i & 31u;
        if (at == 0u) {                                                    // 32 pages at a time: the next ones' numbers are asked for here, their scales half way
          if (i > 0u) { blk = blk2; sc = sc2; }
          raw2 = raw_at(cur, t + i + 32u + lane);
        }
        if (at == 16u) { blk2 = block_of(cur, raw2); sc2 = ld_now(p.c.scales + blk2); }
        const float ks = __shfl_sync(0xffffffffu, sc.x, at), vs = __shfl_sync(0xffffffffu, sc.y, at);
        const uint32_t next = __shfl_sync(0xffffffffu, at == 31u ? blk2 : blk, (at + 1u) & 31u);
        auto follow = [&](uint32_t w) {
          if (i + 1u < codes) load(code_at(next, w), w);
          else if (has_tail) load(tail_at(cur, w), w);
          else next_item(w);
        };
        if (!wait(0u)) break;
#pragma unroll
        for (uint32_t n = 0; n < 8u; n += 4u) {                            // (four sums at a time: a product waits for the one before it on the same sum)
#pragma unroll
          for (uint32_t h = 0; h < 4u; h++) { s[n + h][0] = s[n + h][1] = bias[0]; s[n + h][2] = s[n + h][3] = bias[1]; }
#pragma unroll
          for (uint32_t k = 0; k < 2u; k++) {
            uint32_t w[4][4];
#pragma unroll
            for (uint32_t h = 0; h < 4u; h++) { const uint4 v = ca_lds(ring + (n + h) * 1024u + k * 512u + lane * 16u); w[h][0] = v.x; w[h][1] = v.y; w[h][2] = v.z; w[h][3] = v.w; }
#pragma unroll
            for (uint32_t j = 0; j < 4u; j++)
#pragma unroll
              for (uint32_t h = 0; h < 4u; h++) at_mma(s[n + h], qa[k * 4u + j], __byte_perm(w[h][j], 0u, 0x4140), __byte_perm(w[h][j], 0u, 0x4342));
          }
        }
        __syncwarp();                                                      // the K buffer is read
        follow(0u);
        weigh(cache_vis_page(cur.v, t + i), p0, p1, p.scale_log2 * ks * 16777216.0f, ca_lg2(vs), __fdividef(1.0f, vs));
        const float c0 = -0x1p-17f * zp[0], c1 = -0x1p-17f * zp[2];        // -128 * 2^-24 each
        if (!wait(1u)) break;
#pragma unroll
        for (uint32_t d = 0; d < 16u; d += 4u) {
          uint32_t w[4][4];
#pragma unroll
          for (uint32_t h = 0; h < 4u; h++) { const uint4 v = ca_lds(ring + CACHE_BLOCK + (d + h) * 512u + lane * 16u); w[h][0] = v.x; w[h][1] = v.y; w[h][2] = v.z; w[h][3] = v.w; }
#pragma unroll
          for (uint32_t h = 0; h < 4u; h++) {
            const float2 y = __fadd2_rn(make_float2(o[d + h][0], o[d + h][1]), make_float2(c0, c0)), v = __fadd2_rn(make_float2(o[d + h][2], o[d + h][3]), make_float2(c1, c1));
            o[d + h][0] = y.x; o[d + h][1] = y.y; o[d + h][2] = v.x; o[d + h][3] = v.y;
          }
#pragma unroll
          for (uint32_t j = 0; j < 4u; j++)
#pragma unroll
            for (uint32_t h = 0; h < 4u; h++) at_mma(o[d + h], pa[j], __byte_perm(w[h][j], 0u, 0x4140), __byte_perm(w[h][j], 0u, 0x4342));
        }
        __syncwarp();                                                      // the V buffer is read
        follow(1u);
      }
      if (!ok) { sh.failed = 1u; break; }
      // from here on O is in real units
#pragma unroll
      for (int d = 0; d < 16; d++) { o[d][0] *= 16777216.0f; o[d][1] *= 16777216.0f; o[d][2] *= 16777216.0f; o[d][3] *= 16777216.0f; }
      if (has_tail) {
        auto scores = [&](uint32_t from, uint32_t n0) {                    // of 32 keys
#pragma unroll
          for (uint32_t n = 0; n < 4u; n++) {
            float (&y)[4] = s[n0 + n];
            y[0] = y[1] = y[2] = y[3] = 0.0f;
#pragma unroll
            for (uint32_t k = 0; k < 2u; k++) {
              const uint4 w = ca_lds(from + n * 2048u + k * 1024u + lane * 32u), x = ca_lds(from + n * 2048u + k * 1024u + lane * 32u + 16u);
              at_mma(y, qa[k * 4u], w.x, w.y);
              at_mma(y, qa[k * 4u + 1u], w.z, w.w);
              at_mma(y, qa[k * 4u + 2u], x.x, x.y);
              at_mma(y, qa[k * 4u + 3u], x.z, x.w);
            }
          }
        };
        if (!wait(0u)) { sh.failed = 1u; break; }
        scores(ring, 0u);
        __syncwarp();
        load(tail_at(cur, 2u), 0u);
        if (!wait(1u)) { sh.failed = 1u; break; }
        scores(ring + CACHE_BLOCK, 4u);
        __syncwarp();
        load(tail_at(cur, 3u), 1u);
        weigh(cur.s.L / CACHE_PAGE, p0, p1, p.scale_log2, 0.0f, 1.0f);
        // (behind the sequence's end the tail may hold anything: those values weigh nothing, but 0 * NaN would count)
        const int have = (int)(cur.s.L & (CACHE_PAGE - 1u)) - (int)(4u * t4);
        uint32_t keep[4][2];
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int h = 0; h < 2; h++) { const int r = have - 16 * j - 2 * h; keep[j][h] = r >= 2 ? 0xffffffffu : r == 1 ? 0xffffu : 0u; }
        auto values = [&](uint32_t from, uint32_t d0) {                    // of 64 d
#pragma unroll
          for (uint32_t d = 0; d < 8u; d++) {
            const uint4 w = ca_lds(from + d * 1024u + lane * 32u), x = ca_lds(from + d * 1024u + lane * 32u + 16u);
            at_mma(o[d0 + d], pa[0], w.x & keep[0][0], w.y & keep[0][1]);
            at_mma(o[d0 + d], pa[1], w.z & keep[1][0], w.w & keep[1][1]);
            at_mma(o[d0 + d], pa[2], x.x & keep[2][0], x.y & keep[2][1]);
            at_mma(o[d0 + d], pa[3], x.z & keep[3][0], x.w & keep[3][1]);
          }
        };
        if (!wait(0u)) { sh.failed = 1u; break; }
        values(ring, 0u);
        __syncwarp();
        next_item(0u);
        if (!wait(1u)) { sh.failed = 1u; break; }
        values(ring + CACHE_BLOCK, 8u);
        __syncwarp();
        next_item(1u);
      }
      // ---- the end of the item, or of this warp's share
#pragma unroll
      for (int h = 0; h < 2; h++) { l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1); l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2); }
      if (more) queries(nxt);                                              // (on their way while the result leaves)
      if (done && i0 + 1u >= w0) {
        const float inv[2] = {l[0] > 0.0f ? 1.0f / l[0] : l[0], l[1] > 0.0f ? 1.0f / l[1] : l[1]};
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++) {
          const uint32_t r = cur.rb * 16u + h * 8u + g, i = r / p.group;
          if (r < rows) {
            uint32_t* dst = reinterpret_cast<uint32_t*>(p.O + (size_t)(cur.s.r0 + i) * p.ldo + (cur.hk * p.group + (r - i * p.group)) * 128u + 2u * t4);
#pragma unroll
            for (int d = 0; d < 16; d++) dst[4 * d] = cache_result(o[d][2 * h] * inv[h], o[d][2 * h + 1] * inv[h]);
          }
        }
      } else {
        // a share of an item: the warp's first item goes to a place of its own, its last one over its buffers (nothing is in flight then)
        const uint32_t which = i0 + 1u < w0 ? 0u : 1u;
        float* dst = which ? tailp : headp;
#pragma unroll
        for (int d = 0; d < 16; d++) {
          *reinterpret_cast<float2*>(dst + g * CA_LD + d * 8 + 2 * t4) = make_float2(o[d][0], o[d][1]);
          *reinterpret_cast<float2*>(dst + (g + 8u) * CA_LD + d * 8 + 2 * t4) = make_float2(o[d][2], o[d][3]);
        }
        if (t4 == 0u) { sh.ml[warp][which][g] = make_float2(m[0], l[0]); sh.ml[warp][which][g + 8u] = make_float2(m[1], l[1]); }
        if (lane == 0u) { CaEntry& e = sh.ent[warp * 2u + which]; e.i0 = i0 + 1u; e.i1 = i0 + 1u + cur.v.np; e.b = cur.b; e.hk = cur.hk; e.rb = cur.rb; e.on = 1u; }
      }
      if (!more) break;
      u = end;
      cur = nxt; blk = nxt_blk;
    }
    if (!ok && lane < 2u) mbar_drain(bars + 8u * lane, p.c.status, 613);
  }
  __syncthreads();
  // ---- the warps' shares of one item, merged in order, a row per warp; an item that is all here is finished.  A row of another one goes to memory, and the
  // warp that brings its last share merges the blocks' shares, in order.  (Row by row, with one release and acquire each, instead of a fence and a
  // barrier of the block: 6 -> 2 us from the last page to the end.)
  auto store = [&](const CaEntry& it, uint32_t r, float L, float4 v) {      // columns 4 lane .. of row r of the row block
    const CacheSeq q = sh.seq[it.b];
    const uint32_t x = it.rb * 16u + r, i = x / p.group;
    const float inv = L > 0.0f ? 1.0f / L : L;
    uint32_t* d = reinterpret_cast<uint32_t*>(p.O + (size_t)(q.r0 + i) * p.ldo + (it.hk * p.group + (x - i * p.group)) * 128u + 4u * lane);
    d[0] = cache_result(v.x * inv, v.y * inv); d[1] = cache_result(v.z * inv, v.w * inv);
  };
  auto rows_of = [&](const CaEntry& e) { return min(16u, sh.seq[e.b].n * p.group - e.rb * 16u); };
  // one arrival at row r of an item of blocks c0 .. c1; true for the last one
  auto arrive = [&](uint32_t c0, uint32_t c1, uint32_t r) {
    uint32_t last = 0u;
    __syncwarp();
    if (lane == 0u) {
      uint32_t* at = p.count + c0 * 16u + r;
      uint32_t before;
      asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(at) : "memory");
      last = before == c1 - c0 ? 1u : 0u;
      if (last) *at = 0u;
    }
    last = __shfl_sync(0xffffffffu, last, 0);
    __syncwarp();
    return last != 0u;
  };
  if (sh.failed) {                                                         // a wait ran out: the arrivals still have to be told, or the counters would not return to zero
    if (warp == 0u)
      cache_tell_shares(geo, sh.pre, sh.seq, u0, u1, [&](const CacheCursor& x, uint64_t i0, uint64_t i1) {
        const uint32_t c0 = (uint32_t)deal_owner(i0, U, G), c1 = (uint32_t)deal_owner(i1 - 1u, U, G), rows = min(16u, x.s.n * p.group - x.rb * 16u);
        for (uint32_t r = 0; r < rows; r++) arrive(c0, c1, r);
      });
    return;
  }
  const uint64_t my_i0 = lane < CA_WARPS * 2u && sh.ent[lane].on ? sh.ent[lane].i0 : ~0ull;
  uint32_t before = 0u;                                                    // rows of the items before
  for (uint32_t left = __ballot_sync(0xffffffffu, my_i0 != ~0ull); left;) {
    const uint32_t e0 = __ffs(left) - 1u, run = __ballot_sync(0xffffffffu, my_i0 == __shfl_sync(0xffffffffu, my_i0, e0)) & left;      // (shares of one item stand together, in order)
    left &= ~run;
    const CaEntry it = sh.ent[e0];
    const bool whole = it.i0 >= u0 && it.i1 <= u1;
    const uint32_t n = rows_of(it), r0 = (warp - before) & (CA_WARPS - 1u);
    before += n;
    if (r0 >= n) continue;
    uint32_t c0 = 0u, c1 = 0u;
    if (!whole) {
      const uint32_t own = (uint32_t)deal_owner(lane & 1u ? it.i1 - 1u : it.i0, U, G);
      c0 = __shfl_sync(0xffffffffu, own, 0); c1 = __shfl_sync(0xffffffffu, own, 1);
    }
    for (uint32_t r = r0; r < n; r += CA_WARPS) {
      // lane e has share e's maximum and sum, and its weight
      const bool mine = (run >> lane) & 1u;
      const float2 ml = mine ? sh.ml[lane >> 1][lane & 1u][r] : make_float2(-INFINITY, 0.0f);
      float M = ml.x;
#pragma unroll
      for (uint32_t x = 8; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
      M = __shfl_sync(0xffffffffu, M, 0);                                  // (16 shares: the lower lanes)
      const float f = ml.x == -INFINITY ? 0.0f : at_ex2(ml.x - M);
      float L = mine ? f * ml.y : 0.0f;
#pragma unroll
      for (uint32_t x = 8; x > 0; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
      L = __shfl_sync(0xffffffffu, L, 0);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (uint32_t k = run; k;) {                                         // four at a time
        float4 v[4]; float w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint32_t e = k ? __ffs(k) - 1u : e0;
          w[i] = __shfl_sync(0xffffffffu, f, e) * (k ? 1.0f : 0.0f);
          v[i] = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(gbase + ((e & 1u) ? (e >> 1) * CA_RING : CA_WARPS * CA_RING + (e >> 1) * CA_PART)) + r * CA_LD + 4u * lane);
          if (k) k &= k - 1u;
          else v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) { acc.x = fmaf(w[i], v[i].x, acc.x); acc.y = fmaf(w[i], v[i].y, acc.y); acc.z = fmaf(w[i], v[i].z, acc.z); acc.w = fmaf(w[i], v[i].w, acc.w); }
      }
      if (whole) { store(it, r, L, acc); continue; }
      // (a block has two places: 0 for the item that began before it, 1 for the one that goes on behind it)
      auto at = [&](uint32_t c) { return ((size_t)c * 2u + (c == c0 ? 1u : 0u)) * 16u + r; };
      const size_t here_at = ((size_t)blockIdx.x * 2u + (it.i0 < u0 ? 0u : 1u)) * 16u + r;
      *reinterpret_cast<float4*>(p.part + here_at * 128u + 4u * lane) = acc;
      if (lane == 0u) p.part_ml[here_at] = make_float2(M, L);
      if (!arrive(c0, c1, r)) continue;
      M = -INFINITY; L = 0.0f; acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (uint32_t c = c0; c <= c1; c += 8u) {                            // (eight blocks' shares at a time, the running maximum as elsewhere)
        float4 v[8]; float2 z[8];
        float top = M;
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) { const size_t x = at(min(c + i, c1)); v[i] = __ldcg(reinterpret_cast<const float4*>(p.part + x * 128u) + lane); z[i] = __ldcg(&p.part_ml[x]); }
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) top = fmaxf(top, z[i].x);
        const float a = M == -INFINITY ? 0.0f : at_ex2(M - top);
        M = top; L *= a; acc.x *= a; acc.y *= a; acc.z *= a; acc.w *= a;
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) {
          const float w = c + i <= c1 && z[i].x != -INFINITY ? at_ex2(z[i].x - M) : 0.0f;
          L += w * z[i].y;
          acc.x += w * v[i].x; acc.y += w * v[i].y; acc.z += w * v[i].z; acc.w += w * v[i].w;
        }
      }
      store(it, r, L, acc);
    }
  }
}

}  // namespace p0p
