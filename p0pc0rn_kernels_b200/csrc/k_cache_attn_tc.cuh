// Attention over the 8-bit cache for many new tokens per sequence (prompts), on the 5th-generation tensor cores.  The products, the running maximum
// and tensor memory are those of k_attn_tc.cuh (S = Q K^T, O += P V, two tiles of 128 rows that share every K / V tile, lane = row); what differs:
//   rows    a tile's rows are the queries of ALL heads that share a kv head, query by query (row = query * group + head), so a page is read
//           and converted once for them
//   K, V    arrive as codes (bulk copies) and are turned into fp16 whole numbers - exact - by two warps for K and two for V, into the swizzled
//           tiles that the multiplies read.  The cache's order makes a lane's 16 codes 32 consecutive bytes of a tile: for K 16 d of one key, for V
//           16 keys of one d (so V's tile is K-major).  The keys stand in the order of V's elements in both (cache_col_key).
//   scales  a thread's 64 scores belong to one page: its K scale joins the softmax scale, its V scale the exponent (w = 2^(score + log2 vs - m),
//           and the sum of the weights is weighted with 1 / vs), as in k_cache_attn.cuh
//           The tail has no scale: its weights are up to 2^15 instead (CTC_TAIL).  Scores beyond 2^10 lose their page's largest first (cache_far).
//   work    all items (block of queries, kv head) in one row are dealt out by cost, a unit for each pair of visible pages and CACHE_TC_ITEM for the item itself, to
//           one block per SM, from the numbers on the device.  An item within one block is finished there.  One of two shares is added up by the block that arrives
//           last with one, its own in tensor memory.  One of more shares is added up from memory: by the last block, or, where items are few (p.desc), by k_cache_merge
// Roles: warp 0 keeps the list of work (items, and page by page what the others need to know), warp 1 multiplies, warp 2 loads queries, warps 4-7 convert,
// warps 8-15 and 16-23 are the softmax of the two tiles, two threads per row.  The softmax threads take the registers that the others leave
// (setmaxnreg; per scheduler 4 x 104 + 24 + 40 = the 6 x 80 of the launch; with 32 for each of the others the converting warps spilled: 249 against 246.5 us).
// Bound: 2000 tokens over 6100 of 32:8 heads, 233 GFLOP: 231 to 237 us = 980 to 1010 TFLOP/s, 0.59 to 0.61 of the measured burst, under the power limit (1.6 to 1.7 GHz).  A pair of
// pages takes about 4200 cycles of a block: its multiplies alone 1900 (tensor pipe active 51 to 54 %), its traffic through shared memory 2500 (operands, codes
// in, tiles out), the converting warps about 3500 (latency: a warp's 16 units of 32 bytes, waits and fences in a row), a softmax warp 1700.  Tried and slower: conversion
// by the softmax warps between two tiles (308 us), K as fp16 subnormals with a row sum of q (255 against 260 then, but 147 against 141 for short
// items), 96 registers for the softmax and 48 for the others (390), three slots of tiles and more codes (256).
#pragma once
#include <cuda.h>

#include "attn_tc.cuh"
#include "cache_dev.cuh"
#include "epilogue.cuh"
#include "umma.cuh"

namespace p0p {

struct CacheTcDesc { uint32_t on, row0, q, hk, c1; };      // an item of more than two shares that begins in this block: its first row, its queries, its last block
struct CacheTcP {
  CacheP c;
  __half* O;
  uint32_t ldo;
  CacheTcGeo geo;
  float scale_log2;
  float4* part;          // [block][2][32 groups of 4 columns][256 rows] unnormalised O
  float2* part_ml;       // [block][2][2 halves][256 rows] (maximum, sum)
  uint32_t* count;       // [block][16 warps] arrivals, zero between calls
  CacheTcDesc* desc;     // [block]; NULL: items of more than two shares are added up here as well
};

// Four slots of tiles: with three the K tile two pairs ahead takes the V tile's place, and its conversion waits for that product.  What is left of
// shared memory holds one pair's codes: 4 KB of each page for each converting warp, which asks for the next ones itself as soon as it has read them (one
// warp loading for all four, or a lane for each of the eight, came late: 4000 cycles from the last read to the next codes).
constexpr uint32_t CTC_THREADS = 768u, CTC_SLOTS = 4u, CTC_STAGE = CACHE_BLOCK / 2u;
constexpr int CTC_REGS = 16 * 104 + 4 * 24 + 4 * 40;      // registers per lane of all warps, after setmaxnreg
constexpr float CTC_TAIL = 15.0f;      // log2 of the tail's largest weight
constexpr uint32_t CTC_PAIRS = 4u;     // pairs of pages that are described ahead
constexpr uint32_t CTC_SEGS = 4u;      // items that are announced ahead
// an item's share
struct CtcSeg { uint32_t cnt, t, units, r0, n, L, hk, spent; };
// a page of a pair.  For the softmax: scale_log2 * K scale, log2 and reciprocal of the V scale, its first key | 1 where some key is hidden from some row | 2 in a
// pair that holds the tail | 4 for the tail.
// For the conversion: what it is (codes 0, the tail 1 | its tokens << 8, nothing 2, the end of the work 3), and which block of codes or of the tail.
struct CtcPage { float f, lv, inv_v; uint32_t key0, is, block, pad[2]; };
constexpr uint32_t CTC_SMEM = (2u + CTC_SLOTS) * ATC_TILE + 8u * CTC_STAGE + 512u + 2048u + CTC_PAIRS * 2u * (uint32_t)sizeof(CtcPage) + CTC_SEGS * (uint32_t)sizeof(CtcSeg) + 64u;
static_assert(CTC_SMEM <= 232448u, "shared memory");
static_assert(8u * CTC_STAGE >= CACHE_MAX_SEQS * 8u, "the sequences' costs fit the codes' place while nothing is in it");

template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// 16 codes (code + 128) -> 16 fp16 whole numbers: a byte behind 0x64 is 1024 + code + 128
__device__ __forceinline__ void ctc_convert(uint4 w, uint4& a, uint4& b) {
  const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));      // 1152
  auto two = [&](uint32_t v, uint32_t sel) { const uint32_t r = __byte_perm(v, 0x64646464u, sel); const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&r), off); return *reinterpret_cast<const uint32_t*>(&h); };
  a = make_uint4(two(w.x, 0x4140), two(w.x, 0x4342), two(w.y, 0x4140), two(w.y, 0x4342));
  b = make_uint4(two(w.z, 0x4140), two(w.z, 0x4342), two(w.w, 0x4140), two(w.w, 0x4342));
}
__device__ __forceinline__ void ctc_sts(uint32_t a, uint4 v) { asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }
__device__ __forceinline__ uint4 ctc_lds(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// a named barrier of 64 threads at which all learn whether all are fine
__device__ __forceinline__ bool ctc_agree(int bar, bool fine) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.and.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"(bar), "r"(fine ? 1u : 0u) : "memory");
  return r != 0u;
}

__global__ void __launch_bounds__(CTC_THREADS, 1) k_cache_attn_tc(const CacheTcP p, const __grid_constant__ CUtensorMap mapQ) {
  extern __shared__ __align__(1024) unsigned char ctc_raw[];             // (the swizzled tiles; there is no room to align them by hand, and no static shared memory before them)
  const uint32_t base = smem_u32(ctc_raw);
  unsigned char* gbase = ctc_raw;
  if (base & 1023u) {
    grid_dependency_wait();
    if (threadIdx.x == 0u) { if (p.desc) p.desc[blockIdx.x].on = 0u; cache_tell(p.c.status, 633); }
    return;
  }
  const uint32_t q_sm = base, kv_sm = base + 2u * ATC_TILE, st_sm = kv_sm + CTC_SLOTS * ATC_TILE, bars = st_sm + 8u * CTC_STAGE;
  const uint32_t q_full = bars, q_empty = bars + 8u, st_full = bars + 16u, kv_full = st_full + 64u, kv_empty = kv_full + 8u * CTC_SLOTS, s_full = kv_empty + 8u * CTC_SLOTS, p_full = s_full + 16u;
  const uint32_t o_full = p_full + 16u, seg_full = o_full + 16u, seg_empty = seg_full + 8u * CTC_SEGS, pair_full = seg_empty + 8u * CTC_SEGS, pair_empty = pair_full + 8u * CTC_PAIRS;
  const uint32_t all_done = pair_empty + 8u * CTC_PAIRS, tmem_slot = all_done + 8u;
  float* xch = reinterpret_cast<float*>(gbase + (bars + 512u - base));
  CtcPage* scl = reinterpret_cast<CtcPage*>(xch + 512);                   // [pair][page of it]
  volatile CtcSeg* segs = reinterpret_cast<volatile CtcSeg*>(scl + 2u * CTC_PAIRS);
  volatile uint32_t* at = reinterpret_cast<volatile uint32_t*>(const_cast<CtcSeg*>(segs) + CTC_SEGS);
  const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u;
  if (tid == 0) {
    mbar_init(q_full, 1u); mbar_init(q_empty, 1u); mbar_init(all_done, 1u);
    for (uint32_t s = 0; s < 8u; s++) mbar_init(st_full + 8u * s, 1u);
    for (uint32_t s = 0; s < CTC_SLOTS; s++) { mbar_init(kv_full + 8u * s, 2u); mbar_init(kv_empty + 8u * s, 1u); }
    for (uint32_t t = 0; t < 2u; t++) { mbar_init(s_full + 8u * t, 1u); mbar_init(p_full + 8u * t, 8u); mbar_init(o_full + 8u * t, 1u); }
    for (uint32_t s = 0; s < CTC_SEGS; s++) { mbar_init(seg_full + 8u * s, 1u); mbar_init(seg_empty + 8u * s, 18u); }      // (queries, multiplies, softmax)
    for (uint32_t s = 0; s < CTC_PAIRS; s++) { mbar_init(pair_full + 8u * s, 1u); mbar_init(pair_empty + 8u * s, 1u); }
    fence_mbar_init();
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 512u); tmem_relinquish(); }
  tc_fence_before();
  grid_dependency_wait();
  grid_launch_dependents();
  // ---- this block's share of the work: cost per sequence, their sum, then where the share begins
  {
    uint64_t* per_seq = reinterpret_cast<uint64_t*>(gbase + (st_sm - base));
    uint32_t items = 0u;
    for (uint32_t b = warp; b < p.geo.seqs; b += CTC_THREADS / 32u) {
      const CacheSeq s = cache_seq(p.c, b);
      const uint32_t n = cache_tc_blocks(s, p.geo);
      uint64_t u = 0u;
      for (uint32_t x = lane; x < n; x += 32u) u += cache_tc_cost(cache_tc_part(s, p.geo, x), p.geo);
#pragma unroll
      for (uint32_t o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
      items += n;
      if (lane == 0u) per_seq[b] = u * p.geo.Hkv;
    }
    if (tid == 0) at[5] = 0u;
    __syncthreads();
    if (lane == 0u && items) atomicAdd(const_cast<uint32_t*>(at) + 5, items);
    __syncthreads();
    if (warp == 0u) {
      auto scan = [&](uint64_t v) {
#pragma unroll
        for (uint32_t o = 1; o < 32u; o <<= 1) { const uint64_t w = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += w; }
        return v;
      };
      uint64_t U = 0u;
      for (uint32_t b = 0; b < p.geo.seqs; b += 32u) U += __shfl_sync(0xffffffffu, scan(b + lane < p.geo.seqs ? per_seq[b + lane] : 0u), 31);
      const uint64_t G = cache_tc_workers(U, (uint64_t)at[5] * p.geo.Hkv, gridDim.x);
      uint64_t u0 = 0u, u1 = 0u;
      if (blockIdx.x < G) { u0 = deal_first(blockIdx.x, U, G); u1 = deal_first(blockIdx.x + 1u, U, G); }
      if (lane == 0u) {
        at[4] = (uint32_t)(u1 - u0);
        at[6] = (uint32_t)U; at[7] = (uint32_t)(U >> 32); at[8] = (uint32_t)G; at[9] = (uint32_t)u0; at[10] = (uint32_t)(u0 >> 32);
        if (p.desc) p.desc[blockIdx.x].on = 0u;
      }
      if (u1 > u0) {
        uint64_t r = u0;                                                  // cost before ours, from here on within a sequence, then a block of queries
        uint32_t b = 0u;
        for (uint32_t b0 = 0; b0 < p.geo.seqs; b0 += 32u) {
          const uint64_t mine = b0 + lane < p.geo.seqs ? per_seq[b0 + lane] : 0u, inc = scan(mine), all = __shfl_sync(0xffffffffu, inc, 31);
          const uint32_t hit = __ballot_sync(0xffffffffu, inc > r);
          if (hit) { const uint32_t l = __ffs(hit) - 1u; b = b0 + l; r -= __shfl_sync(0xffffffffu, inc - mine, l); break; }
          r -= all;
        }
        const CacheSeq s = cache_seq(p.c, b);
        const uint32_t n = cache_tc_blocks(s, p.geo);
        for (uint32_t x0 = 0; x0 < n; x0 += 32u) {
          const uint32_t u = x0 + lane < n ? cache_tc_cost(cache_tc_part(s, p.geo, x0 + lane), p.geo) : 0u;
          const uint64_t mine = (uint64_t)u * p.geo.Hkv, inc = scan(mine), all = __shfl_sync(0xffffffffu, inc, 31);
          const uint32_t hit = __ballot_sync(0xffffffffu, inc > r);
          if (hit) {
            const uint32_t l = __ffs(hit) - 1u;
            if (lane == l) { r -= inc - mine; at[0] = b; at[1] = x0 + l; at[2] = (uint32_t)(r / u); at[3] = (uint32_t)(r % u); }
            break;
          }
          r -= all;
        }
      }
    }
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t*>(gbase + (tmem_slot - base)), 0);
  // an item's share, to the other roles: they wait for it here and give it back when they are done with it (every warp of them)
  auto seg_wait = [&](uint32_t seg) { return mbar_wait(seg_full + 8u * (seg % CTC_SEGS), (seg / CTC_SEGS) & 1u, p.c.status, 620, 50u); };
  auto seg_done = [&](uint32_t seg) { __syncwarp(); if (lane == 0u) mbar_arrive(seg_empty + 8u * (seg % CTC_SEGS)); };

  if (warp < 4u) {
    regs_down<24>();
    if (warp == 0u) {
      // ================================================================= the list of work: items, and page by page what the others need to know.  Lane l looks
      // after the l-th of 32 visible pages
      uint32_t pair = 0u, seg = 0u;
      CacheTcWalk w;
      const auto seq = [&](uint32_t b) { return cache_seq(p.c, b); };
      w.begin(p.geo, at[0], at[1], at[2], at[3], at[4], seq);
      bool ok = true;
      for (; ok; w.next(p.geo, seq), seg++) {
        if (seg >= CTC_SEGS) ok = __all_sync(0xffffffffu, mbar_wait(seg_empty + 8u * (seg % CTC_SEGS), (seg / CTC_SEGS - 1u) & 1u, p.c.status, 632, 50u));
        if (!ok) break;
        if (lane == 0u) {
          volatile CtcSeg& g = segs[seg % CTC_SEGS];
          g.cnt = w.cnt; g.t = w.t; g.units = w.units; g.r0 = w.part.r0; g.n = w.part.n; g.L = w.part.L; g.hk = w.hk; g.spent = w.spent;
          mbar_arrive(seg_full + 8u * (seg % CTC_SEGS));
        }
        __syncwarp();
        CtcPage pg{1.0f, 0.0f, 1.0f, 0u, 2u, 0u, {0u, 0u}};
        for (uint32_t j = 0; j < max(w.cnt, 1u) && ok; j++, pair++) {
          const uint32_t l0 = (2u * j) & 31u;
          if (l0 == 0u) {
            const uint32_t k = 2u * (w.t + j) + lane, page = cache_vis_page(w.v, k);
            // (both pages of the tail's pair are marked, as masked too: their rows' threads agree on the maximum)
            const uint32_t marks = (k | 1u) >= w.v.np - 1u && cache_vis_page(w.v, w.v.np - 1u) == w.s.L / CACHE_PAGE ? 3u : 0u;
            pg = CtcPage{1.0f, 0.0f, 1.0f, 0u - CACHE_PAGE | marks | 1u, w.cnt ? 2u : 3u, 0u, {0u, 0u}};      // no page: every key hidden
            if (w.cnt && k < w.v.np) {
              float2 sc = make_float2(1.0f, 1.0f);
              if (page < w.s.L / CACHE_PAGE) {
                uint32_t at_page = ld_now(p.c.table + (size_t)w.b * p.c.max_pages + page);
                if (at_page >= p.c.pages) { cache_tell(p.c.status, CACHE_BAD_PAGE); at_page = 0u; }
                pg.block = at_page * p.c.Hkv + w.hk; pg.is = 0u;
                sc = ld_now(p.c.scales + pg.block);
              } else {
                pg.block = w.b * p.c.Hkv + w.hk; pg.is = 1u | (w.s.L & (CACHE_PAGE - 1u)) << 8;
              }
              pg.f = p.scale_log2 * sc.x; pg.inv_v = __fdividef(1.0f, sc.y);
              asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(pg.lv) : "f"(sc.y));
              pg.key0 = page * CACHE_PAGE | marks | (pg.is & 1u) << 2 | (cache_page_masked(page, w.part.L - w.part.n, w.part.L - 1u, p.geo.window, p.geo.sinks) ? 1u : 0u);
            }
          }
          if (pair >= CTC_PAIRS) ok = __all_sync(0xffffffffu, mbar_wait(pair_empty + 8u * (pair % CTC_PAIRS), (pair / CTC_PAIRS - 1u) & 1u, p.c.status, 622, 20u));
          if (!ok) break;
          if (lane == l0 || lane == l0 + 1u) scl[(pair % CTC_PAIRS) * 2u + (lane - l0)] = pg;
          __syncwarp();
          if (lane == 0u) mbar_arrive(pair_full + 8u * (pair % CTC_PAIRS));
        }
        if (!w.cnt) break;
      }
    } else if (warp == 2u) {
      // ================================================================= queries
      uint32_t seg = 0u;
      for (;; seg++) {
        if (!__all_sync(0xffffffffu, seg_wait(seg))) break;
        volatile CtcSeg& g = segs[seg % CTC_SEGS];
        if (!g.cnt) break;
        const uint32_t r0 = g.r0, hk = g.hk, nt = g.n > p.geo.qpt ? 2u : 1u;
        seg_done(seg);
        if (seg > 0u && !__all_sync(0xffffffffu, mbar_wait(q_empty, (seg - 1u) & 1u, p.c.status, 621, 20u))) break;
        if (lane == 0u) {
          mbar_expect_tx(q_full, nt * 2u * p.geo.qpt * p.geo.group * 128u);
          for (uint32_t t = 0; t < nt; t++)
            for (uint32_t c = 0; c < 2u; c++) tma_load_4d(q_sm + t * ATC_TILE + c * 16384u, &mapQ, (int)(c * 64u), 0, (int)(r0 + t * p.geo.qpt), (int)hk, q_full);
        }
      }
      if (seg > 0u) mbar_wait(q_full, (seg - 1u) & 1u, p.c.status, 635);   // (the last ones are here before the block ends, whatever became of the others)
    } else if (warp == 1u) {
      // ================================================================= multiplies (the whole warp walks the loop, one lane issues)
      const uint32_t idesc = umma_idesc_f16(128u, 128u);
      const uint64_t qd[2] = {umma_desc_sw128(q_sm), umma_desc_sw128(q_sm + ATC_TILE)};
      uint32_t i = 0u, seg = 0u, np[2] = {0u, 0u};                        // tiles of K and V, items, weights consumed per tile of rows
      bool ok = true;
      for (; ok; seg++) {
        if (!__all_sync(0xffffffffu, seg_wait(seg))) break;
        const uint32_t cnt = segs[seg % CTC_SEGS].cnt, nt = segs[seg % CTC_SEGS].n > p.geo.qpt ? 2u : 1u;
        seg_done(seg);
        if (!cnt) break;
        ok = __all_sync(0xffffffffu, mbar_wait(q_full, seg & 1u, p.c.status, 623) && mbar_wait(kv_full + 8u * (i % CTC_SLOTS), (i / CTC_SLOTS) & 1u, p.c.status, 624));
        if (!ok) break;
        tc_fence_after();
        {
          const uint64_t kd = umma_desc_sw128(kv_sm + (i % CTC_SLOTS) * ATC_TILE);
          if (elect_one()) {
            for (uint32_t t = 0; t < nt; t++) {
#pragma unroll
              for (uint32_t kk = 0; kk < 8u; kk++) umma_f16_ss(tmem_base + t * 128u, qd[t] + (kk >> 2) * 1024u + 2u * (kk & 3u), kd + (kk >> 2) * 1024u + 2u * (kk & 3u), idesc, kk);
              umma_commit(s_full + 8u * t);
            }
            umma_commit(kv_empty + 8u * (i % CTC_SLOTS));
            if (cnt == 1u) umma_commit(q_empty);
          }
          __syncwarp();
        }
        for (uint32_t j = 0; j < cnt && ok; j++, i += 2u) {
          const uint32_t iv = i + 1u, sv = iv % CTC_SLOTS, ik = i + 2u, sk = ik % CTC_SLOTS;
          const bool more = j + 1u < cnt;
          bool rdy = mbar_wait(kv_full + 8u * sv, (iv / CTC_SLOTS) & 1u, p.c.status, 625);
          if (more) rdy = rdy && mbar_wait(kv_full + 8u * sk, (ik / CTC_SLOTS) & 1u, p.c.status, 626);
          if (!__all_sync(0xffffffffu, rdy)) { ok = false; break; }
          const uint64_t vd = umma_desc_sw128(kv_sm + sv * ATC_TILE), kd = umma_desc_sw128(kv_sm + sk * ATC_TILE);
          for (uint32_t t = 0; t < nt; t++) {
            if (!__all_sync(0xffffffffu, mbar_wait(p_full + 8u * t, np[t] & 1u, p.c.status, 627))) { ok = false; break; }
            np[t]++;
            tc_fence_after();
            const uint32_t s_col = tmem_base + t * 128u, o_col = tmem_base + 256u + t * 128u;
            const uint64_t qdt = qd[t];
            if (elect_one()) {
#pragma unroll
              for (uint32_t kk = 0; kk < 8u; kk++) umma_f16_ts(o_col, s_col + 8u * kk, vd + (kk >> 2) * 1024u + 2u * (kk & 3u), idesc, j | kk);
              if (more) {
#pragma unroll
                for (uint32_t kk = 0; kk < 8u; kk++) umma_f16_ss(s_col, qdt + (kk >> 2) * 1024u + 2u * (kk & 3u), kd + (kk >> 2) * 1024u + 2u * (kk & 3u), idesc, kk);
                umma_commit(s_full + 8u * t);
              } else
                umma_commit(o_full + 8u * t);
            }
            __syncwarp();
          }
          if (ok && elect_one()) {
            umma_commit(kv_empty + 8u * sv);
            if (more) umma_commit(kv_empty + 8u * sk);
            if (j + 2u == cnt) umma_commit(q_empty);                    // the item's last scores are under way
            mbar_arrive(pair_empty + 8u * ((i >> 1) % CTC_PAIRS));      // (converted, and read by the softmax before it handed over the weights)
          }
          __syncwarp();
        }
      }
      if (elect_one()) umma_commit(all_done);                             // (no multiply is under way when the block ends)
      __syncwarp();
      mbar_wait(all_done, 0u, p.c.status, 636);
    }
  } else if (warp < 8u) {
    // ================================================================= codes (or the tail's fp16) -> fp16 tiles
    regs_down<40>();
    // Two warps for K, two for V; a warp has half of each page: units 256 part + 32 e + lane of its 512 (16 elements each).  A unit's 32 bytes go to row r of the
    // tile's half h, pieces 2 (u % 4) and the next, swizzled
    //   K: r = 64 page + 16 (u / 8 % 4) + 4 (u / 128) + 2 (u / 64 % 2) + u / 4 % 2 (the key's column), h = u / 32 % 2 (which 64 of d);   V: r = u / 4 (d), h = page
    const uint32_t kind = (warp - 4u) >> 1, part = warp & 1u, ch = 2u * (lane & 3u), x = kind ? lane >> 2 : (lane >> 2) & 1u, c0 = (ch ^ x) << 4, c1 = ((ch + 1u) ^ x) << 4;
    const uint32_t to = kv_sm + (kind ? (part * 64u + (lane >> 2)) * 128u : ((lane >> 3) * 16u + part * 8u + x) * 128u), stage = st_sm + (warp - 4u) * 2u * CTC_STAGE, bar = st_full + (warp - 4u) * 16u;
    uint32_t arrived = 0u;                                                // bit h: parity of page h's loads
    const uint8_t* const codes = p.c.codes + kind * CACHE_BLOCK + part * CTC_STAGE;
    auto fetch = [&](uint32_t block, uint32_t half) {                     // one lane
      mbar_expect_tx(bar + 8u * half, CTC_STAGE);
      bulk_g2s(stage + half * CTC_STAGE, codes + (size_t)block * (2u * CACHE_BLOCK), CTC_STAGE, bar + 8u * half);
    };
    auto announced = [&](uint32_t pair) { return __all_sync(0xffffffffu, mbar_wait(pair_full + 8u * (pair % CTC_PAIRS), (pair / CTC_PAIRS) & 1u, p.c.status, 634)); };
    fence_proxy_async();                                                  // (the codes' place held the costs)
    bool ok = announced(0u);
    if (ok && lane < 2u && scl[lane].is == 0u) fetch(scl[lane].block, lane);
    for (uint32_t pair = 0u; ok; pair++) {
      const CtcPage* pg = scl + (pair % CTC_PAIRS) * 2u; const CtcPage* nx = scl + ((pair + 1u) % CTC_PAIRS) * 2u;
      if (pg->is == 3u) break;
      // (whether the next pair is announced is looked at without waiting: that could wait for this one)
      const bool known = __all_sync(0xffffffffu, mbar_test(pair_full + 8u * ((pair + 1u) % CTC_PAIRS), ((pair + 1u) / CTC_PAIRS) & 1u));
      const uint32_t slot = (2u * pair + kind) % CTC_SLOTS, use = (2u * pair + kind) / CTC_SLOTS, dst = to + slot * ATC_TILE;
      if (use > 0u) ok = __all_sync(0xffffffffu, mbar_wait(kv_empty + 8u * slot, (use - 1u) & 1u, p.c.status, 629));
      for (uint32_t half = 0; half < 2u && ok; half++) {
        const uint32_t from = stage + half * CTC_STAGE + lane * 16u, at_h = dst + half * (kind ? 16384u : 8192u), is = pg[half].is;
        uint32_t next = 0xffffffffu;                                      // the block to ask for (a cache has fewer)
        if (known && nx[half].is == 0u) next = nx[half].block;
        if (is == 0u) {
          ok = __all_sync(0xffffffffu, mbar_wait(bar + 8u * half, (arrived >> half) & 1u, p.c.status, 628));
          if (!ok) break;
          arrived ^= 1u << half;
          if (kind == 0u) {
#pragma unroll
            for (uint32_t e = 0; e < 8u; e++) {                           // e = 4 (u / 128 % 2) + 2 (u / 64 % 2) + h: rows, which turn the swizzle, and the half
              constexpr uint32_t HALF = 16384u;
              const uint32_t rows = (e >> 2) * 4u + ((e >> 1) & 1u) * 2u;
              uint4 a, b;
              ctc_convert(ctc_lds(from + e * 512u), a, b);
              ctc_sts(at_h + (e & 1u) * HALF + rows * 128u + (c0 ^ (rows << 4)), a);
              ctc_sts(at_h + (e & 1u) * HALF + rows * 128u + (c1 ^ (rows << 4)), b);
            }
          } else {
#pragma unroll
            for (uint32_t e = 0; e < 8u; e++) {
              uint4 a, b;
              ctc_convert(ctc_lds(from + e * 512u), a, b);
              ctc_sts(at_h + e * 1024u + c0, a);
              ctc_sts(at_h + e * 1024u + c1, b);
            }
          }
        } else {
          const uint4* tl = reinterpret_cast<const uint4*>(p.c.tail + ((size_t)pg[half].block * 2u + kind) * CACHE_BLOCK) + part * 512u + 2u * lane;
#pragma unroll 1
          for (uint32_t e = 0; e < 8u; e++) {
            uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
            if (is != 2u) {
              a = ld_now(tl + e * 64u); b = ld_now(tl + e * 64u + 1u);
              if (kind) {                                                 // keys behind the sequence's end may hold anything: they weigh nothing, but 0 * NaN would count
                const int have = (int)(is >> 8) - (int)(4u * (lane & 3u));
                auto keep = [&](uint32_t v, int at) { return have >= at + 2 ? v : have == at + 1 ? v & 0xffffu : 0u; };
                a.x = keep(a.x, 0); a.y = keep(a.y, 2); a.z = keep(a.z, 16); a.w = keep(a.w, 18);
                b.x = keep(b.x, 32); b.y = keep(b.y, 34); b.z = keep(b.z, 48); b.w = keep(b.w, 50);
              }
            }
            const uint32_t rows = (e >> 2) * 4u + ((e >> 1) & 1u) * 2u, flip = kind ? 0u : rows << 4, at_e = at_h + (kind ? e * 1024u : (e & 1u) * 16384u + rows * 128u);
            ctc_sts(at_e + (c0 ^ flip), a);
            ctc_sts(at_e + (c1 ^ flip), b);
          }
        }
        if (half) fence_proxy_async();
        __syncwarp();
        if (lane == 0u) {
          if (half) mbar_arrive(kv_full + 8u * slot);
          if (next != 0xffffffffu) fetch(next, half);
        }
      }
      if (!ok) break;
      ok = announced(pair + 1u);
      if (ok && !known && lane < 2u && nx[lane].is == 0u) fetch(nx[lane].block, lane);
      __syncwarp();
    }
    if (!ok && lane < 2u) mbar_drain(bar + 8u * lane, p.c.status, 637);
  } else {
    // ================================================================= softmax of one tile: two threads per row, one page of a pair each
    regs_up<104>();
    const uint32_t t = (warp - 8u) >> 3, half = ((warp - 8u) >> 2) & 1u, row = (warp & 3u) * 32u + lane;
    const uint32_t lane_addr = tmem_base + (((warp & 3u) * 32u) << 16), s_addr = lane_addr + t * 128u + half * 64u, p_addr = lane_addr + t * 128u + half * 32u;
    const uint32_t o_addr = lane_addr + 256u + t * 128u + half * 64u, pair_bar = 1u + t * 4u + (warp & 3u);
    float* mine = xch + (t * 2u + half) * 128u + row; const float* other = xch + (t * 2u + (half ^ 1u)) * 128u + row;
    const uint32_t qi = row / p.geo.group, hh = row - qi * p.geo.group;
    uint32_t n = 0u, pair = 0u, items = 0u;                               // this tile's scores and items so far, the block's pairs of pages
    bool ok = true;
    for (uint32_t seg = 0u;; seg++) {
      if (ok && !seg_wait(seg)) ok = false;
      volatile CtcSeg& g = segs[seg % CTC_SEGS];
      ok = ctc_agree((int)pair_bar, ok);                                  // (the two warps of a row meet at barriers: both go on, or neither)
      const uint32_t cnt = ok ? g.cnt : 0u;
      if (!cnt) break;
      if (t == 1u && g.n <= p.geo.qpt) { pair += cnt; seg_done(seg); continue; }
      const uint32_t pos = g.L - g.n + min(t * p.geo.qpt + qi, g.n - 1u);
      float m_used = -INFINITY, l = 0.0f;
      bool far = false;                                                   // the maximum is large
      for (uint32_t j = 0; j < cnt; j++, n++, pair++) {
        // (a wait that ran out: the thread goes on without it, so that its partner is not left at the barrier; the status word is set)
        if (ok && !mbar_wait(s_full + 8u * t, n & 1u, p.c.status, 630)) ok = false;
        tc_fence_after();
        uint32_t s[64];
#pragma unroll
        for (int c = 0; c < 4; c++) tmem_ld16(s_addr + 16u * c, *reinterpret_cast<uint32_t(*)[16]>(&s[16 * c]));
        const float4 pg = *reinterpret_cast<const float4*>(&scl[(pair % CTC_PAIRS) * 2u + half]);      // f, lv, inv_v, key0
        const float sc = pg.x, lv = pg.y;
        const uint32_t key0 = __float_as_uint(pg.w);
        tmem_ld_wait();
        // A page's values are at most 127 times its V scale, the tail's are as they are (scale 1): relative to the tail's largest weight, the weights of the page beside it
        // would be fp16 subnormals where values are small.  So the tail's weights are up to 2^15 (CTC_TAIL), the others below 1 then: its scores count that much
        // less for the maximum, which is exact in its pair (no page comes after it).
        float slack = 8.0f, less = 0.0f;
        if (key0 & 1u) {
          // columns whose key is visible: at most hi, and at least lo or below sk (all relative to the page)
          const uint32_t k0 = key0 & ~(CACHE_PAGE - 1u);
          if (key0 & 2u) slack = 0.0f;
          if (key0 & 4u) less = CTC_TAIL;
          const int hi = (int)min(pos - min(pos, k0), 64u) - (pos < k0 ? 1 : 0);
          int lo = 0, sk = 0;
          if (p.geo.window && pos >= p.geo.window) {
            const uint32_t first = pos - p.geo.window + 1u;
            lo = (int)min(first - min(first, k0), 64u); sk = (int)min(p.geo.sinks - min(p.geo.sinks, k0), 64u);
          }
#pragma unroll
          for (int c = 0; c < 64; c++) {
            const int key = (int)cache_col_key(c);
            s[c] = key <= hi && (key >= lo || key < sk) ? s[c] : 0xff800000u;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 64; c += 8) {
#pragma unroll
          for (int e = 0; e < 4; e++) mx[e] = fmaxf(fmaxf(mx[e], __uint_as_float(s[c + 2 * e])), __uint_as_float(s[c + 2 * e + 1]));      // (one instruction: the maximum of three)
        }
        float mts = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), sc, lv - less);
        *mine = mts;                         // (the partner has read the last one: these scores are there because it handed over the weights before them)
        tc_fence_before();                   // this warp's reads of S end before its partner writes P over columns 32..63 of them
        bar_sync_named((int)pair_bar, 64);
        tc_fence_after();
        mts = fmaxf(mts, *other);
        if (__any_sync(0xffffffffu, mts - m_used > slack)) {      // (the difference: where the maximum is large, 8 more of it may be none, or 16)
          const float m_new = fmaxf(m_used, mts);
          const float alpha = m_new == -INFINITY ? 1.0f : atc_ex2(m_used - m_new);
          l *= alpha;
          if (j > 0u) {
#pragma unroll 1
            for (uint32_t c = 0; c < 4u; c++) {
              uint32_t o[16];
              tmem_ld16(o_addr + 16u * c, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st16(o_addr + 16u * c, o);
            }
          }
          m_used = m_new;
          far = __any_sync(0xffffffffu, qi < p.geo.qpt && cache_far(m_new));      // (rows behind the last query's hold anything)
        }
        float2 ls[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        float nm = m_used == -INFINITY ? 0.0f : lv - m_used;             // (a row that has seen no key yet: all its weights are 0)
        if (far) {                                                        // large scores: see cache_far
          float top = -INFINITY;
#pragma unroll
          for (int c = 0; c < 64; c++) top = fmaxf(top, __uint_as_float(s[c]));
          nm = top == -INFINITY ? 0.0f : *mine - m_used + less;           // (this page's largest, as above; at most slack + less)
          if (top == -INFINITY) top = 0.0f;
#pragma unroll
          for (int c = 0; c < 64; c++) s[c] = __float_as_uint(__uint_as_float(s[c]) - top);
        }
        const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(nm, nm);
#pragma unroll
        for (int c = 0; c < 2; c++) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[32 * c + 2 * e]), __uint_as_float(s[32 * c + 2 * e + 1])), sc2, nm2);
            // (all on the special-function unit: here, where the conversion shares the issue slots, a part of them as polynomials on the FMA pipe, which
            // k_attn_tc.cuh gains from, costs: of 16 pairs 6 260, 148 us; 4 256, 146; 2 254, 140; none 247, 139.6, 2000 tokens over 6100 and four prompts under a window)
            const float2 pr = make_float2(atc_ex2(x.x), atc_ex2(x.y));
            ls[e & 1] = __fadd2_rn(ls[e & 1], pr);
            const __half2 hp = __floats2half2_rn(pr.x, pr.y);
            pk[e] = *reinterpret_cast<const uint32_t*>(&hp);
          }
          tmem_st16(p_addr + 16u * c, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8u * t);
        l = fmaf((ls[0].x + ls[0].y) + (ls[1].x + ls[1].y), pg.z, l);
      }
      bar_sync_named((int)pair_bar, 64);     // (the partner has read the last maximum)
      *mine = l;
      bar_sync_named((int)pair_bar, 64);
      l += *other;
      // ---- the item's end: O / l, or this block's partial result
      if (ok && !mbar_wait(o_full + 8u * t, items & 1u, p.c.status, 631)) ok = false;
      items++;
      tc_fence_after();
      const uint32_t q = t * p.geo.qpt + qi, gt = g.t;                    // the row's query within the block
      const bool live = qi < p.geo.qpt && q < g.n, whole = gt == 0u && cnt == g.units, fine = __all_sync(0xffffffffu, ok);
      const int64_t at_o = live && fine ? (int64_t)(g.r0 + q) * p.ldo + (g.hk * p.geo.group + hh) * 128u + half * 64u : -1;      // the row's half columns in O; -1: not stored
      auto tmem_o = [&](uint32_t c, uint32_t (&o)[32]) {                  // 32 columns
        tmem_ld16(o_addr + 32u * c, *reinterpret_cast<uint32_t(*)[16]>(&o[0]));
        tmem_ld16(o_addr + 32u * c + 16u, *reinterpret_cast<uint32_t(*)[16]>(&o[16]));
        tmem_ld_wait();
      };
      // An item that crosses blocks: each of them leaves (maximum, sum, O) in memory, and the warp that arrives last (of those that have these rows and columns, one in
      // each block) adds them up.  A block has two places: 0 for the item that began before it, 1 for the one that goes on behind it.  Mostly there are two shares, and the
      // first block's, at its end, finds the second's, which that block began with: its own then stays in tensor memory.  Sums of two do not depend on
      // which is whose (both products are rounded); more are all read back and added in block order, or left to k_cache_merge (p.desc).
      bool last = false, two = false;
      uint32_t c0 = blockIdx.x, c1 = c0;
      float m_all = m_used, f = 1.0f, f_other = 0.0f;
      auto part_at = [&](uint32_t b, uint32_t c) { return p.part + ((size_t)(b * 2u + (b == c0 ? 1u : 0u)) * 32u + half * 16u + 8u * c) * 256u + t * 128u + row; };
      auto ml_at = [&](uint32_t b) { return p.part_ml + ((size_t)(b * 2u + (b == c0 ? 1u : 0u)) * 2u + half) * 256u + t * 128u + row; };
      if (!whole && fine) {
        const uint64_t U = (uint64_t)at[6] | (uint64_t)at[7] << 32, u0 = (uint64_t)at[9] | (uint64_t)at[10] << 32, first = u0 + g.spent - gt;      // (the item's unit 0)
        const uint32_t owner = (uint32_t)deal_owner(lane & 1u ? first + g.units - 1u : first, U, at[8]);
        c0 = __shfl_sync(0xffffffffu, owner, 0); c1 = __shfl_sync(0xffffffffu, owner, 1);
        two = c1 == c0 + 1u;
        uint32_t* const arrivals = p.count + c0 * 16u + (warp - 8u);
        uint32_t before = 0u;
        if (two && lane == 0u) asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(before) : "l"(arrivals) : "memory");
        last = __shfl_sync(0xffffffffu, before, 0) == 1u;
        const bool later = !two && p.desc;
        if (!last) {
          *ml_at(blockIdx.x) = make_float2(m_used, l);
#pragma unroll 1
          for (uint32_t c = 0; c < 2u; c++) {
            uint32_t o[32];
            tmem_o(c, o);
            float4* pt = part_at(blockIdx.x, c);
            if (at_o >= 0) {
#pragma unroll
              for (int e = 0; e < 8; e++) pt[e * 256] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
            }
          }
          __syncwarp();
          if (later) {
            if (blockIdx.x == c0 && t == 0u && half == 0u && row == 0u) p.desc[c0] = CacheTcDesc{1u, g.r0, g.n, g.hk, c1};
          } else {
            if (lane == 0u) asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(arrivals) : "memory");
            last = __shfl_sync(0xffffffffu, before, 0) == c1 - c0;
          }
        }
        __syncwarp();
        if (last) {
          if (lane == 0u) *arrivals = 0u;
          if (two) {
            const float2 z = __ldcg(ml_at(blockIdx.x == c0 ? c1 : c0));
            m_all = fmaxf(m_used, z.x);
            f = m_used == -INFINITY ? 0.0f : atc_ex2(m_used - m_all);
            f_other = z.x == -INFINITY ? 0.0f : atc_ex2(z.x - m_all);
            l = __fadd_rn(__fmul_rn(f, l), __fmul_rn(f_other, z.y));
          } else {
            for (uint32_t b = c0; b <= c1; b++) m_all = fmaxf(m_all, __ldcg(ml_at(b)).x);
            l = 0.0f; f = 0.0f;
            for (uint32_t b = c0; b <= c1; b++) { const float2 z = __ldcg(ml_at(b)); l = fmaf(z.x == -INFINITY ? 0.0f : atc_ex2(z.x - m_all), z.y, l); }
          }
        }
      }
      const float inv = l > 0.0f ? 1.0f / l : l;
      const bool vec = ((reinterpret_cast<uintptr_t>(p.O) | ((uintptr_t)p.ldo * 2u)) & 15u) == 0u;
#pragma unroll 1
      for (uint32_t c = 0; c < 2u && (whole || last); c++) {              // 32 columns at a time
        uint32_t o[32];
        tmem_o(c, o);
        if (last) {
#pragma unroll
          for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__fmul_rn(f, __uint_as_float(o[e])));
          for (uint32_t b = c0; b <= c1; b++) {
            if (two && b == blockIdx.x) continue;
            float w = f_other;
            if (!two) { const float zx = __ldcg(ml_at(b)).x; w = zx == -INFINITY ? 0.0f : atc_ex2(zx - m_all); }
            const float4* pt = part_at(b, c);
            if (at_o >= 0) {
#pragma unroll
              for (int e = 0; e < 8; e++) {
                const float4 x = __ldcg(pt + e * 256);
                o[4 * e] = __float_as_uint(__fadd_rn(__uint_as_float(o[4 * e]), __fmul_rn(w, x.x))); o[4 * e + 1] = __float_as_uint(__fadd_rn(__uint_as_float(o[4 * e + 1]), __fmul_rn(w, x.y)));
                o[4 * e + 2] = __float_as_uint(__fadd_rn(__uint_as_float(o[4 * e + 2]), __fmul_rn(w, x.z))); o[4 * e + 3] = __float_as_uint(__fadd_rn(__uint_as_float(o[4 * e + 3]), __fmul_rn(w, x.w)));
              }
            }
          }
        }
        uint32_t v[4][4];                                                 // four pieces of 8 columns
#pragma unroll
        for (int e = 0; e < 16; e++) v[e >> 2][e & 3] = cache_result(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
        if (!vec) {
          if (at_o >= 0) {
#pragma unroll
            for (int e = 0; e < 16; e++) *reinterpret_cast<uint32_t*>(p.O + at_o + 32u * c + 2 * e) = v[e >> 2][e & 3];
          }
          continue;
        }
        // Four lanes swap pieces (a 4 x 4 transposition), so that a store writes 64 consecutive bytes of each of 8 rows: with a row per lane every
        // store touched 32 lines, and nothing else got through to shared memory for 8000 cycles an item.
#pragma unroll
        for (int x = 1; x < 4; x += x) {
          const bool up = (lane & x) != 0u;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            if (i & x) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? v[i][e] : v[i + x][e], x);
              if (up) v[i][e] = got; else v[i + x][e] = got;
            }
          }
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {                                     // this lane's piece of the row of lane r of the four
          const int64_t to = __shfl_sync(0xffffffffu, at_o, (int)((lane & 28u) + r));
          if (to >= 0) *reinterpret_cast<uint4*>(p.O + to + 32u * c + 8u * (lane & 3u)) = make_uint4(v[r][0], v[r][1], v[r][2], v[r][3]);
        }
      }
      tc_fence_before();                     // (the reads of O end before the next item's weights are handed over)
      seg_done(seg);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1u) { tc_fence_after(); tmem_dealloc(tmem_base, 512u); }
}

// ---- items of more than two shares: (maximum, sum, O) of their blocks added up in block order.  A block takes 32 rows of one item's 256.  (8 kv heads, 64 rows over
// 32000 tokens, 18 shares an item: the whole call 49 us; 63 where the block that arrives last reads them all by itself.)
struct CacheMergeP {
  const float4* part; const float2* part_ml; const CacheTcDesc* desc;
  __half* O;
  uint32_t ldo, group, qpt;
};
__global__ void __launch_bounds__(256) k_cache_merge(const CacheMergeP p) {
  __shared__ float tile[32][132];
  grid_dependency_wait();
  grid_launch_dependents();
  const uint32_t c0 = blockIdx.x, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, row = blockIdx.y * 32u + lane;
  const CacheTcDesc d = p.desc[c0];
  if (!d.on) return;
  auto live = [&](uint32_t r) { const uint32_t x = r & 127u, q = (r >> 7) * p.qpt + x / p.group; return x < p.qpt * p.group && q < d.q; };
  if (__syncthreads_or(live(row)) == 0) return;
  auto slab = [&](uint32_t c) { return (size_t)c * 2u + (c == c0 ? 1u : 0u); };
  float M = -INFINITY;
  if (live(row)) for (uint32_t c = c0; c <= d.c1; c++) M = fmaxf(M, p.part_ml[slab(c) * 512u + row].x);
  float L = 0.0f;
  float4 acc[4];
#pragma unroll
  for (int k = 0; k < 4; k++) acc[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (live(row)) {
#pragma unroll 2
    for (uint32_t c = c0; c <= d.c1; c++) {
      const float2 ml = p.part_ml[slab(c) * 512u + row];
      const float f = ml.x == -INFINITY ? 0.0f : atc_ex2(ml.x - M);
      L = fmaf(f, ml.y, L);
#pragma unroll
      for (uint32_t k = 0; k < 4u; k++) {
        const float4 v = p.part[(slab(c) * 32u + warp + 8u * k) * 256u + row];
        acc[k].x = fmaf(f, v.x, acc[k].x); acc[k].y = fmaf(f, v.y, acc[k].y); acc[k].z = fmaf(f, v.z, acc[k].z); acc[k].w = fmaf(f, v.w, acc[k].w);
      }
    }
  }
  const float inv = L > 0.0f ? 1.0f / L : L;
#pragma unroll
  for (uint32_t k = 0; k < 4u; k++) *reinterpret_cast<float4*>(&tile[lane][(warp + 8u * k) * 4u]) = make_float4(acc[k].x * inv, acc[k].y * inv, acc[k].z * inv, acc[k].w * inv);
  __syncthreads();
#pragma unroll
  for (uint32_t k = 0; k < 4u; k++) {
    const uint32_t r = blockIdx.y * 32u + warp * 4u + k;
    if (!live(r)) continue;
    const uint32_t x = r & 127u, q = (r >> 7) * p.qpt + x / p.group, h = d.hk * p.group + x % p.group;
    const float4 v = *reinterpret_cast<const float4*>(&tile[r & 31u][lane * 4u]);
    uint32_t* o = reinterpret_cast<uint32_t*>(p.O + (size_t)(d.row0 + q) * p.ldo + h * 128u + 4u * lane);
    o[0] = cache_result(v.x, v.y); o[1] = cache_result(v.z, v.w);
  }
}

}  // namespace p0p
