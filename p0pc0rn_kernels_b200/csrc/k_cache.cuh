// Writing and reading the 8-bit key/value cache (cache_plan.h says what lies where), and rotary positions.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "cache_dev.cuh"
#include "sync.cuh"

namespace p0p {

// Block x of a call's touched pages: the sequence, and which of its touched pages it is.  False: there are fewer.  All 256 threads.
__device__ __forceinline__ bool cache_find_page(const CacheP& p, uint32_t x, uint32_t per_seq, uint32_t& b, uint32_t& local, CacheSeq& s) {
  if (!p.rows) {                                                         // equal counts: as many blocks for every sequence
    b = x / per_seq; local = x - b * per_seq;
    s = cache_seq(p, b);
    return local < cache_touched(s);
  }
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  auto scan = [&](uint32_t inc) {
#pragma unroll
    for (uint32_t o = 1; o < 32u; o <<= 1) { const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += v; }
    return inc;
  };
  if (p.seqs <= 32u) {                                                   // every warp by itself: one look at the sequences, no barrier
    CacheSeq mine{0u, 0u, 0u};
    if (lane < p.seqs) mine = cache_seq(p, lane);
    const uint32_t c = cache_touched(mine), inc = scan(c), hit = __ballot_sync(0xffffffffu, x < inc && x >= inc - c);
    if (!hit) return false;
    b = __ffs(hit) - 1u;
    local = x - __shfl_sync(0xffffffffu, inc - c, b);
    s.r0 = __shfl_sync(0xffffffffu, mine.r0, b); s.n = __shfl_sync(0xffffffffu, mine.n, b); s.L = __shfl_sync(0xffffffffu, mine.L, b);
    return true;
  }
  __shared__ uint32_t warp_sum[8], found[5];
  if (tid == 0u) found[0] = 0xffffffffu;
  uint64_t base = 0u;
  for (uint32_t b0 = 0; b0 < p.seqs; b0 += 256u) {
    CacheSeq mine{0u, 0u, 0u};
    if (b0 + tid < p.seqs) mine = cache_seq(p, b0 + tid);
    const uint32_t c = cache_touched(mine), inc = scan(c);
    if (lane == 31u) warp_sum[warp] = inc;
    __syncthreads();
    uint32_t before = 0u, all = 0u;
#pragma unroll
    for (uint32_t w = 0; w < 8u; w++) { if (w < warp) before += warp_sum[w]; all += warp_sum[w]; }
    const uint64_t first = base + before + inc - c;
    if (c && x >= first && x < first + c) { found[0] = b0 + tid; found[1] = (uint32_t)(x - first); found[2] = mine.r0; found[3] = mine.n; found[4] = mine.L; }
    base += all;
    __syncthreads();
    if (found[0] != 0xffffffffu || x < base) break;
  }
  b = found[0]; local = found[1]; s.r0 = found[2]; s.n = found[3]; s.L = found[4];
  return b != 0xffffffffu;
}

// NaN -> 0, infinities -> the largest finite value
__device__ __forceinline__ uint32_t cache_clean(uint32_t v) {
  const __half2 h = *reinterpret_cast<const __half2*>(&v);
  uint32_t w = v & __heq2_mask(h, h);
  const __half2 most = __halves2half2(__ushort_as_half(0x7bff), __ushort_as_half(0x7bff));
  const __half2 c = __hmax2(__hmin2(*reinterpret_cast<const __half2*>(&w), most), __hneg2(most));
  return *reinterpret_cast<const uint32_t*>(&c);
}

constexpr uint32_t CW_LD = 136u;        // halves per row of the tile that V is turned in: 16-byte rows, and 4 keys further another half of the banks

// A lane's 16 values of one d (keys 16 j + 4 t + i, t = lane % 4; word w: j = w / 2, i = 2 (w % 2) and the next) into the tile [key][d], together with
// the lane of the other d of the pair (lane ^ 4): the even one's lane takes the even keys, so that a store has two d
__device__ __forceinline__ void cache_turn(__half* tile, uint32_t d, uint32_t lane, const uint32_t (&h)[8]) {
  const bool odd = (lane & 4u) != 0u;
#pragma unroll
  for (uint32_t w = 0; w < 8u; w++) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, h[w], 4);
    const uint32_t both = odd ? __byte_perm(other, h[w], 0x7632) : __byte_perm(h[w], other, 0x5410);
    *reinterpret_cast<uint32_t*>(tile + ((w >> 1) * 16u + 4u * (lane & 3u) + 2u * (w & 1u) + (odd ? 1u : 0u)) * CW_LD + (d & ~1u)) = both;
  }
}
__device__ __forceinline__ void cache_bar(uint32_t id) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(id) : "memory"); }      // of the 128 threads of K or V

// New tokens t0 .. t1 - 1 of the unfinished page `pg` (positions) into the tail.  All 256 threads.
__device__ __forceinline__ void cache_append(__half* tk, __half* tv, const __half* K, const __half* V, uint32_t row_of_pos0, uint32_t pg, uint32_t t0, uint32_t t1) {
  for (uint32_t e = threadIdx.x; e < (t1 - t0) * 16u; e += 256u) {
    const uint32_t pos = t0 + (e >> 4), key = pos - pg * CACHE_PAGE, d = (e & 15u) * 8u;
    const size_t src = (size_t)(row_of_pos0 + pos) * 128u + d;
    uint4 a = ld_now(reinterpret_cast<const uint4*>(K + src)), b = ld_now(reinterpret_cast<const uint4*>(V + src));
    a.x = cache_clean(a.x); a.y = cache_clean(a.y); a.z = cache_clean(a.z); a.w = cache_clean(a.w);
    *reinterpret_cast<uint4*>(tk + cache_k_off(key, d)) = a;
    const uint32_t w[4] = {cache_clean(b.x), cache_clean(b.y), cache_clean(b.z), cache_clean(b.w)};
#pragma unroll
    for (uint32_t i = 0; i < 8u; i++) tv[cache_v_off(key, d + i)] = __ushort_as_half((unsigned short)(w[i >> 1] >> (16u * (i & 1u))));
  }
}

// code + 128 of x in the low byte: x * inv + 768 snaps the quotient to multiples of 2^-14, then the second sum rounds it to the
// nearest whole number, ties to even.  x has 11 significant bits and the scale 12, so that x / scale is either exactly half way between
// two codes or at least 2^-13 away from it, while x * inv is off by 2^-17 at most: the snap restores a tie and moves nothing across one.
__device__ __forceinline__ uint32_t cache_code(float x, float inv) { return __float_as_uint(fmaf(x, inv, 768.0f) + (12582912.0f + 128.0f - 768.0f)); }
__device__ __forceinline__ uint32_t cache_pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// A block of zeros gets the smallest scale that any block has: attention weighs a block's values by it, and zeros are to weigh less than any others.
__device__ __forceinline__ float cache_scale(float amax) { return __uint_as_float((__float_as_uint(__fdiv_rn(fmaxf(amax, 0x1p-24f), 127.0f)) + 4095u) & ~4095u); }

// One block = one touched page of one kv head; 128 threads for K, 128 for V, each half by itself.  A page that the call finishes: its tokens (old ones from
// the tail, new ones from the rows) are read with their largest magnitude found on the way; K's codes leave from the registers, 8 per thread and store, V's
// through a tile in shared memory that turns them.  The unfinished last page only takes its new tokens into the tail; where the call
// also finishes a page that began in the tail, that page's block does it, after it has read the tail.
// Bound: HBM for prompts (256 bytes read and 128 written per token, head and K or V), launch latency for steps.  8000 tokens of 8 heads, 49 MB: 15.3 us =
// 3.2 TB/s, 0.49 of the measured copy (126 pages x 8 heads are 1008 blocks, 1.7 rounds of four per SM; five per SM, at 48 registers, are slower by
// 0.3 us).  One token for each of 64 sequences: 4.9 us.  The heads of a page are neighbours in the grid: the pages that began in the tail take longest and
// stand first (with pages as neighbours the last heads' came in the last round, 17.3 us).
__global__ void __launch_bounds__(256, 4) k_cache_write(const CacheP p, const __half* K, const __half* V, uint32_t ldk, uint32_t ldv, uint32_t per_seq) {
  __shared__ __align__(16) __half tile[CACHE_PAGE * CW_LD];
  __shared__ float sm_max[8];
  const uint32_t tid = threadIdx.x, hk = blockIdx.x % p.Hkv;
  grid_dependency_wait();
  grid_launch_dependents();
  uint32_t b, local;
  CacheSeq s;
  if (!cache_find_page(p, blockIdx.x / p.Hkv, per_seq, b, local, s)) return;
  const uint32_t first = cache_first_page(s), old = s.L - s.n, pg = first + local, last = s.L / CACHE_PAGE;
  const uint32_t row0 = s.r0 - old;                                       // (wraps: only sums with positions >= old are rows)
  __half* tk = p.tail + ((size_t)b * p.Hkv + hk) * 2u * CACHE_BLOCK; __half* tv = tk + CACHE_BLOCK;
  const __half* Kh = K + (size_t)hk * ldk * 128u; const __half* Vh = V + (size_t)hk * ldv * 128u;
  const bool began = (old & (CACHE_PAGE - 1u)) != 0u;                     // page `first` has tokens in the tail
  if (pg == last) {                                                       // unfinished
    if (pg == first || !began) cache_append(tk, tv, Kh, Vh, row0, pg, max(old, pg * CACHE_PAGE), s.L);
    return;
  }
  const uint32_t page = ld_now(p.table + (size_t)b * p.max_pages + pg);
  const uint32_t w = tid >> 7, i = tid & 127u, lane = tid & 31u;
  const uint32_t have = pg == first ? old & (CACHE_PAGE - 1u) : 0u;       // keys that are in the tail
  const __half* src = w ? Vh : Kh; const __half* tl = w ? tv : tk;
  uint4 x[8];
#pragma unroll
  for (uint32_t it = 0; it < 8u; it++) {
    const uint32_t key = it * 8u + (i >> 4), d = (i & 15u) * 8u;
    x[it] = make_uint4(0u, 0u, 0u, 0u);
    if (key >= have) x[it] = ld_now(reinterpret_cast<const uint4*>(src + (size_t)(row0 + pg * CACHE_PAGE + key) * 128u + d));
    else if (w == 0u) x[it] = ld_now(reinterpret_cast<const uint4*>(tl + cache_k_off(key, d)));
  }
  __half2 mx = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
  auto largest = [&](uint32_t v) { mx = __hmax2_nan(mx, __habs2(*reinterpret_cast<const __half2*>(&v))); };
  if (w && have) {                                                        // V's old tokens: pieces of 16 keys of one d
#pragma unroll 1
    for (uint32_t it = 0; it < 4u; it++) {
      const uint32_t u = it * 128u + i;
      const uint4 a = ld_now(reinterpret_cast<const uint4*>(tl) + 2u * u), z = ld_now(reinterpret_cast<const uint4*>(tl) + 2u * u + 1u);
      uint32_t h[8] = {a.x, a.y, a.z, a.w, z.x, z.y, z.z, z.w};
#pragma unroll
      for (int k = 0; k < 8; k++) {                                       // (what lies behind them is of another page or of none: new tokens take its place below)
        const int r = (int)have - (int)(4u * (u & 3u)) - 16 * (k >> 1) - 2 * (k & 1);
        h[k] = r >= 2 ? h[k] : r == 1 ? h[k] & 0xffffu : 0u;
        largest(h[k]);
      }
      cache_turn(tile, u >> 2, lane, h);
    }
    cache_bar(2u);
  }
  // (new tokens are cleaned where something is to clean: the largest magnitude says so, a NaN in it stays one)
  const __half2 old_mx = mx;
#pragma unroll
  for (uint32_t it = 0; it < 8u; it++) { largest(x[it].x); largest(x[it].y); largest(x[it].z); largest(x[it].w); }
  if (!(__low2float(mx) + __high2float(mx) <= 131008.0f)) {
    mx = old_mx;
#pragma unroll
    for (uint32_t it = 0; it < 8u; it++) {
      x[it].x = cache_clean(x[it].x); x[it].y = cache_clean(x[it].y); x[it].z = cache_clean(x[it].z); x[it].w = cache_clean(x[it].w);
      largest(x[it].x); largest(x[it].y); largest(x[it].z); largest(x[it].w);
    }
  }
  if (w) {
#pragma unroll
    for (uint32_t it = 0; it < 8u; it++) {
      const uint32_t key = it * 8u + (i >> 4);
      if (key >= have) *reinterpret_cast<uint4*>(tile + key * CW_LD + (i & 15u) * 8u) = x[it];
    }
  }
  float m = fmaxf(__low2float(mx), __high2float(mx));
#pragma unroll
  for (uint32_t o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0u) sm_max[tid >> 5] = m;
  cache_bar(1u + w);
  const float sc = cache_scale(fmaxf(fmaxf(sm_max[w * 4u], sm_max[w * 4u + 1u]), fmaxf(sm_max[w * 4u + 2u], sm_max[w * 4u + 3u]))), inv = __fdiv_rn(1.0f, sc);
  if (page >= p.pages) { if (tid == 0u) cache_tell(p.status, CACHE_BAD_PAGE); }
  else {
    uint8_t* out = p.codes + (((size_t)page * p.Hkv + hk) * 2u + w) * CACHE_BLOCK;
    if (w == 0u) {
#pragma unroll
      for (uint32_t it = 0; it < 8u; it++) {
        uint32_t q[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const uint32_t v0 = k ? x[it].z : x[it].x, v1 = k ? x[it].w : x[it].y;
          const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&v0)), f1 = __half22float2(*reinterpret_cast<const __half2*>(&v1));
          q[k] = cache_pack4(cache_code(f0.x, inv), cache_code(f0.y, inv), cache_code(f1.x, inv), cache_code(f1.y, inv));
        }
        *reinterpret_cast<uint2*>(out + cache_k_off(it * 8u + (i >> 4), (i & 15u) * 8u)) = make_uint2(q[0], q[1]);
      }
    } else {
#pragma unroll
      for (uint32_t it = 0; it < 2u; it++) {                              // two pieces: keys 16 j + 4 t + e of d and of d + 1
        const uint32_t u = it * 128u + i, d = (u >> 2) * 2u, t = u & 3u;
        uint32_t q0[4], q1[4];
#pragma unroll
        for (uint32_t j = 0; j < 4u; j++) {
          uint32_t c0[4], c1[4];
#pragma unroll
          for (uint32_t e = 0; e < 4u; e++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(tile + (16u * j + 4u * t + e) * CW_LD + d));
            c0[e] = cache_code(f.x, inv); c1[e] = cache_code(f.y, inv);
          }
          q0[j] = cache_pack4(c0[0], c0[1], c0[2], c0[3]); q1[j] = cache_pack4(c1[0], c1[1], c1[2], c1[3]);
        }
        reinterpret_cast<uint4*>(out)[d * 4u + t] = make_uint4(q0[0], q0[1], q0[2], q0[3]);
        reinterpret_cast<uint4*>(out)[(d + 1u) * 4u + t] = make_uint4(q1[0], q1[1], q1[2], q1[3]);
      }
    }
    if (i == 0u) reinterpret_cast<float*>(p.scales + (size_t)page * p.Hkv + hk)[w] = sc;
  }
  // (new tokens behind the last finished page: positions last * 64 >= old, since page `first` is finished)
  if (have) {
    __syncthreads();                                                      // (every read of the tail has ended)
    cache_append(tk, tv, Kh, Vh, row0, last, last * CACHE_PAGE, s.L);
  }
}

// ---- read back: one block = one touched page of one kv head, as in k_cache_write.  K's values go straight to their rows (two lanes swap halves, so
// that a store fills whole 32-byte pieces), V's through the tile that turns them.
// (Here pages are neighbours in the grid: no page takes longer, and 352 MB are read in 66.3 us against 67.3 with heads as neighbours.)
// Bound: HBM.  Four sequences of up to 20000 tokens, 8 heads, 352 MB: 65 us = 5.4 TB/s, 0.83 of the measured copy; 8000 tokens, 49 MB: 12.5 us, 0.60 (the
// launch and one round of blocks); 300 tokens: 4.8 us.
__global__ void __launch_bounds__(256, 5) k_cache_read(const CacheP p, __half* K, __half* V, uint32_t ldk, uint32_t ldv, uint32_t per_seq) {
  __shared__ __align__(16) __half tile[CACHE_PAGE * CW_LD];
  const uint32_t tid = threadIdx.x, hk = blockIdx.y, lane = tid & 31u;
  grid_dependency_wait();
  grid_launch_dependents();
  uint32_t b, local;
  CacheSeq s;
  if (!cache_find_page(p, blockIdx.x, per_seq, b, local, s)) return;
  const uint32_t old = s.L - s.n, pg = cache_first_page(s) + local, row0 = s.r0 - old;
  const uint32_t w = tid >> 7, i = tid & 127u;
  const bool whole = pg < s.L / CACHE_PAGE;
  uint32_t page = 0u;
  if (whole) {
    page = ld_now(p.table + (size_t)b * p.max_pages + pg);
    if (page >= p.pages) { if (tid == 0u) cache_tell(p.status, CACHE_BAD_PAGE); return; }
  }
  uint4 c[4];                                                             // four pieces of 16 codes: of one key (K) or of one d (V)
  float sc = 0.0f;
  if (whole) {
    const uint4* in = reinterpret_cast<const uint4*>(p.codes + (((size_t)page * p.Hkv + hk) * 2u + w) * CACHE_BLOCK);
    sc = ld_now(reinterpret_cast<const float*>(p.scales + (size_t)page * p.Hkv + hk) + w);
#pragma unroll
    for (uint32_t it = 0; it < 4u; it++) c[it] = ld_now(in + it * 128u + i);
  }
  const bool big = sc > 515.0f;                                           // a code of 127 times a scale that was rounded up may pass the largest fp16: it stays finite
  auto values = [&](uint32_t it, uint32_t (&h)[8]) {
    if (whole) {
      // a byte under 0x4b0000 is 2^23 + code + 128 (the conversion instruction has a sixteenth of the lanes)
      const uint32_t q[4] = {c[it].x, c[it].y, c[it].z, c[it].w};
      auto value = [&](int k) {
        const float f = (__uint_as_float(__byte_perm(q[k >> 2], 0x4b000000u, 0x7440 + (k & 3))) - 8388736.0f) * sc;
        return big ? fmaxf(fminf(f, 65504.0f), -65504.0f) : f;
      };
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const __half2 r = __floats2half2_rn(value(2 * j), value(2 * j + 1));
        h[j] = *reinterpret_cast<const uint32_t*>(&r);
      }
    } else {
      const uint4* tl = reinterpret_cast<const uint4*>(p.tail + (((size_t)b * p.Hkv + hk) * 2u + w) * CACHE_BLOCK) + 2u * (it * 128u + i);
      const uint4 a = ld_now(tl), z = ld_now(tl + 1u);
      h[0] = a.x; h[1] = a.y; h[2] = a.z; h[3] = a.w; h[4] = z.x; h[5] = z.y; h[6] = z.z; h[7] = z.w;
    }
  };
  if (w == 0u) {
    __half* dst = K + (size_t)hk * ldk * 128u;
#pragma unroll
    for (uint32_t it = 0; it < 4u; it++) {
      uint32_t h[8];
      values(it, h);
      const uint32_t u = it * 128u + i, key = (u >> 7) * 16u + ((u >> 3) & 3u) * 4u + ((u >> 6) & 1u) * 2u + ((u >> 2) & 1u), d = ((u >> 5) & 1u) * 64u + (u & 3u) * 16u, pos = pg * CACHE_PAGE + key;
      const bool odd = (lane & 1u) != 0u;
      uint32_t got[4];
#pragma unroll
      for (int k = 0; k < 4; k++) got[k] = __shfl_xor_sync(0xffffffffu, odd ? h[k] : h[4 + k], 1);      // (the even lane gives its upper half for the odd one's lower)
      const uint4 a = odd ? make_uint4(got[0], got[1], got[2], got[3]) : make_uint4(h[0], h[1], h[2], h[3]);
      const uint4 z = odd ? make_uint4(h[4], h[5], h[6], h[7]) : make_uint4(got[0], got[1], got[2], got[3]);
      if (pos >= old && pos < s.L) {                                      // (both lanes have the same key)
        __half* r = dst + (size_t)(row0 + pos) * 128u + (d & ~16u) + (odd ? 8u : 0u);
        *reinterpret_cast<uint4*>(r) = a; *reinterpret_cast<uint4*>(r + 16u) = z;
      }
    }
    return;
  }
#pragma unroll
  for (uint32_t it = 0; it < 4u; it++) {
    uint32_t h[8];
    values(it, h);
    cache_turn(tile, (it * 128u + i) >> 2, lane, h);
  }
  cache_bar(2u);
  __half* dst = V + (size_t)hk * ldv * 128u;
#pragma unroll
  for (uint32_t it = 0; it < 8u; it++) {
    const uint32_t key = it * 8u + (i >> 4), d = (i & 15u) * 8u, pos = pg * CACHE_PAGE + key;
    if (pos >= old && pos < s.L) *reinterpret_cast<uint4*>(dst + (size_t)(row0 + pos) * 128u + d) = *reinterpret_cast<const uint4*>(tile + key * CW_LD + d);
  }
}

// ---- rotary positions
struct RopeP {
  const __half* X; __half* Y;
  const uint32_t* lens; const uint32_t* rows;
  uint32_t H, M, ldx, ldy, seqs, each, rot, hpt;      // hpt: heads per thread
  float mscale;
  int* status;
  double turn[64];                                    // turns per position of pair i
};

// cos and sin of pair i at a position: the angle in turns is reduced in 64 bits (a fp32 angle of position 10^6 is off by 0.03), what is left
// of it is within half a turn
__device__ __forceinline__ float2 rope_cs(const RopeP& p, uint32_t i, double pos) {
  if (2u * i >= p.rot) return make_float2(1.0f, 0.0f);
  const double t = pos * p.turn[i];
  float sn, cs;
  sincospif(2.0f * (float)(t - rint(t)), &sn, &cs);
  return make_float2(cs * p.mscale, sn * p.mscale);
}
// the position of row r; false for a row of no sequence.  WHOLE: every lane of the warp asks, for one of four rows (lane / 8) from r & ~3 on
template <bool WHOLE>
__device__ __forceinline__ bool rope_pos(const RopeP& p, uint32_t r, double& pos) {
  uint32_t b, r0, r1;
  if (!p.rows) {
    if (r >= p.M) return false;
    b = r / p.each; r0 = b * p.each; r1 = r0 + p.each;
  } else if (WHOLE && p.seqs <= 32u) {                  // one look at the sequences instead of a search
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t from = 0u, to = 0xffffffffu, len = 0u;
    if (lane < p.seqs) { from = ld_now(p.rows + lane); to = ld_now(p.rows + lane + 1u); len = ld_now(p.lens + lane); }
    b = 0u;
#pragma unroll
    for (uint32_t k = 0; k < 4u; k++) { const uint32_t n = __popc(__ballot_sync(0xffffffffu, to <= (r & ~3u) + k)); if ((r & 3u) == k) b = n; }
    r0 = __shfl_sync(0xffffffffu, from, b & 31u); r1 = __shfl_sync(0xffffffffu, to, b & 31u); len = __shfl_sync(0xffffffffu, len, b & 31u);
    if (b >= p.seqs) return false;
    if (r < r0 || r >= r1) { if (b > 0u) cache_tell(p.status, CACHE_BAD_ROWS); return false; }
    CacheSeq s;
    cache_tell(p.status, cache_seq_check(r0, r1, len, p.M, 0xffffffffu, s));
    if (s.n == 0u) return false;
    pos = (double)(s.L - s.n + (r - r0));
    return true;
  } else {
    uint32_t lo = 0u, hi = p.seqs;                    // the first sequence whose end is behind r
    while (lo < hi) { const uint32_t mid = (lo + hi) >> 1; if (ld_now(p.rows + mid + 1u) > r) hi = mid; else lo = mid + 1u; }
    if (lo == p.seqs) return false;
    b = lo; r0 = ld_now(p.rows + b); r1 = ld_now(p.rows + b + 1u);
    if (r < r0) { if (b > 0u) cache_tell(p.status, CACHE_BAD_ROWS); return false; }
  }
  CacheSeq s;
  const int bad = cache_seq_check(r0, r1, ld_now(p.lens + b), p.M, 0xffffffffu, s);
  cache_tell(p.status, bad);
  if (s.n == 0u) return false;
  pos = (double)(s.L - s.n + (r - r0));
  return true;
}
__device__ __forceinline__ void rope_turn(float2 cs, float& a, float& b) { const float x = a, y = b; a = x * cs.x - y * cs.y; b = fmaf(x, cs.y, y * cs.x); }

// 8 threads per row, 16 elements each as two 16-byte pieces; a thread works out its 8 angles once and turns hpt heads with them.
// HALF: pieces l and l + rot / 16 of the row's first part pair up (rot a multiple of 16: a pair of pieces holds pairs of one
// index each); threads whose pieces lie behind the turned part copy.  Otherwise: pieces 2 l and 2 l + 1, pairs within a piece.
// Bound: HBM for prompts (512 bytes per row and head), launch latency for a step.  4145 rows of 40 heads, 85 MB: 19.6 us = 4.3 TB/s, 0.66 of the measured
// copy (the positions, eight sines each reduced in 64 bits, stand before the first store).  One row: 5.2 us.
template <bool HALF>
__global__ void __launch_bounds__(128) k_rope(const RopeP p) {
  const uint32_t l = threadIdx.x & 7u, r = blockIdx.x * 16u + (threadIdx.x >> 3), h0 = blockIdx.y * p.hpt, h1 = min(h0 + p.hpt, p.H);
  grid_dependency_wait();
  grid_launch_dependents();
  const uint32_t q = p.rot >> 4;                       // HALF: pieces per half of the turned part
  uint32_t c0, c1, i0;                                 // the thread's two pieces, its first pair
  if (HALF) {
    if (l < q) { c0 = l; c1 = l + q; i0 = 8u * l; } else { c0 = 2u * q + 2u * (l - q); c1 = c0 + 1u; i0 = 64u; }
  } else { c0 = 2u * l; c1 = c0 + 1u; i0 = 8u * l; }
  auto x_at = [&](uint32_t h) { return reinterpret_cast<const uint4*>(p.X + ((size_t)h * p.ldx + r) * 128u); };
  auto y_at = [&](uint32_t h) { return reinterpret_cast<uint4*>(p.Y + ((size_t)h * p.ldy + r) * 128u); };
  // the first four heads are asked for before the position is known (a row of the call can be read whether or not it is a sequence's)
  uint4 v[4][2];
  auto four = [&](uint32_t h) {
#pragma unroll
    for (uint32_t k = 0; k < 4u; k++)
      if (r < p.M && h + k < h1) { v[k][0] = ld_now(x_at(h + k) + c0); v[k][1] = ld_now(x_at(h + k) + c1); }
  };
  four(h0);
  double pos = 0.0;
  if (!rope_pos<true>(p, r, pos) || r >= p.M) return;
  float2 cs[8];
#pragma unroll
  for (uint32_t i = 0; i < 8u; i++) cs[i] = rope_cs(p, i0 + i, pos);
  auto turned = [&](uint4 (&v)[2]) {
    __half2* e = reinterpret_cast<__half2*>(v);
    if (HALF) {
      if (i0 < 64u) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float2 a = __half22float2(e[i]), b = __half22float2(e[4 + i]);
          rope_turn(cs[2 * i], a.x, b.x); rope_turn(cs[2 * i + 1], a.y, b.y);
          e[i] = __floats2half2_rn(a.x, a.y); e[4 + i] = __floats2half2_rn(b.x, b.y);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        float2 a = __half22float2(e[i]);
        if (2u * (i0 + i) < p.rot) { rope_turn(cs[i], a.x, a.y); e[i] = __floats2half2_rn(a.x, a.y); }
      }
    }
  };
  for (uint32_t h = h0; h < h1; h += 4u) {
    if (h > h0) four(h);
#pragma unroll
    for (uint32_t k = 0; k < 4u; k++)
      if (h + k < h1) { turned(v[k]); y_at(h + k)[c0] = v[k][0]; y_at(h + k)[c1] = v[k][1]; }
  }
}
// the half layout with a part that is no multiple of 16: a warp per row, one pair (or two elements that are copied) per lane and pass
__global__ void __launch_bounds__(128) k_rope_odd(const RopeP p) {
  const uint32_t lane = threadIdx.x & 31u, r = blockIdx.x * 4u + (threadIdx.x >> 5), h0 = blockIdx.y * p.hpt, h1 = min(h0 + p.hpt, p.H);
  grid_dependency_wait();
  grid_launch_dependents();
  if (r >= p.M) return;
  double pos;
  if (!rope_pos<false>(p, r, pos)) return;
  const uint32_t half = p.rot >> 1;
  float2 cs[2]; uint32_t a[2], b[2];
#pragma unroll
  for (uint32_t k = 0; k < 2u; k++) {
    const uint32_t i = k * 32u + lane;
    cs[k] = rope_cs(p, i, pos);
    if (i < half) { a[k] = i; b[k] = i + half; } else { a[k] = 2u * i; b[k] = 2u * i + 1u; }      // (element 2 i >= rot: behind the turned part)
  }
  for (uint32_t h = h0; h < h1; h++) {
    const __half* x = p.X + ((size_t)h * p.ldx + r) * 128u;
    __half* y = p.Y + ((size_t)h * p.ldy + r) * 128u;
    __half u[2], v[2];
#pragma unroll
    for (int k = 0; k < 2; k++) { u[k] = ld_now(x + a[k]); v[k] = ld_now(x + b[k]); }
    __syncwarp();                                      // (y may be x: a row is read before any of it is written)
#pragma unroll
    for (int k = 0; k < 2; k++) {
      if ((uint32_t)k * 32u + lane < half) {
        float f = __half2float(u[k]), g = __half2float(v[k]);
        rope_turn(cs[k], f, g);
        u[k] = __float2half_rn(f); v[k] = __float2half_rn(g);
      }
      y[a[k]] = u[k]; y[b[k]] = v[k];
    }
  }
}

}  // namespace p0p
