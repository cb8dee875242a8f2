// Flash attention, head_dim 128, on the 5th-generation tensor cores (src/ops/attention.js): the same contract as
// k_attn.cuh (Q [Hq][Lq][128], K / V [Hkv][Lk][128] f16 head-major; O [Lq][ldo] token-major; mask modes 0 / 1 / 2; GQA):
//   S = Q K^T   A = Q tile [128 q][128 d] (shared memory),  B = K tile [128 keys][128 d] (shared memory, K-major: d contiguous)
//   O += P V    A = P tile [128 q][128 keys] (tensor memory), B = V tile [128 keys][128 d] (shared memory, MN-major: d, the N of
//               this product, is contiguous).  V is read as it lies; a transposed copy (so that B would be K-major) was a pass of
//               its own over V (32:8 heads, 1000 causal tokens: 26.7 -> 24.6 us a call, this and two softmax threads per row together)
// One block = two tiles of 128 queries of one head that share every K / V tile (or one tile: see attn_plan).  Tensor memory (512 columns x 128 lanes):
// S of tile A | S of tile B | O of tile A | O of tile B, 128 fp32 columns each; lane = query row.  P (fp16, two keys per
// column) is written over the first 64 columns of its S, which is free once the softmax threads hold the row.
// Roles: warp 0 loads tiles by tensor-map copies into a ring of 32-KB slots (K0 V0 K1 V1 ...); warp 1 issues the
// multiplies in the order  PV_A(j) QK_A(j+1) PV_B(j) QK_B(j+1), so that while the softmax of one tile runs the tensor
// cores work on the other; warps 2-9 are the softmax of tile A, warps 10-17 of tile B: two threads per query row, 64 scores each
// in registers; the two tell each other their row maximum (and at the end their sum) through shared memory, and P is handed to
// the multiplies once both have stored their half.  The running maximum is only raised when it grew by more than 2^8: until
// then P is at most 256 (fine in fp16) and O needs no rescaling, which is a pass over tensor memory.  "S(j+1) ready"
// implies "PV(j) done" (a commit covers every earlier multiply), so the softmax threads may rescale O when they hold S.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>
#include <functional>
#include <vector>

#include "attn_tc.cuh"
#include "epilogue.cuh"
#include "sync.cuh"
#include "umma.cuh"

namespace p0p {

struct AttnTcP {
  __half* O;
  uint32_t Lq, Lk, ldo, Hq, Hkv, mode, nvalid;
  uint32_t np, ns;       // per head: np blocks of two query tiles, then ns blocks of one (2 * np + ns = tiles of 128 queries)
  float scale_log2;      // scale * log2(e)
  int* status;           // bounded waits report here
};

#ifndef ATC_SLOTS_N
#define ATC_SLOTS_N 4
#endif
constexpr uint32_t ATC_THREADS = 576u, ATC_SLOTS = ATC_SLOTS_N;
constexpr uint32_t ATC_SMEM = 1024u + (2u + ATC_SLOTS) * ATC_TILE + 256u + 4096u;      // alignment slack + Q tiles + ring + barriers + the half rows' exchange

__global__ void __launch_bounds__(ATC_THREADS, 1) k_attn_tc(const AttnTcP p, const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK,
                                                            const __grid_constant__ CUtensorMap mapV) {
  extern __shared__ unsigned char atc_raw[];
  const uint32_t base = (smem_u32(atc_raw) + 1023u) & ~1023u;
  unsigned char* gbase = atc_raw + (base - smem_u32(atc_raw));
  const uint32_t q_sm = base, kv_sm = base + 2u * ATC_TILE, bars = kv_sm + ATC_SLOTS * ATC_TILE;
  const uint32_t q_full = bars, kv_full = bars + 8u, kv_empty = kv_full + 8u * ATC_SLOTS, s_full = kv_empty + 8u * ATC_SLOTS;
  const uint32_t p_full = s_full + 16u, o_full = p_full + 16u, tmem_slot = o_full + 16u;
  float* xch = reinterpret_cast<float*>(gbase + (bars + 256u - base));
  // (warp index and tensor-memory base through a shuffle: warp-uniform for the compiler, see k_umma.cuh)
  const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u;
  // the grid: first every head's two-tile blocks, then every head's one-tile blocks (the short ones fill the last wave)
  const bool hasB = blockIdx.x < p.Hq * p.np;
  const uint32_t b1 = blockIdx.x - p.Hq * p.np;
  const uint32_t h = hasB ? blockIdx.x / p.np : b1 / p.ns, q0 = hasB ? (blockIdx.x - h * p.np) * 256u : (2u * p.np + (b1 - h * p.ns)) * 128u;
  const uint32_t hk = h / (p.Hq / p.Hkv);
  // keys any row of this block can see, and the key tiles that covers                        (attention.js:64)
  uint32_t kEnd = p.Lk;
  if (p.mode == 1u) kEnd = min(p.Lk, min(q0 + (hasB ? 255u : 127u), p.nvalid - 1u) + 1u);
  if (p.mode == 2u) kEnd = min(p.Lk, p.nvalid);
  const uint32_t nj = (kEnd + 127u) >> 7;

  if (tid == 0) {
    mbar_init(q_full, 1u);
    for (uint32_t s = 0; s < ATC_SLOTS; s++) { mbar_init(kv_full + 8u * s, 1u); mbar_init(kv_empty + 8u * s, 1u); }
    for (uint32_t t = 0; t < 2u; t++) { mbar_init(s_full + 8u * t, 1u); mbar_init(p_full + 8u * t, 8u); mbar_init(o_full + 8u * t, 1u); }
    fence_mbar_init();
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 512u); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t*>(gbase + (tmem_slot - base)), 0);

  // (every role waits for the kernel before, also those that only meet the loads at barriers: the limit of a bounded wait starts when the
  // inputs exist)
  if (warp == 0) {
    // ================================================================= loads
    if (lane == 0) {
      grid_dependency_wait();
      grid_launch_dependents();
      mbar_expect_tx(q_full, hasB ? 2u * ATC_TILE : ATC_TILE);
      for (uint32_t t = 0; t < (hasB ? 2u : 1u); t++)
        for (uint32_t c = 0; c < 2u; c++) tma_load_3d(q_sm + t * ATC_TILE + c * 16384u, &mapQ, (int)(c * 64u), (int)(q0 + t * 128u), (int)h, q_full);
      for (uint32_t i = 0; i < 2u * nj; i++) {
        const uint32_t slot = i % ATC_SLOTS, use = i / ATC_SLOTS, j = i >> 1, dst = kv_sm + slot * ATC_TILE, bar = kv_full + 8u * slot;
        if (use > 0u && !mbar_wait(kv_empty + 8u * slot, (use - 1u) & 1u, p.status, 401, 100u)) break;
        mbar_expect_tx(bar, ATC_TILE);
        if (i & 1u) { for (uint32_t c = 0; c < 2u; c++) tma_load_3d(dst + c * 16384u, &mapV, (int)(c * 64u), (int)(j * 128u), (int)hk, bar); }
        else { for (uint32_t c = 0; c < 2u; c++) tma_load_3d(dst + c * 16384u, &mapK, (int)(c * 64u), (int)(j * 128u), (int)hk, bar); }
      }
    }
  } else if (warp == 1) {
    // ================================================================= multiplies (the whole warp walks the loop, one lane issues)
    const uint32_t idesc = umma_idesc_f16(128u, 128u), idesc_v = idesc | UMMA_B_MN, nt = hasB ? 2u : 1u;
    const uint64_t qd[2] = {umma_desc_sw128(q_sm), umma_desc_sw128(q_sm + ATC_TILE)};
    grid_dependency_wait();
    bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0u, p.status, 402) && mbar_wait(kv_full, 0u, p.status, 403));
    if (ok) {
      tc_fence_after();
      const uint64_t kd = umma_desc_sw128(kv_sm);
      if (elect_one()) {
        for (uint32_t t = 0; t < nt; t++) {
#pragma unroll
          for (uint32_t kk = 0; kk < 8u; kk++) umma_f16_ss(tmem_base + t * 128u, qd[t] + (kk >> 2) * 1024u + 2u * (kk & 3u), kd + (kk >> 2) * 1024u + 2u * (kk & 3u), idesc, kk);
          umma_commit(s_full + 8u * t);
        }
        umma_commit(kv_empty);
      }
      __syncwarp();
    }
    for (uint32_t j = 0; j < nj && ok; j++) {
      const uint32_t iv = 2u * j + 1u, sv = iv % ATC_SLOTS, ik = iv + 1u, sk = ik % ATC_SLOTS;
      const bool more = j + 1u < nj;
      bool rdy = mbar_wait(kv_full + 8u * sv, (iv / ATC_SLOTS) & 1u, p.status, 404);
      if (more) rdy = rdy && mbar_wait(kv_full + 8u * sk, (ik / ATC_SLOTS) & 1u, p.status, 405);
      if (!__all_sync(0xffffffffu, rdy)) { ok = false; break; }
      const uint64_t vd = umma_desc_sw128_mn(kv_sm + sv * ATC_TILE, 16384u), kd = umma_desc_sw128(kv_sm + sk * ATC_TILE);
      for (uint32_t t = 0; t < nt; t++) {
        if (!__all_sync(0xffffffffu, mbar_spin(p_full + 8u * t, j & 1u, p.status, 406))) { ok = false; break; }
        tc_fence_after();
        const uint32_t s_col = tmem_base + t * 128u, o_col = tmem_base + 256u + t * 128u;
        const uint64_t qdt = qd[t];
        if (elect_one()) {
#pragma unroll
          for (uint32_t kk = 0; kk < 8u; kk++) umma_f16_ts(o_col, s_col + 8u * kk, vd + 128u * kk, idesc_v, j | kk);      // 16 keys further: 2048 bytes
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
      }
      __syncwarp();
    }
  } else {
    // ================================================================= softmax of one tile: two threads per query row, 64 keys each
    const uint32_t t = (warp - 2u) >> 3, half = ((warp - 2u) >> 2) & 1u, qd = warp & 3u, row = qd * 32u + lane, i = q0 + t * 128u + row;
    if (t == 0u || hasB) {
      const uint32_t lane_addr = tmem_base + ((qd * 32u) << 16), s_addr = lane_addr + t * 128u + half * 64u, p_addr = lane_addr + t * 128u + half * 32u;
      const uint32_t o_addr = lane_addr + 256u + t * 128u + half * 64u, pair_bar = 1u + t * 4u + qd;
      // [parity of the key tile][tile][half][row]: what this thread tells its partner (row maximum; at the end, row sum)
      float* mine = xch + (t * 2u + half) * 128u + row; const float* other = xch + (t * 2u + (half ^ 1u)) * 128u + row;
      uint32_t limit = p.Lk;                                                                  // keys [0, limit) are visible to this row
      if (p.mode == 1u) limit = min(p.Lk, min(i, p.nvalid - 1u) + 1u);
      if (p.mode == 2u) limit = min(p.Lk, p.nvalid);
      const float sc = p.scale_log2;
      float m_used = -INFINITY, l = 0.0f;
      bool ok = true;
      grid_dependency_wait();
      for (uint32_t j = 0; j < nj; j++) {
        // (a wait that ran out: the thread goes on without it, so that its partner is not left at the barrier; the status word is set)
        if (ok && !mbar_spin(s_full + 8u * t, j & 1u, p.status, 407)) ok = false;
        tc_fence_after();
        uint32_t s[64];
#pragma unroll
        for (int c = 0; c < 4; c++) tmem_ld16(s_addr + 16u * c, *reinterpret_cast<uint32_t(*)[16]>(&s[16 * c]));
        tmem_ld_wait();
        const int rel = (int)limit - (int)(j * 128u + half * 64u);                            // columns [0, rel) of this half are visible
        if (__any_sync(0xffffffffu, rel < 64)) {
#pragma unroll
          for (int c = 0; c < 64; c++) s[c] = c < rel ? s[c] : 0xff800000u;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 64; c += 4) {
          mx[0] = fmaxf(mx[0], __uint_as_float(s[c])); mx[1] = fmaxf(mx[1], __uint_as_float(s[c + 1]));
          mx[2] = fmaxf(mx[2], __uint_as_float(s[c + 2])); mx[3] = fmaxf(mx[3], __uint_as_float(s[c + 3]));
        }
        float mts = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        mine[(j & 1u) * 512u] = mts;
        tc_fence_before();                   // this warp's reads of S end before its partner writes P over columns 32..63 of them
        bar_sync_named((int)pair_bar, 64);
        tc_fence_after();
        mts = fmaxf(mts, other[(j & 1u) * 512u]) * sc;
        if (__any_sync(0xffffffffu, mts > m_used + 8.0f)) {
          // raise the reference maximum of the warp's rows (its partner has the same rows and decides alike); O and l are rescaled to it
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
        }
        float2 ls[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(-m_used, -m_used);
#pragma unroll
        for (int c = 0; c < 2; c++) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const float2 t = __ffma2_rn(make_float2(__uint_as_float(s[32 * c + 2 * e]), __uint_as_float(s[32 * c + 2 * e + 1])), sc2, nm2);
            float2 pr;
            if ((e * ATC_EMU) % 16 < ATC_EMU) pr = atc_ex2_poly2(t);                              // spread evenly over the chunk
            else pr = make_float2(atc_ex2(t.x), atc_ex2(t.y));
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
        l += (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y);
      }
      mine[(nj & 1u) * 512u] = l;
      bar_sync_named((int)pair_bar, 64);
      l += other[(nj & 1u) * 512u];
      // ---- O / l -> global, token-major, head h at column h * 128
      if (ok && mbar_wait(o_full + 8u * t, 0u, p.status, 408)) {
        tc_fence_after();
        const float inv = 1.0f / l;
        __half* dst = p.O + (size_t)i * p.ldo + h * 128u + half * 64u;
        const bool vec = ((reinterpret_cast<uintptr_t>(p.O) | ((uintptr_t)p.ldo * 2u)) & 15u) == 0u;
#pragma unroll 1
        for (uint32_t c = 0; c < 4u; c++) {
          uint32_t o[16], w[8];
          tmem_ld16(o_addr + 16u * c, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const __half2 hp = __floats2half2_rn(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
            w[e] = *reinterpret_cast<const uint32_t*>(&hp);
          }
          if (i < p.Lq) {
            if (vec) {
              *reinterpret_cast<uint4*>(dst + 16u * c) = make_uint4(w[0], w[1], w[2], w[3]);
              *reinterpret_cast<uint4*>(dst + 16u * c + 8u) = make_uint4(w[4], w[5], w[6], w[7]);
            } else {
#pragma unroll
              for (int e = 0; e < 8; e++) *reinterpret_cast<uint32_t*>(dst + 16u * c + 2 * e) = w[e];
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, 512u); }
}

// How a head's T tiles of 128 queries are cut into blocks.  Two-tile blocks are the efficient ones (K / V tiles shared, the
// softmax of one tile hidden behind the multiplies of the other), but blocks are handed to SMs whole: 15 two-tile blocks
// per head x 24 heads on 148 SMs is 2.4 rounds, of which the third is mostly idle.  One-tile blocks cost ATC_SINGLE_COST of a
// two-tile block (nothing overlaps their softmax: 28 key tiles, 148 heads, 54.6 us against 64.3 in a short run; 50.8 against 72.6, 0.70, in a
// long one, where the power limit slows the denser blocks) and fill that last round.  (24 heads x 3600: 1 to 7 one-tile blocks per
// head within 0.5 % of one another in long runs, 9 are 14 % slower.)  The plan simulates the hardware's in-order hand-out for every split and keeps
// the shortest; cost of a block = its key tiles (they differ under the causal mask).
constexpr double ATC_SINGLE_COST = 0.85;
inline void attn_plan(uint32_t Lq, uint32_t Lk, uint32_t Hq, uint32_t mode, uint32_t nvalid, uint32_t sms, uint32_t& np, uint32_t& ns) {
  const uint32_t T = (Lq + 127u) / 128u;
  np = T / 2u; ns = T & 1u;
  if ((uint64_t)Hq * T > 64ull * sms || sms == 0u) return;         // many rounds: the last one hardly matters
  // the answer depends on these seven numbers only, and a model asks for the same ones call after call
  struct Key { uint32_t v[6]; uint32_t np, ns; };
  static thread_local Key memo = {{0, 0, 0, 0, 0, 0}, 0, 0};
  const uint32_t key[6] = {Lq, Lk, Hq, mode, nvalid, sms};
  if (std::equal(key, key + 6, memo.v)) { np = memo.np; ns = memo.ns; return; }
  auto keys = [&](uint32_t q_last) { uint32_t e = Lk; if (mode == 1u) e = std::min(Lk, std::min(q_last, nvalid - 1u) + 1u); if (mode == 2u) e = std::min(Lk, nvalid); return (e + 127u) / 128u; };
  double best = 1e300;
  std::vector<double> heap(sms);
  for (uint32_t s = T & 1u; s <= T && s <= (T & 1u) + 16u; s += 2u) {
    const uint32_t n2 = (T - s) / 2u;
    std::fill(heap.begin(), heap.end(), 0.0);                       // min-heap of the SMs' finish times (all equal: already a heap)
    auto give = [&](double cost) { std::pop_heap(heap.begin(), heap.end(), std::greater<double>()); heap.back() += cost; std::push_heap(heap.begin(), heap.end(), std::greater<double>()); };
    for (uint32_t h = 0; h < Hq; h++) for (uint32_t i = 0; i < n2; i++) give((double)keys(i * 256u + 255u));
    for (uint32_t h = 0; h < Hq; h++) for (uint32_t i = 0; i < s; i++) give(ATC_SINGLE_COST * keys((2u * n2 + i) * 128u + 127u));
    const double span = *std::max_element(heap.begin(), heap.end());
    if (span < best * 0.995) { best = span; np = n2; ns = s; }
  }
  std::copy(key, key + 6, memo.v); memo.np = np; memo.ns = ns;
}

}  // namespace p0p
