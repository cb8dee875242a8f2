// p0p_cache_write, p0p_cache_read, p0p_rope: host entries.
#include <algorithm>
#include <cmath>

#include "cache_host.h"
#include "k_cache.cuh"

using namespace p0p;

namespace {

template <class Kern, class T>
int cache_move(p0p_ctx* c, const char* op, const p0p_cache_args* a, Kern kern, bool heads_first, T*) {
  P0P_ALIVE(c);
  if (!a || a->struct_size < sizeof(p0p_cache_args)) return fail(c, -1, "%s: bad argument block", op);
  CacheP p{};
  if (int rc = cache_bind(c, op, a->cache, a->M, a->rows, a->rows_off, p)) return rc;
  const uint32_t M = a->M, ldk = a->ldk ? a->ldk : M, ldv = a->ldv ? a->ldv : M;
  if (!M) return 0;
  __half *k, *v;
  if (int rc = cache_heads(c, op, "k", a->k, a->k_off, p.Hkv, M, ldk, k)) return rc;
  if (int rc = cache_heads(c, op, "v", a->v, a->v_off, p.Hkv, M, ldv, v)) return rc;
  const uint64_t per = p.rows ? 0u : cache_touched_bound(p.each, 1u), blocks = p.rows ? cache_touched_bound(M, p.seqs) : per * p.seqs;
  if (blocks * p.Hkv > 0x7fffffffu) return fail(c, -5, "%s: too many rows for one call", op);
  DeviceGuard g(c->device);
  const cudaError_t e = launch_chained(kern, heads_first ? dim3((uint32_t)blocks * p.Hkv) : dim3((uint32_t)blocks, p.Hkv), dim3(256), 0, c->stream, p, (T*)k, (T*)v, ldk, ldv, (uint32_t)per);
  if (e != cudaSuccess) return cuda_fail(c, e, op);
  c->launches += 1;
  return 0;
}

}  // namespace

extern "C" int p0p_cache_write(p0p_ctx* c, const p0p_cache_args* a) { return cache_move(c, "cacheWrite", a, k_cache_write, true, (const __half*)nullptr); }
extern "C" int p0p_cache_read(p0p_ctx* c, const p0p_cache_args* a) { return cache_move(c, "cacheRead", a, k_cache_read, false, (__half*)nullptr); }

extern "C" int p0p_rope(p0p_ctx* c, const p0p_rope_args* a) {
  P0P_ALIVE(c);
  if (!a || a->struct_size < sizeof(p0p_rope_args)) return fail(c, -1, "rope: bad argument block");
  if (!a->seqs || a->seqs > CACHE_MAX_SEQS) return fail(c, -2, "rope: 1 to %u sequences", CACHE_MAX_SEQS);
  if (a->mode > 1u) return fail(c, -2, "rope: unknown mode %u", a->mode);
  if ((a->rot & 1u) || a->rot > 128u) return fail(c, -2, "rope: rot must be even and at most 128");
  if (a->H > 65535u) return fail(c, -2, "rope: at most 65535 heads");
  const double theta = a->theta != 0.0 ? a->theta : 10000.0, factor = a->factor != 0.0 ? a->factor : 1.0, fast = a->fast != 0.0 ? a->fast : 32.0, slow = a->slow != 0.0 ? a->slow : 1.0,
               mscale = a->mscale != 0.0 ? a->mscale : 1.0;
  if (!(theta > 0.0) || !std::isfinite(theta) || !(factor > 0.0) || !std::isfinite(factor) || !(a->original >= 0.0) || !std::isfinite(a->original) || !(fast > slow) || !std::isfinite(fast) ||
      !(slow >= 0.0) || !std::isfinite((float)mscale))
    return fail(c, -2, "rope: theta and factor must be positive, original at least 0, fast above slow, mscale within fp32");
  const uint32_t M = a->M, ldx = a->ldx ? a->ldx : M, ldy = a->ldy ? a->ldy : (a->y ? M : ldx);
  char msg[256];
  if (int rc = cache_rows_check("rope", M, a->seqs, a->rows != nullptr, cache_room(c, a->rows, a->rows_off), a->rows_off, msg, sizeof msg)) return cache_refuse(c, rc, msg);
  if (!cache_live(c, a->lens)) return fail(c, -4, "rope: missing binding (lens)");
  if (a->lens_off & 3u) return fail(c, -5, "rope: lens must lie at a multiple of 4 bytes");
  if (cache_room(c, a->lens, a->lens_off) < a->seqs * 4ull) return fail(c, -7, "rope: lens needs %llu bytes", a->seqs * 4ull);
  if (!M || !a->H) return 0;
  __half *x, *y;
  if (int rc = cache_heads(c, "rope", "x", a->x, a->x_off, a->H, M, ldx, x)) return rc;
  if (a->y) { if (int rc = cache_heads(c, "rope", "y", a->y, a->y_off, a->H, M, ldy, y)) return rc; }
  else if (ldy != ldx) return fail(c, -5, "rope: y.ld without y");
  else y = x;
  RopeP p{};
  p.X = x; p.Y = y; p.lens = cache_at<const uint32_t>(a->lens, a->lens_off); p.rows = a->rows ? cache_at<const uint32_t>(a->rows, a->rows_off) : nullptr;
  if ((reinterpret_cast<uintptr_t>(p.lens) | reinterpret_cast<uintptr_t>(p.rows)) & 3u) return fail(c, -5, "rope: lens and rows must lie at multiples of 4 bytes");
  p.H = a->H; p.M = M; p.ldx = ldx; p.ldy = ldy; p.seqs = a->seqs; p.each = p.rows ? 0u : M / a->seqs; p.rot = a->rot; p.mscale = (float)mscale; p.status = c->dev_status;
  const double pi2 = 6.283185307179586476925286766559;
  for (uint32_t i = 0; 2u * i < a->rot; i++) {
    double f = std::pow(theta, -2.0 * i / a->rot);
    if (factor != 1.0) {
      const double g = a->original > 0.0 ? std::min(1.0, std::max(0.0, (a->original * f / pi2 - slow) / (fast - slow))) : 0.0;
      f *= g + (1.0 - g) / factor;
    }
    p.turn[i] = f / pi2;
    if (!(p.turn[i] <= 0x1p990)) return fail(c, -2, "rope: theta or factor too small: the angle of a far position (2^32) has to be a finite number");
  }
  const bool odd = a->mode == 1u && (a->rot & 15u);
  const uint32_t rows_per_block = odd ? 4u : 16u, gx = (M + rows_per_block - 1u) / rows_per_block;
  // heads per thread: the angles are worked out once per thread, so as many as leave one round of blocks (7 of 128 threads fit an SM).  (5 sequences, 4145
  // tokens, 40 heads: eight heads each, a round and a quarter, 21.5 us; so 19.6)
  const uint32_t gy = (uint32_t)std::min<uint64_t>(p.H, std::max<uint64_t>(1u, 7ull * (uint32_t)c->prop.multiProcessorCount / gx));
  p.hpt = (p.H + gy - 1u) / gy;
  DeviceGuard g(c->device);
  const cudaError_t e = launch_chained(odd ? k_rope_odd : a->mode == 1u ? k_rope<true> : k_rope<false>, dim3(gx, (p.H + p.hpt - 1u) / p.hpt), dim3(128), 0, c->stream, p);
  if (e != cudaSuccess) return cuda_fail(c, e, "rope");
  c->launches += 1;
  return 0;
}
