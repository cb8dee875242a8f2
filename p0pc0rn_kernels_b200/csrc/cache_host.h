// What the entry points of the 8-bit cache share on the host: bindings checked and resolved to pointers.
#pragma once
#include "ctx.h"
#include "cache_dev.cuh"

namespace p0p {

inline bool cache_live(p0p_ctx* c, const p0p_buf* b) { return b && c->bufs.count(const_cast<p0p_buf*>(b)); }
// bytes of a binding from `off` on; 0 where there is none
inline uint64_t cache_room(p0p_ctx* c, const p0p_buf* b, uint64_t off) { return cache_live(c, b) && off < b->size ? b->size - off : 0u; }
template <class T> inline T* cache_at(const p0p_buf* b, uint64_t off) { return reinterpret_cast<T*>(static_cast<char*>(b->ptr) + off); }
inline int cache_refuse(p0p_ctx* c, int rc, const char* msg) { return rc ? fail(c, rc, "%s", msg) : 0; }

inline int cache_bind(p0p_ctx* c, const char* op, const p0p_cache& a, uint32_t M, const p0p_buf* rows, uint64_t rows_off, CacheP& p) {
  char msg[256];
  const CacheShape s{a.Hkv, a.pages, a.seqs, a.max_pages, cache_room(c, a.codes, a.codes_off), cache_room(c, a.scales, a.scales_off), cache_room(c, a.tail, a.tail_off),
                     cache_room(c, a.table, a.table_off), cache_room(c, a.lens, a.lens_off), a.codes_off, a.scales_off, a.tail_off, a.table_off, a.lens_off};
  if (int rc = cache_shape_check(op, s, msg, sizeof msg)) return cache_refuse(c, rc, msg);
  if (int rc = cache_rows_check(op, M, a.seqs, rows != nullptr, cache_room(c, rows, rows_off), rows_off, msg, sizeof msg)) return cache_refuse(c, rc, msg);
  p.codes = cache_at<uint8_t>(a.codes, a.codes_off); p.scales = cache_at<float2>(a.scales, a.scales_off); p.tail = cache_at<__half>(a.tail, a.tail_off);
  p.table = cache_at<const uint32_t>(a.table, a.table_off); p.lens = cache_at<const uint32_t>(a.lens, a.lens_off);
  p.rows = rows ? cache_at<const uint32_t>(rows, rows_off) : nullptr;
  p.Hkv = a.Hkv; p.pages = a.pages; p.seqs = a.seqs; p.max_pages = a.max_pages; p.M = M; p.each = rows ? 0u : M / a.seqs; p.status = c->dev_status;
  // (what is read with 16-byte loads: foreign memory that was wrapped may begin anywhere)
  if ((reinterpret_cast<uintptr_t>(p.codes) | reinterpret_cast<uintptr_t>(p.tail)) & 15u) return fail(c, -5, "%s: codes and tail must lie at multiples of 16 bytes", op);
  if ((reinterpret_cast<uintptr_t>(p.scales) & 7u) || ((reinterpret_cast<uintptr_t>(p.table) | reinterpret_cast<uintptr_t>(p.lens) | reinterpret_cast<uintptr_t>(p.rows)) & 3u))
    return fail(c, -5, "%s: scales must lie at a multiple of 8 bytes, table, lens and rows of 4", op);
  return 0;
}
// an operand of `heads` heads
inline int cache_heads(p0p_ctx* c, const char* op, const char* name, const p0p_buf* b, uint64_t off, uint32_t heads, uint32_t M, uint32_t ld, __half*& out) {
  char msg[256];
  if (!cache_live(c, b)) return fail(c, -4, "%s: missing binding (%s)", op, name);
  if (int rc = cache_heads_check(op, name, heads, M, ld, cache_room(c, b, off), off, msg, sizeof msg)) return cache_refuse(c, rc, msg);
  out = cache_at<__half>(b, off);
  if (reinterpret_cast<uintptr_t>(out) & 15u) return fail(c, -5, "%s: %s must lie at a multiple of 16 bytes", op, name);
  return 0;
}

}  // namespace p0p
