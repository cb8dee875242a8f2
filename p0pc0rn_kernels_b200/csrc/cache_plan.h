// The 8-bit key/value cache: where things lie, which tokens a call touches, which pages a query sees, how the work is dealt out, and
// which arguments are refused.  Plain C++ (host and device), so that all of it can be compiled and tested without a GPU.
//
// Pages of 64 tokens.  codes [page][kv head][K | V][8192] u8 (code + 128); scales [page][kv head][K | V] fp32; tail [sequence][kv head]
// [K | V][8192] fp16: the tokens of the last, unfinished page; table [sequence][max_pages] page numbers; lens [sequence] tokens,
// the ones of the present call included: a call's n tokens of a sequence are its last n.
// Within a page (codes and tail alike) the elements lie in the order in which a warp's lanes want them as operands of m16n8k16
// products, 16 elements per lane (lane = 4 g + t):
//   K: groups of 16 keys x 2 blocks of 8 keys x 2 halves of d; lane: key 4 (g / 2) + 2 block + (g & 1) of the group, 16 consecutive d
//   V: blocks of 8 d; lane: d = g of the block, keys 16 j + 4 t + i (j, i = 0 .. 3)
// so that a product's operand is one 16-byte read per lane, without bank conflicts, and the keys that a lane's probabilities
// belong to are the keys of its V elements.
#pragma once
#include <stdint.h>
#include <stdio.h>

#ifdef __CUDACC__
#define P0P_HD __host__ __device__ __forceinline__
#else
#define P0P_HD inline
#endif

namespace p0p {

constexpr uint32_t CACHE_PAGE = 64u, CACHE_BLOCK = CACHE_PAGE * 128u;      // tokens of a page; elements of a page's K or V of one head
constexpr uint32_t CACHE_MAX_SEQS = 1024u;
enum { CACHE_BAD_ROWS = 601, CACHE_BAD_LENS = 602, CACHE_BAD_PAGE = 603 };

P0P_HD uint32_t cache_k_off(uint32_t key, uint32_t d) {
  return ((key >> 4) * 2u + ((key >> 1) & 1u)) * 1024u + (d >> 6) * 512u + (((key & 15u) >> 2) * 2u + (key & 1u)) * 64u + (d & 63u);
}
P0P_HD uint32_t cache_v_off(uint32_t key, uint32_t d) { return d * 64u + ((key >> 2) & 3u) * 16u + (key >> 4) * 4u + (key & 3u); }

struct CacheSeq { uint32_t r0, n, L; };      // first row of the call, its tokens in the call, tokens altogether
// A sequence whose numbers make no sense is treated as one without new tokens, and the code says why.
// row0, row1: the sequence's entries of `rows`.
P0P_HD int cache_seq_check(uint32_t row0, uint32_t row1, uint32_t len, uint32_t M, uint32_t max_pages, CacheSeq& s) {
  s.r0 = row0; s.n = 0u; s.L = len;
  if (row1 < row0 || row1 > M) return CACHE_BAD_ROWS;
  const uint32_t n = row1 - row0;
  if (n == 0u) return 0;
  if (len < n || (uint64_t)len > (uint64_t)max_pages * CACHE_PAGE) return CACHE_BAD_LENS;
  s.n = n;
  return 0;
}
P0P_HD uint32_t cache_first_page(const CacheSeq& s) { return (s.L - s.n) / CACHE_PAGE; }
P0P_HD uint32_t cache_touched(const CacheSeq& s) { return s.n ? (s.L - 1u) / CACHE_PAGE - cache_first_page(s) + 1u : 0u; }
// the most pages that M tokens in `seqs` sequences touch (a sequence's n tokens touch at most n, and at most n / 64 + 2)
P0P_HD uint64_t cache_touched_bound(uint32_t M, uint32_t seqs) {
  const uint64_t b = (uint64_t)M / CACHE_PAGE + 2ull * seqs;
  return b < M ? b : M;
}

// The pages that the sequence's new queries see: the first `sp` pages (they hold the tokens that always stay visible), then pages
// lo .. lo + (np - sp) - 1, of which the last is the sequence's last.  window 0: all.
struct CacheVis { uint32_t sp, lo, np; };
P0P_HD CacheVis cache_visible(const CacheSeq& s, uint32_t window, uint32_t sinks) {
  const uint32_t first = s.L - s.n, pages = s.L / CACHE_PAGE + (s.L % CACHE_PAGE ? 1u : 0u);
  const uint32_t lo_key = window && first >= window ? first - window + 1u : 0u;
  CacheVis v;
  v.lo = lo_key / CACHE_PAGE;
  const uint32_t sp = sinks / CACHE_PAGE + (sinks % CACHE_PAGE ? 1u : 0u);
  v.sp = sp < v.lo ? sp : v.lo;
  v.np = v.sp + pages - v.lo;
  return v;
}
P0P_HD uint32_t cache_vis_page(const CacheVis& v, uint32_t t) { return t < v.sp ? t : v.lo + t - v.sp; }
// is key visible to the query at position p?
P0P_HD bool cache_key_visible(uint32_t key, uint32_t p, uint32_t window, uint32_t sinks) {
  return key <= p && (window == 0u || p - key < window || key < sinks);
}
// Scores are fp32, and a weight's exponent is score * factor - maximum in one multiply-add.  Where the maximum (in powers of two) is larger than this, the
// rounding of that reference would show in the weights (2^-15 here; at 2^28 it is 16, and weights overflow): the page's largest score is taken off first.
P0P_HD bool cache_far(float m) { return m > 1024.0f || (m < -1024.0f && m > -3.0e38f); }      // (-infinity: no key yet)
// may a page's key be hidden from a query at positions p0 .. p1?
P0P_HD bool cache_page_masked(uint32_t page, uint32_t p0, uint32_t p1, uint32_t window, uint32_t sinks) {
  const uint32_t k0 = page * CACHE_PAGE, k1 = k0 + (CACHE_PAGE - 1u);
  return k1 > p0 || (window != 0u && p1 >= k0 && p1 - k0 >= window && k1 >= sinks);
}

// U units of work in a row are dealt out to G workers, G <= U: worker c has units [deal_first(c), deal_first(c + 1)).
P0P_HD uint64_t div_64(uint64_t a, uint64_t b) { return ((a | b) >> 32) ? a / b : (uint32_t)a / (uint32_t)b; }      // (a 64-bit division takes hundreds of cycles)
P0P_HD uint64_t deal_first(uint64_t c, uint64_t U, uint64_t G) { return div_64(c * U, G); }
P0P_HD uint64_t deal_owner(uint64_t u, uint64_t U, uint64_t G) { return div_64((u + 1u) * G - 1u, U); }

// The split-key attention's units: per sequence [kv head][block of 16 query rows][visible page], one sequence after the other.  The query rows of
// the `group` heads that share a kv head are one matrix of n * group rows, query by query.  An item (all pages of a kv head and row block) costs one
// unit before its pages: its queries and page numbers arrive, its result leaves.
struct CacheGeo { uint32_t Hkv, group, seqs, window, sinks; };
P0P_HD uint64_t cache_units(const CacheSeq& s, const CacheGeo& g) {
  return s.n ? (uint64_t)g.Hkv * ((s.n * g.group + 15u) >> 4) * (1u + cache_visible(s, g.window, g.sinks).np) : 0u;
}
// how many blocks share U units of `items` items: all, unless that cuts items that few blocks (of 8 warps) would do.  Where there are fewer items than blocks
// each gets the same number of them, so that items of one length are cut between blocks as little as can be.
P0P_HD uint64_t cache_workers(uint64_t U, uint64_t items, uint64_t most) {
  uint64_t g = most;
  if (items && items <= most) {
    const uint64_t fit = most / items, per = div_64(U, items), want = per / 9u + (per % 9u ? 1u : 0u);      // (an item's cost: a warp's page each, and the unit before them)
    g = items * (want < fit ? want : fit);
  }
  if (g > most) g = most;
  return g > U ? U : g;
}
// where a warp stands.  pre[b]: units before sequence b; seq[b]: the sequences.
struct CacheCursor {
  CacheSeq s; CacheVis v;
  uint32_t b, hk, rb, rbs, at;      // at 0: before the item's first page; at k > 0: at page k - 1
  P0P_HD void sequence(const CacheGeo& g, const CacheSeq* seq, uint32_t b_) {
    b = b_; s = seq[b];
    v = cache_visible(s, g.window, g.sinks);
    rbs = (s.n * g.group + 15u) >> 4;
  }
  P0P_HD void seek(const CacheGeo& g, const uint64_t* pre, const CacheSeq* seq, uint64_t u) {
    uint32_t lo = 0u, hi = g.seqs - 1u;                                   // the first sequence that ends behind u: it is not empty
    while (lo < hi) { const uint32_t mid = (lo + hi) >> 1; if (pre[mid + 1u] > u) hi = mid; else lo = mid + 1u; }
    sequence(g, seq, lo);
    const uint64_t item = div_64(u - pre[lo], v.np + 1u);
    at = (uint32_t)(u - pre[lo] - item * (v.np + 1u));
    hk = (uint32_t)div_64(item, rbs); rb = (uint32_t)(item - (uint64_t)hk * rbs);
  }
  // the beginning of the next item, which there has to be
  P0P_HD void next_item(const CacheGeo& g, const uint64_t* pre, const CacheSeq* seq) {
    at = 0u;
    if (++rb < rbs) return;
    rb = 0u;
    if (++hk < g.Hkv) return;
    hk = 0u;
    uint32_t n = b + 1u;
    while (n + 1u < g.seqs && pre[n + 1u] == pre[n]) n++;
    if (n < g.seqs) sequence(g, seq, n);
  }
  P0P_HD uint32_t t() const { return at ? at - 1u : 0u; }
  P0P_HD bool tail(uint32_t k) const { return cache_vis_page(v, k) == s.L / CACHE_PAGE; }      // is visible page k the unfinished one?
};

// What a block that has units [u0, u1) and gives up still tells the others: tell(x, i0, i1) once for each item whose pages, units [i0, i1), lie in the block only in part
// (x: where it stands).  That is its first unit's item, its last unit's, or neither; both may be the same one.
template <class Tell>
P0P_HD void cache_tell_shares(const CacheGeo& g, const uint64_t* pre, const CacheSeq* seq, uint64_t u0, uint64_t u1, Tell tell) {
  uint64_t told = ~0ull;
  for (uint32_t k = 0; k < 2u; k++) {
    const uint64_t u = k ? u1 - 1u : u0;
    CacheCursor x;
    x.seek(g, pre, seq, u);
    const uint64_t i0 = u - x.at + 1u, i1 = i0 + x.v.np;
    if (i0 == told || i0 >= u1 || (i0 >= u0 && i1 <= u1)) continue;      // (told already; only the unit before its pages is here; all of it is)
    told = i0;
    tell(x, i0, i1);
  }
}

// The tensor-memory attention's work: an item = up to 2 * qpt queries of a sequence (qpt: those whose heads of one kv head fill a tile of 128
// rows) and one kv head, a unit = two visible pages of it.  Per sequence [block of queries][kv head][pair of pages].
struct CacheTcGeo { uint32_t Hkv, group, seqs, window, sinks, qpt, min_rows; };      // sequences with at most min_rows rows per kv head are the other kernel's
P0P_HD uint32_t cache_tc_blocks(const CacheSeq& s, const CacheTcGeo& g) {
  return s.n && (uint64_t)s.n * g.group > g.min_rows ? (s.n - 1u) / (2u * g.qpt) + 1u : 0u;
}
// the queries of block x, as a sequence that ends with them
P0P_HD CacheSeq cache_tc_part(const CacheSeq& s, const CacheTcGeo& g, uint32_t x) {
  CacheSeq p;
  const uint32_t q0 = x * 2u * g.qpt;
  p.r0 = s.r0 + q0; p.n = s.n - q0 < 2u * g.qpt ? s.n - q0 : 2u * g.qpt; p.L = s.L - s.n + q0 + p.n;
  return p;
}
P0P_HD uint32_t cache_tc_units(const CacheSeq& part, const CacheTcGeo& g) { return (cache_visible(part, g.window, g.sinks).np + 1u) / 2u; }
// the key of column c of a page's 64 score columns (the order in which a lane's V elements lie)
P0P_HD constexpr uint32_t cache_col_key(uint32_t c) { return 16u * ((c >> 2) & 3u) + 4u * (c >> 4) + (c & 3u); }
// The work is dealt out by cost: an item costs CACHE_TC_ITEM units (its queries arrive, its result leaves, the pipeline fills) and then its own.
// (Dealt out by units alone, a block at the start of a prompt, with many items of one unit or two, took 1.7 times as long as the others.)
constexpr uint32_t CACHE_TC_ITEM = 2u;
P0P_HD uint32_t cache_tc_cost(const CacheSeq& part, const CacheTcGeo& g) { return CACHE_TC_ITEM + cache_tc_units(part, g); }
// What a block does next: units [t, t + cnt) of an item; cnt 0: nothing more.  One warp of the block walks the list and announces it to the others.  get(b): sequence b.
struct CacheTcWalk {
  CacheSeq s, part; CacheVis v;
  uint32_t b, x, blocks, hk, t, units, cnt, left, spent;      // spent: the cost, from the beginning of the block's share, of unit t
  P0P_HD void item(const CacheTcGeo& g) {
    part = cache_tc_part(s, g, x);
    v = cache_visible(part, g.window, g.sinks);
    units = (v.np + 1u) / 2u;
  }
  // the share begins `at` into item (b_, x_, hk_) and costs left_
  template <class Get>
  P0P_HD void begin(const CacheTcGeo& g, uint32_t b_, uint32_t x_, uint32_t hk_, uint32_t at, uint32_t left_, Get get) {
    b = b_; x = x_; hk = hk_; left = left_; cnt = 0u; spent = 0u; t = 0u;
    if (!left) return;
    s = get(b);
    blocks = cache_tc_blocks(s, g);
    item(g);
    if (at < CACHE_TC_ITEM) enter(CACHE_TC_ITEM - at);
    else { t = at - CACHE_TC_ITEM; cnt = units - t < left ? units - t : left; }
  }
  P0P_HD void enter(uint32_t first) {
    if (left <= first) { left = 0u; cnt = 0u; return; }
    left -= first; spent += first;
    cnt = units < left ? units : left;
  }
  template <class Get>
  P0P_HD void next(const CacheTcGeo& g, Get get) {
    left -= cnt; spent += cnt; t = 0u; cnt = 0u;
    if (!left) return;
    if (++hk == g.Hkv) {
      hk = 0u;
      if (++x == blocks) {
        x = 0u;
        do { b++; s = get(b); blocks = cache_tc_blocks(s, g); } while (b + 1u < g.seqs && blocks == 0u);
      }
      item(g);
    }
    enter(CACHE_TC_ITEM);
  }
  P0P_HD bool two(const CacheTcGeo& g) const { return part.n > g.qpt; }      // both tiles of rows hold queries
};
// how many blocks share a cost of U: four each at least, but no fewer blocks than items.  (8 kv heads, 256 rows over 4000 tokens: at least six 33.2 us, four 28.8,
// three 30.2)
P0P_HD uint64_t cache_tc_workers(uint64_t U, uint64_t items, uint64_t most) {
  uint64_t g = U / 4u > items ? U / 4u : items;
  if (g > most) g = most;
  return g > U ? U : g;
}

// ---- arguments.  Sizes are the bytes from the given offset to the buffer's end (0: no buffer).
struct CacheShape {
  uint32_t Hkv, pages, seqs, max_pages;
  uint64_t codes, scales, tail, table, lens;
  uint64_t codes_off, scales_off, tail_off, table_off, lens_off;
};
inline int cache_shape_check(const char* op, const CacheShape& s, char* msg, size_t cap) {
#define P0P_REFUSE(code, ...) do { snprintf(msg, cap, __VA_ARGS__); return code; } while (0)
  if (!s.Hkv || !s.pages || !s.seqs || !s.max_pages) P0P_REFUSE(-2, "%s: a cache has at least one kv head, page, sequence and table column", op);
  if (s.Hkv > 65535u) P0P_REFUSE(-2, "%s: at most 65535 kv heads", op);
  if (s.seqs > CACHE_MAX_SEQS) P0P_REFUSE(-2, "%s: at most %u sequences", op, CACHE_MAX_SEQS);
  if (s.max_pages > (1u << 26) - 1u) P0P_REFUSE(-2, "%s: at most 2^26 - 1 pages per sequence", op);
  if (!s.codes || !s.scales || !s.tail || !s.table || !s.lens) P0P_REFUSE(-4, "%s: missing binding (codes, scales, tail, table and lens are needed)", op);
  if ((s.codes_off | s.tail_off) & 15u) P0P_REFUSE(-5, "%s: codes / tail offsets must be multiples of 16 bytes", op);
  if ((s.scales_off & 7u) || ((s.table_off | s.lens_off) & 3u)) P0P_REFUSE(-5, "%s: the scales' offset must be a multiple of 8 bytes, table and lens of 4", op);
  const uint64_t blocks = (uint64_t)s.pages * s.Hkv;
  const uint64_t need[5] = {blocks * 16384u, blocks * 8u, (uint64_t)s.seqs * s.Hkv * 32768u, (uint64_t)s.seqs * s.max_pages * 4u, (uint64_t)s.seqs * 4u};
  const uint64_t have[5] = {s.codes, s.scales, s.tail, s.table, s.lens};
  const char* name[5] = {"codes", "scales", "tail", "table", "lens"};
  for (int i = 0; i < 5; i++)
    if (have[i] < need[i]) P0P_REFUSE(-7, "%s: %s needs %llu bytes", op, name[i], (unsigned long long)need[i]);
  return 0;
}
// rows: bytes of the row offsets (`given`: the caller passes some); without them every sequence has M / seqs rows
inline int cache_rows_check(const char* op, uint32_t M, uint32_t seqs, bool given, uint64_t rows, uint64_t rows_off, char* msg, size_t cap) {
  if (!given) {
    if (M % seqs) P0P_REFUSE(-3, "%s: M must be a multiple of seqs where no row offsets are given", op);
    return 0;
  }
  if (rows_off & 3u) P0P_REFUSE(-5, "%s: the row offsets must lie at a multiple of 4 bytes", op);
  if (rows < (seqs + 1ull) * 4u) P0P_REFUSE(-7, "%s: rows needs %llu bytes", op, (seqs + 1ull) * 4u);
  return 0;
}
// a tensor of `heads` heads with `ld` rows of 128 fp16 each, of which M are used
inline int cache_heads_check(const char* op, const char* name, uint32_t heads, uint32_t M, uint32_t ld, uint64_t bytes, uint64_t off, char* msg, size_t cap) {
  if (ld < M) P0P_REFUSE(-5, "%s: %s.ld must be at least M", op, name);
  if (off & 15u) P0P_REFUSE(-5, "%s: the offset of %s must be a multiple of 16 bytes", op, name);
  const uint64_t need = ((uint64_t)(heads - 1u) * ld + M) * 256u;
  if (bytes < need) P0P_REFUSE(-7, "%s: %s needs %llu bytes", op, name, (unsigned long long)need);
  return 0;
}
#undef P0P_REFUSE

}  // namespace p0p
