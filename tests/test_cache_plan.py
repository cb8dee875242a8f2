"""The arithmetic of the 8-bit cache (csrc/cache_plan.h): orders within a page, touched and visible pages, how attention's work is dealt out,
numbers and arguments that are refused.  Plain C++: compiled and run here without a GPU, with the address sanitizer."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdlib>
#include <cstring>
#include <vector>
#include "cache_plan.h"
using namespace p0p;
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); exit(1); } } while (0)
static uint32_t rnd(uint32_t n) { static uint64_t x = 88172645463325252ull; x ^= x << 13; x ^= x >> 7; x ^= x << 17; return (uint32_t)((x >> 11) % n); }

int main() {
  {   // both orders are permutations of a page
    std::vector<int> k(CACHE_BLOCK, 0), v(CACHE_BLOCK, 0);
    for (uint32_t key = 0; key < 64; key++) for (uint32_t d = 0; d < 128; d++) { k[cache_k_off(key, d)]++; v[cache_v_off(key, d)]++; }
    for (uint32_t i = 0; i < CACHE_BLOCK; i++) CHECK(k[i] == 1 && v[i] == 1);
    // a lane's 16 elements: K 16 consecutive d of one key, V keys 16 j + 4 t + i of one d
    CHECK(cache_k_off(5, 33) == cache_k_off(5, 32) + 1 && cache_k_off(5, 47) == cache_k_off(5, 32) + 15);
    CHECK(cache_v_off(16 + 4, 9) == cache_v_off(4, 9) + 4 && cache_v_off(7, 9) == cache_v_off(4, 9) + 3);
  }
  {   // numbers that make no sense leave a sequence without new tokens
    CacheSeq s;
    CHECK(cache_seq_check(3, 2, 10, 10, 4, s) == CACHE_BAD_ROWS && s.n == 0);
    CHECK(cache_seq_check(3, 11, 10, 10, 4, s) == CACHE_BAD_ROWS && s.n == 0);
    CHECK(cache_seq_check(3, 8, 4, 10, 4, s) == CACHE_BAD_LENS && s.n == 0);
    CHECK(cache_seq_check(3, 8, 257, 10, 4, s) == CACHE_BAD_LENS && s.n == 0);
    CHECK(cache_seq_check(3, 3, 0xffffffffu, 10, 4, s) == 0 && s.n == 0);
    CHECK(cache_seq_check(3, 8, 256, 10, 4, s) == 0 && s.n == 5 && s.r0 == 3 && s.L == 256);
    CHECK(cache_seq_check(0, 5, 0xffffffffu, 10, (1u << 26) - 1u, s) == CACHE_BAD_LENS);
  }
  for (int it = 0; it < 4000; it++) {   // touched pages and their bound
    const uint32_t seqs = 1 + rnd(8);
    uint32_t M = 0; uint64_t all = 0;
    for (uint32_t b = 0; b < seqs; b++) {
      CacheSeq s{M, rnd(4) ? rnd(5) : rnd(300), 0};
      s.L = s.n + rnd(300);
      M += s.n;
      uint32_t want = 0;
      for (uint32_t pg = 0; pg < 20; pg++) { bool t = false; for (uint32_t p = s.L - s.n; p < s.L; p++) t |= p / 64 == pg; want += t; if (t) CHECK(pg >= cache_first_page(s) && pg < cache_first_page(s) + cache_touched(s)); }
      CHECK(cache_touched(s) == want);
      if (s.n) CHECK(want <= cache_touched_bound(s.n, 1));
      all += want;
    }
    CHECK(all <= cache_touched_bound(M, seqs));
  }
  for (int it = 0; it < 4000; it++) {   // visible pages: all that any new query sees, none twice, the last one last
    CacheSeq s{0, 1 + rnd(rnd(2) ? 4 : 200), 0};
    s.L = s.n + rnd(900);
    const uint32_t window = rnd(3) ? 1 + rnd(rnd(2) ? 10 : 500) : 0, sinks = rnd(2) ? rnd(rnd(2) ? 5 : 300) : 0;
    const CacheVis v = cache_visible(s, window, window ? sinks : 0);
    std::vector<int> listed(40, 0);
    CHECK(v.np > 0 && cache_vis_page(v, v.np - 1) == (s.L - 1) / 64);
    for (uint32_t t = 0; t < v.np; t++) { const uint32_t pg = cache_vis_page(v, t); CHECK(pg < 40 && pg <= (s.L - 1) / 64); listed[pg]++; if (t) CHECK(pg > cache_vis_page(v, t - 1)); }
    for (uint32_t pg = 0; pg <= (s.L - 1) / 64; pg++) {
      bool seen = false, hidden = false;
      for (uint32_t p = s.L - s.n; p < s.L; p++) for (uint32_t k = pg * 64; k < pg * 64 + 64; k++) {
        const bool want = k <= p && (!window || k + window > p || k < sinks);
        CHECK(cache_key_visible(k, p, window, sinks) == want);
        if (want) seen = true; else hidden = true;
      }
      CHECK(!seen || listed[pg] == 1);
      if (hidden && listed[pg]) CHECK(cache_page_masked(pg, s.L - s.n, s.L - 1, window, sinks));
    }
  }
  for (int it = 0; it < 600; it++) {   // the units: every worker's items and pages, and whom a unit belongs to
    const uint32_t seqs = 1 + rnd(rnd(2) ? 3 : 40);
    const CacheGeo g{1 + rnd(9), 1 + rnd(20), seqs, rnd(2) ? 1 + rnd(300) : 0, rnd(70)};
    std::vector<CacheSeq> seq(seqs);
    std::vector<uint64_t> pre(seqs + 1, 0);
    uint64_t U = 0, pages = 0;
    struct Unit { uint32_t b, hk, rb, at; };
    std::vector<Unit> all;
    for (uint32_t b = 0; b < seqs; b++) {
      seq[b] = CacheSeq{0, rnd(3) ? rnd(3) : rnd(40), 0};
      seq[b].L = seq[b].n + rnd(400);
      U += cache_units(seq[b], g); pre[b + 1] = U;
      if (!seq[b].n) continue;
      const uint32_t np = cache_visible(seq[b], g.window, g.sinks).np;
      for (uint32_t h = 0; h < g.Hkv; h++) for (uint32_t rb = 0; rb * 16 < seq[b].n * g.group; rb++) { pages += np; for (uint32_t t = 0; t <= np; t++) all.push_back({b, h, rb, t}); }
    }
    CHECK(U == all.size());
    if (!U) continue;
    uint64_t items = 0, seen = 0;
    for (const Unit& y : all) items += y.at == 0;
    const uint64_t G = cache_workers(U, items, 148);
    CHECK(G >= 1 && G <= U && G <= 148);
    CHECK(deal_first(0, U, G) == 0 && deal_first(G, U, G) == U);
    for (uint64_t c = 0; c < G; c++) {
      const uint64_t u0 = deal_first(c, U, G), u1 = deal_first(c + 1, U, G), n = u1 - u0, W = n < 8 ? n : 8;
      CHECK(n > 0);
      for (uint64_t u = u0; u < u1; u++) CHECK(deal_owner(u, U, G) == c);
      for (uint64_t w = 0; w < W; w++) {
        const uint64_t w0 = u0 + deal_first(w, n, W), w1 = u0 + deal_first(w + 1, n, W);
        CHECK(w1 > w0);
        CacheCursor x;
        x.seek(g, pre.data(), seq.data(), w0);
        for (uint64_t u = w0; u < w1;) {                  // as the kernel walks: item by item
          const Unit& y = all[u];
          CHECK(x.b == y.b && x.hk == y.hk && x.rb == y.rb && x.at == y.at);
          const uint64_t end = u + (x.v.np + 1 - x.at) < w1 ? u + (x.v.np + 1 - x.at) : w1;
          const uint32_t first = x.t(), cnt = (uint32_t)(end - u) - (x.at ? 0 : 1);
          for (uint32_t k = first; k < first + cnt; k++, seen++) {
            const Unit& z = all[u + (x.at ? 0 : 1) + (k - first)];
            CHECK(z.b == x.b && z.hk == x.hk && z.rb == x.rb && z.at == k + 1 && cache_vis_page(x.v, k) <= (x.s.L - 1) / 64);
            CHECK(x.tail(k) == (x.s.L % 64 != 0 && k + 1 == x.v.np));
          }
          u = end;
          if (u < w1) x.next_item(g, pre.data(), seq.data());
        }
      }
    }
    CHECK(seen == pages);
  }
  {   // score columns: every key of a page once, in the order of a lane's V elements
    std::vector<int> seen(64, 0);
    for (uint32_t c = 0; c < 64; c++) { seen[cache_col_key(c)]++; CHECK(cache_v_off(cache_col_key(c), 0) == c); }
    for (int x : seen) CHECK(x == 1);
  }
  for (int it = 0; it < 1500; it++) {   // the tensor-memory kernel's units: every block's walk
    const uint32_t seqs = 1 + rnd(rnd(2) ? 3 : 40), group = 1 + rnd(rnd(2) ? 8 : 128);
    const CacheTcGeo g{1 + rnd(5), group, seqs, rnd(2) ? 1 + rnd(300) : 0, rnd(70), 128 / group, rnd(2) ? rnd(100) : 0};
    std::vector<CacheSeq> seq(seqs);
    struct Cost { uint32_t b, x, hk, at, units; };
    std::vector<Cost> all;
    uint64_t items = 0, work = 0, done = 0;
    for (uint32_t b = 0; b < seqs; b++) {
      seq[b] = CacheSeq{0, rnd(3) ? rnd(3) : rnd(200), 0};
      seq[b].L = seq[b].n + rnd(900);
      if ((uint64_t)seq[b].n * group <= g.min_rows) continue;
      for (uint32_t q0 = 0, x = 0; q0 < seq[b].n; q0 += 2 * g.qpt, x++) {
        const CacheSeq part = cache_tc_part(seq[b], g, x);
        CHECK(part.r0 == seq[b].r0 + q0 && part.n == (seq[b].n - q0 < 2 * g.qpt ? seq[b].n - q0 : 2 * g.qpt) && part.L - part.n == seq[b].L - seq[b].n + q0);
        const uint32_t np = cache_visible(part, g.window, g.sinks).np, units = (np + 1) / 2;
        CHECK(cache_tc_units(part, g) == units && cache_tc_cost(part, g) == CACHE_TC_ITEM + units && (part.n <= g.qpt || part.n * group <= 2 * 128));
        for (uint32_t h = 0; h < g.Hkv; h++) { items++; work += units; for (uint32_t c = 0; c < CACHE_TC_ITEM + units; c++) all.push_back({b, x, h, c, units}); }
      }
    }
    const uint64_t U = all.size();
    if (!U) continue;
    const uint64_t G = cache_tc_workers(U, items, 148);
    CHECK(G >= 1 && G <= U && G <= 148);
    const auto get = [&](uint32_t b) { CHECK(b < seqs); return seq[b]; };
    for (uint64_t c = 0; c < G; c++) {
      const uint64_t u0 = deal_first(c, U, G), u1 = deal_first(c + 1, U, G);
      CacheTcWalk w;
      for (w.begin(g, all[u0].b, all[u0].x, all[u0].hk, all[u0].at, (uint32_t)(u1 - u0), get); w.cnt; w.next(g, get)) {
        const uint64_t u = u0 + w.spent;                  // the cost of unit t lies here
        CHECK(u + w.cnt <= u1 && w.t + w.cnt <= w.units);
        for (uint32_t k = 0; k < w.cnt; k++, done++) CHECK(all[u + k].b == w.b && all[u + k].x == w.x && all[u + k].hk == w.hk && all[u + k].at == CACHE_TC_ITEM + w.t + k && all[u + k].units == w.units);
        if (w.t + w.cnt < w.units) {                      // goes on in the next block, which begins with it; the last block of it is the owner of its last unit
          CHECK(u + w.cnt == u1);
          CHECK(deal_owner(u + (w.units - 1 - w.t), U, G) > c);
        }
        if (w.t > 0) CHECK(u == u0);
      }
    }
    CHECK(done == work);
  }
  {   // refusals
    char msg[256];
    CacheShape ok{8, 10, 4, 5, 10 * 8 * 16384, 10 * 8 * 8, 4 * 8 * 32768, 4 * 5 * 4, 16, 0, 0, 0, 0, 0};
    CHECK(cache_shape_check("x", ok, msg, sizeof msg) == 0);
    CacheShape s;
#define BAD(field, value, rc, text) do { s = ok; s.field = value; CHECK(cache_shape_check("x", s, msg, sizeof msg) == rc); CHECK(strstr(msg, text)); } while (0)
    BAD(Hkv, 0, -2, "at least one"); BAD(pages, 0, -2, "at least one"); BAD(seqs, 0, -2, "at least one"); BAD(max_pages, 0, -2, "at least one");
    BAD(Hkv, 65536, -2, "65535"); BAD(seqs, 1025, -2, "1024"); BAD(max_pages, 1u << 26, -2, "2^26");
    BAD(codes, 0, -4, "missing"); BAD(lens, 0, -4, "missing");
    BAD(codes_off, 8, -5, "16 bytes"); BAD(tail_off, 4, -5, "16 bytes"); BAD(scales_off, 4, -5, "8 bytes"); BAD(table_off, 2, -5, "of 4"); BAD(lens_off, 1, -5, "of 4");
    BAD(codes, ok.codes - 1, -7, "codes needs"); BAD(scales, ok.scales - 1, -7, "scales needs"); BAD(tail, ok.tail - 1, -7, "tail needs"); BAD(table, ok.table - 1, -7, "table needs");
    BAD(lens, ok.lens - 1, -7, "lens needs"); BAD(pages, 11, -7, "codes needs"); BAD(pages, 0xffffffffu, -7, "codes needs");
    CHECK(cache_rows_check("x", 12, 4, false, 0, 0, msg, sizeof msg) == 0 && cache_rows_check("x", 13, 4, false, 0, 0, msg, sizeof msg) == -3);
    CHECK(cache_rows_check("x", 13, 4, true, 20, 0, msg, sizeof msg) == 0 && cache_rows_check("x", 13, 4, true, 19, 0, msg, sizeof msg) == -7 && cache_rows_check("x", 13, 4, true, 20, 2, msg, sizeof msg) == -5);
    CHECK(cache_heads_check("x", "k", 3, 5, 7, 19 * 256, 0, msg, sizeof msg) == 0 && cache_heads_check("x", "k", 3, 5, 7, 19 * 256 - 1, 0, msg, sizeof msg) == -7);
    CHECK(cache_heads_check("x", "k", 3, 5, 4, 1 << 20, 0, msg, sizeof msg) == -5 && cache_heads_check("x", "k", 3, 5, 5, 1 << 20, 8, msg, sizeof msg) == -5);
  }
  printf("fine\n");
  return 0;
}
"""


def test_cache_plan(tmp_path):
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "p0pc0rn_kernels_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


def test_code_rounding_is_exact(tmp_path):
    """the two-step rounding of cacheWrite (fused multiply by the reciprocal plus 768, then plus a constant), for every fp16 magnitude under a sweep of
    scales: equal to the quotient in 64 bits rounded to the nearest, ties to even; and no code exceeds 127"""
    src, exe = tmp_path / "code.cpp", tmp_path / "code"
    src.write_text(r"""
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
static float h2f(uint32_t h) { const int e = (h >> 10) & 31, m = h & 1023; return e ? std::ldexp((float)(1024 + m), e - 25) : std::ldexp((float)m, -24); }
static uint32_t bits(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
int main() {
  for (uint32_t a = 1; a < 0x7c00; a += a < 2048 ? 1 : 37) {
    const float amax = h2f(a);
    uint32_t b = (bits(amax / 127.0f) + 4095u) & ~4095u; float s; memcpy(&s, &b, 4);
    int e; const double fr = std::frexp((double)amax / 127.0, &e), up = std::ldexp(std::ceil(fr * 4096.0), e - 12);
    if ((double)s != up) { printf("scale %a %a\n", (double)s, up); return 1; }
    const float inv = 1.0f / s;
    for (uint32_t x = 0; x <= a; x += x + 3000 < a && x > 2048 ? 11 : 1) {
      const float f = h2f(x);
      volatile float t = fmaf(f, inv, 768.0f);
      volatile float r = t + (12582912.0f + 128.0f - 768.0f);
      const int got = (int)(bits(r) & 255u) - 128;
      const double want = std::nearbyint((double)f / (double)s);
      if ((double)got != want || got > 127) { printf("%a / %a: %d, %g\n", (double)f, (double)s, got, want); return 1; }
      volatile float tn = fmaf(-f, inv, 768.0f);
      volatile float rn = tn + (12582912.0f + 128.0f - 768.0f);
      if ((int)(bits(rn) & 255u) - 128 != -got) { printf("sign\n"); return 1; }
    }
  }
  printf("fine\n");
}
""")
    subprocess.run(["g++", "-O2", "-mfma", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


def test_argument_blocks_match_the_header(tmp_path):
    """the packed argument blocks have the header's sizes, and every field the header's place"""
    import struct

    from p0pc0rn_kernels_b200 import cache
    in_cache = ["cache." + f for f in "Hkv pages seqs max_pages codes scales tail table lens codes_off scales_off tail_off table_off lens_off".split()]
    blocks = {"p0p_cache_args": (cache._MOVE, ["struct_size", "M", "ldk", "ldv", *in_cache, "k", "v", "rows", "k_off", "v_off", "rows_off"]),
              "p0p_cache_attn_args": (cache._ATTN, ["struct_size", "Hq", "M", "ldq", "ldo", "max_new", "window", "sinks", "scale", "kernel", *in_cache, "q", "o", "rows", "q_off", "o_off", "rows_off"]),
              "p0p_rope_args": (cache._ROPE, "struct_size H M ldx ldy seqs mode rot theta factor original fast slow mscale x y lens rows x_off y_off lens_off rows_off".split())}
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    lines = "".join(f'printf("%zu\\n", sizeof({n}));' + "".join(f'printf("%zu\\n", offsetof({n}, {f}));' for f in fields) for n, (_, fields) in blocks.items())
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "p0p.h"\nint main(void){' + lines + "return 0;}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for layout, fields in blocks.values():
        want.append(layout.size)
        zero = [0.0 if c in "fd" else 0 for c in _codes(layout.format)]
        for i, c in enumerate(_codes(layout.format)):                      # where a value put into field i shows up first
            raw = layout.pack(*zero[:i], -1.0 if c in "fd" else 255, *zero[i + 1:])
            at = next(k for k, b in enumerate(raw) if b)
            want.append(at - at % struct.calcsize(c))
        assert len(fields) == len(zero)
    assert got == want


def _codes(fmt):
    """a struct format as one letter per value"""
    import re
    return "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([IQfd])", fmt))


def test_bad_numbers_are_refused_before_the_call():
    import p0pc0rn_kernels_b200 as P
    import pytest

    class Gpu:
        _h = _check = None
    for bad in (-1, 1 << 32, 1.5):
        with pytest.raises(ValueError, match="rope: bad argument"):
            P.rope(Gpu(), {"x": {"buf": type("B", (), {"handle": None})()}, "H": 1, "M": bad, "seqs": 1, "lens": None})
    with pytest.raises(ValueError, match="unknown mode"):
        P.rope(Gpu(), {"x": {}, "H": 1, "M": 1, "seqs": 1, "lens": None, "mode": "both"})
    with pytest.raises(ValueError, match="unknown kernel"):
        P.cacheAttention(Gpu(), {"q": {}, "o": {}, "kernel": "warp"})


TOLD = r"""
#include <cstdlib>
#include <map>
#include <vector>
#include "cache_plan.h"
using namespace p0p;
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); exit(1); } } while (0)
static uint32_t rnd(uint32_t n) { static uint64_t x = 88172645463325252ull; x ^= x << 13; x ^= x >> 7; x ^= x << 17; return (uint32_t)((x >> 11) % n); }

int main() {
  uint64_t both = 0;
  for (int it = 0; it < 2000; it++) {
    const uint32_t seqs = 1 + rnd(rnd(2) ? 2 : 20), most = rnd(2) ? 148 : 1 + rnd(20);
    const CacheGeo g{1 + rnd(4), 1 + rnd(20), seqs, rnd(2) ? 1 + rnd(300) : 0, rnd(70)};
    std::vector<CacheSeq> seq(seqs);
    std::vector<uint64_t> pre(seqs + 1, 0);
    uint64_t U = 0, items = 0;
    struct Item { uint64_t i0, i1; uint32_t b, hk, rb; };
    std::vector<Item> all;
    for (uint32_t b = 0; b < seqs; b++) {
      seq[b] = CacheSeq{0, rnd(3) ? rnd(3) : rnd(40), 0};
      seq[b].L = seq[b].n + rnd(rnd(2) ? 400 : 9000);
      if (seq[b].n) {
        const uint32_t np = cache_visible(seq[b], g.window, g.sinks).np;
        uint64_t u = U;
        for (uint32_t h = 0; h < g.Hkv; h++) for (uint32_t rb = 0; rb * 16 < seq[b].n * g.group; rb++, u += np + 1, items++) all.push_back({u + 1, u + 1 + np, b, h, rb});
      }
      U += cache_units(seq[b], g); pre[b + 1] = U;
    }
    if (!U) continue;
    const uint64_t G = cache_workers(U, items, most);
    std::map<uint64_t, std::vector<uint64_t>> told;      // an item's first page -> the blocks that told
    for (uint64_t c = 0; c < G; c++)
      cache_tell_shares(g, pre.data(), seq.data(), deal_first(c, U, G), deal_first(c + 1, U, G), [&](const CacheCursor& x, uint64_t i0, uint64_t i1) {
        bool known = false;
        for (const Item& y : all) if (y.i0 == i0) { known = true; CHECK(y.i1 == i1 && y.b == x.b && y.hk == x.hk && y.rb == x.rb); }
        CHECK(known);
        told[i0].push_back(c);
      });
    for (const Item& y : all) {                          // every block that has a page of an item that crosses blocks, once
      const uint64_t c0 = deal_owner(y.i0, U, G), c1 = deal_owner(y.i1 - 1, U, G);
      std::vector<uint64_t> want;
      if (c0 != c1) for (uint64_t c = c0; c <= c1; c++) want.push_back(c);
      CHECK(told[y.i0] == want);
      if (c0 != c1 && (deal_first(c0, U, G) == y.i0 || deal_first(c0, U, G) + 1 == y.i0)) both++;
    }
  }
  CHECK(both > 100);                                     // (blocks that are a share of one item, which begins with them)
  printf("fine\n");
  return 0;
}
"""


def test_a_block_that_gives_up_tells_each_item_once(tmp_path):
    src, exe = tmp_path / "told.cpp", tmp_path / "told"
    src.write_text(TOLD)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "p0pc0rn_kernels_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


def test_a_cache_that_does_not_fit_leaves_no_buffers_behind():
    import p0pc0rn_kernels_b200 as P
    import pytest

    class Gpu:
        def __init__(self, room): self.room, self.held = room, []

        def buffer(self, size, label=""):
            if len(self.held) == self.room: raise P.GpuError("no room")
            self.held.append(label)
            return label

        def free(self, b): self.held.remove(b)
    a = {"Hkv": 1, "pages": 2, "seqs": 1, "maxPages": 2}
    for room in range(5):
        g = Gpu(room)
        with pytest.raises(P.GpuError, match="no room"): P.kvCache(g, a)
        assert g.held == []
    g = Gpu(5)
    c = P.kvCache(g, a)
    assert [c[k]["buf"] for k in ("codes", "scales", "tail", "table", "lens")] == g.held and len(g.held) == 5
    g = Gpu(2)                                            # (a shared table and lengths are another cache's)
    with pytest.raises(P.GpuError, match="no room"): P.kvCache(g, {**a, "table": {"buf": "t"}, "lens": {"buf": "l"}})
    assert g.held == []
    g = Gpu(3)
    assert P.kvCache(g, {**a, "table": {"buf": "t"}, "lens": {"buf": "l"}})["lens"] == {"buf": "l"}


SHARES = r"""
#include <cstdlib>
#include <vector>
#include "cache_plan.h"
using namespace p0p;
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); exit(1); } } while (0)
// the longest run of one item's pages in a warp's share (split keys, 148 blocks of 8 warps)
static uint32_t split_run(uint32_t Hkv, uint32_t group, std::vector<CacheSeq> seq, uint32_t window, uint32_t sinks) {
  const CacheGeo g{Hkv, group, (uint32_t)seq.size(), window, sinks};
  std::vector<uint64_t> pre(seq.size() + 1, 0);
  uint64_t U = 0, items = 0;
  for (size_t b = 0; b < seq.size(); b++) { U += cache_units(seq[b], g); pre[b + 1] = U; items += (uint64_t)Hkv * ((seq[b].n * group + 15) / 16); }
  const uint64_t G = cache_workers(U, items, 148);
  uint32_t most = 0;
  for (uint64_t c = 0; c < G; c++) {
    const uint64_t u0 = deal_first(c, U, G), n = deal_first(c + 1, U, G) - u0, W = n < 8 ? n : 8;
    for (uint64_t w = 0; w < W; w++) {
      const uint64_t w0 = u0 + deal_first(w, n, W), w1 = u0 + deal_first(w + 1, n, W);
      CacheCursor x;
      x.seek(g, pre.data(), seq.data(), w0);
      for (uint64_t u = w0; u < w1;) {
        const uint64_t end = u + (x.v.np + 1 - x.at) < w1 ? u + (x.v.np + 1 - x.at) : w1;
        const uint32_t cnt = (uint32_t)(end - u) - (x.at ? 0 : 1);
        if (cnt > most) most = cnt;
        u = end;
        if (u < w1) x.next_item(g, pre.data(), seq.data());
      }
    }
  }
  return most;
}
// the longest run of one item's pairs of pages in a block's share (tensor memory)
static uint32_t tc_run(uint32_t Hkv, uint32_t group, std::vector<CacheSeq> seq, uint32_t window, uint32_t sinks) {
  const CacheTcGeo g{Hkv, group, (uint32_t)seq.size(), window, sinks, 128 / group, 0};
  struct At { uint32_t b, x, hk, at; };
  std::vector<At> all;
  uint64_t items = 0;
  for (uint32_t b = 0; b < seq.size(); b++)
    for (uint32_t x = 0; x < cache_tc_blocks(seq[b], g); x++)
      for (uint32_t h = 0; h < Hkv; h++) { items++; const uint32_t n = cache_tc_cost(cache_tc_part(seq[b], g, x), g); for (uint32_t c = 0; c < n; c++) all.push_back({b, x, h, c}); }
  const uint64_t U = all.size(), G = cache_tc_workers(U, items, 148);
  uint32_t most = 0;
  for (uint64_t c = 0; c < G; c++) {
    const uint64_t u0 = deal_first(c, U, G), u1 = deal_first(c + 1, U, G);
    CacheTcWalk w;
    const auto get = [&](uint32_t b) { return seq[b]; };
    for (w.begin(g, all[u0].b, all[u0].x, all[u0].hk, all[u0].at, (uint32_t)(u1 - u0), get); w.cnt; w.next(g, get)) if (w.cnt > most) most = w.cnt;
  }
  return most;
}
static CacheSeq s(uint32_t r0, uint32_t n, uint32_t L) { return CacheSeq{r0, n, L}; }
int main() {
  // (the kernels take an item's page numbers and scales 32 pages at a time)
  const uint32_t a = split_run(8, 16, {s(0, 310, 400), s(310, 12, 20000), s(322, 20, 37)}, 0, 0), b = tc_run(8, 4, {s(0, 1100, 8000)}, 0, 0), c = split_run(4, 16, {s(0, 700, 9000)}, 0, 0);
  printf("%u %u %u\n", a, b, c);
  CHECK(a > 32 && b > 32 && c > 64);
  printf("fine\n");
  return 0;
}
"""


def test_the_long_cases_hand_over_page_numbers(tmp_path):
    """cases of test_cache_gpu.py whose shares of one item are longer than the 32 pages that are looked up at a time"""
    src, exe = tmp_path / "shares.cpp", tmp_path / "shares"
    src.write_text(SHARES)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "p0pc0rn_kernels_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr
