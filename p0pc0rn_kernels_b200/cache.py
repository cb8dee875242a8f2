"""The 8-bit key/value cache and what works on it.  No counterpart in the reference: the step between a language model's `heads` projections
and the attention over everything that came before.

  kvCache           the buffers of one layer's cache (page table and lengths may be shared between layers)
  rope              rotary positions of the newest tokens' heads, from positions that live on the device
  cacheWrite        the newest tokens' keys and values into the cache: finished pages of 64 tokens as 8-bit codes, the rest in an fp16 tail
  cacheRead         the inverse: the newest tokens as fp16 keys and values
  cacheAttention    causal attention of the newest tokens over the cache, with or without a sliding window and first tokens that stay visible

A cache is a dict: {Hkv, pages, seqs, maxPages, codes: {buf, off}, scales, tail, table, lens}.  `lens` (u32 per sequence) counts the tokens of
the present call too, `table` (u32 [seqs][maxPages]) names the page that holds tokens 64 i .. 64 i + 63.  The program fills both, for
instance with gpu.upload(..., dst=...); they are read on the device when a call runs, so one recording serves every step.  The newest tokens of all sequences
are consecutive rows; `rows` ({buf, off}: u32 [seqs + 1]) says where each sequence's begin, without it every sequence has M / seqs.
include/p0p.h has the layouts, the arithmetic and what is refused.
"""
from __future__ import annotations

import struct

from ._lib import lib

PAGE = 64
_SPLIT, _TMEM = 24, 25
# The argument blocks of include/p0p.h, packed: a decoding step makes these calls for every layer, and filling a ctypes structure takes longer than the call
_CACHE = "4I 5Q 5Q"
_MOVE = struct.Struct("@4I" + _CACHE + "3Q 3Q")
_ATTN = struct.Struct("@8I f I" + _CACHE + "3Q 3Q")
_ROPE = struct.Struct("@8I 6d 4Q 4Q")


def _h(t) -> int:
    if not t: return 0
    h = t["buf"].handle
    return (h.value or 0) if h is not None else 0


def _o(t) -> int:
    return t.get("off") or 0 if t else 0


def _cache(c) -> tuple:
    k, s, t, p, n = c["codes"], c["scales"], c["tail"], c["table"], c["lens"]
    return c["Hkv"], c["pages"], c["seqs"], c["maxPages"], _h(k), _h(s), _h(t), _h(p), _h(n), _o(k), _o(s), _o(t), _o(p), _o(n)


def cacheBytes(pages: int, Hkv: int, seqs: int, maxPages: int) -> dict:
    """bytes of each buffer of a cache"""
    return {"codes": pages * Hkv * 2 * PAGE * 128, "scales": pages * Hkv * 8, "tail": seqs * Hkv * 2 * PAGE * 256, "table": seqs * maxPages * 4, "lens": seqs * 4}


def kvCache(gpu, a: dict) -> dict:
    """a: {Hkv, pages, seqs, maxPages, table?, lens?}: the buffers of one layer's cache, zeroed.  `table` and `lens` of another layer's cache
    can be passed to share them.  The buffers are freed with gpu.free."""
    n = cacheBytes(a["pages"], a["Hkv"], a["seqs"], a["maxPages"])
    c = {k: a[k] for k in ("Hkv", "pages", "seqs", "maxPages")}
    made = []
    try:
        for k in ("codes", "scales", "tail", "table", "lens"):
            if not a.get(k): made.append(gpu.buffer(n[k], "cache " + k))
            c[k] = a.get(k) or {"buf": made[-1], "off": 0}
    except Exception:
        for b in made: gpu.free(b)           # (no room for a later one: none is left behind)
        raise
    return c


def _pack(op, layout, *values) -> bytes:
    try:
        return layout.pack(*values)
    except struct.error as e:                # a negative or fractional number, or one that no 32 (64) bits hold
        raise ValueError(f"{op}: bad argument ({e})") from None


def _move(op, fn, gpu, a):
    k, v, rows = a["k"], a["v"], a.get("rows")
    gpu._check(fn(gpu._h, _pack(op, _MOVE, _MOVE.size, a["M"], k.get("ld") or 0, v.get("ld") or 0, *_cache(a["cache"]), _h(k), _h(v), _h(rows), _o(k), _o(v), _o(rows))))


def cacheWrite(gpu, a: dict) -> None:
    """a: {cache, k: {buf, off, ld}, v, M, rows?}: k / v [Hkv][ld][128] f16 (ld rows per head, default M): the M newest tokens"""
    _move("cacheWrite", lib.p0p_cache_write, gpu, a)


def cacheRead(gpu, a: dict) -> None:
    """a: {cache, k: {buf, off, ld}, v, M, rows?}: writes to k / v, [Hkv][ld][128] f16, the last tokens of each sequence as the cache holds them"""
    _move("cacheRead", lib.p0p_cache_read, gpu, a)


def cacheAttention(gpu, a: dict) -> None:
    """a: {cache, q: {buf, off, ld}, o: {buf, off, ld}, Hq, M, rows?, new?, window?, sinks?, scale?}: q [Hq][ld][128] f16, o [M][ld] f16 token-major at
    column h * 128.  cacheWrite of the same tokens comes first.  A query sees the keys up to its own; with `window`, the last `window` of
    them and the first `sinks` tokens.  `new`: the most new tokens any sequence has, where the program knows it.  `kernel`
    ('split' | 'tmem', for tests) forces one of the two kernels."""
    q, o, rows = a["q"], a["o"], a.get("rows")
    kernel = a.get("kernel")
    if kernel not in (None, "split", "tmem"):
        raise ValueError("cacheAttention: unknown kernel " + str(kernel))
    gpu._check(lib.p0p_cache_attention(gpu._h, _pack("cacheAttention", _ATTN, _ATTN.size, a["Hq"], a["M"], q.get("ld") or 0, o.get("ld") or 0, a.get("new") or 0, a.get("window") or 0, a.get("sinks") or 0,
                                                     a.get("scale") or 0.0, 0 if kernel is None else _SPLIT if kernel == "split" else _TMEM, *_cache(a["cache"]), _h(q), _h(o), _h(rows),
                                                     _o(q), _o(o), _o(rows))))


def rope(gpu, a: dict) -> None:
    """a: {x: {buf, off, ld}, y? (default x), H, M, seqs, lens: {buf, off}, rows?, mode: 'interleaved' | 'half', rot (default 128), theta, factor,
    original, fast, slow, mscale}: turns the first `rot` elements of H heads of the M newest tokens by their positions"""
    x, y, lens, rows, mode, rot = a["x"], a.get("y"), a["lens"], a.get("rows"), a.get("mode"), a.get("rot")
    if mode not in (None, "interleaved", "half"):
        raise ValueError("rope: unknown mode " + str(mode))
    gpu._check(lib.p0p_rope(gpu._h, _pack("rope", _ROPE, _ROPE.size, a["H"], a["M"], x.get("ld") or 0, (y.get("ld") or 0) if y else 0, a["seqs"], 1 if mode == "half" else 0, 128 if rot is None else rot,
                                          a.get("theta") or 0.0, a.get("factor") or 0.0, a.get("original") or 0.0, a.get("fast") or 0.0, a.get("slow") or 0.0, a.get("mscale") or 0.0,
                                          _h(x), _h(y), _h(lens), _h(rows), _o(x), _o(y), _o(lens), _o(rows))))
