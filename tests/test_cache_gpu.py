"""The 8-bit key/value cache, attention over it and rotary positions, against the definitions in 64 bits.

Tolerances.  Codes, scales and what is read back are exact.  Attention: a weight is rounded to fp16 (half a step, 2^-11, relative; below fp16's
normal range 2^-25 of the largest weight), its exponential is off by less than 1e-4, the result is rounded to fp16 (2^-11).  Weights that are
off by d each move the weighted mean by at most d * 2 max|v|, so |error| <= max|v| * (2 * (2^-11 + 1e-4) + 2^-11 + keys * 2^-25).  Rotary
positions: one rounding to fp16 (2^-11 of the result, 2^-25 where it is subnormal) and four in fp32 (2^-24 of |a| + |b| each)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
PAGE = 64


def _clean(x):
    x = np.where(np.isnan(x), np.float16(0), x)
    return np.clip(x, np.float16(-65504), np.float16(65504)).astype(np.float16)


def _quantise(x):
    """64 x 128 values -> (codes, scale), from the definition in 64 bits"""
    x = x.astype(np.float64); a = np.abs(x).max()
    if a == 0: return np.zeros_like(x), 1.0
    m, e = np.frexp(a / 127.0)
    s = float(np.ldexp(np.ceil(m * 4096.0), e - 12))
    return np.rint(x / s), s


def _offsets():
    key, d = np.arange(PAGE)[:, None], np.arange(128)[None]
    k = ((key >> 4) * 2 + ((key >> 1) & 1)) * 1024 + (d >> 6) * 512 + (((key & 15) >> 2) * 2 + (key & 1)) * 64 + (d & 63)
    v = d * 64 + ((key >> 2) & 3) * 16 + (key >> 4) * 4 + (key & 3)
    return k, v


class Cache:
    """a cache on the GPU and what it should hold"""

    def __init__(self, P, gpu, Hkv, seqs, maxPages, spare=3, seed=0, pages=None, first_page=0):
        self.P, self.gpu, self.Hkv, self.seqs, self.maxp = P, gpu, Hkv, seqs, maxPages
        rng = np.random.default_rng(seed)
        self.pages = pages or seqs * maxPages + spare
        self.table = (first_page + rng.permutation(self.pages - first_page)[:seqs * maxPages]).reshape(seqs, maxPages).astype(np.uint32)
        self.d = P.kvCache(gpu, {"Hkv": Hkv, "pages": self.pages, "seqs": seqs, "maxPages": maxPages})
        self.poison()
        gpu.upload(self.table, dst=self.d["table"]["buf"])
        self.lens = np.zeros(seqs, np.uint32)
        self.tok = [(np.zeros((Hkv, 0, 128), np.float16),) * 2 for _ in range(seqs)]      # every token, as written

    def poison(self):
        """what nobody has written yet: codes of any kind with a scale that is no number, a tail of NaN"""
        n = self.P.cacheBytes(self.pages, self.Hkv, self.seqs, self.maxp)
        if n["codes"] < 1 << 28: self.gpu.upload(np.full(n["codes"], 0xA5, np.uint8), dst=self.d["codes"]["buf"])
        self.gpu.upload(np.full(n["scales"] // 4, np.nan, np.float32), dst=self.d["scales"]["buf"])
        self.gpu.upload(np.full(n["tail"] // 2, 0x7E01, np.uint16), dst=self.d["tail"]["buf"])

    def free(self):
        for k in ("codes", "scales", "tail", "table", "lens"): self.gpu.free(self.d[k]["buf"])

    def advance(self, news):
        self.lens = self.lens + np.asarray(news, np.uint32)
        self.gpu.upload(self.lens, dst=self.d["lens"]["buf"])

    def write(self, news, k, v, rows=True, ld=None, extra=0):
        """k / v: lists per sequence of [Hkv][n][128] fp16"""
        M = int(sum(news)) + extra; ld = ld or M
        bufs, offs = [], np.concatenate([[0], np.cumsum(news)]).astype(np.uint32)
        for x in (k, v):
            t = np.full((self.Hkv, ld, 128), 0x7E01, np.uint16).view(np.float16)
            for b, xb in enumerate(x): t[:, offs[b]:offs[b + 1]] = xb
            bufs.append(self.gpu.upload(t))
        self.advance(news)
        rb = self.gpu.upload(offs) if rows else None
        self.P.cacheWrite(self.gpu, {"cache": self.d, "k": {"buf": bufs[0], "ld": ld}, "v": {"buf": bufs[1], "ld": ld}, "M": M, "rows": {"buf": rb} if rows else None})
        for b in bufs + [rb]: self.gpu.free(b)
        for b in range(self.seqs):
            self.tok[b] = tuple(np.concatenate([o, _clean(x[b])], 1) for o, x in zip(self.tok[b], (k, v)))

    def held(self, b):
        """K, V [Hkv][L][128] in 64 bits, as the cache should stand for them"""
        out = []
        for x in self.tok[b]:
            y = x.astype(np.float64)
            for pg in range(x.shape[1] // PAGE):
                for h in range(self.Hkv):
                    q, s = _quantise(x[h, pg * PAGE:(pg + 1) * PAGE])
                    y[h, pg * PAGE:(pg + 1) * PAGE] = q * s
            out.append(y)
        return out

    def fill(self, lens, seed=1, std=(1.0, 1.0)):
        rng = np.random.default_rng(seed)
        k, v = ([rng.normal(0, s, (self.Hkv, int(L), 128)).astype(np.float16) for L in lens] for s in std)
        self.write(list(lens), k, v)

    def read(self, news, rows=True, extra=0):
        M = int(sum(news)) + extra
        offs = np.concatenate([[0], np.cumsum(news)]).astype(np.uint32)
        kb, vb = (self.gpu.upload(np.full((self.Hkv, M, 128), 0x7E01, np.uint16)) for _ in range(2))
        rb = self.gpu.upload(offs) if rows else None
        self.P.cacheRead(self.gpu, {"cache": self.d, "k": {"buf": kb}, "v": {"buf": vb}, "M": M, "rows": {"buf": rb} if rows else None})
        out = [self.gpu.read(x).view(np.uint16)[:self.Hkv * M * 128].reshape(self.Hkv, M, 128) for x in (kb, vb)]
        for x in (kb, vb, rb): self.gpu.free(x)
        return out, offs


def _attn_want(q, K, V, window, sinks, scale=None):
    """q [Hq][n][128], K / V [Hkv][L][128] -> [n][Hq][128] in 64 bits"""
    import torch
    q, K, V = (torch.from_numpy(np.asarray(t, np.float64)).cuda() for t in (q, K, V))
    Hq, n = q.shape[:2]; Hkv, L = K.shape[:2]
    p = torch.arange(L - n, L, device="cuda")[:, None]; j = torch.arange(L, device="cuda")[None]
    see = j <= p
    if window: see = see & ((p - j < window) | (j < sinks))
    s = torch.einsum("hgnd,hld->hgnl", q.view(Hkv, Hq // Hkv, n, 128), K) * (scale or 128 ** -0.5)
    o = torch.einsum("hgnl,hld->hgnd", torch.softmax(s.masked_fill(~see, -torch.inf), -1), V)
    return o.permute(2, 0, 1, 3).reshape(n, Hq, 128).cpu().numpy()


def _attend(cache, news, group, window=0, sinks=0, scale=None, rows=True, new=None, kernel=None, seed=5, qstd=1.0, extra=0, ldo=None, nan_row=None, ldq=0):
    """runs cacheAttention for the last `news` tokens of each sequence; returns (out [M][Hq][128], wanted list, q list)"""
    P, gpu, Hq = cache.P, cache.gpu, cache.Hkv * group
    rng = np.random.default_rng(seed)
    offs = np.concatenate([[0], np.cumsum(news)]).astype(np.uint32); M = int(offs[-1]) + extra
    q = rng.normal(0, qstd, (Hq, M + ldq, 128)).astype(np.float16)
    if ldq: q[:, M:] = np.nan                                                                  # rows of another call between the heads
    if nan_row is not None: q[nan_row[0], nan_row[1], 3] = np.nan
    ldo = ldo or Hq * 128
    qb, ob, rb = gpu.upload(q), gpu.upload(np.full((M, ldo), 0x7E01, np.uint16)), gpu.upload(offs)
    P.cacheAttention(gpu, {"cache": cache.d, "q": {"buf": qb, "ld": M + ldq}, "o": {"buf": ob, "ld": ldo}, "Hq": Hq, "M": M, "rows": {"buf": rb} if rows else None, "new": new, "window": window,
                           "sinks": sinks, "scale": scale, "kernel": kernel})
    raw = gpu.read(ob).view(np.uint16)[:M * ldo].reshape(M, ldo)
    for b in (qb, ob, rb): gpu.free(b)
    assert (raw[:, Hq * 128:] == 0x7E01).all() and (raw[offs[-1]:] == 0x7E01).all(), "written outside the rows"
    out = np.ascontiguousarray(raw[:, :Hq * 128]).view(np.float16).reshape(M, Hq, 128)
    return out, [q[:, offs[b]:offs[b + 1]] for b in range(cache.seqs)], offs


def _check(cache, news, group, window=0, sinks=0, scale=None, **kw):
    out, q, offs = _attend(cache, news, group, window, sinks, scale, **kw)
    for b in range(cache.seqs):
        if not news[b]: continue
        K, V = cache.held(b)
        want = _attn_want(q[b], K, V, window, sinks, scale)
        got = out[offs[b]:offs[b + 1]].astype(np.float64)
        top = np.abs(V).max()
        tol = top * (2 * (2.0 ** -11 + 1e-4) + 2.0 ** -11 + K.shape[1] * 2.0 ** -25)
        err = np.abs(got - want)
        assert err.max() <= tol, (b, err.max(), tol, np.unravel_index(err.argmax(), err.shape))


# ------------------------------------------------------------------------------------------------------------- writing, reading back
STEPS = [
    dict(label="one sequence, token by token over a page's end", Hkv=2, maxp=3, steps=[[62]] + [[1]] * 4, rows=False),
    dict(label="chunks that begin and end inside pages", Hkv=3, maxp=8, steps=[[37], [64], [27], [130], [1], [63], [65]], rows=False),
    dict(label="several sequences, some without new tokens", Hkv=1, maxp=6, steps=[[5, 0, 70, 1], [60, 1, 0, 63], [1, 0, 64, 0], [130, 200, 3, 1]], rows=True),
    dict(label="equal counts", Hkv=2, maxp=4, steps=[[40] * 5, [1] * 5, [23] * 5, [1] * 5, [100] * 5], rows=False),
    dict(label="33 sequences", Hkv=2, maxp=4, steps=[[(b * 7) % 66 for b in range(33)], [b % 3 for b in range(33)], [64 + b for b in range(33)]], rows=True),
    dict(label="128 sequences", Hkv=1, maxp=3, steps=[[(b * 11) % 66 for b in range(128)], [b % 2 for b in range(128)], [70] * 128], rows=True),
    dict(label="more sequences than a block has threads", Hkv=1, maxp=2, steps=[[(b * 7) % 66 for b in range(300)], [1 + b % 3 for b in range(300)]], rows=True),
]


@pytest.mark.parametrize("c", STEPS, ids=lambda c: c["label"])
def test_write_and_read(gpu, c):
    """whatever the calls, each page is quantised once, from its 64 tokens; the rest is in the tail; nothing else is touched"""
    import p0pc0rn_kernels_b200 as P
    Hkv, seqs = c["Hkv"], len(c["steps"][0])
    cache = Cache(P, gpu, Hkv, seqs, c["maxp"], seed=3)
    rng = np.random.default_rng(11)
    try:
        for news in c["steps"]:
            k, v = ([(rng.normal(0, 1, (Hkv, n, 128)) * np.exp(rng.normal(0, 1, (Hkv, 1, 1)))).astype(np.float16) for n in news] for _ in range(2))
            cache.write(news, k, v, rows=c["rows"], extra=2 if c["rows"] else 0, ld=sum(news) + 5)
            got, offs = cache.read(news, rows=c["rows"], extra=1 if c["rows"] else 0)
            for b in range(0, seqs, max(1, seqs // 20)):
                for g, w in zip(got, cache.held(b)):
                    n = news[b]
                    assert np.array_equal(g[:, offs[b]:offs[b + 1]].view(np.float16), w[:, w.shape[1] - n:].astype(np.float16)), (b, news)
            if c["rows"]: assert all((g[:, offs[-1]:] == 0x7E01).all() for g in got)
        # the bytes themselves
        n = P.cacheBytes(cache.pages, Hkv, seqs, c["maxp"])
        codes = gpu.read(cache.d["codes"]["buf"], 0, n["codes"]).reshape(cache.pages, Hkv, 2, -1)
        scales = gpu.read(cache.d["scales"]["buf"], 0, n["scales"]).view(np.float32).reshape(cache.pages, Hkv, 2)
        tail = gpu.read(cache.d["tail"]["buf"], 0, n["tail"]).view(np.float16).reshape(seqs, Hkv, 2, -1)
        used = np.zeros(cache.pages, bool)
        for b in range(0, seqs, max(1, seqs // 20)):
            L = int(cache.lens[b])
            for pg in range(L // PAGE):
                page = cache.table[b, pg]; used[page] = True
                for h in range(Hkv):
                    for w, off in enumerate(_offsets()):
                        q, s = _quantise(cache.tok[b][w][h, pg * PAGE:(pg + 1) * PAGE])
                        assert scales[page, h, w] == s and np.array_equal(codes[page, h, w][off], (q + 128).astype(np.uint8))
            for h in range(Hkv):
                for w, off in enumerate(_offsets()):
                    assert np.array_equal(tail[b, h, w][off][:L % PAGE], cache.tok[b][w][h, L - L % PAGE:])
        if seqs < 20: assert (codes[~used] == 0xA5).all() and np.isnan(scales[~used]).all()
        all_, offs = cache.read([int(x) for x in cache.lens])                                  # whole sequences
        for b in range(0, seqs, max(1, seqs // 20)):
            for g, w in zip(all_, cache.held(b)): assert np.array_equal(g[:, offs[b]:offs[b + 1]].view(np.float16), w.astype(np.float16))
    finally:
        cache.free()


def test_write_special_values(gpu):
    """NaN is stored as 0, infinities as the largest finite value; blocks of zeros, of subnormals, and one whose largest value stands alone"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 5, 1, 3)
    rng = np.random.default_rng(2)
    k = rng.normal(0, 1, (5, 100, 128)).astype(np.float16); v = rng.normal(0, 1, (5, 100, 128)).astype(np.float16)
    k[0, 3, 7] = np.nan; v[0, 90, 0] = np.nan; k[1, 63, 127] = np.inf; v[1, 64, 5] = -np.inf; v[1, 0, 0] = -np.inf
    k[2, :64] = 0; v[2, :64] = -0.0
    k[3] = (rng.integers(-40, 41, (100, 128)) * 2.0 ** -24).astype(np.float16); v[3] = 0; v[3, 5, 5] = 2.0 ** -24
    k[4, :64] = 0; k[4, 10, 10] = -65504; v[4, :64] = 1.0; v[4, 2, 3] = 2.0                   # 63.5 steps: a tie
    try:
        cache.write([100], [k], [v], rows=False)
        got, _ = cache.read([100], rows=False)
        for g, w in zip(got, cache.held(0)):
            w = np.clip(w, -65504, 65504).astype(np.float16)
            assert np.isfinite(g.view(np.float16)).all() and np.array_equal(g.view(np.float16), w)
    finally:
        cache.free()


# ------------------------------------------------------------------------------------------------------------- attention
ATT = [
    dict(label="one token of context", Hkv=2, group=4, lens=[1], news=[1]),
    dict(label="a tail only", Hkv=1, group=1, lens=[63], news=[1]),
    dict(label="a whole page, no tail", Hkv=3, group=4, lens=[64], news=[1]),
    dict(label="a page and one token", Hkv=2, group=8, lens=[65], news=[1]),
    dict(label="one token, 300 of context", Hkv=8, group=4, lens=[301], news=[1]),
    dict(label="one token, several pages per warp", Hkv=4, group=4, lens=[40000], news=[1]),
    dict(label="ragged batch", Hkv=2, group=4, lens=[1, 64, 500, 65, 3000, 128, 129, 7], news=[1] * 8),
    dict(label="sequences without new tokens, rows behind the last", Hkv=2, group=3, lens=[100, 0, 300, 64, 200], news=[2, 0, 0, 5, 1], extra=3),
    dict(label="a batch of short contexts: many items per warp", Hkv=2, group=2, lens=[1 + (b * 37) % 150 for b in range(700)], news=[1] * 700),
    dict(label="16 rows exactly", Hkv=1, group=16, lens=[200], news=[1]),
    dict(label="17 rows: two row blocks", Hkv=1, group=17, lens=[200], news=[1]),
    dict(label="several new tokens, odd group", Hkv=2, group=5, lens=[333, 70], news=[7, 66]),
    dict(label="the first tokens of a prompt", Hkv=2, group=2, lens=[150], news=[150]),
    dict(label="prompts of several sequences", Hkv=1, group=4, lens=[500, 129, 90], news=[300, 129, 1]),
    dict(label="window inside a page", Hkv=2, group=4, lens=[300], news=[1], window=10),
    dict(label="window 1", Hkv=2, group=4, lens=[300, 65], news=[3, 1], window=1),
    dict(label="window and sinks far apart", Hkv=2, group=4, lens=[5000, 900, 30], news=[1, 4, 2], window=200, sinks=4),
    dict(label="sinks over several pages", Hkv=1, group=2, lens=[2000], news=[5], window=64, sinks=130),
    dict(label="sinks that meet the window", Hkv=1, group=2, lens=[300], news=[2], window=100, sinks=250),
    dict(label="window wider than the context", Hkv=1, group=2, lens=[300], news=[2], window=1000, sinks=2),
    dict(label="prompt longer than its window", Hkv=2, group=3, lens=[700, 400], news=[700, 150], window=100, sinks=3),
    dict(label="own scale", Hkv=2, group=2, lens=[200], news=[3], scale=0.02),
    dict(label="peaked scores", Hkv=2, group=2, lens=[700], news=[2], qstd=12.0),
    dict(label="output rows with a stride, 4-byte aligned", Hkv=2, group=2, lens=[200], news=[3], ldo=4 * 128 + 6),
    dict(label="heads with a stride", Hkv=2, group=2, lens=[200, 70], news=[3, 40], ldq=7),
]


def _att_cache(P, gpu, c):
    cache = Cache(P, gpu, c["Hkv"], len(c["lens"]), max(1, -(-max(c["lens"]) // PAGE)) + 1, seed=9)
    cache.fill(c["lens"], std=(1.0, np.float16(0.7)))
    return cache


PROMPTS = [
    dict(label="a block of queries exactly", Hkv=1, group=4, lens=[64], news=[64]),
    dict(label="one query more than a tile", Hkv=2, group=4, lens=[33], news=[33]),
    dict(label="an odd number of pages, history that ends in one", Hkv=2, group=4, lens=[700], news=[130]),
    dict(label="few queries over a long context: items that cross many blocks", Hkv=2, group=4, lens=[20000], news=[70]),
    dict(label="a long prompt: blocks with several items", Hkv=4, group=4, lens=[1500], news=[1500]),
    dict(label="groups that do not divide a tile", Hkv=2, group=7, lens=[600, 300], news=[200, 300]),
    dict(label="one head per kv head", Hkv=5, group=1, lens=[1000], news=[400]),
    dict(label="many heads per kv head", Hkv=1, group=100, lens=[200], news=[70]),
    dict(label="128 heads per kv head", Hkv=1, group=128, lens=[300], news=[3]),
    dict(label="long window over long contexts", Hkv=2, group=4, lens=[9000, 4000], news=[300, 1000], window=700, sinks=70),
    dict(label="wide scores: the maximum moves by more than the lazy threshold", Hkv=2, group=4, lens=[2000], news=[200], qstd=6.0),
    dict(label="steps and prompts in one batch", Hkv=2, group=4, lens=[5000, 300, 2000, 64, 900], news=[1, 300, 2, 64, 500], extra=1),
]


@pytest.mark.parametrize("kernel", [None, "split", "tmem"])
@pytest.mark.parametrize("c", ATT + PROMPTS, ids=lambda c: c["label"])
def test_attention(gpu, c, kernel):
    import p0pc0rn_kernels_b200 as P
    cache = _att_cache(P, gpu, c)
    try:
        kw = {k: c[k] for k in ("window", "sinks", "scale", "qstd", "extra", "ldo", "ldq") if k in c}
        kw["kernel"] = kernel
        for _ in range(2): _check(cache, c["news"], c["group"], **kw)                          # (twice: a counter left over would show)
        if len(set(c["news"])) == 1: _check(cache, c["news"], c["group"], rows=False, new=c["news"][0], **{k: v for k, v in kw.items() if k != "extra"})
    finally:
        cache.free()


def test_attention_chooses_by_rows(gpu):
    """few query rows per kv head go to the split-key kernel, many to the tensor-memory kernel; a batch of both kinds, or one the host cannot know, to both"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 8, 3, 5)
    cache.fill([300, 200, 250])
    try:
        for news, group, rows, new, want in (([1, 1, 1], 4, False, None, 24), ([48, 48, 48], 1, False, None, 24), ([13, 13, 13], 4, False, None, 25), ([1, 0, 2], 4, True, 2, 24),
                                             ([1, 100, 2], 4, True, 100, 26), ([1, 100, 2], 4, True, None, 26), ([1, 1, 1], 200, False, None, 24)):
            _check(cache, news, group, rows=rows, new=new)
            assert gpu.lastKernel == want, (news, group, gpu.lastKernel)
    finally:
        cache.free()
    one = Cache(P, gpu, 8, 1, 5)
    one.fill([300])
    try:
        for n, want in ((24, 24), (25, 25)):
            _check(one, [n], 4, rows=False)
            assert gpu.lastKernel == want
    finally:
        one.free()


def test_attention_scales_far_apart(gpu):
    """pages whose values differ by a factor of 2^20, an all-zero page, a page of the largest values"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 2, 1, 8)
    rng = np.random.default_rng(4)
    k = rng.normal(0, 1, (2, 400, 128)); v = rng.normal(0, 1, (2, 400, 128))
    v[:, :64] *= 2.0 ** -14; v[:, 64:128] = 0; v[:, 128:192] *= 2.0 ** 6; k[:, 192:256] *= 2.0 ** -10; k[0, 256:320] = 0; v[1, 300, :] = 60000.0
    try:
        cache.write([400], [k.astype(np.float16)], [v.astype(np.float16)], rows=False)
        for kernel in ("split", "tmem"):
            _check(cache, [2], 4, kernel=kernel)
            _check(cache, [2], 4, window=330, kernel=kernel)
            _check(cache, [200], 4, window=330, kernel=kernel)
    finally:
        cache.free()


@pytest.mark.parametrize("kernel", ["split", "tmem"])
@pytest.mark.parametrize("shift", [14, 20, 26])
def test_attention_sum_where_a_small_page_weighs_most(gpu, shift, kernel):
    """half of the weight, or nearly all of it, lies on pages whose values are 2^-shift of the others': it counts in full"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 2, 1, 6)
    rng = np.random.default_rng(6)
    k = rng.normal(0, 0.02, (2, 300, 128)); v = rng.normal(0, 1, (2, 300, 128))
    k[1, :128] *= 30.0                                                                         # (the second head: weights that vary)
    v[:, :128] *= 2.0 ** (9 - shift); v[:, 128:] *= 2.0 ** 9
    try:
        cache.write([300], [k.astype(np.float16)], [v.astype(np.float16)], rows=False)
        _check(cache, [2], 4, kernel=kernel)
        _check(cache, [170], 4, kernel=kernel)
    finally:
        cache.free()


@pytest.mark.parametrize("kernel", ["split", "tmem"])
@pytest.mark.parametrize("scale", [1e-45, 1e-30, 1e-6, 300.0])
def test_attention_scales_of_any_size(gpu, scale, kernel):
    """a scale that leaves nothing of the scores is an average; a large one is the largest score's value, kept apart here by their distance"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 1, 1, 4)
    rng = np.random.default_rng(7)
    k = np.zeros((1, 200, 128)); k[0, :, 0] = rng.permutation(200) - 100.0                     # (scores apart by |q0|: nothing is rounded, a second key has no weight)
    v = rng.normal(0, 1, (1, 200, 128))
    try:
        cache.write([200], [k.astype(np.float16)], [v.astype(np.float16)], rows=False)
        _check(cache, [3], 2, scale=scale, kernel=kernel)
        _check(cache, [3], 2, window=90, sinks=3, scale=scale, kernel=kernel)
    finally:
        cache.free()


@pytest.mark.parametrize("window", [0, 9000])
def test_attention_long_items_among_many(gpu, window):
    """a long context among many short items: its items lie over many blocks, which add them up without another kernel; the same again, bit for bit"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 8, 3, 320)
    cache.fill([400, 20000, 37])
    try:
        for _ in range(2): _check(cache, [310, 12, 20], 16, window=window, kernel="tmem")
        got = [_attend(cache, [310, 12, 20], 16, window=window, kernel="tmem")[0].view(np.uint16) for _ in range(3)]
        assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
    finally:
        cache.free()


@pytest.mark.parametrize("kernel", ["split", "tmem"])
def test_pages_behind_the_window_can_be_given_away(gpu, kernel):
    """the table's entries of pages that no query sees, and that hold no sink, are not followed: they name no page here"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 2, 2, 20)
    cache.fill([1000, 520])
    try:
        table = cache.table.copy()
        for b, (L, n) in enumerate(((1000, 70), (520, 3))):                                    # window 200: the oldest query, L - n, sees L - n - 199 and later ones; sinks: 130 tokens
            table[b, 3:(L - n - 199) // 64] = 0xFFFFFFFF
            table[b, L // 64:] = 0xFFFFFFFF
        assert (table[0, 3:11] == 0xFFFFFFFF).all() and table[1, 3] == 0xFFFFFFFF and table[1, 4] != 0xFFFFFFFF
        gpu.upload(table, dst=cache.d["table"]["buf"])
        _check(cache, [70, 3], 4, window=200, sinks=130, kernel=kernel)
        gpu.done()
    finally:
        cache.free()


def test_layers_that_share_table_and_lengths(gpu):
    """two layers' caches with one table and one set of lengths, which a program uploads once a step"""
    import p0pc0rn_kernels_b200 as P
    one = Cache(P, gpu, 2, 2, 4)
    two = Cache(P, gpu, 1, 2, 4, seed=0)
    for k in ("table", "lens"): gpu.free(two.d[k]["buf"])
    two.d = {**two.d, **{k: P.kvCache(gpu, {"Hkv": 1, "pages": two.pages, "seqs": 2, "maxPages": 4, "table": one.d["table"], "lens": one.d["lens"]})[k] for k in ("table", "lens")}}
    try:
        assert two.d["table"]["buf"] is one.d["table"]["buf"] and two.d["lens"]["buf"] is one.d["lens"]["buf"]
        rng = np.random.default_rng(3)
        for news in ([100, 7], [1, 1], [30, 60]):
            for c in (one, two):
                c.write(news, *([rng.normal(0, 1, (c.Hkv, n, 128)).astype(np.float16) for n in news] for _ in range(2)))
        for c in (one, two): _check(c, [30, 60], 2)
    finally:
        for k in ("codes", "scales", "tail"): gpu.free(two.d[k]["buf"])
        one.free()


def test_attention_nan_query_stays_in_its_row(gpu):
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 2, 2, 10)
    cache.fill([500, 200])
    try:
        for kernel in ("split", "tmem"):
            out, q, offs = _attend(cache, [3, 2], 4, nan_row=(5, 1), kernel=kernel)
            bad = np.zeros(out.shape[:2], bool); bad[1, 5] = True
            assert np.isnan(out[bad]).all() and np.isfinite(out[~bad]).all()
    finally:
        cache.free()


def test_attention_of_a_later_token_does_not_reach_back(gpu):
    """an infinite value in the newest token's value (kept as the largest finite one): the queries before it do not see it"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 1, 1, 4)
    rng = np.random.default_rng(4)
    k, v = (rng.normal(0, 1, (1, 70, 128)).astype(np.float16) for _ in range(2))
    v[0, 69] = np.inf; k[0, 69] = np.nan
    try:
        cache.write([70], [k], [v], rows=False)
        for kernel in ("split", "tmem"):
            out, q, offs = _attend(cache, [4], 2, kernel=kernel)
            want = _attn_want(q[0][:, :3], *(x[:, :69] for x in cache.held(0)), 0, 0)
            top = np.abs(v[0, :69].astype(np.float64)).max()
            assert np.abs(out[:3] - want).max() <= top * (2 * (2.0 ** -11 + 1e-4) + 2.0 ** -11 + 70 * 2.0 ** -25)
    finally:
        cache.free()


def test_cache_past_32_bit_offsets(gpu):
    """pages that lie more than 2^32 bytes into the codes"""
    import p0pc0rn_kernels_b200 as P
    Hkv = 8
    cache = Cache(P, gpu, Hkv, 2, 5, pages=34000, first_page=33800)
    try:
        assert int(cache.table.min()) * Hkv * 16384 > 1 << 32
        cache.fill([300, 130])
        got, offs = cache.read([300, 130])
        for b in range(2):
            for g, w in zip(got, cache.held(b)): assert np.array_equal(g[:, offs[b]:offs[b + 1]].view(np.float16), w.astype(np.float16))
        _check(cache, [3, 1], 4)
    finally:
        cache.free(); gpu.drainPool()


# ------------------------------------------------------------------------------------------------------------- rotary positions
def _freq(rot, theta=10000.0, factor=1.0, original=0.0, fast=32.0, slow=1.0):
    i = np.arange(rot // 2); f = theta ** (-2.0 * i / rot) if rot else np.zeros(0)
    if factor == 1.0: return f
    g = np.clip((original * f / (2 * np.pi) - slow) / (fast - slow), 0, 1) if original else 0.0
    return f * (g + (1 - g) / factor)


ROPE = [
    dict(label="half", mode="half", H=5, news=[1], lens=[1]),
    dict(label="interleaved, far out", mode="interleaved", H=3, news=[4, 1, 0, 30], lens=[4, 900000, 7, 4000000000]),
    dict(label="part of the head, half", mode="half", rot=64, H=2, news=[33], lens=[500]),
    dict(label="part of the head, half, odd", mode="half", rot=38, H=2, news=[33, 2], lens=[500, 70]),
    dict(label="half of an odd half", mode="half", rot=6, H=3, news=[5], lens=[5]),
    dict(label="part of the head, interleaved", mode="interleaved", rot=90, H=2, news=[33], lens=[500]),
    dict(label="nothing turned", mode="half", rot=0, H=2, news=[3], lens=[5]),
    dict(label="scaled linearly", mode="half", H=2, news=[40], lens=[100000], factor=4.0),
    dict(label="scaled by parts", mode="interleaved", H=2, news=[40], lens=[100000], factor=8.0, original=4096, mscale=1.2, theta=500000.0),
    dict(label="scaled by parts, own limits, half", mode="half", rot=96, H=70, news=[40, 3], lens=[100000, 10], factor=8.0, original=8192, fast=16.0, slow=2.0),
    dict(label="many tokens and heads", mode="half", H=40, news=[1000, 37], lens=[1000, 5000]),
]


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("c", ROPE, ids=lambda c: c["label"])
def test_rope(gpu, c, inplace):
    import p0pc0rn_kernels_b200 as P
    rng = np.random.default_rng(1)
    H, rot, news = c["H"], c.get("rot", 128), c["news"]
    offs = np.concatenate([[0], np.cumsum(news)]).astype(np.uint32); M, ld = int(offs[-1]) + 2, int(offs[-1]) + 5
    x = rng.normal(0, 1, (H, ld, 128)).astype(np.float16)
    xb, yb, lb, rb = gpu.upload(x), gpu.upload(np.full((H, M, 128), 0x7E01, np.uint16)), gpu.upload(np.array(c["lens"], np.uint32)), gpu.upload(offs)
    extra = {k: c[k] for k in ("theta", "factor", "original", "fast", "slow", "mscale") if k in c}
    try:
        P.rope(gpu, {"x": {"buf": xb, "ld": ld}, "y": None if inplace else {"buf": yb}, "H": H, "M": M, "seqs": len(news), "lens": {"buf": lb}, "rows": {"buf": rb}, "mode": c["mode"], "rot": rot, **extra})
        got = gpu.read(xb).view(np.float16)[:x.size].reshape(x.shape) if inplace else gpu.read(yb).view(np.float16)[:H * M * 128].reshape(H, M, 128)
        if inplace: assert np.array_equal(got[:, offs[-1]:], x[:, offs[-1]:])
        else: assert (got[:, offs[-1]:].view(np.uint16) == 0x7E01).all()
        pos = np.concatenate([np.arange(L - n, L, dtype=np.float64) for L, n in zip(c["lens"], news)])
        ang = pos[:, None] * _freq(rot, **{k: v for k, v in extra.items() if k != "mscale"})
        ms = c.get("mscale", 1.0); cs, sn = np.cos(ang) * ms, np.sin(ang) * ms
        x = x[:, :offs[-1]].astype(np.float64); want = x.copy()
        first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if c["mode"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
        a, b = x[..., first], x[..., second]
        want[..., first], want[..., second] = a * cs - b * sn, a * sn + b * cs
        mag = np.zeros_like(want); mag[..., first] = mag[..., second] = (np.abs(a) + np.abs(b)) * ms
        # (an angle in 64 bits: position * frequency in turns and the oracle's own product are each off by 2^-53 of the angle)
        tol = np.abs(want) * 2.0 ** -11 + 2.0 ** -25 + mag * (6 * 2.0 ** -24 + float(pos.max(initial=1.0)) * 8 * 2.0 ** -53)
        assert (np.abs(got[:, :offs[-1]].astype(np.float64) - want) <= tol).all()
        assert np.array_equal(got[:, :offs[-1], rot:], x[..., rot:].astype(np.float16))
    finally:
        for t in (xb, yb, lb, rb): gpu.free(t)


# ------------------------------------------------------------------------------------------------------------- together
def test_decoding_loop_recorded_once(gpu):
    """rotary positions, write and attention of a decoding step, recorded once and replayed over pages' ends with new lengths: as a program runs
    them.  A second recording, of another batch, shares the scratch memory and is replayed in between."""
    import p0pc0rn_kernels_b200 as P
    rng = np.random.default_rng(8)
    own = P.createGpu({"device": 0})
    Hkv, group, seqs = 2, 4, 3
    Hq = Hkv * group
    rot = {"mode": "half", "rot": 128, "theta": 10000.0}

    def turn(x, p):
        cs, sn = np.cos(p * _freq(128)), np.sin(p * _freq(128)); x = x.astype(np.float64)
        a, b = x[..., :64], x[..., 64:]
        return np.concatenate([a * cs - b * sn, a * sn + b * cs], -1)
    sets = []
    for start in ([60, 127, 0], [700, 3, 64]):
        cache = Cache(P, own, Hkv, seqs, 14, seed=sum(start))
        cache.fill(start)
        heads, ob = own.buffer((Hq + 2 * Hkv) * seqs * 256), own.buffer(seqs * Hq * 256)
        n = seqs * 256

        def step(cache=cache, heads=heads, ob=ob, n=n):
            P.rope(own, {"x": {"buf": heads}, "H": Hq + Hkv, "M": seqs, "seqs": seqs, "lens": cache.d["lens"], **rot})
            P.cacheWrite(own, {"cache": cache.d, "k": {"buf": heads, "off": Hq * n}, "v": {"buf": heads, "off": (Hq + Hkv) * n}, "M": seqs})
            P.cacheAttention(own, {"cache": cache.d, "q": {"buf": heads}, "o": {"buf": ob}, "Hq": Hq, "M": seqs})
        sets.append([cache, heads, ob, step, None])
    try:
        for s in sets:                                   # one eager step each, then recorded
            s[0].advance([1] * seqs); x = rng.normal(0, 1, (Hq + 2 * Hkv, seqs, 128)).astype(np.float16); own.upload(x, dst=s[1]); s[3](); _step_check(s, x, turn, own, Hq, Hkv)
            s[4] = own.record(s[3])
        for it in range(8):
            for s in sets:
                s[0].advance([1] * seqs); x = rng.normal(0, 1, (Hq + 2 * Hkv, seqs, 128)).astype(np.float16); own.upload(x, dst=s[1]); s[4].launch(); _step_check(s, x, turn, own, Hq, Hkv)
        assert not own.lost
    finally:
        for s in sets:
            if s[4]: s[4].free()
            s[0].free()
        own.close()


def _step_check(s, x, turn, own, Hq, Hkv):
    cache, heads, ob = s[:3]
    seqs = cache.seqs
    y = own.read(heads).view(np.float16)[:x.size].reshape(x.shape)
    out = own.read(ob).view(np.float16)[:seqs * Hq * 128].reshape(seqs, Hq, 128)
    for b in range(seqs):
        p = float(cache.lens[b] - 1)
        want = turn(x[:Hq + Hkv, b], p)
        assert np.abs(y[:Hq + Hkv, b] - want).max() <= np.abs(want).max() * 2.0 ** -11 + 1e-5
        cache.tok[b] = tuple(np.concatenate([o, t[:, b:b + 1]], 1) for o, t in zip(cache.tok[b], (y[Hq:Hq + Hkv], x[Hq + Hkv:])))
        K, V = cache.held(b)
        w = _attn_want(y[:Hq, b:b + 1], K, V, 0, 0)[0]
        assert np.abs(out[b] - w).max() <= np.abs(V).max() * (2 * (2.0 ** -11 + 1e-4) + 2.0 ** -11 + K.shape[1] * 2.0 ** -25)


def test_attention_recorded_before_its_scratch_memory_exists(gpu):
    import p0pc0rn_kernels_b200 as P
    own = P.createGpu({"device": 0})
    cache = Cache(P, own, 2, 1, 3)
    cache.fill([130])
    q, o = own.buffer(4 * 256), own.buffer(4 * 256)
    call = lambda: P.cacheAttention(own, {"cache": cache.d, "q": {"buf": q}, "o": {"buf": o}, "Hq": 4, "M": 1})  # noqa: E731
    try:
        with pytest.raises(ValueError, match="run it once before"): own.record(call)
        assert not own.lost
        call()
        g = own.record(call)
        g.launch(); own.done(); g.free()
    finally:
        cache.free(); own.close()


def test_same_result_twice_and_in_one_call_of_many(gpu):
    """bit for bit the same from run to run; a prefix shared by two sequences (one page in two tables) is read by both"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 2, 2, 8)
    cache.fill([400, 0])
    try:
        for kernel in ("split", "tmem"):
            outs = [_attend(cache, [5, 0], 4, kernel=kernel)[0].tobytes() for _ in range(3)]
            assert outs[0] == outs[1] == outs[2]
        t = cache.table.copy(); t[1, :6] = t[0, :6]
        gpu.upload(t, dst=cache.d["table"]["buf"])
        rng = np.random.default_rng(3)
        k, v = (rng.normal(0, 1, (2, 3, 128)).astype(np.float16) for _ in range(2))
        cache.tok[1] = tuple(x[:, :384] for x in cache.tok[0]); cache.lens[1] = 384
        empty = np.zeros((2, 0, 128), np.float16)
        cache.write([0, 3], [empty, k], [empty, v])                        # its own tail behind the shared pages
        for kernel in ("split", "tmem"): _check(cache, [5, 3], 4, kernel=kernel)
    finally:
        cache.free()


def test_another_stream(gpu):
    """a context on the host framework's stream: tensors made there, no waiting in between"""
    import torch

    import p0pc0rn_kernels_b200 as P
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        own = P.createGpu({"device": 0, "stream": st.cuda_stream})
        try:
            cache = Cache(P, own, 2, 2, 6)
            cache.fill([300, 100])
            _check(cache, [2, 1], 4)
            cache.free()
        finally:
            own.close()


# ------------------------------------------------------------------------------------------------------------- refusals
def test_refusals(gpu):
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 2, 3, 2)
    b = gpu.buffer(1 << 20)
    t = {"buf": b}
    kv = {"cache": cache.d, "k": t, "v": t, "M": 6}
    at = {"cache": cache.d, "q": t, "o": t, "Hq": 4, "M": 6}
    ro = {"x": t, "H": 4, "M": 6, "seqs": 3, "lens": cache.d["lens"]}

    def no(op, args, text, **change):
        a = dict(args); a.update(change)
        with pytest.raises(ValueError, match=text): op(gpu, a)

    def but(**kw):
        return dict(cache.d, **kw)
    try:
        for op, a in ((P.cacheWrite, kv), (P.cacheRead, kv), (P.cacheAttention, at)):
            no(op, a, "multiple of seqs", M=7)
            no(op, a, "codes needs", cache=but(pages=1000)); no(op, a, "table needs", cache=but(maxPages=2000)); no(op, a, "at least one", cache=but(pages=0))
            no(op, a, "at most 1024", cache=but(seqs=1025)); no(op, a, "missing", cache=but(tail={"buf": type("B", (), {"handle": None})()}))
            no(op, a, "16 bytes", cache=but(codes={"buf": cache.d["codes"]["buf"], "off": 8}))
            no(op, a, "rows needs", rows={"buf": gpu.bufs and b, "off": (1 << 20) - 8})
        no(P.cacheWrite, kv, "k needs", M=3000); no(P.cacheWrite, kv, "v.ld", v={"buf": b, "ld": 5}); no(P.cacheWrite, kv, "multiple of 16", k={"buf": b, "off": 4})
        no(P.cacheAttention, at, "multiple of Hkv", Hq=3); no(P.cacheAttention, at, "o needs", o={"buf": b, "ld": 1 << 18}); no(P.cacheAttention, at, "o.ld", o={"buf": b, "ld": 511})
        no(P.cacheAttention, dict(at, Hq=2 * 130), "128 heads", kernel="tmem", q={"buf": b}, o={"buf": b})
        no(P.cacheAttention, at, "finite", scale=float("nan")); no(P.cacheAttention, at, "not negative", scale=-0.1); no(P.cacheAttention, at, "q needs", M=3000)
        no(P.rope, ro, "even", rot=7); no(P.rope, ro, "even", rot=130); no(P.rope, ro, "unknown mode", mode="x"); no(P.rope, ro, "positive", theta=-1.0); no(P.rope, ro, "fast above slow", fast=1.0, slow=2.0)
        no(P.rope, ro, "multiple of seqs", M=7); no(P.rope, ro, "x needs", M=3000); no(P.rope, ro, "sequences", seqs=0); no(P.rope, ro, "multiple of 16", x={"buf": b, "off": 2})
        assert not gpu.lost
        for op, a in ((P.cacheWrite, kv), (P.cacheRead, kv), (P.cacheAttention, at), (P.rope, ro)): op(gpu, dict(a, M=0))      # nothing to do
        gpu.done()
    finally:
        gpu.free(b); cache.free()


def test_numbers_on_the_device_that_make_no_sense(gpu):
    """row offsets, lengths and page numbers are checked where they are read: the sequence is left out (a page not followed), the next wait says
    so, and the context goes on"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 2, 2, 4, spare=0)
    cache.fill([100, 130])
    ok, _ = cache.read([100, 130])
    lens, table = cache.d["lens"]["buf"], cache.d["table"]["buf"]
    b, r = gpu.buffer(1 << 20), gpu.upload(np.array([0, 2, 3], np.uint32))
    calls = [lambda: P.cacheWrite(gpu, {"cache": cache.d, "k": {"buf": b}, "v": {"buf": b}, "M": 3, "rows": {"buf": r}}),
             lambda: P.cacheRead(gpu, {"cache": cache.d, "k": {"buf": b}, "v": {"buf": b}, "M": 3, "rows": {"buf": r}}),
             lambda: P.cacheAttention(gpu, {"cache": cache.d, "q": {"buf": b}, "o": {"buf": b, "off": 1 << 19}, "Hq": 4, "M": 3, "rows": {"buf": r}})]
    rope = lambda: P.rope(gpu, {"x": {"buf": b}, "H": 4, "M": 3, "seqs": 2, "lens": {"buf": lens}, "rows": {"buf": r}})  # noqa: E731

    def fails(call, text):
        call()
        with pytest.raises(P.GpuError, match=text): gpu.done()
        gpu.done()
    try:
        for bad in ([0, 3, 2], [0, 2, 4], [0, 4, 4]):
            gpu.upload(np.array(bad, np.uint32), dst=r)
            for call in calls: fails(call, "row offsets")
        gpu.upload(np.array([0, 2, 3], np.uint32), dst=r)
        for bad in ([1, 130], [100, 0], [100, 257], [0xffffffff, 130]):
            gpu.upload(np.array(bad, np.uint32), dst=lens)
            for call in calls: fails(call, "fewer tokens than rows")
        gpu.upload(np.array([1, 130], np.uint32), dst=lens)
        fails(rope, "fewer tokens")
        gpu.upload(np.array([128, 130], np.uint32), dst=lens)                                  # (the write would finish page 1 of sequence 0)
        for bad in (cache.pages, 0xffffffff):
            t = cache.table.copy(); t[0, 1] = bad
            gpu.upload(t, dst=table)
            for call in calls: fails(call, "page number")
        gpu.upload(cache.table, dst=table); gpu.upload(cache.lens, dst=lens)
        again, offs = cache.read([100, 130])
        assert all(np.array_equal(x[:, :64], y[:, :64]) and np.array_equal(x[:, 100:228], y[:, 100:228]) for x, y in zip(ok, again)) and not gpu.lost
        _check_ok = [int(x) for x in cache.lens]
        assert _check_ok == [100, 130]
    finally:
        for x in (b, r): gpu.free(x)
        cache.free()


# ------------------------------------------------------------------------------------------------------------- errors against the result's own size
def _check_rms(cache, news, group, window=0, sinks=0, scale=None, without=None, **kw):
    """The error's root mean square, per sequence and query head, against the wanted result's.  Each weight is off by at most d = 2^-11 + 1e-4, independently
    of the others (rounding), so that the weighted mean of values that vary around it is off by d of that mean's own spread, at most of its size; the result's
    rounding adds 2^-11 (2^-25 where it is subnormal): sqrt(d^2 + 2^-22) = 7.6e-4 of the result.  The limit is 1e-3 of it, where one page in a
    thousand left out, taken twice or given another's scale moves it by more.  `without`: pages (sequence, page) of which that is checked, on the wanted result."""
    out, q, offs = _attend(cache, news, group, window, sinks, scale, **kw)
    for b in range(cache.seqs):
        if not news[b]: continue
        K, V = cache.held(b)
        want = _attn_want(q[b], K, V, window, sinks, scale)
        err = out[offs[b]:offs[b + 1]].astype(np.float64) - want
        limit = 1e-3 * np.sqrt((want ** 2).mean((0, 2))) + 2.0 ** -25
        got = np.sqrt((err ** 2).mean((0, 2)))
        assert (got <= limit).all(), (b, (got / limit).max(), int((got / limit).argmax()))
        for at, pg in without or ():
            if at != b: continue
            keep = np.arange(K.shape[1]) // PAGE != pg
            less = _attn_want(q[b][:, -1:], K[:, keep], V[:, keep], 0, 0, scale)                 # (the newest query alone: it sees them all)
            assert (np.sqrt(((less - want[-1:]) ** 2).mean((0, 2))) > limit).all(), (b, pg)


@pytest.mark.parametrize("kernel", ["split", "tmem"])
@pytest.mark.parametrize("scale", [2.0 ** 16, 2.0 ** 22, 2.0 ** 24, 2.0 ** 27, 2.0 ** 31, 2.0 ** 64])
def test_attention_large_scores(gpu, scale, kernel):
    """scores of any size that fp32 holds: the value of the largest one (they are far apart: nothing else has weight), never more than that"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 2, 1, 5)
    rng = np.random.default_rng(7)
    k = np.zeros((2, 300, 128)); k[:, :, 0] = rng.permutation(300) - 150.0
    v = rng.normal(0, 1, (2, 300, 128))
    try:
        cache.write([300], [k.astype(np.float16)], [v.astype(np.float16)], rows=False)
        for n in (3, 90):
            _check_rms(cache, [n], 2, scale=scale, kernel=kernel)
            _check_rms(cache, [n], 2, window=90, sinks=3, scale=scale, kernel=kernel)
    finally:
        cache.free()


@pytest.mark.parametrize("kernel", ["split", "tmem"])
def test_attention_large_scores_from_large_values(gpu, kernel):
    """the same with the usual scale, from queries and keys of the largest values, positive and negative: products up to 10^11"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 1, 1, 4)
    rng = np.random.default_rng(7)
    k = np.repeat(rng.permutation(200)[None, :, None] * 600.0 - 60000.0, 128, 2)
    v = rng.normal(0, 1, (1, 200, 128))
    try:
        cache.write([200], [k.astype(np.float16)], [v.astype(np.float16)], rows=False)
        for std in (100.0, 10000.0):
            _check_rms(cache, [3], 2, qstd=std, kernel=kernel)
            _check_rms(cache, [70], 2, qstd=std, kernel=kernel)
    finally:
        cache.free()


@pytest.mark.parametrize("kernel", ["split", "tmem"])
@pytest.mark.parametrize("size", [0, 8, 10, 12, 14])
def test_attention_beside_a_page_of_zeros(gpu, size, kernel):
    """a page of zero values costs the other pages' weights nothing, however small their values are (its keys are zero as well in the second head)"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 2, 1, 6)
    rng = np.random.default_rng(size)
    k = rng.normal(0, 1, (2, 320, 128)); v = rng.normal(0, 2.0 ** -size, (2, 320, 128))
    v[:, :64] = 0; v[:, 192:256] = 0; k[1, :64] = 0
    try:
        cache.write([320], [k.astype(np.float16)], [v.astype(np.float16)], rows=False)
        scales = gpu.read(cache.d["scales"]["buf"]).view(np.float32)[:cache.pages * 4].reshape(cache.pages, 2, 2)
        assert (scales[cache.table[0, 0], :, 1] == _quantise(np.full((64, 128), 2.0 ** -24))[1]).all() and scales[cache.table[0, 0], 1, 0] == scales[cache.table[0, 3], 0, 1]
        for n in (2, 60): _check_rms(cache, [n], 4, kernel=kernel)
    finally:
        cache.free()


@pytest.mark.parametrize("kernel", ["split", "tmem"])
@pytest.mark.parametrize("size", [0, 7, 10, 12, 14, 16])
def test_attention_beside_a_tail_of_small_values(gpu, size, kernel):
    """the unfinished page's values are no larger than the others': its weights cost theirs nothing"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 2, 2, 6)
    rng = np.random.default_rng(size)
    lens = [101, 4 * 64 + 37]
    k, v = ([rng.normal(0, s, (2, L, 128)).astype(np.float16) for L in lens] for s in (1.0, 2.0 ** -size))
    v[1][1, 256:] = 0
    try:
        cache.write(lens, k, v)
        for n in ([1, 2], [40, 70]): _check_rms(cache, n, 4, kernel=kernel)
    finally:
        cache.free()


def test_rope_refuses_what_ends_in_no_number(gpu):
    """a factor that fp32 does not hold, frequencies whose angles are infinite: refused; what is large or small and still a number is not"""
    import p0pc0rn_kernels_b200 as P
    b, lens = gpu.upload(np.ones((2, 3, 128), np.float16)), gpu.upload(np.array([4000000000], np.uint32))
    args = {"x": {"buf": b}, "H": 2, "M": 3, "seqs": 1, "lens": {"buf": lens}, "mode": "half"}
    try:
        for kw in (dict(mscale=1e39), dict(mscale=-1e300), dict(mscale=float("nan")), dict(theta=5e-324), dict(factor=1e-308), dict(theta=1e-300, factor=1e-20), dict(factor=1e-308, original=1.0)):
            with pytest.raises(ValueError, match="rope"): P.rope(gpu, {**args, **kw})
        for kw in (dict(theta=1e300), dict(factor=1e300), dict(theta=1e-200), dict(factor=1e-200), dict(mscale=0.5)): P.rope(gpu, {**args, **kw})
        got = gpu.read(b).view(np.float16)[:2 * 3 * 128]
        # (five turns of pairs of ones, each off by the rounding to fp16, one of them by half: no pair is longer than sqrt 2)
        assert np.isfinite(got).all() and np.abs(got).max() <= 0.5 * 2.0 ** 0.5 * (1 + 2.0 ** -11) ** 5 + 5 * 2.0 ** -25
        assert not gpu.lost
    finally:
        gpu.free(b); gpu.free(lens)


def _pages_apart(cache, lens, seed=1, std=1.0):
    """fills a cache with values that have a mean of their own in each page, and keys of a size of their own"""
    rng = np.random.default_rng(seed)
    k, v = [], []
    for L in lens:
        n = -(-int(L) // PAGE)
        size, mean = np.exp(rng.normal(0, 0.1, (cache.Hkv, n, 1))), rng.normal(0, 1, (cache.Hkv, n, 128))
        spread = np.exp(rng.normal(0, 0.3, (cache.Hkv, n, 1)))
        def tokens(scale, add):
            x = rng.normal(0, std, (cache.Hkv, n * PAGE, 128))
            return (x * np.repeat(scale, PAGE, 1) + np.repeat(add, PAGE, 1))[:, :int(L)].astype(np.float16)
        k.append(tokens(size, 0 * mean)); v.append(tokens(0.7 * spread, mean))
    cache.write(list(lens), k, v)


LONG = [
    # (first three: more than 32 and 64 pages of an item in a warp's share, more than 32 pairs of pages in a block's: test_cache_plan.py)
    dict(label="long contexts among many: shares of many pages", Hkv=8, group=16, lens=[400, 20000, 37], news=[310, 12, 20], kernel="split"),
    dict(label="a long prompt over a long context: blocks with many pairs of an item", Hkv=8, group=4, lens=[8000], news=[1100], kernel="tmem"),
    dict(label="a chunk of a prompt, split keys: shares of more pages still", Hkv=4, group=16, lens=[9000], news=[700], kernel="split"),
    dict(label="one token, four pages per warp", Hkv=4, group=4, lens=[40000], news=[1], kernel="split"),
    dict(label="few queries over a long context", Hkv=2, group=4, lens=[20000], news=[70], kernel="tmem"),
    dict(label="few queries over a long context, split keys", Hkv=2, group=4, lens=[20000], news=[70], kernel="split"),
    dict(label="several long contexts", Hkv=8, group=4, lens=[3000, 9001, 5000, 64 * 70], news=[1, 2, 1, 1], kernel="split"),
    dict(label="several contexts, prompts", Hkv=2, group=7, lens=[3000, 5001, 64 * 30], news=[40, 90, 150], kernel="tmem"),
]


@pytest.mark.parametrize("c", LONG, ids=lambda c: c["label"])
def test_attention_reads_every_page_once(gpu, c):
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, c["Hkv"], len(c["lens"]), -(-max(c["lens"]) // PAGE), seed=13)
    try:
        _pages_apart(cache, c["lens"])
        some = [(b, pg) for b, L in enumerate(c["lens"]) for pg in sorted({0, 1, 31, 32, 33, 64, L // PAGE // 2, (L - 1) // PAGE - 1, (L - 1) // PAGE}) if pg <= (L - 1) // PAGE and L > 100]
        _check_rms(cache, c["news"], c["group"], kernel=c["kernel"], without=some)
        _check_rms(cache, c["news"], c["group"], kernel=c["kernel"], window=2500, sinks=70)
    finally:
        cache.free()


ROPE_MORE = [
    dict(label="many heads per thread, half", mode="half", H=41, M=4200, seqs=3),
    dict(label="many heads per thread, interleaved", mode="interleaved", H=40, M=4200, seqs=2),
    dict(label="many heads per thread, half, odd part", mode="half", rot=38, H=23, M=1700, seqs=2),
    dict(label="part of the head, many heads", mode="half", rot=64, H=33, M=3001, seqs=1),
    dict(label="equal counts", mode="half", H=3, M=35, seqs=5, rows=False),
    dict(label="equal counts, odd part", mode="half", rot=10, H=3, M=35, seqs=5, rows=False),
    dict(label="equal counts, interleaved, many heads", mode="interleaved", H=40, M=4200, seqs=100, rows=False),
    dict(label="40 sequences, some empty", mode="half", H=3, M=211, seqs=40),
    dict(label="300 sequences, some empty", mode="interleaved", H=2, M=1201, seqs=300),
    dict(label="300 sequences, odd part", mode="half", rot=22, H=2, M=1201, seqs=300),
    dict(label="32 sequences", mode="half", H=2, M=77, seqs=32),
]


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("c", ROPE_MORE, ids=lambda c: c["label"])
def test_rope_heads_and_sequences(gpu, c, inplace):
    """more heads than a thread holds at once, equal counts, more sequences than a warp looks at; tolerances as in test_rope"""
    import p0pc0rn_kernels_b200 as P
    rng = np.random.default_rng(3)
    H, M, seqs, rot, equal = c["H"], c["M"], c["seqs"], c.get("rot", 128), c.get("rows") is False
    cuts = np.arange(seqs + 1) * (M // seqs) if equal else np.concatenate([[0], np.sort(rng.integers(0, M + 1, seqs - 1)), [M]])
    if not equal and seqs > 5: cuts[3] = cuts[2]; cuts[-2] = M                                 # (sequences without tokens, the last one too)
    offs = cuts.astype(np.uint32); news = np.diff(cuts)
    lens = (news + rng.integers(0, 100000, seqs)).astype(np.uint32)
    x = rng.normal(0, 1, (H, M, 128)).astype(np.float16)
    xb, lb = gpu.upload(x), gpu.upload(lens)
    yb, rb = (None if inplace else gpu.upload(np.full((H, M + 3, 128), 0x7E01, np.uint16))), (None if equal else gpu.upload(offs))
    try:
        P.rope(gpu, {"x": {"buf": xb}, "y": {"buf": yb, "ld": M + 3} if yb else None, "H": H, "M": M, "seqs": seqs, "lens": {"buf": lb}, "rows": {"buf": rb} if rb else None, "mode": c["mode"], "rot": rot})
        got = gpu.read(yb or xb).view(np.float16)[:H * (M if inplace else M + 3) * 128].reshape(H, -1, 128)
        if not inplace: assert (got[:, M:].view(np.uint16) == 0x7E01).all()
        got = got[:, :M]
        pos = np.concatenate([np.arange(L - n, L, dtype=np.float64) for L, n in zip(lens.astype(np.int64), news)])
        ang = pos[:, None] * _freq(rot); cs, sn = np.cos(ang), np.sin(ang)
        first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if c["mode"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
        for h in range(H):
            z = x[h].astype(np.float64); want = z.copy(); mag = np.zeros_like(z)
            a, b = z[:, first], z[:, second]
            want[:, first], want[:, second] = a * cs - b * sn, a * sn + b * cs
            mag[:, first] = mag[:, second] = np.abs(a) + np.abs(b)
            tol = np.abs(want) * 2.0 ** -11 + 2.0 ** -25 + mag * (6 * 2.0 ** -24 + float(pos.max()) * 8 * 2.0 ** -53)
            assert (np.abs(got[h].astype(np.float64) - want) <= tol).all(), h
            assert np.array_equal(got[h][:, rot:], x[h][:, rot:])
    finally:
        for t in (xb, yb, lb, rb): gpu.free(t)


@pytest.mark.parametrize("kernel", ["split", "tmem"])
def test_attention_over_the_largest_values_stays_finite(gpu, kernel):
    """values of the largest fp16 of either sign (infinities among them, which are stored so): their means are no infinities"""
    import p0pc0rn_kernels_b200 as P
    for L, news in ((64, (3, 40)), (40, (3, 40)), (230, (3, 100)), (20000, (3, 70))):
        cache = Cache(P, gpu, 2, 1, -(-L // PAGE))
        rng = np.random.default_rng(L)
        k = rng.normal(0, 1, (2, L, 128)).astype(np.float16)
        v = np.full((2, L, 128), 65504, np.float16); v[:, ::3, 5] = np.inf; v[1, :, 64:] = -65504; v[1, 1::7, 70] = -np.inf
        try:
            cache.write([L], [k], [v], rows=False)
            for n in news:
                out, q, offs = _attend(cache, [n], 4, kernel=kernel)
                want = np.broadcast_to(np.repeat(_clean(v[:, 0]), 4, 0).astype(np.float64), out.shape)
                # (codes of 127 times a scale rounded up by at most 2^-11, weights off by 2^-11 + 1e-4, the result's rounding; never beyond the largest fp16)
                assert np.isfinite(out).all() and np.abs(out.astype(np.float64) - want).max() <= 65504 * (3 * 2.0 ** -11 + 1e-4)
        finally:
            cache.free()


@pytest.mark.parametrize("kernel", [None, "split", "tmem"])
def test_attention_of_empty_batches(gpu, kernel):
    """no sequence has new tokens; and as many sequences as a call can have, most of them without any"""
    import p0pc0rn_kernels_b200 as P
    cache = Cache(P, gpu, 2, 1024, 2)
    try:
        cache.fill([70 if b % 100 == 7 or b == 1023 else 0 for b in range(1024)])
        out, _, _ = _attend(cache, [0] * 1024, 4, extra=5, kernel=kernel)
        assert out.shape[0] == 5                                                               # (and nothing was written: _attend looks)
        _check(cache, [1 + b % 3 if cache.lens[b] else 0 for b in range(1024)], 4, extra=2, kernel=kernel)
        _check(cache, [70 if cache.lens[b] else 0 for b in range(1024)], 4, kernel=kernel)
        gpu.done()
    finally:
        cache.free()
