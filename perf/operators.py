"""The 8-bit key/value cache, the attention over it and rotary positions, as measurable cases.

  rope    rotary positions of a step's heads: both layouts, whole or part of a head, plain or scaled for long contexts
  write   a step's (or a prompt's) keys and values into the cache, and the touched pages read back
  read    whole sequences read back from the cache as fp16 keys and values
  attn    attention of the newest tokens over the cache: one token or a chunk of a prompt per sequence, with or without a sliding
          window and first tokens that stay visible

The cache: pages of 64 tokens, found through a table per sequence; per page and kv head 64 x 128 8-bit codes for K and for V, each with one
fp32 scale (the largest magnitude / 127, rounded up to 12 significant bits); the tokens of a sequence's last, unfinished page stay in
fp16 (the tail).  `lens` counts the newest tokens too: a call's n tokens of a sequence are its last n.  Codes are stored with 128 added, in
the order  K: [key / 16][key bit 1][d / 64][key bits 2..3][key bit 0][d % 64],  V: [d][key bits 2..3][key / 16][key bits 0..1].
"""
import math
import random

import torch

own = False
PAGE, D = 64, 128
_context = None


# ------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one user's decoding step, ordinary layout: the smallest call, all latency
        {"name": "rope_b1", "op": "rope", "heads": 40, "seqs": 1, "new": 1, "past": 4000, "spread": False, "ragged": False, "mode": "half", "rot": 128, "theta": 10000.0,
         "factor": 1.0, "original": 0, "mscale": 1.0, "salt": 1},
        # prompts of several users, a quarter of the head left alone, frequencies scaled by parts, positions far out
        {"name": "rope_prompts_far", "op": "rope", "heads": 40, "seqs": 5, "new": 1000, "past": 900000, "spread": True, "ragged": True, "mode": "interleaved", "rot": 96, "theta": 500000.0,
         "factor": 8.0, "original": 8192, "mscale": 1.2, "salt": 2},
        # one step of 64 users: 64 tokens, of which three complete their page
        {"name": "write_step_b64", "op": "write", "hkv": 8, "seqs": 64, "new": 1, "past": 4000, "spread": True, "ragged": False, "salt": 20},
        # a chunk of a prompt that begins and ends inside a page
        {"name": "write_prompt_8000", "op": "write", "hkv": 8, "seqs": 1, "new": 8000, "past": 101, "spread": False, "ragged": False, "salt": 4},
        # a short conversation read back
        {"name": "read_300", "op": "read", "hkv": 8, "seqs": 1, "past": 300, "spread": False, "salt": 5},
        # several long ones, for an fp16 consumer
        {"name": "read_b4_20000", "op": "read", "hkv": 8, "seqs": 4, "past": 20000, "spread": True, "salt": 6},
        # one user, one token, a short context: latency
        {"name": "attn_b1_300", "op": "attn", "hkv": 8, "group": 4, "seqs": 1, "new": 1, "past": 300, "spread": False, "ragged": False, "window": 0, "sinks": 0, "salt": 7},
        # one user, one token, a long context
        {"name": "attn_b1_32000", "op": "attn", "hkv": 8, "group": 4, "seqs": 1, "new": 1, "past": 32000, "spread": False, "ragged": False, "window": 0, "sinks": 0, "salt": 8},
        # 64 users of mixed context lengths, one token each
        {"name": "attn_b64_4096", "op": "attn", "hkv": 8, "group": 4, "seqs": 64, "new": 1, "past": 4096, "spread": True, "ragged": False, "window": 0, "sinks": 0, "salt": 9},
        # 16 users with far longer contexts than the window; one head per kv head, and a few tokens of speculation each
        {"name": "attn_window_b16", "op": "attn", "hkv": 16, "group": 1, "seqs": 16, "new": 5, "past": 16000, "spread": True, "ragged": True, "window": 2048, "sinks": 4, "salt": 10},
        # a chunk of a prompt over what the cache holds already
        {"name": "attn_prompt_2000", "op": "attn", "hkv": 8, "group": 4, "seqs": 1, "new": 2000, "past": 6100, "spread": False, "ragged": False, "window": 0, "sinks": 0, "salt": 11},
        # ragged prompts from their first token on, under a sliding window
        {"name": "attn_prompts_window", "op": "attn", "hkv": 4, "group": 7, "seqs": 4, "new": 2500, "past": 0, "spread": False, "ragged": True, "window": 1000, "sinks": 8, "salt": 12},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op, salt = rng.choice(["attn"] * 5 + ["write"] * 2 + ["read", "rope"]), rng.randrange(1 << 20)
    seqs = _log(rng, 1, 128)
    if op == "rope":
        return {"op": op, "heads": _log(rng, 2, 80), "seqs": seqs, "new": _log(rng, 1, 4000), "past": _log(rng, 1, 1000000), "spread": rng.random() < 0.5, "ragged": rng.random() < 0.5,
                "mode": rng.choice(["half", "interleaved"]), "rot": rng.choice([128, 128, 64, 32, rng.randrange(1, 65) * 2]), "theta": rng.choice([10000.0, 500000.0, 1000000.0]),
                "factor": rng.choice([1.0, 4.0, 8.0, 32.0]), "original": rng.choice([0, 4096, 8192]), "mscale": rng.choice([1.0, 1.0, 1.35]), "salt": salt}
    hkv = rng.choice([1, 2, 3, 4, 8, 8, 16])
    if op == "read":
        return {"op": op, "hkv": hkv, "seqs": seqs, "past": _log(rng, 16, 40000), "spread": rng.random() < 0.7, "salt": salt}
    step = rng.random() < 0.6
    new = rng.choice([1, 1, 1, 2, 4, 7]) if step else _log(rng, 8, 8000)
    past = rng.choice([0, _log(rng, 1, 60000), _log(rng, 64, 60000), _log(rng, 500, 60000), _log(rng, 500, 60000)])
    c = {"op": op, "hkv": hkv, "seqs": seqs, "new": new, "past": past, "spread": rng.random() < 0.7, "ragged": new > 1 and rng.random() < 0.7, "salt": salt}
    if op == "attn":
        w = rng.choice([0, 0, _log(rng, 1, 8000)])
        c.update(group=rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 12, 16]), window=w, sinks=rng.choice([0, 4, _log(rng, 1, 200)]) if w else 0)
    return c


def draw(rng):
    """a case of the same kinds over the whole range, at most as much work as the largest listed one and a bounded plain form"""
    most = {op: [max(work(c)[k] for c in listed() if c["op"] == op) for k in ("bytes", "flops")] for op in ("rope", "write", "read", "attn")}
    while True:
        c = _draw(rng)
        w, (lens, news) = work(c), _lens(c)
        longest, n = max(lens), max(news)
        if w["bytes"] <= most[c["op"]][0] and w["flops"] <= most[c["op"]][1] and len(lens) * c.get("hkv", 1) * longest <= 5e6 and len(lens) * c.get("hkv", 1) * c.get("group", 1) * n * longest <= 1e9:
            return c


def _lens(c):
    """(tokens of each sequence with the newest, how many of them are new); a `read` reads all of them"""
    r, past, new = random.Random(c["salt"]), c["past"], c.get("new", 0)
    pasts = [past if not c["spread"] else r.randint((past + 3) // 4, past) for _ in range(c["seqs"])]
    news = [new if i == 0 or not c.get("ragged") else r.randint(1, new) for i in range(c["seqs"])]
    if c["op"] == "read": return pasts, pasts
    return [p + n for p, n in zip(pasts, news)], news


# ------------------------------------------------------------------------------------------------------------- the inputs
def _up12(s):
    """positive fp32 values rounded up to 12 significant bits"""
    return ((s.view(torch.int32) + 4095) & ~4095).view(torch.float32)


class _State:
    """what a program holds before the call: the cache, the step's tensors, the argument dicts of its calls"""

    def __init__(self, case, seed):
        self.c = case
        self.gen = torch.Generator(device="cuda"); self.gen.manual_seed(seed)
        lens, news = _lens(case)
        self.lens_list, self.news_list, self.M = lens, news, sum(news)
        self.calls = self.gpu = None
        self.wrapped = []
        self.lens = self.ints(lens)
        offs = [0]
        for n in news: offs.append(offs[-1] + n)
        self.offs, self.row_offs = offs, self.ints(offs)              # (a program with as many rows for each sequence need not pass them)
        self.equal = len(set(news)) == 1

    def ints(self, v):
        return torch.tensor(v, device="cuda", dtype=torch.int32)

    def randn(self, *shape, std=1.0):
        return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, std, generator=self.gen).half()

    def cache(self, extra=0):
        """a cache that holds the sequences: codes as quantised normal values leave them, a spread of scales, pages in any order"""
        c = self.c
        hkv, self.maxp = c["hkv"], max(1, -(-max(self.lens_list) // PAGE)) + extra
        self.pages = c["seqs"] * self.maxp
        self.codes = torch.empty(self.pages, hkv, 2, PAGE * D, device="cuda", dtype=torch.uint8)
        step = max(1, (1 << 26) // (hkv * 2 * PAGE * D))
        for p in range(0, self.pages, step):
            part = self.codes[p:p + step]
            part.copy_(torch.empty(part.shape, device="cuda", dtype=torch.float16).normal_(128.0, 29.0, generator=self.gen).round_().clamp_(1, 255))
        self.scales = _up12(torch.empty(self.pages, hkv, 2, device="cuda").normal_(0.0, 0.3, generator=self.gen).exp_().mul_(4.3 / 127))
        self.tail = self.randn(c["seqs"], hkv, 2, PAGE * D)
        self.table = torch.randperm(self.pages, device="cuda", generator=self.gen).to(torch.int32).view(c["seqs"], self.maxp)

    def wrap(self, t):
        b = self.gpu.wrap(t.data_ptr(), t.numel() * t.element_size())
        self.wrapped.append(b)
        return {"buf": b}

    def cache_args(self):
        return {"Hkv": self.c["hkv"], "pages": self.pages, "seqs": self.c["seqs"], "maxPages": self.maxp, "codes": self.wrap(self.codes), "scales": self.wrap(self.scales),
                "tail": self.wrap(self.tail), "table": self.wrap(self.table), "lens": self.wrap(self.lens)}

    def __del__(self):
        for b in self.wrapped: self.gpu.free(b)


def prepare(case, seed):
    s = _State(case, seed)
    op = case["op"]
    if op == "rope":
        s.x = s.randn(case["heads"], s.M, D); s.y = torch.zeros_like(s.x)
        return s
    # (`write`: as many pages more as a plain form needs to treat every sequence alike)
    s.cache(extra=(case["new"] + PAGE - 1) // PAGE + 1 if op == "write" else 0)
    if op == "write":
        s.k = s.randn(case["hkv"], s.M, D); s.v = s.randn(case["hkv"], s.M, D)
        # the pages that this call touches, whole: from the first one's first token to the newest token
        back = [L - (L - n) // PAGE * PAGE for L, n in zip(s.lens_list, s.news_list)]
        offs = [0]
        for n in back: offs.append(offs[-1] + n)
        s.back_offs, s.back_M = s.ints(offs), offs[-1]
        s.k_back = torch.zeros(case["hkv"], s.back_M, D, device="cuda", dtype=torch.float16); s.v_back = torch.zeros_like(s.k_back)
    elif op == "read":
        s.k = torch.zeros(case["hkv"], s.M, D, device="cuda", dtype=torch.float16); s.v = torch.zeros_like(s.k)
    else:
        s.q = s.randn(case["hkv"] * case["group"], s.M, D)
        s.o = torch.zeros(s.M, case["hkv"] * case["group"] * D, device="cuda", dtype=torch.float16)
    return s


# ------------------------------------------------------------------------------------------------------------- the framework's calls
def _calls(s):
    """a program's handles and argument dicts, made once"""
    global _context
    import p0pc0rn_kernels_b200 as P
    if _context is None:
        _context = P.createGpu({"device": 0, "stream": torch.cuda.current_stream().cuda_stream})
    s.gpu, c, op = _context, s.c, s.c["op"]
    rows = None if s.equal else s.wrap(s.row_offs)
    if op == "rope":
        return [(P.rope, {"x": s.wrap(s.x), "y": s.wrap(s.y), "H": c["heads"], "M": s.M, "seqs": c["seqs"], "lens": s.wrap(s.lens), "rows": rows, "mode": c["mode"], "rot": c["rot"],
                          "theta": c["theta"], "factor": c["factor"], "original": c["original"], "mscale": c["mscale"]})], s.y
    cache = s.cache_args()
    if op == "write":
        return [(P.cacheWrite, {"cache": cache, "k": s.wrap(s.k), "v": s.wrap(s.v), "M": s.M, "rows": rows}),
                (P.cacheRead, {"cache": cache, "k": s.wrap(s.k_back), "v": s.wrap(s.v_back), "M": s.back_M, "rows": s.wrap(s.back_offs)})], (s.k_back, s.v_back)
    if op == "read":
        return [(P.cacheRead, {"cache": cache, "k": s.wrap(s.k), "v": s.wrap(s.v), "M": s.M, "rows": rows})], (s.k, s.v)
    return [(P.cacheAttention, {"cache": cache, "q": s.wrap(s.q), "o": s.wrap(s.o), "Hq": c["hkv"] * c["group"], "M": s.M, "rows": rows, "new": c["new"], "window": c["window"],
                                "sinks": c["sinks"]})], s.o


def run(state):
    if own:
        if state.calls is None: state.calls = _calls(state)
        for op, args in state.calls[0]: op(state.gpu, args)
        return state.calls[1]
    return {"rope": _plain_rope, "write": _plain_write, "read": _plain_read, "attn": _plain_attn}[state.c["op"]](state)


# ------------------------------------------------------------------------------------------------------------- the plain forms
def _ordered(kv):
    """[..., 2, 8192] in the cache's order -> [..., 2, 64 keys, 128]"""
    lead = kv.shape[:-2]; n = len(lead)
    k = kv[..., 0, :].reshape(*lead, 4, 2, 2, 4, 2, 64).permute(*range(n), n, n + 3, n + 1, n + 4, n + 2, n + 5).reshape(*lead, PAGE, D)
    v = kv[..., 1, :].reshape(*lead, D, 4, 4, 4).permute(*range(n), n + 2, n + 1, n + 3, n).reshape(*lead, PAGE, D)
    return torch.stack([k, v], -3)


def _stored(kv):
    """the inverse of _ordered"""
    lead = kv.shape[:-3]; n = len(lead)
    k = kv[..., 0, :, :].reshape(*lead, 4, 4, 2, 2, 2, 64).permute(*range(n), n, n + 2, n + 4, n + 1, n + 3, n + 5).reshape(*lead, PAGE * D)
    v = kv[..., 1, :, :].reshape(*lead, 4, 4, 4, D).permute(*range(n), n + 3, n + 1, n, n + 2).reshape(*lead, PAGE * D)
    return torch.stack([k, v], -2)


def _rows(s, offs, M):
    """(sequence, index among its rows) of M rows"""
    r = torch.arange(M, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(offs[1:], r, right=True)
    return b, (r - offs[b]).long()


def _held(s, first, count):
    """fp32 [seqs][hkv][2][count * 64][128] of pages first[b] .. first[b] + count of every sequence"""
    at = first[:, None] + torch.arange(count, device="cuda")
    page = s.table.long().gather(1, at.clamp(max=s.maxp - 1))
    x = _ordered(s.codes[page].float() - 128.0) * s.scales[page][..., None, None]                 # [seqs][count][hkv][2][64][128]
    x = torch.where((at == (s.lens // PAGE).long()[:, None])[..., None, None, None, None], _ordered(s.tail.float())[:, None], x)
    return x.permute(0, 2, 3, 1, 4, 5).reshape(x.shape[0], x.shape[2], 2, count * PAGE, D)


def _plain_rope(s):
    c = s.c; b, i = _rows(s, s.row_offs, s.M)
    half = c["rot"] // 2
    f = torch.tensor(_frequencies(c), device="cuda", dtype=torch.float64)
    pos = (s.lens[b] - (s.row_offs[1:] - s.row_offs[:-1])[b]).double() + i.double()
    ang = pos[:, None] * f                                                                         # (64 bits: positions go far)
    cos, sin = (ang.cos() * c["mscale"]).float(), (ang.sin() * c["mscale"]).float()
    x = s.x.float(); y = x.clone()
    first, second = (slice(0, half), slice(half, 2 * half)) if c["mode"] == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    y[..., first] = x[..., first] * cos - x[..., second] * sin
    y[..., second] = x[..., first] * sin + x[..., second] * cos
    return s.y.copy_(y)


def _plain_write(s):
    n = s.row_offs[1:] - s.row_offs[:-1]; old = s.lens - n
    first, count = (old // PAGE).long(), (s.c["new"] + PAGE - 1) // PAGE + 1
    pos = first[:, None] * PAGE + torch.arange(count * PAGE, device="cuda")                        # every touched page's tokens
    row = (s.row_offs[:-1, None] + pos - old[:, None]).clamp(0, s.M - 1)
    new = torch.stack([s.k, s.v], 1)[:, :, row].permute(2, 0, 1, 3, 4).float()                     # [seqs][hkv][2][tokens][128]
    new = torch.where(torch.isnan(new), torch.zeros_like(new), new.clamp(-65504.0, 65504.0))
    seqs, hkv = new.shape[:2]
    tail = _ordered(s.tail.float())
    x = torch.where((pos < old[:, None])[:, None, None, :, None], tail.repeat(1, 1, 1, count, 1), new)
    x = x.view(seqs, hkv, 2, count, PAGE, D).permute(0, 3, 1, 2, 4, 5)                             # [seqs][page][hkv][2][64][128]
    amax = x.abs().amax((-1, -2))
    scale = torch.where(amax > 0, _up12(amax / 127.0), torch.ones_like(amax))
    code = (x / scale[..., None, None]).round()
    at = first[:, None] + torch.arange(count, device="cuda")
    full = (at + 1) * PAGE <= s.lens[:, None]
    page = s.table.long().gather(1, at)
    s.codes[page] = torch.where(full[..., None, None, None], _stored(code + 128.0).to(torch.uint8), s.codes[page])
    s.scales[page] = torch.where(full[..., None, None], scale, s.scales[page])
    # the unfinished page, if any: its new tokens join (or begin) the tail
    last = (s.lens // PAGE).long()
    t = torch.arange(PAGE, device="cuda") + last[:, None] * PAGE
    took = (t >= old[:, None]) & (t < s.lens[:, None])
    row = (s.row_offs[:-1, None] + t - old[:, None]).clamp(0, s.M - 1)
    end = torch.stack([s.k, s.v], 1)[:, :, row].permute(2, 0, 1, 3, 4).float()
    end = torch.where(torch.isnan(end), torch.zeros_like(end), end.clamp(-65504.0, 65504.0))
    s.tail.copy_(_stored(torch.where(took[:, None, None, :, None], end, tail)))
    # read back
    held = _held(s, first, count)
    b, i = _rows(s, s.back_offs, s.back_M)
    kv = held[b, :, :, i].permute(2, 1, 0, 3).half()
    return s.k_back.copy_(kv[0]), s.v_back.copy_(kv[1])


def _plain_read(s):
    held = _held(s, torch.zeros_like(s.lens, dtype=torch.long), s.maxp)
    b, i = _rows(s, s.row_offs, s.M)
    kv = held[b, :, :, i].permute(2, 1, 0, 3).half()
    return s.k.copy_(kv[0]), s.v.copy_(kv[1])


def _plain_attn(s):
    c = s.c; hkv, g, seqs, nmax = c["hkv"], c["group"], c["seqs"], c["new"]
    held = _held(s, torch.zeros_like(s.lens, dtype=torch.long), s.maxp)
    key = torch.arange(s.maxp * PAGE, device="cuda")
    k, v = held[:, :, 0], torch.where((key < s.lens[:, None])[:, None, :, None], held[:, :, 1], torch.zeros((), device="cuda"))
    n = s.row_offs[1:] - s.row_offs[:-1]
    i = torch.arange(nmax, device="cuda")
    q = s.q[:, (s.row_offs[:-1, None] + torch.minimum(i, (n - 1)[:, None])).long()].float()        # [heads][seqs][new][128]
    q = q.view(hkv, g, seqs, nmax, D).permute(2, 0, 1, 3, 4).reshape(seqs, hkv, g * nmax, D)
    sc = torch.matmul(q, k.transpose(-1, -2)).view(seqs, hkv, g, nmax, -1) / math.sqrt(D)
    p = (s.lens - n)[:, None] + i                                                                  # positions [seqs][new]
    see = key <= p[..., None]
    if c["window"]: see = see & ((key > p[..., None] - c["window"]) | (key < c["sinks"]))
    sc = sc.masked_fill_(~see[:, None, None], float("-inf"))
    sc = (sc - sc.amax(-1, keepdim=True)).exp_()
    sc = sc / sc.sum(-1, keepdim=True)
    o = torch.matmul(sc.view(seqs, hkv, g * nmax, -1), v).view(seqs, hkv, g, nmax, D).permute(0, 3, 1, 2, 4).reshape(seqs, nmax, hkv * g * D)
    b, r = _rows(s, s.row_offs, s.M)
    return s.o.copy_(o[b, r])


# ------------------------------------------------------------------------------------------------------------- in 64 bits
def _frequencies(c):
    """the angle that each pair turns by from one position to the next"""
    out = []
    for i in range(c["rot"] // 2):
        f = c["theta"] ** (-2.0 * i / c["rot"])
        if c["factor"] != 1.0:
            part = 0.0
            if c["original"]: part = min(1.0, max(0.0, (c["original"] * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)))
            f = f * (part + (1.0 - part) / c["factor"])
        out.append(f)
    return out


def _offsets():
    """where a page's (key, d) lies: for K, for V"""
    key = torch.arange(PAGE, device="cuda")[:, None]; d = torch.arange(D, device="cuda")[None]
    k = ((key // 16) * 2 + (key // 2) % 2) * 1024 + (d // 64) * 512 + ((key % 16) // 4 * 2 + key % 2) * 64 + d % 64
    v = d * 64 + (key // 4) % 4 * 16 + key // 16 * 4 + key % 4
    return k.reshape(-1), v.reshape(-1)


def _sequence(s, b, h):
    """K and V of sequence b, kv head h in 64 bits, [tokens][128]"""
    L = s.lens_list[b]; full = L // PAGE; got = []
    for w, off in enumerate(_offsets()):
        page = s.table[b, :full].long()
        x = (s.codes[page, h, w][:, off].double() - 128.0) * s.scales[page, h, w].double()[:, None]
        t = s.tail[b, h, w][off].double().view(PAGE, D)[:L - full * PAGE]
        got.append(torch.cat([x.reshape(-1, D), t]))
    return got


def exact(case, seed):
    s = prepare(case, seed); op = case["op"]
    pairs = range(case["seqs"])
    if op == "rope":
        y = s.x.double()
        for b in pairs:
            r0, r1 = s.offs[b], s.offs[b + 1]
            pos = torch.arange(s.lens_list[b] - (r1 - r0), s.lens_list[b], device="cuda", dtype=torch.float64)
            for i, f in enumerate(_frequencies(case)):
                a, z = (i, i + case["rot"] // 2) if case["mode"] == "half" else (2 * i, 2 * i + 1)
                turn = torch.polar(torch.full_like(pos, case["mscale"]), pos * f)
                both = torch.complex(s.x[:, r0:r1, a].double(), s.x[:, r0:r1, z].double()) * turn
                y[:, r0:r1, a], y[:, r0:r1, z] = both.real, both.imag
        return y
    if op in ("write", "read"):
        outs = [[], []]
        for b in pairs:
            L, n = s.lens_list[b], s.news_list[b]; old = L - n; head = [[], []]
            for h in range(case["hkv"]):
                kv = _sequence(s, b, h) if op == "read" else None
                for w in range(2):
                    if op == "read":
                        head[w].append(kv[w])
                        continue
                    t0 = old // PAGE * PAGE
                    x = torch.cat([s.tail[b, h, w][_offsets()[w]].double().view(PAGE, D)[:old - t0], (s.k, s.v)[w][h, s.offs[b]:s.offs[b + 1]].double()])
                    full = x.shape[0] // PAGE * PAGE
                    blk = x[:full].view(-1, PAGE * D)
                    a = blk.abs().amax(1, keepdim=True)
                    # the largest magnitude / 127 in 12 significant bits, rounded up: a power of two times a whole number of them
                    m, e = torch.frexp(a / 127.0)
                    sc = torch.where(a > 0, torch.ldexp(torch.ceil(m * 4096.0), e - 12), torch.ones_like(a))
                    head[w].append(torch.cat([((blk / sc).round() * sc).view(-1, D), x[full:]]))
            for w in range(2): outs[w].append(torch.stack(head[w]))
        return torch.cat(outs[0], 1), torch.cat(outs[1], 1)
    if work(case)["flops"] > 4e12: return None
    o, g = torch.zeros(s.o.shape, device="cuda", dtype=torch.float64), case["group"]
    for b in pairs:
        r0, r1, L = s.offs[b], s.offs[b + 1], s.lens_list[b]
        p = torch.arange(L - (r1 - r0), L, device="cuda")[:, None]; j = torch.arange(L, device="cuda")[None]
        hide = j > p
        if case["window"]: hide = hide | ((p - j >= case["window"]) & (j >= case["sinks"]))
        for h in range(case["hkv"]):
            k, v = _sequence(s, b, h)
            for x in range(h * g, h * g + g):
                z = (s.q[x, r0:r1].double() @ k.T) * D ** -0.5
                o[r0:r1, x * D:(x + 1) * D] = torch.softmax(z.masked_fill(hide, -math.inf), 1) @ v
    return o


# ------------------------------------------------------------------------------------------------------------- the accounting
def _seen(L, n, window, sinks):
    """(query, visible key) pairs of a sequence, and how many of its keys any query sees"""
    if not window: return n * L - n * (n - 1) / 2.0, L
    pairs = 0.0
    for p in range(L - n, L): pairs += min(p + 1, window) + min(sinks, max(0, p + 1 - window))
    lo = max(0, L - n + 1 - window)
    return pairs, L - lo + min(sinks, lo)


def work(case):
    c = case; lens, news = _lens(c); M = sum(news)
    if c["op"] == "rope": return {"bytes": 512.0 * c["heads"] * M, "flops": 6.0 * c["heads"] * M * c["rot"] / 2}
    hkv = c["hkv"]
    if c["op"] == "read":
        tail = sum(L % PAGE for L in lens)
        return {"bytes": hkv * ((256.0 + 512.0) * (M - tail) + 1024.0 * tail), "flops": 256.0 * hkv * (M - tail)}
    if c["op"] == "write":
        total = 0.0
        for L, n in zip(lens, news):
            old = L - n; done = L // PAGE * PAGE - old // PAGE * PAGE           # tokens that this call quantises
            back = L - old // PAGE * PAGE; end = L % PAGE
            total += 512.0 * n + 512.0 * (old % PAGE if done else 0) + 256.0 * done + 512.0 * min(n, end)       # written
            total += 256.0 * (back - end) + 512.0 * end + 512.0 * back                                          # read back
        return {"bytes": hkv * total, "flops": 5.0 * 256 * hkv * M}
    pairs = keys = 0.0
    for L, n in zip(lens, news):
        p, k = _seen(L, n, c["window"], c["sinks"])
        pairs += p
        tail = min(L % PAGE, k)
        keys += (k - tail) * 256.0 + tail * 512.0
    return {"bytes": keys * hkv + 512.0 * hkv * c["group"] * M, "flops": 512.0 * hkv * c["group"] * pairs}
