"""Timed cases of the operators around a cache that many sequences share or hold in 8 bits: quantising cache rows as they are
written and reading them back, attention over the quantised cache, attention of a batch that shares a long prefix, and the log
probabilities of the tokens that came out, with entropy and the top alternatives.

Listed cases (what each stands for in real use):
  cache_row1           the new token of one chat: the smallest write, where latency counts
  cache_prompt_t20000  a long prompt's rows, appended behind 13 cells that are there already
  q8_one_short         one sequence a few dozen tokens in, over the 8-bit cache
  q8_chat_b24          24 chats of uneven length at the 32-on-4-heads layout, an ordinary step of a server
  q8_batch_b128        128 sequences of up to 8192 tokens: the largest step over the 8-bit cache
  shared_b6            6 answers to one short prompt at the two-layer test model's head layout
  shared_b128          128 answers to a prompt of 8000 tokens, up to 500 tokens into each
  shared_long_b64      64 answers to a document of 30001 tokens at the 64-on-4-heads layout
  shared_q8_b32        32 answers to a prompt of 16000 tokens, each answer's own cells in 8 bits
  logp_one             the drawn token of one row of a 151936-token vocabulary with 5 alternatives
  logp_b64             those of 64 rows with 20 alternatives each
  logp_score_t1000     1000 rows of a text that is scored, without alternatives
Drawn cases also have 32-bit rows, head sizes of 64 and 256, windows, empty sequences and rows of which most tokens may not come.

A quantised cache is a tensor of bytes [pages][KV heads][68 head_dim]. A record of a page (32 cells) and a KV head holds, one after
the other: K's whole numbers q [head_dim / 32][4][4][4][2][8], where [m][a][b][c][t][j] is cell 8 b + 4 t + c, dim 32 m + 8 a + j;
K's scales d (fp16) [head_dim / 32][32 cells]; V's q [head_dim / 32][4][16][2][8], where [m][a][r][t][c] is cell 8 a + c, dim
32 m + 16 t + r; V's scales, as K's. A value is d q. d of 32 dims of a row is the smallest fp16 number that is no less than their
largest magnitude over 127, q = value / d rounded to the nearest whole number, halves to the even one.

The plain forms are written with elementary torch operations. What decides a whole number (scales, quotients, the order of the
alternatives) and the sums over a vocabulary are 64-bit there.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
BLOCK = 32  # cells of a page
VOCAB = 151936
# head layouts: (query heads, KV heads, head size)
HEADS = {"32x4": (32, 4, 128), "64x4": (64, 4, 128), "tiny": (4, 2, 64), "16x2": (16, 2, 256), "24x24": (24, 24, 64),
         "40x8": (40, 8, 128)}
MOST_CELLS = 128 * 8192   # cells of the largest step over the 8-bit cache
MOST_BYTES = 6.4e8        # and the bytes it reads, about
MOST_SCORES = 1.2e8       # query heads times cells of the largest shared prefix
MOST_ROWS = 20000         # rows of the largest write


def _cache(name, heads, T, mode, dtype):
    return {"name": name, "op": "cache", "heads": heads, "T": T, "mode": mode, "dtype": dtype}


def _q8(name, heads, B, lo, hi, window=0, sinks=0):
    """B sequences of lo .. hi cells (spread evenly, in an order of the case's own)."""
    return {"name": name, "op": "q8", "heads": heads, "B": B, "lo": lo, "hi": hi, "window": window, "sinks": sinks}


def _shared(name, heads, B, prefix, lo, hi, bits=16):
    return {"name": name, "op": "shared", "heads": heads, "B": B, "prefix": prefix, "lo": lo, "hi": hi, "bits": bits}


def _logp(name, B, V, top, masked=False):
    return {"name": name, "op": "logp", "B": B, "V": V, "top": top, "masked": masked}


def listed():
    return [_cache("cache_row1", "32x4", 1, "step", "f16"),
            _cache("cache_prompt_t20000", "32x4", 20000, "prompt", "f16"),
            _q8("q8_one_short", "32x4", 1, 45, 45),
            _q8("q8_chat_b24", "32x4", 24, 100, 4100),
            _q8("q8_batch_b128", "32x4", 128, 1000, 8192),
            _shared("shared_b6", "tiny", 6, 300, 0, 40),
            _shared("shared_b128", "32x4", 128, 8000, 1, 500),
            _shared("shared_long_b64", "64x4", 64, 30001, 10, 2000),
            _shared("shared_q8_b32", "40x8", 32, 16000, 100, 3000, bits=8),
            _logp("logp_one", 1, VOCAB, 5),
            _logp("logp_b64", 64, VOCAB, 20),
            _logp("logp_score_t1000", 1000, VOCAB, 0)]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cache", "q8", "q8", "shared", "shared", "logp"])
    heads = rng.choice(sorted(HEADS))
    H, kv, hd = HEADS[heads]
    if op == "cache":
        c = _cache("", heads, _log_int(rng, 1, max(1, MOST_ROWS * 512 // (kv * hd))), rng.choice(["step", "prompt"]),
                   rng.choice(["f16", "f32"]))
        if c["dtype"] == "f32":
            c["T"] = max(1, c["T"] // 2)
    elif op == "q8":
        cells = min(MOST_CELLS // 2, int(MOST_BYTES / (2.125 * kv * hd)))
        B = _log_int(rng, 1, 128)
        hi = _log_int(rng, 1, min(131072, max(1, cells // B)))
        c = _q8("", heads, B, rng.randint(0 if hi < 64 else 1, hi), hi)
        if rng.random() < 0.4:
            c["window"], c["sinks"] = _log_int(rng, 1, 8192), rng.choice([0, 1, 4, 33, 128])
    elif op == "shared":
        B = _log_int(rng, 1, 128)
        prefix = _log_int(rng, 1, min(65536, int(MOST_SCORES * 128 / (B * H * max(hd, 128)))))
        hi = _log_int(rng, 1, min(4096, max(1, int(MOST_BYTES / (16 * B * kv * hd)))))
        c = _shared("", heads, B, prefix, rng.randint(0, hi), hi, rng.choice([16, 16, 8]))
    else:
        V = rng.choice([VOCAB, _log_int(rng, 100, 200000), _log_int(rng, 1000, 200000)])
        c = _logp("", _log_int(rng, 1, max(1, min(2000, 500 * VOCAB // V))), V, rng.choice([0, 1, 5, 20, rng.randint(1, 32)]),
                  rng.random() < 0.3)
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------

def _lens(case):
    """The sequences' lengths: part of the case, not of the seed."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    n = [hi] if B == 1 else [lo + (hi - lo) * i // (B - 1) for i in range(B)]
    random.Random(B * 1000003 + lo * 31 + hi).shuffle(n)
    return n


def _visible(case, n):
    w, s = case["window"], case["sinks"]
    return n if w <= 0 or n <= w else min(n, w + min(s, n - w))


def _record_views(cache, hd):
    """(K's q, K's scales, V's q, V's scales) of a quantised cache, as views."""
    P, kv, _ = cache.shape
    m, half = hd // 32, cache.view(torch.float16)
    return (cache[:, :, :32 * hd].view(torch.int8).unflatten(2, (m, 4, 4, 4, 2, 8)),
            half[:, :, 16 * hd:17 * hd].unflatten(2, (m, BLOCK)),
            cache[:, :, 34 * hd:66 * hd].view(torch.int8).unflatten(2, (m, 4, 16, 2, 8)),
            half[:, :, 33 * hd:].unflatten(2, (m, BLOCK)))


def _tables(lens, g):
    """Lists of pages for these lengths, in the order sequences took and gave them back: any order."""
    pages = [-(-n // BLOCK) for n in lens]
    total = max(8, -(-sum(pages) // 8) * 8)
    order = torch.randperm(total, generator=g, device=DEV)[:max(1, sum(pages))].to(torch.int32)
    first = [0]
    for n in pages[:-1]:
        first.append(first[-1] + n)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    return total, dict(lens=i32(lens), first=i32(first), blocks=order, max_len=max(1, max(lens)))


def _random_f16_cache(total, kv, hd, randn):
    cells = total * BLOCK
    return (randn(kv, hd // 4, cells, 4, dtype=torch.float16), randn(kv, cells // 4, hd, 4, dtype=torch.float16))


def _random_q8_cache(total, kv, hd, g):
    """Whole numbers and scales as rows of about unit spread give them."""
    cache = torch.empty(total, kv, 68 * hd, dtype=torch.uint8, device=DEV)
    kq, kd, vq, vd = _record_views(cache, hd)
    for q, d in ((kq, kd), (vq, vd)):
        q.copy_((50.0 * torch.randn(q.shape, generator=g, device=DEV, dtype=torch.float16)).clamp_(-127, 127).round_())
        d.copy_((0.016 + 0.008 * torch.rand(d.shape, generator=g, device=DEV)).half())
    return cache


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    rand = lambda *s: torch.rand(*s, generator=g, device=DEV)
    randn = lambda *s, **k: torch.randn(*s, generator=g, device=DEV, **k)
    if case["op"] == "logp":
        B, V = case["B"], case["V"]
        x = 2.2 * randn(B, V)
        # a few hundred likely tokens above the rest
        n = min(300, V)
        at = rand(B, V).topk(n, dim=1).indices
        x.scatter_(1, at, (13.0 - 1.4 * torch.log(torch.arange(1, n + 1, device=DEV, dtype=torch.float32)) + 0.3 * randn(B, n)))
        if case["masked"]:  # an answer held to a form: most tokens may not come
            x.masked_fill_(rand(B, V) < 0.6, -math.inf)
            at[:, 0] = torch.argmax(x, 1)
        # what came: one of the likely tokens
        pick = at[:, :1] if case["masked"] else at.gather(1, torch.randint(0, n, (B, 1), generator=g, device=DEV))
        return dict(case=case, x=x, tokens=pick[:, 0].to(torch.int32).contiguous(), work=None)
    H, kv, hd = HEADS[case["heads"]]
    if case["op"] == "cache":
        T = case["T"]
        if case["mode"] == "prompt":
            pages = -(-(T + 13) // BLOCK)
            order = torch.randperm(pages + 3, generator=g, device=DEV)
            i = torch.arange(13, 13 + T, device=DEV)
            cells = order[i // BLOCK] * BLOCK + i % BLOCK
        else:
            pages = 2 * T
            cells = torch.randperm(pages + 3, generator=g, device=DEV)[:T] * BLOCK + torch.randint(0, BLOCK, (T,), generator=g, device=DEV)
        rows = randn(T, 2, kv, hd) * torch.exp(0.5 * randn(1, 2, kv, hd))  # K and V of a token side by side; some dims are larger
        rows = rows.half() if case["dtype"] == "f16" else rows
        return dict(case=case, hd=hd, kv=kv, k=rows[:, 0], v=rows[:, 1], cells=cells.to(torch.int32),
                    cache=torch.zeros(pages + 3, kv, 68 * hd, dtype=torch.uint8, device=DEV))
    lens = _lens(case)
    total, s = _tables(lens, g)
    s.update(case=case, H=H, kv=kv, hd=hd, q=(2.0 * randn(len(lens), H, hd)).half(), scale=1.0 / math.sqrt(hd), work=None)
    if case["op"] == "q8" or case["bits"] == 8:
        s["cache"] = _random_q8_cache(total, kv, hd, g)
    else:
        s["k"], s["v"] = _random_f16_cache(total, kv, hd, randn)
    if case["op"] == "shared":
        ptotal, p = _tables([case["prefix"]], g)
        pk, pv = _random_f16_cache(ptotal, kv, hd, randn)
        s["prefix"] = dict(k=pk, v=pv, length=p["lens"], blocks=p["blocks"], max_len=case["prefix"])
    return s


# ---- plain forms -------------------------------------------------------------------------------

def _f16_cells(k, v, page):
    """K [..., kv, hd, cells] and V [..., kv, cells, hd] in 32 bits of the pages `page` [..., n] of a cache in the cell layouts."""
    kv, hd = k.shape[0], v.shape[2]
    lead, n = page.shape[:-1], page.shape[-1]
    kp = k.unflatten(2, (-1, BLOCK)).permute(2, 0, 1, 4, 3).reshape(-1, kv, hd, BLOCK)          # [page][kv][hd][32]
    vp = v.unflatten(1, (-1, BLOCK // 4)).permute(1, 0, 2, 4, 3).reshape(-1, kv, BLOCK, hd)     # [page][kv][32][hd]
    return _in_order(kp[page.reshape(-1)].float(), vp[page.reshape(-1)].float(), lead, n)


def _q8_cells(cache, hd, page):
    lead, n = page.shape[:-1], page.shape[-1]
    kq, kd, vq, vd = _record_views(cache[page.reshape(-1)], hd)
    P, kv, m = kd.shape[:3]
    # [m][a][b][c][t][j] -> dim (m, a, j), cell (b, t, c), and [m][a][r][t][c] -> cell (a, c), dim (m, t, r)
    k = kq.permute(0, 1, 2, 3, 7, 4, 6, 5).reshape(P, kv, m, 32, BLOCK).float() * kd[:, :, :, None].float()
    v = vq.permute(0, 1, 3, 6, 2, 5, 4).reshape(P, kv, BLOCK, m, 32).float() * vd.transpose(2, 3)[..., None].float()
    return _in_order(k.reshape(P, kv, hd, BLOCK), v.reshape(P, kv, BLOCK, hd), lead, n)


def _in_order(k, v, lead, n):
    kv, hd = k.shape[1], k.shape[2]
    k = k.reshape(-1, n, kv, hd, BLOCK).permute(0, 2, 3, 1, 4).reshape(*lead, kv, hd, n * BLOCK)
    v = v.reshape(-1, n, kv, BLOCK, hd).permute(0, 2, 1, 3, 4).reshape(*lead, kv, n * BLOCK, hd)
    return k, v


def _own_cells(s):
    """K, V of the sequences' own cells, and which of them are visible."""
    c = s["case"]
    L = -(-s["max_len"] // BLOCK)
    page = s["first"][:, None] + torch.arange(L, device=DEV)
    page = s["blocks"][page.clamp(max=s["blocks"].numel() - 1)].long()
    k, v = _q8_cells(s["cache"], s["hd"], page) if "cache" in s else _f16_cells(s["k"], s["v"], page)
    i, n = torch.arange(L * BLOCK, device=DEV), s["lens"][:, None]
    seen = i < n
    if c["op"] == "q8" and c["window"] > 0:
        seen = seen & ((i >= n - c["window"]) | (i < c["sinks"]))
    return k, v, seen[:, None, None]


def _plain_q8(s):
    B, H = s["q"].shape[:2]
    k, v, seen = _own_cells(s)
    q = s["q"].float().reshape(B, s["kv"], H // s["kv"], s["hd"])
    score = ((q @ k) * s["scale"]).masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
    return out.reshape(B, H, s["hd"]).half()


def _plain_shared(s):
    B, H = s["q"].shape[:2]
    kv, hd, x = s["kv"], s["hd"], s["prefix"]
    k, v, seen = _own_cells(s)
    pk, pv = _f16_cells(x["k"], x["v"], x["blocks"][None].long())
    q = s["q"].float().reshape(B, kv, H // kv, hd)
    score = ((q @ k) * s["scale"]).masked_fill(~seen, -math.inf)
    rows = q.transpose(0, 1).reshape(kv, -1, hd)  # a KV head's queries of all sequences
    ps = (rows @ pk[0]) * s["scale"]
    ps = ps.masked_fill(torch.arange(ps.shape[-1], device=DEV) >= x["length"], -math.inf)
    ptop = ps.amax(-1).reshape(kv, B, -1, 1).transpose(0, 1)
    top = torch.maximum(score.amax(-1, keepdim=True), ptop)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(score - top)
    pp = torch.exp(ps - top.transpose(0, 1).reshape(kv, -1, 1))
    total = p.sum(-1, keepdim=True) + pp.sum(-1).reshape(kv, B, -1, 1).transpose(0, 1)
    out = p @ v + (pp @ pv[0]).reshape(kv, B, -1, hd).transpose(0, 1)
    return (out / torch.where(total == 0, torch.ones_like(total), total)).reshape(B, H, hd).half()


def _rounded(x, hd):
    """Scales [T][kv][hd / 32] and whole numbers [T][kv][hd / 32][32] of rows."""
    x = x.double().unflatten(2, (hd // 32, 32))
    most = x.abs().amax(-1)
    scale = (most / 127).half()
    scale = torch.where(scale.double() * 127 < most, (scale.view(torch.int16) + 1).view(torch.float16), scale)
    step = torch.where(scale == 0, torch.ones_like(scale), scale).double()[..., None]
    return scale, torch.round(x / step).to(torch.int8)


def _plain_cache(s):
    hd, dtype = s["hd"], s["k"].dtype
    kq, kd, vq, vd = _record_views(s["cache"], hd)
    page, cell = (s["cells"] // BLOCK).long(), (s["cells"] % BLOCK).long()
    in_k, in_v = (page, slice(None), slice(None), slice(None), cell // 8, cell % 4, cell // 4 % 2), \
        (page, slice(None), slice(None), cell // 8, slice(None), slice(None), cell % 8)
    at = (page, slice(None), slice(None), cell)
    kd[at], k = _rounded(s["k"], hd)
    vd[at], v = _rounded(s["v"], hd)
    kq[in_k] = k.unflatten(3, (4, 8))
    vq[in_v] = v.unflatten(3, (2, 16)).transpose(3, 4)
    back = lambda q, d: (q.float() * d[..., None].float()).flatten(2).to(dtype)
    return back(kq[in_k].flatten(3), kd[at]), back(vq[in_v].transpose(3, 4).flatten(3), vd[at])


def _plain_logp(s):
    x, n = s["x"], s["case"]["top"]
    z = x.double()
    z = z - z.amax(1, keepdim=True)
    w = torch.exp(z)
    total = w.sum(1, keepdim=True)
    lse = torch.log(total)
    entropy = lse[:, 0] - (w * torch.where(w > 0, z, 0.0)).sum(1) / total[:, 0]
    of = (z.gather(1, s["tokens"].long()[:, None]) - lse)[:, 0].float()
    if n == 0:
        return of, entropy.float()
    value, token = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits: the lowest index first
    value, token = value[:, :n], token[:, :n]
    at = (z.gather(1, token) - lse).float()
    return of, entropy.float(), torch.where(value == -math.inf, -1, token).to(torch.int32), at


# ---- the framework's calls ---------------------------------------------------------------------

def _own_run(s):
    import localstack_amd as L
    c = s["case"]
    if c["op"] == "cache":
        L.store_q8(s["cache"], s["k"], s["v"], s["cells"])
        return L.load_q8(s["cache"], s["cells"], dtype=s["k"].dtype)
    if c["op"] == "logp":
        if s["work"] is None:  # a server keeps its workspace
            s["work"] = torch.empty(L.token_logprobs_work_bytes(c["B"], c["V"], c["top"]), dtype=torch.uint8, device=DEV)
        r = L.token_logprobs(s["x"], s["tokens"], n_top=c["top"], work=s["work"])
        return r if c["top"] else r[:2]
    seqs = (s["lens"], s["first"], s["blocks"], s["max_len"])
    if s["work"] is None:
        n = L.paged_attention_q8_work_bytes(c["B"], s["H"], s["kv"], s["hd"], s["max_len"], c["window"], c["sinks"]) if c["op"] == "q8" \
            else L.shared_attention_work_bytes(c["B"], s["H"], s["kv"], s["hd"], s["max_len"], c["prefix"])
        s["work"], s["out"] = torch.empty(n, dtype=torch.uint8, device=DEV), torch.empty_like(s["q"])
    kept = dict(scale=s["scale"], out=s["out"], work=s["work"])
    if c["op"] == "q8":
        return L.paged_attention_q8(s["q"], s["cache"], *seqs, window=c["window"], n_sink=c["sinks"], **kept)
    x = s["prefix"]
    prefix = L.SharedPrefix(x["k"], x["v"], x["length"], x["blocks"], x["max_len"])
    if c["bits"] == 8:
        return L.shared_attention_q8(s["q"], prefix, s["cache"], *seqs, **kept)
    return L.shared_attention(s["q"], prefix, s["k"], s["v"], *seqs, **kept)


def run(state):
    if own:
        return _own_run(state)
    return {"cache": _plain_cache, "q8": _plain_q8, "shared": _plain_shared, "logp": _plain_logp}[state["case"]["op"]](state)


def work(case):
    if case["op"] == "logp":
        return {"bytes": case["B"] * (4 * case["V"] + 12 + 8 * case["top"]), "flops": 4 * case["B"] * case["V"]}
    H, kv, hd = HEADS[case["heads"]]
    q8, f16 = 2 * kv * (hd + hd // 16), 4 * kv * hd  # a cell's bytes
    if case["op"] == "cache":
        rows = 2 * kv * hd * (2 if case["dtype"] == "f16" else 4)
        return {"bytes": 2 * case["T"] * (rows + q8 + 4), "flops": 8 * case["T"] * kv * hd}
    io = 4 * case["B"] * H * hd
    if case["op"] == "q8":
        seen = sum(_visible(case, n) for n in _lens(case))
        return {"bytes": q8 * seen + io + seen // 8, "flops": 4 * H * hd * seen}
    seen, p = sum(_lens(case)), case["prefix"]
    return {"bytes": (q8 if case["bits"] == 8 else f16) * seen + f16 * p + io + (seen + p) // 8,
            "flops": 4 * H * hd * (seen + p * case["B"])}


# ---- 64-bit results ----------------------------------------------------------------------------

def _pages_of(s, b, n):
    i = torch.arange(n, device=DEV)
    return s["blocks"][int(s["first"][b]) + i // BLOCK].long(), i % BLOCK


def _f16_rows(k, v, page, at, g):
    """K [n][hd] and V [n][hd] of these cells of KV head g, in 64 bits."""
    cell = page * BLOCK + at
    return k[g].index_select(1, cell).double().transpose(1, 2).reshape(v.shape[2], cell.numel()).t(), v[g, cell // 4, :, cell % 4].double()


def _q8_offsets(hd):
    """Where K's and V's whole number of (cell, dim), and the scale of (cell, block of dims), lie in a record."""
    i, d = torch.arange(BLOCK, device=DEV)[:, None], torch.arange(hd, device=DEV)[None]
    k = d // 32 * 1024 + d % 32 // 8 * 256 + i // 8 * 64 + i % 4 * 16 + i // 4 % 2 * 8 + d % 8
    v = d // 32 * 1024 + i // 8 * 256 + d % 16 * 16 + d // 16 % 2 * 8 + i % 8
    return k, v, d // 32 * BLOCK + i


def _q8_rows(cache, hd, page, at, g):
    ko, vo, so = _q8_offsets(hd)
    rec = cache[page, g]
    num = lambda off: rec.view(torch.int8).gather(1, off[at]).double()
    sc = lambda off: rec.view(torch.float16).gather(1, off[at]).double()
    return num(ko) * sc(so + 16 * hd), num(vo + 34 * hd) * sc(so + 33 * hd)


def _exact_attention(s):
    c, kv, hd, H = s["case"], s["kv"], s["hd"], s["H"]
    grp = H // kv
    out = torch.zeros(c["B"], H, hd, dtype=torch.float64, device=DEV)
    lens = s["lens"].tolist()
    for g in range(kv):
        q = s["q"][:, g * grp:(g + 1) * grp].double()
        if c["op"] == "shared":
            x = s["prefix"]
            i = torch.arange(c["prefix"], device=DEV)
            pk, pv = _f16_rows(x["k"], x["v"], x["blocks"][i // BLOCK].long(), i % BLOCK, g)
        for b, n in enumerate(lens):
            page, at = _pages_of(s, b, n)
            if c["op"] == "q8" and c["window"] > 0:
                i = torch.arange(n, device=DEV)
                keep = (i >= n - c["window"]) | (i < c["sinks"])
                page, at = page[keep], at[keep]
            k, v = _q8_rows(s["cache"], hd, page, at, g) if "cache" in s else _f16_rows(s["k"], s["v"], page, at, g)
            score = [q[b].mm(k.t())] + ([q[b].mm(pk.t())] if c["op"] == "shared" else [])
            p = torch.cat(score, 1) * s["scale"]
            if p.shape[1] == 0:
                continue
            p = torch.softmax(p, 1)
            o = p[:, :v.shape[0]].mm(v)
            if c["op"] == "shared":
                o = o + p[:, v.shape[0]:].mm(pv)
            out[b, g * grp:(g + 1) * grp] = o
    return out


def _exact_cache(s):
    import numpy as np
    out = []
    for x in (s["k"], s["v"]):
        x = x.cpu().numpy().astype(np.float64)
        T, kv, hd = x.shape
        x = x.reshape(T, kv, hd // 32, 32)
        most = np.abs(x).max(3)
        d = (most / 127).astype(np.float16)
        d = np.where(d.astype(np.float64) * 127 < most, np.nextafter(d, np.float16(np.inf)), d).astype(np.float64)[..., None]
        out.append((np.rint(x / np.where(d == 0, 1.0, d)) * d).reshape(T, kv, hd))
    return tuple(out)


def _exact_logp(s):
    x, n = s["x"].double(), s["case"]["top"]
    p = torch.log_softmax(x, 1)
    of = p[torch.arange(p.shape[0], device=DEV), s["tokens"].long()]
    entropy = torch.special.entr(torch.exp(p)).sum(1)
    if n == 0:
        return of, entropy
    ids = torch.argsort(s["x"], dim=1, descending=True, stable=True)[:, :n]
    at = p.gather(1, ids)
    return of, entropy, torch.where(at == -math.inf, -1, ids).to(torch.int32), at


def exact(case, seed):
    s = prepare(case, seed)
    return {"cache": _exact_cache, "q8": _exact_attention, "shared": _exact_attention, "logp": _exact_logp}[case["op"]](s)
