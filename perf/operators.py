"""Timed cases of the operators of a decode step of many sequences: attention of one new token per sequence over the paged
KV cache, routing of tokens to experts by a given rule, and sampling of the next tokens.

Listed cases (what each stands for in real use):
  attn_one_short     one sequence a few dozen tokens in: the smallest call, where latency counts
  attn_one_tiny      one sequence at the two-layer test model's head layout (4 query heads on 2, head size 64)
  attn_chat_b24      24 chats of uneven length at the 32-on-4-heads layout, an ordinary step of a server
  attn_long_b2       two documents of about a hundred thousand tokens at the 64-on-4-heads layout
  attn_batch_b128    128 sequences of up to 8192 tokens: the largest step
  attn_window_b48    48 long sequences of which each token sees the last 4000 and the first 4 cells
  sample_one         one row of a 151936-token vocabulary, temperature with top-k and top-p: a single user
  sample_b64         64 rows of that vocabulary, every request with settings of its own, greedy ones among them
  sample_free_b200   200 rows drawn with a temperature alone (no filter) from an odd vocabulary
  route_t1           one token, softmax over 128 experts, 8 used: a decode step of one sequence
  route_t512         a prompt step, sigmoid scores of 256 experts with a balance bias, 4 of 8 groups
  route_t60000       a very long batch of prompts routed at once by that rule

The plain forms are written with elementary torch operations. Scores whose order decides an answer (router choices, sampled
tokens) are 64-bit there, since a 32-bit rounding would decide between close candidates.
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
MOST_CELLS = 128 * 8192  # cells of the largest step
MOST_BYTES = 1.2e9       # and the K and V bytes it reads, about


def _attn(name, heads, B, lo, hi, window=0, sinks=0):
    """B sequences of lo .. hi cells (spread evenly, in an order of the case's own)."""
    return {"name": name, "op": "attn", "heads": heads, "B": B, "lo": lo, "hi": hi, "window": window, "sinks": sinks}


def _sample(name, B, V, mode):
    return {"name": name, "op": "sample", "B": B, "V": V, "mode": mode}


def _route(name, T, E, k, score, groups=1, used=1, top=1, bias=False, renorm=True, scale=1.0):
    return {"name": name, "op": "route", "T": T, "E": E, "k": k, "score": score, "groups": groups, "used": used, "top": top,
            "bias": bias, "renorm": renorm, "scale": scale}


def listed():
    return [_attn("attn_one_short", "32x4", 1, 45, 45),
            _attn("attn_one_tiny", "tiny", 1, 300, 300),
            _attn("attn_chat_b24", "32x4", 24, 100, 4100),
            _attn("attn_long_b2", "64x4", 2, 90001, 110007),
            _attn("attn_batch_b128", "32x4", 128, 1000, 8192),
            _attn("attn_window_b48", "32x4", 48, 5000, 20000, window=4000, sinks=4),
            _sample("sample_one", 1, VOCAB, "chat"),
            _sample("sample_b64", 64, VOCAB, "mixed"),
            _sample("sample_free_b200", 200, 50259, "free"),
            _route("route_t1", 1, 128, 8, "softmax"),
            _route("route_t512", 512, 256, 8, "sigmoid", 8, 4, 2, True, True, 2.5),
            _route("route_t60000", 60000, 256, 8, "sigmoid", 8, 4, 2, True, True, 2.5)]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "sample", "route"])
    if op == "attn":
        heads = rng.choice(sorted(HEADS))
        _, kv, hd = HEADS[heads]
        cells = min(MOST_CELLS // 2, int(MOST_BYTES / (4 * kv * hd)))
        B = _log_int(rng, 1, 128)
        hi = _log_int(rng, 1, min(131072, max(1, cells // B)))
        c = _attn("", heads, B, rng.randint(0 if hi < 64 else 1, hi), hi)
        if rng.random() < 0.4:
            c["window"], c["sinks"] = _log_int(rng, 1, 8192), rng.choice([0, 1, 4, 33, 128])
    elif op == "sample":
        V = rng.choice([VOCAB, _log_int(rng, 100, 200000), _log_int(rng, 1000, 200000)])
        c = _sample("", _log_int(rng, 1, max(1, min(256, 64 * VOCAB // V))), V, rng.choice(["chat", "mixed", "free", "minp", "topp"]))
    else:
        E = rng.choice([8, 60, 64, 96, 128, 160, 256, rng.randint(2, 256)])
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if E % g == 0 and E // g >= 2] or [1])
        used = rng.randint(1, groups)
        k = rng.randint(1, min(10, used * (E // groups)))
        score = rng.choice(["softmax", "sigmoid"])
        c = _route("", _log_int(rng, 1, 60000), E, k, score, groups, used, rng.choice([1, 2]) if E // groups >= 2 else 1,
                   rng.random() < 0.5, rng.random() < 0.7, rng.choice([1.0, 2.5]))
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


def _settings(mode, B):
    """Per row: (temperature, top_k, top_p, min_p)."""
    rows = {"chat": [(0.7, 20, 0.8, 0.0)], "free": [(0.9, 0, 1.0, 0.0)], "minp": [(1.1, 0, 1.0, 0.05)],
            "topp": [(1.0, 0, 0.95, 0.0)],
            "mixed": [(0.7, 20, 0.8, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.95, 0.0), (0.6, 0, 1.0, 0.1), (1.3, 1000, 0.99, 0.01),
                      (1.0, 0, 1.0, 0.0), (0.8, 50, 1.0, 0.0)]}[mode]
    return [rows[i % len(rows)] for i in range(B)]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    rand = lambda *s: torch.rand(*s, generator=g, device=DEV)
    randn = lambda *s, **k: torch.randn(*s, generator=g, device=DEV, **k)
    if case["op"] == "attn":
        H, kv, hd = HEADS[case["heads"]]
        lens = _lens(case)
        pages = [-(-n // BLOCK) for n in lens]
        total = max(8, -(-sum(pages) // 8) * 8)
        cells = total * BLOCK
        # pages lie in the cache in the order sequences took and gave them back: any order
        order = torch.randperm(total, generator=g, device=DEV)[:max(1, sum(pages))].to(torch.int32)
        first = [0]
        for n in pages[:-1]:
            first.append(first[-1] + n)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        return dict(case=case, H=H, kv=kv, hd=hd, k=randn(kv, hd // 4, cells, 4, dtype=torch.float16),
                    v=randn(kv, cells // 4, hd, 4, dtype=torch.float16),
                    q=(2.0 * randn(len(lens), H, hd)).half(), lens=i32(lens), first=i32(first), blocks=order,
                    max_len=max(1, max(lens)), scale=1.0 / math.sqrt(hd), work=None)
    if case["op"] == "sample":
        B, V = case["B"], case["V"]
        x = 2.2 * randn(B, V)
        # a few hundred likely tokens above the rest, the first of them well ahead in every other row
        n = min(300, V)
        at = rand(B, V).topk(n, dim=1).indices
        lift = 13.0 - 1.4 * torch.log(torch.arange(1, n + 1, device=DEV, dtype=torch.float32)) * (1.0 + (torch.arange(B, device=DEV) % 2)[:, None])
        x.scatter_add_(1, at, lift.expand(B, n).contiguous())
        s = _settings(case["mode"], B)
        col = lambda i, t: torch.tensor([r[i] for r in s], dtype=t, device=DEV)
        return dict(case=case, x=x, u=rand(B), temperature=col(0, torch.float32), top_k=col(1, torch.int32),
                    top_p=col(2, torch.float32), min_p=col(3, torch.float32), work=None)
    T, E = case["T"], case["E"]
    x = 1.5 * randn(T, E) + randn(1, E)  # some experts are asked for more often
    return dict(case=case, x=x, bias=0.1 * randn(E) if case["bias"] else None)


# ---- plain forms -------------------------------------------------------------------------------

def _plain_attention(s):
    c, kv, hd = s["case"], s["kv"], s["hd"]
    B, H = s["q"].shape[:2]
    L = -(-s["max_len"] // BLOCK) * BLOCK
    page = s["first"][:, None] + torch.arange(L // BLOCK, device=DEV)
    page = s["blocks"][page.clamp(max=s["blocks"].numel() - 1)].long()
    cell = (page[:, :, None] * BLOCK + torch.arange(BLOCK, device=DEV)).reshape(-1)
    # [kv][hd / 4][cell][4] -> [B][kv][hd][L], and [kv][cell / 4][hd][4] -> [B][kv][L][hd]
    k = s["k"][:, :, cell].reshape(kv, hd // 4, B, L, 4).permute(2, 0, 1, 4, 3).reshape(B, kv, hd, L).float()
    quad = cell[::4] // 4
    v = s["v"][:, quad].reshape(kv, B, L // 4, hd, 4).permute(1, 0, 2, 4, 3).reshape(B, kv, L, hd).float()
    q = s["q"].float().reshape(B, kv, H // kv, hd)
    score = (q @ k) * s["scale"]
    i, n = torch.arange(L, device=DEV), s["lens"][:, None]
    seen = i < n
    if c["window"] > 0:
        seen = seen & ((i >= n - c["window"]) | (i < c["sinks"]))
    seen = seen[:, None, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
    return out.reshape(B, H, hd).half()


def _plain_sample(s):
    x, u = s["x"], s["u"].double()
    B, V = x.shape
    greedy = ~(s["temperature"] > 0)
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None]
    value, token = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits: the lowest index first
    w = torch.exp((value.double() - value[:, :1].double()) / t)
    rank = torch.arange(V, device=x.device)
    k = torch.where(s["top_k"] > 0, s["top_k"], V)[:, None]
    w = torch.where((rank < k) & ((w >= s["min_p"].double()[:, None]) | (rank == 0)), w, 0.0)
    cum = torch.cumsum(w, 1)
    p = s["top_p"].double()[:, None]
    keep = (p >= 1) | (rank == 0) | (cum - w < p * cum[:, -1:])
    w = torch.where(keep, w, 0.0)
    cum = torch.cumsum(w, 1)
    total = cum[:, -1:]
    at = (cum <= u[:, None] * total).sum(1, keepdim=True)
    at = torch.minimum(at, (w > 0).sum(1, keepdim=True) - 1)
    at = torch.where(greedy[:, None], torch.zeros_like(at), at)
    prob = torch.where(greedy[:, None], torch.ones_like(total), w.gather(1, at) / total)
    return token.gather(1, at)[:, 0].to(torch.int32), prob[:, 0].float()


def _plain_route(s):
    c, x = s["case"], s["x"].double()
    T, E, G, k = c["T"], c["E"], c["groups"], c["k"]
    if c["score"] == "softmax":
        p = torch.exp(x - x.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-x))
    choice = p if s["bias"] is None else p + s["bias"].double()
    if c["used"] < G:
        best = torch.sort(choice.reshape(T, G, E // G), dim=2, descending=True).values[:, :, :c["top"]].sum(2)
        group = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["used"]]
        kept = torch.zeros(T, G, dtype=torch.bool, device=x.device).scatter_(1, group, True)
        choice = choice.masked_fill(~kept.repeat_interleave(E // G, dim=1), -math.inf)
    ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :k]
    w = p.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True).clamp(min=2.0 ** -14)
    return ids.to(torch.int32), (w * c["scale"]).float()


# ---- the framework's calls ---------------------------------------------------------------------

def _own_run(s):
    import localstack_amd as L
    c = s["case"]
    if c["op"] == "attn":
        if s["work"] is None:  # a server keeps its workspace and output buffer
            s["work"] = torch.empty(L.paged_attention_work_bytes(c["B"], s["H"], s["kv"], s["hd"], s["max_len"], c["window"], c["sinks"]),
                                    dtype=torch.uint8, device=DEV)
            s["out"] = torch.empty_like(s["q"])
        return L.paged_attention(s["q"], s["k"], s["v"], s["lens"], s["first"], s["blocks"], s["max_len"], window=c["window"],
                                 n_sink=c["sinks"], scale=s["scale"], out=s["out"], work=s["work"])
    if c["op"] == "sample":
        if s["work"] is None:
            s["work"] = torch.empty(L.sample_work_bytes(c["B"], c["V"]), dtype=torch.uint8, device=DEV)
        return L.sample(s["x"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                        work=s["work"])
    rule = L.RouterRule(score=c["score"], n_group=c["groups"], n_group_used=c["used"], group_top=c["top"], renorm=c["renorm"],
                        scale=c["scale"])
    return L.moe_select(s["x"], c["k"], rule, bias=s["bias"])


def run(state):
    if own:
        return _own_run(state)
    return {"attn": _plain_attention, "sample": _plain_sample, "route": _plain_route}[state["case"]["op"]](state)


def work(case):
    if case["op"] == "attn":
        H, kv, hd = HEADS[case["heads"]]
        seen = sum(_visible(case, n) for n in _lens(case))
        return {"bytes": 4 * kv * hd * seen + 4 * case["B"] * H * hd + seen // 8, "flops": 4 * H * hd * seen}
    if case["op"] == "sample":
        return {"bytes": case["B"] * (4 * case["V"] + 28), "flops": 2 * case["B"] * case["V"]}
    return {"bytes": case["T"] * (4 * case["E"] + 8 * case["k"]), "flops": 4 * case["T"] * case["E"]}


# ---- 64-bit results ----------------------------------------------------------------------------

def _exact_attention(s):
    c, kv, hd, H = s["case"], s["kv"], s["hd"], s["H"]
    out = []
    for b, n in enumerate(s["lens"].tolist()):
        ids = [i for i in range(n) if c["window"] <= 0 or i >= n - c["window"] or i < c["sinks"]]
        if not ids:
            out.append(torch.zeros(H, hd, dtype=torch.float64, device=DEV))
            continue
        ids = torch.tensor(ids, device=DEV)
        f = int(s["first"][b])
        cell = s["blocks"][f + ids // BLOCK].long() * BLOCK + ids % BLOCK
        rows = []
        for g in range(kv):
            kg = s["k"][g].index_select(1, cell).double().transpose(1, 2).reshape(hd, -1)         # [hd][n]
            vg = s["v"][g, cell // 4, :, cell % 4].double()                                       # [n][hd]
            q = s["q"][b, g * (H // kv):(g + 1) * (H // kv)].double()
            rows.append(torch.softmax(q.mm(kg) * s["scale"], dim=1).mm(vg))
        out.append(torch.cat(rows))
    return torch.stack(out)


def _exact_sample(s):
    """Row by row with numpy: sort by (logit, index), cut, walk."""
    import numpy as np
    x, u = s["x"].cpu().numpy(), s["u"].cpu().numpy().astype(np.float64)
    col = {n: s[n].cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p")}
    tokens, probs = [], []
    for b in range(x.shape[0]):
        row = x[b].astype(np.float64)
        if not col["temperature"][b] > 0:
            tokens.append(int(np.argmax(row)))
            probs.append(1.0)
            continue
        z = (row - row.max()) / np.float64(col["temperature"][b])
        live = np.flatnonzero(z > -700)
        order = live[np.argsort(-row[live], kind="stable")]
        if col["top_k"][b] > 0:
            order = order[:col["top_k"][b]]
        w = np.exp(z[order])
        n = max(1, int(np.count_nonzero(w >= np.float64(col["min_p"][b]))))
        order, w = order[:n], w[:n]
        if col["top_p"][b] < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w), np.float64(col["top_p"][b]) * w.sum(), side="left"))
            order, w = order[:n], w[:n]
        cum = np.cumsum(w)
        i = min(len(w) - 1, int(np.searchsorted(cum, u[b] * cum[-1], side="right")))
        tokens.append(int(order[i]))
        probs.append(float(w[i] / cum[-1]))
    return np.array(tokens, np.int32), np.array(probs, np.float64)


def _exact_route(s):
    import numpy as np
    c = s["case"]
    x = s["x"].cpu().numpy().astype(np.float64)
    if c["score"] == "softmax":
        p = np.exp(x - x.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    else:
        p = 1.0 / (1.0 + np.exp(-x))
    choice = p + (0.0 if s["bias"] is None else s["bias"].cpu().numpy().astype(np.float64))
    T, E, G = c["T"], c["E"], c["groups"]
    per = E // G
    if c["used"] < G:
        value = -np.sort(-choice.reshape(T, G, per), axis=2)[:, :, :c["top"]]
        rank = np.argsort(np.argsort(-value.sum(2), axis=1, kind="stable"), axis=1)
        choice = np.where(np.repeat(rank < c["used"], per, axis=1), choice, -np.inf)
    ids = np.argsort(-choice, axis=1, kind="stable")[:, :c["k"]]
    w = np.take_along_axis(p, ids, 1)
    if c["renorm"]:
        w = w / np.maximum(w.sum(1, keepdims=True), 2.0 ** -14)
    return ids.astype(np.int32), w * c["scale"]


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attention, "sample": _exact_sample, "route": _exact_route}[case["op"]](s)
