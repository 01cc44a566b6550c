"""What is timed of the paged-serving operators: their cases, inputs, plain forms and exact values.

Four operators make one decoding or prompt step over a paged key-value cache:

  append   per-head RMSNorm of q and k, rotary position, K and V rows written to their pages
  decode   attention of one new token per sequence over the pages (window and sink tokens optional)
  prompt   attention of a ragged batch of prompt chunks over the pages (causal, the same options)
  sample   one token per row of logits: temperature, top-k, top-p, min-p and a given uniform number

`own` false computes them with elementary torch operations; `own` true calls the package.
"""
import math

import torch

own = False

D = 128
_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases --------------------------------------------------------------------------------------

def listed():
    return [
        # the first decoding steps of a short prompt: one sequence, latency is all there is
        {"name": "append 1x1", "op": "append", "batch": 1, "new": 1, "ctx": 8, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dtype": "f32", "cache": "f16", "page": 16},
        # one step of a batch of 64 at ragged contexts, 16-bit activations
        {"name": "append 64x1 ragged bf16", "op": "append", "batch": 64, "new": 1, "ctx": 2047, "ragged": True,
         "q_heads": 32, "kv_heads": 4, "dtype": "bf16", "cache": "bf16", "page": 32},
        # a prompt pass of 32 prompts of 512 tokens
        {"name": "append 32x512", "op": "append", "batch": 32, "new": 512, "ctx": 0, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dtype": "f32", "cache": "f16", "page": 64},
        # one sequence just after its prompt
        {"name": "decode 1x31", "op": "decode", "batch": 1, "len": 31, "ragged": False, "q_heads": 16, "kv_heads": 8,
         "dtype": "f32", "cache": "f16", "page": 16, "window": 0, "sinks": 0},
        # one sequence at the model's whole context: the cache's length is the only parallelism
        {"name": "decode 1x32768", "op": "decode", "batch": 1, "len": 32768, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dtype": "f16", "cache": "f16", "page": 64, "window": 0, "sinks": 0},
        # the batched-decode workload: 64 sequences of 2048 positions
        {"name": "decode 64x2048", "op": "decode", "batch": 64, "len": 2048, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dtype": "f32", "cache": "f16", "page": 64, "window": 0, "sinks": 0},
        # ragged lengths with a sliding window and sink tokens, eight queries to a KV head
        {"name": "decode 37 ragged window", "op": "decode", "batch": 37, "len": 19001, "ragged": True, "q_heads": 32,
         "kv_heads": 4, "dtype": "bf16", "cache": "bf16", "page": 16, "window": 4097, "sinks": 4},
        # the short prompt of the greedy benchmark
        {"name": "prompt 1x8", "op": "prompt", "batch": 1, "new": 8, "ctx": 0, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dtype": "f32", "cache": "f16", "page": 16, "window": 0, "sinks": 0},
        # ragged prompt chunks behind ragged contexts, window and sinks
        {"name": "prompt 5 ragged window", "op": "prompt", "batch": 5, "new": 1500, "ctx": 4500, "ragged": True,
         "q_heads": 32, "kv_heads": 4, "dtype": "bf16", "cache": "bf16", "page": 32, "window": 1025, "sinks": 4},
        # one long prompt, causal over itself
        {"name": "prompt 1x8192", "op": "prompt", "batch": 1, "new": 8192, "ctx": 0, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dtype": "f16", "cache": "f16", "page": 64, "window": 0, "sinks": 0},
        # one row of the model's logits, a usual setting
        {"name": "sample 1x151936", "op": "sample", "rows": 1, "vocab": 151936, "dtype": "f32", "spread": 3.0,
         "mixed": False, "top_k": 40, "top_p": 0.9, "min_p": 0.0, "temperature": 0.8},
        # a batch in which every request has its own setting, full-vocabulary nuclei among them
        {"name": "sample 64x151936 mixed", "op": "sample", "rows": 64, "vocab": 151936, "dtype": "f32", "spread": 2.5,
         "mixed": True, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "prompt", "sample"])
    if op == "sample":
        vocab = _log(rng, 33, 200003)
        rows = min(_log(rng, 1, 200), max(1, 64 * 151936 // vocab))
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["f32", "f16", "bf16"]),
                "spread": round(rng.uniform(0.5, 4.0), 2), "mixed": rng.random() < 0.5,
                "top_k": rng.choice([0, 0, 5, 50, 777]), "top_p": rng.choice([1.0, 0.95, 0.7, 0.3]),
                "min_p": rng.choice([0.0, 0.0, 0.02, 0.2]), "temperature": round(rng.uniform(0.3, 1.6), 2)}
    q_heads, kv_heads = rng.choice([(16, 8), (16, 8), (32, 4), (4, 4), (8, 1), (12, 4), (10, 2), (16, 1)])
    cache = rng.choice(["f16", "bf16"])
    c = {"op": op, "batch": 1, "q_heads": q_heads, "kv_heads": kv_heads, "ragged": rng.random() < 0.7,
         "dtype": rng.choice(["f32", cache]), "cache": cache, "page": rng.choice([16, 32, 64, 128])}
    if op == "append":
        c["new"] = _log(rng, 1, 512)
        c["batch"] = _log(rng, 1, max(1, min(64, 16384 * 32 // (c["new"] * (q_heads + 2 * kv_heads)))))
        c["ctx"] = rng.choice([0, _log(rng, 1, 4000)])
        return c
    if op == "decode":
        c["len"] = _log(rng, 1, 32768)
        c["batch"] = _log(rng, 1, max(1, min(64, 64 * 2048 * 8 // (c["len"] * kv_heads * 2))))
    else:
        c["new"] = _log(rng, 1, 2500)
        c["batch"] = _log(rng, 1, max(1, min(32, 5000 // c["new"])))
        c["ctx"] = rng.choice([0, _log(rng, 1, 3500)])
    c["window"], c["sinks"] = rng.choice([(0, 0), (0, 0), (_log(rng, 1, 5000), 0), (_log(rng, 1, 5000), 4),
                                          (_log(rng, 16, 2000), _log(rng, 1, 200))])
    return c


def _part(c, key, b):
    """Sequence b's share of c[key]: all of it, or spread from the whole down to a twentieth."""
    n = c[key]
    if not c["ragged"] or b == 0 or n == 0:
        return n
    f = (b * 0.6180339887498949 + (0.37 if key == "ctx" else 0.0)) % 1.0
    return max(1, int(n * (0.05 + 0.95 * f * f)))


def _lens(c):
    """(new tokens, total length) of every sequence."""
    if c["op"] == "decode":
        return [(1, _part(c, "len", b)) for b in range(c["batch"])]
    new = [1 if c["new"] == 1 else _part(c, "new", b) for b in range(c["batch"])]
    return [(n, n + _part(c, "ctx", b)) for b, n in enumerate(new)]


# ---- inputs -------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "sample":
        R, V = case["rows"], case["vocab"]
        s["logits"] = (torch.randn(R, V, device="cuda", generator=g) * case["spread"]).to(_T[case["dtype"]])
        s["u"] = torch.rand(R, device="cuda", generator=g)
        ones = torch.ones(R, device="cuda")
        s["temperature"], s["top_p"] = ones * case["temperature"], ones * case["top_p"]
        s["min_p"] = ones * case["min_p"]
        s["top_k"] = torch.full((R,), case["top_k"], device="cuda", dtype=torch.int32)
        if case["mixed"]:  # requests with settings of their own: every fourth keeps the case's
            i = torch.arange(R, device="cuda")
            s["temperature"] = torch.where(i % 4 == 1, ones * 0.6, s["temperature"])
            s["temperature"] = torch.where(i % 8 == 7, ones * 0.0, s["temperature"])
            s["top_k"] = torch.where(i % 4 == 2, torch.full_like(s["top_k"], 64), s["top_k"])
            s["top_p"] = torch.where(i % 4 == 3, ones * 0.9, s["top_p"])
            s["min_p"] = torch.where(i % 8 == 4, ones * 0.05, s["min_p"])
        return s
    lens = _lens(case)
    B, page, kvh, H = case["batch"], case["page"], case["kv_heads"], case["q_heads"]
    per = [-(-n // page) for _, n in lens]
    width, pages = max(per), sum(per) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).cpu()
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    new = [n for n, _ in lens]
    T = sum(new)
    s["table"] = table.cuda()
    s["lens"] = torch.tensor([n for _, n in lens], dtype=torch.int32, device="cuda")
    s["starts"] = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda")
    s["k"] = torch.randn(pages, kvh, page, D, device="cuda", generator=g).to(_T[case["cache"]])
    s["v"] = torch.randn(pages, kvh, page, D, device="cuda", generator=g).to(_T[case["cache"]])
    s["rows"] = T
    if case["op"] == "append":
        s["qkv"] = torch.randn(T, (H + 2 * kvh) * D, device="cuda", generator=g).to(_T[case["dtype"]])
        s["q_norm"] = 1 + 0.1 * torch.randn(D, device="cuda", generator=g)
        s["k_norm"] = 1 + 0.1 * torch.randn(D, device="cuda", generator=g)
        far = torch.arange(max(n for _, n in lens), device="cuda", dtype=torch.float64)
        a = far[:, None] * (1.0e6 ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2)))[None]
        s["cos"], s["sin"] = a.cos().float(), a.sin().float()
    else:  # normalised and rotated queries: of unit size by element
        s["q"] = (torch.randn(T, H, D, device="cuda", generator=g) * 1.5).to(_T[case["dtype"]])
    return s


# ---- one pass -----------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        from kernel_optimization_webgpu_b200 import runtime as R
        if op == "append":
            q = R.paged_append(s["qkv"], s["k"], s["v"], s["table"], s["lens"], s["cos"], s["sin"], c["q_heads"],
                               q_norm=s["q_norm"], k_norm=s["k_norm"], q_starts=s["starts"])
            return q.view(s["rows"], c["q_heads"], D), s["k"], s["v"]
        if op == "decode":
            return R.paged_attn_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], window=c["window"],
                                       sinks=c["sinks"])
        if op == "prompt":
            return R.paged_attn_prompt(s["q"], s["k"], s["v"], s["table"], s["lens"], s["starts"],
                                       window=c["window"], sinks=c["sinks"])
        return R.sample_rows(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                             min_p=s["min_p"])
    return {"append": _append, "decode": _attend, "prompt": _attend, "sample": _sample}[op](s)


def _rows(s):
    """Sequence and position of every new token."""
    t = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(s["starts"].long(), t, right=True) - 1
    return b, s["lens"].long()[b] - (s["starts"].long()[b + 1] - t)


def _append(s):
    c = s["case"]
    H, kvh, page = c["q_heads"], c["kv_heads"], c["page"]
    x = s["qkv"].float().view(s["rows"], H + 2 * kvh, D)
    b, pos = _rows(s)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turned(h, w):
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w
        lo, hi = h[..., :D // 2], h[..., D // 2:]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)

    q, k, v = turned(x[:, :H], s["q_norm"]), turned(x[:, H:H + kvh], s["k_norm"]), x[:, H + kvh:]
    at = s["table"].long()[b, pos // page]
    s["k"][at, :, pos % page] = k.to(s["k"].dtype)
    s["v"][at, :, pos % page] = v.to(s["v"].dtype)
    return q.to(s["qkv"].dtype), s["k"], s["v"]


def _attend(s):
    c = s["case"]
    H, kvh, B = c["q_heads"], c["kv_heads"], c["batch"]
    b, pos = _rows(s)
    n = max(m for m, _ in _lens(c))  # rows of the padded batch
    at = torch.arange(s["rows"], device="cuda") - s["starts"].long()[b]
    q = torch.zeros(B, n, H, D, device="cuda")
    q[b, at] = s["q"].float()
    p = torch.full((B, n), -1, device="cuda")
    p[b, at] = pos
    held = s["table"].long().clamp(min=0)
    k, v = (x[held].transpose(2, 3).reshape(B, -1, kvh, D).float() for x in (s["k"], s["v"]))
    j = torch.arange(k.shape[1], device="cuda")
    seen = j <= p[..., None]
    if c["window"]:
        seen = seen & ((j > p[..., None] - c["window"]) | (j < c["sinks"]))
    q = q.view(B, n, kvh, H // kvh, D).permute(0, 2, 3, 1, 4).reshape(B, kvh, -1, D)
    w = torch.matmul(q, k.permute(0, 2, 3, 1)).view(B, kvh, H // kvh, n, -1).mul_(D ** -0.5)
    w.masked_fill_(~seen[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w = w.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = w.sum(-1, keepdim=True)
    held = (j < s["lens"][:, None])[..., None, None]
    y = torch.matmul(w.view(B, kvh, -1, k.shape[1]), v.masked_fill_(~held, 0.0).transpose(1, 2))
    y = y.view(B, kvh, H // kvh, n, D) / total.masked_fill_(total == 0, 1.0)
    return y.permute(0, 3, 1, 2, 4).reshape(B, n, H, D)[b, at].to(s["q"].dtype)


def _sample(s):
    c = s["case"]
    V = c["vocab"]
    v, order = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True)
    T = s["temperature"][:, None]
    x = (v.double() - v[:, :1].double()) / torch.where(T > 0, T, 1.0).double()
    w = x.exp()
    i = torch.arange(V, device="cuda")
    k = torch.where(s["top_k"] > 0, s["top_k"], V).long()
    k = torch.where(s["temperature"] > 0, k, 1)[:, None]
    w = torch.where(i < k, w, 0.0)
    run_ = w.cumsum(-1)
    total = run_[:, -1:]
    # the shortest prefix that reaches top_p of the top-k sum, then the weights of at least min_p
    before = run_ - w
    top_p = s["top_p"].double()[:, None]
    keep = (i == 0) | ((i < k) & ((before < top_p * total) | (top_p >= 1)) & (w >= s["min_p"].double()[:, None]))
    w = torch.where(keep, w, 0.0)
    run_ = torch.where(keep, run_, 0.0).amax(-1, keepdim=True)
    cum = w.cumsum(-1)
    past = keep & (cum > s["u"].double()[:, None] * run_)
    last = keep.long().sum(-1) - 1
    pick = torch.where(past.any(-1), past.long().argmax(-1), last)[:, None]
    logp = w.gather(1, pick).log() - run_.log()
    return order.gather(1, pick)[:, 0].to(torch.int32), logp[:, 0].float()


# ---- what a pass cannot do without --------------------------------------------------------------

def _visible(c, p):
    """Keys that a query at position p sees."""
    if not c["window"]:
        return p + 1
    lo = max(0, p + 1 - c["window"])
    return p + 1 - lo + min(lo, c["sinks"])


def work(case):
    c = case
    if c["op"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * _SIZE[c["dtype"]] + c["rows"] * 28, "flops": 4 * n}
    H, kvh = c["q_heads"], c["kv_heads"]
    lens = _lens(c)
    T = sum(n for n, _ in lens)
    act, kv = _SIZE[c["dtype"]], _SIZE[c["cache"]]
    if c["op"] == "append":
        far = max(n for _, n in lens) - min(t - n for n, t in lens)
        return {"bytes": T * D * ((2 * H + 2 * kvh) * act + 2 * kvh * kv) + min(far, T) * D * 4,
                "flops": T * D * (8 * H + 8 * kvh)}
    pairs = sum(_visible(c, p) for n, t in lens for p in range(t - n, t))
    keys = sum(t if not c["window"] else t - max(0, t - n + 1 - c["window"])
               + min(max(0, t - n + 1 - c["window"]), c["sinks"]) for n, t in lens)
    return {"bytes": keys * kvh * D * 2 * kv + 2 * T * H * D * act, "flops": 4 * D * H * pairs}


# ---- the definitions in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "sample":
        return _exact_sample(s)
    H, kvh, page = c["q_heads"], c["kv_heads"], c["page"]
    outs = []
    ks, vs = s["k"].double(), s["v"].double()
    first = 0
    for b, (n, t) in enumerate(_lens(c)):
        rows = slice(first, first + n)
        first += n
        where = torch.arange(t, device="cuda")
        pages = s["table"][b].long()[where // page]
        if c["op"] == "append":
            x = s["qkv"][rows].double().reshape(n, -1, D)
            at = where[t - n:]
            turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
            heads = []
            for part, w in ((x[:, :H], s["q_norm"]), (x[:, H:H + kvh], s["k_norm"])):
                part = part / (part.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
                z = torch.complex(part[..., :D // 2].contiguous(), part[..., D // 2:].contiguous()) * turn
                heads.append(torch.cat([z.real, z.imag], -1))
            ks[pages[t - n:], :, at % page] = heads[1]
            vs[pages[t - n:], :, at % page] = x[:, H + kvh:]
            outs.append(heads[0])
            continue
        k, v = ks[pages, :, where % page], vs[pages, :, where % page]  # [t][kvh][D]
        y = torch.zeros(n, H, D, device="cuda", dtype=torch.float64)
        p = torch.arange(t - n, t, device="cuda")[:, None]
        gone = where[None] > p
        if c["window"]:
            gone |= (p - where[None] >= c["window"]) & (where[None] >= c["sinks"])
        for h in range(H):
            g = h * kvh // H
            z = s["q"][rows, h].double() @ k[:, g].T / math.sqrt(D)
            y[:, h] = torch.softmax(z.masked_fill(gone, -math.inf), -1) @ v[:, g]
        outs.append(y)
    out = torch.cat(outs)
    return (out, ks, vs) if c["op"] == "append" else out


def _exact_sample(s):
    ids, logps = [], []
    V = s["case"]["vocab"]
    for r in range(s["case"]["rows"]):
        v = s["logits"][r].double()
        T, u = float(s["temperature"][r]), float(s["u"][r])
        k, top_p, min_p = int(s["top_k"][r]), float(s["top_p"][r]), float(s["min_p"][r])
        if T <= 0:
            ids.append(int((v == v.max()).nonzero()[0, 0]))
            logps.append(0.0)
            continue
        rank = torch.argsort(-v, stable=True)[:k if 0 < k < V else V]
        w = torch.exp((v[rank] - v[rank[0]]) / T)
        run_ = torch.cumsum(w, 0)
        m = w.numel()
        if top_p < 1:
            m = min(m, int((run_ < top_p * run_[-1]).sum()) + 1)
        m = max(1, min(m, int((w >= min_p).sum())))
        i = min(m - 1, int((run_[:m] <= u * run_[m - 1]).sum()))
        ids.append(int(rank[i]))
        logps.append(math.log(float(w[i]) / float(run_[m - 1])))
    return (torch.tensor(ids, dtype=torch.int32), torch.tensor(logps, dtype=torch.float64))
