"""What is timed of the operators beside the paged-serving ones: cases, inputs, plain forms, exact values.

Five operators serve many answers to long prompts from a cache in 8 bits:

  store    per-head RMSNorm of q and k, rotary position, K and V rows as 8-bit integers with a
           scale per row into their pages, and the same positions read back in 16 bits
  read     whole sequences of the 8-bit cache read back into the 16-bit pages of a prompt pass
  decode   attention of one new token per sequence over the 8-bit cache
  shared   attention of one new token per sequence, groups of sequences sharing their first positions
  score    log probability of a given token, entropy and the largest alternatives per row of logits

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
        {"name": "store 1x1", "op": "store", "batch": 1, "new": 1, "ctx": 8, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dtype": "f32", "out": "f16", "page": 16},
        # a prompt pass of 32 prompts of 512 tokens, its attention reading 16-bit pages
        {"name": "store 32x512", "op": "store", "batch": 32, "new": 512, "ctx": 0, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dtype": "f32", "out": "f16", "page": 64},
        # the context of one conversation before its next turn's prompt pass
        {"name": "read 1x700 bf16", "op": "read", "batch": 1, "len": 700, "ragged": False, "q_heads": 32,
         "kv_heads": 4, "out": "bf16", "page": 16},
        # the contexts of a ragged batch of chunked prompts
        {"name": "read 24 ragged", "op": "read", "batch": 24, "len": 9001, "ragged": True, "q_heads": 16,
         "kv_heads": 8, "out": "f16", "page": 64},
        # one sequence just after its prompt
        {"name": "decode 1x31", "op": "decode", "batch": 1, "len": 31, "ragged": False, "q_heads": 16, "kv_heads": 8,
         "dtype": "f32", "page": 16, "window": 0, "sinks": 0},
        # one sequence at the model's whole context: the cache's length is the only parallelism
        {"name": "decode 1x32768", "op": "decode", "batch": 1, "len": 32768, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dtype": "f16", "page": 64, "window": 0, "sinks": 0},
        # the batched-decode workload: 64 sequences of 2048 positions
        {"name": "decode 64x2048", "op": "decode", "batch": 64, "len": 2048, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dtype": "f32", "page": 64, "window": 0, "sinks": 0},
        # four answers to one question of ordinary length
        {"name": "shared 4 of 1000", "op": "shared", "groups": 1, "batch": 4, "shared": 1000, "tail": 40,
         "ragged": False, "q_heads": 16, "kv_heads": 8, "dtype": "f32", "cache": "f16", "page": 16},
        # a batch of answers to one long prompt
        {"name": "shared 64 of 16384", "op": "shared", "groups": 1, "batch": 64, "shared": 16384, "tail": 300,
         "ragged": True, "q_heads": 16, "kv_heads": 8, "dtype": "f16", "cache": "f16", "page": 64},
        # several prompts with unequal numbers of answers, eight queries to a KV head
        {"name": "shared 7 groups bf16", "op": "shared", "groups": 7, "batch": 75, "shared": 5003, "tail": 701,
         "ragged": True, "q_heads": 32, "kv_heads": 4, "dtype": "bf16", "cache": "bf16", "page": 32},
        # the token just sampled, with five alternatives
        {"name": "score 1x151936", "op": "score", "rows": 1, "vocab": 151936, "dtype": "f32", "spread": 3.0,
         "masked": False, "top": 5},
        # the tokens of a prompt of 512 scored
        {"name": "score 512x151936 bf16", "op": "score", "rows": 512, "vocab": 151936, "dtype": "bf16",
         "spread": 2.5, "masked": False, "top": 20},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "read", "decode", "shared", "score"])
    if op == "score":
        vocab = _log(rng, 100, 200003)
        return {"op": op, "rows": min(_log(rng, 1, 2000), max(1, 300 * 151936 // vocab)), "vocab": vocab,
                "dtype": rng.choice(["f32", "f16", "bf16"]), "spread": round(rng.uniform(0.5, 4.0), 2),
                "masked": rng.random() < 0.3, "top": rng.choice([0, 1, 5, 20, 32])}
    q_heads, kv_heads = rng.choice([(16, 8), (16, 8), (32, 4), (4, 4), (8, 1), (12, 4), (10, 2), (16, 1)])
    c = {"op": op, "batch": 1, "q_heads": q_heads, "kv_heads": kv_heads, "ragged": rng.random() < 0.7,
         "page": rng.choice([16, 32, 64, 128])}
    if op == "store":
        c["dtype"], c["out"] = rng.choice(["f32", "f16", "bf16"]), rng.choice(["f16", "bf16"])
        c["new"] = _log(rng, 1, 512)
        c["batch"] = _log(rng, 1, max(1, min(64, 16384 * 32 // (c["new"] * (q_heads + 2 * kv_heads)))))
        c["ctx"] = rng.choice([0, _log(rng, 1, 4000)])
    elif op == "read":
        c["out"] = rng.choice(["f16", "bf16"])
        c["len"] = _log(rng, 1, 12000)
        c["batch"] = _log(rng, 1, max(1, min(64, 24 * 3600 * 8 // (c["len"] * kv_heads))))
    elif op == "decode":
        c["dtype"] = rng.choice(["f32", "f16", "bf16"])
        c["len"] = _log(rng, 1, 32768)
        c["batch"] = _log(rng, 1, max(1, min(64, 64 * 2048 * 8 // (c["len"] * kv_heads))))
        c["window"], c["sinks"] = rng.choice([(0, 0), (0, 0), (_log(rng, 1, 5000), 0), (_log(rng, 1, 5000), 4),
                                              (_log(rng, 16, 2000), _log(rng, 1, 200))])
    else:
        c["cache"] = rng.choice(["f16", "bf16"])
        c["dtype"] = rng.choice(["f32", c["cache"]])
        c["shared"], c["tail"] = _log(rng, 16, 16384), _log(rng, 1, 800)
        c["batch"] = _log(rng, 1, max(2, min(80, 64 * 16384 * 8 // ((c["shared"] + c["tail"]) * max(kv_heads, 4)))))
        c["groups"] = _log(rng, 1, max(1, min(c["batch"] // 2, 400000 // (c["shared"] * kv_heads))))
    return c


def _share(c, key, b):
    """Sequence (or group) b's share of c[key]: all of it, or spread from the whole down to a twentieth."""
    n = c[key]
    if not c["ragged"] or b == 0 or n == 0:
        return n
    f = (b * 0.6180339887498949 + (0.37 if key in ("ctx", "tail") else 0.0)) % 1.0
    return max(1, int(n * (0.05 + 0.95 * f * f)))


def _groups(c):
    """Sequences of every group, one at least."""
    if not c["ragged"]:
        return [c["batch"] * (g + 1) // c["groups"] - c["batch"] * g // c["groups"] for g in range(c["groups"])]
    at = [1 + (c["batch"] - c["groups"]) * g * g // (c["groups"] * c["groups"]) + g for g in range(c["groups"])]
    return [b - a for a, b in zip([0] + at[1:], at[1:] + [c["batch"]])]


def _lens(c):
    """(new tokens, total length) of every sequence."""
    if c["op"] in ("decode", "read"):
        return [(1, _share(c, "len", b)) for b in range(c["batch"])]
    if c["op"] == "shared":
        held = [_share(c, "shared", g) for g, n in enumerate(_groups(c)) for _ in range(n)]
        return [(1, n + _share(c, "tail", b)) for b, n in enumerate(held)]
    new = [1 if c["new"] == 1 else _share(c, "new", b) for b in range(c["batch"])]
    return [(n, n + _share(c, "ctx", b)) for b, n in enumerate(new)]


# ---- inputs -------------------------------------------------------------------------------------

def _tables(c, s, lens, g):
    """A shuffled block table; of a group's sequences the pages that its prefix fills are the same ones."""
    page = c["page"]
    per = [-(-n // page) for n in lens]
    full, lead = [0] * len(lens), list(range(len(lens)))
    if c["op"] == "shared":
        b = 0
        for i, n in enumerate(_groups(c)):
            for k in range(b, b + n):
                lead[k], full[k] = b, _share(c, "shared", i) // page if k > b else 0
            b += n
    pages = sum(per) - sum(full) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).cpu()
    table = torch.full((len(lens), max(per)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :full[b]] = table[lead[b], :full[b]]
        table[b, full[b]:n] = order[at:at + n - full[b]]
        at += n - full[b]
    s["table"] = table.cuda()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return pages, lead


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c, s = case, {"case": case}
    if c["op"] == "score":
        R, V = c["rows"], c["vocab"]
        x = torch.randn(R, V, device="cuda", generator=g) * c["spread"]
        s["tokens"] = torch.randint(0, V, (R,), device="cuda", generator=g, dtype=torch.int32)
        if c["masked"]:  # a grammar allows two thirds of the tokens
            x.masked_fill_(torch.rand(V, device="cuda", generator=g) < 1 / 3, -math.inf)
        # every other token is the likeliest; a forbidden one is never scored
        best = x.argmax(-1).to(torch.int32)
        likely = (torch.arange(R, device="cuda") % 2 == 0) | (x.gather(1, s["tokens"].long()[:, None])[:, 0] == -math.inf)
        s["tokens"] = torch.where(likely, best, s["tokens"])
        s["logits"] = x.to(_T[c["dtype"]])
        return s
    lens = _lens(c)
    B, page, kvh, H = c["batch"], c["page"], c["kv_heads"], c["q_heads"]
    pages, lead = _tables(c, s, [n for _, n in lens], g)
    new = [n for n, _ in lens]
    T = s["rows"] = sum(new)
    s["starts"] = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda")
    if c["op"] == "shared":
        s["k"], s["v"] = (torch.randn(pages, kvh, page, D, device="cuda", generator=g).to(_T[c["cache"]]) for _ in "kv")
        sizes = _groups(c)
        held = [_share(c, "shared", i) for i, n in enumerate(sizes) for _ in range(n)]
        s["shared"] = torch.tensor(held, dtype=torch.int32, device="cuda")
        s["groups"] = torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + 1)], dtype=torch.int32, device="cuda")
        table = s["table"].cpu()
        for b in range(B):  # the page in which the prefix ends is copied for every sequence behind the first
            i, n = held[b] // page, held[b] % page
            if n and lead[b] != b:
                for x in (s["k"], s["v"]):
                    x[table[b, i], :, :n] = x[table[lead[b], i], :, :n]
    else:  # rows as the model's: K normalised, V smaller; 8-bit integers with a scale per row
        for n, size in (("k", 1.5), ("v", 0.7)):
            x = torch.randn(pages, kvh, page, D, device="cuda", generator=g) * size
            s[n + "s"] = x.abs().amax(-1) / 127
            s[n] = (x / s[n + "s"][..., None]).round().to(torch.int8)
    if c["op"] in ("store", "read"):  # the 16-bit pages of a prompt pass, in order
        per = [-(-n // page) for _, n in lens]
        s["out_table"] = torch.zeros(B, max(per), dtype=torch.int32)
        for b in range(B):
            s["out_table"][b, :per[b]] = torch.arange(per[b]) + sum(per[:b])
        s["out_table"] = s["out_table"].cuda()
        s["k_out"], s["v_out"] = (torch.zeros(sum(per), kvh, page, D, device="cuda", dtype=_T[c["out"]]) for _ in "kv")
        s["first"] = torch.tensor([n - m for m, n in lens], dtype=torch.int32, device="cuda")
    if c["op"] == "store":
        s["qkv"] = torch.randn(T, (H + 2 * kvh) * D, device="cuda", generator=g).to(_T[c["dtype"]])
        s["q_norm"] = 1 + 0.1 * torch.randn(D, device="cuda", generator=g)
        s["k_norm"] = 1 + 0.1 * torch.randn(D, device="cuda", generator=g)
        far = torch.arange(max(n for _, n in lens), device="cuda", dtype=torch.float64)
        a = far[:, None] * (1.0e6 ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2)))[None]
        s["cos"], s["sin"] = a.cos().float(), a.sin().float()
    elif c["op"] != "read":  # normalised and rotated queries
        s["q"] = (torch.randn(T, H, D, device="cuda", generator=g) * 1.5).to(_T[c["dtype"]])
    return s


# ---- one pass -----------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        from kernel_optimization_webgpu_b200 import runtime as R
        if op == "score":
            return R.score_rows(s["logits"], s["tokens"], top=c["top"])
        if op == "shared":
            return R.paged_attn_decode_shared(s["q"], s["k"], s["v"], s["table"], s["lens"], s["groups"], s["shared"])
        cache = (s["k"], s["v"], s["ks"], s["vs"], s["table"], s["lens"])
        if op == "decode":
            return R.paged_attn_decode_q8(s["q"], *cache, window=c["window"], sinks=c["sinks"])
        if op == "read":
            return R.paged_read_q8(*cache, s["k_out"], s["v_out"], s["out_table"])
        q = R.paged_append_q8(s["qkv"], *cache, s["cos"], s["sin"], c["q_heads"], q_norm=s["q_norm"],
                              k_norm=s["k_norm"], q_starts=s["starts"])
        k, v = R.paged_read_q8(*cache, s["k_out"], s["v_out"], s["out_table"], first=s["first"])
        return q.view(s["rows"], c["q_heads"], D), k, v
    return {"store": _store, "read": _read, "decode": _attend, "shared": _attend, "score": _score}[op](s)


def _rows(s, first):
    """Sequence and position of every position from first[b] on."""
    n = s["lens"].long() - first.long()
    b = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n, output_size=s["counted"])
    at = torch.arange(s["counted"], device="cuda") - (n.cumsum(0) - n)[b]
    return b, first.long()[b] + at


def _copy(s, b, pos):
    c = s["case"]
    src, dst = s["table"].long()[b, pos // c["page"]], s["out_table"].long()[b, pos // c["page"]]
    at = pos % c["page"]
    for n in "kv":
        s[n + "_out"][dst, :, at] = (s[n][src, :, at].float() * s[n + "s"][src, :, at][..., None]).to(_T[c["out"]])
    return s["k_out"], s["v_out"]


def _read(s):
    s["counted"] = sum(n for _, n in _lens(s["case"]))
    return _copy(s, *_rows(s, torch.zeros_like(s["lens"])))


def _store(s):
    c = s["case"]
    H, kvh, page = c["q_heads"], c["kv_heads"], c["page"]
    s["counted"] = s["rows"]
    x = s["qkv"].float().view(s["rows"], H + 2 * kvh, D)
    b, pos = _rows(s, s["first"])
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turned(h, w):
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w
        lo, hi = h[..., :D // 2], h[..., D // 2:]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)

    q, k, v = turned(x[:, :H], s["q_norm"]), turned(x[:, H:H + kvh], s["k_norm"]), x[:, H + kvh:]
    at = s["table"].long()[b, pos // page]
    for n, rows in (("k", k), ("v", v)):
        scale = rows.abs().amax(-1) / 127
        s[n + "s"][at, :, pos % page] = scale
        s[n][at, :, pos % page] = (rows / scale[..., None]).round().to(torch.int8)
    return (q.to(s["qkv"].dtype), *_copy(s, b, pos))


def _attend(s):
    """One query per sequence; every sequence's keys gathered side by side."""
    c = s["case"]
    H, kvh, B = c["q_heads"], c["kv_heads"], c["batch"]
    held = s["table"].long().clamp(min=0)
    k, v = (s[n][held].transpose(2, 3).reshape(B, -1, kvh, D).float() for n in "kv")
    if c["op"] == "decode":
        ks, vs = (s[n][held].transpose(2, 3).reshape(B, -1, kvh) for n in ("ks", "vs"))
        k, v = k.mul_(ks[..., None]), v.mul_(vs[..., None])
    j = torch.arange(k.shape[1], device="cuda")
    n = s["lens"][:, None].long()
    seen = j < n
    if c.get("window"):
        seen = seen & ((j >= n - c["window"]) | (j < c["sinks"]))
    w = torch.matmul(s["q"].float().view(B, kvh, H // kvh, D), k.permute(0, 2, 3, 1)).mul_(D ** -0.5)
    w.masked_fill_(~seen[:, None, None], -math.inf)
    w = w.sub_(w.amax(-1, keepdim=True)).exp_()
    total = w.sum(-1, keepdim=True)
    y = torch.matmul(w, v.masked_fill_((j >= n)[..., None, None], 0.0).transpose(1, 2)) / total
    return y.reshape(B, H, D).to(s["q"].dtype)


def _score(s):
    x = s["logits"].float()
    V, n = x.shape[1], s["case"]["top"]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    entropy = total.log() - e.mul_(torch.where(e > 0, d, 0.0)).sum(-1, keepdim=True) / total
    d -= total.log()
    logp = d.gather(1, s["tokens"].long()[:, None])
    # by value, ties to the lower index: one whole number each
    bits = x.add_(0.0).view(torch.int32).long()
    keys = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 20) + (V - 1 - torch.arange(V, device="cuda"))
    top = keys.topk(n, -1).values % (1 << 20)
    ids = V - 1 - top
    return logp[:, 0], entropy[:, 0], ids.to(torch.int32), d.gather(1, ids)


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "score":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * _SIZE[c["dtype"]] + c["rows"] * (12 + 8 * c["top"]), "flops": 6 * n}
    H, kvh = c["q_heads"], c["kv_heads"]
    lens = _lens(c)
    T, total = sum(n for n, _ in lens), sum(n for _, n in lens)
    row8 = 2 * kvh * (D + 4)  # K and V of a position, with their scales
    if c["op"] == "store":
        act = _SIZE[c["dtype"]]
        far = max(n for _, n in lens) - min(t - n for n, t in lens)
        return {"bytes": T * (D * ((2 * H + 2 * kvh) * act + 2 * kvh * 2) + row8) + min(far, T) * D * 4,
                "flops": T * D * (8 * H + 16 * kvh)}
    if c["op"] == "read":
        return {"bytes": total * (row8 + 2 * kvh * D * 2), "flops": total * 2 * kvh * D}
    act = _SIZE[c["dtype"]]
    if c["op"] == "shared":
        sizes = _groups(c)
        once = sum(_share(c, "shared", g) for g in range(len(sizes)))
        keys = once + total - sum(n * _share(c, "shared", g) for g, n in enumerate(sizes))
        return {"bytes": keys * kvh * D * 4 + 2 * T * H * D * act, "flops": 4 * D * H * total}
    keys = total
    if c["window"]:
        keys = sum(n if n <= c["window"] else c["window"] + min(n - c["window"], c["sinks"]) for _, n in lens)
    return {"bytes": keys * row8 + 2 * T * H * D * act, "flops": 4 * D * H * keys}


# ---- the definitions in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "score":
        return _exact_score(s)
    H, kvh, page = c["q_heads"], c["kv_heads"], c["page"]
    ys, row = [], 0
    kd, vd = (s[n].double() for n in ("k_out", "v_out")) if c["op"] in ("store", "read") else (None, None)
    lead = s["groups"].tolist() if c["op"] == "shared" else None
    for b, (new, n) in enumerate(_lens(c)):
        where = torch.arange(n, device="cuda")
        at = s["table"][b].long()[where // page]
        if lead:  # the shared positions from the group's first sequence
            first = max(x for x in lead[:-1] if x <= b)
            at = torch.where(where < s["shared"][b], s["table"][first].long()[where // page], at)
            k, v = (s[x][at, :, where % page].double() for x in "kv")
        else:
            k, v = (s[x][at, :, where % page].double() * s[x + "s"][at, :, where % page].double()[..., None] for x in "kv")
        if c["op"] == "store":
            x = s["qkv"][row:row + new].double().reshape(new, -1, D)
            row += new
            where, turn = where[n - new:], torch.complex(s["cos"][n - new:n].double(), s["sin"][n - new:n].double())[:, None]
            heads = []
            for part, w in ((x[:, :H], s["q_norm"]), (x[:, H:H + kvh], s["k_norm"])):
                part = part / (part.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
                z = torch.complex(part[..., :D // 2].contiguous(), part[..., D // 2:].contiguous()) * turn
                heads.append(torch.cat([z.real, z.imag], -1))
            ys.append(heads[0])
            k, v = (torch.round(h / h.abs().amax(-1, keepdim=True) * 127) * h.abs().amax(-1, keepdim=True) / 127
                    for h in (heads[1], x[:, H + kvh:]))
        if c["op"] in ("store", "read"):
            to = s["out_table"][b].long()[where // page]
            kd[to, :, where % page], vd[to, :, where % page] = k, v
            continue
        gone = torch.zeros(n, dtype=torch.bool, device="cuda")
        if c.get("window"):
            gone = (n - 1 - where >= c["window"]) & (where >= c["sinks"])
        y = torch.empty(H, D, device="cuda", dtype=torch.float64)
        for g in range(kvh):
            own_heads = slice(g * (H // kvh), (g + 1) * (H // kvh))
            z = s["q"][b, own_heads].double() @ k[:, g].T / math.sqrt(D)
            y[own_heads] = torch.softmax(z.masked_fill(gone, -math.inf), -1) @ v[:, g]
        ys.append(y)
    if c["op"] == "read":
        return kd, vd
    return (torch.cat(ys), kd, vd) if c["op"] == "store" else torch.stack(ys)


def _exact_score(s):
    n, out = s["case"]["top"], []
    for r in range(s["case"]["rows"]):
        x = s["logits"][r].double()
        logp = torch.log_softmax(x, -1)
        p = logp.exp()
        order = torch.argsort(-x, stable=True)[:n]
        out.append((logp[s["tokens"][r].long()], -(p * logp.clamp(min=-1e300)).sum(), order.to(torch.int32), logp[order]))
    return tuple(torch.stack(x) for x in zip(*out))
