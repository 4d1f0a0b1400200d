"""Cases of the device operators: page plans, K/V append, attention over a shared prefix, token log probabilities.

Every operator has a plain form in elementary torch operations (32 bits, rounded once at the end) and the call of
laya_goish_b200.device that a user's program makes.  Ragged sizes come from the case itself ("sizes" seeds them), values
from the seed."""
import math
import random

import torch

own = False

PAGE = 64  # tokens per K/V page
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one decode step of a running batch: a token each, now and then a new page
        {"name": "plan decode step", "op": "plan", "n": 64, "max_past": 4000, "max_count": 1, "pad": 0, "base": 768,
         "sizes": 1},
        # a large batch of prompts and continuations planned at once, capacity beyond what is used
        {"name": "plan ragged prompts", "op": "plan", "n": 4096, "max_past": 700, "max_count": 513, "pad": 4097,
         "base": 0, "sizes": 2},
        # the new rows of one decode step
        {"name": "append decode rows", "op": "append", "rows": 64, "kv": 8, "hd": 64, "src": "f16", "type": "f16",
         "token_major": False, "skip": 0.0, "sizes": 3},
        # a prefill chunk whose projections came in 32 bits, padded rows skipped
        {"name": "append prompt rows", "op": "append", "rows": 16381, "kv": 4, "hd": 128, "src": "f32", "type": "bf16",
         "token_major": True, "skip": 0.02, "sizes": 4},
        # options of one short prompt, one token each
        {"name": "attend 8 options", "op": "attend", "n": 8, "max_q": 1, "fixed_q": True, "heads": 32, "kv": 8,
         "hd": 64, "prefix": 512, "max_own": 63, "type": "f16", "token_major": False, "pad": 0, "sizes": 5},
        # generation of many answers over one document, a length that ends inside a page, heads in groups of seven
        {"name": "attend 64 answers", "op": "attend", "n": 64, "max_q": 1, "fixed_q": True, "heads": 28, "kv": 4,
         "hd": 128, "prefix": 4001, "max_own": 300, "type": "f16", "token_major": False, "pad": 0, "sizes": 6},
        # question suffixes of different lengths over one prompt, a padded batch, some without tokens
        {"name": "attend suffixes", "op": "attend", "n": 24, "max_q": 48, "fixed_q": False, "heads": 32, "kv": 8,
         "hd": 64, "prefix": 1024, "max_own": 48, "type": "f16", "token_major": True, "pad": 37, "sizes": 7},
        # wide heads, an odd batch
        {"name": "attend wide heads", "op": "attend", "n": 33, "max_q": 1, "fixed_q": True, "heads": 8, "kv": 2,
         "hd": 256, "prefix": 6000, "max_own": 700, "type": "bf16", "token_major": False, "pad": 0, "sizes": 8},
        # a full serving batch over a long document, two tokens a sequence
        {"name": "attend long document", "op": "attend", "n": 256, "max_q": 2, "fixed_q": True, "heads": 32, "kv": 8,
         "hd": 128, "prefix": 16384, "max_own": 512, "type": "bf16", "token_major": False, "pad": 0, "sizes": 9},
        # one answer token with its alternatives
        {"name": "logprobs one row", "op": "logprobs", "rows": 1, "vocab": 152064, "tokens": 1, "top": 20,
         "type": "f32", "masked": 0.0, "lowest": False, "gap": 0},
        # option candidates read from a restricted vocabulary, rows of a wider buffer
        {"name": "logprobs candidates", "op": "logprobs", "rows": 48, "vocab": 32000, "tokens": 16, "top": 5,
         "type": "f16", "masked": 0.5, "lowest": False, "gap": 24},
        # the log probabilities of whole prompts
        {"name": "logprobs prompts", "op": "logprobs", "rows": 2048, "vocab": 152064, "tokens": 1, "top": 5,
         "type": "bf16", "masked": 0.0, "lowest": False, "gap": 0},
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "logprobs", "logprobs"])
    sizes = rng.randrange(1 << 30)
    if op == "plan":
        return {"op": op, "n": _log(rng, 1, 4096), "max_past": _log(rng, 1, 4000), "max_count": _log(rng, 1, 512),
                "pad": rng.choice([0, 0, rng.randrange(1, 5000)]), "base": rng.choice([0, rng.randrange(1, 20000)]),
                "sizes": sizes}
    if op == "append":
        kind = rng.choice(["f16", "bf16"])
        return {"op": op, "rows": _log(rng, 1, 16384), "kv": rng.choice([1, 2, 4, 8]), "hd": rng.choice([64, 128, 256]),
                "src": rng.choice([kind, "f32"]), "type": kind, "token_major": rng.random() < 0.5,
                "skip": rng.choice([0.0, 0.1]), "sizes": sizes}
    if op == "attend":
        heads, kv, hd = rng.choice([(32, 8, 64), (28, 4, 128), (32, 8, 128), (8, 2, 256), (16, 16, 64), (12, 1, 128),
                                    (5, 1, 64)])
        max_q = rng.choice([1, 1, _log(rng, 2, 64)])
        n = _log(rng, 1, max(1, min(256, 1024 // max_q)))
        most = (256 * 2 * 32 * 16384) // (n * max_q * heads)
        prefix = _log(rng, 1, max(1, min(16384, most)))
        return {"op": op, "n": n, "max_q": max_q, "fixed_q": rng.random() < 0.5, "heads": heads, "kv": kv, "hd": hd,
                "prefix": rng.choice([prefix, prefix, prefix, 0]), "max_own": max(max_q, _log(rng, 1, 1000)),
                "type": rng.choice(["f16", "bf16"]), "token_major": rng.random() < 0.5,
                "pad": rng.choice([0, 0, rng.randrange(1, 40)]), "sizes": sizes}
    vocab = rng.choice([32000, 152064, _log(rng, 300, 150000), _log(rng, 300, 150000)])
    return {"op": op, "rows": _log(rng, 1, max(1, min(2048, (2048 * 152064) // (vocab * 2)))), "vocab": vocab,
            "tokens": rng.choice([1, rng.randrange(1, 17)]), "top": rng.choice([0, 1, 5, rng.randrange(2, 65)]),
            "type": rng.choice(["f32", "f16", "bf16"]), "masked": rng.choice([0.0, 0.0, 0.5, 0.999]),
            "lowest": rng.random() < 0.3, "gap": rng.choice([0, 0, rng.randrange(1, 50)])}


def _plan_sizes(c):
    """(past, count) of each sequence: half of them fresh where whole prompts come in, empty ones among them."""
    r = random.Random(c["sizes"])
    if c["max_count"] == 1:
        return [r.randint(0, c["max_past"]) for _ in range(c["n"])], [1] * c["n"]
    past = [r.randint(0, c["max_past"]) if r.random() < 0.5 else 0 for _ in range(c["n"])]
    return past, [0 if r.random() < 0.05 else r.randint(1, c["max_count"]) for _ in range(c["n"])]


def _attend_sizes(c):
    """(new tokens, own tokens with them) of each sequence."""
    r = random.Random(c["sizes"])
    new = [c["max_q"] if c["fixed_q"] else r.randint(0, c["max_q"]) for _ in range(c["n"])]
    if not c["fixed_q"]:
        new[r.randrange(c["n"])] = c["max_q"]
    return new, [r.randint(q, max(q, c["max_own"])) for q in new]


def _pages(n):
    return -(-n // PAGE)


def work(case):
    c = case
    if c["op"] == "plan":
        past, count = _plan_sizes(c)
        touched = sum(_pages(p + q) - p // PAGE for p, q in zip(past, count) if q)
        fresh = sum(_pages(p + q) - _pages(p) for p, q in zip(past, count))
        n, t = c["n"], sum(count) + c["pad"]
        return {"bytes": 8 * n + 4 * touched + 16 * t + 4 * (2 * n + 1) + 4 * fresh, "flops": 0}
    if c["op"] == "append":
        x = c["rows"] * c["kv"] * c["hd"] * 2
        return {"bytes": 8 * c["rows"] + x * (4 if c["src"] == "f32" else 2) + x * 2, "flops": 0}
    if c["op"] == "attend":
        new, held = _attend_sizes(c)
        t, row = sum(new), c["heads"] * c["hd"]
        seen = t * c["prefix"] + sum(q * (h - q) + q * (q + 1) // 2 for q, h in zip(new, held))
        keys = c["prefix"] + sum(h for q, h in zip(new, held) if q)
        return {"bytes": 2 * keys * c["kv"] * c["hd"] * 2 + 2 * t * row * 2 + 4 * t * c["heads"],
                "flops": 4 * row * seen}
    size = 4 if c["type"] == "f32" else 2
    return {"bytes": c["rows"] * (c["vocab"] * size + 8 * c["tokens"] + 8 + 8 * c["top"]),
            "flops": 5 * c["rows"] * c["vocab"]}


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def _shuffled(r, n):
    x = list(range(n))
    r.shuffle(x)
    return x


def _cache(c, pages, g):
    """K and V pages, [pages][kv heads][64][hd] or that view of pages held token by token."""
    shape = (pages, PAGE, c["kv"], c["hd"]) if c["token_major"] else (pages, c["kv"], PAGE, c["hd"])
    both = [torch.randn(shape, device="cuda", generator=g).to(TYPES[c["type"]]) for _ in range(2)]
    return [x.permute(0, 2, 1, 3) for x in both] if c["token_major"] else both


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    if c["op"] == "plan":
        past, count = _plan_sizes(c)
        have = [_pages(p) for p in past]
        need = [_pages(p + q) for p, q in zip(past, count)]
        total = sum(need) + 16
        ids = _shuffled(r, total)
        width = max(need) + 2
        rows, at = [], 0
        for h in have:
            rows.append(ids[at:at + h] + [-1] * (width - h))
            at += h
        return {"c": c, "past": _ints(past), "count": _ints(count), "free": _ints(ids[at:]), "tables": _ints(rows),
                "capacity": sum(count) + c["pad"], "base": c["base"]}
    if c["op"] == "append":
        t = c["rows"]
        pages = _pages(t) + 8
        slots = _shuffled(r, pages * PAGE)[:t] if t < 2000 else torch.randperm(
            pages * PAGE, device="cuda", generator=g)[:t].tolist()
        slots = _ints([-1 if r.random() < c["skip"] else s for s in slots], torch.int64)
        k, v = _cache(c, pages, g)
        kv = torch.randn((2, t, c["kv"], c["hd"]), device="cuda", generator=g).to(TYPES[c["src"]])
        return {"c": c, "k": k, "v": v, "new_k": kv[0], "new_v": kv[1], "slots": slots}
    if c["op"] == "attend":
        new, held = _attend_sizes(c)
        pre = _pages(c["prefix"])
        each = [_pages(h) for h in held]
        pages = pre + sum(each) + 3
        ids = _shuffled(r, pages)
        width = max(each) + 1
        rows, at = [], pre
        for e in each:
            rows.append(ids[at:at + e] + [-1] * (width - e))
            at += e
        k, v = _cache(c, pages, g)
        offsets = [0]
        for q in new:
            offsets.append(offsets[-1] + q)
        t = offsets[-1] + c["pad"]
        # queries wide enough that the softmax is neither flat nor a single key
        q = (1.5 * torch.randn((t, c["heads"], c["hd"]), device="cuda", generator=g)).to(TYPES[c["type"]])
        return {"c": c, "q": q, "k": k, "v": v, "prefix_pages": _ints(ids[:pre]), "prefix": c["prefix"],
                "tables": _ints(rows), "lens": _ints(held), "offsets": _ints(offsets), "max_q": c["max_q"],
                "out": torch.zeros_like(q), "lse": torch.zeros((t, c["heads"]), device="cuda")}
    n, vocab = c["rows"], c["vocab"]
    wide = torch.empty((n, vocab + c["gap"]), device="cuda", dtype=TYPES[c["type"]])
    for at in range(0, n, 256):
        x = 2.5 * torch.randn((min(256, n - at), vocab + c["gap"]), device="cuda", generator=g)
        if c["masked"]:
            gone = torch.rand(x.shape, device="cuda", generator=g) < c["masked"]
            x = x.masked_fill(gone, torch.finfo(wide.dtype).min if c["lowest"] else -math.inf)
            x[:, vocab // 2] = 1.0
        wide[at:at + 256] = x.to(wide.dtype)
    tokens = torch.randint(0, vocab, (n, c["tokens"]), device="cuda", generator=g, dtype=torch.int32)
    tokens[:, c["tokens"] - 1] = vocab // 2  # an allowed one
    return {"c": c, "logits": wide[:, :vocab], "tokens": tokens, "top": c["top"]}


def _plan(s):
    past, count, free, tables, cap = s["past"].long(), s["count"].long(), s["free"], s["tables"], s["capacity"]
    n, width = tables.shape
    have, need = (past + PAGE - 1) // PAGE, (past + count + PAGE - 1) // PAGE
    fresh = (need.clamp(max=width) - have).clamp(min=0)
    first = torch.cumsum(fresh, 0) - fresh
    col = torch.arange(width, device=past.device)
    new = (col >= have[:, None]) & (col < (have + fresh)[:, None])
    at = first[:, None] + col - have[:, None]
    ok = (at >= 0) & (at < free.numel())
    tables.copy_(torch.where(new, torch.where(ok, free[at.clamp(0, free.numel() - 1)], -1), tables))
    ends = torch.cumsum(count, 0)
    offsets = torch.cat([ends.new_zeros(1), ends])
    t = torch.arange(cap, device=past.device)
    seq = torch.searchsorted(ends, t, right=True)
    real = seq < n
    i = seq.clamp(max=n - 1)
    u = past[i] + t - offsets[i]
    page = tables[i, (u // PAGE).clamp(max=width - 1)].long()
    held = real & (u // PAGE < width) & (page >= 0)
    return {"tables": tables, "slots": torch.where(held, page * PAGE + u % PAGE, -1),
            "positions": torch.where(real, u + s["base"], 0).int(), "seqs": torch.where(real, seq, -1).int(),
            "offsets": offsets.clamp(max=cap).int(), "lens": (past + count).int(),
            "totals": torch.stack([ends[-1], fresh.sum()])}


def _append(s):
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    s["k"][at // PAGE, :, at % PAGE] = s["new_k"][keep].to(s["k"].dtype)
    s["v"][at // PAGE, :, at % PAGE] = s["new_v"][keep].to(s["v"].dtype)
    return {"k": s["k"], "v": s["v"]}


def _part(scores, values):
    """(maximum, sum, weighted values) of a softmax over the last axis; masked scores are -inf."""
    m = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - m.masked_fill(m == -math.inf, 0.0))
    return m[..., 0], e.sum(-1), e @ values


def _attend(s):
    q, k, v, offsets, lens = s["q"], s["k"], s["v"], s["offsets"].long(), s["lens"].long()
    t, heads, hd = q.shape
    kv, n = k.shape[1], lens.numel()
    group, most = heads // kv, s["max_q"]
    x = q.float().view(t, kv, group, hd) * (1.0 / math.sqrt(hd))
    # the prefix, for all rows
    held = s["prefix_pages"].numel() * PAGE
    kp = k[s["prefix_pages"].long()].permute(1, 0, 2, 3).reshape(kv, held, hd)[:, :s["prefix"]].float()
    vp = v[s["prefix_pages"].long()].permute(1, 0, 2, 3).reshape(kv, held, hd)[:, :s["prefix"]].float()
    rows = x.permute(1, 0, 2, 3).reshape(kv, t * group, hd)
    if s["prefix"]:
        m1, l1, o1 = _part(rows @ kp.transpose(1, 2), vp)
    else:
        m1, l1, o1 = torch.full_like(rows[..., 0], -math.inf), torch.zeros_like(rows[..., 0]), torch.zeros_like(rows)
    m1, l1, o1 = (y.reshape(kv, t, group, -1).permute(1, 0, 2, 3) for y in (m1, l1, o1))
    # each sequence's own keys, its queries padded to the longest
    j = torch.arange(most, device=q.device)
    new = offsets[1:] - offsets[:-1]
    own_q = x[(offsets[:-1, None] + j).clamp(max=t - 1)].permute(0, 2, 1, 3, 4).reshape(n, kv, most * group, hd)
    pages = s["tables"].long().clamp(min=0)
    ks = k[pages].permute(0, 2, 1, 3, 4).reshape(n, kv, -1, hd).float()
    vs = v[pages].permute(0, 2, 1, 3, 4).reshape(n, kv, -1, hd).float()
    key = torch.arange(ks.shape[2], device=q.device)
    seen = key < (lens[:, None] - new[:, None] + j + 1)[..., None]
    seen = seen[:, :, None].expand(n, most, group, -1).reshape(n, 1, most * group, -1)
    m2, l2, o2 = _part((own_q @ ks.transpose(2, 3)).masked_fill(~seen, -math.inf), vs)
    at = torch.arange(t, device=q.device)
    b = torch.searchsorted(offsets[1:].contiguous(), at, right=True)
    real = b < n
    b = b.clamp(max=n - 1)
    m2, l2, o2 = (y.reshape(n, kv, most, group, -1)[b, :, (at - offsets[b]).clamp(0, most - 1)] for y in (m2, l2, o2))
    # joined
    m = torch.maximum(m1, m2)
    safe = m.masked_fill(m == -math.inf, 0.0)
    w1, w2 = torch.exp(m1 - safe), torch.exp(m2 - safe)
    total = w1 * l1 + w2 * l2
    o = torch.where(total > 0, (w1 * o1 + w2 * o2) / total, 0.0).reshape(t, heads, hd).to(q.dtype)
    lse = (safe + torch.log(total)).reshape(t, heads)
    return {"out": torch.where(real[:, None, None], o, s["out"]), "lse": torch.where(real[:, None], lse, s["lse"])}


def _logprobs(s):
    x = s["logits"].float() + 0.0
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(-1)
    lse = m[:, 0] + torch.log(total)
    out = {"logprobs": x.gather(1, s["tokens"].long()) - lse[:, None],
           "entropy": torch.log(total) - torch.where(e > 0, e * d, 0.0).sum(-1) / total, "lse": lse}
    if s["top"]:
        # values as whole numbers of the same order, then the lowest index first among equals
        bits = x.view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
        index = torch.arange(x.shape[1], device=x.device)
        best = torch.topk((order << 20) - index, min(s["top"], x.shape[1]), dim=1).values
        ids = -best & 0xfffff
        top = x.gather(1, ids)
        gone = top == -math.inf
        out["top_ids"] = torch.where(gone, -1, ids).int()
        out["top_logprobs"] = torch.where(gone, -math.inf, top - lse[:, None])
    return out


def _pages_of(device, s):
    """The cache's handle, which a program makes once for a layer."""
    if "pages" not in s:
        s["pages"] = device.KVPages(s["k"], s["v"])
    return s["pages"]


def run(state):
    s = state
    op = s["c"]["op"]
    if own:
        from laya_goish_b200 import device
        if op == "plan":
            p = device.page_plan(s["past"], s["count"], s["free"], s["tables"], s["capacity"], base=s["base"])
            return {"tables": s["tables"], "slots": p.slots, "positions": p.positions, "seqs": p.seqs,
                    "offsets": p.offsets, "lens": p.lens, "totals": p.totals}
        if op == "append":
            device.kv_append(_pages_of(device, s), s["new_k"], s["new_v"], s["slots"])
            return {"k": s["k"], "v": s["v"]}
        if op == "attend":
            device.prefix_attention(s["q"], _pages_of(device, s), s["prefix_pages"], s["prefix"], s["tables"],
                                    s["lens"], s["offsets"], s["max_q"], out=s["out"], lse=s["lse"])
            return {"out": s["out"], "lse": s["lse"]}
        p = device.token_logprobs(s["logits"], s["tokens"], top=s["top"])
        out = {"logprobs": p.logprobs, "entropy": p.entropy, "lse": p.lse}
        return dict(out, top_ids=p.top_ids, top_logprobs=p.top_logprobs) if s["top"] else out
    return {"plan": _plan, "append": _append, "attend": _attend, "logprobs": _logprobs}[op](s)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "plan":
        return None  # whole numbers throughout
    if c["op"] == "append":
        k, v = s["k"].double(), s["v"].double()
        for row, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                k[slot // PAGE, :, slot % PAGE] = s["new_k"][row].double()
                v[slot // PAGE, :, slot % PAGE] = s["new_v"][row].double()
        return {"k": k, "v": v}
    if c["op"] == "attend":
        new, held = _attend_sizes(c)
        group, hd = c["heads"] // c["kv"], c["hd"]
        out, lse = s["out"].double(), s["lse"].double()

        def tokens(x, pages, n):
            return x[pages[:_pages(n)].long()].double().transpose(0, 1).reshape(c["kv"], _pages(n) * PAGE, hd)[:, :n]

        kp, vp = tokens(s["k"], s["prefix_pages"], c["prefix"]), tokens(s["v"], s["prefix_pages"], c["prefix"])
        first = 0
        for b, (n, h) in enumerate(zip(new, held)):
            if n:
                keys = torch.cat([kp, tokens(s["k"], s["tables"][b], h)], 1)
                vals = torch.cat([vp, tokens(s["v"], s["tables"][b], h)], 1)
                x = s["q"][first:first + n].double().view(n, c["kv"], group, hd)
                a = torch.einsum("nkgd,ksd->nkgs", x, keys) / math.sqrt(hd)
                last = c["prefix"] + h - n + torch.arange(n, device="cuda")
                a = a.masked_fill((torch.arange(keys.shape[1], device="cuda") > last[:, None])[:, None, None],
                                  -math.inf)
                lse[first:first + n] = torch.logsumexp(a, -1).view(n, -1)
                out[first:first + n] = torch.einsum("nkgs,ksd->nkgd", torch.softmax(a, -1), vals).reshape(n, -1, hd)
            first += n
        return {"out": out, "lse": lse}
    lp, ent, lse, top = [], [], [], []
    for at in range(0, c["rows"], 128):
        x = s["logits"][at:at + 128].double()
        y = torch.log_softmax(x, -1)
        lse.append(torch.logsumexp(x, -1))
        lp.append(y.gather(1, s["tokens"][at:at + 128].long()))
        ent.append(-torch.where(y > -math.inf, torch.exp(y) * y, 0.0).sum(-1))
        if c["top"]:
            top.append(torch.topk(y, min(c["top"], c["vocab"]), dim=1).values)
    out = {"logprobs": torch.cat(lp), "entropy": torch.cat(ent), "lse": torch.cat(lse)}
    return dict(out, top_ids=None, top_logprobs=torch.cat(top)) if c["top"] else out
