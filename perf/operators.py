"""Measured cases of the paged KV cache operators.

Four operators of a serving step, each in two forms: `own` false, elementary
torch operations in 32 bits; `own` true, the library's calls.

tables  block tables and slot maps from request lengths: pages of a free list
        handed to the requests that grow, pages of ended requests put back,
        and for each new token its position and its slot in the cache
store   rows of new K and V written to their slots
paged   attention of each request's new tokens (one, or a chunk of a prompt)
        over its pages, causal, grouped heads, sinks, sliding window
packed  attention over whole prompts of different lengths packed into one
        tensor, causal, grouped heads, sinks, sliding window
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the bookkeeping of one decode step: 64 requests, one token each
        {"name": "tables, decode step of 64", "op": "tables", "requests": 64, "page": 16, "max_pages": 256, "ctx": 4000,
         "chunks": 0, "chunk": 1, "ended": 0, "tokens": 64, "spare": 64, "pick": 1},
        # the same when prompts join in chunks, requests end and pages run short
        {"name": "tables, 512 with chunks", "op": "tables", "requests": 512, "page": 16, "max_pages": 512, "ctx": 7000,
         "chunks": 60, "chunk": 512, "ended": 25, "tokens": 16384, "spare": 1500, "pick": 2},
        # K and V of one decode step, fp32 activations into a bf16 cache
        {"name": "store, decode step of 64", "op": "store", "tokens": 64, "kv_heads": 8, "dim": 64, "page": 16,
         "src": "f32", "dtype": "bf16", "fused": False, "pad": 0, "slots": 8192},
        # K and V of prefill steps out of a fused projection's rows, some of them padding
        {"name": "store, prompt of 16k", "op": "store", "tokens": 16401, "kv_heads": 8, "dim": 128, "page": 32,
         "src": "bf16", "dtype": "bf16", "fused": True, "pad": 100, "slots": 32768},
        # batch-1 decode at context 4096, 64 query heads over 8 KV heads: the smallest call
        {"name": "paged, one token at 4096", "op": "paged", "requests": 1, "heads": 64, "kv_heads": 8, "dim": 64,
         "page": 16, "dtype": "bf16", "lo": 4096, "hi": 4096, "chunks": 0, "chunk": 1, "new": 1, "sinks": True,
         "window": 0, "pick": 5},
        # batched decode over long ragged contexts
        {"name": "paged, decode of 64 to 8k", "op": "paged", "requests": 64, "heads": 64, "kv_heads": 8, "dim": 64,
         "page": 16, "dtype": "bf16", "lo": 500, "hi": 8000, "chunks": 0, "chunk": 1, "new": 1, "sinks": True,
         "window": 0, "pick": 6},
        # the same in the engine's default precision, a few guessed tokens at a time
        {"name": "paged, f32 guesses of 3", "op": "paged", "requests": 15, "heads": 64, "kv_heads": 8, "dim": 64,
         "page": 16, "dtype": "f32", "lo": 100, "hi": 1500, "chunks": 0, "chunk": 1, "new": 3, "sinks": True,
         "window": 0, "pick": 7},
        # chunks of prompts beside decoding requests in one step
        {"name": "paged, chunks with decode", "op": "paged", "requests": 21, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "dtype": "f16", "lo": 300, "hi": 6000, "chunks": 5, "chunk": 500, "new": 1, "sinks": False,
         "window": 0, "pick": 8},
        # a prefill batch of ordinary prompts
        {"name": "packed, 16 prompts to 2k", "op": "packed", "requests": 16, "heads": 64, "kv_heads": 8, "dim": 64,
         "dtype": "bf16", "lo": 100, "hi": 2048, "sinks": True, "window": 0, "pick": 9},
        # the same of a layer with a 128-token sliding window
        {"name": "packed, window of 128", "op": "packed", "requests": 4, "heads": 64, "kv_heads": 8, "dim": 64,
         "dtype": "bf16", "lo": 1500, "hi": 4000, "sinks": True, "window": 128, "pick": 10},
        # one long prompt with wide heads: the largest
        {"name": "packed, one prompt of 8k", "op": "packed", "requests": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "f16", "lo": 8191, "hi": 8191, "sinks": False, "window": 0, "pick": 11},
        # a few short prompts in the engine's default precision
        {"name": "packed, f32 short prompts", "op": "packed", "requests": 3, "heads": 64, "kv_heads": 8, "dim": 64,
         "dtype": "f32", "lo": 17, "hi": 301, "sinks": True, "window": 0, "pick": 12},
    ]


def draw(rng):
    def size(lo, hi):  # over the logarithm
        return odd(int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    def odd(n):  # 3072 is not among the sizes
        return n + (n == 3072)

    pick = rng.randrange(1 << 30)
    op = rng.choice(["tables", "store", "paged", "paged", "packed", "packed"])
    if op == "tables":
        n, page = size(1, 700), rng.choice([8, 16, 32, 64])
        ctx = size(30, 8000)
        chunks = rng.randint(0, n // 4)
        chunk = size(2, 600)
        return {"op": op, "requests": n, "page": page, "max_pages": (ctx + chunk) // page + rng.randint(1, 9), "ctx": ctx,
                "chunks": chunks, "chunk": chunk, "ended": rng.randint(0, n // 8),
                "tokens": odd(n + chunks * chunk - rng.randint(0, n // 2)), "spare": size(1, 3000), "pick": pick}
    if op == "store":
        n = size(1, 16000)
        return {"op": op, "tokens": n, "kv_heads": rng.choice([1, 2, 4, 8]), "dim": rng.choice([64, 64, 80, 128]),
                "page": rng.choice([8, 16, 32, 64]), "src": rng.choice(["f32", "bf16", "f16"]),
                "dtype": rng.choice(["f32", "bf16", "f16"]), "fused": rng.random() < 0.5, "pad": rng.randint(0, n // 10),
                "slots": 64 * (2 * (n // 128) + 2 * rng.randint(0, 100) + 3)}
    kv_heads, dtype = rng.choice([2, 4, 8]), rng.choice(["bf16", "bf16", "f16", "f32"])
    shape = {"kv_heads": kv_heads, "heads": kv_heads * rng.choice([1, 4, 5, 8]), "dim": rng.choice([64, 64, 80, 128]), "dtype": dtype,
             "sinks": rng.random() < 0.5, "window": rng.choice([0, 0, 128, size(20, 2000)]), "pick": pick}
    if (shape["heads"] + 2 * kv_heads) * shape["dim"] == 3072:
        shape["heads"] += kv_heads
    if op == "paged":
        hi = size(20, 7000 if dtype != "f32" else 2500)
        n = min(size(1, 100), max(1, 400000 // hi))
        chunk = min(size(2, 500), hi)
        chunks = rng.choice([0, rng.randint(0, min(n, 4))])
        return {"op": op, "requests": n, "page": rng.choice([8, 16, 32, 64]), "lo": max(1, hi // rng.randint(1, 9)),
                "hi": hi, "chunks": chunks, "chunk": chunk, "new": rng.choice([1, 1, 1, rng.randint(2, 6)]), **shape}
    hi = size(10, 6000 if dtype != "f32" else 1500)
    n = min(size(1, 30), max(1, 36_000_000 // (hi * hi)))
    return {"op": op, "requests": n, "lo": max(1, hi // rng.randint(1, 9)), "hi": hi, **shape}


def lengths(case):
    """The lengths a case stands for, by its own `pick`: (tokens held, new tokens) of each request."""
    r = random.Random(case["pick"])
    n = case["requests"]
    if case["op"] == "tables":
        held = [r.randint(1, case["ctx"]) for _ in range(n)]
        new = [1] * n
        order = r.sample(range(n), n)
        for b in order[:case["chunks"]]:
            new[b] = r.randint(1, case["chunk"])
        for b in order[n - case["ended"]:]:
            new[b] = -1
        return held, new
    total = [r.randint(case["lo"], case["hi"]) for _ in range(n)]
    if case["op"] == "packed":
        return [0] * n, total
    new = [min(t, case["new"]) for t in total]
    for b in r.sample(range(n), case["chunks"]):
        new[b] = min(total[b], r.randint((case["chunk"] + 1) // 2, case["chunk"]))
    return [t - q for t, q in zip(total, new)], new


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prefix(v):
    return ints([sum(v[:i]) for i in range(len(v) + 1)])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    s = {"op": case["op"]}
    if case["op"] == "store":
        n, h, d, dt = case["tokens"], case["kv_heads"], case["dim"], DTYPES[case["src"]]
        if case["fused"]:  # rows of a projection that holds q, k and v
            rows = normal(n, 7 * h * d, dtype=dt)
            s["k"], s["v"] = rows[:, 5 * h * d:6 * h * d].view(n, h, d), rows[:, 6 * h * d:].view(n, h, d)
        else:
            s["k"], s["v"] = normal(n, h, d, dtype=dt), normal(n, h, d, dtype=dt)
        pages = case["slots"] // case["page"]
        s["k_pages"] = normal(pages, case["page"], h, d, dtype=DTYPES[case["dtype"]])
        s["v_pages"] = normal(pages, case["page"], h, d, dtype=DTYPES[case["dtype"]])
        order = torch.randperm(pages, generator=g, device="cuda")  # consecutive positions, pages in any order
        at = torch.arange(n, device="cuda")
        s["slots"] = order[at // case["page"]] * case["page"] + at % case["page"]
        if case["pad"]:
            s["slots"][n - case["pad"]:] = -1
        return s
    held, new = lengths(case)
    if case["op"] == "tables":
        page, width = case["page"], case["max_pages"]
        have = [-(-t // page) for t in held]
        total = sum(have) + case["spare"]
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        s["kv_len"], s["new_len"] = ints(held), ints(new)
        owns = torch.arange(width, device="cuda") < ints(have)[:, None]
        s["page_table"] = torch.full((len(held), width), -1, dtype=torch.int32, device="cuda")
        s["page_table"][owns] = order[case["spare"]:]
        s["free_pages"] = torch.zeros(total, dtype=torch.int32, device="cuda")
        s["free_pages"][:case["spare"]] = order[:case["spare"]]
        s["n_free"] = ints([case["spare"]])
        s["page_size"], s["n_tokens"] = page, case["tokens"]
        return s
    h, kh, d, dt = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    t = sum(new)
    rows = normal(t, (h + 2 * kh) * d + 16, dtype=dt)  # a projection's rows: q, k, v, and what follows them
    rows[:, :h * d] *= 1.5
    s["q"] = rows[:, :h * d].view(t, h, d)
    s["sinks"] = normal(h) if case["sinks"] else None
    s["window"] = case["window"]
    s["cu_new"], s["most_new"] = prefix(new), max(new)
    if case["op"] == "packed":
        s["k"], s["v"] = rows[:, h * d:(h + kh) * d].view(t, kh, d), rows[:, (h + kh) * d:-16].view(t, kh, d)
        return s
    page = case["page"]
    total = [a + b for a, b in zip(held, new)]
    have = [-(-n // page) for n in total]
    pages = sum(have) + 7
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    owns = torch.arange(max(have), device="cuda") < ints(have)[:, None]
    s["page_table"] = torch.full((len(total), max(have)), -1, dtype=torch.int32, device="cuda")
    s["page_table"][owns] = order[:sum(have)]
    s["kv_len"] = ints(total)
    s["k_pages"], s["v_pages"] = normal(pages, page, kh, d, dtype=dt), normal(pages, page, kh, d, dtype=dt)
    return s


def run(s):
    if own:
        return RUN_OWN[s["op"]](s)
    return RUN_PLAIN[s["op"]](s)


# ---- the library's calls ----------------------------------------------------


def own_tables(s):
    from picchio_b200 import kv_tables
    t = kv_tables(s["kv_len"], s["new_len"], s["page_table"], s["free_pages"], s["n_free"],
                  page_size=s["page_size"], n_tokens=s["n_tokens"])
    return {"page_table": s["page_table"], "free_pages": s["free_pages"], "n_free": t.n_free, "kv_len": t.kv_len,
            "cu_new": t.cu_new, "served": t.served, "positions": t.positions, "slots": t.slots}


def own_store(s):
    from picchio_b200 import kv_store
    kv_store(s["k_pages"], s["v_pages"], s["k"], s["v"], s["slots"])
    return {"k": s["k_pages"], "v": s["v_pages"]}


_attention = []


def attention():
    """The handle that a program keeps beside its model (workspace of the split sums)."""
    if not _attention:
        from picchio_b200 import Attention
        _attention.append(Attention())
    return _attention[0]


def own_paged(s):
    return {"out": attention().paged(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["cu_new"], s["kv_len"],
                                     sinks=s["sinks"], window=s["window"])}


def own_packed(s):
    return {"out": attention().packed(s["q"], s["k"], s["v"], s["cu_new"], sinks=s["sinks"], window=s["window"])}


RUN_OWN = {"tables": own_tables, "store": own_store, "paged": own_paged, "packed": own_packed}

# ---- the plain forms --------------------------------------------------------


def plain_tables(s):
    kv, new, page, n_tokens = s["kv_len"].long(), s["new_len"].long(), s["page_size"], s["n_tokens"]
    table, free, n_free = s["page_table"].long(), s["free_pages"].long(), s["n_free"].long()
    width, room = table.shape[1], free.shape[0]
    ended = new < 0
    held = (kv + page - 1) // page
    fits = ~ended & (kv + new <= width * page)
    add = torch.where(fits, new, 0)
    want = torch.where(fits, (kv + add + page - 1) // page - held, 0)
    give = torch.where(ended, held, 0)
    column = torch.arange(width, device=kv.device)
    back = n_free + (give.cumsum(0) - give)[:, None] + column  # where each page of an ended request goes
    back = torch.where(column < give[:, None], back, room).clamp(max=room)
    free = torch.cat([free, free.new_zeros(1)]).scatter(0, back.reshape(-1), table.reshape(-1))[:room]
    avail = n_free + give.sum()
    upto, tokens = want.cumsum(0), add.cumsum(0)
    served = fits & ((want == 0) | (upto <= avail)) & ((add == 0) | (tokens <= n_tokens))
    nth = (upto - want)[:, None] + column - held[:, None]
    grows = served[:, None] & (column >= held[:, None]) & (column < (held + want)[:, None])
    table = torch.where(grows, free[(avail - 1 - nth).clamp(0, room - 1)], table)
    took = torch.where(served, add, 0)
    cu = torch.cat([took.new_zeros(1), took.cumsum(0)])
    at = torch.arange(n_tokens, device=kv.device)
    b = torch.searchsorted(cu[1:].contiguous(), at, right=True).clamp(max=kv.shape[0] - 1)
    live = at < cu[-1]
    pos = kv[b] + at - cu[b]
    slot = table[b, (pos // page).clamp(0, width - 1)] * page + pos % page
    return {"page_table": table.int(), "free_pages": free.int(),
            "n_free": (avail - torch.where(served, want, 0).sum()).int(),
            "kv_len": torch.where(ended, 0, kv + took).int(), "cu_new": cu.int(), "served": served.int(),
            "positions": torch.where(live, pos, -1).int(), "slots": torch.where(live, slot, -1)}


def plain_store(s):
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    for pages, rows in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])):
        pages.view(-1, *pages.shape[2:])[at] = rows[keep].float().to(pages.dtype)
    return {"k": s["k_pages"], "v": s["v_pages"]}


def attend(q, k, v, q_pos, k_len, sinks, window):
    """q [B, Q, H, D] at positions q_pos [B, Q], k and v [B, L, KH, D] of which k_len [B] are there."""
    n, most, h, d = q.shape
    length, kh = k.shape[1], k.shape[2]
    at = torch.arange(length, device=q.device)
    there = at < k_len[:, None]
    sees = there[:, None, :] & (at <= q_pos[:, :, None])
    if window:
        sees &= at > q_pos[:, :, None] - window
    q = (q.float() / math.sqrt(d)).view(n, most, kh, h // kh, d).permute(0, 2, 3, 1, 4)
    k = k.float().permute(0, 2, 3, 1)[:, :, None]
    v = torch.where(there[:, :, None, None], v.float(), 0.0).permute(0, 2, 1, 3)[:, :, None]
    p = torch.matmul(q, k).masked_fill_(~sees[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    if sinks is not None:
        sinks = sinks.float().view(1, kh, h // kh, 1, 1)
        top = torch.maximum(top, sinks)
    top = torch.where(top == -math.inf, 0.0, top)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks - top)
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 3, 1, 2, 4).reshape(n, most, h, d)


def padded(s):
    """For each request its rows of the packed tensors, padded to the longest; and where each packed row is among them."""
    cu = s["cu_new"].long()
    i = torch.arange(s["most_new"], device=cu.device)
    rows = (cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    t = torch.arange(s["q"].shape[0], device=cu.device)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return cu[1:] - cu[:-1], i, rows, (b, t - cu[b])


def plain_paged(s):
    n_new, i, rows, back = padded(s)
    kv = s["kv_len"].long()
    table = s["page_table"].long().clamp(min=0)
    k, v = (p[table].flatten(1, 2) for p in (s["k_pages"], s["v_pages"]))
    out = attend(s["q"][rows], k, v, (kv - n_new)[:, None] + i, kv, s["sinks"], s["window"])
    return {"out": out[back].to(s["q"].dtype)}


def plain_packed(s):
    n_new, i, rows, back = padded(s)
    out = attend(s["q"][rows], s["k"][rows], s["v"][rows], i.expand(rows.shape), n_new, s["sinks"], s["window"])
    return {"out": out[back].to(s["q"].dtype)}


RUN_PLAIN = {"tables": plain_tables, "store": plain_store, "paged": plain_paged, "packed": plain_packed}

# ---- what a pass cannot do without, and the same in 64 bits -----------------


def work(case):
    if case["op"] == "store":
        size = {"f32": 4, "f16": 2, "bf16": 2}
        rows = (case["tokens"] - case["pad"]) * case["kv_heads"] * case["dim"] * 2
        return {"bytes": rows * (size[case["src"]] + size[case["dtype"]]) + 8 * case["tokens"], "flops": 0}
    held, new = lengths(case)
    if case["op"] == "tables":
        page = case["page"]
        moved = sum(-(-t // page) if a < 0 else -(-(t + a) // page) - -(-t // page) for t, a in zip(held, new))
        # each length and count in and out, each page that changes hands read and written, each token's two numbers
        return {"bytes": 20 * len(held) + 8 * moved + 12 * case["tokens"] + 12, "flops": 0}
    size = 4 if case["dtype"] == "f32" else 2
    keys = pairs = 0
    for a, q in zip(held, new):
        w = case["window"] or a + q
        keys += min(a + q, w + q - 1)
        n = min(max(w - a, 0), q)  # rows that see all positions before them
        pairs += n * a + n * (n + 1) // 2 + (q - n) * w
    rows = sum(new) * case["heads"] * case["dim"] * 2 + keys * case["kv_heads"] * case["dim"] * 2
    pages = 4 * sum(-(-(a + q) // case["page"]) for a, q in zip(held, new)) if case["op"] == "paged" else 0
    return {"bytes": rows * size + pages + 8 * len(new) + (4 * case["heads"] if case["sinks"] else 0),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    if case["op"] == "store":
        out = {}
        for name in ("k", "v"):
            page = s[name + "_pages"].double().flatten(0, 1)
            n = case["tokens"] - case["pad"]
            page.index_copy_(0, s["slots"][:n], s[name][:n].double())
            out[name] = page.view(s[name + "_pages"].shape)
        return out
    held, new = lengths(case)
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    group = h // kh
    out = torch.zeros(sum(new), h, d, dtype=torch.float64, device="cuda")
    first = 0
    for b, (a, n) in enumerate(zip(held, new)):
        if case["op"] == "paged":
            pages = s["page_table"][b, :-(-(a + n) // case["page"])].long()
            k, v = (p[pages].flatten(0, 1)[:a + n].double() for p in (s["k_pages"], s["v_pages"]))
        else:
            k, v = s["k"][first:first + n].double(), s["v"][first:first + n].double()
        for r0 in range(0, n, 2048):
            r1 = min(n, r0 + 2048)
            row = torch.arange(a + r0, a + r1, device="cuda")[:, None]
            key = torch.arange(a + n, device="cuda")[None]
            hidden = (key > row) | (key <= row - (case["window"] or a + n))
            for head in range(h):
                z = s["q"][first + r0:first + r1, head].double() @ k[:, head // group].T * d ** -0.5
                z = z.masked_fill(hidden, -math.inf)
                sink = s["sinks"][head].double().expand(r1 - r0, 1) if case["sinks"] else z[:, :0]
                p = torch.softmax(torch.cat([z, sink], 1), 1)[:, :a + n]
                out[first + r0:first + r1, head] = p @ v[:, head // group]
        first += n
    return {"out": out}
