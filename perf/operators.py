"""Measured cases of the paged key / value cache and the operators around it.

Four operators of ``domino_b200.paged.PagedKVCache``:

* ``write``   query / key norm, rotary positions, and the store of a chunk's keys and values into pages;
* ``attend``  attention of a chunk of new tokens (one or many) over the paged cache, causal or over the whole block,
              also with a sliding window and first tokens that stay visible;
* ``fork`` + ``reserve``  rows that share pages, and the copy of a shared last page before it is written;
* ``compact`` pages in use moved to the front of the pool.

``run`` computes them in a plain form (elementary torch operations in 32 bits) or, with ``own`` set, through the
framework's calls.  ``exact`` restates the definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    served = {"heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64}
    att = {"op": "attend", "causal": True, "window": 0, "sinks": 0}
    return [
        # one request, one new token after a short prompt: the smallest call of plain decoding, all latency
        {"name": "attend_one_token", **att, **served, "batch": 1, "tokens": 1, "past_min": 528, "past_max": 528},
        # the verify pass of the end-to-end loop: 2 requests, blocks of 16, prompt 512, 2048 new tokens
        {"name": "attend_verify_b2", **att, **served, "batch": 2, "tokens": 16, "past_min": 512, "past_max": 2560},
        # the verify pass of a full server: 32 requests of very different lengths
        {"name": "attend_verify_b32", **att, **served, "batch": 32, "tokens": 16, "past_min": 4001, "past_max": 16383},
        # plain decoding of many requests, some of them just begun, small pages, fp16
        {"name": "attend_decode_b64", **att, **served, "dtype": "fp16", "page": 16, "batch": 64, "tokens": 1,
         "past_min": 0, "past_max": 8190},
        # the second chunk of a long prompt: as many new tokens as cached ones
        {"name": "attend_prefill_8k", **att, **served, "batch": 1, "tokens": 8192, "past_min": 8192, "past_max": 8192},
        # odd chunk over a long past with a window and sinks; five query heads per key head, 96 wide
        {"name": "attend_window_sinks", **att, "heads": 40, "kv_heads": 8, "dim": 96, "dtype": "fp16", "page": 32,
         "batch": 4, "tokens": 515, "past_min": 900, "past_max": 30011, "window": 1024, "sinks": 4},
        # the drafter's block: every position of the block sees the whole block, 32-bit weights
        {"name": "attend_draft_block_fp32", **att, "heads": 16, "kv_heads": 4, "dim": 64, "dtype": "fp32", "page": 32,
         "batch": 3, "tokens": 16, "past_min": 300, "past_max": 1500, "causal": False},
        # the block's queries and keys on their way into the cache, as the verify pass writes them
        {"name": "write_verify_b2", "op": "write", **served, "batch": 2, "tokens": 16, "past_min": 512, "past_max": 2560,
         "rotary": 128, "interleaved": False, "norm": True, "stretch": 1.0},
        # a prompt batch on its way into the cache
        {"name": "write_prefill", "op": "write", **served, "batch": 4, "tokens": 8192, "past_min": 0, "past_max": 0,
         "rotary": 128, "interleaved": False, "norm": True, "stretch": 1.0},
        # odd chunks far behind the trained length: half of the head rotated in interleaved pairs, stretched frequencies
        {"name": "write_far_interleaved", "op": "write", "heads": 28, "kv_heads": 4, "dim": 128, "dtype": "fp16",
         "page": 32, "batch": 7, "tokens": 333, "past_min": 700001, "past_max": 1000003, "rotary": 64,
         "interleaved": True, "norm": False, "stretch": 4.0},
        # 32 requests continue one prompt: shared pages, and a copy of its last page for each
        {"name": "fork_b32", "op": "fork", "layers": 4, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64,
         "batch": 32, "tokens": 16, "past": 4021},
        # a pool half given back: the pages still in use move to the front
        {"name": "compact_512", "op": "compact", "layers": 4, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64,
         "pages": 512, "batch": 16, "row_pages": 17},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = [work(c) for c in listed()]
    most_bytes, most_flops = max(w["bytes"] for w in top), max(w["flops"] for w in top)
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return c


def _draw(rng):
    op = rng.choice(["attend"] * 4 + ["write"] * 2 + ["fork", "compact"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    page = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    if op == "fork":
        return {"op": op, "layers": rng.randint(1, 6), "kv_heads": kv_heads, "dim": rng.choice([64, 96, 128]),
                "dtype": dtype, "page": page, "batch": _log(rng, 2, 64), "tokens": _log(rng, 1, 40),
                "past": _log(rng, 3, 5000)}
    if op == "compact":
        batch = rng.randint(2, 24)
        row_pages = _log(rng, 1, 24)
        return {"op": op, "layers": rng.randint(1, 4), "kv_heads": kv_heads, "dim": rng.choice([64, 96, 128]),
                "dtype": dtype, "page": page, "pages": batch * row_pages + _log(rng, 1, 200), "batch": batch,
                "row_pages": row_pages}
    group = rng.choice([1, 2, 3, 4, 5, 8])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128])
    batch = _log(rng, 1, 64)
    base = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page}
    if op == "write":
        past = _log(rng, 1, 1000000)
        rotary = rng.choice([dim, dim, dim // 2, dim // 4])
        return {**base, "batch": batch, "tokens": _log(rng, 1, 4000), "past_min": past // 2, "past_max": past,
                "rotary": rotary - rotary % 2, "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.5,
                "stretch": rng.choice([1.0, 1.0, 4.0])}
    tokens = 1 if rng.random() < 0.35 else _log(rng, 2, 24) if rng.random() < 0.6 else _log(rng, 25, 4000)
    if dtype == "fp32":  # 32-bit products: the drafter's blocks and short chunks
        tokens, batch = min(tokens, 48), min(batch, 8)
    past = _log(rng, 1, 30000 if dtype != "fp32" else 3000)
    causal = rng.random() < 0.8
    window = _log(rng, 1, 4000) if causal and rng.random() < 0.35 else 0
    return {**base, "batch": batch, "tokens": tokens, "past_min": rng.randint(0, past), "past_max": past,
            "causal": causal, "window": window, "sinks": rng.choice([0, 1, 4, 64]) if window else 0}


def _pasts(case):
    """Cached tokens of each row before the chunk: spread evenly between the case's bounds."""
    n, lo, hi = case["batch"], case["past_min"], case["past_max"]
    return [hi if n == 1 else lo + (hi - lo) * b // (n - 1) for b in range(n)]


def _lens(case):
    """New tokens of each row: all of the chunk, but every fifth row ends early."""
    return [case["tokens"] if b % 5 != 4 else max(1, case["tokens"] * 2 // 3) for b in range(case["batch"])]


def _visible(past, n, causal, window, sinks):
    """(query, key) pairs that see one another, and keys that any query sees, for n new tokens after `past`."""
    if not causal:
        return n * (past + n), past + n
    if not window:
        return n * past + n * (n + 1) // 2, past + n
    pairs = 0
    for t in range(n):
        p = past + t
        near = min(window, p + 1)
        pairs += near + min(sinks, p + 1 - near)
    first = max(0, past - window + 1)
    return pairs, past + n - first + min(sinks, first)


def work(case):
    w = _DT[case["dtype"]].itemsize
    if case["op"] == "attend":
        nbytes = flops = 0
        for past, n in zip(_pasts(case), _lens(case)):
            pairs, keys = _visible(past, n, case["causal"], case["window"], case["sinks"])
            nbytes += 2 * keys * case["kv_heads"] * case["dim"] * w + 2 * n * case["heads"] * case["dim"] * w
            flops += 4 * pairs * case["heads"] * case["dim"]
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "write":
        n = sum(_lens(case))
        return {"bytes": 2 * n * (case["heads"] + 2 * case["kv_heads"]) * case["dim"] * w,
                "flops": n * (case["heads"] + case["kv_heads"]) * (3 * case["rotary"] + 4 * case["dim"] * case["norm"])}
    page = 2 * case["layers"] * case["kv_heads"] * case["page"] * case["dim"] * w
    if case["op"] == "fork":  # each row but one copies the shared last page, where it is not full
        moved = (case["batch"] - 1) * (case["past"] % case["page"] > 0)
        return {"bytes": 2 * moved * page + 2 * 4 * case["batch"] * (case["past"] // case["page"] + 1), "flops": 0}
    used, _ = _holes(case)
    table = case["batch"] * case["row_pages"]
    return {"bytes": 2 * page * sum(p >= len(used) for p in used) + 2 * 4 * table, "flops": 0}


def _holes(case):
    """Pages in use of a pool whose odd rows were given back (ascending), and the rows that hold them."""
    step = _stride(case["pages"])
    rows = [b for b in range(case["batch"]) if b % 2 == 0]
    used = [(b * case["row_pages"] + s) * step % case["pages"] for b in rows for s in range(case["row_pages"])]
    return sorted(used), rows


def _stride(pages):
    """A step that visits every page once, scattered."""
    step = max(1, int(pages * 0.618))
    while math.gcd(step, pages) != 1:
        step += 1
    return step


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inv_freq(case):
    """Rotary frequencies: theta 1e6, the slow half of them stretched for a longer context, and the factor on cos and sin."""
    half = case["rotary"] // 2
    inv = 1e6 ** (-torch.arange(half, dtype=torch.float64) * 2 / case["rotary"])
    ramp = ((torch.arange(half, dtype=torch.float64) - half / 4) / max(half / 2, 1)).clamp(0, 1)
    inv = inv * (1 - ramp) + inv / case["stretch"] * ramp
    factor = 1.0 if case["stretch"] == 1.0 else 0.1 * math.log(case["stretch"]) + 1.0
    return inv.to(torch.float32).cuda(), factor


def _inputs(case, seed):
    """Everything a call takes, as plain tensors: pool, tables and the chunk's own data."""
    g = _generator(seed)
    dt, op = _DT[case["dtype"]], case["op"]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32 if dt == torch.float32 else torch.float16)
                * scale).to(dt)

    D, KV, page, B = case["dim"], case["kv_heads"], case["page"], case["batch"]
    s = {"case": case, "page": page}
    if op in ("attend", "write"):
        T = case["tokens"]
        pasts, lens = _pasts(case), _lens(case)
        row_pages = max(-(-(p + T) // page) for p in pasts) + 1
        # a write touches the pages from the row's past on; the attention reads them all
        first = [p // page if op == "write" else 0 for p in pasts]
        count = [-(-(p + n) // page) - f for p, n, f in zip(pasts, lens, first)]
        pages = sum(count) + 3
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
        table = torch.full((B, row_pages), -1, dtype=torch.int32)
        at = 0
        for b in range(B):
            table[b, first[b]: first[b] + count[b]] = order[at: at + count[b]]
            at += count[b]
        refs = torch.zeros(pages, dtype=torch.int32)
        refs[order[:at].long()] = 1
        s.update(table=table.cuda(), refs=refs.cuda(), start=torch.tensor(pasts, device="cuda"),
                 lens=torch.tensor(lens, device="cuda"))
        s["data"] = randn(1, 2, pages, KV, page, D)
        s["length"] = s["start"].clone()
        s["q"] = randn(B, T, case["heads"], D, scale=2.0)  # attention that prefers some keys
        if op == "write":
            s["k"], s["v"] = randn(B, T, KV, D), randn(B, T, KV, D)
            s["inv_freq"], s["factor"] = _inv_freq(case)
            s["q_norm"] = (1 + 0.1 * randn(D).float()).to(dt) if case["norm"] else None
            s["k_norm"] = (1 + 0.1 * randn(D).float()).to(dt) if case["norm"] else None
        return s
    if op == "fork":
        n = -(-case["past"] // page)
        row_pages = -(-(case["past"] + case["tokens"]) // page)
        pages = n + B * (row_pages - n + 1) + 2
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        s["table"] = torch.full((B, row_pages), -1, dtype=torch.int32, device="cuda")
        s["table"][0, :n] = order[:n]
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
        s["refs"][order[:n].long()] = 1
        s["length"] = torch.zeros(B, dtype=torch.long, device="cuda")
        s["length"][0] = case["past"]
        s["src"] = torch.zeros(B, dtype=torch.long, device="cuda")
        s["upto"] = torch.full((B,), case["past"] + case["tokens"], dtype=torch.long, device="cuda")
    else:
        pages, n = case["pages"], case["row_pages"]
        used, rows = _holes(case)
        step = _stride(pages)
        table = torch.full((B, n), -1, dtype=torch.int32)
        for b in rows:
            table[b] = torch.tensor([(b * n + i) * step % pages for i in range(n)], dtype=torch.int32)
        refs = torch.zeros(pages, dtype=torch.int32)
        refs[torch.tensor(used)] = 1
        s["table"], s["refs"] = table.cuda(), refs.cuda()
        s["length"] = torch.tensor([n * page if b in rows else 0 for b in range(B)], device="cuda")
        s["saved"] = (s["table"].clone(), s["refs"].clone())
    s["data"] = randn(case["layers"], 2, pages, KV, page, D)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from domino_b200 import PagedKVCache, Rope

        layers, _, pages, kv_heads, page, dim = s["data"].shape
        cache = PagedKVCache(layers, case["batch"], kv_heads, pages, dim, s["data"].dtype, s["data"].device,
                             page_size=page, row_pages=s["table"].shape[1])
        for name in ("data", "table", "length", "refs"):
            getattr(cache, name).copy_(s[name])
            s[name] = getattr(cache, name)
        s["cache"] = cache
        if case["op"] == "write":
            s["rope"] = Rope(dim, inv_freq=s["inv_freq"], factor=s["factor"], interleaved=case["interleaved"])
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    return {"attend": _attend, "write": _write, "fork": _fork, "compact": _compact}[c["op"]](s, c)


def _attend(s, c):
    if own:
        return s["cache"].attend(0, s["q"], s["start"], s["lens"], causal=c["causal"], window=c["window"],
                                 sinks=c["sinks"])
    q = s["q"]
    out = torch.zeros_like(q)
    group = c["heads"] // c["kv_heads"]
    for b, (past, n) in enumerate(zip(_pasts(c), _lens(c))):  # the plain form knows the lengths on the host
        # with a window only its own pages and the sinks' are gathered
        total = past + n
        far = max(0, past - c["window"] + 1) if c["window"] else 0
        pos = torch.arange(far, total, device=q.device)
        if far:
            pos = torch.cat([torch.arange(min(c["sinks"], far), device=q.device), pos])
        at, off = s["table"][b].long()[pos // s["page"]], pos % s["page"]
        k = s["data"][0, 0][at, :, off].float().transpose(0, 1)  # [KV, keys, D]
        v = s["data"][0, 1][at, :, off].float().transpose(0, 1)
        step = max(1, (1 << 28) // (c["heads"] * len(pos)))
        for t0 in range(0, n, step):
            t1 = min(n, t0 + step)
            qq = q[b, t0:t1].float().transpose(0, 1).reshape(c["kv_heads"], group * (t1 - t0), -1)
            w = torch.bmm(qq, k.transpose(1, 2)) * c["dim"] ** -0.5
            if c["causal"]:
                p = past + torch.arange(t0, t1, device=q.device)[:, None]
                hidden = pos[None] > p
                if c["window"]:
                    hidden = hidden | ((pos[None] <= p - c["window"]) & (pos[None] >= c["sinks"]))
                w.view(c["kv_heads"], group, t1 - t0, -1).masked_fill_(hidden, float("-inf"))
            w = torch.exp(w - w.amax(-1, keepdim=True))
            o = torch.bmm(w, v) / w.sum(-1, keepdim=True)
            out[b, t0:t1] = o.reshape(c["heads"], t1 - t0, -1).transpose(0, 1).to(q.dtype)
    return out


def _write(s, c):
    if own:
        q = s["cache"].write(0, s["q"], s["k"], s["v"], s["rope"], s["start"], s["lens"], q_norm=s["q_norm"],
                             k_norm=s["k_norm"], eps=1e-6)
        return {"q": q, "data": s["data"]}
    T, r = c["tokens"], c["rotary"]
    t = torch.arange(T, device=s["q"].device)
    pos = s["start"][:, None] + t[None]
    live = t[None] < s["lens"][:, None]
    angle = pos.double()[..., None] * s["inv_freq"].double()  # far positions: 32 bits lose the angle
    cos, sin = (angle.cos() * s["factor"]).float()[:, :, None], (angle.sin() * s["factor"]).float()[:, :, None]

    def place(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
        y = x.clone()
        a, b = (slice(0, r, 2), slice(1, r, 2)) if c["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
        return y.to(s["q"].dtype)

    q = place(s["q"], s["q_norm"]) * live[:, :, None, None]
    k = place(s["k"], s["k_norm"])
    b, i = live.nonzero(as_tuple=True)
    p = pos[b, i]
    at = s["table"][b, p // s["page"]].long()
    s["data"][0, 0][at, :, p % s["page"]] = k[b, i]
    s["data"][0, 1][at, :, p % s["page"]] = s["v"][b, i]
    return {"q": q, "data": s["data"]}


def _reserve_plain(table, length, refs, upto, page, data):
    """Pages for positions length .. upto - 1 of every row, lowest free page first; a shared page that will be written
    is copied, unless no row but the first that needs it holds it."""
    slots = torch.arange(table.shape[1], device=table.device)[None]
    first, last = length // page, (upto + page - 1) // page
    grows = upto > length
    want = grows[:, None] & (slots >= first[:, None]) & (slots < last[:, None])
    fresh = want & (table < 0)
    at = table.long().clamp(min=0)
    edge = want & (slots == first[:, None]) & (table >= 0)
    b, i = edge.nonzero(as_tuple=True)
    held = table[b, i].long()
    same = held[:, None] == held[None]
    rank = torch.tril(same, -1).sum(1)
    copies = (refs[held] > 1) & ((rank > 0) | (refs[held] > same.sum(1)))
    fresh[b[copies], i[copies]] = True
    old = at[b[copies], i[copies]]
    rows, cols = fresh.nonzero(as_tuple=True)
    free = (refs == 0).nonzero()[:, 0][: rows.numel()]
    table[rows, cols] = free.to(table.dtype)
    refs[free] = 1
    refs.index_put_((old,), torch.full_like(old, -1, dtype=refs.dtype), accumulate=True)
    data[:, :, table[b[copies], i[copies]].long()] = data[:, :, old]


def _fork(s, c):
    if own:
        s["cache"].fork(s["src"])
        s["cache"].reserve(s["upto"])
    else:
        table, length, refs, src = s["table"], s["length"], s["refs"], s["src"]
        slots = torch.arange(table.shape[1], device=table.device)[None]
        moved = src != torch.arange(len(src), device=src.device)
        kept = slots * s["page"] < length[src][:, None]
        new = torch.where(kept, table[src], torch.full_like(table, -1))
        new = torch.where(moved[:, None], new, table)
        for t, sign in ((table, -1), (new, 1)):
            pages = t[t >= 0].long()
            refs.index_put_((pages,), torch.full_like(pages, sign, dtype=refs.dtype), accumulate=True)
        table.copy_(new)
        length.copy_(length[src])
        _reserve_plain(table, length, refs, s["upto"], s["page"], s["data"])
    return {"table": s["table"], "length": s["length"], "refs": s["refs"], "data": s["data"]}


def _compact(s, c):
    # the pool as the retired rows left it, so that each pass has the same pages to move
    s["table"].copy_(s["saved"][0])
    s["refs"].copy_(s["saved"][1])
    if own:
        s["cache"].compact()
    else:
        table, refs, data = s["table"], s["refs"], s["data"]
        used = refs > 0
        n = used.sum()
        index = torch.arange(len(refs), device=refs.device)
        src = (used & (index >= n)).nonzero()[:, 0]
        dst = (~used & (index < n)).nonzero()[:, 0]
        data[:, :, dst] = data[:, :, src]
        refs[dst] = refs[src]
        refs[src] = 0
        index[src] = dst
        table.copy_(torch.where(table >= 0, index[table.long().clamp(min=0)].to(table.dtype), table))
    return {"table": s["table"], "refs": s["refs"], "data": s["data"]}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    c, page = case, case["page"]
    if c["op"] == "attend":
        group, D = c["heads"] // c["kv_heads"], c["dim"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, (past, n) in enumerate(zip(_pasts(c), _lens(c))):
            slots = s["table"][b, : -(-(past + n) // page)].long()
            for h in range(c["kv_heads"]):
                k = s["data"][0, 0, slots, h].reshape(-1, D)[: past + n].double()
                v = s["data"][0, 1, slots, h].reshape(-1, D)[: past + n].double()
                j = torch.arange(past + n, device="cuda")
                for t0 in range(0, n, 512):
                    t1 = min(n, t0 + 512)
                    qh = s["q"][b, t0:t1, h * group: (h + 1) * group].double()
                    logits = torch.einsum("tgd,jd->tgj", qh, k) / math.sqrt(D)
                    if c["causal"]:
                        p = past + torch.arange(t0, t1, device="cuda")
                        see = j[None] <= p[:, None]
                        if c["window"]:
                            see &= (p[:, None] - j[None] < c["window"]) | (j[None] < c["sinks"])
                        logits = torch.where(see[:, None], logits, -math.inf)
                    out[b, t0:t1, h * group: (h + 1) * group] = torch.softmax(logits, -1) @ v
        return out
    if c["op"] == "write":
        data, q_out = s["data"].double(), torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        r = c["rotary"]
        for b, (past, n) in enumerate(zip(_pasts(c), _lens(c))):
            p = torch.arange(past, past + n, device="cuda")
            turn = torch.polar(torch.full((n, r // 2), s["factor"], dtype=torch.float64, device="cuda"),
                               p.double()[:, None] * s["inv_freq"].double()[None])
            done = []
            for x, weight in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
                x = x[b, :n].double()
                if weight is not None:
                    x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + 1e-6) * weight.double()
                pairs = x[..., :r].unflatten(-1, (r // 2, 2) if c["interleaved"] else (2, r // 2))
                if not c["interleaved"]:
                    pairs = pairs.transpose(-1, -2)
                z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
                z = z if c["interleaved"] else z.transpose(-1, -2)
                done.append(torch.cat([z.flatten(-2), x[..., r:]], -1))
            q_out[b, :n] = done[0]
            where = s["table"][b].long()[p // page]
            data[0, 0, where, :, p % page] = done[1]
            data[0, 1, where, :, p % page] = s["v"][b, :n].double()
        return {"q": q_out, "data": data}
    table, refs, data = s["table"].tolist(), s["refs"].tolist(), s["data"]
    if c["op"] == "fork":
        B, n = c["batch"], -(-c["past"] // page)
        need = -(-(c["past"] + c["tokens"]) // page)
        for b in range(1, B):
            table[b][:n] = table[0][:n]
            for q in table[0][:n]:
                refs[q] += 1
        shared = c["past"] % page > 0 and B > 1
        for b in range(B):
            for i in range(c["past"] // page, need):
                if i < n and not (shared and b > 0):
                    continue
                new = refs.index(0)
                if i < n:
                    old = table[b][i]
                    refs[old] -= 1
                    data[:, :, new] = data[:, :, old]
                table[b][i], refs[new] = new, 1
        return {"table": torch.tensor(table, dtype=torch.int32, device="cuda"),
                "length": torch.full((B,), c["past"], dtype=torch.long, device="cuda"),
                "refs": torch.tensor(refs, dtype=torch.int32, device="cuda"), "data": data.double()}
    n = sum(x > 0 for x in refs)
    goes = dict(zip([p for p in range(n, len(refs)) if refs[p] > 0], [p for p in range(n) if refs[p] == 0]))
    for old, new in goes.items():
        data[:, :, new] = data[:, :, old]
        refs[new], refs[old] = refs[old], 0
    table = [[goes.get(p, p) for p in row] for row in table]
    return {"table": torch.tensor(table, dtype=torch.int32, device="cuda"),
            "refs": torch.tensor(refs, dtype=torch.int32, device="cuda"), "data": data.double()}
