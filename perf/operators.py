"""Cases of the paged-cache operators: attention over 16-bit paged caches, attention with a sliding window and first
tokens that stay visible, and the upkeep of the pages (copy, fork, free, compact).

``run`` computes them in their plain form, from elementary torch operations in 32 bits, or, where ``own`` is true,
through the framework's entry points; ``exact`` says in 64 bits what comes out.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}


# ----------------------------------------------------------------------------------------------------- the cases


def _attn(name, dtype, batch, q, keys, page, heads, hd, window=-1, sinks=0, spread=0):
    return {"name": name, "kind": "attn", "dtype": dtype, "batch": batch, "qlo": q[0], "qhi": q[1], "lo": keys[0],
            "hi": keys[1], "page": page, "qh": heads[0], "kvh": heads[1], "hd": hd, "window": window, "sinks": sinks,
            "spread": spread}


def listed():
    return [
        # a few short requests of a small model, one new token each: a chat server that is nearly idle (latency)
        _attn("decode16 short", "bf16", 4, (1, 1), (64, 512), 16, (8, 2), 128),
        # a full batch with ragged contexts, one new token each: the steady state of a server with a 16-bit cache
        _attn("decode16 ragged", "bf16", 64, (1, 1), (1024, 8192), 64, (64, 8), 128),
        # half precision, narrow heads, an odd number of them, pages of one token (the serving default)
        _attn("decode16 page1 hd64", "fp16", 48, (1, 1), (17, 4097), 1, (15, 5), 64),
        # speculative verify: five new tokens for each request on an 8k prefix
        _attn("verify16", "bf16", 32, (5, 5), (8192, 8192), 64, (32, 8), 128),
        # endless streams: a window of 4096 keys and the first 4 tokens; the pages between them are gone
        _attn("stream decode bf16", "bf16", 128, (1, 1), (4096, 131072), 64, (64, 8), 128, 4095, 4),
        # the same over the framework's 8-bit cache: wide heads, the 1024-key window of a hybrid model's local layers
        _attn("stream decode e4m3 hd256", "e4m3", 16, (1, 1), (500, 20000), 64, (16, 8), 256, 1024, 4),
        # a chunk of each prompt on top of a cached prefix, windowed layers with wide heads
        _attn("stream extend hd256", "bf16", 8, (2048, 2048), (18432, 18432), 64, (16, 8), 256, 1024, 4),
        # ragged prompts in half precision from an empty cache, odd lengths, window and sinks
        _attn("stream prompts hd128", "fp16", 5, (33, 4099), (33, 4099), 16, (32, 8), 128, 1500, 5),
        # one request of a small model forked into four samples (latency)
        {"name": "fork small", "kind": "fork", "layers": 2, "page": 16, "kvh": 2, "hd": 128, "parents": 1, "ways": 4,
         "lo": 300, "hi": 300, "spare": 40, "spread": 1},
        # beam search over a batch: every parent into four, eight layers
        {"name": "fork batch", "kind": "fork", "layers": 8, "page": 64, "kvh": 8, "hd": 128, "parents": 24, "ways": 4,
         "lo": 500, "hi": 3000, "spare": 32, "spread": 2},
        # requests of a batch end and others take their pages: free, close the gaps, grow, drop what left the window
        {"name": "churn", "kind": "churn", "layers": 4, "page": 64, "kvh": 8, "hd": 128, "rows": 64, "lo": 64,
         "hi": 2048, "window": 1024, "sinks": 4, "spread": 3},
        # pages moved within every layer's pool: swapping in a prefix, moving requests between two halves of a pool
        {"name": "copy pages", "kind": "copy", "layers": 8, "page": 64, "kvh": 8, "hd": 128, "pages": 640, "n": 250,
         "spread": 4},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["decode", "decode", "verify", "stream", "stream", "extend", "fork", "churn", "copy"])
    spread = rng.randrange(1 << 20)
    page = rng.choice([1, 8, 16, 32, 64, 128])
    if kind in ("fork", "churn", "copy"):
        c = {"layers": rng.randint(1, 8), "page": max(page, 8), "kvh": rng.choice([1, 2, 5, 8]), "hd": rng.choice([64, 128, 256]),
             "spread": spread}
        if kind == "fork":
            lo = _log(rng, 1, 2000)
            return {"kind": "fork", **c, "parents": _log(rng, 1, 32), "ways": rng.randint(1, 6), "lo": lo,
                    "hi": lo + rng.randint(0, 1000), "spare": rng.randint(1, 64)}
        if kind == "churn":
            return {"kind": "churn", **c, "rows": _log(rng, 2, 80), "lo": rng.randint(1, 200), "hi": _log(rng, 200, 2048),
                    "window": rng.randint(1, 1500), "sinks": rng.randint(0, 70)}
        n = _log(rng, 1, 250)
        return {"kind": "copy", **c, "pages": 2 * n + rng.randint(1, 60), "n": n}
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    hd = rng.choice([64, 128, 128, 256])
    kvh = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
    gqa = rng.choice([1, 2, 3, 4, 6, 8, 8, 16])
    heads = (kvh * gqa, kvh)
    batch = _log(rng, 1, 96)
    window, sinks = -1, 0
    if kind == "decode":
        q, keys = (1, 1), (rng.randint(0, 600), _log(rng, 600, 8192))
    elif kind == "verify":
        t = rng.randint(2, 16)
        q, keys = (1, t), (rng.randint(16, 600), _log(rng, 600, 8192))
    elif kind == "stream":
        dtype = rng.choice(["bf16", "fp16", "e4m3"])
        t = rng.choice([1, 1, 1, rng.randint(2, 8)])
        q, keys = (1, t), (rng.randint(0, 600), _log(rng, 600, 131072))
        window, sinks = _log(rng, 1, 4096), _log(rng, 1, 129) - 1
    else:
        batch = min(batch, 8)
        t = _log(rng, 17, 4096)
        q, keys = (max(1, t // 3), t), (t, t + rng.choice([0, rng.randint(1, 4000)]))
        window, sinks = rng.choice([(-1, 0), (_log(rng, 1, 3000), _log(rng, 1, 129) - 1)])
    return {k: v for k, v in _attn("", dtype, batch, q, keys, page, heads, hd, window, sinks, spread).items() if k != "name"}


def draw(rng):
    most = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]
    while True:
        c = _draw(rng)
        w = work(c)
        if c["kind"] == "attn":
            _, ql, _ = _lens(c)
            room = c["batch"] * c["qh"] * max(ql) * _width(c)[1] * 4  # bytes of the plain form's scores
            gathered = c["batch"] * _width(c)[1] * c["kvh"] * c["hd"] * 4
        else:
            room = gathered = 0
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and room <= 9e9 and gathered <= 5e9:
            return c


# ------------------------------------------------------------------------------------------------- sizes of a case


def _lens(c):
    """Keys and new tokens of each request, and the first position each still needs besides the sinks."""
    r = random.Random(c["spread"])
    keys = [r.randint(c["lo"], c["hi"]) for _ in range(c["batch"])]
    ql = [r.randint(c["qlo"], c["qhi"]) for _ in keys]
    if c["qhi"] > 16:  # prompts: no more new tokens than keys
        ql = [min(a, b) for a, b in zip(ql, keys)]
    first = [max(0, k - n - c["window"]) if c["window"] >= 0 else 0 for k, n in zip(keys, ql)]
    return keys, ql, first


def _width(c):
    """(sinks, sinks and the longest run of other keys that a request's queries see)."""
    keys, _, first = _lens(c)
    s = c["sinks"] if c["window"] >= 0 else 0
    return s, s + max(1, max(max(0, k - max(f, s)) for k, f in zip(keys, first)))


def _seen(c):
    """Keys that each query sees, summed over queries, and distinct keys that some query sees, over requests."""
    pairs = distinct = 0
    w, s = c["window"], c["sinks"]
    for k, n, f in zip(*_lens(c)):
        if w < 0:
            lo, hi = max(0, k - n), k  # positions of the queries that see anything: p + 1 keys each
            pairs += (hi * (hi + 1) - lo * (lo + 1)) // 2
        else:
            for p in range(max(0, k - n), k):
                a = max(0, p - w)
                pairs += p + 1 - a + min(s, a)
        distinct += k - f + min(s, f) if w >= 0 else k
    return pairs, distinct


def _row_lens(c):
    r = random.Random(c["spread"])
    n = c["parents"] if c["kind"] == "fork" else c["rows"]
    return [r.randint(c["lo"], c["hi"]) for _ in range(n)]


def _pages_of(n, page):
    return -(-n // page)


def work(case):
    c = case
    if c["kind"] == "attn":
        pairs, distinct = _seen(c)
        tokens = sum(_lens(c)[1])
        el = 1 if c["dtype"] == "e4m3" else 2
        q = tokens * c["qh"] * c["hd"]
        return {"bytes": 2 * distinct * c["kvh"] * c["hd"] * el + q * (el + 2) + tokens * c["qh"] * 4,
                "flops": 4 * pairs * c["qh"] * c["hd"]}
    tok = c["kvh"] * c["hd"] * 2 * 2 * c["layers"]  # bytes of one token in every pool
    if c["kind"] == "copy":
        return {"bytes": 2 * c["n"] * c["page"] * tok, "flops": 0}
    if c["kind"] == "fork":
        lens = _row_lens(c)
        tails = sum(n % c["page"] for n in lens)
        entries = sum(_pages_of(n, c["page"]) for n in lens) * c["ways"]
        return {"bytes": tails * tok * (1 + c["ways"]) + 16 * entries, "flops": 0}
    moved, entries = _churn(c)
    return {"bytes": 2 * moved * c["page"] * tok + 16 * entries, "flops": 0}


def _churn(c):
    """Pages that the closing of gaps moves in a first pass, and table entries that the pass touches."""
    lens, page = _row_lens(c), c["page"]
    rows = []
    top = 0
    for n in lens:
        rows.append(list(range(top, top + _pages_of(n, page))))
        top += len(rows[-1])
    live = set(range(top))
    moved = entries = 0
    for half in (0, 1):
        mine = [i for i in range(len(lens)) if i % 2 == half]
        for i in mine:
            live -= set(rows[i])
            entries += len(rows[i])
            rows[i] = []
        low = len(live)
        to = dict(zip(sorted(p for p in live if p >= low), (p for p in range(low) if p not in live)))
        moved += len(to)
        rows = [[to.get(p, p) if p >= 0 else p for p in r] for r in rows]
        entries += sum(len(r) for r in rows)
        live = set(range(low))
        at = low
        for i in mine:
            n = _pages_of(lens[i], page)
            rows[i] = list(range(at, at + n))
            at += n
            gone = range(_pages_of(c["sinks"], page), max(0, lens[i] - c["window"]) // page)
            for j in gone:
                rows[i][j] = -1
            live |= {p for p in rows[i] if p >= 0}
            entries += n
    return moved, entries


# --------------------------------------------------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _normal(shape, std, g, dtype):
    """Normal values in chunks, so that a large pool needs no copy of itself in 32 bits."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    for part in out.flatten().split(1 << 28):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * std)
    return out


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] != "attn":
        return _prepare_pages(c, g)
    keys, ql, first = _lens(c)
    page, dt = c["page"], DTYPES[c["dtype"]]
    cols = _pages_of(max(keys), page) + 1
    table = torch.full((c["batch"], cols), -1, dtype=torch.int64)
    sink_pages = _pages_of(c["sinks"], page)
    where = []
    for b, (n, f) in enumerate(zip(keys, first)):
        held = torch.arange(_pages_of(n, page))
        if c["window"] >= 0:  # the pages between the sinks and the window have been released
            held = held[(held < sink_pages) | (held >= f // page)]
        where.append(torch.stack([torch.full_like(held, b), held]))
    b, col = torch.cat(where, 1)
    pages = b.numel() + 3
    table[b, col] = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[: b.numel()]
    shape = (pages, page, c["kvh"], c["hd"])
    std = 0.5 if c["dtype"] == "e4m3" else 1.0
    call = {
        "q": _normal((sum(ql), c["qh"], c["hd"]), 1.0, g, dt), "k_cache": _normal(shape, std, g, dt),
        "v_cache": _normal(shape, std, g, dt), "page_table": table.to(torch.int32).cuda(),
        "cache_seqlens": _ints(keys), "cu_seqlens_q": torch.cat([_ints([0]), _ints(ql).cumsum(0).to(torch.int32)]),
        "max_seqlen_q": max(ql), "softmax_scale": c["hd"] ** -0.5, "causal": True, "return_softmax_lse": True,
    }
    if c["window"] >= 0:
        call["window_size"], call["sink_tokens"] = (c["window"], 0), c["sinks"]
    if c["dtype"] == "e4m3":
        for name in ("k_descale", "v_descale"):
            call[name] = torch.rand((c["batch"], c["kvh"]), generator=g, device="cuda") * 1.5 + 0.5
    return {"case": c, "call": call}


def _prepare_pages(c, g):
    r = random.Random(c["spread"])
    page = c["page"]
    if c["kind"] == "copy":
        total = c["pages"]
        ids = r.sample(range(total), 2 * c["n"])
        s = {"src": _ints(ids[: c["n"]]), "dst": _ints(ids[c["n"]:])}
        table, lens, refs = _ints([[-1]]), _ints([0]), _ints([1] * total)
    else:
        lens = _row_lens(c)
        held = [_pages_of(n, page) for n in lens]
        if c["kind"] == "fork":
            n = c["parents"]
            total = sum(held) + n * c["ways"] + c["spare"]
            ids = r.sample(range(total), sum(held))  # scattered, as after a while of serving
            rows = n * (1 + c["ways"])
            s = {"parents": _ints([i for i in range(n) for _ in range(c["ways"])]), "children": _ints(list(range(n, rows)))}
        else:
            total = sum(held) + 5
            ids = list(range(sum(held)))
            rows = c["rows"]
            s = {"halves": [(_ints(list(range(h, rows, 2))), _ints(lens[h::2])) for h in (0, 1) if h < rows]}
        at, own_rows = 0, []
        for h in held:
            own_rows.append(ids[at:at + h])
            at += h
        cols = max(held) + 2
        table = _ints([p + [-1] * (cols - len(p)) for p in own_rows] + [[-1] * cols] * (rows - len(lens)))
        lens = _ints(lens + [0] * (rows - len(lens)))
        refs = torch.zeros(total, dtype=torch.int32, device="cuda")
        refs[torch.tensor(ids, device="cuda")] = 1
    pool = _normal((c["layers"], 2, total, page, c["kvh"], c["hd"]), 1.0, g, torch.bfloat16)
    s |= {"case": c, "pool": pool, "table": table, "lens": lens, "refs": refs}
    if own:
        from greenattention_b200 import kv_pages

        s["handle"] = kv_pages.PagePool([t for layer in pool for t in layer], table, lens, refs)
    return s


# ------------------------------------------------------------------------------------------------------ one pass


def run(state):
    c = state["case"]
    if c["kind"] == "attn":
        if own:
            from greenattention_b200 import attn_paged

            out, lse = attn_paged.attend(**state["call"])
        else:
            out, lse = _plain_attend(c, state["call"])
        return {"out": out, "lse": lse}
    h = state["handle"] if own else _PlainPages(state["pool"], state["table"], state["lens"], state["refs"])
    if c["kind"] == "copy":
        h.copy(state["src"], state["dst"])
        return {"pool": state["pool"]}
    if c["kind"] == "fork":  # the branches of the step before end, and each parent branches again
        h.free(state["children"])
        h.fork(state["parents"], state["children"])
    else:
        for rows, lens in state["halves"]:
            h.free(rows)
            h.compact()
            h.grow(rows, lens)
            h.evict(rows, window_left=c["window"], sink_tokens=c["sinks"])
    return {"pool": state["pool"], "table": state["table"], "lens": state["lens"], "refs": state["refs"]}


def _plain_attend(c, a):
    q, kc, vc, table = a["q"], a["k_cache"], a["v_cache"], a["page_table"]
    page, kvh, hd, w = c["page"], c["kvh"], c["hd"], c["window"]
    keys, cu = a["cache_seqlens"].long(), a["cu_seqlens_q"].long()
    dev, batch, most_q = q.device, keys.numel(), a["max_seqlen_q"]
    ql = cu[1:] - cu[:-1]
    sinks, width = _width(c)
    # positions whose keys some query of the request sees: the sinks, then one run that ends with the last key
    first = (keys - ql - w).clamp(min=0) if w >= 0 else torch.zeros_like(keys)
    pos = first.clamp(min=sinks)[:, None] + torch.arange(width - sinks, device=dev)
    pos = torch.cat([torch.arange(sinks, device=dev).expand(batch, sinks), pos], 1)
    there = pos < keys[:, None]
    at = table.gather(1, (pos // page).clamp(max=table.shape[1] - 1)).long().clamp(min=0) * page + pos % page

    def rows(cache):
        flat = cache.view(-1, kvh, hd)
        if c["dtype"] == "e4m3":
            return flat.view(torch.uint8)[at].view(cache.dtype).float()
        return flat[at].float()

    t = torch.arange(most_q, device=dev)
    qat = (cu[:-1, None] + t).clamp(max=q.shape[0] - 1)
    qf = q.float()[qat].view(batch, most_q, kvh, -1, hd)
    s = torch.einsum("bqhgd,bkhd->bhgqk", qf, rows(kc)) * a["softmax_scale"]
    if "k_descale" in a:
        s = s * a["k_descale"][:, :, None, None, None]
    qpos = (keys - ql)[:, None] + t
    sees = there[:, None] & (pos[:, None] <= qpos[:, :, None])
    if w >= 0:
        sees &= (pos[:, None] >= qpos[:, :, None] - w) | (pos[:, None] < sinks)
    s = s.masked_fill_(~sees[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = s.sub_(m).exp_()
    total = e.sum(-1, keepdim=True)
    o = torch.einsum("bhgqk,bkhd->bhgqd", e, rows(vc)) / total
    o = torch.where(total > 0, o, 0.0)
    if "v_descale" in a:
        o = o * a["v_descale"][:, :, None, None, None]
    lse = (m + total.log())[..., 0]
    b_of = torch.repeat_interleave(torch.arange(batch, device=dev), ql, output_size=q.shape[0])
    t_of = torch.arange(q.shape[0], device=dev) - cu[b_of]
    o = o.permute(0, 3, 1, 2, 4)[b_of, t_of].reshape(q.shape[0], -1, hd)
    lse = lse.permute(0, 3, 1, 2)[b_of, t_of].reshape(q.shape[0], -1)
    return o.to(torch.bfloat16 if c["dtype"] == "e4m3" else q.dtype), lse.T.contiguous()


class _PlainPages:
    """The pages' upkeep in elementary operations. ``pool`` holds every layer's K and V; a page is free while no
    table entry holds it (its count in ``refs`` is 0), and new pages are the lowest free ones, in the rows' order."""

    def __init__(self, pool, table, lens, refs):
        self.pool, self.table, self.lens, self.refs, self.page = pool, table, lens, refs, pool.shape[3]

    def copy(self, src, dst):
        self.pool[:, :, dst.long()] = self.pool[:, :, src.long()]

    def _held(self, rows):
        cols = torch.arange(self.table.shape[1], device=rows.device)
        n = (self.lens[rows] + self.page - 1) // self.page
        return cols, cols < n[:, None]

    def _drop(self, rows, gone):
        old = self.table[rows]
        gone = gone & (old >= 0)
        self.refs.index_add_(0, old.clamp(min=0).flatten(), -gone.flatten().to(torch.int32))
        self.table[rows] = torch.where(gone, -1, old)

    def free(self, rows):
        rows = rows.long()
        self._drop(rows, self._held(rows)[1])
        self.lens[rows] = 0

    def evict(self, rows, window_left, sink_tokens):
        rows = rows.long()
        cols, held = self._held(rows)
        last = (self.lens[rows] - window_left).clamp(min=0) // self.page
        self._drop(rows, held & (cols >= -(-sink_tokens // self.page)) & (cols < last[:, None]))

    def _free_ids(self):
        return torch.argsort((self.refs > 0).to(torch.int8), stable=True)

    def grow(self, rows, lens):
        rows = rows.long()
        cols, held = self._held(rows)
        new = (cols < ((lens + self.page - 1) // self.page)[:, None]) & ~held
        rank = new.flatten().cumsum(0).view(new.shape) - 1
        ids = self._free_ids()[rank.clamp(min=0)].to(torch.int32)
        self.table[rows] = torch.where(new, ids, self.table[rows])
        self.refs.index_add_(0, ids.flatten(), new.flatten().to(torch.int32))
        self.lens[rows] = lens

    def fork(self, parents, children):
        parents, children = parents.long(), children.long()
        cols, held = self._held(parents)
        lens = self.lens[parents]
        tail = lens % self.page
        shared = cols < (lens // self.page)[:, None]
        old = self.table[parents]
        last = ((lens - 1) // self.page).clamp(min=0).long()
        src = old.gather(1, last[:, None])[:, 0].long()
        new = self._free_ids()[((tail > 0).cumsum(0) - 1).clamp(min=0)]
        keep = torch.arange(self.page, device=src.device) < tail[:, None]
        to = torch.where(tail > 0, new, src)  # a length that ends with its page needs no copy: onto itself
        self.pool[:, :, to] = torch.where(keep[None, None, :, :, None, None], self.pool[:, :, src], self.pool[:, :, to])
        mine = self.table[children]
        mine = torch.where(shared, old, mine)
        self.table[children] = torch.where(held & ~shared, new[:, None].to(torch.int32), mine)
        self.refs.index_add_(0, old.clamp(min=0).flatten(), (shared & (old >= 0)).flatten().to(torch.int32))
        self.refs.index_add_(0, new, (tail > 0).to(torch.int32))
        self.lens[children] = lens

    def compact(self):
        live = self.refs > 0
        low = live.sum()
        ids = torch.arange(live.numel(), device=live.device)
        src = (live & (ids >= low)).nonzero()[:, 0]
        dst = (~live & (ids < low)).nonzero()[:, 0]
        self.pool[:, :, dst] = self.pool[:, :, src]
        to = torch.where(live, ids, -1)
        to[src] = dst
        rows = torch.arange(self.table.shape[0], device=ids.device)
        held = self._held(rows)[1] & (self.table >= 0)
        self.table.copy_(torch.where(held, to[self.table.clamp(min=0).long()].to(torch.int32), self.table))
        counts = self.refs[src]
        self.refs[src] = 0
        self.refs[dst] = counts


# ------------------------------------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    global own
    c, was = case, own
    own = False
    s = prepare(c, seed)
    own = was
    return _exact_attend(c, s["call"]) if c["kind"] == "attn" else _exact_pages(c, s)


def _exact_attend(c, a):
    """Request by request and in blocks of queries: softmax(q k^T scale + mask) v from the definition."""
    hd, kvh, gqa, page = c["hd"], c["kvh"], c["qh"] // c["kvh"], c["page"]
    out = torch.zeros(a["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full((c["qh"], out.shape[0]), -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    raw = {n: (a[n].view(torch.uint8) if c["dtype"] == "e4m3" else a[n]) for n in ("k_cache", "v_cache")}
    for b, (n, new) in enumerate(zip(*_lens(c)[:2])):
        for q0 in range(0, new, 512):
            q1 = min(new, q0 + 512)
            p = torch.arange(n - new + q0, n - new + q1, device="cuda")
            lo = max(0, n - new + q0 - c["window"]) if c["window"] >= 0 else 0
            hi = n - new + q1
            pos = torch.cat([torch.arange(min(lo, c["sinks"]), device="cuda"), torch.arange(lo, max(lo, hi), device="cuda")])
            pos = pos[pos < max(0, hi)]
            if pos.numel() == 0:
                continue
            ids = a["page_table"][b, pos // page].long()
            k, v = (raw[x][ids, pos % page].view(a[x].dtype).double().transpose(0, 1) for x in ("k_cache", "v_cache"))
            q = a["q"][at + q0:at + q1].double().view(q1 - q0, kvh, gqa, hd).permute(1, 2, 0, 3).reshape(kvh, -1, hd)
            s = (q @ k.transpose(1, 2)).view(kvh, gqa, q1 - q0, -1) * a["softmax_scale"]
            if "k_descale" in a:
                s = s * a["k_descale"][b].double()[:, None, None, None]
            hidden = pos > p[:, None]
            if c["window"] >= 0:
                hidden |= (pos < p[:, None] - c["window"]) & (pos >= c["sinks"])
            s[:, :, hidden] = -math.inf
            z = torch.logsumexp(s, -1)
            w = torch.exp(s - torch.where(z == -math.inf, 0.0, z)[..., None]).view(kvh, -1, pos.numel())
            o = (w @ v).view(kvh, gqa, q1 - q0, hd)
            if "v_descale" in a:
                o = o * a["v_descale"][b].double()[:, None, None, None]
            out[at + q0:at + q1] = o.permute(2, 0, 1, 3).reshape(q1 - q0, -1, hd)
            lse[:, at + q0:at + q1] = z.reshape(-1, q1 - q0)
        at += new
    return {"out": out, "lse": lse}


def _exact_pages(c, s):
    """The pages' books kept with lists, and every page or part of a page copied for itself, in the books' order."""
    pool, page = s["pool"], c["page"]

    def move(dst, src, tokens=page):
        pool[:, :, dst, :tokens] = pool[:, :, src, :tokens]

    if c["kind"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            move(b, a)
        return {"pool": pool}
    table, lens, refs = s["table"].tolist(), s["lens"].tolist(), s["refs"].tolist()

    def release(row, cols):
        for j in cols:
            if table[row][j] >= 0:
                refs[table[row][j]] -= 1
                table[row][j] = -1

    def free(row):
        release(row, range(_pages_of(lens[row], page)))
        lens[row] = 0

    if c["kind"] == "fork":
        spare = [i for i, n in enumerate(refs) if n == 0]
        for a, b in zip(s["parents"].tolist(), s["children"].tolist()):
            for j in range(lens[a] // page):
                table[b][j] = table[a][j]
                refs[table[a][j]] += 1
            if lens[a] % page:
                j, new = lens[a] // page, spare.pop(0)
                move(new, table[a][j], lens[a] % page)
                table[b][j], refs[new] = new, 1
            lens[b] = lens[a]
    else:
        for rows, to in s["halves"]:
            rows, to = rows.tolist(), to.tolist()
            for r in rows:
                free(r)
            live = sum(n > 0 for n in refs)
            gaps = [i for i in range(live) if refs[i] == 0]
            moved = {}
            for i in [i for i in range(live, len(refs)) if refs[i] > 0]:
                moved[i] = gaps.pop(0)
                move(moved[i], i)
                refs[moved[i]], refs[i] = refs[i], 0
            for r, n in enumerate(lens):
                for j in range(_pages_of(n, page)):
                    table[r][j] = moved.get(table[r][j], table[r][j])
            for r, n in zip(rows, to):
                for j in range(_pages_of(n, page)):
                    table[r][j] = refs.index(0)
                    refs[table[r][j]] = 1
                lens[r] = n
            for r, n in zip(rows, to):
                release(r, range(_pages_of(c["sinks"], page), max(0, n - c["window"]) // page))
    return {"pool": pool, "table": _ints(table), "lens": _ints(lens), "refs": _ints(refs)}
