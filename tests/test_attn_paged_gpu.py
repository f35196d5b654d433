"""Attention over 16-bit and e4m3 paged caches with a window and first tokens, against the 64-bit definition. The bounds
are the oracle's (``oracle/paged_oracle.attend``): roundings counted by half steps, the 32-bit sums by their lengths."""

import pytest
import torch

from oracle import paged_oracle

pytestmark = pytest.mark.gpu
BF16, FP16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def make(dtype, lens, new, page, qh, kvh, hd, window=-1, sinks=0, seed=0, q_dtype=None, descale=False, stacked=False,
         heads_first=False, q_wide=False, scale=None):
    """A call over a shuffled pool. Pages without a visible key are not in the table (-1), what no query may see is NaN."""
    g = torch.Generator().manual_seed(seed)
    cols = max(1, max(-(-n // page) for n in lens)) + 2
    table = torch.full((len(lens), cols), -1, dtype=torch.int64)
    seen, b_of = [], []
    for b, (n, t) in enumerate(zip(lens, new)):
        lo = max(0, n - t - window) if window >= 0 else 0
        vis = [j for j in range(n) if j >= lo or j < sinks] if n - t + t > 0 else []
        held = sorted({j // page for j in vis})
        seen.append(vis)
        b_of += [(b, c) for c in held]
    pages = len(b_of) + 2
    ids = torch.randperm(pages, generator=g)[: len(b_of)]
    for (b, c), i in zip(b_of, ids.tolist()):
        table[b, c] = i
    shape = (pages, kvh, page, hd) if heads_first else (pages, page, kvh, hd)
    if stacked:
        buf = torch.full((pages, 2, *shape[1:]), float("nan"))
        caches = [buf[:, 0], buf[:, 1]]
    else:
        caches = [torch.full(shape, float("nan")) for _ in range(2)]
    views = [c.transpose(1, 2) if heads_first else c for c in caches]
    for b, vis in enumerate(seen):
        if vis:
            at = torch.tensor(vis)
            for c in views:
                c[table[b, at // page], at % page] = torch.randn((len(vis), kvh, hd), generator=g)
    if stacked:
        buf = buf.to(dtype).cuda()
        kc, vc = buf[:, 0], buf[:, 1]
    else:
        kc, vc = (c.to(dtype).cuda() for c in caches)
    if heads_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    total = sum(new)
    q = torch.randn((total, qh, hd), generator=g)
    q = q.to(q_dtype or (BF16 if dtype == FP8 else dtype)).cuda()
    if q_wide:
        wide = torch.zeros((total, qh + 1, hd + 8), dtype=q.dtype, device="cuda")
        wide[:, :qh, :hd] = q
        q = wide[:, :qh, :hd]
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    kw = dict(q=q, k_cache=kc, v_cache=vc, page_table=table.to(torch.int32).cuda(),
              cache_seqlens=torch.tensor(lens, dtype=torch.int32).cuda(), cu_seqlens_q=cu, max_seqlen_q=max(1, max(new)),
              causal=True, return_softmax_lse=True, softmax_scale=scale)
    if window >= 0:
        kw |= dict(window_size=(window, 0), sink_tokens=sinks)
    if descale:
        kw |= {n: (torch.rand((len(lens), kvh), generator=g) + 0.5).cuda() for n in ("k_descale", "v_descale")}
    return kw


def check(kw, got=None):
    from greenattention_b200 import attn_paged

    out, lse = attn_paged.attend(**kw) if got is None else got
    torch.cuda.synchronize()
    want = paged_oracle.attend(kw)
    rows = ~want["out"].isnan()
    off = (out.cpu().double() - want["out"]).abs()
    assert (off <= want["out_tol"])[rows].all(), f"out: {(off / want['out_tol'].clamp(min=1e-30))[rows].max()} of the bound"
    zl, gl = want["lse"], lse.cpu().double()
    fin = zl.isfinite()
    assert torch.equal(gl[zl == -torch.inf], zl[zl == -torch.inf])
    assert ((gl - zl).abs() <= want["lse_tol"])[fin].all()
    assert attn_paged.check_status() == 0
    return out, lse


SHAPES = [(8, 2, 128), (6, 6, 64), (5, 1, 64), (16, 8, 128), (15, 5, 128), (12, 3, 256), (20, 10, 256), (24, 12, 64)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP8])
@pytest.mark.parametrize("qh,kvh,hd", SHAPES)
def test_decode(dtype, qh, kvh, hd):
    check(make(dtype, [1, 137, 64, 300, 0, 33], [1] * 6, 16, qh, kvh, hd, seed=hd + qh, descale=dtype == FP8))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP8])
@pytest.mark.parametrize("page", [1, 2, 8, 64, 256])
def test_page_sizes(dtype, page):
    check(make(dtype, [1, 255, 256, 257, 90], [1] * 5, page, 8, 4, 128, seed=page))


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 1), (1, 0), (15, 4), (16, 16), (63, 5), (100, 33), (100, 129), (64, 0), (5000, 3)])
def test_window_and_first_tokens(dtype, hd, window, sinks):
    check(make(dtype, [1, 5, 129, 400, 97], [1] * 5, 16, 8, 4, hd, window, sinks, seed=window + sinks, descale=dtype == FP8))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP8])
@pytest.mark.parametrize("qh,kvh,hd", [(8, 2, 128), (8, 8, 64), (16, 1, 128), (4, 1, 256), (64, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (40, 3)])
def test_verify(dtype, qh, kvh, hd, window, sinks):
    """Several new tokens, more of them than keys among them (their first rows see nothing), requests without any."""
    check(make(dtype, [200, 3, 64, 31, 9], [5, 5, 1, 0, 16], 16, qh, kvh, hd, window, sinks, seed=qh))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP8])
@pytest.mark.parametrize("qh,kvh,hd,page", [(8, 2, 128, 16), (4, 4, 64, 1), (6, 2, 256, 64), (7, 1, 128, 32), (34, 2, 128, 128)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (50, 7), (0, 2), (200, 0)])
def test_prompts(dtype, qh, kvh, hd, page, window, sinks):
    check(make(dtype, [130, 257, 40, 1, 300], [130, 100, 17, 1, 64], page, qh, kvh, hd, window, sinks, seed=page + qh,
               descale=dtype == FP8))


def test_prompt_with_more_tokens_than_keys():
    check(make(BF16, [20, 0, 70], [40, 33, 70], 16, 8, 2, 128, seed=5))


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("new", [1, 5, 40])
def test_layouts(dtype, new):
    """Interleaved K / V, head-major pages, strided queries and outputs, an e4m3 query, a scalar descale."""
    base = dict(page=16, qh=8, kvh=2, hd=128, window=70, sinks=4, seed=new)
    check(make(dtype, [200, 90], [new, new], stacked=True, **base))
    check(make(dtype, [200, 90], [new, new], heads_first=True, **base))
    kw = make(dtype, [200, 90], [new, new], q_wide=True, **base)
    wide = torch.full((2 * new + 3, 8, 136), float("nan"), dtype=BF16, device="cuda")
    kw["out"] = wide[: 2 * new, :, :128]
    check(kw)
    assert wide[:, :, 128:].isnan().all() and wide[2 * new:].isnan().all()
    if dtype == FP8:
        kw = make(dtype, [200, 90], [new, new], q_dtype=FP8, **base)
        kw |= dict(k_descale=torch.tensor([0.4], device="cuda").expand(2, 2), v_descale=torch.full((1, 2), 1.7, device="cuda"))
        check(kw)


@pytest.mark.parametrize("new", [1, 4, 50])
def test_rows_behind_the_last_request_stay(new):
    kw = make(BF16, [60, 99], [new, new], 16, 8, 2, 128, seed=3)
    q = torch.cat([kw["q"], torch.full_like(kw["q"][:3], float("nan"))])
    out = torch.full_like(q, 7.0)
    kw |= dict(q=q, out=out)
    from greenattention_b200 import attn_paged

    got, lse = attn_paged.attend(**kw)
    assert got is out and (out[2 * new:] == 7).all()
    kw2 = dict(kw, q=q[: 2 * new], out=None)
    check(kw2, (out[: 2 * new], lse[:, : 2 * new]))


@pytest.mark.parametrize("batch,n", [(1, 20000), (300, 40), (3, 3000)])
@pytest.mark.parametrize("kvh", [1, 8])
def test_splits(batch, n, kvh):
    """One long sequence over all SMs, and more requests than SMs; the split must not change what comes out."""
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(n // 2, n + 1, (batch,), generator=g).tolist()
    kw = make(BF16, lens, [1] * batch, 64, 2 * kvh, kvh, 64, seed=n)
    from greenattention_b200 import attn_paged

    a, la = attn_paged.attend(**kw)
    b, lb = attn_paged.attend(**kw)
    assert torch.equal(a, b) and torch.equal(la, lb)
    few = list(range(0, batch, max(1, batch // 3)))[:3]
    sub = dict(kw, q=kw["q"][few], page_table=kw["page_table"][few], cache_seqlens=kw["cache_seqlens"][few],
               cu_seqlens_q=torch.arange(len(few) + 1, dtype=torch.int32, device="cuda"))
    want = paged_oracle_fast(sub)
    assert ((a[few].double() - want).abs() <= 2.0**-7 * want.abs() + 2.0**-8 * 4).all()


def paged_oracle_fast(kw):
    """One new token, no window: the definition on the GPU in 64 bits."""
    page, kvh, hd = kw["k_cache"].shape[1:]
    out = torch.empty(kw["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(kw["cache_seqlens"].tolist()):
        at = torch.arange(n, device="cuda")
        ids = kw["page_table"][b, at // page].long()
        k, v = (kw[x][ids, at % page].double().transpose(0, 1) for x in ("k_cache", "v_cache"))
        q = kw["q"][b].double().view(kvh, -1, hd)
        out[b] = (torch.softmax(q @ k.transpose(1, 2) * hd**-0.5, -1) @ v).reshape(-1, hd)
    return out


def test_offsets_beyond_32_bits():
    """The call's pages lie behind 2^32 elements of the pool."""
    page, kvh, hd = 64, 8, 128
    pages = (1 << 32) // (page * kvh * hd) + 3
    kw = make(BF16, [150, 70], [1, 1], page, 16, kvh, hd, seed=2)
    for n in ("k_cache", "v_cache"):
        big = torch.empty((pages, page, kvh, hd), dtype=BF16, device="cuda")
        small = kw[n]
        big[-small.shape[0]:] = small
        kw["big_" + n] = big
    shift = pages - kw["k_cache"].shape[0]
    from greenattention_b200 import attn_paged

    moved = {k: v for k, v in kw.items() if not k.startswith("big_")}
    want = attn_paged.attend(**moved)
    moved |= dict(k_cache=kw["big_k_cache"], v_cache=kw["big_v_cache"],
                  page_table=torch.where(kw["page_table"] >= 0, kw["page_table"] + shift, kw["page_table"]))
    got = attn_paged.attend(**moved)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_non_finite_values_count_where_they_are_seen():
    kw = make(BF16, [50, 50, 50], [1, 1, 1], 16, 4, 2, 64, seed=8)
    pt = kw["page_table"].tolist()
    kw["v_cache"][pt[0][1], 3, 0, 5] = float("inf")
    kw["k_cache"][pt[1][1], 3, 1, 0] = float("nan")
    from greenattention_b200 import attn_paged

    out, lse = attn_paged.attend(**kw)
    out = out.view(3, 2, 2, 64)
    assert (out[0, 0, :, 5] == float("inf")).all() and out[0, 0, :, :5].isfinite().all() and out[0, 1].isfinite().all()
    assert out[1, 1].isnan().all() and lse[2:, 1].isnan().all() and out[1, 0].isfinite().all()
    assert out[2].isfinite().all()


@pytest.mark.parametrize("new", [1, 40])
def test_bad_pages_and_lengths_are_flagged(new):
    from greenattention_b200 import attn_paged

    kw = make(BF16, [100, 100], [new, new], 16, 4, 2, 64, seed=9)
    good = attn_paged.attend(**kw)[0]
    bad = dict(kw, page_table=kw["page_table"].clone())
    bad["page_table"][0, 2] = kw["k_cache"].shape[0]
    out, _ = attn_paged.attend(**bad)
    assert attn_paged.check_status() == 3 and attn_paged.check_status() == 0
    assert out[:new].isfinite().all() and torch.equal(out[new:], good[new:])
    long = dict(kw, cache_seqlens=torch.tensor([100, 1 << 20], dtype=torch.int32, device="cuda"))
    out, _ = attn_paged.attend(**long)
    assert attn_paged.check_status() != 0
    assert torch.equal(out[:new], good[:new])


@pytest.mark.parametrize("new", [1, 33])
def test_graph_replays_with_live_lengths(new):
    """Two captured graphs and eager calls in turn, lengths and table changed between replays."""
    from greenattention_b200 import attn_paged

    attn_paged.ensure_ready()
    kws = [make(BF16, [200, 130], [new, new], 16, 8, 2, 128, 90, 4, seed=s) for s in (1, 2)]
    outs, graphs = [], []
    for kw in kws:
        out = torch.empty_like(kw["q"])
        outs.append(out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            attn_paged.attend(**dict(kw, out=out))
        graphs.append(g)
    for step in range(2):
        want = [attn_paged.attend(**kw)[0] for kw in kws]
        for o in outs:
            o.fill_(3)
        streams = [torch.cuda.Stream() for _ in graphs]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        # bit by bit: with the shorter lengths the window reaches back to keys that the inputs hold as NaN
        for w, o in zip(want, outs):
            assert torch.equal(w.view(torch.int16), o.view(torch.int16))
        assert want[0].isfinite().all() == (step == 0)
        for kw in kws:
            kw["cache_seqlens"].copy_(torch.tensor([190, 125], dtype=torch.int32))


def test_calls_on_two_streams():
    from greenattention_b200 import attn_paged

    kws = [make(FP16, [3000, 500], [1, 1], 16, 8, 2, 128, seed=s) for s in (1, 2)]
    want = [attn_paged.attend(**kw) for kw in kws]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in kws]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(attn_paged.attend(**kws[i])[0])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w[0], x) for x in g)


def test_through_the_backend_entry(monkeypatch):
    """``with_kvcache``: calls with first tokens are served, 16-bit caches without them when the server asked."""
    import importlib

    from greenattention_b200 import attn_decode, attn_paged, dispatch

    attn_decode.ensure_ready()
    attn_paged.ensure_ready()
    importlib.reload(attn_paged)
    attn_paged.ensure_ready()
    entry = dispatch.with_kvcache(lambda **kw: "stock")
    for new in (1, 4, 40):
        kw = make(FP8, [100, 70], [new, new], 16, 8, 2, 128, 30, 4, seed=new)
        check(kw, entry(**kw))
        kw = make(BF16, [100, 70], [new, new], 16, 8, 2, 128, seed=new)
        assert entry(**kw) == "stock"
        monkeypatch.setattr(dispatch, "KV16", True)
        check(kw, entry(**kw))
        assert entry(**dict(kw, softcap=30.0)) == "stock"
        monkeypatch.setattr(dispatch, "KV16", False)
    with pytest.raises(dispatch.Declined, match="softcap"):
        entry(**dict(make(BF16, [9], [1], 16, 8, 2, 128, 30, 4), softcap=30.0))


def definition_on_gpu(kw, rows):
    """The definition in 64 bits on the GPU for some rows of a call: out, sum_j p_j |v_j|, lse of those rows, and how far
    32-bit scores may be off (see the oracle)."""
    page, kvh, hd = kw["k_cache"].shape[1:]
    window, sinks = kw.get("window_size", (-1, 0))[0], kw.get("sink_tokens") or 0
    cu, lens = kw["cu_seqlens_q"].tolist(), kw["cache_seqlens"].tolist()
    outs, spreads, lses, offs = [], [], [], []
    fp8 = kw["k_cache"].dtype == FP8
    for row in rows:
        b = max(i for i in range(len(lens)) if cu[i] <= row)
        p = lens[b] - (cu[b + 1] - cu[b]) + row - cu[b]
        at = torch.arange(p + 1, device="cuda")
        if window >= 0:
            at = at[(at >= p - window) | (at < sinks)]
        ids = kw["page_table"][b, at // page].long()
        k, v = (kw[x].view(torch.uint8 if fp8 else torch.int16)[ids, at % page].view(kw[x].dtype).double().transpose(0, 1)
                for x in ("k_cache", "v_cache"))
        q = kw["q"][row].to(FP8 if fp8 else kw["q"].dtype).double().view(kvh, -1, hd)
        kd, vd = (1.0 if kw.get(n) is None else kw[n][b].double()[:, None, None] for n in ("k_descale", "v_descale"))
        s = q @ k.transpose(1, 2) * hd**-0.5 * kd
        w = torch.softmax(s, -1)
        outs.append((w @ v * vd).reshape(-1, hd))
        spreads.append((w @ v.abs() * vd).reshape(-1, hd))
        lses.append(torch.logsumexp(s, -1).reshape(-1))
        offs.append(((q.abs() @ k.abs().transpose(1, 2) * hd**-0.5 * kd).amax() * hd * 2.0**-23 + len(at) * 2.0**-23 + 2.0**-16))
    return torch.stack(outs), torch.stack(spreads), torch.stack(lses, 1), max(float(x) for x in offs)


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("page", [4, 16, 64])
@pytest.mark.parametrize("new,keys", [(700, 3000), (1500, 1500), (5, 6000), (24, 6000)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (700, 40)])
def test_many_tiles_and_items(dtype, hd, page, new, keys, window, sinks):
    """Long enough that every CTA goes through many tiles and several items: rings, buffers and barriers wrap round."""
    from greenattention_b200 import attn_paged

    g = torch.Generator(device="cuda").manual_seed(hd + new)
    qh, kvh, batch = 16, 4, 5
    lens = [keys - 37 * b for b in range(batch)]
    cols = -(-keys // page)
    pool = [torch.randn((batch * cols, page, kvh, hd), generator=g, device="cuda").to(dtype) for _ in range(2)]
    table = torch.randperm(batch * cols, generator=g, device="cuda").view(batch, cols).to(torch.int32)
    news = [min(new, n) for n in lens]
    q = torch.randn((sum(news), qh, hd), generator=g, device="cuda").to(BF16)
    kw = dict(q=q, k_cache=pool[0], v_cache=pool[1], page_table=table, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
              cu_seqlens_q=torch.tensor([0] + news, device="cuda").cumsum(0).to(torch.int32), max_seqlen_q=max(news), causal=True,
              return_softmax_lse=True)
    if window >= 0:
        kw |= dict(window_size=(window, 0), sink_tokens=sinks)
    if dtype == FP8:
        kw |= {n: torch.rand((batch, kvh), generator=g, device="cuda") + 0.5 for n in ("k_descale", "v_descale")}
    out, lse = attn_paged.attend(**kw)
    again, _ = attn_paged.attend(**kw)
    assert attn_paged.check_status() == 0
    assert torch.equal(out, again)
    rows = sorted({0, len(q) - 1, *torch.randint(0, len(q), (20,), generator=torch.Generator().manual_seed(1)).tolist()})
    want, spread, want_lse, off = definition_on_gpu(kw, rows)
    p_step = 2.0**-11 if dtype == FP8 else 2.0**-8
    # the oracle's bound: half a step of the bf16 output, of P, and the scores' part (twice)
    bound = (2.0**-8 * want.abs() + (p_step + 2 * off) * spread) * (1 + 2.0**-6) + 2.0**-25
    assert ((out[rows].double() - want).abs() <= bound).all()
    assert ((lse[:, rows].double() - want_lse).abs() <= off + 2.0**-20 * (1 + want_lse.abs())).all()


@pytest.mark.parametrize("new", [40, 400])
def test_query_offsets_that_do_not_ascend_stay_in_bounds(new):
    """Malformed offsets ask for more rows than there are: nothing is written outside, the rest of the call is served."""
    from greenattention_b200 import attn_paged

    kw = make(BF16, [500, 500, 500], [new, new, new], 16, 8, 2, 64, seed=4)
    kw["cu_seqlens_q"] = torch.tensor([0, 3 * new, 0, 9 * new], dtype=torch.int32, device="cuda")
    guard = torch.full((3 * new + 64, 8, 64), 3.0, dtype=BF16, device="cuda")
    kw["out"] = guard[32:32 + 3 * new]
    attn_paged.attend(**kw)
    torch.cuda.synchronize()
    assert (guard[:32] == 3).all() and (guard[32 + 3 * new:] == 3).all()
    attn_paged.check_status()
    check(make(BF16, [50, 60], [40, 40], 16, 8, 2, 64, seed=6))


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (FP8, 256)])
@pytest.mark.parametrize("new", [1, 20, 200])
def test_lengths_up_to_the_largest(dtype, hd, new):
    """The last keys of a request of 2^30 tokens, and lengths beyond, which a wide table would address: cut to 2^30."""
    from greenattention_b200 import attn_paged

    page, cols, most = 4096, 1 << 20, 1 << 30
    g = torch.Generator(device="cuda").manual_seed(new)
    kc, vc = (torch.randn((2, page, 2, hd), generator=g, device="cuda").to(dtype) for _ in range(2))
    table = torch.full((2, cols), -1, dtype=torch.int32, device="cuda")
    table[0, most // page - 1], table[0, 0], table[1, 0] = 1, 0, 0
    kw = dict(q=torch.randn((2 * new, 4, hd), generator=g, device="cuda").to(BF16), k_cache=kc, v_cache=vc, page_table=table,
              cu_seqlens_q=torch.tensor([0, new, 2 * new], dtype=torch.int32, device="cuda"), max_seqlen_q=new, causal=True,
              window_size=(300, 0), sink_tokens=5, return_softmax_lse=True)
    near = dict(kw, page_table=torch.tensor([[0, 1], [0, -1]], dtype=torch.int32, device="cuda"),
                cache_seqlens=torch.tensor([2 * page, 1000], dtype=torch.int32, device="cuda"))
    want = paged_oracle.attend(near)
    for n in (most, most + 1, (1 << 31) - 1):
        out, lse = attn_paged.attend(**kw, cache_seqlens=torch.tensor([n, 1000], dtype=torch.int32, device="cuda"))
        assert attn_paged.check_status() == (0 if n == most else 5)
        assert ((out.cpu().double() - want["out"]).abs() <= want["out_tol"]).all()
        assert ((lse.cpu().double() - want["lse"]).abs() <= want["lse_tol"]).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP8])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 5, 17, 300])
def test_a_long_flat_tail_under_one_dominant_key(dtype, hd, new):
    """Key 3 scores 18 above all others and its value is 0: what comes out is the tail's share, n e^-18 / (1 + n e^-18), of
    values of 1, each probability of it 2^-26. The bound is the oracle's: half a step of the output and of P (relative), the
    32-bit scores and sums, and 2^-32 a key where fp16 P are subnormal."""
    from greenattention_b200 import attn_paged

    page, kvh, gqa, batch, keys = 64, 2, 4, 3, 20000
    cols = -(-keys // page)
    g = torch.Generator().manual_seed(new)
    table = torch.randperm(batch * cols, generator=g).view(batch, cols).to(torch.int32).cuda()
    kc, vc = (torch.zeros((batch * cols, page, kvh, hd), device="cuda") for _ in range(2))
    vc += 1
    q = torch.zeros((batch * new, kvh * gqa, hd), device="cuda")
    q[..., 7] = 12
    first = table[:, 0].long()
    kc[first, 3, :, 7], vc[first, 3] = 12, 0
    q_type = BF16 if dtype == FP8 else dtype
    kw = dict(q=q.to(q_type), k_cache=kc.to(dtype), v_cache=vc.to(dtype), page_table=table,
              cache_seqlens=torch.full((batch,), keys, dtype=torch.int32, device="cuda"),
              cu_seqlens_q=torch.arange(batch + 1, dtype=torch.int32, device="cuda") * new, max_seqlen_q=new, causal=True,
              return_softmax_lse=True, softmax_scale=0.125)
    out, lse = attn_paged.attend(**kw)
    assert attn_paged.check_status() == 0
    n = (keys - new + torch.arange(new, device="cuda").repeat(batch)).double()
    tail = n * torch.exp(torch.tensor(-18.0, dtype=torch.float64, device="cuda"))
    want = (tail / (1 + tail))[:, None, None].expand(out.shape)
    off = hd * 2.0**-23 * 18 + 18 * 2.0**-22
    p_step, o_step = (2.0**-8 if dtype == BF16 else 2.0**-11), (2.0**-11 if dtype == FP16 else 2.0**-8)
    bound = (o_step + p_step + 2 * off + (keys + 64) * 2.0**-23) * want * (1 + 2.0**-6)
    if dtype != BF16:
        bound = bound + 2.0**-32 * n[:, None, None]
    if dtype == FP16:
        bound = bound + 2.0**-25
    err = (out.double() - want).abs()
    assert (err <= bound).all(), f"{(err / bound).max()} of the bound"
    z = (18 + torch.log1p(tail)).expand(lse.shape)
    assert ((lse.double() - z).abs() <= off + keys * 2.0**-23 + 2.0**-20 * (1 + z)).all()


@pytest.mark.parametrize("qh,new", [(8, 1), (8, 5), (32, 6), (8, 100)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (40, 3)])
def test_descales_of_zero_below_it_and_no_number(qh, new, window, sinks):
    """The same pattern of numbers and NaN whichever kernel the count of rows selects (warp level, slices, prompts)."""
    from greenattention_b200 import attn_paged

    kw = make(FP8, [200, 130, 160], [new] * 3, 16, qh, 2, 128, window, sinks, seed=new, descale=True)
    kw["k_descale"].copy_(torch.tensor([[0.0, -0.7], [float("nan"), -0.0], [1.0, 0.25]]))
    kw["v_descale"].copy_(torch.tensor([[-1.5, 1.0], [1.0, 0.5], [0.0, float("nan")]]))
    out, lse = attn_paged.attend(**kw)
    want = paged_oracle.attend(kw)
    assert torch.equal(out.cpu().isnan(), want["out"].isnan()) and torch.equal(lse.cpu().isnan(), want["lse"].isnan())
    fine, zfine = ~want["out"].isnan(), ~want["lse"].isnan()
    assert ((out.cpu().double() - want["out"]).abs() <= want["out_tol"])[fine].all()
    assert ((lse.cpu().double() - want["lse"]).abs() <= want["lse_tol"])[zfine].all()
    assert attn_paged.check_status() == 0


def narrow(kw):
    """The call with query and output rows at multiples of 4 elements that are not multiples of 8: no 16-byte loads."""
    total, qh, hd = kw["q"].shape
    q = torch.zeros((total, qh, hd + 4), dtype=kw["q"].dtype, device="cuda")
    q[..., :hd] = kw["q"]
    out = torch.full((total, qh, hd + 4), 7.0, dtype=BF16 if kw["k_cache"].dtype == FP8 else kw["k_cache"].dtype, device="cuda")
    return dict(kw, q=q[..., :hd], out=out[..., :hd])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP8])
@pytest.mark.parametrize("qh,kvh,hd,page", [(8, 2, 128, 16), (5, 5, 64, 1), (6, 2, 256, 64)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (50, 7)])
@pytest.mark.parametrize("new", [1, 5, 90])
def test_queries_that_only_allow_loads_of_four_elements(dtype, qh, kvh, hd, page, window, sinks, new):
    kw = narrow(make(dtype, [130, 257, 40, 300], [new, new, 40 if new > 16 else new, 0], page, qh, kvh, hd, window, sinks, seed=hd,
                     descale=dtype == FP8))
    check(kw)
    assert (kw["out"]._base[..., hd:] == 7).all()
    if dtype == FP8:
        q = torch.zeros(kw["q"]._base.shape, dtype=FP8, device="cuda")
        q[..., :hd] = kw["q"].to(FP8)
        check(dict(kw, q=q[..., :hd], out=None))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP8])
@pytest.mark.parametrize("qh,new", [(8, 1), (8, 5), (32, 6), (8, 100)])
@pytest.mark.parametrize("scale", [0.03, 0.5, 0.0, -0.1])
def test_given_scales(dtype, qh, new, scale):
    check(make(dtype, [200, 130, 90], [new, new, min(new, 90)], 16, qh, 2, 128, 60, 4, seed=new, scale=scale, descale=dtype == FP8))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("qh,new", [(8, 1), (8, 5), (32, 6), (8, 100)])
def test_descales_beside_16_bit_caches(dtype, qh, new):
    kw = make(dtype, [200, 130, 90], [new, new, min(new, 90)], 16, qh, 2, 128, 60, 4, seed=new, descale=True)
    kw["k_descale"].copy_(torch.tensor([[0.0, -0.7], [0.4, -0.0], [1.0, 0.25]]))
    kw["v_descale"].copy_(torch.tensor([[-1.5, 1.0], [1.0, 0.5], [0.0, 3.0]]))
    check(kw)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 64])
@pytest.mark.parametrize("new,keys", [(700, 3000), (5, 6000), (24, 6000)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (700, 40)])
def test_many_tiles_and_items_fp16(hd, page, new, keys, window, sinks):
    """As above with queries, keys and values in half precision."""
    from greenattention_b200 import attn_paged

    g = torch.Generator(device="cuda").manual_seed(hd + new)
    qh, kvh, batch = 16, 4, 5
    lens = [keys - 37 * b for b in range(batch)]
    cols = -(-keys // page)
    pool = [torch.randn((batch * cols, page, kvh, hd), generator=g, device="cuda").to(FP16) for _ in range(2)]
    table = torch.randperm(batch * cols, generator=g, device="cuda").view(batch, cols).to(torch.int32)
    q = torch.randn((batch * new, qh, hd), generator=g, device="cuda").to(FP16)
    kw = dict(q=q, k_cache=pool[0], v_cache=pool[1], page_table=table, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
              cu_seqlens_q=torch.arange(batch + 1, dtype=torch.int32, device="cuda") * new, max_seqlen_q=new, causal=True,
              return_softmax_lse=True)
    if window >= 0:
        kw |= dict(window_size=(window, 0), sink_tokens=sinks)
    out, lse = attn_paged.attend(**kw)
    assert attn_paged.check_status() == 0
    rows = sorted({0, len(q) - 1, *torch.randint(0, len(q), (20,), generator=torch.Generator().manual_seed(1)).tolist()})
    want, spread, want_lse, off = definition_on_gpu(kw, rows)
    seen = keys if window < 0 else window + 1 + sinks
    # the oracle's bound; subnormal P: |v| is below 8, so a key loses at most 2^-32 * 8
    bound = (2.0**-11 * want.abs() + (2.0**-11 + 2 * off) * spread) * (1 + 2.0**-6) + 2.0**-25 + seen * 2.0**-29
    assert ((out[rows].double() - want).abs() <= bound).all()
    assert ((lse[:, rows].double() - want_lse).abs() <= off + 2.0**-20 * (1 + want_lse.abs())).all()


def repeated(dtype, hd, kvh, gqa, lens, new, seed):
    """A call over requests whose page tables go round 8 pages of 128 tokens, values between 0.5 and 1.5."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    page, pages = 128, 8
    kc = (torch.randn((pages, page, kvh, hd), generator=g, device="cuda") * 0.3).to(dtype)
    vc = (torch.rand((pages, page, kvh, hd), generator=g, device="cuda") + 0.5).to(dtype)
    cols = -(-max(lens) // page)
    table = ((torch.arange(cols, device="cuda") + torch.arange(len(lens), device="cuda")[:, None]) % pages).to(torch.int32)
    news = [min(new, n) for n in lens]
    q = torch.randn((sum(news), kvh * gqa, hd), generator=g, device="cuda").to(BF16 if dtype == FP8 else dtype)
    return dict(q=q, k_cache=kc, v_cache=vc, page_table=table, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                cu_seqlens_q=torch.tensor([0] + news, device="cuda").cumsum(0).to(torch.int32), max_seqlen_q=max(news), causal=True,
                return_softmax_lse=True)


def check_repeated(kw, rows, fold=32768):
    """Some rows against the definition in 64 bits, every token of the pool weighed by how often the row sees it. The bound is
    the oracle's, with the 32-bit sums (a product cut to the accumulator's last place, at most 2^-23 of it) over `fold` keys:
    behind so many the sum is put aside. Values are positive, so sum_j p_j |v_j| is the output."""
    from greenattention_b200 import attn_paged

    out, lse = attn_paged.attend(**kw)
    again, _ = attn_paged.attend(**kw)
    assert attn_paged.check_status() == 0 and torch.equal(out, again)
    page, kvh, hd = kw["k_cache"].shape[1:]
    dtype, cu, lens = kw["k_cache"].dtype, kw["cu_seqlens_q"].tolist(), kw["cache_seqlens"].tolist()
    p_step, o_step = (2.0**-8 if dtype == BF16 else 2.0**-11), (2.0**-11 if dtype == FP16 else 2.0**-8)
    k, v = (kw[x].double().flatten(0, 1).transpose(0, 1) for x in ("k_cache", "v_cache"))
    for row in rows:
        b = max(i for i in range(len(lens)) if cu[i] <= row)
        n = lens[b] - (cu[b + 1] - cu[b]) + row - cu[b] + 1
        full = torch.bincount(kw["page_table"][b, : n // page].long(), minlength=len(kw["k_cache"])).repeat_interleave(page)
        if n % page:
            full[kw["page_table"][b, n // page].long() * page:][: n % page] += 1
        q = kw["q"][row].to(dtype).double().view(kvh, -1, hd)
        s = q @ k.transpose(1, 2) * hd**-0.5
        off = hd * 2.0**-23 * float((q.abs() @ k.abs().transpose(1, 2)).amax()) * hd**-0.5 + float(s.abs().amax()) * 2.0**-22
        z = torch.logsumexp(s + full.double().log(), -1)
        want = (torch.exp(s - z[..., None]) * full) @ v
        bound = (o_step + (p_step + 2 * off + (min(n, fold) + 64) * 2.0**-23)) * want * (1 + 2.0**-6)
        err = (out[row].double().view(want.shape) - want).abs()
        assert (err <= bound).all(), f"row {row}, {n} keys: {(err / bound).max()} of the bound"
        zerr = (lse[:, row].double().view(z.shape) - z).abs()
        assert (zerr <= off + (min(n, fold) + 64) * 2.0**-23 + 2.0**-20 * (1 + z)).all()


LONG = [1 << 21, 70000, 33000, 5, 90000, 131072, 32768, 32769, 65537, 200, 40000]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP8])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kvh,gqa,new", [(512, 1, 1), (100, 2, 40), (2, 2, 100)])
def test_sums_over_many_keys(dtype, hd, kvh, gqa, new):
    """Few gangs with long slices (warp level, split prompts' kernel), and prompts: segments end inside requests and with them."""
    kw = repeated(dtype, hd, kvh, gqa, LONG, new, hd + new)
    cu = kw["cu_seqlens_q"].tolist()
    check_repeated(kw, sorted({x for a, b in zip(cu, cu[1:]) for x in (a, b - 1)}))


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_sums_over_many_keys_without_16_byte_queries(dtype, hd):
    kw = narrow(repeated(dtype, hd, 2, 2, [1 << 20, 70000, 90], 50, hd))
    cu = kw["cu_seqlens_q"].tolist()
    check_repeated(kw, sorted({x for a, b in zip(cu, cu[1:]) for x in (a, b - 1)}))


def test_an_item_that_lasts_seconds():
    """A prompt on 2^27 keys (one page, named by every entry) in front of more items than SMs: the queries of the item behind
    it wait that long. Keys are 0 and values 1, so every output is 1 and the LSE is the logarithm of the count."""
    from greenattention_b200 import attn_paged

    page, new, gqa, hd, keys, others = 1024, 20, 8, 64, 1 << 27, 320
    kc = torch.zeros((1, page, 1, hd), dtype=BF16, device="cuda")
    lens = torch.tensor([keys] + [100 + i for i in range(others)], dtype=torch.int32, device="cuda")
    table = torch.zeros((others + 1, keys // page), dtype=torch.int32, device="cuda")
    total = (others + 1) * new
    q = torch.randn((total, gqa, hd), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(BF16)
    out, lse = attn_paged.attend(q=q, k_cache=kc, v_cache=torch.ones_like(kc), page_table=table, cache_seqlens=lens,
                                 cu_seqlens_q=torch.arange(others + 2, dtype=torch.int32, device="cuda") * new, max_seqlen_q=new,
                                 causal=True, return_softmax_lse=True)
    assert attn_paged.check_status() == 0
    seen = (lens[:, None] - new + 1 + torch.arange(new, device="cuda")).flatten().double()
    # sums of at most 32768 equal numbers are exact; each of the folds behind rounds the shares and the LSE a few times
    folds = (seen / 32768).ceil()
    assert ((out.double() - 1).abs() <= (2.0**-8 + folds * 2.0**-22)[:, None, None]).all()
    assert ((lse.double() - seen.log()).abs() <= (2.0**-20 + folds * 2.0**-22) * (1 + seen.log())).all()


def poison(kw, where):
    """Values put into (cache, request, key, head, dim) places."""
    page = kw["k_cache"].shape[1]
    table = kw["page_table"].tolist()
    for cache, b, key, h, d, x in where:
        kw[cache][table[b][key // page], key % page, h, d] = x


def check_with_non_finite(kw):
    from greenattention_b200 import attn_paged

    out, lse = attn_paged.attend(**kw)
    assert attn_paged.check_status() == 0
    want = paged_oracle.attend(kw)
    got, ref = out.cpu().double(), want["out"]
    odd = (got.isnan() != ref.isnan()).nonzero()
    assert len(odd) == 0, f"{odd[:5].tolist()} of {len(odd)}"
    inf = ref.isinf()
    odd = ((got.isinf() != inf) | inf & (got != ref)).nonzero()
    assert len(odd) == 0, f"{odd[:5].tolist()} of {len(odd)}"
    fin = ref.isfinite()
    assert ((got - ref).abs() <= want["out_tol"])[fin].all()
    glse, rlse = lse.cpu().double(), want["lse"]
    assert torch.equal(glse.isnan(), rlse.isnan()) and torch.equal(glse[rlse == -torch.inf], rlse[rlse == -torch.inf])
    fin = rlse.isfinite()
    assert ((glse - rlse).abs() <= want["lse_tol"])[fin].all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP8])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("qh,new", [(8, 2), (8, 16), (40, 6), (8, 90)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (50, 7), (3, 130)])
def test_non_finite_values_that_only_some_rows_see(dtype, hd, qh, new, window, sinks):
    """Infinities and NaN among the new tokens, around the far edge of the first and the last row's window and among the first
    tokens: they reach the rows that see them and no others. The last request has more new tokens than keys."""
    inf, nan = (float("nan") if dtype == FP8 else float("inf")), float("nan")
    lens = [200, 300, 70, new - 1 or 1]
    where = []
    for b, n in enumerate(lens[:3]):
        at = {n - 1: inf, n - new: nan, n - new // 2: -inf, n - new + 1: inf, 2: inf, 5: nan}
        if window >= 0:
            at |= {max(0, n - new - window): -inf, max(0, n - new - window + 1): nan, max(0, n - 1 - window): inf, max(0, n - 2 - window): nan}
        where += [("v_cache", b, j, i % 2, (5 * i + b) % hd, x) for i, (j, x) in enumerate(at.items()) if 0 <= j < n]
    where += [("v_cache", 3, lens[3] - 1, 0, 9, nan), ("v_cache", 3, 0, 1, 3, inf), ("k_cache", 1, 300 - new // 2, 1, 4, nan)]
    kw = make(dtype, lens, [new] * 4, 16, qh, 2, hd, window, sinks, seed=new, descale=dtype == FP8)
    seen = [(n - new - window if window >= 0 else 0, n) for n in lens]  # what the pool holds pages for
    poison(kw, [w for w in where if w[2] >= seen[w[1]][0] or w[2] < sinks])
    check_with_non_finite(kw)
    if new == 90:
        check_with_non_finite(narrow(kw))


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("kvh,gqa,new", [(2, 2, 3), (16, 10, 9), (2, 4, 70)])
def test_non_finite_values_in_split_requests_and_behind_segments(dtype, kvh, gqa, new):
    """One long request over many CTAs, and over few, in segments: the new tokens' values lie in its last piece."""
    kw = repeated(dtype, 64, kvh, gqa, [70000, 33000], new, new)
    own = [torch.empty_like(kw[n][:1]).expand(4, *kw[n].shape[1:]).contiguous() for n in ("k_cache", "v_cache")]
    for t, n in zip(own, ("k_cache", "v_cache")):  # the last two pages of each request are its own
        t.copy_(kw[n][:4])
        kw[n] = torch.cat([kw[n].view(torch.uint8 if dtype == FP8 else torch.int16), t.view(torch.uint8 if dtype == FP8 else torch.int16)]).view(dtype)
    for b, n in enumerate((70000, 33000)):
        last = (n - 1) // 128
        kw["page_table"][b, last - 1], kw["page_table"][b, last] = 8 + 2 * b, 9 + 2 * b
    clean = dict(kw, v_cache=kw["v_cache"].clone())
    poison(kw, [("v_cache", 0, 69999, 0, 3, float("nan")), ("v_cache", 0, 70000 - new + 1, 1, 60, float("nan")),
                ("v_cache", 1, 33000 - new // 2, 1, 0, float("nan"))])
    from greenattention_b200 import attn_paged

    out, lse = attn_paged.attend(**kw)
    want, wlse = attn_paged.attend(**clean)
    assert attn_paged.check_status() == 0 and torch.equal(lse, wlse)
    hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda").view(2, new, kvh, gqa, 64)
    hit[0, new - 1:, 0, :, 3] = True
    hit[0, 1:, 1, :, 60] = True
    hit[1, new - new // 2:, 1, :, 0] = True
    hit = hit.view(out.shape)
    # rows that are computed anew are rounded elsewhere: both results are within the oracle's bound of the definition
    bound = 2 * (2.0**-8 + (2.0**-11 if dtype == FP8 else 2.0**-8) + (32768 + 64) * 2.0**-23) * want.double()
    odd = ((out.isnan() != hit) | ~hit & ((out.double() - want.double()).abs() > bound)).nonzero()
    assert len(odd) == 0, f"{odd[:5].tolist()} of {len(odd)}"
