"""The pages' upkeep against the rules kept with lists (``oracle/paged_oracle.Books``): counts, table, lengths and every
byte of the pools, random histories and the calls that contradict themselves, and a run with the attention."""

import random

import pytest
import torch

from oracle import paged_oracle

pytestmark = pytest.mark.gpu


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def setup(pages, page, rows, cols, layers=2, seed=0, tail=(2, 32), wide_table=False, interleaved=False):
    from greenattention_b200 import kv_pages

    g = torch.Generator().manual_seed(seed)
    caches = []
    for _ in range(layers):
        if interleaved:
            buf = torch.randint(0, 255, (pages, 2, page, *tail), generator=g, dtype=torch.uint8).cuda()
            caches += [buf[:, 0], buf[:, 1]]
        else:
            caches += [torch.randint(0, 255, (pages, page, *tail), generator=g, dtype=torch.uint8).cuda() for _ in range(2)]
    table = torch.full((rows, cols + 3 * wide_table), -1, dtype=torch.int32, device="cuda")[:, :cols]
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    pool = kv_pages.PagePool(caches, table, lens, refs)
    books = paged_oracle.Books([c.cpu() for c in caches], table.tolist(), lens.tolist(), refs.tolist())
    return pool, books


def same(pool, books):
    torch.cuda.synchronize()
    assert pool.seqlens.tolist() == books.lens and pool.refs.tolist() == books.refs
    assert pool.page_table.tolist() == books.table
    for a, b in zip(pool.caches, books.caches):
        assert torch.equal(a.cpu(), b)
    assert pool.check_status() == books.status
    books.status = 0


def both(pool, books, name, *lists, dtype=torch.int32, **kw):
    getattr(pool, name)(*[ints(v, dtype) for v in lists], **kw)
    getattr(books, name)(*lists, **kw)


@pytest.mark.parametrize("page", [1, 4, 16, 128])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_histories(page, dtype):
    r = random.Random(page)
    rows, cols = 12, 9
    pool, books = setup(300, page, rows, cols, seed=page, wide_table=True, interleaved=page == 4)
    for step in range(40):
        some = r.sample(range(rows), r.randint(1, 5))
        what = r.choice(["grow", "grow", "free", "evict", "fork", "compact", "copy"])
        if what == "grow":
            both(pool, books, "grow", some, [min(cols * page, books.lens[x] + r.randint(0, 3 * page)) for x in some], dtype=dtype)
        elif what == "free":
            both(pool, books, "free", some[:2], dtype=dtype)
        elif what == "evict":
            both(pool, books, "evict", some, window_left=r.randint(0, 4 * page), sink_tokens=r.randint(0, 2 * page), dtype=dtype)
        elif what == "fork":
            empty = [x for x in range(rows) if books.lens[x] == 0][:3]
            full = [x for x in range(rows) if books.lens[x] > 0]
            if empty and full:
                both(pool, books, "fork", [r.choice(full) for _ in empty], empty, dtype=dtype)
        elif what == "compact":
            to, live = pool.compact()
            want, n = books.compact()
            assert to.tolist() == want and live.item() == n
        else:
            ids = r.sample(range(300), 8)
            both(pool, books, "copy", ids[:4], ids[4:], dtype=dtype)
        same(pool, books)


def test_entries_that_contradict_one_another():
    pool, books = setup(40, 8, 6, 4)
    both(pool, books, "grow", [0, 1, 0, 2], [20, 9, 30, 0])
    same(pool, books)
    both(pool, books, "copy", [5, 6, 7, 3, 9, 9], [20, 20, 21, 3, 7, 22])  # two writers of 20, a source that is written, onto itself
    assert books.status == 10
    same(pool, books)
    both(pool, books, "copy", [1, -1, 40, 2, 3], [30, 31, 32, 40, 33])
    assert books.status == 7
    same(pool, books)
    both(pool, books, "fork", [0, 0, 1, 3, 0], [4, 4, 1, 5, 2])  # named twice, not empty, an empty parent
    assert books.status == 10
    same(pool, books)
    both(pool, books, "fork", [9, -1, 0], [3, 3, 6])
    same(pool, books)
    both(pool, books, "free", [0, 0, 7, -2, 4])
    same(pool, books)
    both(pool, books, "evict", [1, 1], window_left=0)
    same(pool, books)
    both(pool, books, "grow", [3, 5], [33, 12])  # beyond the table's row
    assert books.status == 5
    same(pool, books)


@pytest.mark.parametrize("page", [1, 16])
def test_no_free_page_left(page):
    pool, books = setup(10, page, 6, 8)
    both(pool, books, "grow", [0, 1, 2, 3], [4 * page, 0, 5 * page, 2 * page])  # one page short for row 3
    assert books.status == 8
    same(pool, books)
    both(pool, books, "grow", [4, 5], [page + 1, 1])
    same(pool, books)
    if page > 1:
        both(pool, books, "free", [4])
        both(pool, books, "grow", [0], [3 * page + 1])
        both(pool, books, "grow", [5], [3])
        both(pool, books, "fork", [5, 0, 5], [1, 3, 4])
        same(pool, books)


def test_counts_that_do_not_match_are_not_driven_below_zero():
    pool, books = setup(20, 4, 3, 5)
    both(pool, books, "grow", [0, 1], [17, 9])
    pool.refs[1] = 0
    books.refs[1] = 0
    pool.page_table[1, 1] = 99
    books.table[1][1] = 99
    both(pool, books, "free", [0])
    assert books.status == 9
    same(pool, books)
    both(pool, books, "free", [1])
    assert books.status == 3
    same(pool, books)


@pytest.mark.parametrize("pages", [1, 15, 16384, 16385, 70001])
def test_compact_over_pool_sizes(pages):
    """Spans of the kernels begin and end inside the pool; counts that are not 16-byte aligned."""
    from greenattention_b200 import kv_pages

    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        share = (0.1, 0.5, 0.95)[seed]
        store = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
        refs = store[seed % 2:seed % 2 + pages]
        refs.copy_((torch.rand(pages, generator=g, device="cuda") < share) * 3)
        cache = torch.arange(pages, dtype=torch.int32, device="cuda").view(-1, 1, 1).expand(pages, 1, 4).contiguous()
        held = refs.nonzero()[:, 0]
        table = held.to(torch.int32)[None].contiguous() if len(held) else torch.zeros((1, 1), dtype=torch.int32, device="cuda")
        lens = ints([len(held)])
        pool = kv_pages.PagePool([cache], table, lens, refs)
        to, live = pool.compact()
        n = len(held)
        low, moved = held[held < n], held[held >= n]
        gaps = torch.tensor(sorted(set(range(n)) - set(low.tolist())), device="cuda", dtype=torch.int64)
        want = torch.full((pages,), -1, device="cuda", dtype=torch.int64)
        want[low], want[moved] = low, gaps
        assert live.item() == n and torch.equal(to.long(), want)
        assert torch.equal(refs, (torch.arange(pages, device="cuda") < n) * 3) and pool.check_status() == 0
        if n:
            assert torch.equal(table[0].long(), want[held]) and torch.equal(cache[table[0].long(), 0, 0].long(), held)


def test_many_rows_and_pages_of_a_large_pool():
    pool, books = setup(40000, 1, 3000, 24, layers=1, tail=(16,))
    r = random.Random(1)
    rows = r.sample(range(3000), 2500)
    both(pool, books, "grow", rows, [r.randint(0, 15) for _ in rows])
    same(pool, books)
    both(pool, books, "free", rows[::2])
    both(pool, books, "fork", rows[1:1000:2], rows[0:999:2])
    want, n = books.compact()
    to, live = pool.compact()
    assert to.tolist() == want and live.item() == n
    same(pool, books)


def test_offsets_beyond_32_bits():
    from greenattention_b200 import kv_pages

    pages, page = 70000, 64
    cache = torch.empty((pages, page, 8, 128), dtype=torch.uint8, device="cuda")  # 4.6 GB
    cache[-3:] = torch.arange(3, device="cuda", dtype=torch.uint8).view(3, 1, 1, 1) + 5
    cache[0] = 1
    pool = kv_pages.PagePool([cache], ints([[0]]), ints([0]), torch.ones(pages, dtype=torch.int32, device="cuda"))
    pool.copy(ints([pages - 1, 0]), ints([1, pages - 2]))
    assert (cache[1] == 7).all() and (cache[pages - 2] == 1).all() and (cache[pages - 3] == 5).all() and (cache[-1] == 7).all()


def test_in_a_graph_and_on_another_stream():
    pool, books = setup(60, 8, 6, 6)
    rows, lens = ints([0, 1]), ints([20, 31])
    kids, parents = ints([2, 3]), ints([0, 1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pool.free(kids)
        pool.free(rows)
        pool.grow(rows, lens)
        pool.fork(parents, kids)
        pool.compact()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for n in (20, 7):
        lens[0] = n
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        books.free([2, 3])
        books.free([0, 1])
        books.grow([0, 1], [n, 31])
        books.fork([0, 1], [2, 3])
        books.compact()
        same(pool, books)


def test_refusals_of_calls():
    from greenattention_b200 import dispatch

    pool, _ = setup(10, 4, 3, 3)
    for bad in (lambda: pool.free([1]), lambda: pool.free(torch.tensor([1])), lambda: pool.free(ints([1]).float()),
                lambda: pool.free(ints([[1]])), lambda: pool.free(ints([0, 1, 2, 0])[::2]), lambda: pool.copy(ints([1]), ints([1, 2])),
                lambda: pool.copy(ints([1]), ints([1], torch.int64)), lambda: pool.evict(ints([1]), -1), lambda: pool.evict(ints([1]), 3, True),
                lambda: pool.grow(ints([1]), ints([1, 2])), lambda: pool.grow(ints([0] * 40000), ints([0] * 40000))):
        with pytest.raises(dispatch.Declined):
            bad()
    none = ints([])
    pool.free(none), pool.grow(none, none), pool.fork(none, none), pool.copy(none, none), pool.evict(none, 1)
    assert pool.check_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_serving_run(dtype):
    """Prompts, forks, decode steps that write each new token, eviction behind the window, compaction, the end: every
    step's attention is that of an unpaged history kept beside it."""
    from greenattention_b200 import attn_paged, kv_pages

    page, kvh, qh, hd, rows, cols, window, sinks = 16, 2, 8, 128, 6, 20, 40, 3
    pages = 48
    g = torch.Generator(device="cuda").manual_seed(1)
    kc, vc = (torch.full((pages, page, kvh, hd), float("nan"), device="cuda").to(dtype) for _ in range(2))
    table = torch.full((rows, cols), -1, dtype=torch.int32, device="cuda")
    lens, refs = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(pages, dtype=torch.int32, device="cuda")
    pool = kv_pages.PagePool([kc, vc], table, lens, refs)
    history = {}

    def step(live, new):
        """New tokens of the rows `live` are written to their pages, then attended."""
        have = lens.tolist()
        pool.grow(ints(live), ints([have[x] + n for x, n in zip(live, new)]))
        for x, n in zip(live, new):
            k, v = (torch.randn((n, kvh, hd), generator=g, device="cuda").to(dtype) for _ in range(2))
            at = torch.arange(have[x], have[x] + n, device="cuda")
            for c, t in ((kc, k), (vc, v)):
                c.view(torch.uint8)[table[x, at // page].long(), at % page] = t.view(torch.uint8)
            old = history.get(x)
            history[x] = [k, v] if old is None else [torch.cat([a.view(torch.uint8), b.view(torch.uint8)]).view(dtype) for a, b in zip(old, (k, v))]
        q = torch.randn((sum(new), qh, hd), generator=g, device="cuda").to(torch.bfloat16)
        kw = dict(q=q, cu_seqlens_q=ints([0] + new).cumsum(0).to(torch.int32), max_seqlen_q=max(new), causal=True,
                  window_size=(window, 0), sink_tokens=sinks, return_softmax_lse=True)
        got = attn_paged.attend(k_cache=kc, v_cache=vc, page_table=table[live], cache_seqlens=lens[live], **kw)
        flat = dict(kw, cache_seqlens=lens[live])
        most = max(len(history[x][0]) for x in live)
        whole = [torch.zeros((len(live), 512, kvh, hd), device="cuda").to(dtype) for _ in range(2)]
        for i, x in enumerate(live):
            for w, h in zip(whole, history[x]):
                w.view(torch.uint8)[i, : len(h)] = h.view(torch.uint8)
        assert most <= 512
        want = attn_paged.attend(k_cache=whole[0], v_cache=whole[1], page_table=ints([[i] for i in range(len(live))]), **flat)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        oracle = paged_oracle.attend(dict(flat, k_cache=whole[0], v_cache=whole[1], page_table=ints([[i] for i in range(len(live))])))
        assert ((got[0].cpu().double() - oracle["out"]).abs() <= oracle["out_tol"]).all()

    step([0, 1], [75, 33])
    pool.fork(ints([0, 0, 1]), ints([2, 3, 4]))
    for a, c in ((0, 2), (0, 3), (1, 4)):
        history[c] = list(history[a])
    for n in range(4):
        step([0, 1, 2, 3, 4], [1 + n % 2] * 5)
        pool.evict(ints([0, 1, 2, 3, 4]), window, sinks)
    pool.free(ints([0, 3]))
    history.pop(0), history.pop(3)
    to, live = pool.compact()
    assert (refs[: live.item()] > 0).all() and (refs[live.item():] == 0).all()
    step([1, 2, 4], [5, 1, 3])
    step([1, 0, 2, 4], [1, 50, 1, 1])
    pool.free(ints(list(range(rows))))
    assert (refs == 0).all() and (lens == 0).all() and pool.check_status() == 0 and attn_paged.check_status() == 0


@pytest.mark.parametrize("pages", [1, 15, 16383, 16384, 16385, 32768])
@pytest.mark.parametrize("left", [0, -1, 7])
@pytest.mark.parametrize("hole", [None, 0, -1])
def test_compact_of_a_full_pool(pages, left, hole):
    """Every page held, or all but the first or last: whatever words the scratch holds before the call, nothing but the
    page into the hole moves."""
    import ctypes

    from greenattention_b200 import _C, kv_pages

    held = [i for i in range(pages) if hole is None or i != hole % pages]
    refs = torch.full((pages,), 2, dtype=torch.int32, device="cuda")
    if hole is not None:
        refs[hole] = 0
    cache = torch.arange(pages, dtype=torch.int32, device="cuda").view(-1, 1, 1).expand(pages, 1, 4).contiguous()
    table = ints([held or [-1]])
    pool = kv_pages.PagePool([cache], table, ints([len(held)]), refs)
    lib = _C.lib()
    p = _C.GaPagePool.from_buffer_copy(pool._p)
    nbytes = lib.ga_pages_scratch_bytes(ctypes.byref(p), 0)
    scratch = torch.full((nbytes // 4,), left, dtype=torch.int32, device="cuda")
    p.scratch, p.scratch_bytes = scratch.data_ptr(), nbytes
    to, live = torch.full((pages,), -9, dtype=torch.int32, device="cuda"), ints([-9])
    _C.check(lib.ga_pages_compact(ctypes.byref(p), to.data_ptr(), live.data_ptr(), _C.raw_stream(pool.device.index)), "compact")
    n = len(held)
    want = [-1] * pages
    for i in held:
        want[i] = i if i < n else hole % pages
    assert live.item() == n and to.tolist() == want and pool.check_status() == 0
    assert refs.tolist() == [2] * n + [0] * (pages - n)
    if n:
        assert table[0].tolist() == [want[i] for i in held]
        assert torch.equal(cache[table[0].long(), 0, 0].long(), torch.tensor(held, device="cuda"))


@pytest.mark.parametrize("page", [1, 2, 16])
@pytest.mark.parametrize("window,sinks", [(0, (1 << 31) - 1), ((1 << 31) - 1, 0), ((1 << 31) - 1, (1 << 31) - 1), (0, (1 << 31) - 257), (3, 5)])
def test_evict_with_the_largest_window_and_first_tokens(page, window, sinks):
    pool, books = setup(400, page, 3, 300 // page + 1)
    both(pool, books, "grow", [0, 1, 2], [290, 0, 7])
    both(pool, books, "evict", [0, 1, 2], window_left=window, sink_tokens=sinks)
    same(pool, books)


def test_grow_past_32_bits_of_pages():
    """All rows of a wide table ask for all columns: more pages than an int counts. None are there for any row."""
    from greenattention_b200 import kv_pages

    rows, cols, pages = 32768, 65537, 100
    cache = torch.zeros((pages, 1, 16), dtype=torch.uint8, device="cuda")
    table = torch.full((rows, cols), -1, dtype=torch.int32, device="cuda")  # 8.6 GB
    lens, refs = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(pages, dtype=torch.int32, device="cuda")
    pool = kv_pages.PagePool([cache], table, lens, refs)
    every = torch.arange(rows, dtype=torch.int32, device="cuda")
    pool.grow(every, torch.full_like(every, cols))
    assert pool.check_status() == 8
    assert not lens.any() and not refs.any() and (table[:, :200] == -1).all()
    some = torch.full_like(every, cols)
    some[0], some[-1] = 60, 0  # the first row fits; no other does
    pool.grow(every, some)
    assert pool.check_status() == 8
    assert lens[0] == 60 and lens.sum() == 60 and refs.sum() == 60 and (table[1:, :200] == -1).all()
    assert table[0, :60].tolist() == list(range(60))
    some[1:] = 0  # rows that need no page, in the shadow of one that finds none
    some[0], some[1], some[5] = 60, cols, 0
    lens[7] = 3
    some[7] = 2
    pool.grow(every, some)
    assert pool.check_status() == 8 and lens[0] == 60 and lens[7] == 3 and lens.sum() == 63


@pytest.mark.parametrize("want", [(1 << 31) - 1, 1 << 31, (1 << 31) + 5, (1 << 32) + 7, (1 << 62)])
def test_grow_to_lengths_that_no_int_holds(want):
    from greenattention_b200 import kv_pages

    page, cols = 4096, 1 << 20  # 2^32 tokens a row
    cache = torch.zeros((3, page, 16), dtype=torch.uint8, device="cuda")
    table = torch.full((2, cols), -1, dtype=torch.int32, device="cuda")
    pool = kv_pages.PagePool([cache], table, ints([0, 0]), ints([0, 0, 0]))
    pool.grow(ints([0, 1], torch.int64), ints([want, 5000], torch.int64))
    first = pool.check_status()
    assert first == (8 if want < 1 << 31 else 5)
    if want < 1 << 31:  # asks for 2^19 pages; the row behind it is left as it was
        assert pool.seqlens.tolist() == [0, 0] and pool.refs.tolist() == [0, 0, 0]
    else:
        assert pool.seqlens.tolist() == [0, 5000] and pool.refs.tolist() == [1, 1, 0] and table[1, :2].tolist() == [0, 1]
