"""Refusals and routing of the attention over 16-bit and e4m3 paged caches, without a GPU."""

import pytest
import torch

from greenattention_b200 import attn_paged, dispatch, kv_pages

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


def call(device="meta", dtype=BF16, **over):
    z = lambda *s, dt=dtype: torch.zeros(s, dtype=dt, device=device)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)  # noqa: E731
    kw = dict(q=z(4, 8, 128), k_cache=z(9, 16, 2, 128), v_cache=z(9, 16, 2, 128), page_table=i(2, 5), cache_seqlens=i(2),
              cu_seqlens_q=i(3), max_seqlen_q=2, causal=True, window_size=(64, 0), sink_tokens=4)
    return kw | over


@pytest.mark.parametrize("over,needle", [
    (dict(softcap=30.0), "softcap"), (dict(sinks=torch.zeros(8)), "unsupported arg sinks"), (dict(sink_tokens=-1), "sink_tokens"),
    (dict(sink_tokens=1.5), "sink_tokens"), (dict(sink_tokens=True), "sink_tokens"), (dict(window_size=(64, 3)), "window right"),
    (dict(causal=False, window_size=(64, -1)), "non-causal"), (dict(max_seqlen_q=0), "max_seqlen_q"), (dict(max_seqlen_q=None), "max_seqlen_q"),
    (dict(page_table=None), "paged"), (dict(cache_seqlens=7), "paged"),
    (dict(q=torch.zeros(4, 8, 128, dtype=torch.float16, device="meta")), "q dtype"),
    (dict(q=torch.zeros(4, 8, 96, dtype=BF16, device="meta")), "head_dim"),
    (dict(q=torch.zeros(4, 7, 128, dtype=BF16, device="meta")), "q_heads"),
    (dict(q=torch.zeros(4, 8, 256, dtype=BF16, device="meta")[:, :, ::2]), "q layout"),
    (dict(q=torch.zeros(4, 8, 130, dtype=BF16, device="meta")[:, :, :128]), "q layout"),
    (dict(k_cache=torch.zeros(9, 12, 2, 128, dtype=BF16, device="meta"), v_cache=torch.zeros(9, 12, 2, 128, dtype=BF16, device="meta")), "power of two"),
    (dict(v_cache=torch.zeros(8, 16, 2, 128, dtype=BF16, device="meta")), "shapes differ"),
    (dict(v_cache=torch.zeros(9, 16, 2, 128, dtype=torch.float16, device="meta")), "kv dtype"),
    (dict(k_cache=torch.zeros(9, 16, 2, 132, dtype=BF16, device="meta")[..., :128]), "kv layout"),
    (dict(page_table=torch.zeros(2, 5, dtype=torch.int64, device="meta")), "page_table"),
    (dict(cu_seqlens_q=torch.zeros(4, dtype=torch.int32, device="meta")), "batch mismatch"),
    (dict(cache_seqlens=torch.zeros(2, dtype=torch.int32)), "on cpu"), (dict(k_descale=torch.ones(2, 2)), "k_descale is on cpu"),
    (dict(k_descale=torch.ones(3, 2, device="meta")), "k_descale"), (dict(out=torch.zeros(4, 8, 128, dtype=torch.float32, device="meta")), "out must be"),
    (dict(out=torch.zeros(1, 8, 128, dtype=BF16, device="meta").expand(4, 8, 128)), "overlap"), (dict(), "on the host"),
])
def test_refusals(over, needle):
    why = attn_paged.select(call(**over))
    assert isinstance(why, str) and needle in why, why
    with pytest.raises(dispatch.Declined, match="attn_paged"):
        attn_paged.attend(**call(**over))


def test_routing(monkeypatch):
    kw = call()
    assert dispatch.owns(kw) and not dispatch.takes_kv16(kw)
    plain = call(sink_tokens=None)
    assert not dispatch.owns(plain) and "GREEN_ATTN_KV16" in attn_paged._select_routed(plain)
    assert "GREEN_ATTN_KV16" in attn_paged._select_routed(call(dtype=FP8, sink_tokens=None))
    monkeypatch.setattr(dispatch, "KV16", True)
    assert dispatch.takes_kv16(plain) and not dispatch.owns(plain)
    assert "on the host" in attn_paged._select_routed(plain)
    assert "GREEN_ATTN_KV16" in attn_paged._select_routed(call(dtype=FP8, sink_tokens=None))


def pool(**over):
    c = [torch.zeros(6, 16, 2, 64, dtype=BF16) for _ in range(4)]
    kw = dict(caches=c, page_table=torch.zeros(3, 4, dtype=torch.int32), seqlens=torch.zeros(3, dtype=torch.int32),
              refs=torch.zeros(6, dtype=torch.int32))
    return kv_pages.PagePool(**(kw | over))


@pytest.mark.parametrize("over,needle", [
    (dict(caches=[]), "no tensors"), (dict(caches=[torch.zeros(5, 16, 2, 64)]), "tensor 0"),
    (dict(caches=[torch.zeros(6, 12, 2, 64)]), "power of two"), (dict(caches=[torch.zeros(6, 16, 3, dtype=torch.uint8)]), "16 bytes"),
    (dict(caches=[torch.zeros(6, 16, 4, 64).transpose(1, 2).contiguous().transpose(1, 2)]), "not dense"),
    (dict(caches=[torch.zeros(1, 16, 2, 64).expand(6, 16, 2, 64)]), "overlap"), (dict(caches=[torch.zeros(6, 16, 2, 64)] * 2), "twice"),
    (dict(page_table=torch.zeros(3, 4, dtype=torch.int64)), "int32"), (dict(seqlens=torch.zeros(4, dtype=torch.int32)), "as long as"),
    (dict(refs=torch.zeros(6, dtype=torch.int32, device="meta")), "different devices"),
    (dict(page_table=torch.zeros(1, 4, dtype=torch.int32).expand(3, 4)), "overlap"),
])
def test_pool_refusals(over, needle):
    with pytest.raises(dispatch.Declined, match=needle):
        pool(**over)


def test_pool_has_no_cpu_path():
    from greenattention_b200 import _C

    with pytest.raises(_C.GreenAttentionError, match="no CPU path"):
        pool()


def test_struct_layouts_match_the_header():
    """Field names and order of the ctypes mirrors follow the C structs."""
    import os
    import re

    from greenattention_b200 import _C

    with open(os.path.join(os.path.dirname(os.path.dirname(__file__)), "include", "green_attention.h")) as f:
        header = f.read()
    for name, mirror in (("GaPagedParams", _C.GaPagedParams), ("GaPagePool", _C.GaPagePool)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header, flags=re.S).group(1)
        fields = []
        for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
            parts = [x.strip() for x in decl.strip().split(",")]
            if parts[0]:
                fields += [re.split(r"[\s*]+", parts[0])[-1]] + [x.lstrip("*").strip() for x in parts[1:]]
        assert fields == [n for n, _ in mirror._fields_], name


def test_pool_of_more_pages_than_the_kernels_count():
    n = (1 << 31) - 32768
    m = dict(dtype=torch.int32, device="meta")
    for pages, needle in ((n, "at most"), (n - 1, "no CPU path")):
        with pytest.raises(Exception, match=needle):
            kv_pages.PagePool([torch.zeros(pages, 1, 4, **m)], torch.zeros(1, 4, **m), torch.zeros(1, **m), torch.zeros(pages, **m))


@pytest.mark.parametrize("strides,ok", [
    ((1024, 128, 1), True), ((128, 512, 1), True), ((1028, 128, 1), True), ((128, 516, 1), True), ((1152, 144, 1), True),
    ((128, 128, 1), False), ((1020, 128, 1), False), ((128, 508, 1), False), ((256, 128, 1), False), ((128, 384, 1), False),
])
def test_rows_of_out_that_overlap_are_refused(strides, ok):
    out = torch.empty_strided((4, 8, 128), strides, dtype=BF16, device="meta")
    why = attn_paged.select(call(out=out))
    assert ("on the host" if ok else "overlap") in why
