"""Front-end of the attention over 16-bit and e4m3 paged caches, with first tokens that stay visible beside a window.

The call contract is that of ``attn_decode`` (same names, layouts, causal and window rules), with these differences:

* ``k_cache`` / ``v_cache`` are bf16, fp16 or e4m3; ``q`` has the cache's type (beside e4m3: e4m3, or bf16, which is
  rounded to e4m3 in the kernel), ``out`` too (beside e4m3: bf16). ``head_dim`` 64, 128 or 256, any number of query
  heads per kv head, any power-of-two page size from 1 token, any ``max_seqlen_q``;
* ``sink_tokens=S`` with ``window_size=(W, 0)``: the query at position ``p`` attends the keys ``[p - W, p]`` and the
  request's first ``S`` keys. The pages between the first tokens and the window are never read, so their page-table
  entries may be those of released pages (``kv_pages.PagePool.evict``) and the lengths go on counting;
* a row that sees no key gets zeros and an LSE of -inf; rows of ``out`` and ``lse`` behind the last request's are left
  as they were. Non-finite values count where they are visible, and reach no row that does not see them; a K or V row
  that no query of the call's request sees is not read.

Every call brings its own scratch (from torch's caching allocator, on the current stream), so calls on several streams
and captured graphs do not share any. What the kernels cannot serve is declined with a reason (``dispatch.Declined``).

``attend(**kw)`` is the direct entry. ``select`` is registered for the ops ``decode``, ``verify`` and ``extend``: calls with
``sink_tokens`` come here, and with ``GREEN_ATTN_KV16=1`` every call over a paged bf16 / fp16 cache does.
"""

from __future__ import annotations

import ctypes
import logging
from typing import Callable, Union

import torch

from greenattention_b200 import _C, attn_decode, dispatch

HEAD_DIMS = (64, 128, 256)
MAX_KV_HEADS = 512
KV_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float8_e4m3fn: 2}
FP8 = torch.float8_e4m3fn
STATUS_NAMES = {
    1: "a bounded wait for a full stage ran out", 2: "a bounded wait for a free stage ran out", 4: "shared memory was misplaced",
    3: "a page id was out of range (its keys were taken as zeros)",
    5: "a cache_seqlens entry exceeded page_table.shape[1] * page_size, or 2^30",
}
_ALLOWED = attn_decode._ALLOWED | {"sink_tokens"}
logger = logging.getLogger(__name__)

_status: dict = {}           # device index -> int32 word the kernels leave a non-zero value in
_workspace_bytes: dict = {}  # (device index, batch) -> bytes


def ensure_ready(device: Union[torch.device, int, None] = None) -> None:
    """Load the library and set up ``device``. Idempotent; runs at the first call and has to have run before a CUDA
    graph is captured."""
    if not torch.cuda.is_available():
        raise _C.GreenAttentionError("no CUDA device: the green kernels have no CPU path")
    dev = torch.device("cuda") if device is None else torch.device(device)
    index = torch.cuda.current_device() if dev.index is None else dev.index
    if index in _status:
        return
    if torch.cuda.is_current_stream_capturing():
        raise _C.GreenAttentionError("ensure_ready() has to run before a CUDA graph is captured")
    _C.init(index)
    _status[index] = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", index))
    torch.cuda.synchronize(index)  # the word is zero before a kernel on any stream may set it


def check_status(device: Union[torch.device, int, None] = None, reset: bool = True) -> int:
    """The status word (0 = fine; ``STATUS_NAMES``), logged when it is not 0 and put back. Synchronises."""
    dev = torch.device("cuda") if device is None else torch.device(device)
    index = torch.cuda.current_device() if dev.index is None else dev.index
    if index not in _status:
        return 0
    val = int(_status[index].item())
    if val:
        logger.error("green_attention: paged attention status %d on cuda:%d: %s", val, index, STATUS_NAMES.get(val, "unknown"))
        if reset:
            _status[index].zero_()
    return val


def _prepare(kw: dict):
    """What a call needs at launch, or the reason (a str) why there is no kernel for it: from shapes, types and Python
    scalars only."""
    more = kw.keys() - _ALLOWED
    for name in more:
        if kw[name] is not None:
            return f"unsupported arg {name}"
    get = kw.get
    q, kc, vc, pt, cs, cu = get("q"), get("k_cache"), get("v_cache"), get("page_table"), get("cache_seqlens"), get("cu_seqlens_q")
    for t in (q, kc, vc, pt, cs, cu):
        if not isinstance(t, torch.Tensor):
            return "not a paged varlen call"
    kv, qt = kc.dtype, q.dtype
    if kv not in KV_TYPES or vc.dtype != kv:
        return f"kv dtype {kv} / {vc.dtype}"
    if qt != kv and not (kv == FP8 and qt == torch.bfloat16):
        return f"q dtype {qt} beside a {kv} cache"
    shape, kshape = q.shape, kc.shape
    if len(shape) != 3 or len(kshape) != 4 or kshape != vc.shape:
        return "q or kv rank, or k/v shapes differ"
    total, qh, hd = shape
    pages, page, kvh, khd = kshape
    if hd not in HEAD_DIMS or khd != hd or not kvh or not qh or qh % kvh or kvh > MAX_KV_HEADS:
        return f"q shape: no kernel for (head_dim={hd}, q_heads={qh}, kv_heads={kvh})"
    if page <= 0 or page & (page - 1):
        return "page_size not a power of two"
    align = 15 if kv == FP8 else 7  # elements of 16 bytes
    k0, k1, k2, k3 = kc.stride()
    v0, v1, v2, v3 = vc.stride()
    kp, vp = kc.data_ptr(), vc.data_ptr()
    if k3 != 1 or v3 != 1 or (k0 | k1 | k2 | v0 | v1 | v2) & align or (kp | vp) & 15:
        return "kv layout: last stride 1, other strides and the base multiples of 16 bytes"
    q0, q1, q2 = q.stride()
    qp = q.data_ptr()
    if q2 != 1 or (q0 | q1) & 3 or qp & (3 if qt == FP8 else 7):
        return "q layout: last stride 1, other strides and the base multiples of 4 elements"
    i32 = torch.int32
    ps = pt.shape
    if pt.dtype != i32 or cs.dtype != i32 or cu.dtype != i32 or len(ps) != 2 or cs.dim() != 1 or cu.dim() != 1:
        return "page_table / cache_seqlens / cu_seqlens_q dtype or rank"
    batch = cs.shape[0]
    if batch == 0 or ps[0] != batch or cu.shape[0] != batch + 1:
        return "batch mismatch"
    if batch > 1 and cs.stride(0) != 1 or cu.stride(0) != 1:
        return "cache_seqlens / cu_seqlens_q stride"
    mq = get("max_seqlen_q")
    if type(mq) is not int or mq < 1:
        return f"max_seqlen_q {mq} is not a positive int"
    if mq > 1 and not get("causal", False):
        return "non-causal call with several query tokens"
    if get("softcap"):
        return "softcap"
    left = -1
    if get("window_size") is not None:
        left = attn_decode._window_left(kw)
        if isinstance(left, str):
            return left
        left = min(max(left, -1), 1 << 30)
    sinks = get("sink_tokens") or 0
    if type(sinks) is not int or not 0 <= sinks < 1 << 31:
        return f"sink_tokens {sinks} is not a count"
    dev = q.device
    for t in (kc, vc, pt, cs, cu):
        if t.device != dev:
            return f"a tensor is on {t.device}, q on {dev}"
    scales = []
    for name in ("k_descale", "v_descale"):
        t = get(name)
        if t is None:
            scales += (None, 0, 0)
            continue
        if not isinstance(t, torch.Tensor) or t.device != dev:
            return f"{name} is on {getattr(t, 'device', None)}, q on {dev}"
        why = attn_decode._descale_reason(t, batch, kvh, name)
        if why:
            return why
        scales += (t.data_ptr(), t.stride(0) if t.shape[0] > 1 else 0, t.stride(1))
    out = get("out")
    want = torch.bfloat16 if kv == FP8 else kv
    if out is not None:
        if not isinstance(out, torch.Tensor) or out.device != dev:
            return "out is not a tensor on q's device"
        if out.dtype != want or out.shape != shape or out.stride(2) != 1:
            return f"out must be {want} of q's shape with last stride 1"
        s0, s1, _ = out.stride()
        if (s0 | s1) & 3 or out.data_ptr() & 7 or (qh > 1 and s1 < hd) or (total > 1 and s0 < hd) or (
                qh > 1 and total > 1 and s0 < (qh - 1) * s1 + hd and s1 < (total - 1) * s0 + hd):
            return "out layout: rows must not overlap, strides and the base multiples of 4 elements"
    if dev.type != "cuda":
        return "tensors are on the host: the green kernels have no CPU path"
    scale = get("softmax_scale")
    head = (KV_TYPES[kv], qp, qt == torch.bfloat16, q0, q1, kp, vp, k0, k1, k2, v0, v1, v2, pages, page, qh, kvh, hd,
            pt.data_ptr(), *pt.stride(), ps[1], cs.data_ptr(), cu.data_ptr(), *scales)
    tail = (total, batch, mq, left, sinks, hd**-0.5 if scale is None else scale)
    return q, out, want, get("return_softmax_lse", False), head, tail


def _fire(q, out, want, with_lse, head, tail):
    dev = q.device
    index = dev.index
    if index not in _status:
        ensure_ready(dev)
    total, batch = tail[0], tail[1]
    if out is None:
        out = q.new_empty(q.shape, dtype=want)
    o0, o1, _ = out.stride()
    lse = q.new_empty((q.shape[1], total), dtype=torch.float32) if with_lse else None
    lib = _C.lib()
    nbytes = _workspace_bytes.get((index, batch))
    if nbytes is None:
        nbytes = _workspace_bytes[(index, batch)] = lib.ga_paged_workspace_bytes(index, batch)
    ws = q.new_empty(nbytes, dtype=torch.uint8)
    p = _C.GaPagedParams(*head, out.data_ptr(), o0, o1, lse.data_ptr() if with_lse else None, *tail,
                         _status[index].data_ptr(), ws.data_ptr(), nbytes)
    if torch.cuda.current_device() == index:
        rc = lib.ga_paged_attend(ctypes.byref(p), _C.raw_stream(index))
    else:
        with torch.cuda.device(dev):  # the library launches on the current device
            rc = lib.ga_paged_attend(ctypes.byref(p), _C.raw_stream(index))
    if rc:
        _C.check(rc, "ga_paged_attend")
    return (out, lse) if with_lse else out


def attend(**kw):
    """Attention over a paged cache (see the module); ``out``, or ``(out, lse)`` with ``return_softmax_lse``. Raises
    ``dispatch.Declined`` with the reason for a call outside what the kernels serve."""
    call = _prepare(kw)
    if type(call) is str:
        raise dispatch.Declined(f"attn_paged: {call}")
    return _fire(*call)


def select(kw: dict) -> Union[Callable, str]:
    """The launcher for this call or why there is none, from shapes, types and Python scalars only."""
    call = _prepare(kw)
    if type(call) is str:
        return call
    if kw["q"].device.index not in _status:
        return "kernel not prewarmed for this device"
    return attend


def _select_routed(kw: dict) -> Union[Callable, str]:
    if kw.get("sink_tokens") is None and not dispatch.takes_kv16(kw):
        return "attn_paged: no sink_tokens, and no 16-bit cache with GREEN_ATTN_KV16=1"
    return select(kw)


def _prewarm(backend) -> None:
    ensure_ready()
    check_status()


dispatch.register("decode", _select_routed, prewarm=_prewarm)
dispatch.register("verify", _select_routed)
dispatch.register("extend", _select_routed)
