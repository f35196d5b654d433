"""64-bit definition of the attention over paged caches with a window and first tokens (``attn_paged``), and the books of a
page pool kept with lists (``kv_pages``). Pure torch / Python on the CPU; used by the tests only."""

from __future__ import annotations

import math

import torch

FP8 = torch.float8_e4m3fn
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def attend(kw: dict) -> dict:
    """``out``, ``lse`` and how far a right kernel may be from them, from the definition, in 64 bits.

    ``out_tol``: half a step of the output's type for its rounding; half a step of P's 16-bit type (fp16 beside an e4m3
    cache) for every probability, i.e. that share of ``sum_j p_j |v_j|``; half the fp16 subnormal step where out is fp16, and
    2^-32 of the row's largest probability for every key where P is (fp16 P are taken up to 2^7 and more);
    and the 32-bit scores: a dot product of ``hd`` terms is off by at most ``hd 2^-23 sum |q_d k_d|`` in any order of
    summation with truncation, which changes every probability by that factor twice (numerator and sum). ``lse_tol``: the
    scores' part, ``n 2^-23`` for the sum of n terms and 2^-20 for the exponentials and the logarithm."""
    q, kc, vc = (kw[n].cpu() for n in ("q", "k_cache", "v_cache"))
    pt, lens, cu = (kw[n].cpu().tolist() for n in ("page_table", "cache_seqlens", "cu_seqlens_q"))
    total, qh, hd = q.shape
    page, kvh = kc.shape[1], kc.shape[2]
    gqa = qh // kvh
    scale = hd**-0.5 if kw.get("softmax_scale") is None else kw["softmax_scale"]
    window = kw.get("window_size") or (-1, -1)
    window = -1 if window[0] is None else window[0]
    sinks = kw.get("sink_tokens") or 0
    if kc.dtype == FP8 and q.dtype == torch.bfloat16:
        q = q.float().clamp(-448, 448).to(FP8)
    out_type = torch.bfloat16 if kc.dtype == FP8 else kc.dtype
    p_type = torch.float16 if kc.dtype == FP8 else kc.dtype
    q = q.double()
    out = torch.full((total, qh, hd), math.nan, dtype=torch.float64)
    tol = torch.zeros_like(out)
    lse = torch.full((qh, total), math.nan, dtype=torch.float64)
    lse_tol = torch.zeros_like(lse)
    kd, vd = (None if kw.get(n) is None else kw[n].cpu().double().expand(len(lens), kvh) for n in ("k_descale", "v_descale"))
    for b, n in enumerate(lens):
        new = cu[b + 1] - cu[b]
        for t in range(new):
            p = n - new + t
            keys = [j for j in range(0, p + 1) if window < 0 or j >= p - window or j < sinks]
            row = cu[b] + t
            if not keys:
                out[row] = 0
                lse[:, row] = -math.inf
                continue
            at = [(pt[b][j // page], j % page) for j in keys]
            k = torch.stack([kc[a, c].double() for a, c in at])  # [n, kvh, hd]
            v = torch.stack([vc[a, c].double() for a, c in at])
            for h in range(kvh):
                ks = scale * (1.0 if kd is None else kd[b, h].item())
                vs = 1.0 if vd is None else vd[b, h].item()
                rows = q[row, h * gqa:(h + 1) * gqa]
                s = rows @ k[:, h].T * ks
                z = torch.logsumexp(s, -1)
                w = torch.exp(s - z[:, None])
                o = w @ v[:, h] * vs
                spread = (w @ v[:, h].abs()) * abs(vs)
                off = (hd * 2.0**-23 * (rows.abs() @ k[:, h].abs().T) * abs(ks)).amax(-1) + s.abs().amax(-1) * 2.0**-22
                heads = slice(h * gqa, (h + 1) * gqa)
                out[row, heads] = o
                e = HALF_STEP[out_type] * o.abs() + (HALF_STEP[p_type] + 2 * off[:, None] + (len(keys) + 64) * 2.0**-23) * spread
                if p_type == torch.float16:
                    # P is 2^7 at least at the largest probability: half its smallest fp16 step, over the sum
                    e = e + 2.0**-32 * v[:, h].abs().sum(0) * abs(vs) * w.amax(-1)[:, None]
                if out_type == torch.float16:
                    e = e + 2.0**-25
                tol[row, heads] = e * (1 + 2.0**-6)  # products of two of these terms
                lse[heads, row] = z
                lse_tol[heads, row] = off + len(keys) * 2.0**-23 + 2.0**-20 * (1 + z.abs())
    return {"out": out, "out_tol": tol, "lse": lse, "lse_tol": lse_tol}


class Books:
    """The rules of ``kv_pages.PagePool``, one entry after the other."""

    def __init__(self, caches, table, lens, refs):
        self.caches = [c.clone() for c in caches]
        self.table, self.lens, self.refs = [list(r) for r in table], list(lens), list(refs)
        self.page, self.status = caches[0].shape[1], 0

    def pages(self, n):
        return -(-max(0, n) // self.page)

    def _move(self, dst, src, tokens):
        for c in self.caches:
            c[dst, :tokens] = c[src, :tokens]

    def copy(self, src, dst):
        n = len(self.refs)
        ok = [0 <= a < n and 0 <= b < n for a, b in zip(src, dst)]
        written = {b for a, b, o in zip(src, dst, ok) if o and a != b}
        last = {b: i for i, (a, b, o) in enumerate(zip(src, dst, ok)) if o and a != b}
        if not all(ok):
            self.status = 7
        for i, (a, b, o) in enumerate(zip(src, dst, ok)):
            if o and a != b and last[b] == i:
                if a in written:
                    self.status = 10
                else:
                    self._move(b, a, self.page)

    def _release(self, row, cols):
        for j in cols:
            e = self.table[row][j]
            if e >= 0:
                self.table[row][j] = -1
                if e >= len(self.refs):
                    self.status = 3
                elif self.refs[e] <= 0:
                    self.status = 9
                else:
                    self.refs[e] -= 1

    def _rows(self, rows):
        for r in dict.fromkeys(rows):
            if 0 <= r < len(self.lens):
                yield r
            else:
                self.status = 7

    def free(self, rows):
        for r in self._rows(rows):
            self._release(r, range(self.pages(self.lens[r])))
            self.lens[r] = 0

    def evict(self, rows, window_left, sink_tokens=0):
        for r in self._rows(rows):
            self._release(r, range(self.pages(sink_tokens), max(0, self.lens[r] - window_left) // self.page))

    def grow(self, rows, lens):
        spare = [i for i, n in enumerate(self.refs) if n == 0]
        seen, short = set(), False
        for r, n in zip(rows, lens):
            if not 0 <= r < len(self.lens):
                self.status = 7
                continue
            if r in seen:
                self.status = 10
                continue
            seen.add(r)
            if self.pages(n) > len(self.table[r]):
                self.status = 5
                continue
            have = self.pages(self.lens[r])
            need = max(0, self.pages(n) - have)
            short |= need > len(spare)
            if need and short:
                self.status = 8
                continue
            for j in range(have, have + need):
                self.table[r][j] = spare.pop(0)
                self.refs[self.table[r][j]] = 1
            self.lens[r] = max(self.lens[r], n)

    def fork(self, parents, children):
        spare = [i for i, n in enumerate(self.refs) if n == 0]
        was = list(self.lens)
        seen = set()
        for a, c in zip(parents, children):
            if not (0 <= a < len(was) and 0 <= c < len(was)):
                self.status = 7
                continue
            if c in seen or was[c] != 0:
                self.status = 10
                seen.add(c)
                continue
            seen.add(c)
            n, tail = was[a], was[a] % self.page
            if n == 0:
                continue
            if tail:
                src = self.table[a][n // self.page]
                if not 0 <= src < len(self.refs):
                    self.status = 3
                    continue
                if not spare:
                    self.status = 8
                    continue
                new = spare.pop(0)
                self._move(new, src, tail)
                self.table[c][n // self.page] = new
                self.refs[new] = 1
            for j in range(n // self.page):
                e = self.table[c][j] = self.table[a][j]
                if e >= 0:
                    self.refs[e] += 1
            self.lens[c] = n

    def compact(self):
        live = [i for i, n in enumerate(self.refs) if n > 0]
        gaps = [i for i in range(len(live)) if self.refs[i] <= 0]
        to = {i: i for i in live}
        for i in live:
            if i >= len(live):
                to[i] = gaps.pop(0)
                self._move(to[i], i, self.page)
                self.refs[to[i]], self.refs[i] = self.refs[i], 0
        for r, n in enumerate(self.lens):
            for j in range(self.pages(n)):
                e = self.table[r][j]
                if e >= 0:
                    if e in to:
                        self.table[r][j] = to[e]
                    else:
                        self.status = 9
        return [to.get(i, -1) for i in range(len(self.refs))], len(live)
