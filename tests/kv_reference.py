"""Plain 64-bit and fp32 restatements of the paged INT8 key/value cache, for the tests: quantisation step by
step in numpy fp32 (each operation rounded to nearest, as the operator is defined), attention in float64."""
from __future__ import annotations

import numpy as np
import torch

INV127 = np.float32(1.0) / np.float32(127.0)
TINY = np.float32(1e-30)


class CacheRef:
    """The cache on the host: codes, scales and sums, with the write rule applied page by page."""

    def __init__(self, pages, heads, dim, page):
        self.page = page
        self.code = {n: np.zeros((pages, heads, page, dim), np.int8) for n in "kv"}
        self.scale = {n: np.zeros((pages, heads), np.float32) for n in "kv"}
        self.k_sum = np.zeros((pages, heads, dim), np.int16)

    def write(self, table, start, count, k, v):
        """table: the sequence's pages; k, v fp32 [heads, count, dim]."""
        ps = self.page
        if not count:
            return
        for slot in range(start // ps, -(-(start + count) // ps)):
            p, lo, hi = table[slot], max(start, slot * ps), min(start + count, slot * ps + ps)
            for name, src in (("k", k), ("v", v)):
                for h in range(src.shape[0]):
                    x = src[h, lo - start: hi - start].astype(np.float32)
                    old = lo - slot * ps
                    codes, had = self.code[name][p, h], self.scale[name][p, h]
                    if not np.isfinite(x).all() or (old and np.isnan(had)):
                        self.scale[name][p, h] = np.nan
                        codes[old: hi - slot * ps] = 0
                        continue
                    s = max(np.abs(x).max() * INV127, TINY)
                    if old:
                        s = max(s, had)
                        if s > had:
                            codes[:old] = np.rint(codes[:old].astype(np.float32) * (had / s)).astype(np.int8)
                    codes[old: hi - slot * ps] = np.rint(x * (np.float32(1.0) / s)).astype(np.int8)
                    self.scale[name][p, h] = s
            if hi == slot * ps + ps:
                self.k_sum[p] = self.code["k"][p].astype(np.int32).sum(1).astype(np.int16)

    def dense(self, name, table, n):
        """float64 [heads, n, dim]."""
        at = np.asarray(table[: -(-n // self.page)], np.int64)
        if not len(at):
            return np.zeros((self.scale[name].shape[1], 0, self.code[name].shape[-1]))
        x = self.code[name][at].astype(np.float64) * self.scale[name][at].astype(np.float64)[..., None, None]
        return np.moveaxis(x, 0, 1).reshape(x.shape[1], -1, x.shape[-1])[:, :n]

    def tensors(self, device="cuda"):
        t = lambda a: torch.from_numpy(a).to(device)  # noqa: E731
        return dict(k=t(self.code["k"]), v=t(self.code["v"]), k_scale=t(self.scale["k"]), v_scale=t(self.scale["v"]),
                    k_sum=t(self.k_sum))


def attend(q, k, v, vs, pos, scale, causal=True, window=0, pages=None, page=0):
    """One kv head.  q float64 [rows, D] with position pos[row] (-1: padding), k and v [n, D], vs [n] the V scale of
    each key's page; pages: per row the
    page ordinals it may see.  Returns (out, lse, bound): `bound` is the error a kernel may make before its output
    is rounded, per element (see below)."""
    n = k.shape[0]
    out, lse, bound = np.zeros((len(q), v.shape[1])), np.full(len(q), -np.inf), np.zeros((len(q), v.shape[1]))
    for r, p in enumerate(pos):
        if p < 0:
            continue
        at = np.arange(n)
        see = np.ones(n, bool)
        if causal:
            see = (at <= p) & (at > (p - window if window else -1))
        if pages is not None:
            see &= np.isin(at // page, pages[r])
        at = at[see]
        if not len(at):
            continue
        x = (k[at] @ q[r]) * scale
        top = x.max()
        w = np.exp(x - top)
        total = w.sum()
        w = w / total
        out[r], lse[r] = w @ v[at], top + np.log(total)
        # The weights may be rounded to fp16 once (2^-11 relative, 2^-25 of the largest weighted magnitude where
        # they are subnormal); fp32 arithmetic of the scores moves a weight by |x| log2(e) * 2^-22 relative at
        # most, the base-2 exponential by 2^-22, and the fp32 sums by n * 2^-24 of their absolute terms.
        weight = w @ np.abs(v[at])
        rel = 2.0 ** -11 + (np.abs(x).max() * 1.5 + 4) * 2.0 ** -22 + 2 * len(at) * 2.0 ** -24
        peak = (w * 127 * vs[at]).max()
        bound[r] = rel * weight + len(at) * 2.0 ** -25 * peak
    return out, lse, bound


HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 1e-40}


def check(got, out, bound, dtype):
    """got (torch) against the float64 result, within the bound and one rounding to dtype."""
    got = got.double().cpu().numpy()
    limit = bound + HALF_ULP[dtype] * (np.abs(out) + bound) + SMALLEST[dtype]
    bad = ~(np.abs(got - out) <= limit)
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - out).max()), float(limit.max()),
                           np.argwhere(bad)[:4].tolist())


def select(q, scales_k, sums, pos, n, page, group):
    """Page choice of one (sequence, kv head): q fp32 [group, T, D], sums int [P, D], scales_k fp32 [P]."""
    t = q.shape[1]
    out = np.full((t, n), -1, np.int32)
    s = np.maximum(np.abs(q).max(-1) * INV127, TINY).astype(np.float32)
    q8 = np.rint(q * (np.float32(1.0) / s)[..., None]).astype(np.int64)
    for i in range(t):
        if pos[i] < 0:
            continue
        last = pos[i] // page
        score = np.full(last, -np.inf, np.float32)
        for j in range(last):
            best = max(np.float32(int(q8[g, i] @ sums[j].astype(np.int64))) * s[g, i] for g in range(group))
            score[j] = best * scales_k[j]
        order = np.argsort(-score.astype(np.float64), kind="stable")[: n - 1]
        kept = sorted(order.tolist()) + [last]
        out[i, : len(kept)] = kept
    return out
