"""Cases of the 8-bit key/value cache: writing it, reading it back, attending over it, and attending
over the pages that a score selects.

A decoder that emits its clip piece by piece (one latent frame, a row of tokens, a single token)
attends over everything before the piece.  The cache keeps those keys and values as INT8 codes with
one fp32 scale per (page, head); the sequences of a batch share one pool of pages through a page table.

`own` false: elementary torch operations in fp32, each output rounded once.  `own` true: the calls a
user of h3vae_b200 makes.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
INV127 = float(torch.tensor(1.0, dtype=torch.float32) / 127.0)
TINY = 1e-30      # smallest scale
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _case(name, op, dtype, batch, q_heads, kv_heads, dim, page, length, tokens, **more):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "length": length, "tokens": tokens, "causal": True, "window": 0, "pages": 0,
            "ragged": False, **more}


def listed():
    return [
        # one token appended per step, 32 streams: pages that end, start and are half full
        _case("write_step", "write", "fp16", 32, 16, 16, 64, 64, 5120, 1, ragged=True),
        # a whole decoder tile (5 frames of 32 x 32 tokens) stored after an odd number of earlier tokens
        _case("write_tile", "write", "fp16", 4, 16, 16, 64, 64, 6917, 5120),
        # a grouped-head prompt in bf16, four sequences of different lengths
        _case("write_prompt", "write", "bf16", 4, 32, 8, 128, 128, 16384, 16001, ragged=True),
        # the context handed back to a dense consumer: one latent frame's worth, and a long one
        _case("read_frame", "read", "fp16", 1, 16, 16, 64, 64, 1797, 0),
        _case("read_long", "read", "bf16", 8, 32, 8, 128, 64, 32768, 0, ragged=True),
        # single tokens: the smallest call (one short stream) and a batch of long grouped-head streams
        _case("step_short", "attend", "fp16", 1, 16, 16, 64, 64, 1797, 1),
        _case("step_long", "attend", "bf16", 16, 32, 8, 128, 64, 32768, 1, ragged=True),
        # one latent frame (1024 tokens, every token sees the whole frame) over five frames of context
        _case("frame_chunk", "attend", "fp16", 2, 16, 16, 64, 64, 5120, 1024, causal=False),
        # a causal grouped-head prompt, its length a multiple of nothing
        _case("prompt_causal", "attend", "bf16", 2, 32, 8, 128, 128, 8101, 8101),
        # 32 of 2048 pages per query: one long stream, a batch of grouped-head streams, a piece of 17 tokens
        _case("sparse_step", "sparse", "fp16", 1, 16, 16, 64, 64, 131072, 1, pages=32),
        _case("sparse_batch", "sparse", "bf16", 16, 32, 8, 128, 64, 32768, 1, pages=48, ragged=True),
        _case("sparse_piece", "sparse", "fp16", 2, 16, 16, 64, 64, 20001, 17, pages=24),
    ]


def _logint(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(max(v, lo), hi)
    return v + 1 if v == 3 * 1024 else v


def _cost(case):
    """What a case asks of the plain form: score values and cache values, the largest listed ones' at most."""
    t, n = max(case["tokens"], 1), case["length"]
    if case["op"] == "sparse":
        n = min(n, case["pages"] * case["page"]) * case["dim"] // 16 + n // case["page"]
    scores = case["batch"] * case["q_heads"] * t * n * case["dim"] / 128 if case["op"] in ("attend", "sparse") else 0
    return scores, case["batch"] * case["kv_heads"] * case["length"] * case["dim"]


def draw(rng):
    most = [max(c) for c in zip(*(_cost(c) for c in listed()))]
    while True:
        op = rng.choice(["write", "read", "attend", "attend", "sparse"])
        kv, group = rng.choice([(16, 1), (32, 1), (8, 4), (4, 8), (1, 16), (2, 7), (5, 2)])
        dim = rng.choice([64, 64, 128])
        page = rng.choice([16, 32, 64, 128])
        batch = _logint(rng, 1, 32)
        length = _logint(rng, 8, 131072 if op == "sparse" else 32768)
        tokens, pages = 0, 0
        if op in ("write", "attend"):
            tokens = rng.choice([1, 1, _logint(rng, 2, 96), _logint(rng, 97, 8192)])
        if op == "sparse":
            tokens, pages = rng.choice([1, 1, _logint(rng, 2, 24)]), _logint(rng, 1, 64)
        if tokens > length:
            continue
        causal = op != "attend" or rng.random() < 0.7
        case = _case("", op, rng.choice(["fp16", "bf16"]), batch, kv * group, kv, dim, page, length, tokens,
                     pages=pages, causal=causal, ragged=rng.random() < 0.5,
                     window=_logint(rng, 1, length) if op == "attend" and causal and rng.random() < 0.3 else 0)
        del case["name"]
        if all(c <= m for c, m in zip(_cost(case), most)) and kv * group * dim != 3 * 1024:
            return case


def _lengths(case):
    """Tokens in the cache per sequence after the call, and how many of them the call brings."""
    b, n, t = case["batch"], case["length"], case["tokens"]
    if not case["ragged"]:
        return [n] * b, [t] * b
    part = [1.0 - 0.8 * ((i * 0.6180339887) % 1.0) for i in range(b)]
    lens = [max(1, int(n * p)) for p in part]
    counts = [min(t, m) if case["op"] != "write" else max(1, min(m, int(t * p + 0.5))) for m, p in zip(lens, part)]
    return lens, (counts if t > 1 else [min(t, m) for m in lens])


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _unit(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    b, h, d, ps, t = case["batch"], case["kv_heads"], case["dim"], case["page"], case["tokens"]
    lens, counts = _lengths(case)
    held = [n - c if case["op"] == "write" else n for n, c in zip(lens, counts)]   # in the cache before the call
    width = max(-(-n // ps) for n in lens) + 1
    total = sum(-(-n // ps) for n in lens) + 3
    order = torch.randperm(total, generator=gen, device=DEV).tolist()
    table = [[-1] * width for _ in range(b)]
    s = {"case": case, "lens": lens, "counts": counts, "held": held}
    cache = {
        "k": torch.zeros(total, h, ps, d, dtype=torch.int8, device=DEV),
        "v": torch.zeros(total, h, ps, d, dtype=torch.int8, device=DEV),
        "k_scale": torch.zeros(total, h, device=DEV), "v_scale": torch.zeros(total, h, device=DEV),
        "k_sum": torch.zeros(total, h, d, dtype=torch.int16, device=DEV),
    }
    q_centre = []
    for i, n in enumerate(lens):
        np_ = -(-n // ps)
        pages = [order.pop() for _ in range(np_)]
        table[i][:np_] = pages
        pages = torch.tensor(pages, device=DEV)
        # keys of one page resemble one another (neighbouring tokens), values are wider and off centre
        centre = rnd(np_, h, 1, d)
        valid = (torch.arange(np_ * ps, device=DEV) < held[i]).view(np_, 1, ps, 1)
        for name, x in (("k", _unit(0.6 * centre + 0.8 * rnd(np_, h, ps, d))), ("v", 0.7 * rnd(np_, h, ps, d) + 0.1)):
            scale = ((x * valid).abs().amax((2, 3)) * INV127).clamp_min(TINY)
            codes = torch.round(x / scale[:, :, None, None]).clamp_(-127, 127).to(torch.int8)
            cache[name][pages], cache[name + "_scale"][pages] = codes, scale
        full = torch.arange(np_, device=DEV) * ps + ps <= held[i]
        sums = cache["k"][pages].sum(2, dtype=torch.int32) * full[:, None, None]
        cache["k_sum"][pages] = sums.to(torch.int16)
        q_centre.append(centre[torch.randint(np_, (max(t, 1),), generator=gen, device=DEV), :, 0].transpose(0, 1))
    s["table"] = torch.tensor(table, dtype=torch.int32, device=DEV)
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["start"] = torch.tensor(held, dtype=torch.int32, device=DEV)
    s["count"] = torch.tensor(counts, dtype=torch.int32, device=DEV)
    ty, g = TYPES[case["dtype"]], case["q_heads"] // h
    if case["op"] == "write":
        # tokens as a fused projection leaves them: [B, T, H, D] storage seen as [B, H, T, D]
        s["new_k"] = _unit(rnd(b, t, h, d)).to(ty).transpose(1, 2)
        s["new_v"] = (0.7 * rnd(b, t, h, d) + 0.1).to(ty).transpose(1, 2)
        # a first page, and the page read back with it, starts where the page of the first new token does
        s["first"] = torch.tensor([x - x % ps for x in held], dtype=torch.int32, device=DEV)
        s["back"] = max(n - (x - x % ps) for n, x in zip(lens, held))
    if case["op"] in ("attend", "sparse"):
        q = _unit(torch.stack(q_centre)[:, :, None] * 0.7 + rnd(b, h, g, t, d))
        s["q"] = q.reshape(b, h * g, t, d).to(ty)
        s["scale"] = d ** -0.5
    s["cache"] = cache
    if own:
        root = str(Path(__file__).resolve().parents[1] / "comfyui-h3vae-pyopt_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        from h3vae_b200 import kernels
        from h3vae_b200.kv_cache import KVCacheI8
        s["lib"], s["cache"] = kernels, KVCacheI8(**cache)
        # a uniform batch passes no counts
        s["count"] = s["count"] if any(c != t for c in counts) else None
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    case, lib, cache = s["case"], s["lib"], s["cache"]
    ty = TYPES[case["dtype"]]
    if case["op"] == "write":
        lib.kv_write_i8(cache, s["table"], s["start"], s["new_k"], s["new_v"], counts=s["count"])
        k, v = lib.kv_read_i8(cache, s["table"], s["lengths"], s["back"], start=s["first"], dtype=ty)
        return {"k": k, "v": v, "k_scale": cache.k_scale, "v_scale": cache.v_scale, "k_sum": cache.k_sum}
    if case["op"] == "read":
        k, v = lib.kv_read_i8(cache, s["table"], s["lengths"], case["length"], dtype=ty)
        return {"k": k, "v": v}
    if case["op"] == "attend":
        return lib.attention_kv_i8(s["q"], cache, s["table"], s["lengths"], s["scale"], counts=s["count"],
                                   causal=case["causal"], window=case["window"])
    pages = lib.kv_select_i8(s["q"], cache, s["table"], s["lengths"], case["pages"], counts=s["count"])
    out = lib.attention_kv_i8(s["q"], cache, s["table"], s["lengths"], s["scale"], counts=s["count"], selected=pages)
    return {"out": out, "pages": pages}


def _run_plain(s):
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "sparse": _plain_sparse}[
        s["case"]["op"]](s)


def _tokens(s, name, table):
    """The values [B, H, N, D] in fp32 that the pages of `table` [B, P] hold."""
    c = s["cache"]
    at = table.clamp_min(0).long()
    x = c[name][at].float() * c[name + "_scale"][at][..., None, None]     # [B, P, H, page, D]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_read(s, start=None, n=None):
    case, ps = s["case"], s["case"]["page"]
    n = case["length"] if n is None else n
    first = torch.zeros_like(s["lengths"]) if start is None else start
    slots = first[:, None] // ps + torch.arange(-(-n // ps) + 1, device=DEV)
    table = torch.gather(s["table"], 1, slots.clamp_max(s["table"].shape[1] - 1).long())
    at = torch.arange(n, device=DEV)
    there = (at < (s["lengths"] - first)[:, None])[:, None, :, None]      # every `first` begins a page
    return {x: torch.where(there, _tokens(s, x, table)[:, :, :n], 0.0).to(TYPES[case["dtype"]]) for x in "kv"}


def _plain_write(s):
    case, cache, ps = s["case"], s["cache"], s["case"]["page"]
    start, count, t = s["start"], s["count"], s["case"]["tokens"]
    touched = (t + ps - 2) // ps + 1
    slots = start[:, None] // ps + torch.arange(touched, device=DEV)             # page of each sequence
    pos = slots[..., None] * ps + torch.arange(ps, device=DEV)                   # [B, P, page]
    new = (pos >= start[:, None, None]) & (pos < (start + count)[:, None, None])
    here = new.any(-1)
    table = torch.gather(s["table"], 1, slots.clamp_max(s["table"].shape[1] - 1).long()).long()
    src = (pos - start[:, None, None]).clamp(0, t - 1)
    rows = torch.arange(case["batch"], device=DEV)[:, None, None]
    for name in "kv":
        x = s["new_" + name].transpose(1, 2)[rows, src].float()                  # [B, P, page, H, D]
        x = torch.where(new[..., None, None], x, 0.0).transpose(2, 3)            # [B, P, H, page, D]
        scale = (x.abs().amax((3, 4)) * INV127).clamp_min(TINY)
        codes, had = cache[name][table.clamp_min(0)].float(), cache[name + "_scale"][table.clamp_min(0)]
        old = (slots * ps < start[:, None])[..., None]                           # the page held tokens before
        scale = torch.where(old, torch.maximum(scale, had), scale)
        codes = torch.where((old & (scale > had))[..., None, None],
                            torch.round(codes * (had / scale)[..., None, None]).clamp(-127, 127), codes)
        fresh = torch.round(x * (1.0 / scale)[..., None, None]).clamp(-127, 127)
        keep = (pos < start[:, None, None])[:, :, None, :, None]
        codes = torch.where(new[:, :, None, :, None], fresh, torch.where(keep, codes, cache[name][
            table.clamp_min(0)].float())).to(torch.int8)
        cache[name][table[here]] = codes[here]
        cache[name + "_scale"][table[here]] = scale[here]
    done = here & ((slots + 1) * ps <= (start + count)[:, None])
    cache["k_sum"][table[done]] = cache["k"][table[done]].sum(2, dtype=torch.int32).to(torch.int16)
    back = _plain_read(s, s["first"], s["back"])
    return {**back, "k_scale": cache["k_scale"], "v_scale": cache["v_scale"], "k_sum": cache["k_sum"]}


def _softmax_times(scores, seen, v):
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    return (scores @ v) / scores.sum(-1, keepdim=True).clamp_min(1e-37)


def _places(s):
    """Position of each query token [B, T], -1 where there is none."""
    i = torch.arange(s["case"]["tokens"], device=DEV)
    pos = (s["lengths"] - s["count"])[:, None] + i
    return torch.where(i < s["count"][:, None], pos, -1)


def _plain_attend(s):
    case, q = s["case"], s["q"]
    b, hq, t, d = q.shape
    h, g = case["kv_heads"], hq // case["kv_heads"]
    k, v = (_tokens(s, x, s["table"]) for x in "kv")
    pos = _places(s)[:, :, None]
    at = torch.arange(k.shape[2], device=DEV)
    seen = (at < s["lengths"][:, None, None]) & (pos >= 0)
    if case["causal"]:
        seen = seen & (at <= pos)
        if case["window"]:
            seen = seen & (at > pos - case["window"])
    q = q.float().view(b, h, g, t, d)
    outs = []
    for i in range(0, b, max(1, (1 << 31) // max(1, hq * t * k.shape[2]))):       # up to 8 GB of scores at once
        j = slice(i, i + max(1, (1 << 31) // max(1, hq * t * k.shape[2])))
        scores = q[j].flatten(2, 3) @ k[j].transpose(2, 3)
        n = scores.shape[0]
        scores = scores.mul_(s["scale"]).view(n, h, g, t, -1)
        outs.append(_softmax_times(scores, seen[j][:, None, None], v[j][:, :, None]).view(n, hq, t, d))
    return torch.cat(outs).to(s["q"].dtype)


def _plain_select(s):
    """Pages [B, H, T, n]: the last visible one and the best of those before it, ascending, -1 where none is left."""
    case, c, ps, n = s["case"], s["cache"], s["case"]["page"], s["case"]["pages"]
    q = s["q"].float()
    b, hq, t, d = q.shape
    h, g = case["kv_heads"], hq // case["kv_heads"]
    scale = (q.abs().amax(-1, keepdim=True) * INV127).clamp_min(TINY)
    codes = torch.round(q * (1.0 / scale)).clamp(-127, 127).view(b, h, g * t, d)
    at = s["table"].clamp_min(0).long()
    sums = c["k_sum"][at].transpose(1, 2).int()                                   # [B, H, P, D]
    # whole numbers up to 2^28: two products that fp32 holds exactly
    low = sums & 127
    dots = (codes @ low.float().transpose(2, 3)).int() + 128 * (codes @ (sums >> 7).float().transpose(2, 3)).int()
    score = (dots.float().view(b, h, g, t, -1) * scale.view(b, h, g, t, 1)).amax(2)
    score = score * c["k_scale"][at].transpose(1, 2)[:, :, None]
    pos = _places(s)
    last = torch.where(pos >= 0, pos // ps, -1)[:, None, :, None]
    slot = torch.arange(score.shape[-1], device=DEV)
    score = torch.where(slot < last, score, -math.inf)
    score = torch.where(slot == last, math.inf, score)
    best, index = torch.sort(score, dim=-1, descending=True, stable=True)
    best, index = best[..., :n], index[..., :n]
    index = torch.where(best == -math.inf, score.shape[-1], index).sort(-1).values
    pages = torch.full((b, h, t, n), -1, dtype=torch.int32, device=DEV)
    pages[..., : index.shape[-1]] = torch.where(index == score.shape[-1], -1, index).int()
    return pages


def _plain_sparse(s):
    case, c, ps = s["case"], s["cache"], s["case"]["page"]
    pages = _plain_select(s)
    b, h, t, n = pages.shape
    g, d = case["q_heads"] // h, case["dim"]
    at = torch.gather(s["table"][:, None, None].expand(b, h, t, -1), 3, pages.clamp_min(0).long()).clamp_min(0).long()
    heads = torch.arange(h, device=DEV)[None, :, None, None]
    k, v = ((c[x][at, heads].float() * c[x + "_scale"][at, heads][..., None, None]).flatten(3, 4) for x in "kv")
    where = (pages[..., None] * ps + torch.arange(ps, device=DEV)).flatten(3)     # [B, H, T, n * page]
    seen = (pages >= 0).repeat_interleave(ps, -1) & (where <= _places(s)[:, None, :, None])
    q = s["q"].float().view(b, h, g, t, d).transpose(2, 3)                        # [B, H, T, g, D]
    out = _softmax_times((q @ k.transpose(3, 4)) * s["scale"], seen[:, :, :, None], v)
    return {"out": out.transpose(2, 3).reshape(b, h * g, t, d).to(s["q"].dtype), "pages": pages}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    lens, counts = _lengths(case)
    h, hq, d, ps = case["kv_heads"], case["q_heads"], case["dim"], case["page"]
    row = 2 * h * d                                                # one token's keys and values, in codes
    if case["op"] == "read":
        return {"bytes": sum(lens) * row + case["batch"] * case["length"] * row * 2, "flops": sum(lens) * row}
    if case["op"] == "write":
        back = [n - (n - c - (n - c) % ps) for n, c in zip(lens, counts)]
        moved = sum(c * row * 3 for c in counts) + sum(x * row for x in back) + case["batch"] * max(back) * row * 2
        return {"bytes": moved, "flops": sum(counts) * row * 4 + sum(back) * row}
    q_out = sum(counts) * hq * d * 2 * 2
    pairs = bytes_ = 0
    for n, c in zip(lens, counts):
        if case["op"] == "sparse":
            kept = [min(case["pages"], (n - c + i) // ps + 1) for i in range(c)]
            full = n // ps
            pairs += sum(kept) * ps
            bytes_ += min(sum(kept) * ps, n) * row + full * h * d * 2
            pairs += full * c // 2
        elif case["causal"]:
            w = case["window"] or n
            pairs += sum(min(n - c + i + 1, w) for i in range(c))
            bytes_ += min(n, w + c - 1) * row
        else:
            pairs += n * c
            bytes_ += n * row
    return {"bytes": bytes_ + q_out, "flops": 4 * hq * d * pairs}


# ---------------------------------------------------------------------------
# The same from the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"write": _exact_write, "read": _exact_read, "attend": _exact_attend, "sparse": _exact_sparse}[
        case["op"]](s)


def _exact_tokens(s, i, name, head):
    """float64 [N, D]: what sequence i's pages hold for one head."""
    at = [p for p in s["table"][i].tolist() if p >= 0]
    c = s["cache"]
    return (c[name][at, head].double() * c[name + "_scale"][at, head].double()[:, None, None]).flatten(0, 1)


def _exact_read(s):
    case = s["case"]
    out = {x: torch.zeros(case["batch"], case["kv_heads"], case["length"], case["dim"], dtype=torch.float64,
                          device=DEV) for x in "kv"}
    for x in "kv":
        for i, n in enumerate(s["lens"]):
            for head in range(case["kv_heads"]):
                out[x][i, head, :n] = _exact_tokens(s, i, x, head)[:n]
    return out


def _exact_write(s):
    case, ps = s["case"], s["case"]["page"]
    got = {"k_sum": None}
    for name in "kv":
        scales = s["cache"][name + "_scale"].double().clone()
        dense = torch.zeros(case["batch"], case["kv_heads"], s["back"], case["dim"], dtype=torch.float64, device=DEV)
        for i, (had, count) in enumerate(zip(s["held"], s["counts"])):
            first, end = had - had % ps, had + count
            for slot in range(first // ps, -(-end // ps)):
                page, lo, hi = int(s["table"][i, slot]), max(had, slot * ps), min(end, slot * ps + ps)
                x = s["new_" + name][i, :, lo - had: hi - had].double()
                scale = (x.abs().amax((1, 2)) / 127).clamp_min(TINY)
                if lo > slot * ps:
                    before = scales[page].clone()
                    scale = torch.maximum(scale, before)
                    codes = s["cache"][name][page, :, : lo - slot * ps].double() * (before / scale)[:, None, None]
                    dense[i, :, slot * ps - first: lo - first] = codes.round() * scale[:, None, None]
                dense[i, :, lo - first: hi - first] = (x / scale[:, None, None]).round() * scale[:, None, None]
                scales[page] = scale
        got[name], got[name + "_scale"] = dense, scales
    return got


def _exact_rows(q, k, v, seen, scale):
    """softmax(q k^T * scale) v in float64; a row that sees nothing is zero."""
    w = (q.double() @ k.T) * scale
    w = torch.where(seen, w, -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp_min(-1e300))
    total = w.sum(-1, keepdim=True)
    return torch.where(total > 0, (w @ v) / torch.where(total > 0, total, 1.0), 0.0)


def _exact_attend(s):
    case, q = s["case"], s["q"]
    h, g = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    if 4 * case["dim"] * case["q_heads"] * sum(n * max(c, 1) for n, c in zip(s["lens"], s["counts"])) > 6e12:
        return None
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for i, (n, c) in enumerate(zip(s["lens"], s["counts"])):
        pos = torch.arange(n - c, n, device=DEV)[:, None]
        at = torch.arange(n, device=DEV)
        seen = torch.ones(c, n, dtype=torch.bool, device=DEV)
        if case["causal"]:
            seen = (at <= pos) & (at > (pos - case["window"] if case["window"] else -1))
        for head in range(h):
            k, v = (_exact_tokens(s, i, x, head)[:n] for x in "kv")
            for j in range(head * g, head * g + g):
                out[i, j, :c] = _exact_rows(q[i, j, :c], k, v, seen, s["scale"])
    return out


def _exact_sparse(s):
    case, q, ps = s["case"], s["q"], s["case"]["page"]
    h, g, t, n = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["tokens"], case["pages"]
    if case["batch"] * h * t > 4096:
        return None
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    pages = torch.full((case["batch"], h, t, n), -1, dtype=torch.int64, device=DEV)
    for i, (total, c) in enumerate(zip(s["lens"], s["counts"])):
        at = [p for p in s["table"][i].tolist() if p >= 0]
        for head in range(h):
            k, v = (_exact_tokens(s, i, x, head) for x in "kv")
            sums = s["cache"]["k_sum"][at, head].double()
            for j in range(c):
                place = total - c + j
                last = place // ps
                rows = q[i, head * g: head * g + g, j].float()
                # the score is defined on 8-bit queries, whole-number products and fp32 factors
                unit = (rows.abs().amax(-1, keepdim=True) * INV127).clamp_min(TINY)
                whole = torch.round(rows * (1.0 / unit)).clamp(-127, 127).double() @ sums[:last].T
                score = (whole.float() * unit).amax(0) * s["cache"]["k_scale"][at[:last], head]
                best = score.double().sort(descending=True, stable=True).indices[: n - 1]
                kept = torch.cat([best.sort().values, torch.tensor([last], device=DEV)])
                pages[i, head, j, : kept.numel()] = kept
                where = (kept[:, None] * ps + torch.arange(ps, device=DEV)).flatten()
                out[i, head * g: head * g + g, j] = _exact_rows(rows, k[where], v[where], where <= place, s["scale"])
    return {"out": out, "pages": pages}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c.get("name", "drawn"), work(c), c)
