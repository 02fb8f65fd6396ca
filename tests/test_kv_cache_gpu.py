"""The paged INT8 key/value cache on the B200 against plain restatements (kv_reference): codes, scales, sums and
page choices bit for bit, attention against float64 within derived bounds."""
import numpy as np
import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(rng, lens, page, spare=3, width=None):
    """Scattered pages for every sequence, -1 past its end, and the pool's size."""
    need = [-(-max(n, 1) // page) for n in lens]
    order = rng.permutation(sum(need) + spare).tolist()
    rows = [[order.pop() for _ in range(n)] for n in need]
    width = width or max(need) + 1
    return rows, _i32([r + [-1] * (width - len(r)) for r in rows]), sum(need) + spare


def _wide(table, pages=20000):
    """The same table in rows of many more pages: calls are planned for what a table could hold, so small lengths
    then run on the kernels for long sequences (parts joined by a second kernel, tensor-core row tiles)."""
    return torch.nn.functional.pad(table, (0, pages - table.shape[1]), value=-1).contiguous()


def _rounded(x, dtype):
    """fp32 numpy of x rounded to dtype."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TYPES[dtype]).float().numpy()


def _same(cache, ref):
    for name, got in (("k", cache.k), ("v", cache.v), ("k_sum", cache.k_sum)):
        want = ref.k_sum if name == "k_sum" else ref.code[name]
        assert np.array_equal(got.cpu().numpy(), want), (name, np.argwhere(got.cpu().numpy() != want)[:4])
    for name, got in (("k", cache.k_scale), ("v", cache.v_scale)):
        assert np.array_equal(got.cpu().numpy(), ref.scale[name], equal_nan=True), name


def _filled(rng, lens, heads, dim, page, v_spread=None, garbage=True):
    """A reference cache holding `lens` tokens (scattered pages), with garbage in slots no token uses."""
    rows, table, pages = _tables(rng, lens, page)
    ref = R.CacheRef(pages, heads, dim, page)
    for row, n in zip(rows, lens):
        k = rng.standard_normal((heads, n, dim)).astype(np.float32)
        v = rng.standard_normal((heads, n, dim)).astype(np.float32)
        if v_spread is not None:
            v *= (10.0 ** rng.uniform(*v_spread, (1, -(-n // page), 1))).repeat(page, 1)[:, :n].astype(np.float32)
        ref.write(row, 0, n, k, v)
        if garbage and n % page:
            ref.code["k"][row[-1], :, n % page:] = rng.integers(-127, 128, (heads, page - n % page, dim))
            ref.code["v"][row[-1], :, n % page:] = rng.integers(-127, 128, (heads, page - n % page, dim))
    used = {p for row, n in zip(rows, lens) for p in row[: -(-n // page)]}
    for p in set(range(pages)) - used if garbage else ():
        ref.scale["k"][p] = ref.scale["v"][p] = np.nan
    return ref, rows, table


def _cache(ref):
    from h3vae_b200.kv_cache import KVCacheI8
    return KVCacheI8(**ref.tensors())


# ---------------------------------------------------------------------------
# Writing
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,page,dim,heads", [("fp16", 64, 64, 3), ("bf16", 128, 128, 2), ("fp16", 16, 128, 1),
                                                  ("fp32", 32, 64, 5), ("bf16", 16, 64, 2), ("fp16", 128, 64, 2)])
@pytest.mark.parametrize("layout", ["bhtd", "bthd", "odd"])
def test_write_steps(cuda_lib, dtype, page, dim, heads, layout):
    """Pieces of 1..130 tokens appended (ragged, some empty), growing so that pages requantise."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(page + dim)
    batch, cap = 3, 400
    rows, table, pages = _tables(rng, [cap] * batch, page)
    ref = R.CacheRef(pages, heads, dim, page)
    cache = _cache(ref)
    at = [0, 5, page - 1]
    for step, t in enumerate([1, 1, page, 130, 1, 7, 1]):
        counts = [t, max(0, t - 1 - step), t]
        k, v = (_rounded(rng.standard_normal((batch, heads, t, dim)) * (1 + step), dtype) for _ in "kv")
        tensors = []
        for x in (k, v):
            x = torch.from_numpy(x).to(TYPES[dtype])
            if layout == "bthd":
                x = x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
            elif layout == "odd":   # rows that start on no 16-byte boundary
                wide = torch.zeros(batch, heads, t, dim + 3, dtype=x.dtype)
                wide[..., 1:dim + 1] = x
                x = wide.cuda()[..., 1:dim + 1]
            tensors.append(x.cuda())
        for b in range(batch):
            if step == 0 and at[b]:   # earlier tokens that the sequence starts with
                first = _rounded(rng.standard_normal((2, heads, at[b], dim)), dtype)
                ref.write(rows[b], 0, at[b], *first)
                one = [torch.from_numpy(x[None]).to(TYPES[dtype]).cuda() for x in first]
                K.kv_write_i8(cache, table[b: b + 1], _i32([0]), *one)
            ref.write(rows[b], at[b], counts[b], k[b, :, : counts[b]], v[b, :, : counts[b]])
        K.kv_write_i8(cache, table, _i32(at), *tensors, counts=_i32(counts) if counts != [t] * batch else None)
        _same(cache, ref)
        at = [x + c for x, c in zip(at, counts)]
    # within half a step of what came last: the newest token of each sequence
    for b in range(batch):
        if counts[b]:
            got = ref.dense("k", rows[b], at[b])[:, -1]
            s = ref.scale["k"][rows[b][(at[b] - 1) // page]]
            assert (np.abs(got - k[b, :, counts[b] - 1]) <= s[:, None] * (0.5 + 2.0 ** -15)).all()


def test_write_replaces_and_rewinds(cuda_lib):
    """A start before the old end replaces tokens; slot 0 starts the page's scale anew."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(1)
    rows, table, pages = _tables(rng, [96], 32)
    ref = R.CacheRef(pages, 2, 64, 32)
    cache = _cache(ref)
    for start, n, size in ((0, 70, 8.0), (40, 30, 1.0), (64, 32, 0.5), (0, 1, 0.1), (1, 31, 0.2), (0, 0, 1.0)):
        k, v = (_rounded(rng.standard_normal((1, 2, n, 64)) * size, "fp16") for _ in "kv")
        ref.write(rows[0], start, n, k[0], v[0])
        K.kv_write_i8(cache, table, _i32([start]), *(torch.from_numpy(x).half().cuda() for x in (k, v)))
        _same(cache, ref)


def test_write_zeros_nan_and_infinity(cuda_lib):
    """Zero pages take the smallest scale; a page that takes a NaN or infinity reads NaN until slot 0 is rewritten,
    and only for its head."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(2)
    rows, table, pages = _tables(rng, [64], 16)
    ref = R.CacheRef(pages, 2, 64, 16)
    cache = _cache(ref)
    k, v = (_rounded(rng.standard_normal((1, 2, 48, 64)), "fp16") for _ in "kv")
    k[0, :, 0:16] = 0.0
    k[0, 1, 20, 3] = np.nan
    v[0, 0, 40, 9] = -np.inf
    v[0, 1, 47] = 65504.0
    for start, n in ((0, 48), (24, 4), (16, 16), (32, 16)):
        part = [x[:, :, start: start + n].copy() for x in (k, v)]
        if (start, n) != (0, 48):
            part = [np.nan_to_num(x, nan=0.5, posinf=1.0, neginf=-1.0) for x in part]
        ref.write(rows[0], start, n, part[0][0], part[1][0])
        K.kv_write_i8(cache, table, _i32([start]), *(torch.from_numpy(x).half().cuda() for x in part))
        for name, got in (("k", cache.k_scale), ("v", cache.v_scale)):
            assert np.array_equal(got.cpu().numpy(), ref.scale[name], equal_nan=True)
        for name, got in (("k", cache.k), ("v", cache.v)):
            fine = ~np.isnan(ref.scale[name])
            assert np.array_equal(got.cpu().numpy()[fine], ref.code[name][fine])
    assert np.isfinite(ref.scale["k"]).all() and np.isfinite(ref.scale["v"]).all()
    assert ref.scale["k"][rows[0][0], 0] == R.TINY


def test_bad_pages_are_not_touched(cuda_lib):
    """Page numbers outside the pool and positions outside the table: skipped, and bit 3 of the error word."""
    from h3vae_b200 import _lib, kernels as K
    rng = np.random.default_rng(3)
    ref, rows, table = _filled(rng, [40, 40], 2, 64, 16, garbage=False)
    cache = _cache(ref)
    bad = table.clone()
    bad[0, 1], bad[1, 0] = cache.num_pages, -7
    assert _lib.device_error() == 0
    k, v = K.kv_read_i8(cache, bad, _i32([40, 40]), 40)
    assert _lib.device_error() == 8
    want = [torch.from_numpy(np.stack([ref.dense(n, r, 40) for r in rows])).cuda() for n in "kv"]
    for got, w in zip((k, v), want):
        w = w.float().half()
        w[0, :, 16:32] = 0
        w[1, :, :16] = 0
        assert torch.equal(got, w)
    before = [x.clone() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_sum)]
    x = torch.ones(2, 2, 16, 64, device="cuda", dtype=torch.float16)
    K.kv_write_i8(cache, bad, _i32([16, 0]), x, x)                # both land on a bad page number
    K.kv_write_i8(cache, table, _i32([16 * table.shape[1], -1]), x, x)   # past the table, before it
    assert _lib.device_error() == 8
    for a, b in zip(before, (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_sum)):
        assert torch.equal(a, b)
    # attention leaves the bad pages out; a length past the table counts as the table's end
    q = torch.randn(2, 2, 1, 64, device="cuda").half()
    out = K.attention_kv_i8(q, cache, bad, _i32([40, 40]), 0.125)
    assert _lib.device_error() == 8
    for b, keep in ((0, list(range(16)) + list(range(32, 40))), (1, list(range(16, 40)))):
        for h in range(2):
            kk, vv = (ref.dense(n, rows[b], 40)[h][keep] for n in "kv")
            vs = ref.scale["v"][rows[b], h].astype(np.float64).repeat(16)[keep]
            o, _, bound = R.attend(q[b, h].double().cpu().numpy(), kk, vv, vs, [len(keep) - 1], 0.125)
            R.check(out[b, h], o, bound, torch.float16)
    out = K.attention_kv_i8(q, cache, table[:, :2].contiguous(), _i32([2 ** 31 - 1, 32]), 0.125)
    same = K.attention_kv_i8(q, cache, table[:, :2].contiguous(), _i32([32, 32]), 0.125)
    assert _lib.device_error() == 8 and torch.equal(out, same)
    sel = _i32([[[[0, 99, 1]], [[1, 0, -1]]], [[[0, 1, 2]], [[2 ** 31 - 1, 1, 0]]]])
    out = K.attention_kv_i8(q, cache, table, _i32([40, 40]), 0.125, selected=sel)
    assert torch.isfinite(out).all()
    _lib.device_error()


# ---------------------------------------------------------------------------
# Reading
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128), (128, 64)])
def test_read(cuda_lib, dtype, page, dim):
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(dim)
    lens = [0, 1, page, 333]
    ref, rows, table = _filled(rng, lens, 3, dim, page)
    cache = _cache(ref)
    for start, n in (([0, 0, 0, 0], 340), ([0, 1, page - 1, 7], 129), ([5, 0, 0, 332], 1), ([0, 0, 0, 0], 0)):
        k, v = K.kv_read_i8(cache, table, _i32(lens), n, start=_i32(start), dtype=TYPES[dtype])
        assert k.shape == v.shape == (4, 3, n, dim) and k.dtype == TYPES[dtype]
        for name, got in (("k", k), ("v", v)):
            want = np.zeros((4, 3, n, dim), np.float32)
            for b, ln in enumerate(lens):
                codes = ref.code[name][rows[b]].astype(np.float32) * ref.scale[name][rows[b]][..., None, None]
                x = np.moveaxis(codes, 0, 1).reshape(3, -1, dim)[:, start[b]: min(ln, start[b] + n)]
                want[b, :, : x.shape[1]] = x
            assert torch.equal(got.cpu(), torch.from_numpy(want).to(TYPES[dtype]))
    if dtype == "fp16":
        k0, _ = K.kv_read_i8(cache, table, _i32(lens), 340)
        k1, _ = K.kv_read_i8(cache, table, _i32(lens), 340, start=_i32([0] * 4))
        assert torch.equal(k0, k1)


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def _attend_all(ref, rows, q, lens, counts, scale, page, **kw):
    """float64 result, lse and bound of a whole batch; kw["selected"]: [B, H, T, n]."""
    b, hq, t, d = q.shape
    heads = ref.scale["k"].shape[1]
    g = hq // heads
    out, lse, bound = np.zeros(q.shape), np.full((b, hq, t), -np.inf), np.zeros(q.shape)
    sel = kw.pop("selected", None)
    qn = q.double().cpu().numpy()
    for i, n in enumerate(lens):
        pos = [n - counts[i] + j if j < counts[i] and n - counts[i] + j >= 0 else -1 for j in range(t)]
        with np.errstate(invalid="ignore"):
            k, v = ref.dense("k", rows[i], n), ref.dense("v", rows[i], n)
        for h in range(heads):
            vs = ref.scale["v"][rows[i], h].astype(np.float64).repeat(page)[:n]
            for j in range(h * g, h * g + g):
                pages = None if sel is None else sel[i, h]
                out[i, j], lse[i, j], bound[i, j] = R.attend(qn[i, j], k[h], v[h], vs, pos, scale, pages=pages,
                                                             page=page, **kw)
    return out, lse, bound


CASES = [
    # dtype, dim, page, kv heads, group, tokens, lens, counts, causal, window
    ("fp16", 64, 64, 4, 1, 1, [1797, 1, 0, 64], None, True, 0),
    ("bf16", 128, 64, 2, 4, 1, [700, 65, 0, 129], None, True, 0),
    ("fp16", 128, 128, 1, 16, 1, [1000, 3], None, True, 37),
    ("bf16", 64, 16, 2, 7, 1, [513, 16], None, True, 1),
    ("fp16", 64, 32, 1, 33, 2, [300, 1], None, True, 0),
    ("fp16", 64, 64, 2, 1, 5, [5, 3, 130, 64], None, True, 0),         # more queries than tokens: empty rows
    ("bf16", 64, 64, 2, 3, 17, [200, 17, 90], [17, 0, 4], True, 0),
    ("fp16", 64, 128, 2, 1, 100, [777, 100, 0], None, False, 0),
    ("fp16", 64, 16, 1, 2, 257, [257, 300], [257, 250], True, 0),
    ("bf16", 128, 32, 1, 5, 70, [411, 70], None, True, 50),
    ("bf16", 128, 64, 1, 1, 300, [300, 1000], [1, 300], True, 0),
    ("fp16", 128, 16, 1, 4, 129, [640, 129], None, False, 0),
    ("fp16", 64, 64, 1, 1, 513, [1100], None, True, 200),
    ("fp16", 64, 64, 1, 8, 40, [2500, 40], [40, 33], True, 0),
]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(cuda_lib, case, wide):
    from h3vae_b200 import kernels as K
    dtype, dim, page, heads, group, t, lens, counts, causal, window = CASES[case]
    rng = np.random.default_rng(100 + case)
    ref, rows, table = _filled(rng, lens, heads, dim, page)
    cache = _cache(ref)
    table = _wide(table) if wide else table
    batch = len(lens)
    q = torch.from_numpy(rng.standard_normal((batch, heads * group, t, dim)) * 2).to(TYPES[dtype]).cuda()
    args = dict(causal=causal, window=window)
    got, lse = K.attention_kv_i8(q, cache, table, _i32(lens), dim ** -0.5, counts=None if counts is None else
                                 _i32(counts), return_lse=True, **args)
    out, want_lse, bound = _attend_all(ref, rows, q, lens, counts or [t] * batch, dim ** -0.5, page, **args)
    R.check(got, out, bound, TYPES[dtype])
    lse = lse.double().cpu().numpy()
    assert np.array_equal(np.isinf(lse), np.isinf(want_lse))
    fine = np.isfinite(want_lse)
    assert np.abs(lse[fine] - want_lse[fine]).max(initial=0.0) <= 2.0 ** -10
    again = K.attention_kv_i8(q, cache, table, _i32(lens), dim ** -0.5, counts=None if counts is None else
                              _i32(counts), **args)
    assert torch.equal(got, again)       # the same bits on every call


@pytest.mark.parametrize("t,group", [(1, 1), (1, 12), (3, 8), (150, 1), (40, 4)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_layouts(cuda_lib, t, group, dtype, wide):
    """Transposed, interleaved and unaligned q and out give the bits of dense ones."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(5)
    lens = [310, 151]
    ref, rows, table = _filled(rng, lens, 2, 64, 64)
    cache = _cache(ref)
    table = _wide(table) if wide else table
    q = torch.from_numpy(rng.standard_normal((2, 2 * group, t, 64))).to(TYPES[dtype]).cuda()
    want = K.attention_kv_i8(q, cache, table, _i32(lens), 0.125)
    wide = torch.zeros(2, t, 2 * group, 3 * 64 + 1, dtype=q.dtype, device="cuda")
    wide[..., 65:129] = q.transpose(1, 2)
    view = wide[..., 65:129].transpose(1, 2)
    assert torch.equal(K.attention_kv_i8(view, cache, table, _i32(lens), 0.125), want)
    out = torch.full((2, 2 * group, t, 3 * 64 + 1), 7.0, dtype=q.dtype, device="cuda")
    got = K.attention_kv_i8(view, cache, table, _i32(lens), 0.125, out=out[..., 3:67])
    assert torch.equal(got, want) and (out[..., :3] == 7).all() and (out[..., 67:] == 7).all()


@pytest.mark.parametrize("t", [1, 9, 140])
@pytest.mark.parametrize("wide", [False, True])
def test_masked_places_have_no_effect(cuda_lib, t, wide):
    """NaN scales and any codes in pages and slots past what a row sees; a NaN page that some rows see makes
    exactly those rows NaN."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(6)
    lens, page = [150, 200], 16
    ref, rows, table = _filled(rng, lens, 2, 64, page)
    cache = _cache(ref)
    more = torch.cat([table, _i32([[rows[1][0]] * 3, [rows[0][0]] * 3])], 1).contiguous()   # more table than tokens
    table, more = (_wide(table), _wide(more)) if wide else (table, more)
    q = torch.from_numpy(rng.standard_normal((2, 4, t, 64))).half().cuda()
    out, _, bound = _attend_all(ref, rows, q, lens, [t, t], 0.125, page)
    R.check(K.attention_kv_i8(q, cache, more, _i32(lens), 0.125), out, bound, torch.float16)
    # the last page of sequence 0 turns NaN
    last = rows[0][149 // page]
    cache.k_scale[last] = float("nan")
    got = K.attention_kv_i8(q, cache, table, _i32(lens), 0.125)
    pos = np.array([150 - t + i for i in range(t)])
    hit = torch.from_numpy(pos // page >= 149 // page).cuda()
    assert torch.isnan(got[0][:, hit]).all()
    if (~hit).any():
        R.check(got[0][:, ~hit], out[0][:, ~hit.cpu().numpy()], bound[0][:, ~hit.cpu().numpy()], torch.float16)
    R.check(got[1], out[1], bound[1], torch.float16)
    # a V scale instead
    cache.k_scale[last] = torch.from_numpy(ref.scale["k"][last]).cuda()
    cache.v_scale[last] = float("nan")
    assert torch.isnan(K.attention_kv_i8(q, cache, table, _i32(lens), 0.125)[0][:, hit]).all()


@pytest.mark.parametrize("t,group", [(1, 2), (6, 12), (130, 2)])
@pytest.mark.parametrize("scale", [0.125, 4.0, 0.0, -0.2])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_spread_scales(cuda_lib, t, group, scale, wide):
    """V pages whose scales differ by 10^8, zero pages among them, and near one-hot rows."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(7)
    lens, page = [500, 333], 32
    ref, rows, table = _filled(rng, lens, 1, 64, page, v_spread=(-5, 3))
    for row in rows:
        ref.code["v"][row[2]] = 0
        ref.scale["v"][row[2]] = R.TINY
        ref.code["k"][row[4]] = 0
        ref.scale["k"][row[4]] = R.TINY
    cache = _cache(ref)
    q = torch.from_numpy(rng.standard_normal((2, group, t, 64))).half().cuda()
    got = K.attention_kv_i8(q, cache, _wide(table) if wide else table, _i32(lens), scale)
    out, _, bound = _attend_all(ref, rows, q, lens, [t, t], scale, page)
    R.check(got, out, bound, torch.float16)


def test_attention_bf16_wide_queries(cuda_lib):
    """bf16 queries beyond fp16's range, and tiny ones."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(8)
    ref, rows, table = _filled(rng, [200], 1, 64, 64)
    cache = _cache(ref)
    table = _wide(table)
    for size in (1e6, 1e-6, 1e-30):
        for t in (1, 130):
            q = torch.from_numpy(rng.standard_normal((1, 2, t, 64)) * size).to(torch.bfloat16).cuda()
            q[0, 1, 0] = 0
            got = K.attention_kv_i8(q, cache, table, _i32([200]), 0.125 / size if size > 1 else 0.125)
            out, _, bound = _attend_all(ref, rows, q, [200], [t], 0.125 / size if size > 1 else 0.125, 64)
            R.check(got, out, bound, torch.bfloat16)


def test_long_cache_offsets(cuda_lib):
    """Pages beyond 2^31 bytes into the pool, for every operation."""
    from h3vae_b200 import kernels as K
    from h3vae_b200.kv_cache import KVCacheI8
    heads, page, dim = 8, 128, 128
    pages = (2 ** 31) // (heads * page * dim) * 2 + 40
    cache = KVCacheI8.empty(pages, heads, dim, page)
    rng = np.random.default_rng(9)
    n = 300
    ids = [pages - 1, 3, pages - 17]
    table = _i32([ids])
    x = torch.from_numpy(rng.standard_normal((2, 1, heads, n, dim))).half().cuda()
    K.kv_write_i8(cache, table, _i32([0]), x[0], x[1])
    small = KVCacheI8.empty(3, heads, dim, page)
    K.kv_write_i8(small, _i32([[0, 1, 2]]), _i32([0]), x[0], x[1])
    assert torch.equal(cache.k[ids], small.k) and torch.equal(cache.k_sum[ids], small.k_sum)
    for a, b in zip(K.kv_read_i8(cache, table, _i32([n]), n), K.kv_read_i8(small, _i32([[0, 1, 2]]), _i32([n]), n)):
        assert torch.equal(a, b)
    for t in (1, 150):
        q = torch.from_numpy(rng.standard_normal((1, heads, t, dim))).half().cuda()
        a = K.attention_kv_i8(q, cache, table, _i32([n]), 0.1)
        assert torch.equal(a, K.attention_kv_i8(q, small, _i32([[0, 1, 2]]), _i32([n]), 0.1))
        a = K.attention_kv_i8(q, cache, _wide(table), _i32([n]), 0.1)
        assert torch.equal(a, K.attention_kv_i8(q, small, _wide(_i32([[0, 1, 2]])), _i32([n]), 0.1))
        sel = K.kv_select_i8(q, cache, table, _i32([n]), 2)
        assert torch.equal(sel, K.kv_select_i8(q, small, _i32([[0, 1, 2]]), _i32([n]), 2))
        a = K.attention_kv_i8(q, cache, table, _i32([n]), 0.1, selected=sel)
        assert torch.equal(a, K.attention_kv_i8(q, small, _i32([[0, 1, 2]]), _i32([n]), 0.1, selected=sel))


def test_attention_long_rows(cuda_lib):
    """A long stream: many splits of the keys joined, single tokens and a piece."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(10)
    lens = [20011, 64]
    ref, rows, table = _filled(rng, lens, 1, 64, 64)
    cache = _cache(ref)
    for t, group in ((1, 1), (1, 9), (70, 1)):
        q = torch.from_numpy(rng.standard_normal((2, group, t, 64)) * 3).half().cuda()
        got = K.attention_kv_i8(q, cache, table, _i32(lens), 0.125)
        counts = [t, t]
        out, _, bound = _attend_all(ref, rows, q, lens, counts, 0.125, 64)
        R.check(got, out, bound, torch.float16)


# ---------------------------------------------------------------------------
# Selection
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,dim,page,heads,group,t,lens,counts,n", [
    ("fp16", 64, 16, 2, 1, 1, [1000, 16, 0, 1], None, 7),
    ("bf16", 128, 32, 1, 4, 3, [2000, 70], None, 20),
    ("fp16", 64, 64, 1, 3, 9, [900, 400], [9, 4], 1),
    ("fp16", 64, 16, 1, 70, 2, [333], None, 5),
    ("bf16", 64, 16, 1, 1, 1, [15000], None, 400),
    ("fp16", 64, 16, 1, 2, 5, [5, 3], None, 40),
])
def test_select(cuda_lib, dtype, dim, page, heads, group, t, lens, counts, n):
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(n)
    ref, rows, table = _filled(rng, lens, heads, dim, page)
    cache = _cache(ref)
    q = torch.from_numpy(rng.standard_normal((len(lens), heads * group, t, dim))).to(TYPES[dtype]).cuda()
    got = K.kv_select_i8(q, cache, table, _i32(lens), n, counts=None if counts is None else _i32(counts))
    qn = q.float().cpu().numpy()
    for b, ln in enumerate(lens):
        c = t if counts is None else counts[b]
        pos = [ln - c + i if i < c else -1 for i in range(t)]
        for h in range(heads):
            want = R.select(qn[b, h * group: h * group + group], ref.scale["k"][rows[b], h], ref.k_sum[rows[b], h], pos,
                            n, page, group)
            assert np.array_equal(got[b, h].cpu().numpy(), want), (b, h)
    # and attention over them
    out, _, bound = _attend_all(ref, rows, q, lens, counts or [t] * len(lens), dim ** -0.5, page,
                                selected=got.cpu().numpy())
    att = K.attention_kv_i8(q, cache, table, _i32(lens), dim ** -0.5, selected=got,
                            counts=None if counts is None else _i32(counts))
    R.check(att, out, bound, TYPES[dtype])
    # in any order, with gaps
    perm = torch.randperm(n, generator=torch.Generator().manual_seed(0)).cuda()
    gaps = torch.full((*got.shape[:3], 2), -1, dtype=torch.int32, device="cuda")
    mixed = torch.cat([got[..., perm], gaps], -1)[..., torch.randperm(
        n + 2, generator=torch.Generator().manual_seed(1)).cuda()].contiguous()
    att = K.attention_kv_i8(q, cache, table, _i32(lens), dim ** -0.5, selected=mixed,
                            counts=None if counts is None else _i32(counts))
    R.check(att, out, bound, TYPES[dtype])


def test_select_ties_go_to_the_lower_page(cuda_lib):
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(11)
    ref, rows, table = _filled(rng, [16 * 700 + 3], 1, 64, 16)
    ref.k_sum[:] = 5
    ref.scale["k"][rows[0]] = 0.5
    ref.k_sum[rows[0][300]] = 6
    cache = _cache(ref)
    q = torch.ones(1, 1, 1, 64, dtype=torch.float16, device="cuda")
    got = K.kv_select_i8(q, cache, table, _i32([16 * 700 + 3]), 260)[0, 0, 0].cpu().tolist()
    assert got == list(range(258)) + [300, 700]
    got = K.kv_select_i8(-q, cache, table, _i32([16 * 700 + 3]), 302)[0, 0, 0].cpu().tolist()
    assert got == list(range(300)) + [301, 700]
    cache.k_sum.zero_()
    got = K.kv_select_i8(q, cache, table, _i32([16 * 700 + 3]), 5)[0, 0, 0].cpu().tolist()
    assert got == [0, 1, 2, 3, 700]
    cache.k_scale[rows[0][77]] = float("nan")       # a NaN page is chosen, not hidden
    got = K.kv_select_i8(q, cache, table, _i32([16 * 700 + 3]), 3)[0, 0, 0].cpu().tolist()
    assert got == [0, 77, 700]


# ---------------------------------------------------------------------------
# Streams, graphs, refusals
# ---------------------------------------------------------------------------
def test_side_stream_and_graph(cuda_lib):
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(12)
    lens = [321, 65]
    ref, rows, table = _filled(rng, lens, 2, 64, 64)
    cache = _cache(ref)
    n = _i32(lens)
    table = _wide(table)
    for t in (1, 130):
        q = torch.from_numpy(rng.standard_normal((2, 4, t, 64))).half().cuda()

        def step(q):
            sel = K.kv_select_i8(q, cache, table, n, 3)
            return K.attention_kv_i8(q, cache, table, n, 0.125), K.attention_kv_i8(q, cache, table, n, 0.125,
                                                                                   selected=sel), sel
        want = step(q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step(q)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        held = torch.zeros_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(held)
        held.copy_(q)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals(cuda_lib):
    from h3vae_b200 import kernels as K
    from h3vae_b200.kv_cache import KVCacheI8
    cache = KVCacheI8.empty(4, 2, 64, 16)
    table, one = _i32([[0, 1]]), _i32([1])
    k = torch.zeros(1, 2, 3, 64, device="cuda", dtype=torch.float16)
    q = torch.zeros(1, 4, 3, 64, device="cuda", dtype=torch.float16)
    bad = [
        lambda: KVCacheI8.empty(4, 2, 80, 16), lambda: KVCacheI8.empty(4, 2, 64, 24),
        lambda: KVCacheI8(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_sum.int()),
        lambda: KVCacheI8(cache.k, cache.v.transpose(0, 1), cache.k_scale, cache.v_scale, cache.k_sum),
        lambda: KVCacheI8(*(getattr(cache, n).cpu() for n in ("k", "v", "k_scale", "v_scale", "k_sum"))),
        lambda: K.kv_write_i8(cache, table.long(), one, k, k), lambda: K.kv_write_i8(cache, table[0], one, k, k),
        lambda: K.kv_write_i8(cache, table, one, k, k.float()), lambda: K.kv_write_i8(cache, table, one, k[..., :32], k),
        lambda: K.kv_write_i8(cache, table, one, k[:, :1], k[:, :1]), lambda: K.kv_write_i8(cache, table, None, k, k),
        lambda: K.kv_write_i8(cache, table, _i32([1, 2]), k, k), lambda: K.kv_write_i8(cache, table, one, k, k[:, :, :2]),
        lambda: K.kv_write_i8(cache, table, one, k.cpu(), k.cpu()), lambda: K.kv_write_i8(cache, table, one.cpu(), k, k),
        lambda: K.kv_write_i8(cache, table, one, k.int(), k.int()),
        lambda: K.kv_read_i8(cache, table, one, -1), lambda: K.kv_read_i8(cache, table, one, 4, dtype=torch.int8),
        lambda: K.kv_read_i8(cache, table, None, 4),
        lambda: K.attention_kv_i8(q[:, :3], cache, table, one, 1.0), lambda: K.attention_kv_i8(q.float(), cache, table, one, 1.0),
        lambda: K.attention_kv_i8(q, cache, table, None, 1.0), lambda: K.attention_kv_i8(q, cache, table, one, 1.0, window=-1),
        lambda: K.attention_kv_i8(q, cache, table, one, 1.0, causal=False, window=4),
        lambda: K.attention_kv_i8(q, cache, table, one, 1.0, out=k),
        lambda: K.attention_kv_i8(q, cache, table, one, 1.0, selected=_i32([[[[0]]]])),
        lambda: K.attention_kv_i8(q, cache, table, one, 1.0, causal=False, selected=torch.zeros(1, 2, 3, 1, dtype=torch.int32, device="cuda")),
        lambda: K.attention_kv_i8(q, cache, table, one, 1.0, window=2, selected=torch.zeros(1, 2, 3, 1, dtype=torch.int32, device="cuda")),
        lambda: K.kv_select_i8(q, cache, table, one, 0), lambda: K.kv_select_i8(q, cache, table, one, 2, counts=_i32([1, 1])),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail(f"call {i} was not refused")
    # nothing to do is no error
    K.kv_write_i8(cache, table, one, k[:, :, :0], k[:, :, :0])
    assert K.attention_kv_i8(q[:, :, :0], cache, table, one, 1.0).shape == (1, 4, 0, 64)
    assert K.kv_select_i8(q[:, :, :0], cache, table, one, 2).shape == (1, 2, 0, 2)


def test_attention_over_many_selected_pages(cuda_lib):
    """More pages than one cluster's blocks hold: the parts go through the workspace."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(13)
    lens = [16 * 2600 + 5]
    ref, rows, table = _filled(rng, lens, 1, 64, 16)
    cache = _cache(ref)
    q = torch.from_numpy(rng.standard_normal((1, 2, 2, 64)) * 2).half().cuda()
    sel = K.kv_select_i8(q, cache, table, _i32(lens), 2300)
    got = K.attention_kv_i8(q, cache, table, _i32(lens), 0.125, selected=sel)
    out, _, bound = _attend_all(ref, rows, q, lens, [2], 0.125, 16, selected=sel.cpu().numpy())
    R.check(got, out, bound, torch.float16)


def test_long_single_streams(cuda_lib):
    """One and three long streams of one head: more runs of keys than a cluster has blocks."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(14)
    lens = [30000, 17, 9001]
    ref, rows, table = _filled(rng, lens, 1, 128, 128)
    cache = _cache(ref)
    for t, group, pick in ((1, 1, [0]), (1, 10, [0, 1, 2]), (4, 1, [1, 2, 0])):
        q = torch.from_numpy(rng.standard_normal((len(pick), group, t, 128)) * 2).to(torch.bfloat16).cuda()
        n = [lens[i] for i in pick]
        got = K.attention_kv_i8(q, cache, table[pick].contiguous(), _i32(n), 0.09)
        out, _, bound = _attend_all(ref, [rows[i] for i in pick], q, n, [t] * len(pick), 0.09, 128)
        R.check(got, out, bound, torch.bfloat16)


@pytest.mark.parametrize("heads,group,dim,lens", [
    (8, 1, 64, [4000, 17, 2900, 0, 3333, 1, 640, 3969, 64, 2500]),            # cut to fit one wave of blocks
    (8, 20, 64, [3100, 900, 2047, 33]),                                       # two row tiles
    (8, 2, 128, [1800, 5, 2100, 700] * 4),
    (8, 2, 64, [5000, 3000] + [(37 * i) % 200 for i in range(43)]),           # more than a warp's, three waves
    (8, 1, 64, [2500] + [(53 * i) % 150 for i in range(62)] + [1900]),        # more rows than blocks
    (8, 1, 64, [(29 * i) % 120 for i in range(127)] + [4100, 0, 2000]),       # more than twice as many
    (8, 1, 64, [(29 * i) % 120 for i in range(130)]),                         # and none long enough to cut
])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attention_uneven_batches(cuda_lib, heads, group, dim, lens, dtype):
    """Sequences of very different lengths, cut into runs that fit the device."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(len(lens))
    ref, rows, table = _filled(rng, lens, heads, dim, 64)
    cache = _cache(ref)
    q = torch.from_numpy(rng.standard_normal((len(lens), heads * group, 1, dim)) * 2).to(TYPES[dtype]).cuda()
    got = K.attention_kv_i8(q, cache, _wide(table, 2000), _i32(lens), dim ** -0.5)
    out, _, bound = _attend_all(ref, rows, q, lens, [1] * len(lens), dim ** -0.5, 64)
    R.check(got, out, bound, TYPES[dtype])


@pytest.mark.parametrize("heads,group,t,width,n", [(2, 3, 1, 60, 5), (1, 1, 3, 900, 40), (2, 2, 8, 1600, 33), (3, 8, 8, 2100, 64),
                                                   (1, 1, 1, 4096, 9), (16, 1, 8, 1030, 16), (1, 9, 8, 1600, 12), (2, 1, 9, 1600, 7)])
@pytest.mark.parametrize("dim", [64, 128])
def test_select_wide_tables(cuda_lib, heads, group, t, width, n, dim):
    """One launch or two, by tokens and the table's width: the same choice as with a table no wider than needed."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(width + n)
    lens = [1000, 0, 16 * min(width, 1200) - 3]
    ref, rows, table = _filled(rng, lens, heads, dim, 16)
    cache = _cache(ref)
    q = torch.from_numpy(rng.standard_normal((3, heads * group, t, dim))).half().cuda()
    wide = torch.nn.functional.pad(table, (0, max(0, width - table.shape[1])), value=-1).contiguous()
    got = K.kv_select_i8(q, cache, wide, _i32(lens), n)
    for other in (table, _wide(table, 5000)):
        assert torch.equal(got, K.kv_select_i8(q, cache, other, _i32(lens), n))
    counts = [t, t, max(t - 1, 0)]
    got = K.kv_select_i8(q, cache, wide, _i32(lens), n, counts=_i32(counts))
    assert torch.equal(got, K.kv_select_i8(q, cache, _wide(table, 5000), _i32(lens), n, counts=_i32(counts)))
