"""The cache operators on the B200 at the edges of what they promise, against the restatements of kv_reference."""
import numpy as np
import pytest
import torch

import kv_reference as R
from test_kv_cache_gpu import TYPES, _attend_all, _cache, _filled, _i32, _wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,page,t,group", [(64, 64, 137, 1), (128, 32, 137, 1), (128, 128, 43, 5), (64, 16, 67, 3)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_tiles_into_an_unaligned_output(cuda_lib, dim, page, t, group, dtype):
    """Row tiles whose last warps have rows past the end, written element by element: the bits of an aligned output,
    and nothing beside it."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(20 + dim + t)
    lens = [300, t]
    ref, rows, table = _filled(rng, lens, 2, dim, page)
    cache, table = _cache(ref), _wide(table)
    q = torch.from_numpy(rng.standard_normal((2, 2 * group, t, dim)) * 2).to(TYPES[dtype]).cuda()
    want = K.attention_kv_i8(q, cache, table, _i32(lens), dim ** -0.5)
    out, _, bound = _attend_all(ref, rows, q, lens, [t, t], dim ** -0.5, page)
    R.check(want, out, bound, TYPES[dtype])
    room = torch.full((2, 2 * group, t, dim + 5), 7.0, dtype=q.dtype, device="cuda")
    got = K.attention_kv_i8(q, cache, table, _i32(lens), dim ** -0.5, out=room[..., 3: dim + 3])
    assert torch.equal(got, want) and (room[..., :3] == 7).all() and (room[..., dim + 3:] == 7).all()


# ---------------------------------------------------------------------------
# A page with a NaN scale
# ---------------------------------------------------------------------------
def _sees(pos, page, size, causal, window):
    """Whether a row at `pos` (-1: none) sees a key of page ordinal `page`."""
    first = max(0, pos + 1 - window) if window else 0
    return pos >= 0 and page * size + size > first and (not causal or page * size <= pos)


@pytest.mark.parametrize("t,causal,window", [(1, True, 0), (1, True, 4), (5, True, 4), (9, True, 0), (30, True, 0), (30, True, 7),
                                             (20, False, 0), (140, True, 0), (140, True, 30)])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_scales_reach_the_rows_that_see_them_alone(cuda_lib, t, causal, window, wide, which):
    """One page of a sequence takes a NaN scale, for keys or for values: the rows that see a key of it are NaN, the
    others and the other sequence are what they were."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(30 + t)
    lens, size = [150, 200], 16
    ref, rows, table = _filled(rng, lens, 2, 64, size)
    q = torch.from_numpy(rng.standard_normal((2, 4, t, 64))).half().cuda()
    args = dict(causal=causal, window=window)
    out, _, bound = _attend_all(ref, rows, q, lens, [t, t], 0.125, size, **args)
    for page in (9, 8, 3):
        cache = _cache(ref)
        getattr(cache, which + "_scale")[rows[0][page]] = float("nan")
        got = K.attention_kv_i8(q, cache, _wide(table) if wide else table, _i32(lens), 0.125, **args)
        hit = np.array([_sees(150 - t + i if 150 - t + i >= 0 else -1, page, size, causal, window) for i in range(t)])
        assert torch.isnan(got[0][:, torch.from_numpy(hit).cuda()]).all()
        if not hit.all():
            R.check(got[0][:, torch.from_numpy(~hit).cuda()], out[0][:, ~hit], bound[0][:, ~hit], torch.float16)
        R.check(got[1], out[1], bound[1], torch.float16)


@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_scales_and_rows_without_keys(cuda_lib, which):
    """Padding rows and rows before the first key are zero, whatever the pages hold."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(31)
    lens, counts, t = [70, 5], [3, 9], 12
    ref, rows, table = _filled(rng, lens, 1, 64, 16)
    q = torch.from_numpy(rng.standard_normal((2, 2, t, 64))).half().cuda()
    cache = _cache(ref)
    for row in rows:
        for page in row:
            getattr(cache, which + "_scale")[page] = float("nan")
    for tab in (table, _wide(table)):
        got, lse = K.attention_kv_i8(q, cache, tab, _i32(lens), 0.125, counts=_i32(counts), return_lse=True)
        assert torch.isnan(got[0, :, :3]).all() and (got[0, :, 3:] == 0).all() and (lse[0, :, 3:] == -np.inf).all()
        assert (got[1, :, :4] == 0).all() and torch.isnan(got[1, :, 4:9]).all() and (got[1, :, 9:] == 0).all()


@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_scales_of_selected_pages_past_a_row(cuda_lib, which):
    """A selected page that lies behind a row's position adds nothing to it."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(32)
    lens, t, size = [150], 20, 16
    ref, rows, table = _filled(rng, lens, 2, 64, size)
    q = torch.from_numpy(rng.standard_normal((1, 4, t, 64))).half().cuda()
    sel = torch.arange(10, dtype=torch.int32, device="cuda").expand(1, 2, t, 10).contiguous()
    out, _, bound = _attend_all(ref, rows, q, lens, [t], 0.125, size, selected=sel.cpu().numpy())
    cache = _cache(ref)
    getattr(cache, which + "_scale")[rows[0][9]] = float("nan")
    got = K.attention_kv_i8(q, cache, table, _i32(lens), 0.125, selected=sel)
    hit = torch.arange(130, 150) >= 144
    assert torch.isnan(got[:, :, hit.cuda()]).all()
    R.check(got[:, :, ~hit.cuda()], out[:, :, ~hit.numpy()], bound[:, :, ~hit.numpy()], torch.float16)


# ---------------------------------------------------------------------------
# Selection with NaN and infinities in the queries
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("t,wide", [(1, False), (1, True), (6, False), (12, False)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_select_leaves_out_heads_that_are_not_finite(cuda_lib, t, wide, dtype):
    """A head whose query holds a NaN or an infinity has no say in its group's choice; where no head is left, all
    pages count alike and the lowest are taken."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(50 + t)
    lens, size, n, group = [700, 333], 16, 6, 3
    ref, rows, table = _filled(rng, lens, 2, 64, size)
    cache = _cache(ref)
    table = _wide(table, 5000) if wide else table
    q = torch.from_numpy(rng.standard_normal((2, 2 * group, t, 64))).to(TYPES[dtype])
    fine = q.float().numpy().copy()
    q[0, 0, :, 5] = float("nan")
    q[0, 2, :, 63] = float("inf")
    q[0, 4, :, 0] = -float("inf")
    q[1, 3:, t - 1, 17] = float("nan")
    got = K.kv_select_i8(q.cuda(), cache, table, _i32(lens), n).cpu().numpy()
    left = {(0, 0): [1], (0, 1): [3, 5], (1, 0): [0, 1, 2], (1, 1): [3, 4, 5]}
    for (b, h), heads in left.items():
        pos = [lens[b] - t + i for i in range(t)]
        want = R.select(fine[b, heads], ref.scale["k"][rows[b], h], ref.k_sum[rows[b], h], pos, n, size, len(heads))
        if (b, h) == (1, 1):
            want[t - 1] = [*range(n - 1), pos[-1] // size]
        assert np.array_equal(got[b, h], want), (b, h)


# ---------------------------------------------------------------------------
# Sequences without queries
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("t,group,wide", [(1, 1, False), (1, 4, True), (7, 2, False), (40, 1, True), (140, 1, True)])
def test_sequences_without_queries_are_not_looked_at(cuda_lib, t, group, wide):
    """A count of zero: zero rows, and no page of the sequence is looked up (its table holds no page numbers, which a
    lookup would report)."""
    from h3vae_b200 import _lib, kernels as K
    rng = np.random.default_rng(40 + t)
    lens, counts = [500, 700, 333], [t, 0, max(0, t - 1)]
    ref, rows, table = _filled(rng, lens, 2, 64, 16)
    cache = _cache(ref)
    table = _wide(table) if wide else table
    q = torch.from_numpy(rng.standard_normal((3, 2 * group, t, 64))).half().cuda()
    args = dict(counts=_i32(counts))
    want = K.attention_kv_i8(q, cache, table, _i32(lens), 0.125, **args)
    pages = K.kv_select_i8(q, cache, table, _i32(lens), 4, **args)
    kept = K.attention_kv_i8(q, cache, table, _i32(lens), 0.125, selected=pages, **args)
    assert _lib.device_error() == 0
    gone = table.clone()
    gone[1] = -1
    got, lse = K.attention_kv_i8(q, cache, gone, _i32(lens), 0.125, return_lse=True, **args)
    assert _lib.device_error() == 0
    assert torch.equal(got, want) and (got[1] == 0).all() and (lse[1] == -np.inf).all()
    assert torch.equal(K.kv_select_i8(q, cache, gone, _i32(lens), 4, **args), pages) and (pages[1] == -1).all()
    assert _lib.device_error() == 0
    every = torch.arange(4, dtype=torch.int32, device="cuda").expand(1, 2, t, 4)     # pages named for rows that are none
    sel = torch.cat([pages[:1], every, pages[2:]]).contiguous()
    assert torch.equal(K.attention_kv_i8(q, cache, gone, _i32(lens), 0.125, selected=sel, **args), kept)
    assert _lib.device_error() == 0


# ---------------------------------------------------------------------------
# V scales far apart
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("t,group", [(1, 2), (6, 12), (130, 2)])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("big", [1e4, 1e10, 1e18])
@pytest.mark.parametrize("order", ["zeros first", "zeros last", "mixed"])
@pytest.mark.parametrize("k_size", [1.0, 8.0])
def test_value_pages_of_zeros_beside_large_ones(cuda_lib, t, group, wide, big, order, k_size):
    """Keys whose values are zero count in the denominator like any other, however large the other pages' values are."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(60 + t)
    lens, size = [500, 333], 32
    ref, rows, table = _filled(rng, lens, 1, 64, size)
    for row in rows:
        pages = row[: len(row)]
        zero = {"zeros first": pages[: len(pages) // 2], "zeros last": pages[len(pages) // 2:], "mixed": pages[::2]}[order]
        for page in pages:
            ref.scale["k"][page] *= np.float32(k_size)
            ref.scale["v"][page] = R.TINY if page in zero else np.float32(ref.scale["v"][page] * big)
        for page in zero:
            ref.code["v"][page] = 0
    cache = _cache(ref)
    q = torch.from_numpy(rng.standard_normal((2, group, t, 64))).to(torch.bfloat16).cuda()
    got, lse = K.attention_kv_i8(q, cache, _wide(table) if wide else table, _i32(lens), 0.125, return_lse=True)
    out, want_lse, bound = _attend_all(ref, rows, q, lens, [t, t], 0.125, size)
    R.check(got, out, bound, torch.bfloat16)
    lse = lse.double().cpu().numpy()
    assert np.abs(lse - want_lse).max() <= 2.0 ** -10


@pytest.mark.parametrize("t", [1, 12, 130])
def test_value_pages_of_zeros_in_parts_of_their_own(cuda_lib, t):
    """The same where parts of the keys are joined: whole runs of zero pages beside runs of large values."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(61)
    lens, size = [12000], 64
    ref, rows, table = _filled(rng, lens, 1, 64, size)
    ref.scale["v"][rows[0]] *= np.float32(1e12)
    half = rows[0][: len(rows[0]) // 2]
    ref.scale["v"][half] = R.TINY
    ref.code["v"][half] = 0
    cache = _cache(ref)
    q = torch.from_numpy(rng.standard_normal((1, 1, t, 64))).to(torch.bfloat16).cuda()
    sel = torch.arange(len(rows[0]), dtype=torch.int32, device="cuda").expand(1, 1, t, -1).contiguous()
    out, _, bound = _attend_all(ref, rows, q, lens, [t], 0.125, size)
    for tab, more in ((table, {}), (_wide(table), {}), (table, dict(selected=sel))):
        R.check(K.attention_kv_i8(q, cache, tab, _i32(lens), 0.125, **more), out, bound, torch.bfloat16)


# ---------------------------------------------------------------------------
# Selected pages for a frame of tokens
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,dim,group,t,lens,n", [("fp16", 64, 1, 192, [1500, 192], 7), ("bf16", 128, 3, 150, [900, 77], 4)])
def test_selected_pages_for_a_frame(cuda_lib, dtype, dim, group, t, lens, n):
    """Hundreds of tokens a call: every token's own choice, and attention over it."""
    from h3vae_b200 import kernels as K
    rng = np.random.default_rng(70 + t)
    ref, rows, table = _filled(rng, lens, 2, dim, 64)
    cache = _cache(ref)
    q = torch.from_numpy(rng.standard_normal((2, 2 * group, t, dim))).to(TYPES[dtype]).cuda()
    got = K.kv_select_i8(q, cache, table, _i32(lens), n)
    qn = q.float().cpu().numpy()
    for b, ln in enumerate(lens):
        pos = [ln - t + i if ln - t + i >= 0 else -1 for i in range(t)]
        for h in range(2):
            want = R.select(qn[b, h * group: h * group + group], ref.scale["k"][rows[b], h], ref.k_sum[rows[b], h], pos,
                            n, 64, group)
            assert np.array_equal(got[b, h].cpu().numpy(), want), (b, h)
    out, _, bound = _attend_all(ref, rows, q, lens, [t, t], dim ** -0.5, 64, selected=got.cpu().numpy())
    R.check(K.attention_kv_i8(q, cache, table, _i32(lens), dim ** -0.5, selected=got), out, bound, TYPES[dtype])
