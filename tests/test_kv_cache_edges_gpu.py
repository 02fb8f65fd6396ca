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
