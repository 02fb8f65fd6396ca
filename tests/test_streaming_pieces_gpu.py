"""TokenStream on the B200 in pieces of whole frames: against the decoder's own chain, and with selected pages."""
import pytest
import torch

from test_streaming_gpu import _decoder, _rel

pytestmark = pytest.mark.gpu


def test_one_dense_piece_is_the_transformer(cuda_lib):
    """A clip in one piece sees what H3Decoder.transformer sees; keys and values are INT8 instead of fp16.  Their noise
    (a step of amax / 127 with amax about 4 rms: 1 % of the rms) reaches the output through two residual blocks: 3 %."""
    from h3vae_b200.streaming import TokenStream
    dec = _decoder()
    x = torch.randn(2, 3 * 96, 256, generator=torch.Generator().manual_seed(2)).half().cuda()
    got = TokenStream(dec, 2, (8, 12), max_frames=3).append(x)
    assert _rel(got, dec.transformer(x, (3, 8, 12))) < 3e-2


def test_frames_with_selected_pages(cuda_lib, monkeypatch):
    """Whole frames with as many pages as the context has: every page is chosen, so causal attention without selection
    gives the same but for the order of fp32 sums, whose fp16 rounding moves INT8 codes (the 0.5 % of the block chain).
    With fewer pages a stream's first frame, whose context they hold, is the same."""
    from h3vae_b200 import kernels as K
    from h3vae_b200.streaming import TokenStream
    dec = _decoder()
    x = torch.randn(2, 4 * 96, 256, generator=torch.Generator().manual_seed(3)).half().cuda()
    pieces = [x[:, :96], x[:, 96: 288], x[:, 288:]]
    every, few = (TokenStream(dec, 2, (8, 12), 4, pages=p) for p in (6, 2))
    got, less = [every.append(p) for p in pieces], [few.append(p) for p in pieces]
    monkeypatch.setattr(K, "kv_select_i8", lambda *args, **kw: None)
    causal = TokenStream(dec, 2, (8, 12), 4, pages=1)
    want = [causal.append(p) for p in pieces]
    for a, b in zip(got, want):
        assert _rel(a, b) < 5e-3
    assert _rel(less[0], want[0]) < 5e-3 and all(torch.isfinite(y).all() for y in less)
    assert _rel(less[2], want[2]) > 5e-3         # the last frame's tokens see a third of the context
