"""The INT8 decoder blocks over a clip that arrives piece by piece.

H3Decoder.transformer sees a clip's tokens at once.  TokenStream takes them in pieces (a few latent frames, one
frame): every block keeps the keys and values of the earlier pieces in a paged INT8 cache, and a piece attends to
itself and everything before it.  The rest of the chain is H3Decoder's: INT8 linears, QK norm + RoPE in the QKV
GEMM's epilogue, fused residual norms.

A piece does not see what comes after it, so the output is not that of H3Decoder.transformer over the whole clip (but
for a clip in one piece, where keys and values are INT8 instead of fp16).  The page table is made for max_frames at
once and calls are planned for its width, so a stream much shorter than max_frames runs on plans for the longest.

    stream = TokenStream(decoder, batch=4, grid_hw=(32, 32), max_frames=40)
    for piece in pieces:                 # fp16 [4, frames * 1024, hidden]
        y = stream.append(piece)         # the blocks' output for the piece, after the final LayerNorm
"""
from __future__ import annotations

import torch

from . import kernels as K
from .kv_cache import PAGE_SIZES, KVCacheI8
from .model import H3Decoder, rope_tables


class TokenStream:
    """State of one batch of clips.  `pages` > 0: each token attends to that many cache pages of earlier tokens
    (its own among them) instead of all, chosen per head by K.kv_select_i8, and to no later token.  That is for pieces
    of one or a few tokens over a long context: every token reads its own pages, so for whole frames attention to all
    is faster (4 clips x 16 heads x 1024 tokens, 32 pages: 3.4 ms a block over 5120 tokens and 3.7 ms over 40960;
    attention to all 0.18 and 1.2 ms)."""

    def __init__(self, decoder: H3Decoder, batch: int, grid_hw: tuple[int, int], max_frames: int, *,
                 page_size: int = 64, pages: int = 0):
        if not decoder.int8:
            raise ValueError("TokenStream runs the INT8 block chain (H3Decoder(int8=True))")
        if batch < 1 or max_frames < 1 or min(grid_hw) < 1 or pages < 0:
            raise ValueError("batch, grid and max_frames must be positive, pages at least 0")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        cfg = decoder.cfg
        self.decoder, self.batch, self.pages = decoder, batch, pages
        self.per_frame = grid_hw[0] * grid_hw[1]
        self.max_tokens = max_frames * self.per_frame
        per_clip = -(-self.max_tokens // page_size)
        dev = decoder.device
        self.caches = [KVCacheI8.empty(batch * per_clip, cfg.heads, 64, page_size, dev) for _ in decoder.blocks]
        self.page_table = torch.arange(batch * per_clip, dtype=torch.int32, device=dev).view(batch, per_clip)
        self.tokens = 0                                              # per clip, so far
        self.start = torch.zeros(batch, dtype=torch.int32, device=dev)
        cos, sin = rope_tables(max_frames, *grid_hw, cfg.rot_dims, dev)
        self._rope = [t.view(1, self.max_tokens, 1, -1).expand(batch, -1, 1, t.shape[-1]) for t in (cos, sin)]

    @torch.no_grad()
    def append(self, x: torch.Tensor) -> torch.Tensor:
        """x: fp16 [batch, n, hidden], the next n tokens (whole frames or part of one) -> fp16 [batch, n, hidden]."""
        dec, cfg = self.decoder, self.decoder.cfg
        b, n, d = x.shape
        if b != self.batch or d != cfg.hidden or x.dtype != torch.float16:
            raise ValueError(f"tokens must be fp16 [{self.batch}, n, {cfg.hidden}]")
        if n == 0 or self.tokens + n > self.max_tokens:
            raise ValueError(f"{n} tokens do not fit after {self.tokens} of at most {self.max_tokens}")
        cos, sin = (t[:, self.tokens: self.tokens + n].contiguous() for t in self._rope)
        lengths = self.start + n
        h = x = x.reshape(b * n, d).contiguous()
        out = scale2 = None
        for i, (blk, cache) in enumerate(zip(dec.blocks, self.caches)):
            if i == 0:
                q1, s1 = K.rms_quant(x, blk.norm1_w, cfg.eps)
            else:
                h, q1, s1 = K.residual_rms_quant(h, out, scale2, blk.norm1_w, cfg.eps, h_out=h)
                x = h
            q, k, v = K.gemm_i8_qkv_rope(q1, s1, blk.qkv_q, blk.qkv_s, blk.qkv_b, b, n, cfg.heads, cos, sin,
                                         cfg.qk_eps)
            K.kv_write_i8(cache, self.page_table, self.start, k, v)
            if self.pages:
                chosen = K.kv_select_i8(q, cache, self.page_table, lengths, self.pages)
                y = K.attention_kv_i8(q, cache, self.page_table, lengths, 1.0 / 8.0, selected=chosen)
            else:
                y = K.attention_kv_i8(q, cache, self.page_table, lengths, 1.0 / 8.0, causal=False)
            qy, sy = K.row_quant(y.transpose(1, 2).reshape(b * n, d))
            h, sumsq = K.gemm_i8_residual(qy, sy, blk.out_q, blk.out_s, blk.out_b, x, blk.scale1)
            q2, s2 = K.rms_quant_parts(h, sumsq, blk.norm2_w, cfg.eps)
            act = K.gemm_i8_swiglu(q2, s2, blk.up_q, blk.up_s, blk.up_b)
            qf, sf = K.row_quant(act)
            out = K.gemm_i8(qf, sf, blk.down_q, blk.down_s, blk.down_b)
            scale2 = blk.scale2
        self.tokens += n
        self.start = lengths
        return K.final_residual_layernorm(h, out, scale2, dec.ln_w, dec.ln_b, cfg.eps).view(b, n, d)

    def context(self, block: int, dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values a block has kept, dense [batch, heads, tokens, 64]."""
        return K.kv_read_i8(self.caches[block], self.page_table, self.start, self.tokens, dtype=dtype)
