"""One decoder layer of a Llama-style model on this library's kernels (decode step).

The layer the reference's model loader wires (onnx-rt/src/model_loader/gemma.rs:13-36,
Llama without Gemma's embedding scale), one token per sequence:

    pre1 = x + resid                    h1 = RMSNorm(pre1) * input_norm     (SkipSimplifiedLayerNormalization)
    q, k, v = h1 . Wqkv^T, RoPE(q), RoPE(k) and v appended to the cache   (sa_qkv_project_append)
    a = GroupQueryAttention over the cache                               (sa_gqa_attend, rotary done)
    o = a . Wo^T                                                         (MatMulNBits)
    pre2 = o + pre1                     h2 = RMSNorm(pre2) * post_norm      (SkipSimplifiedLayerNormalization)
    g|u = h2 . Wgu^T                                                     (MatMulNBits, packed gate|up rows)
    m = Silu(g) * u                                                      (SwiGLU)
    d = m . Wdown^T                                                      (MatMulNBits)

and returns (d, pre2): the next layer adds them in its own first norm
(x = d, resid = pre2), so every residual add is fused into a norm.  All weights
are int4 MatMulNBits (block 32, zero point 8) with scales of the activation type.
The cache position is not advanced (once per forward pass, after the last layer).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ._lib import SA_BLOCK_TOKENS
from .ops import (gqa_attend, gqa_select_blocks, gqa_sparse_attend, gqa_tree_attend, kv_block_means, matmul_nbits,
                  qkv_project_append, rms_norm, rotary_embedding, silu_mul)


@dataclass
class LayerWeights:
    """Int4 MatMulNBits weights ([N][K/32][16] codes, [N][K/32] scales) of one layer."""

    wqkv_codes: torch.Tensor   # (Hq + 2*Hkv)*D rows: Wq, then Wk, then Wv
    wqkv_scales: torch.Tensor
    wo_codes: torch.Tensor     # hidden rows, K = Hq*D
    wo_scales: torch.Tensor
    wgu_codes: torch.Tensor    # 2*F rows: gate rows, then up rows, K = hidden
    wgu_scales: torch.Tensor
    wdown_codes: torch.Tensor  # hidden rows, K = F
    wdown_scales: torch.Tensor
    input_norm: torch.Tensor   # (hidden,)
    post_norm: torch.Tensor    # (hidden,)
    epsilon: float = 1e-5


def decoder_layer_step(x: torch.Tensor, resid: torch.Tensor | None, w: LayerWeights, cache, layer: int, *,
                       cos_cache=None, sin_cache=None, do_rotary: bool = True, rotary_interleaved: bool = False,
                       block_means: torch.Tensor | None = None, max_blocks: int = 0):
    """One decode step of one layer: ``x`` (B, hidden) plus residual ``resid`` (None for
    the first layer) -> ``(d, pre2)``, the input and residual of the next layer.

    With ``block_means`` -- this layer's bf16 (B, H, blocks, D) means of every full block
    before the new token, as ``kv_block_means`` fills them -- the token attends to the
    ``max_blocks`` blocks of 64 that ``gqa_select_blocks`` picks instead of the whole cache,
    and the mean of a block that the token fills is added.
    """
    b, hidden = x.shape
    cfg = cache.config
    hq = cfg.kv_head_count * (cfg.num_heads // cfg.num_kv_heads)
    d_head = cfg.head_dim
    h1, pre1 = rms_norm(x, w.input_norm, skip=resid, epsilon=w.epsilon)
    q, _, _ = qkv_project_append(h1, w.wqkv_codes, w.wqkv_scales, cache, layer, do_rotary=do_rotary,
                                 rotary_interleaved=rotary_interleaved, cos_cache=cos_cache, sin_cache=sin_cache)
    q = q.view(b, 1, hq * d_head)
    if block_means is None:
        a = gqa_attend(q, cache, layer, num_heads=hq, do_rotary=False)
    else:
        ids = gqa_select_blocks(q, cache, layer, block_means, num_heads=cfg.num_heads, max_blocks=max_blocks)
        a = gqa_sparse_attend(q, cache, layer, ids, num_heads=cfg.num_heads)
        blk, last = divmod(cache.current_position(), SA_BLOCK_TOKENS)
        if last == SA_BLOCK_TOKENS - 1:
            kv_block_means(cache, layer, blk, blk + 1, out=block_means[:, :, blk:blk + 1])
    return _after_attention(a.view(b, hq * d_head), pre1, w)


def _after_attention(a: torch.Tensor, pre1: torch.Tensor, w: LayerWeights):
    """Output projection, second norm and MLP of rows ``a`` (rows, Hq*D)."""
    hidden = pre1.shape[1]
    o = matmul_nbits(a, w.wo_codes, w.wo_scales, K=a.shape[1], N=hidden)
    h2, pre2 = rms_norm(o, w.post_norm, skip=pre1, epsilon=w.epsilon)
    f2 = w.wgu_scales.shape[0]
    gu = matmul_nbits(h2, w.wgu_codes, w.wgu_scales, K=hidden, N=f2)
    m = silu_mul(gu)
    return matmul_nbits(m, w.wdown_codes, w.wdown_scales, K=f2 // 2, N=hidden), pre2


def tree_layer_step(x: torch.Tensor, resid: torch.Tensor | None, w: LayerWeights, cache, layer: int, *,
                    parents: torch.Tensor, position_ids: torch.Tensor, cos_cache: torch.Tensor,
                    sin_cache: torch.Tensor, rotary_interleaved: bool = False):
    """One layer over a tree of drafted tokens per sequence: ``x`` (B*N, hidden) plus ``resid`` -> ``(d, pre2)``.

    ``parents`` int32 (B, N) as gqa_tree_attend takes them; ``position_ids`` int32 (B, N) the nodes' positions,
    cache position + depth (any row of the tables for a slot without a node).  The drafts' K/V go to the cache
    behind its position, which is not advanced.  A verification step runs this for every layer, accepts a path
    from the last one's output and keeps it:

        cache.keep_drafts(path, drafted=N); cache.advance_position(path.shape[1])
    """
    batch, nodes = parents.shape
    hidden = x.shape[1]
    if x.shape[0] != batch * nodes:
        raise ValueError("tree_layer_step: x must have batch * nodes rows")
    cfg = cache.config
    hkv, d_head = cfg.kv_head_count, cfg.head_dim
    hq = hkv * (cfg.num_heads // cfg.num_kv_heads)
    qd, kd = hq * d_head, hkv * d_head
    h1, pre1 = rms_norm(x, w.input_norm, skip=resid, epsilon=w.epsilon)
    proj = []
    for r0, n in ((0, qd), (qd, kd), (qd + kd, kd)):
        proj.append(matmul_nbits(h1, w.wqkv_codes[r0:r0 + n], w.wqkv_scales[r0:r0 + n], K=hidden, N=n))
    q, k, v = (t.view(batch, nodes, -1) for t in proj)
    for t, heads in ((q, hq), (k, hkv)):
        rotary_embedding(t, cos_cache, sin_cache, position_ids=position_ids, interleaved=rotary_interleaved,
                         num_heads=heads, out=t)
    cache.append(layer, k, v)
    a = gqa_tree_attend(q, cache, layer, parents, num_heads=cfg.num_heads)
    return _after_attention(a.view(batch * nodes, qd), pre1, w)


def prefill_layer_step(x: torch.Tensor, resid: torch.Tensor | None, w: LayerWeights, cache, layer: int, *,
                       batch: int, seq_len: int, cos_cache=None, sin_cache=None, do_rotary: bool = True,
                       rotary_interleaved: bool = False):
    """One layer over whole prompts: ``x`` (batch*seq_len, hidden) plus ``resid`` -> ``(d, pre2)``.

    The same layer as decoder_layer_step with every projection a tcgen05 MatMulNBits of
    batch*seq_len rows.  Q, K and V are three MatMulNBits calls on the row blocks of the packed
    Wqkv (GroupQueryAttention takes separate contiguous Q/K/V), and GroupQueryAttention appends
    the prompts' K/V at the cache position (RoPE, quantize-on-append) and runs the causal
    prefill attention of every query over them.  The position is not advanced.
    """
    m, hidden = x.shape
    if m != batch * seq_len:
        raise ValueError("prefill_layer_step: x must have batch * seq_len rows")
    from .ops import group_query_attention

    cfg = cache.config
    hkv = cfg.kv_head_count
    hq = hkv * (cfg.num_heads // cfg.num_kv_heads)
    d_head = cfg.head_dim
    qd, kd = hq * d_head, hkv * d_head
    h1, pre1 = rms_norm(x, w.input_norm, skip=resid, epsilon=w.epsilon)
    proj = []
    for r0, n in ((0, qd), (qd, kd), (qd + kd, kd)):
        proj.append(matmul_nbits(h1, w.wqkv_codes[r0:r0 + n], w.wqkv_scales[r0:r0 + n], K=hidden, N=n))
    q, k, v = (t.view(batch, seq_len, -1) for t in proj)
    a = group_query_attention(q, k, v, cache, layer, num_heads=cfg.num_heads, kv_num_heads=cfg.num_kv_heads,
                              do_rotary=do_rotary,
                              rotary_interleaved=rotary_interleaved, cos_cache=cos_cache, sin_cache=sin_cache)
    return _after_attention(a.view(m, qd), pre1, w)
