"""ViT-B/16 (and friends) with torchvision-compatible ``state_dict`` keys.

"ViT-B/16 DDP bf16 (GEMM-heavy path, fused softmax-CE
+ SGD/AdamW)".  Keys: ``class_token``, ``conv_proj.{weight,bias}``,
``encoder.pos_embedding``, ``encoder.layers.encoder_layer_{i}.{ln_1,ln_2}.*``,
``...self_attention.{in_proj_weight,in_proj_bias,out_proj.weight,out_proj.bias}``,
``...mlp.{0,3}.{weight,bias}``, ``encoder.ln.*``, ``heads.head.*``.

197 tokens per image: ordinary single-device attention, no sequence
parallelism.  Projections, MLP, patch embedding and head run on
the own MFMA GEMM (csrc/kernels/gemm.hip) with bias / GELU / residual fused in
its epilogues; loss and optimizer are the fused HIP kernels.

Options beyond torchvision's model, all off by default (its keys and numbers are then unchanged): ``rel_pos_bias`` adds a learned
relative position bias to every layer's attention, ``layer_scale`` a learned gate per channel to every branch (``post_norm``:
and a LayerNorm before the gate), with the block ends fused into the next block's norm, and ``pool="attention"`` replaces the
class token's row by one learned query that attends to all tokens.
"""
from __future__ import annotations

import math
from collections import OrderedDict

import torch
import torch.nn as tnn

from .. import nn as pnn
from ..nn.functional import (attention, cross_attention, gated_residual_norm, layer_norm, linear, mlp_gelu, patch_embed,
                             rel_bias_attention, vit_embed)


class MultiheadSelfAttention(tnn.Module):
    """Packed-QKV self attention, parameters named like ``nn.MultiheadAttention``.  ``positions`` (what
    ``nn.grid_position_buckets`` returns): with a learned bias per bucket of relative positions and head."""

    def __init__(self, dim: int, heads: int, positions=None):
        super().__init__()
        assert dim % heads == 0
        self.embed_dim, self.num_heads, self.head_dim = dim, heads, dim // heads
        self.in_proj_weight = tnn.Parameter(torch.empty(3 * dim, dim))
        self.in_proj_bias = tnn.Parameter(torch.zeros(3 * dim))
        self.out_proj = pnn.Linear(dim, dim)
        tnn.init.xavier_uniform_(self.in_proj_weight)
        tnn.init.zeros_(self.out_proj.bias)
        self.relative_position_bias_table = None
        if positions is not None:
            self.relative_position_bias_table = tnn.Parameter(torch.zeros(int(positions[2].max()) + 1, heads))
            for name, codes in zip(("_q_codes", "_k_codes", "_bucket_of"), positions):
                self.register_buffer(name, codes, persistent=False)

    def forward(self, x, residual=None):
        qkv = linear(x, self.in_proj_weight, self.in_proj_bias)   # own MFMA GEMM, bias in the epilogue
        if self.relative_position_bias_table is not None:
            out = rel_bias_attention(qkv, self.relative_position_bias_table, self._q_codes, self._k_codes, self._bucket_of,
                                     self.num_heads)
        else:
            out = attention(qkv, self.num_heads)  # [b, s, d]: fused kernel on GPU/bf16, matmul-softmax oracle elsewhere
        return self.out_proj(out, residual)   # bias + residual in the GEMM epilogue


class EncoderBlock(tnn.Module):
    """Pre-LN block.  Every elementwise op rides in a GEMM or LayerNorm kernel: bias / GELU / residual add in GEMM
    epilogues, GELU' in the data-gradient GEMM's epilogue, and the two gradients that meet at a residual fork are
    summed inside the LayerNorm backward kernel (``layer_norm(..., with_skip=True)``)."""

    def __init__(self, dim, heads, mlp_dim, dropout=0.0, positions=None, layer_scale=None, post_norm=False):
        super().__init__()
        self.ln_1 = tnn.LayerNorm(dim, eps=1e-6)
        self.self_attention = MultiheadSelfAttention(dim, heads, positions)
        self.dropout = tnn.Dropout(dropout)
        self.ln_2 = tnn.LayerNorm(dim, eps=1e-6)
        self.mlp = tnn.Sequential(
            pnn.Linear(dim, mlp_dim), tnn.GELU(), tnn.Dropout(dropout), pnn.Linear(mlp_dim, dim), tnn.Dropout(dropout))
        for m in (self.mlp[0], self.mlp[3]):
            tnn.init.xavier_uniform_(m.weight)
            tnn.init.normal_(m.bias, std=1e-6)
        self.gated = layer_scale is not None
        if self.gated:
            self.gate_1 = tnn.Parameter(torch.full((dim,), float(layer_scale)))
            self.gate_2 = tnn.Parameter(torch.full((dim,), float(layer_scale)))
            self.post_ln_1 = tnn.LayerNorm(dim, eps=1e-6) if post_norm else None
            self.post_ln_2 = tnn.LayerNorm(dim, eps=1e-6) if post_norm else None
        elif post_norm:
            raise ValueError("post_norm goes with layer_scale")

    @staticmethod
    def _ln(ln, x, with_skip=False):
        return layer_norm(x, ln.weight, ln.bias, ln.eps, with_skip)

    @staticmethod
    def _end(x, branch, gate, post, ln):
        return gated_residual_norm(x, branch, gate, ln.weight, ln.bias, ln.eps, None if post is None else post.weight,
                                   None if post is None else post.bias)

    def gated_forward(self, x, xn, next_ln):
        """``(x, ln_1(x)) -> (x', next_ln(x'))``: each branch's end (norm, gate, residual add) and the norm that follows it are
        one kernel."""
        x, xn = self._end(x, self.dropout(self.self_attention(xn)), self.gate_1, self.post_ln_1, self.ln_2)
        if self.dropout.p > 0.0 and self.training:
            y = self.mlp(xn)
        else:
            y = mlp_gelu(xn, self.mlp[0].weight, self.mlp[0].bias, self.mlp[3].weight, self.mlp[3].bias)
        return self._end(x, y, self.gate_2, self.post_ln_2, next_ln)

    def forward(self, x):
        if self.gated:
            return self.gated_forward(x, self._ln(self.ln_1, x), self.ln_1)[0]
        if self.dropout.p > 0.0 and self.training:  # unfused composition (the reference configuration uses p = 0)
            y = self.dropout(self.self_attention(self._ln(self.ln_1, x)))
            x = x + y
            return x + self.mlp(self._ln(self.ln_2, x))
        xn, skip = self._ln(self.ln_1, x, True)
        x = self.self_attention(xn, skip)
        xn, skip = self._ln(self.ln_2, x, True)
        return mlp_gelu(xn, self.mlp[0].weight, self.mlp[0].bias, self.mlp[3].weight, self.mlp[3].bias, skip)


class Encoder(tnn.Module):
    def __init__(self, seq_len, layers, heads, dim, mlp_dim, dropout=0.0, positions=None, layer_scale=None, post_norm=False):
        super().__init__()
        self.pos_embedding = tnn.Parameter(torch.empty(1, seq_len, dim).normal_(std=0.02))
        self.dropout = tnn.Dropout(dropout)
        self.layers = tnn.Sequential(OrderedDict(
            (f"encoder_layer_{i}", EncoderBlock(dim, heads, mlp_dim, dropout, positions, layer_scale, post_norm))
            for i in range(layers)))
        self.ln = tnn.LayerNorm(dim, eps=1e-6)

    def forward(self, x, cls_only: bool = False):
        """``x`` already carries the position embedding.  ``cls_only``: normalise just the class-token row (LayerNorm
        is row-wise, and the classifier reads nothing else)."""
        x = self.dropout(x)
        if len(self.layers) and self.layers[0].gated:
            xn = EncoderBlock._ln(self.layers[0].ln_1, x)
            norms = [blk.ln_1 for blk in self.layers][1:] + [self.ln]
            for blk, ln in zip(self.layers, norms):
                x, xn = blk.gated_forward(x, xn, ln)
            return xn[:, 0] if cls_only else xn
        x = self.layers(x)
        if cls_only:
            x = x[:, 0]
        return EncoderBlock._ln(self.ln, x)


class AttentionPool(tnn.Module):
    """``[B, S, D] -> [B, D]``: one learned query per head attends to all tokens."""

    def __init__(self, dim: int, heads: int):
        super().__init__()
        self.num_heads = heads
        self.query = tnn.Parameter(torch.empty(1, 1, dim).normal_(std=0.02))
        self.kv_proj = pnn.Linear(dim, 2 * dim)
        self.out_proj = pnn.Linear(dim, dim)
        for m in (self.kv_proj, self.out_proj):
            tnn.init.xavier_uniform_(m.weight)
            tnn.init.zeros_(m.bias)

    def forward(self, x):
        q = self.query.to(x.dtype).expand(x.shape[0], -1, -1)
        return self.out_proj(cross_attention(q, self.kv_proj(x), self.num_heads)[:, 0])


class VisionTransformer(tnn.Module):
    def __init__(self, image_size=224, patch_size=16, layers=12, heads=12, dim=768, mlp_dim=3072,
                 num_classes=1000, dropout=0.0, rel_pos_bias=False, layer_scale=None, post_norm=False, pool="token"):
        super().__init__()
        if pool not in ("token", "attention"):
            raise ValueError(f"pool {pool!r}: 'token' or 'attention'")
        assert image_size % patch_size == 0
        self.image_size, self.patch_size, self.hidden_dim = image_size, patch_size, dim
        self.conv_proj = pnn.Conv2d(3, dim, patch_size, patch_size)
        seq = (image_size // patch_size) ** 2 + 1
        self.class_token = tnn.Parameter(torch.zeros(1, 1, dim))
        side = image_size // patch_size
        positions = pnn.grid_position_buckets(side, side) if rel_pos_bias else None
        self.encoder = Encoder(seq, layers, heads, dim, mlp_dim, dropout, positions, layer_scale, post_norm)
        self.pool = AttentionPool(dim, heads) if pool == "attention" else None
        self.heads = tnn.Sequential(OrderedDict(head=pnn.Linear(dim, num_classes)))
        fan_in = 3 * patch_size * patch_size
        tnn.init.trunc_normal_(self.conv_proj.weight, std=math.sqrt(1.0 / fan_in))
        tnn.init.zeros_(self.conv_proj.bias)
        tnn.init.zeros_(self.heads.head.weight)
        tnn.init.zeros_(self.heads.head.bias)

    def forward(self, x):
        # patch embedding: a stride = kernel conv is a GEMM over the extracted patches; then class token +
        # position embedding in one pass
        tok = patch_embed(x, self.conv_proj.weight, self.conv_proj.bias, self.patch_size)  # [b, tokens, dim]
        x = vit_embed(tok, self.class_token, self.encoder.pos_embedding)
        if self.pool is not None:
            return self.heads(self.pool(self.encoder(x)))
        x = self.encoder(x, cls_only=True)
        return self.heads(x)


def vit_b_16(num_classes=1000, image_size=224, **kw):
    return VisionTransformer(image_size, 16, 12, 12, 768, 3072, num_classes, **kw)


def vit_ti_16(num_classes=1000, image_size=224, **kw):
    """ViT-Tiny/16: width 192, 3 heads of 64."""
    return VisionTransformer(image_size, 16, 12, 3, 192, 768, num_classes, **kw)


def vit_s_16(num_classes=1000, image_size=224, **kw):
    """ViT-Small/16: width 384, 6 heads of 64."""
    return VisionTransformer(image_size, 16, 12, 6, 384, 1536, num_classes, **kw)


def vit_l_16(num_classes=1000, image_size=224, **kw):
    """ViT-Large/16 (torchvision ``vit_l_16`` keys): 24 layers, width 1024, 16 heads of 64."""
    return VisionTransformer(image_size, 16, 24, 16, 1024, 4096, num_classes, **kw)


def vit_tiny_test(num_classes=10, image_size=32, **kw):
    """A 2-layer toy of the same architecture for CPU tests: width 32, ONE head of 32 (the smallest head the fused
    attention kernels take, so that the toy runs without an oracle op on a GPU too)."""
    return VisionTransformer(image_size, 8, 2, 1, 32, 64, num_classes, **kw)
