"""LLaMA-style decoder hosting the MoC FFN (build_model of moc/model.py:147-148).

Only the FFN is this library's hot path.  The rest of the decoder is the
smallest host that keeps build_model(config, ffn_type=...) and its
state_dict keys interchangeable with the reference (moc/model.py:20-148):
pre-norm blocks of RMSNorm (f32 statistics), rotary position embedding on
interleaved (even, odd) feature pairs, causal SDPA attention, and a tied or
separate LM head with the shifted next-token loss.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from .block import (attention_half, attention_half_ok, bare, final_norm, lm_head, lm_head_ok, next_token_loss,
                    next_token_loss_ok, plain, runs_stock, stock_method)
from .config import MoCConfig
from .ffn import MoCSwiGLUFFN, block_ffn, block_ffn_f32_ok, block_ffn_ok, build_ffn
from .losses import cross_entropy_f32, linear_cross_entropy, linear_distillation

FFN_TYPES = ("dense", "moc", "moc_gcp", "moc_2_8", "moc_post_silu_abs")


@stock_method()
class RMSNorm(nn.Module):
    """y = bf16/f32-cast(x / rms(x)) * weight, statistics in float32."""

    def __init__(self, dim: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x):
        xf = x.float()
        inv_rms = torch.rsqrt(torch.mean(xf * xf, dim=-1, keepdim=True) + self.eps)
        return (xf * inv_rms).to(x.dtype) * self.weight


def rotary_tables(head_dim: int, max_len: int, theta: float = 10000.0):
    """cos/sin [max_len, head_dim // 2] of the angle pos * theta^(-2i / head_dim)."""
    inv_freq = 1.0 / torch.pow(theta, torch.arange(0, head_dim, 2, dtype=torch.float32) / head_dim)
    angle = torch.arange(max_len, dtype=torch.float32)[:, None] * inv_freq[None, :]
    return torch.cos(angle), torch.sin(angle)


def rotate_pairs(x, cos, sin):
    """Rotate features (2i, 2i+1) of x [batch, heads, seq, head_dim] by the
    angle of (position, i)."""
    seq = x.shape[-2]
    c, s = cos[:seq], sin[:seq]
    even, odd = x.unflatten(-1, (-1, 2)).unbind(-1)
    return torch.stack((even * c - odd * s, even * s + odd * c), dim=-1).flatten(-2)


@stock_method()
class CausalSelfAttention(nn.Module):
    def __init__(self, config: MoCConfig):
        super().__init__()
        d = config.hidden_size
        self.num_heads = config.num_attention_heads
        self.head_dim = d // self.num_heads
        self.qkv_proj = nn.Linear(d, 3 * d, bias=False)
        self.out_proj = nn.Linear(d, d, bias=False)
        cos, sin = rotary_tables(self.head_dim, config.max_seq_len, config.rope_theta)
        self.register_buffer("rope_cos", cos, persistent=False)
        self.register_buffer("rope_sin", sin, persistent=False)

    def forward(self, x):
        batch, seq, d = x.shape
        # [batch, seq, 3 * d] -> three [batch, heads, seq, head_dim] views
        heads = self.qkv_proj(x).view(batch, seq, 3, self.num_heads, self.head_dim).permute(2, 0, 3, 1, 4)
        q = rotate_pairs(heads[0], self.rope_cos, self.rope_sin)
        k = rotate_pairs(heads[1], self.rope_cos, self.rope_sin)
        ctx = F.scaled_dot_product_attention(q, k, heads[2], is_causal=True)
        return self.out_proj(ctx.permute(0, 2, 1, 3).reshape(batch, seq, d))


class TransformerBlock(nn.Module):
    """Pre-norm residual block: x + attn(norm(x)), then x + ffn(norm(x))."""

    def __init__(self, config: MoCConfig, ffn_type: str = "dense"):
        super().__init__()
        self.attn_norm = RMSNorm(config.hidden_size, eps=config.rms_norm_eps)
        self.attn = CausalSelfAttention(config)
        self.ffn_norm = RMSNorm(config.hidden_size, eps=config.rms_norm_eps)
        self.ffn = build_ffn(config.hidden_size, config.intermediate_size, ffn_type=ffn_type,
                             k=config.k)

    def forward(self, x):
        if isinstance(self.ffn, MoCSwiGLUFFN) and attention_half_ok(x, self.attn_norm, RMSNorm, self.attn,
                                                                    CausalSelfAttention):
            # one Function over the library's kernels (same result within bf16
            # rounding)
            h = attention_half(x, self.attn_norm, self.attn)
        else:
            h = x + self.attn(self.attn_norm(x))
        if type(self.ffn_norm) is RMSNorm and bare(self.ffn_norm, self.ffn) and (
                block_ffn_ok(h, self.ffn_norm.weight, self.ffn) or
                block_ffn_f32_ok(h, self.ffn_norm.weight, self.ffn)):
            # MoC FFN: ffn_norm as one row kernel in front of it, the residual
            # add in its Down GEMM's epilogue (same result within bf16 rounding)
            return block_ffn(h, self.ffn_norm.weight, self.ffn_norm.eps, self.ffn)
        return h + self.ffn(self.ffn_norm(h))


@stock_method("_logits")
class LLaMAModel(nn.Module):
    def __init__(self, config: MoCConfig, ffn_type: str = "dense"):
        super().__init__()
        if ffn_type not in FFN_TYPES:
            raise ValueError(
                "ffn_type must be 'dense', 'moc', 'moc_gcp', 'moc_2_8', "
                f"or 'moc_post_silu_abs', got {ffn_type!r}"
            )
        self.config = config
        self.ffn_type = ffn_type
        self.tok_emb = nn.Embedding(config.vocab_size, config.hidden_size)
        self.blocks = nn.ModuleList(
            TransformerBlock(config, ffn_type=ffn_type) for _ in range(config.num_hidden_layers))
        self.norm = RMSNorm(config.hidden_size, eps=config.rms_norm_eps)
        self.lm_head = (None if config.tie_word_embeddings
                        else nn.Linear(config.hidden_size, config.vocab_size, bias=False))
        self._init_weights()

    @staticmethod
    def _init_module(module: nn.Module) -> None:
        # every projection and embedding table ~ N(0, 0.02); norms keep ones
        if isinstance(module, (nn.Linear, nn.Embedding)):
            nn.init.normal_(module.weight, mean=0.0, std=0.02)

    def _init_weights(self):
        self.apply(self._init_module)

    def num_parameters(self) -> int:
        return sum(p.numel() for p in self.parameters())

    def _logits(self, h):
        if self.lm_head is not None:
            return self.lm_head(h)
        return torch.matmul(h, self.tok_emb.weight.t())

    def _hidden(self, input_ids):
        h = self.tok_emb(input_ids)
        for block in self.blocks:
            h = block(h)
        return h

    def _head_weight(self):
        return self.tok_emb.weight if self.lm_head is None else getattr(self.lm_head, "weight", None)

    def _loss_rows(self, h):
        """The rows that the logits are made of, norm(h), and whether that is a product with
        the head's weight of which the losses' kernels read both."""
        head, weight = self.lm_head, self._head_weight()
        if not (h.is_cuda and runs_stock(self, "_logits") and plain(h, weight) and
                (head is None or (type(head) is nn.Linear and head.bias is None and bare(head)))):
            return self.norm(h), False
        x = final_norm(h, self.norm, RMSNorm)
        types = {x.dtype, weight.dtype}
        if torch.is_autocast_enabled("cuda"):
            taken = torch.get_autocast_dtype("cuda") == torch.bfloat16 and types <= {torch.bfloat16, torch.float32}
        else:
            taken = types in ({torch.bfloat16}, {torch.float32})
        return x, taken and plain(x)

    def loss(self, input_ids, labels, row_weight=None):
        """forward(input_ids, labels)[1] in f32 without the logits, which exist for a
        piece of the positions at a time (losses.linear_cross_entropy); of all positions
        off the device, in other types than distill's and where the head is not a plain
        product.  row_weight [batch, seq] (f32): the weight of position t's loss, against
        label t + 1."""
        x, taken = self._loss_rows(self._hidden(input_ids))
        target = F.pad(labels[:, 1:], (0, 1), value=-100)
        if taken:
            return linear_cross_entropy(x, self._head_weight(), target, row_weight)
        return cross_entropy_f32(self._logits(x), target, row_weight)

    def distill(self, input_ids, teacher_ids, teacher_logits, row_weight=None, *, temperature: float = 1.0):
        """The divergence of the model's logits from a teacher's top ones at the same
        positions, [batch, seq, words] ids and logits (losses.linear_distillation, which
        describes them and row_weight).  Device tensors in bf16 or f32, or either under
        bf16 autocast."""
        x, taken = self._loss_rows(self._hidden(input_ids))
        if not taken:
            raise ValueError("distill takes a plain LM head on the device, in bf16 or f32 or under bf16 autocast")
        return linear_distillation(x, self._head_weight(), teacher_ids, teacher_logits, row_weight, temperature=temperature)

    def forward(self, input_ids, labels=None):
        h = self._hidden(input_ids)
        weight = self._head_weight()
        if self.ffn_type != "dense" and runs_stock(self, "_logits") and \
                lm_head_ok(h, self.norm, RMSNorm, self.lm_head, weight):
            logits = lm_head(h, self.norm, weight)
        else:
            logits = self._logits(self.norm(h))
        if labels is None:
            return logits
        # next-token loss: position t is scored against label t + 1
        if self.ffn_type != "dense" and next_token_loss_ok(logits, labels):
            return logits, next_token_loss(logits, labels)
        pred = logits[:, :-1].flatten(0, 1)
        target = labels[:, 1:].flatten()
        return logits, F.cross_entropy(pred, target, ignore_index=-100)


def build_model(config: MoCConfig, ffn_type: str = "dense") -> LLaMAModel:
    return LLaMAModel(config, ffn_type=ffn_type)
