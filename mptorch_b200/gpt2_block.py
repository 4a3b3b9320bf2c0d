"""A GPT-2-small-shaped transformer block built from the quantized layers: the caller-side workload of
benchmark config 5 (d=768, 12 heads, MLP 3072), wired like the reference's example
``examples/gpt/mptorch_shakespeare_softmax_gpt.py:246-337`` (pre-LN block: QLayerNorm -> attention with QLinear
projections, qmatmul for QK^T and PV, QSoftmax -> QLayerNorm -> QLinear MLP with GELU).
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from .number import FloatingPoint
from .quant import (MXCache, QAffineFormats, QLayerNorm, QLayerNormFormats, QLinear, QPackedLinear, QSoftmax, QSoftmaxFormats, mx_attention,
                    mx_cache_write)
from .quant.functional import qmatmul

__all__ = ["BlockConfig", "QBlock", "QTinyGPT", "ServedBlock", "ServedGPT", "default_formats"]


class BlockConfig:
    def __init__(self, d_model=768, n_head=12, d_mlp=3072, vocab=50257, seq_len=1024):
        self.d_model, self.n_head, self.d_mlp, self.vocab, self.seq_len = d_model, n_head, d_mlp, vocab, seq_len


def default_formats(add=FloatingPoint(5, 10, True, False), mul=FloatingPoint(4, 3, True, False)):
    """fwd_mac = bwd_mac = (add e5m10, mul e4m3) for the GEMMs (tuple order is (add, mul)); softmax and layernorm in
    the add format."""
    affine = QAffineFormats(fwd_mac=(add, mul), bwd_mac=(add, mul), fwd_rnd="nearest", bwd_rnd="nearest")
    softmax = QSoftmaxFormats(fwd_off=add, fwd_exp=add, fwd_acc=add, bwd_add=add, bwd_mul=add)
    lnorm = QLayerNormFormats(fwd_acc=add, fwd_mul=add, fwd_div=add, fwd_sqrt=add, bwd_acc=add, bwd_mul=add, bwd_div=add)
    return affine, softmax, lnorm


class QBlock(nn.Module):
    def __init__(self, cfg: BlockConfig, formats=None):
        super().__init__()
        affine, softmax, lnorm = formats or default_formats()
        self.cfg, self.affine = cfg, affine
        d = cfg.d_model
        self.ln1 = QLayerNorm(d, lnorm)
        self.qkv = QLinear(d, 3 * d, affine)
        self.proj = QLinear(d, d, affine)
        self.softmax = QSoftmax(-1, softmax)
        self.ln2 = QLayerNorm(d, lnorm)
        self.fc = QLinear(d, cfg.d_mlp, affine)
        self.out = QLinear(cfg.d_mlp, d, affine)
        for m in (self.qkv, self.proj, self.fc, self.out):
            nn.init.normal_(m.weight, std=0.02)
            nn.init.zeros_(m.bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        B, T, d = x.shape
        h = self.cfg.n_head
        q, k, v = self.qkv(self.ln1(x)).split(d, dim=2)
        q = q.view(B, T, h, d // h).transpose(1, 2).contiguous()
        k = k.view(B, T, h, d // h).transpose(1, 2).contiguous()
        v = v.view(B, T, h, d // h).transpose(1, 2).contiguous()
        att = qmatmul(q, k.transpose(-2, -1), self.affine) * (1.0 / math.sqrt(d // h))
        mask = torch.ones(T, T, device=x.device, dtype=torch.bool).tril()
        att = self.softmax(att.masked_fill(~mask, float("-inf")))
        y = qmatmul(att, v, self.affine).transpose(1, 2).contiguous().view(B, T, d)
        x = x + self.proj(y)
        return x + self.out(torch.nn.functional.gelu(self.fc(self.ln2(x))))


class QTinyGPT(nn.Module):
    """Token embedding -> one quantized block -> plain fp32 head (the head and the loss stay in fp32)."""

    def __init__(self, cfg: BlockConfig, formats=None):
        super().__init__()
        self.cfg = cfg
        self.wte = nn.Embedding(cfg.vocab, cfg.d_model)
        self.wpe = nn.Embedding(cfg.seq_len, cfg.d_model)
        self.block = QBlock(cfg, formats)
        nn.init.normal_(self.wte.weight, std=0.02)
        nn.init.normal_(self.wpe.weight, std=0.02)

    def forward(self, idx: torch.Tensor) -> torch.Tensor:
        T = idx.shape[1]
        x = self.wte(idx) + self.wpe(torch.arange(T, device=idx.device))
        return self.block(x)

    def macs_per_step(self, batch: int, seq: int) -> int:
        """Simulated MACs of one forward+backward pass (backward = 2x forward for every GEMM)."""
        c = self.cfg
        rows = batch * seq
        fwd = rows * c.d_model * (3 * c.d_model + c.d_model + 2 * c.d_mlp) + 2 * batch * c.n_head * seq * seq * (c.d_model // c.n_head)
        return 3 * fwd


class ServedBlock(nn.Module):
    """A trained ``QBlock`` as it answers: the four weights packed in a 4-bit block format, K and V in the pages of an MX cache.
    New tokens come in chunks or one by one; ``pages``, ``lens`` and ``starts`` are those of ``quant.mx_attention``."""

    def __init__(self, block: QBlock, weights: str = "mxfp4"):
        super().__init__()
        self.n_head, self.ln1, self.ln2 = block.cfg.n_head, block.ln1, block.ln2
        self.qkv, self.proj, self.fc, self.out = (QPackedLinear.from_linear(m, weights) for m in (block.qkv, block.proj, block.fc, block.out))

    @torch.no_grad()
    def forward(self, x: torch.Tensor, cache: MXCache, pages: torch.Tensor, lens: torch.Tensor, starts: torch.Tensor | None = None) -> torch.Tensor:
        q, k, v = (t.unflatten(-1, (self.n_head, -1)) for t in self.qkv(self.ln1(x)).chunk(3, dim=-1))
        mx_cache_write(k, v, cache, pages, lens, starts)
        x = x + self.proj(mx_attention(q, cache, pages, lens, starts).flatten(-2))
        return x + self.out(torch.nn.functional.gelu(self.fc(self.ln2(x))))


class ServedGPT(nn.Module):
    """A trained ``QTinyGPT`` as it answers: ``ServedBlock`` between the embeddings and the (tied) packed vocabulary head."""

    def __init__(self, model: QTinyGPT, weights: str = "mxfp4"):
        super().__init__()
        self.cfg, self.wte, self.wpe = model.cfg, model.wte, model.wpe
        self.block = ServedBlock(model.block, weights)
        self.head = QPackedLinear(model.wte.weight, None, weights)

    def new_cache(self, pages: int, page: int = 64, elem_format: str = "e4m3") -> MXCache:
        return MXCache.empty(pages, self.cfg.n_head, self.cfg.d_model // self.cfg.n_head, page, elem_format, self.wte.weight.device)

    @torch.no_grad()
    def forward(self, idx: torch.Tensor, cache: MXCache, pages: torch.Tensor, lens: torch.Tensor) -> torch.Tensor:
        """Logits of the new tokens ``idx`` [sequences, new]; ``lens`` counts each sequence with them."""
        at = lens[:, None] - idx.shape[1] + torch.arange(idx.shape[1], device=idx.device)
        x = self.wte(idx) + self.wpe(at.clamp(0, self.cfg.seq_len - 1))
        return self.head(self.block(x, cache, pages, lens))

    @torch.no_grad()
    def generate(self, idx: torch.Tensor, new: int, page: int = 64, elem_format: str = "e4m3") -> torch.Tensor:
        """The most likely continuation of prompts of one length: [sequences, prompt + new] tokens."""
        b, t = idx.shape
        if t < 1 or t + new > self.cfg.seq_len:
            raise ValueError("prompt and continuation must fit seq_len")
        width = -(-(t + new) // page)
        cache = self.new_cache(b * width, page, elem_format)
        pages = torch.arange(b * width, device=idx.device, dtype=torch.int32).view(b, width)
        lens, chunk = torch.full((b,), t, device=idx.device, dtype=torch.int32), idx
        for _ in range(new):
            chunk = self(chunk, cache, pages, lens)[:, -1].argmax(-1, keepdim=True)
            idx = torch.cat([idx, chunk], dim=1)
            lens = lens + 1
        return idx
