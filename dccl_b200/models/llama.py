"""Llama-style decoder used by the data-parallel training benchmark.

Plain PyTorch: RMSNorm, rotary position embedding, grouped-query attention through
``scaled_dot_product_attention``, SwiGLU MLP, untied output head. ``LlamaConfig.tinyllama_1b`` is
the benchmark's shape: 22 layers, hidden 2048, 32 heads, 4 KV heads, FFN 5632, vocabulary 32000
(about 1.1 B parameters). The model is only the workload whose gradients the library all-reduces;
the "no library GEMM" rule of this project applies to the communication paths, not to it.

With ``LlamaConfig(fused=True)`` the same modules compute with the operators of ``dccl_b200.ops.decoder``: each residual add in one pass with
the norm after it, rotary positions of queries and keys in one launch, and the gated projections as one product (parameters and state
dict stay the same). A module that is more than what stands here (another one put in its place, a bias, hooks) is called, and so is what an
operator does not take (the gated projections in float32 on the GPU or under autocast, fake and transformed tensors); the others around it stay fused.
"""
import functools
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.nn.modules.module import _has_any_global_hook

from ..ops import decoder as ops


@dataclass
class LlamaConfig:
    vocab_size: int = 32000
    hidden: int = 2048
    layers: int = 22
    heads: int = 32
    kv_heads: int = 4
    ffn: int = 5632
    max_seq: int = 2048
    rope_theta: float = 10000.0
    eps: float = 1e-5
    fused: bool = False

    @staticmethod
    def tinyllama_1b():
        return LlamaConfig()

    @staticmethod
    def tiny():
        return LlamaConfig(vocab_size=512, hidden=128, layers=2, heads=4, kv_heads=2, ffn=256, max_seq=128)

    def num_params(self):
        hd = self.hidden // self.heads
        attn = self.hidden * self.hidden * 2 + 2 * self.hidden * hd * self.kv_heads
        mlp = 3 * self.hidden * self.ffn
        return self.layers * (attn + mlp + 2 * self.hidden) + 2 * self.vocab_size * self.hidden + self.hidden


class RMSNorm(nn.Module):
    def __init__(self, dim, eps):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim))
        self.eps = eps

    def forward(self, x):
        v = x.float()
        v = v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + self.eps)
        return (v * self.weight.float()).to(x.dtype)


def rope_tables(seq, head_dim, theta, device):
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, device=device, dtype=torch.float32) / head_dim))
    t = torch.arange(seq, device=device, dtype=torch.float32)
    f = torch.outer(t, inv)
    return f.cos(), f.sin()


def apply_rope(x, cos, sin):
    # x: [B, H, S, D]; rotate pairs (even, odd halves)
    d = x.shape[-1] // 2
    x1, x2 = x[..., :d].float(), x[..., d:].float()
    c, s = cos[None, None, : x.shape[2]], sin[None, None, : x.shape[2]]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).to(x.dtype)


class Attention(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.h, self.kv, self.hd = cfg.heads, cfg.kv_heads, cfg.hidden // cfg.heads
        self.q = nn.Linear(cfg.hidden, cfg.heads * self.hd, bias=False)
        self.k = nn.Linear(cfg.hidden, cfg.kv_heads * self.hd, bias=False)
        self.v = nn.Linear(cfg.hidden, cfg.kv_heads * self.hd, bias=False)
        self.o = nn.Linear(cfg.heads * self.hd, cfg.hidden, bias=False)

    def forward(self, x, cos, sin):
        b, s, _ = x.shape
        q = self.q(x).view(b, s, self.h, self.hd).transpose(1, 2)
        k = self.k(x).view(b, s, self.kv, self.hd).transpose(1, 2)
        v = self.v(x).view(b, s, self.kv, self.hd).transpose(1, 2)
        q, k = apply_rope(q, cos, sin), apply_rope(k, cos, sin)
        out = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=self.kv != self.h)
        return self.o(out.transpose(1, 2).reshape(b, s, self.h * self.hd))

    def fused(self, x, at):
        b, s, _ = x.shape
        return self.o(attend(self.q(x).view(b, s, self.h, self.hd), self.k(x).view(b, s, self.kv, self.hd), self.v(x).view(b, s, self.kv, self.hd), at,
                             self.kv != self.h))


# ---- the fused form. Every operator stands for modules that are then not called, so each use asks first whether calling them would do more.

_OWN_FORWARD = {kind: kind.forward for kind in (nn.Linear, RMSNorm, Attention)}


def untouched(module, kind):
    """Whether a call of `module` computes what `kind` says and nothing else: of that very class, with neither a bias nor hooks nor another forward."""
    return (type(module) is kind and kind.forward is _OWN_FORWARD[kind] and "forward" not in module.__dict__
            and getattr(module, "bias", None) is None and module._compiled_call_impl is None and not _has_any_global_hook()
            and not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks))


class Positions:
    """The frequencies of the rotary positions, and their tables where a module has to be called that takes those."""

    def __init__(self, seq, head_dim, theta, device):
        self.freqs, self._tables = ops.rotary_frequencies(head_dim, theta, device=device), (seq, head_dim, theta, device)

    @functools.cached_property
    def tables(self):
        return rope_tables(*self._tables)


_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def taken(x):
    """Whether x is a tensor that the operators take: of their types and devices, with values of its own."""
    return x.dtype in _TYPES and x.device.type in ("cpu", "cuda") and type(x) in (torch.Tensor, nn.Parameter) and not torch._C._functorch.is_functorch_wrapped_tensor(x)


def attend(q, k, v, at, grouped):
    """Causal attention of [batch, seq, heads, head dim], whose queries and keys are turned by their positions first: [batch, seq, heads * head dim].
    grouped: k and v have fewer heads."""
    if taken(q):
        q, k = ops.rotary(q, k, at.freqs)
    else:
        q, k = (apply_rope(t.transpose(1, 2), *at.tables).transpose(1, 2) for t in (q, k))
    out = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True, enable_gqa=grouped)
    return out.transpose(1, 2).flatten(2)


def attention(module, n, at, kind):
    return module.fused(n, at) if untouched(module, kind) else module(n, *at.tables)


def gated(n, gate, up):
    if (untouched(gate, nn.Linear) and untouched(up, nn.Linear) and taken(n) and n.dtype in _TYPES[:3 - n.is_cuda] and gate.weight.dtype == up.weight.dtype == n.dtype
            and not torch.is_autocast_enabled(n.device.type)):
        return ops.gated_linear(n, gate.weight, up.weight)
    return F.silu(gate(n)) * up(n)


def norms(norm, x):
    """Whether the operators compute what `norm` does with x."""
    return untouched(norm, RMSNorm) and taken(x) and norm.weight.dtype in (x.dtype, torch.float32)


def norm_of(x, norm):
    if norm is None:
        return None
    return ops.rms_norm(x, norm.weight, eps=norm.eps) if norms(norm, x) else norm(x)


def add_norm(x, branch, norm):
    """x + branch, and the norm of it; None where what comes next takes no norm."""
    if norm is not None and norms(norm, x) and torch.promote_types(x.dtype, branch.dtype) == x.dtype:
        return ops.residual_norm(x, branch.to(x.dtype), norm.weight, eps=norm.eps)
    x = x + branch
    return x, norm_of(x, norm)


def run_fused(x, blocks, last, at, kind):
    """The blocks and the last norm. A block that is not an untouched one of its kind is called as a module."""
    entries = [blk.n1 if untouched(blk, kind) else None for blk in blocks] + [last]
    n = norm_of(x, entries[0])
    for blk, entry, after in zip(blocks, entries, entries[1:]):
        if entry is None:
            x = blk(x, *at.tables)
            n = norm_of(x, after)
        else:
            x, n = blk.fused(x, n, at, after)
    return n


class Block(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.n1, self.n2 = RMSNorm(cfg.hidden, cfg.eps), RMSNorm(cfg.hidden, cfg.eps)
        self.attn = Attention(cfg)
        self.gate = nn.Linear(cfg.hidden, cfg.ffn, bias=False)
        self.up = nn.Linear(cfg.hidden, cfg.ffn, bias=False)
        self.down = nn.Linear(cfg.ffn, cfg.hidden, bias=False)

    def forward(self, x, cos, sin):
        x = x + self.attn(self.n1(x), cos, sin)
        h = self.n2(x)
        return x + self.down(F.silu(self.gate(h)) * self.up(h))

    def fused(self, x, n, at, after):
        """(x, n) after this block, from x and its norm n: n is the norm of x by `after`, which comes next."""
        x, n = add_norm(x, attention(self.attn, n, at, Attention), self.n2)
        return add_norm(x, self.down(gated(n, self.gate, self.up)), after)


_OWN_FORWARD[Block] = Block.forward


class LlamaDecoder(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.cfg = cfg
        self.embed = nn.Embedding(cfg.vocab_size, cfg.hidden)
        self.blocks = nn.ModuleList([Block(cfg) for _ in range(cfg.layers)])
        self.norm = RMSNorm(cfg.hidden, cfg.eps)
        self.head = nn.Linear(cfg.hidden, cfg.vocab_size, bias=False)
        self.apply(self._init)

    @staticmethod
    def _init(m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, std=0.02)

    def forward(self, tokens):
        x = self.embed(tokens)
        if self.cfg.fused:
            at = Positions(tokens.shape[1], self.cfg.hidden // self.cfg.heads, self.cfg.rope_theta, tokens.device)
            return self.head(run_fused(x, self.blocks, self.norm, at, Block))
        cos, sin = rope_tables(tokens.shape[1], self.cfg.hidden // self.cfg.heads, self.cfg.rope_theta, tokens.device)
        for blk in self.blocks:
            x = blk(x, cos, sin)
        return self.head(self.norm(x))

    def loss(self, tokens):
        """Next-token cross entropy on a batch of token ids [B, S]."""
        logits = self.forward(tokens[:, :-1])
        return F.cross_entropy(logits.reshape(-1, logits.shape[-1]).float(), tokens[:, 1:].reshape(-1))
