"""A linear-attention language model: trained on whole sequences, served token by token.

Each block is pre-norm residual
    x += mixer(layer_norm(x));  x += swiglu(layer_norm(x))
and the mixer a linear attention with one learned decay a head:
    q, k, v, gate = x W;  o = linear_attention(q, k, v, log decay)
    y = (layer_norm(o) per head * silu(gate)) Wout
Training and prompts run the chunked form and single tokens the recurrent one, on the state that a
prompt leaves.  The MLP keeps its hidden activation in 8 bits between the passes (delta_kernels'
swiglu_q8): 2.06 M bytes a token of width M, where the activation and its product in bfloat16 take 6 M.
Projections and the MLP are GEMMs in `compute_dtype`, over float32 weights.  It has no counterpart in the
reference; delta_mixers.model holds the gated-delta-rule model.

    python -m delta_mixers.linear     trains a small model for a few steps and continues a prompt
"""
from __future__ import annotations

import functools
import math
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

import delta_kernels as dk


@dataclass
class LinearLMConfig:
    vocab: int = 32768
    d_model: int = 512
    layers: int = 8
    heads: int = 8
    key_dim: int = 64
    value_dim: int = 64
    mlp_width: int = 1408
    norm_epsilon: float = 1e-5
    compute_dtype: torch.dtype = torch.bfloat16


def _linear(i: int, o: int, device) -> torch.nn.Parameter:
    return torch.nn.Parameter(torch.randn(o, i, device=device) * i ** -0.5)


def _mm(x, w):
    return F.linear(x, w.to(x.dtype))


class LayerNorm(torch.nn.Module):
    def __init__(self, width: int, epsilon: float, bias: bool = True, device=None):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(width, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(width, device=device)) if bias else None
        self.epsilon = epsilon

    def forward(self, x):
        return dk.layer_norm(x, self.weight, self.bias, self.epsilon)


class LinearMixer(torch.nn.Module):
    """Input projections packed in one weight, rows [q | k | v | gate]."""

    def __init__(self, cfg: LinearLMConfig, device=None):
        super().__init__()
        self.cfg = cfg
        D, H, K, V = cfg.d_model, cfg.heads, cfg.key_dim, cfg.value_dim
        self.in_proj = _linear(D, 2 * H * K + 2 * H * V, device)
        self.out = _linear(H * V, D, device)
        self.norm = LayerNorm(V, cfg.norm_epsilon, False, device)
        # exp(-softplus(decay)): memories from 4 to 512 tokens over the heads
        rate = torch.logspace(math.log10(1 / 4), math.log10(1 / 512), H, device=device)
        self.decay = torch.nn.Parameter(torch.log(torch.expm1(rate)))

    def _split(self, x):
        B, T, _ = x.shape
        H, K, V = self.cfg.heads, self.cfg.key_dim, self.cfg.value_dim
        q, k, v, gate = _mm(x, self.in_proj).split((H * K, H * K, H * V, H * V), -1)
        return ((q * K ** -0.5).view(B, T, H, K), k.view(B, T, H, K), v.view(B, T, H, V), gate)

    def _join(self, o, gate):
        return _mm(self.norm(o).reshape(gate.shape) * F.silu(gate), self.out)

    def forward(self, x, valid=None, reset=None, state=None):
        """x [B, T, d_model]; returns (y, state after the last token)."""
        q, k, v, gate = self._split(x)
        o, state = dk.linear_attention(q, k, v, -F.softplus(self.decay), valid, reset, state)
        return self._join(o, gate), state

    def step(self, x, state):
        """One token a sequence, x [B, 1, d_model]; the state is updated in place.  Without gradients."""
        q, k, v, gate = self._split(x)
        return self._join(dk.linear_attention_step(state, q, k, v, -F.softplus(self.decay)), gate)


class _Q8Mlp(torch.autograd.Function):
    """r = swiglu(x w13^T) w2^T, keeping only x and the hidden activation in 8 bits for the backward,
    which recomputes the product that w2's gradient reads."""

    @staticmethod
    def forward(ctx, x, w13, w2):
        a, codes, exps = dk.swiglu_q8_forward(torch.mm(x, w13.t()))
        ctx.save_for_backward(x, codes, exps, w13, w2)
        return torch.mm(a, w2.t())

    @staticmethod
    @once_differentiable
    def backward(ctx, dr):
        x, codes, exps, w13, w2 = ctx.saved_tensors
        dr = dr.contiguous()
        dh, a = dk.swiglu_q8_backward(codes, exps, torch.mm(dr, w2), ctx.needs_input_grad[2])
        dx = torch.mm(dh, w13) if ctx.needs_input_grad[0] else None
        dw13 = torch.mm(dh.t(), x) if ctx.needs_input_grad[1] else None
        dw2 = torch.mm(dr.t(), a) if ctx.needs_input_grad[2] else None
        return dx, dw13, dw2


class Q8SwiGLU(torch.nn.Module):
    """w13 packs the gate and up projections ([w1 | w3] rows)."""

    def __init__(self, cfg: LinearLMConfig, device=None):
        super().__init__()
        self.w13 = _linear(cfg.d_model, 2 * cfg.mlp_width, device)
        self.w2 = _linear(cfg.mlp_width, cfg.d_model, device)

    def forward(self, x):
        rows = x.reshape(-1, x.shape[-1])
        return _Q8Mlp.apply(rows, self.w13.to(x.dtype), self.w2.to(x.dtype)).view(x.shape)


class LinearBlock(torch.nn.Module):
    def __init__(self, cfg: LinearLMConfig, device=None):
        super().__init__()
        self.cfg = cfg
        self.norm1 = LayerNorm(cfg.d_model, cfg.norm_epsilon, True, device)
        self.norm2 = LayerNorm(cfg.d_model, cfg.norm_epsilon, True, device)
        self.mixer = LinearMixer(cfg, device)
        self.mlp = Q8SwiGLU(cfg, device)

    def _mlp(self, x):
        return x + self.mlp(self.norm2(x).to(self.cfg.compute_dtype)).float()

    def forward(self, x, valid=None, reset=None, state=None):
        """x [B, T, d_model] float32 residual stream; returns (x, state)."""
        y, state = self.mixer(self.norm1(x).to(self.cfg.compute_dtype), valid, reset, state)
        return self._mlp(x + y.float()), state

    def step(self, x, state):
        y = self.mixer.step(self.norm1(x).to(self.cfg.compute_dtype), state)
        return self._mlp(x + y.float())


def scored(valid, present, reset):
    """Which of tokens 1 .. T - 1 have a score, [B, T - 1] or None (all), from the masks [B, T] of score."""
    if present is None and reset is None:
        return None if valid is None else valid[:, 1:]
    on = [] if valid is None else [valid[:, 1:] != 0]
    if present is not None:
        on += [present[:, 1:] != 0, present[:, :-1] != 0]
    if reset is not None:
        on.append(reset[:, 1:] == 0)
    return functools.reduce(torch.logical_and, on)


class LinearLM(torch.nn.Module):
    def __init__(self, cfg: LinearLMConfig, device=None):
        super().__init__()
        self.cfg = cfg
        self.embed = torch.nn.Parameter(torch.randn(cfg.vocab, cfg.d_model, device=device) * 0.02)
        self.blocks = torch.nn.ModuleList(LinearBlock(cfg, device) for _ in range(cfg.layers))
        self.norm = LayerNorm(cfg.d_model, cfg.norm_epsilon, True, device)

    def _logits(self, x):
        return _mm(self.norm(x).to(self.cfg.compute_dtype), self.embed)

    def features(self, tokens, valid=None, reset=None,
                 states: Optional[List[torch.Tensor]] = None) -> Tuple[torch.Tensor, list]:
        """tokens [B, T] -> (final-norm features [B, T, d_model] in compute_dtype, the blocks' states
        after the last token)."""
        x, out = self.embed[tokens], []
        for i, blk in enumerate(self.blocks):
            x, s = blk(x, valid, reset, None if states is None else states[i])
            out.append(s)
        return self.norm(x).to(self.cfg.compute_dtype), out

    def forward(self, tokens, valid=None, reset=None):
        """tokens [B, T] -> logits [B, T, vocab] in compute_dtype."""
        return _mm(self.features(tokens, valid, reset)[0], self.embed)

    def loss(self, tokens):
        """Mean next-token cross entropy (the tied head and the loss in one operator)."""
        h, _ = self.features(tokens[:, :-1])
        return dk.linear_cross_entropy(h.reshape(-1, self.cfg.d_model),
                                       self.embed.to(self.cfg.compute_dtype),
                                       tokens[:, 1:].reshape(-1))

    def score(self, tokens, valid=None, top: int = 0, temperature: float = 1.0, present=None,
              reset=None) -> dk.TokenLogProbs:
        """Log probabilities of tokens 1 .. T - 1 after those before them, [B, T - 1], their entropy and
        the top alternatives; zeros where valid [B, T] is 0.  valid says which tokens are scored, all are
        read (a prompt, say); present [B, T], 0 at padding, and reset [B, T], 1 where a document begins,
        are forward's valid and reset: a token is scored after the one right before it, so padding, what
        follows it, and a document's first token give zeros."""
        logits = self(tokens[:, :-1], *(None if m is None else m[:, :-1] for m in (present, reset)))
        return dk.token_log_probs(logits, tokens[:, 1:], top, scored(valid, present, reset), temperature)

    @torch.no_grad()
    def prefill(self, tokens, states=None):
        """A prompt, or its continuation: (logits of the last token [B, vocab], states)."""
        h, states = self.features(tokens, None, None, states)
        return _mm(h[:, -1], self.embed), states

    @torch.no_grad()
    def step(self, tokens, states):
        """One token a sequence, tokens [B]; the states are updated in place.  Returns logits."""
        x = self.embed[tokens][:, None]
        for blk, s in zip(self.blocks, states):
            x = blk.step(x, s)
        return self._logits(x)[:, 0]


def main():
    torch.manual_seed(0)
    cfg = LinearLMConfig(vocab=256, d_model=256, layers=2, heads=4, mlp_width=704)
    model = LinearLM(cfg, device="cuda")
    opt = dk.FusedAdamW(model.parameters(), lr=3e-3)
    text = torch.tensor(list(__doc__.encode()), device="cuda")
    for i in range(200):
        start = torch.randint(0, len(text) - 129, (16, 1), device="cuda")
        tokens = text[start + torch.arange(129, device="cuda")]
        opt.zero_grad(set_to_none=True)
        loss = model.loss(tokens)
        loss.backward()
        opt.step()
        if i % 50 == 49:
            print(f"step {i + 1}: loss {loss.item():.3f}", flush=True)
    logits, states = model.prefill(text[None, :40])
    out = []
    for _ in range(60):
        token = logits.argmax(-1)
        out.append(int(token))
        logits = model.step(token, states)
    print(repr(bytes(text[:40].tolist()).decode()), "->", repr(bytes(out).decode("latin1")))


if __name__ == "__main__":
    main()
