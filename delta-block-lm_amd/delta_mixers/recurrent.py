"""A language model whose mixers are gated linear recurrences: a state of one value a channel.

Each block is pre-norm residual
    x += mixer(layer_norm(x));  x += swiglu(layer_norm(x))
and the mixer a recurrence with a decay for each token and channel:
    u, r, gate = x W;  g = -2 sigmoid(r) softplus(decay)                       (log decay)
    h_t = exp(g_t) h_{t-1} + sqrt(1 - exp(2 g_t)) u_t;  y = (h * silu(gate)) Wout
Training and prompts run the scan, single tokens the step on the states that a prompt leaves: 4 bytes a
channel, where linear attention's heads (delta_mixers.linear) keep 4 K.  Matrices are trained by Muon, the
rest by FusedAdamW (make_optimizers).  A trained model is scored by the log probabilities of given tokens
(score), which also make a policy's loss (policy_loss).  It has no counterpart in the reference.

    python -m delta_mixers.recurrent     trains a small model for a few steps and continues a prompt
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch
import torch.nn.functional as F

import delta_kernels as dk

from .linear import LayerNorm, Q8SwiGLU, _linear, _mm, scored


@dataclass
class RecurrentLMConfig:
    vocab: int = 32768
    d_model: int = 512
    layers: int = 8
    width: int = 512  # channels of a mixer's recurrence
    mlp_width: int = 1408
    norm_epsilon: float = 1e-5
    compute_dtype: torch.dtype = torch.bfloat16


class RecurrentMixer(torch.nn.Module):
    """Input projections packed in one weight, rows [u | r | gate]."""

    def __init__(self, cfg: RecurrentLMConfig, device=None):
        super().__init__()
        self.in_proj = _linear(cfg.d_model, 3 * cfg.width, device)
        self.out = _linear(cfg.width, cfg.d_model, device)
        # at r = 0 exp(-softplus(decay)): memories from 2 to 512 tokens over the channels
        rate = torch.logspace(math.log10(1 / 2), math.log10(1 / 512), cfg.width, device=device)
        self.decay = torch.nn.Parameter(torch.log(torch.expm1(rate)))

    def _split(self, x):
        u, r, gate = _mm(x, self.in_proj).chunk(3, -1)
        g = -2 * torch.sigmoid(r.float()) * F.softplus(self.decay)
        rest = -torch.expm1(2 * g)
        if torch.is_grad_enabled():
            # for the gradient alone: 0 where a gate is closed (g = 0), where the root's is infinite
            rest = F.relu(rest)
        return (torch.sqrt(rest) * u).to(x.dtype), g, gate

    def _join(self, h, gate):
        return _mm(h * F.silu(gate), self.out)

    def forward(self, x, valid=None, reset=None, state=None):
        """x [B, T, d_model]; returns (y, state [B, width] after the last token)."""
        u, g, gate = self._split(x)
        h, state = dk.gated_recurrence(u, g, valid, reset, state)
        return self._join(h, gate), state

    def step(self, x, state):
        """One token a sequence, x [B, 1, d_model]; the state is updated in place.  Without gradients."""
        u, g, gate = self._split(x)
        return self._join(dk.gated_recurrence_step(state, u, g), gate)


class RecurrentBlock(torch.nn.Module):
    def __init__(self, cfg: RecurrentLMConfig, device=None):
        super().__init__()
        self.cfg = cfg
        self.norm1 = LayerNorm(cfg.d_model, cfg.norm_epsilon, True, device)
        self.norm2 = LayerNorm(cfg.d_model, cfg.norm_epsilon, True, device)
        self.mixer = RecurrentMixer(cfg, device)
        self.mlp = Q8SwiGLU(cfg, device)

    def _mlp(self, x):
        return x + self.mlp(self.norm2(x).to(self.cfg.compute_dtype)).float()

    def forward(self, x, valid=None, reset=None, state=None):
        """x [B, T, d_model] float32 residual stream; returns (x, state)."""
        y, state = self.mixer(self.norm1(x).to(self.cfg.compute_dtype), valid, reset, state)
        return self._mlp(x + y.float()), state

    def step(self, x, state):
        return self._mlp(x + self.mixer.step(self.norm1(x).to(self.cfg.compute_dtype), state).float())


class RecurrentLM(torch.nn.Module):
    def __init__(self, cfg: RecurrentLMConfig, device=None):
        super().__init__()
        self.cfg = cfg
        self.embed = torch.nn.Parameter(torch.randn(cfg.vocab, cfg.d_model, device=device) * 0.02)
        self.blocks = torch.nn.ModuleList(RecurrentBlock(cfg, device) for _ in range(cfg.layers))
        self.norm = LayerNorm(cfg.d_model, cfg.norm_epsilon, True, device)

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

    def policy_loss(self, tokens, advantages, valid=None, entropy_weight: float = 0.0, present=None,
                    reset=None):
        """Minus the mean over the scored tokens of advantage times log probability, less entropy_weight
        times their mean entropy; advantages [B, T - 1], the masks as for score."""
        r = self.score(tokens, valid, present=present, reset=reset)
        on = scored(valid, present, reset)
        n = r.log_probs.numel() if on is None else on.sum().clamp(min=1)
        return -((advantages * r.log_probs).sum() + entropy_weight * r.entropy.sum()) / n

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
        return _mm(self.norm(x).to(self.cfg.compute_dtype), self.embed)[:, 0]


def make_optimizers(model, lr: float = 0.02, other_lr: float = 1e-3, weight_decay: float = 0.01):
    """(Muon for the blocks' projections, FusedAdamW for the rest): the embedding, which is the head too,
    convolutions, norms and gates.  Any of the models here.  A packed projection (u, r and gate; q, k, v and
    what goes with them; w1 and w3) is one matrix, and orthogonalised as one."""
    matrices = [p for n, p in model.named_parameters()
                if n.startswith("blocks.") and p.dim() == 2 and "conv" not in n]
    own = {id(p) for p in matrices}
    rest = [p for p in model.parameters() if id(p) not in own]
    return (dk.Muon(matrices, lr=lr, weight_decay=weight_decay),
            dk.FusedAdamW(rest, lr=other_lr, weight_decay=weight_decay))


def train_step(model, optimizers, loss_of) -> torch.Tensor:
    """One forward, backward and update; loss_of(model) is the loss.  Returns it detached."""
    for o in optimizers:
        o.zero_grad(set_to_none=True)
    loss = loss_of(model)
    loss.backward()
    for o in optimizers:
        o.step()
    return loss.detach()


def main(steps: int = 200):
    torch.manual_seed(0)
    cfg = RecurrentLMConfig(vocab=256, d_model=256, layers=2, width=256, mlp_width=704)
    model = RecurrentLM(cfg, device="cuda")
    optimizers = make_optimizers(model, other_lr=3e-3)
    text = torch.tensor(list(__doc__.encode()), device="cuda")
    for i in range(steps):
        start = torch.randint(0, len(text) - 129, (16, 1), device="cuda")
        tokens = text[start + torch.arange(129, device="cuda")]
        loss = train_step(model, optimizers, lambda m: m.loss(tokens))
        if i % 50 == 49:
            print(f"step {i + 1}: loss {loss.item():.3f}", flush=True)
    logits, states = model.prefill(text[None, :40])
    out = []
    for _ in range(60):
        token = logits.argmax(-1)
        out.append(int(token))
        logits = model.step(token, states)
    print(repr(bytes(text[:40].tolist()).decode()), "->", repr(bytes(out).decode("latin1")))
    with torch.no_grad():
        r = model.score(text[None, :40], top=3)
    print(f"the prompt: mean log probability {r.log_probs.mean().item():.3f}, entropy "
          f"{r.entropy.mean().item():.3f}; after it, most likely "
          f"{[chr(t) for t in r.top_tokens[0, -1].tolist()]}")


if __name__ == "__main__":
    main()
