"""A small language model of Mamba mixers and gated feed-forward blocks: trained as a
module, served with states in a pool, answering under controlled logits.

    python -m ossm_amd.decoder        # on a GPU: trains on a counting task and answers

It is the example of the library's language-model operators together: training runs
``MambaMixer`` and ``gated_linear`` with their backwards, a prompt runs
``mixer_prompt``, each further token ``mixer_step`` and ``gated_linear`` on a few rows, and
``control_logits`` shapes what is answered.
"""

from __future__ import annotations

from typing import List, Optional, Sequence

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from . import decode
from .gated import GatedFeedForward
from .logits import control_logits, pack_allowed
from .mamba import MambaMixer

__all__ = ["MambaDecoder"]


class _Block(nn.Module):
    def __init__(self, d_model: int, d_hidden: int, d_state: int, d_conv: int, expand: int, activation: str) -> None:
        super().__init__()
        self.norm1, self.norm2 = nn.LayerNorm(d_model), nn.LayerNorm(d_model)
        self.mixer = MambaMixer(d_model, d_state=d_state, d_conv=d_conv, expand=expand)
        self.feed_forward = GatedFeedForward(d_model, d_hidden, activation=activation)

    def forward(self, x: Tensor, mix=None) -> Tensor:
        x = x + (mix or self.mixer)(self.norm1(x))
        return x + self.feed_forward(self.norm2(x))


class MambaDecoder(nn.Module):
    """Embedding, blocks of mixer and feed-forward, logits on the embedding's weights."""

    def __init__(self, vocab: int, d_model: int, n_layers: int, *, d_hidden: Optional[int] = None, d_state: int = 16,
                 d_conv: int = 4, expand: int = 2, activation: str = "silu") -> None:
        super().__init__()
        self.embedding = nn.Embedding(vocab, d_model)
        nn.init.normal_(self.embedding.weight, std=d_model ** -0.5)
        self.blocks = nn.ModuleList(_Block(d_model, d_hidden or 4 * d_model, d_state, d_conv, expand, activation)
                                    for _ in range(n_layers))
        self.norm = nn.LayerNorm(d_model)

    def _logits(self, x: Tensor) -> Tensor:
        return F.linear(self.norm(x), self.embedding.weight)

    def forward(self, tokens: Tensor) -> Tensor:
        """Logits [batch, length, vocab] of tokens [batch, length], differentiable."""
        x = self.embedding(tokens)
        for block in self.blocks:
            x = block(x)
        return self._logits(x)

    def states(self, slots: int) -> List[decode.MixerState]:
        """A pool of ``slots`` sequences' states, a ``MixerState`` a block."""
        return [decode.MixerState.of(b.mixer, slots) for b in self.blocks]

    @torch.no_grad()
    def prompt(self, tokens: Tensor, offsets: Tensor, states: Sequence[decode.MixerState], slots: Tensor,
               resume: Optional[Tensor] = None) -> Tensor:
        """Logits after each of the packed prompts, tokens [rows], offsets [prompts + 1]
        (``mixer_prompt``); their states go to ``slots``.  An empty prompt's are its
        predecessor's last token's and mean nothing."""
        x = self.embedding(tokens)
        for block, state in zip(self.blocks, states):
            x = block(x, lambda h, b=block, s=state: decode.prompt(b.mixer, h, s, slots, offsets, resume))
        return self._logits(x[(offsets[1:] - 1).clamp(min=0).long()])

    @torch.no_grad()
    def step(self, tokens: Tensor, states: Sequence[decode.MixerState], slots: Tensor) -> Tensor:
        """Logits [rows, vocab] after one more token of each sequence, tokens [rows]."""
        x = self.embedding(tokens)
        for block, state in zip(self.blocks, states):
            x = block(x, lambda h, b=block, s=state: decode.step(b.mixer, h, s, slots))
        return self._logits(x)

    @torch.no_grad()
    def answer(self, prompts: Sequence[Tensor], tokens: int, *, allowed: Optional[Tensor] = None, **control) -> Tensor:
        """The most likely ``tokens`` further tokens of each prompt (1-D tensors of at least
        one token), [prompts, tokens].  allowed: bool [vocab] or [prompts, vocab];
        repetition, presence, frequency, bias_ids, bias_values as ``control_logits``'s."""
        dev = self.embedding.weight.device
        S, lengths = len(prompts), [int(p.numel()) for p in prompts]
        if S == 0 or min(lengths) == 0:
            raise ValueError("answer needs at least one prompt, each of at least one token")
        history = torch.zeros(S, max(lengths) + tokens, dtype=torch.int32, device=dev)
        for i, p in enumerate(prompts):
            history[i, :lengths[i]] = p.to(dev)
        first = torch.tensor(lengths, dtype=torch.int32, device=dev)
        count, slots = first.clone(), torch.arange(S, dtype=torch.int32, device=dev)
        offsets = torch.zeros(S + 1, dtype=torch.int32, device=dev)
        offsets[1:] = first.cumsum(0)
        mask = None if allowed is None else pack_allowed(allowed.to(dev))
        states = self.states(S)
        logits = self.prompt(torch.cat([p.to(dev) for p in prompts]), offsets, states, slots)
        out = torch.empty(S, tokens, dtype=torch.int64, device=dev)
        for t in range(tokens):
            out[:, t] = control_logits(logits, history, count, first, allowed=mask, **control).argmax(-1)
            history.scatter_(1, count[:, None].long(), out[:, t:t + 1].int())
            count += 1
            if t + 1 < tokens:
                logits = self.step(out[:, t], states, slots)
        return out


def main() -> None:
    """Trains a small model to count on modulo 20, then lets it go on counting."""
    torch.manual_seed(0)
    V, L = 20, 32
    model = MambaDecoder(V, 64, 2).cuda()
    opt = torch.optim.AdamW(model.parameters(), lr=3e-3)
    for i in range(60):
        start, stride = torch.randint(0, V, (64, 1)).cuda(), torch.randint(1, 4, (64, 1)).cuda()
        seq = (start + stride * torch.arange(L + 1).cuda()) % V
        loss = F.cross_entropy(model(seq[:, :-1]).flatten(0, 1), seq[:, 1:].flatten())
        opt.zero_grad()
        loss.backward()
        opt.step()
        if i % 20 == 19:
            print(f"step {i + 1}: loss {loss.item():.3f}", flush=True)
    prompts = [torch.tensor([3, 4, 5]), torch.tensor([0, 2, 4, 6, 8]), torch.tensor([1, 4, 7, 10])]
    print("goes on:", model.answer(prompts, 8).tolist(), flush=True)
    even = torch.arange(V) % 2 == 0
    print("even tokens only, repeats penalised:", model.answer(prompts, 8, allowed=even, frequency=2.0).tolist(), flush=True)


if __name__ == "__main__":
    main()
