"""A small language model of mixers (Mamba's or the gated recurrence's) and gated
feed-forward blocks: trained as a module, served with states in a pool, answering under
controlled logits.

    python -m ossm_amd.decoder        # on a GPU: trains on a counting task and answers

It is the example of the library's language-model operators together: training runs
``MambaMixer`` or ``RecurrentMixer``, ``gated_linear`` and ``add_layer_norm`` with their
backwards, a prompt runs ``mixer_prompt`` or ``recurrence_prompt``, each further token
``mixer_step`` or ``recurrence_step`` and ``gated_linear`` on a few rows, ``control_logits``
shapes what is answered and ``sample_logits`` draws it.
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from . import decode
from .gated import GatedFeedForward
from .linear import calls_only
from .logits import control_logits, pack_allowed
from .mamba import MambaMixer
from .norm import LayerNorm, norm_of_sum
from .recurrence import RecurrentMixer, RecurrentState
from .sampling import sample_logits

__all__ = ["MambaDecoder"]

_State = Union[decode.MixerState, RecurrentState]


class _Block(nn.Module):
    def __init__(self, mixer: nn.Module, d_model: int, d_hidden: int, activation: str) -> None:
        super().__init__()
        self.norm1, self.norm2 = LayerNorm(d_model), LayerNorm(d_model)
        self.mixer = mixer
        self.feed_forward = GatedFeedForward(d_model, d_hidden, activation=activation)

    def forward(self, x: Tensor, mix=None) -> Tensor:
        x, added = self.parts(x, None, mix)
        return x + added

    def parts(self, x: Tensor, added: Optional[Tensor], mix=None) -> Tuple[Tensor, Tensor]:
        """The residual stream and what the block adds to it, from those of the block before
        (nothing added yet: None); each sum is taken with the norm that follows it."""
        h, x = (self.norm1(x), x) if added is None else norm_of_sum(self.norm1, added, x)
        h, x = norm_of_sum(self.norm2, (mix or self.mixer)(h), x)
        return x, self.feed_forward(h)


def _through(block: nn.Module, x: Tensor, added: Optional[Tensor], *mix) -> Tuple[Tensor, Optional[Tensor]]:
    """``block`` on ``x + added``, as such a pair; a replaced or hooked one is called as it is."""
    if calls_only(block, _Block):
        return block.parts(x, added, *mix)
    return block(x if added is None else x + added, *mix), None


class MambaDecoder(nn.Module):
    """Embedding, blocks of mixer and feed-forward, logits on the embedding's weights.
    mixer: "mamba" (``MambaMixer``) or "recurrent" (``RecurrentMixer``), of all blocks or one a
    block; d_state and d_conv are the Mamba mixer's."""

    def __init__(self, vocab: int, d_model: int, n_layers: int, *, d_hidden: Optional[int] = None, d_state: int = 16,
                 d_conv: int = 4, expand: int = 2, activation: str = "silu", mixer: Union[str, Sequence[str]] = "mamba") -> None:
        super().__init__()
        mixers = [mixer] * n_layers if isinstance(mixer, str) else list(mixer)
        if len(mixers) != n_layers or any(m not in ("mamba", "recurrent") for m in mixers):
            raise ValueError(f'mixer must be "mamba" or "recurrent", for all {n_layers} blocks or one for each, not {mixer!r}')
        self.embedding = nn.Embedding(vocab, d_model)
        nn.init.normal_(self.embedding.weight, std=d_model ** -0.5)
        self.blocks = nn.ModuleList(
            _Block(MambaMixer(d_model, d_state=d_state, d_conv=d_conv, expand=expand) if m == "mamba"
                   else RecurrentMixer(d_model, expand=expand), d_model, d_hidden or 4 * d_model, activation) for m in mixers)
        self.norm = LayerNorm(d_model)

    def _logits(self, x: Tensor, added: Optional[Tensor]) -> Tensor:
        h = self.norm(x) if added is None else norm_of_sum(self.norm, added, x)[0]
        return F.linear(h, self.embedding.weight)

    def forward(self, tokens: Tensor) -> Tensor:
        """Logits [batch, length, vocab] of tokens [batch, length], differentiable."""
        x, added = self.embedding(tokens), None
        for block in self.blocks:
            x, added = _through(block, x, added)
        return self._logits(x, added)

    def states(self, slots: int) -> List[_State]:
        """A pool of ``slots`` sequences' states, a ``MixerState`` or ``RecurrentState`` a block."""
        return [(RecurrentState if isinstance(b.mixer, RecurrentMixer) else decode.MixerState).of(b.mixer, slots)
                for b in self.blocks]

    @torch.no_grad()
    def prompt(self, tokens: Tensor, offsets: Tensor, states: Sequence[_State], slots: Tensor,
               resume: Optional[Tensor] = None) -> Tensor:
        """Logits after each of the packed prompts, tokens [rows], offsets [prompts + 1]
        (``mixer_prompt``); their states go to ``slots``.  An empty prompt's are its
        predecessor's last token's and mean nothing."""
        x, added = self.embedding(tokens), None
        for block, state in zip(self.blocks, states):
            if isinstance(block.mixer, RecurrentMixer):
                mix = lambda h, b=block, s=state: b.mixer.prompt(h, s, slots, offsets, resume)  # noqa: E731
            else:
                mix = lambda h, b=block, s=state: decode.prompt(b.mixer, h, s, slots, offsets, resume)  # noqa: E731
            x, added = _through(block, x, added, mix)
        last = (offsets[1:] - 1).clamp(min=0).long()
        return self._logits(x[last], None if added is None else added[last])

    @torch.no_grad()
    def step(self, tokens: Tensor, states: Sequence[_State], slots: Tensor) -> Tensor:
        """Logits [rows, vocab] after one more token of each sequence, tokens [rows]."""
        x, added = self.embedding(tokens), None
        for block, state in zip(self.blocks, states):
            if isinstance(block.mixer, RecurrentMixer):
                mix = lambda h, b=block, s=state: b.mixer.step(h, s, slots)  # noqa: E731
            else:
                mix = lambda h, b=block, s=state: decode.step(b.mixer, h, s, slots)  # noqa: E731
            x, added = _through(block, x, added, mix)
        return self._logits(x, added)

    @torch.no_grad()
    def answer(self, prompts: Sequence[Tensor], tokens: int, *, allowed: Optional[Tensor] = None,
               temperature: Union[float, Tensor, None] = None, top_k: Union[int, Tensor, None] = None,
               top_p: Union[float, Tensor, None] = None, min_p: Union[float, Tensor, None] = None,
               generator: Optional[torch.Generator] = None, **control) -> Tensor:
        """``tokens`` further tokens of each prompt (1-D tensors of at least one token),
        [prompts, tokens]: the most likely ones, or with a temperature drawn as
        ``sample_logits`` draws them, by random numbers of ``generator`` (the device's by
        default).  allowed: bool [vocab] or [prompts, vocab]; repetition, presence, frequency,
        bias_ids, bias_values as ``control_logits``'s."""
        dev = self.embedding.weight.device
        S, lengths = len(prompts), [int(p.numel()) for p in prompts]
        if S == 0 or min(lengths) == 0:
            raise ValueError("answer needs at least one prompt, each of at least one token")
        if temperature is None and any(v is not None for v in (top_k, top_p, min_p, generator)):
            raise ValueError("answer draws tokens only with a temperature: top_k, top_p, min_p and generator need one")
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
            logits = control_logits(logits, history, count, first, allowed=mask, **control)
            if temperature is None:
                out[:, t] = logits.argmax(-1)
            else:
                chosen = sample_logits(logits, torch.rand(S, device=dev, generator=generator), temperature=temperature,
                                       top_k=top_k, top_p=top_p, min_p=min_p, out=out[:, t])
                chosen.clamp_(min=0)  # a mask that allows nothing: token 0, as argmax's
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
    print("drawn:", model.answer(prompts, 8, temperature=1.0, top_p=0.95).tolist(), flush=True)


if __name__ == "__main__":
    main()
