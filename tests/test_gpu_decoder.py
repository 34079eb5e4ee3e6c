"""GPU tests of the example model: what it answers step by step is what its training
form computes over the whole sequence.

Tolerance, derived before the first run: both forms hold float32 sums and states and
differ in the order of sums (products of up to 256 terms) and in which kernel forms
them; two blocks' roundings stay below 2^-24 * 256 of the logits' size each way, 1e-4
of the largest logit bounds them."""

from __future__ import annotations

import pytest
import torch

from tests.gpu_util import announce, need_gpu, no_device_errors

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    need_gpu()
    from ossm_amd.decoder import MambaDecoder

    torch.manual_seed(0)
    return MambaDecoder(97, 64, 2, d_hidden=120).cuda()


def close(a, b):
    assert (a - b).abs().max() <= 1e-4 * b.abs().max()


def test_prompts_and_tokens_match_the_whole_sequence(model):
    tokens = torch.randint(0, 97, (3, 40)).cuda()
    announce("decoder prompt and steps against forward")
    with torch.no_grad():
        whole = model(tokens)
    states = model.states(8)
    slots = torch.tensor([5, 0, 7]).cuda()
    cuts = [30, 1, 37]
    offsets = torch.tensor([0, 30, 31, 68]).cuda()
    packed = torch.cat([tokens[i, :n] for i, n in enumerate(cuts)])
    logits = model.prompt(packed, offsets, states, slots)
    for i, n in enumerate(cuts):
        close(logits[i], whole[i, n - 1])
    for t in range(3):
        at = torch.tensor([n + t for n in cuts]).cuda()
        logits = model.step(tokens[torch.arange(3).cuda(), at], states, slots)
        for i, n in enumerate(cuts):
            close(logits[i], whole[i, n + t])
    # a second piece of each prompt
    offsets = torch.tensor([0, 2, 8, 8]).cuda()
    packed = torch.cat([tokens[0, 33:35], tokens[1, 4:10]])
    logits = model.prompt(packed, offsets, states, slots, torch.ones(3, dtype=torch.bool).cuda())
    close(logits[0], whole[0, 34])
    close(logits[1], whole[1, 9])
    no_device_errors()


def test_training_step_reaches_every_parameter(model):
    tokens = torch.randint(0, 97, (2, 50)).cuda()
    announce("decoder training step")
    loss = torch.nn.functional.cross_entropy(model(tokens)[:, :-1].flatten(0, 1), tokens[:, 1:].flatten())
    grads = torch.autograd.grad(loss, list(model.parameters()))
    assert all(torch.isfinite(g).all() and g.abs().max() > 0 for g in grads)


def test_answers_follow_the_controls(model):
    prompts = [torch.tensor([1, 2, 3]), torch.tensor([50]), torch.arange(20)]
    allowed = torch.zeros(3, 97, dtype=torch.bool)
    allowed[0, 10:20] = allowed[1, ::7] = allowed[2, 96] = True
    announce("decoder answers")
    out = model.answer(prompts, 12, allowed=allowed, frequency=100.0)
    for i in range(3):
        assert allowed[i].cuda()[out[i]].all()
    # a penalty past every logit uses each of ten tokens once before any twice
    assert sorted(out[0][:10].tolist()) == list(range(10, 20))
    assert (out[2] == 96).all()
    # without controls: the training form's own choice, token by token
    free = model.answer(prompts, 6)
    for i, p in enumerate(prompts):
        seq = p.cuda()
        for t in range(6):
            with torch.no_grad():
                logits = model(seq[None])[0, -1]
            top = logits.topk(2).values
            if top[0] - top[1] > 1e-3 * top[0].abs():  # not a tie to rounding
                assert int(logits.argmax()) == int(free[i, t])
            seq = torch.cat([seq, free[i, t:t + 1]])
    with pytest.raises(ValueError, match="at least one"):
        model.answer([], 3)


def test_bfloat16_weights(model):
    """The same model cast to bfloat16 serves, and agrees to bfloat16's rounding."""
    import copy

    half = copy.deepcopy(model).bfloat16()
    tokens = torch.randint(0, 97, (2, 20)).cuda()
    announce("decoder in bfloat16")
    offsets = torch.tensor([0, 20, 40]).cuda()
    slots = torch.arange(2).cuda()
    a = model.prompt(tokens.flatten(), offsets, model.states(2), slots)
    b = half.prompt(tokens.flatten(), offsets, half.states(2), slots)
    assert b.dtype == torch.bfloat16
    assert (a - b.float()).abs().max() <= 0.1 * a.abs().max()
    assert half.step(tokens[:, 0], half.states(2), slots).shape == (2, 97)
