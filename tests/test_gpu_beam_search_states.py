"""Beam search's carried states: scores and texts near enough to a whole pass that a state
left behind, or moved in part, shows.

A step and a whole pass compute the same logits in other orders.  A logit of at most L is
off by some 64 roundings of 2^-24 between them, a log-probability by twice that, a text's
sum by its length times that: with L = 35 and 12 tokens 3.2e-3.  (One layer's recurrent state
left out of the reordering changes scores by 0.2 and more.)"""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu


def build(vocab):
    from fhe_mamba_b200.mamba2_layer import Mamba2Model
    return Mamba2Model(layers=2, d_model=64, d_state=32, heads=4, vocab=vocab, std=0.2, calib_sequences=2, calib_tokens=4,
                       calib_prompt=2).plain_sequences()


def bound(net, rows, length):
    """The bound for texts of `length` tokens, from the largest logit of whole passes over rows of tokens."""
    return length * 2 * net.logits(net(rows)[0]).abs().max().item() * 64 * 2.0 ** -24


def text_scores(net, rows, prompt, lengths):
    return net.score(rows, lengths=(prompt + lengths).int()).logprob[:, prompt - 1:].sum(1)


@torch.no_grad()
@pytest.mark.parametrize("beams", [1, 2, 4, 9])
@pytest.mark.parametrize("ends", [False, True])
def test_scores_of_texts(beams, ends):
    net = build(211)
    g = torch.Generator(device="cuda").manual_seed(beams)
    prompt = torch.randint(0, 211, (3, 6), generator=g, device="cuda")
    lengths = torch.tensor([6, 2, 4], dtype=torch.int32, device="cuda")
    eos = int(net.beam_search(prompt, beams, 12, lengths=lengths).tokens[0, 0, 3]) if ends else None
    out = net.beam_search(prompt, beams, 12, eos, lengths)
    for i, n in enumerate(lengths.tolist()):
        rows = torch.cat([prompt[i, :n].expand(beams, -1), out.tokens[i]], 1)
        b = bound(net, rows, 12)
        assert b < 1e-2  # far below what a state left behind changes
        own = text_scores(net, rows, n, out.lengths[i])
        assert (own - out.scores[i]).abs().max() <= b


@torch.no_grad()
def test_every_text_of_two_tokens():
    """With as many beams as tokens the search finds the best texts of two, and no others."""
    net = build(7)
    prompt = torch.tensor([[1, 5, 2], [6, 0, 0]], device="cuda")
    out = net.beam_search(prompt, 7, 2)
    every = torch.tensor(list(itertools.product(range(7), repeat=2)), device="cuda")
    for i in range(2):
        rows = torch.cat([prompt[i].expand(49, -1), every], 1)
        b = bound(net, rows, 2)
        best = text_scores(net, rows, 3, torch.full((49,), 2, device="cuda")).topk(8)
        assert (best.values[:-1] - best.values[1:]).min() > 2 * b  # far enough apart to be told
        assert torch.equal(out.tokens[i], every[best.indices[:7]])
        assert (out.scores[i] - best.values[:7]).abs().max() <= b
