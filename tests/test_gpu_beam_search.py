"""Beam search with the plaintext model: every operator of a generation loop
together, against the model's own scores of whole texts and against plain loops."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu


def build(vocab, dtype=None):
    from fhe_mamba_b200.mamba2_layer import Mamba2Model
    return Mamba2Model(layers=2, d_model=64, d_state=32, heads=4, vocab=vocab, std=0.2, calib_sequences=2, calib_tokens=4,
                       calib_prompt=2).plain_sequences(dtype=dtype)


@pytest.fixture(scope="module")
def net():
    return build(211)


# Scores of one text by steps and by a whole pass differ by the roundings of both: 2 layers and 3000 roundings of 2^-24
# each, passed on by a factor of 8 a layer, of logits below 20, for each token.
def tol(length):
    return length * 2 * 8 * 3000 * 2.0 ** -24 * 20


def text_scores(net, prompt, texts, lengths):
    """Sums of log-probabilities of texts [beams, length] behind a prompt, one whole pass."""
    rows = torch.cat([prompt.expand(len(texts), -1), texts], 1)
    n = (prompt.shape[-1] + lengths).int()
    return net.score(rows, lengths=n).logprob[:, prompt.shape[-1] - 1:].sum(1)


def test_exhaustive():
    """With as many beams as texts of one token fewer the search finds the best of all."""
    net = build(7)
    prompt = torch.tensor([[1, 5, 2], [6, 0, 0]], device="cuda")
    with torch.no_grad():
        out = net.beam_search(prompt, 7, 2)
        every = torch.tensor(list(itertools.product(range(7), repeat=2)), device="cuda")
        for i in range(2):
            s = text_scores(net, prompt[i], every, torch.full((49,), 2, device="cuda"))
            best = s.topk(7)
            assert (out.scores[i] - best.values).abs().max() <= tol(2)
            own = text_scores(net, prompt[i], out.tokens[i], out.lengths[i])
            assert (own - out.scores[i]).abs().max() <= tol(2)


@pytest.mark.parametrize("beams", [1, 4, 9])
def test_scores_belong_to_the_texts(net, beams):
    """Prompts of different lengths; the carried states have moved with their texts, ended ones stay as they were."""
    g = torch.Generator(device="cuda").manual_seed(beams)
    prompt = torch.randint(0, 211, (3, 6), generator=g, device="cuda")
    lengths = torch.tensor([6, 2, 4], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        free = net.beam_search(prompt, beams, 12, lengths=lengths)
    eos = int(free.tokens[0, 0, 3])  # a token that the search meets
    with torch.no_grad():
        ending = net.beam_search(prompt, beams, 12, eos, lengths, 0.7)
        for out in (free, ending):
            assert out.tokens.shape == (3, beams, 12)
            for i, n in enumerate(lengths.tolist()):
                own = text_scores(net, prompt[i, :n], out.tokens[i], out.lengths[i])
                assert (own - out.scores[i]).abs().max() <= tol(12)
                assert len({tuple(t) for t in out.tokens[i].tolist()}) == beams
    assert (free.lengths == 12).all() and (free.scores[:, 1:] <= free.scores[:, :-1]).all()
    rank = ending.scores / ending.lengths ** 0.7
    assert (rank[:, 1:] <= rank[:, :-1]).all()
    for text, n in zip(ending.tokens.flatten(0, 1).tolist(), ending.lengths.flatten().tolist()):
        assert eos not in text[:n - 1] and (n == 12 or all(t == eos for t in text[n - 1:]))
    assert (ending.lengths < 12).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_one_beam_is_greedy(dtype):
    """The same steps with the first of the largest logits, in every type of activations."""
    net = build(211, dtype)
    prompt = torch.randint(0, 211, (4, 5), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    with torch.no_grad():
        out = net.beam_search(prompt, 1, 8)
        hidden, state = net(prompt)
        logits = net.logits(hidden[:, -1])
        for i in range(8):
            t = logits.argmax(-1)
            assert torch.equal(out.tokens[:, 0, i], t)
            logits = net.logits(net.step(t, state))


def test_refusals_and_small_calls(net):
    prompt = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    for args, message in (((prompt[0], 2, 2), "tokens"), ((prompt[:, :0], 2, 2), "tokens"), ((prompt, 0, 2), "beams"),
                          ((prompt, 65, 2), "beams"), ((prompt, 2, 0), "length"),
                          ((prompt, 2, 2, None, torch.tensor([1, 0], dtype=torch.int32, device="cuda")), "needs a token"),
                          ((prompt, 2, 2, 211), "eos")):
        with pytest.raises(ValueError, match=message):
            net.beam_search(*args)
    assert net.beam_search(prompt[:0], 2, 3).tokens.shape == (0, 2, 3)
    assert net.beam_search(prompt.cpu(), 2, 1).tokens.shape == (2, 2, 1)


def test_rows_without_tokens(net):
    """Rows of no tokens come out empty and leave the state as it was."""
    hidden, state = net(torch.zeros(3, 0, dtype=torch.int64, device="cuda"))
    assert hidden.shape == (3, 0, 64)
    assert all(not w.any() and not s.any() for w, s in state)


def test_training_pass_reaches_every_parameter(net):
    """Tied embedding included, padded rows with and without a token id in the padding."""
    tokens = torch.randint(0, 211, (2, 20), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    lengths = torch.tensor([20, 9], dtype=torch.int32, device="cuda")
    padded = tokens.clone()
    padded[1, 9:] = -1
    grads = []
    for t in (tokens, padded):
        net.zero_grad()
        net.loss(t, lengths).backward()
        grads.append({n: p.grad.clone() for n, p in net.named_parameters()})
    for n, a in grads[0].items():
        assert torch.isfinite(a).all() and a.any(), n
        assert torch.equal(a, grads[1][n]), n
