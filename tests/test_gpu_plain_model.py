"""The plaintext model over whole sequences (convolution, recurrence and scores
together) against the float64 token-by-token layers, and the client's scores."""
import json
import math
import os

import numpy as np
import pytest
import torch

from conftest import GOLDEN

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    from fhe_mamba_b200.mamba2_layer import Mamba2Model
    return Mamba2Model(layers=3, d_model=64, d_state=32, heads=4, vocab=211, std=0.05, calib_sequences=2,
                       calib_tokens=4, calib_prompt=2)


def exact_hidden(model, tokens):
    """Normalised final hidden vectors of token rows, float64 (exact_step)."""
    from fhe_mamba_b200.mamba2_layer import _rms, exact_step
    b = tokens.shape[0]
    state = [([np.zeros((b, W.conv_dim)) for _ in range(W.conv_kernel - 1)],
              np.zeros((b, W.heads, W.head_dim, W.d_state))) for W in model.layers]
    out = []
    for t in range(tokens.shape[1]):
        h = model.embedding[tokens[:, t]]
        for i, W in enumerate(model.layers):
            h, c, s = exact_step(W, h, *state[i])
            state[i] = (c, s)
        out.append(_rms(h, model.norm_f, model.layers[0].eps))
    return np.stack(out, 1), state


# A layer passes fewer than 3000 roundings of u = 2^-24 relative to its largest
# value (dot products of 64 and 128, 80 tokens of recurrence, the norms), and
# its norms and gates pass a relative change on at most a few times; 3 layers
# with a factor of 8 each for that: 3 * 8 * 3000 u = 4.3e-3 of the largest.
TOL = 3 * 8 * 3000 * 2.0 ** -24


def test_sequences_match_the_token_layers(model):
    tokens = np.random.default_rng(1).integers(0, 211, (3, 80))
    want, state = exact_hidden(model, tokens)
    net = model.plain_sequences()
    got, new = net(torch.as_tensor(tokens, device="cuda"))
    assert np.abs(got.detach().cpu().numpy() - want).max() <= TOL * np.abs(want).max()
    for (window, s), (conv, exact) in zip(new, state):
        assert np.abs(s.detach().cpu().numpy() - exact).max() <= TOL * np.abs(exact).max()
        w = np.stack(conv, 1)
        assert np.abs(window.detach().cpu().numpy() - w).max() <= TOL * np.abs(w).max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prefill_then_steps(model, dtype):
    """Prompts of different lengths prefilled in one padded batch, then continued token by token, give the hidden
    vectors of the whole rows (the same arithmetic in float32; 2^-8 per rounded activation, some 30 of them, in bfloat16)."""
    g = torch.Generator(device="cuda").manual_seed(2)
    tokens = torch.randint(0, 211, (3, 90), generator=g, device="cuda")
    lengths = torch.tensor([80, 1, 37], device="cuda", dtype=torch.int32)
    net = model.plain_sequences(dtype=dtype)
    with torch.no_grad():
        whole, _ = net(tokens)
        part, state = net(tokens[:, :80], lengths=lengths)
    tol = (TOL if dtype == torch.float32 else 30 * 2.0 ** -8) * whole.float().abs().max()
    for r, n in enumerate(lengths.tolist()):
        assert (part[r, :n].float() - whole[r, :n].float()).abs().max() <= tol
    state = [(w.detach(), s.detach()) for w, s in state]
    for i in range(10):
        at = lengths.long() + i
        h = net.step(tokens[torch.arange(3), at], state)
        assert (h.float() - whole[torch.arange(3), at].float()).abs().max() <= tol


def test_scores(model):
    tokens = np.random.default_rng(3).integers(0, 211, (2, 40))
    hidden, _ = exact_hidden(model, tokens)
    logits = hidden[:, :-1] @ model.embedding.T
    m = logits.max(-1, keepdims=True)
    lse = m + np.log(np.exp(logits - m).sum(-1, keepdims=True))
    want = np.take_along_axis(logits - lse, tokens[:, 1:, None], -1)[..., 0]
    net = model.plain_sequences()
    lengths = torch.tensor([40, 25], device="cuda", dtype=torch.int32)
    s = net.score(torch.as_tensor(tokens, device="cuda"), lengths=lengths, top_k=4)
    # a logit is a product of 64: the hidden vector's error times the row's absolute sum
    tol = 2 * TOL * np.abs(hidden).max() * np.abs(model.embedding).sum(1).max()
    got = s.logprob.detach().cpu().numpy()
    assert np.abs(got[0] - want[0]).max() <= tol and np.abs(got[1, :24] - want[1, :24]).max() <= tol
    assert (got[1, 24:] == 0).all() and s.top_ids.shape == (2, 39, 4)
    loss = net.loss(torch.as_tensor(tokens, device="cuda"), lengths=lengths).item()
    assert abs(loss + (want[0].sum() + want[1, :24].sum()) / 63) <= tol


def test_rows_with_nothing_to_score(model):
    """Rows of one token: no scores, a loss of 0 and gradients of 0; rows of none are refused."""
    net = model.plain_sequences()
    one = torch.tensor([[3], [5]], device="cuda")
    assert net.score(one, top_k=4).top_ids.shape == (2, 0, 4)
    for lengths in (None, torch.tensor([1, 0], dtype=torch.int32, device="cuda")):
        loss = net.loss(one, lengths)
        assert loss.item() == 0
        grad = torch.autograd.grad(loss, net.embedding)[0]
        assert not grad.any()
    with pytest.raises(ValueError, match="at least 1"):
        net.score(one[:, :0])


def test_loss_has_the_gradients_of_differences(model):
    """The loss's gradient along a direction against the central difference: the loss is rounded by at most
    2 TOL x (log vocab + spread of the logits) and its curvature along the step is of the size of the loss."""
    net = model.plain_sequences()
    tokens = torch.randint(0, 211, (2, 70), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    net.loss(tokens).backward()
    g = torch.Generator(device="cuda").manual_seed(5)
    for name, p in net.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    with torch.no_grad():
        v = {n: p.grad * (p.abs().max() / p.grad.abs().max().clamp(min=1e-20)) for n, p in net.named_parameters()}
        ana = sum((p.grad.double() * v[n].double()).sum() for n, p in net.named_parameters()).item()
        step = 2.0 ** -8

        def at(e):
            for n, p in net.named_parameters():
                p.add_(v[n], alpha=e)
            out = net.loss(tokens).double().item()
            for n, p in net.named_parameters():
                p.add_(v[n], alpha=-e)
            return out
        num = (at(step) - at(-step)) / (2 * step)
    base = net.loss(tokens).item()
    assert math.isfinite(base)
    # directions follow the gradient: the derivative is positive, and the third-order term of a step of 2^-8 of the
    # parameters' size stays far below a tenth of it
    assert ana > 0 and abs(num - ana) <= 0.1 * ana


def test_client_loop_scores():
    """--client-alternatives' scores in the chain's result, over the slot model of the encrypted schedule."""
    import sys
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
    from slot_sim import SlotContext

    from fhe_mamba_b200.chain_payload import PayloadError, client_logits, read_chain_payload, run_chain
    p = read_chain_payload(os.path.join(GOLDEN, "mamba2_chain"), 0, True)
    cc = SlotContext(2048)
    cc.device = 0
    plain = run_chain(SlotContext(2048), p, 3, 1e-3, autoregressive_client_loop=True)["measurements"]
    m = run_chain(cc, p, 3, 1e-3, autoregressive_client_loop=True, client_alternatives=3)["measurements"]
    assert "autoregressive_selected_scores" not in plain
    scores = m["autoregressive_selected_scores"]
    assert [s["token"] for s in scores] == m["autoregressive_selected_ids"] == plain["autoregressive_selected_ids"]
    prompt = int(p.autoregressive["prompt_tokens"])
    for i, s in enumerate(scores):
        z = client_logits(p, np.asarray(p.ar_expected_poly_final[prompt - 1 + i], dtype=np.float64))
        lp = z - z.max() - np.log(np.exp(z - z.max()).sum())
        assert s["alternatives"][0][0] == s["token"] and len(s["alternatives"]) == 3
        # the decrypted vector is within 1e-3 of the reference: each logit within 1e-3 of the head's absolute row sum
        tol = 2e-3 * np.abs(p.client_embedding_w).sum(1).max()
        assert abs(s["logprob"] - lp[s["token"]]) <= tol
        assert abs(s["entropy"] + (np.exp(lp) * lp).sum()) <= 20 * tol
    json.dumps(scores)
    with pytest.raises(PayloadError, match="client-alternatives"):
        run_chain(cc, p, 2, 1e-3, client_alternatives=3)


def test_model_client_scores(model):
    from types import SimpleNamespace

    from fhe_mamba_b200.mamba2_layer import EncryptedMamba2Model
    em = EncryptedMamba2Model.__new__(EncryptedMamba2Model)
    em.cc, em.m = SimpleNamespace(device=0), model
    h = np.random.default_rng(5).normal(size=(2, 64))
    z = h @ model.embedding.T
    s = em.client_scores(h, z.argmax(1), 2)
    assert [x["alternatives"][0][0] for x in s] == z.argmax(1).tolist()
