"""What the plaintext model takes: tokens counted from the vocabulary's end."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def net():
    from fhe_mamba_b200.mamba2_layer import Mamba2Model
    return Mamba2Model(layers=2, d_model=64, d_state=32, heads=4, vocab=211, std=0.2, calib_sequences=2, calib_tokens=4,
                       calib_prompt=2).plain_sequences()


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_negative_tokens_count_from_the_end(net, dtype):
    tokens = torch.tensor([[-1, 3, -211], [210, -208, 0]], device="cuda", dtype=dtype)
    want = tokens.long() % 211
    with torch.no_grad():
        assert torch.equal(net._embed(tokens), net.embedding[tokens.long()].float())
        (a, s), (b, t) = net(tokens), net(want)
        assert torch.equal(a, b) and all(torch.equal(u, v) for x, y in zip(s, t) for u, v in zip(x, y))
        assert torch.equal(net.step(tokens[:, 0], s), net.step(want[:, 0], t))
        assert torch.equal(net(tokens.cpu())[0], b)
    grads = []
    for v in (tokens, want):
        net.zero_grad()
        net(v)[0].square().sum().backward()
        grads.append(net.embedding.grad.clone())
    assert torch.equal(*grads)


def test_tokens_outside_the_vocabulary(net):
    with torch.no_grad():
        e = net._embed(torch.tensor([[211, -212, 5]], device="cuda"))
    assert torch.isnan(e[0, 0]).all() and not e[0, 1].any() and torch.equal(e[0, 2], net.embedding[5].float())
