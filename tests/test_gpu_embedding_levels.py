"""The embedding's gradient where its positions are merged in three and four levels
(past 262144 and 8388608 of them).  Gradients are small whole numbers, whose sums float32
holds whole in any order, so every row has to be equal to the sum."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n, vocab, width", [(262144, 50280, 8), (262145, 50280, 8), (300001, 50280, 8), (300001, 3, 5),
                                             (524289, 1, 4), (600000, 1 << 20, 1), (8388700, 50280, 1)])
def test_many_positions(n, vocab, width):
    from fhe_mamba_b200 import mamba_ops as ops
    g = torch.Generator(device="cuda").manual_seed(n + vocab)
    tokens = (torch.rand(n, generator=g, device="cuda") ** 4 * vocab).long().clamp(max=vocab - 1)  # a few have most positions
    u = torch.rand(n, generator=g, device="cuda")
    tokens[u < 0.1] = -1
    tokens[(u > 0.5) & (u < 0.52)] = vocab + 3
    table = torch.zeros(vocab, width, device="cuda", requires_grad=True)
    dy = torch.randint(-1, 2, (n, width), generator=g, device="cuda").float()  # sums below 2^24
    dw, = torch.autograd.grad(ops.embedding(tokens, table), table, dy)
    used = (tokens >= 0) & (tokens < vocab)
    want = torch.zeros(vocab, width, dtype=torch.float64, device="cuda").index_add_(0, tokens[used], dy[used].double())
    assert torch.equal(dw.double(), want)
