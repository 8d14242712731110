"""Selections whose totals are easily got wrong: equal rows at different
alignments, and rows whose mask leaves nothing but the type's lowest numbers."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
    from fhe_mamba_b200 import mamba_ops
    return mamba_ops


def rand(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [131, 1003, 10007])
def test_equal_rows_at_every_alignment(ops, dtype, vocab):
    """Equal beams of rows of odd length, whose largest token comes first: their totals are equal, whichever 16-byte
    words the rows begin in, and go to the lower beam."""
    b, k = 300, 4
    row = (2 * torch.rand(b, 1, vocab, generator=rand(vocab), device="cuda") - 1).to(dtype)
    row[..., 0] = 3
    logits = row.expand(b, k, vocab).contiguous()
    got = ops.beam_select(logits, torch.zeros(b, k, device="cuda"))
    assert not got.tokens.any()
    assert torch.equal(got.parents, torch.arange(k, device="cuda").expand(b, k))
    assert (got.scores == got.scores[:, :1]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_the_lowest_number(ops, dtype):
    """A beam whose every token is masked with a number far below zero has the total that the formula says, its score
    less the logarithm of the vocabulary, not one that outranks the others.  A total is rounded to float32 from a sum
    off by at most 2^-24 (2.2 (log2 of the vocabulary + 12) + 32) relative to itself: 4e-6, and half a step of 2^-20
    of the rounding."""
    vocab = 5003
    low = torch.finfo(dtype).min
    logits = (2 * torch.randn(6, vocab, generator=rand(1), device="cuda")).to(dtype)
    logits[1] = low
    logits[4] = low if dtype == torch.float16 else -1e30
    logits[5, 1:] = low
    logits[5, 0] = low if dtype == torch.float16 else low / 2
    scores = torch.tensor([[-9.0, -9.0, -11.0], [-3.0, -2.0, -4.0]], device="cuda")
    got = ops.beam_select(logits, scores, width=8)
    z = logits.double().view(2, 3, vocab)
    top = z.max(-1, keepdim=True).values
    want = scores.double()[..., None] + ((z - top) - torch.log(torch.exp(z - top).sum(-1, keepdim=True)))
    best, at = torch.sort(want.flatten(1), dim=1, descending=True, stable=True)
    assert torch.equal(got.parents, at[:, :8] // vocab) and torch.equal(got.tokens, at[:, :8] % vocab)
    assert ((got.scores.double() - best[:, :8]).abs() <= 4e-6 + 2.0 ** -21 * 2).all()
    # all beams masked: the lower tokens of the beam with the best score
    same = torch.full((3, vocab), low, device="cuda", dtype=dtype)
    got = ops.beam_select(same, scores[1:])
    assert got.parents.tolist() == [[1, 1, 1]] and got.tokens.tolist() == [[0, 1, 2]]
    assert ((got.scores - (-2 - math.log(vocab))).abs() <= 4e-6 + 2.0 ** -21 * 2).all()
