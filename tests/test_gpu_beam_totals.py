"""Selections whose totals are easily got wrong: equal rows at different alignments."""
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
