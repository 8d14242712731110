"""The state scan's gradients where counts pass 32 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_gradients_of_more_than_two_to_the_32_threads():
    """2^27 tokens and a row more, one head of one row and one column (9 GB): a warp per token makes more than 2^32
    threads.  The last row's gradients are a call's of that row alone, bit for bit (the same segments)."""
    from fhe_mamba_b200 import mamba_ops as ops
    b, l = 1025, 1 << 17
    g = torch.Generator(device="cuda").manual_seed(1)
    shape = dict(x=(b, l, 1, 1), write=(b, l, 1), log_decay=(b, l, 1), B=(b, l, 1, 1), C=(b, l, 1, 1))
    i = {n: torch.rand(s, generator=g, device="cuda") for n, s in shape.items()}
    i["log_decay"].neg_()
    dy = torch.rand((b, l, 1, 1), generator=g, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        t = lambda n, v: v.to(dtype) if n in ("x", "B", "C") else v  # noqa: E731

        def grads(first):
            leaf = {n: t(n, v[first:]).detach().requires_grad_() for n, v in i.items()}
            y, _ = ops.ssm_scan(**leaf)
            return dict(zip(leaf, torch.autograd.grad(y, list(leaf.values()), dy[first:].to(dtype))))
        whole = {n: v[-1:].clone() for n, v in grads(0).items()}
        for n, v in grads(b - 1).items():
            assert torch.equal(whole[n], v), n
