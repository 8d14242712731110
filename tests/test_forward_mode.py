"""Inputs with forward-mode derivatives are refused: outputs without a tangent would pass for constants."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from fhe_mamba_b200 import mamba_ops as ops


def test_tangents_are_found():
    x, w = torch.randn(3, 4), torch.randn(4)
    assert not ops._wants_grad(x, None, w) and ops._wants_grad(x.clone().requires_grad_(), None)
    with fwd.dual_level():
        assert not ops._wants_grad(x, None, w)
        dual = fwd.make_dual(x, torch.ones_like(x))
        for tensors in ((dual,), (w, None, dual), (dual.view(12)[:5],)):
            with pytest.raises(ValueError, match="forward-mode"):
                ops._wants_grad(*tensors)
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                ops._wants_grad(*tensors)
    assert not ops._wants_grad(x, w)


def test_steps_and_beams_refuse_before_the_device():
    z = torch.zeros
    with fwd.dual_level():
        d = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ops.ssm_step(z(1, 2, 3, 4), d(z(1, 2, 3)), z(1, 2), z(1, 2), z(1, 1, 4), z(1, 1, 4)),
                     lambda: ops.causal_conv_step(z(1, 3, 4), z(1, 4), d(z(4, 4)))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()


@pytest.mark.gpu
def test_every_operator_refuses():
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    tokens = torch.tensor([1, 0], device="cuda")
    table, w = r(5, 8), r(8)
    cases = [
        (lambda x: ops.rms_norm(x, w), r(2, 8)),
        (lambda v: ops.rms_norm(table, v), w),
        (lambda x: ops.add_rms_norm(x, table, w), r(5, 8)),
        (lambda s: ops.add_rms_norm(table, table, w, scale=s), r(8)),
        (lambda z: ops.gated_rms_norm(table, z, w), r(5, 8)),
        (lambda t: ops.embedding(tokens, t), table),
        (lambda z: ops.token_logprobs(z, tokens), r(2, 7)),
        (lambda z: ops.beam_select(z, torch.zeros(1, 2, device="cuda")), r(2, 7)),
        (lambda s: ops.beam_select(table, s), r(1, 5)),
        (lambda s: ops.beam_reorder([s], torch.zeros(1, 5, dtype=torch.int64, device="cuda")), r(5, 8)),
        (lambda x: ops.causal_conv(x, table.T[:, :4].contiguous()), r(2, 3, 8)),
        (lambda x: ops.ssm_scan(x, r(1, 3, 2), -r(1, 3, 2).abs(), r(1, 3, 1, 8), r(1, 3, 1, 8)), r(1, 3, 2, 4)),
    ]
    for f, x in cases:
        f(x)
        with fwd.dual_level():
            dual = fwd.make_dual(x, torch.ones_like(x))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                    f(dual)
