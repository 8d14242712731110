"""What the plaintext model takes: tokens counted from the vocabulary's end, and
norms that the operators refuse (rows of more than 16384 channels, an eps of 0)."""
from types import SimpleNamespace

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


# A mean of n squares in float32 is off by at most 41 2^-24 (16 additions in a thread, 5 in a warp, 16 of warps, four
# roundings) in the operators and by no more in torch's sums; half of that and 5 roundings for a normalised value; SiLU by
# (8 + 3 |z|) 2^-24.  Both sides together, with |z| < 10: 2 (21 + 5 + 38) 2^-24.
NEAR = 2 * 64 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wide_rows(net, dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    n = 16392
    h, branch, w = r(2, 3, n), r(2, 3, n).to(dtype), 1 + r(n)
    half = torch.finfo(dtype).eps / 2
    saved = net.dtype
    try:
        net.dtype = dtype
        for b in (None, branch):
            u, stream = net._norm(h, b, w, 1e-5)
            want = h if b is None else h + b.float()
            assert torch.equal(stream, want) and u.dtype == dtype
            want = want.double()
            want = want * torch.rsqrt(want.square().mean(-1, keepdim=True) + 1e-5) * w.double()
            assert ((u.double() - want).abs() <= (NEAR + half) * want.abs() * (1 + half)).all()
        y, z = r(2, 4, n // 4).to(dtype), r(2, n).to(dtype)
        p = {"gn_w": w, "w_out": torch.eye(8, n, device="cuda", dtype=dtype)}
        got = net._finish(SimpleNamespace(eps=1e-5), p, y, z)
        v = y.flatten(-2).double() * z.double() * torch.sigmoid(z.double())
        want = (v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * w.double())[:, :8]
        # times the identity: one product of 1 and exact zeros
        assert got.dtype == dtype and ((got.double() - want).abs() <= (NEAR + half) * want.abs() * (1 + half)).all()
    finally:
        net.dtype = saved


def test_no_eps(net):
    """An eps of 0: whole passes, steps and gradients, near those of an eps that the operators take."""
    tokens = torch.randint(0, 211, (2, 9), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    eps = [W.eps for W in net.weights]
    outs = []
    try:
        for e in (0.0, 2.0 ** -100):  # rows of the embedding have mean squares of about 0.04
            for W in net.weights:
                W.eps = e
            net.zero_grad()
            net.loss(tokens).backward()
            with torch.no_grad():
                hidden, state = net(tokens[:, :-1])
                last = net.step(tokens[:, -1], state)
            outs.append([hidden, last, *(p.grad.clone() for p in net.parameters())])
    finally:
        for W, e in zip(net.weights, eps):
            W.eps = e
    # 2 layers, roundings of 3000 x 2^-24 each, passed on by a factor of 8 a layer
    for a, b in zip(*outs):
        assert torch.isfinite(a).all() and (a - b).norm() <= 2 * 8 * 3000 * 2.0 ** -24 * b.norm()
