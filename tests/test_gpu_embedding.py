"""The token embedding on the GPU.  The lookup is one fp32 product rounded once
and has to be equal; a row of the gradient is a sum of n terms in fp32 and a
product, off by at most (n + 2) u of the sum of their magnitudes, u = 2^-24, plus
half a step of its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
    from fhe_mamba_b200 import mamba_ops
    return mamba_ops


def rand(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def some_tokens(seed, n, vocab, how):
    g = rand(seed)
    t = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    if how == "skewed":  # a third of the positions are one token, many are none
        u = torch.rand(n, generator=g, device="cuda")
        t[u < 0.33] = vocab // 2
        t[u > 0.8] = -1
        t[(u > 0.7) & (u < 0.72)] = vocab + 3
    if how == "one":
        t[:] = vocab - 1
    if how == "none":
        t[:] = -5
    return t


def want_grad(tokens, dy, vocab, scale):
    used = (tokens >= 0) & (tokens < vocab)
    t = tokens[used].long()
    d = torch.zeros(vocab, dy.shape[-1], dtype=torch.float64, device="cuda").index_add_(0, t, dy[used].double())
    mag = torch.zeros_like(d).index_add_(0, t, dy[used].double().abs())
    n = torch.bincount(t, minlength=vocab)[:, None]
    return d * scale, mag * abs(scale) * (n + 2) * U


CASES = [(1, 7, 3, "even"), (5, 1, 64, "one"), (31, 50280, 8, "even"), (33, 1000, 1, "skewed"), (2047, 1000, 768, "skewed"),
         (2048, 100, 4, "none"), (2049, 5003, 769, "skewed"), (4097, 3, 20, "even"), (16383, 50280, 64, "even"),
         (16400, 211, 1300, "skewed"), (65537, 5003, 8, "skewed"), (70001, 1, 24, "one"), (140000, 1 << 20, 2, "skewed")]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, vocab, width, how", CASES)
def test_embedding(ops, dtype, n, vocab, width, how):
    for out, scale, kind in ((dtype, 1.0, torch.int64), (torch.float32, 0.37, torch.int32)):
        table = torch.randn(vocab, width, generator=rand(1), device="cuda").to(dtype).requires_grad_()
        tokens = some_tokens(2, n, vocab, how).to(kind)
        y = ops.embedding(tokens, table, scale, out)
        used = (tokens >= 0) & (tokens < vocab)
        want = (table.detach()[torch.where(used, tokens, 0).long()].float() * scale).to(out)
        want[tokens < 0] = 0
        want[tokens >= vocab] = math.nan
        assert y.dtype == out and torch.equal(torch.nan_to_num(y.detach(), 7.0), torch.nan_to_num(want, 7.0))
        dy = torch.randn(n, width, generator=rand(3), device="cuda").to(out)
        dy[tokens >= vocab] = math.nan  # what no row gets is not read into any
        dw, = torch.autograd.grad(y, table, dy, retain_graph=True)
        exact, err = want_grad(tokens, dy, vocab, scale)
        half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal
        assert dw.dtype == dtype and torch.isfinite(dw).all()
        worst = ((dw.double() - exact).abs() / (err + half * (exact.abs() + err) + tiny)).max().item()
        assert worst <= 1, worst
        assert (dw[torch.bincount(tokens[used].long(), minlength=vocab) == 0] == 0).all()
        assert torch.equal(torch.autograd.grad(y, table, dy)[0], dw)


def test_shapes_and_strides(ops):
    wide = torch.randn(50, 100, generator=rand(1), device="cuda").bfloat16()
    tokens = torch.randint(0, 50, (3, 4, 6), generator=rand(2), device="cuda")
    for table in (wide[:, 4:68], wide[:, 8:72], wide[::2, :64], wide[:, :64], wide.t()[:64].t(), wide[:1, :64].expand(50, 64)):
        for t in (tokens % table.shape[0], (tokens % table.shape[0])[:, 1], (tokens % table.shape[0])[..., ::2], tokens[0, 0, 0] * 0,
                  tokens[:0]):
            assert torch.equal(ops.embedding(t, table, 0.5), (table[t].float() * 0.5).bfloat16())
    leaf = wide.clone().requires_grad_()
    view = leaf[::2, 3:67]
    dy = torch.randn(3, 4, 6, 64, generator=rand(3), device="cuda").bfloat16().transpose(0, 1).contiguous().transpose(0, 1)
    g, = torch.autograd.grad(ops.embedding(tokens % 25, view), leaf, dy)
    exact, err = want_grad((tokens % 25).flatten(), dy.reshape(-1, 64), 25, 1.0)
    got = g[::2, 3:67].double()
    assert ((got - exact).abs() <= err + 2.0 ** -8 * (exact.abs() + err)).all()
    assert not g[1::2].any() and not g[:, :3].any() and not g[:, 67:].any()
    none = torch.empty(0, 5, dtype=torch.int64, device="cuda")
    g, = torch.autograd.grad(ops.embedding(none, leaf), leaf, torch.empty(0, 5, 100, device="cuda", dtype=torch.bfloat16))
    assert g.shape == leaf.shape and not g.any()


def test_table_changed_or_empty(ops):
    """The gradient needs no value of the table; a table without rows has nothing but absent tokens."""
    leaf = torch.ones(5, 16, device="cuda", requires_grad=True)
    tokens = torch.tensor([1, 1, 4], device="cuda")
    y = ops.embedding(tokens, leaf)
    with torch.no_grad():
        leaf.add_(1)
    g, = torch.autograd.grad(y.sum(), leaf)
    assert torch.equal(g.sum(1), torch.tensor([0.0, 32, 0, 0, 16], device="cuda"))
    none = torch.empty(0, 16, device="cuda", requires_grad=True)
    y = ops.embedding(torch.tensor([0, -1], device="cuda"), none)
    assert torch.isnan(y[0]).all() and (y[1] == 0).all()
    assert torch.autograd.grad(y.sum(), none)[0].shape == (0, 16)


def test_large_offsets(ops):
    """Rows past 2^31 elements of the table, its gradient and the outputs."""
    table = torch.zeros(40000, 1 << 16, device="cuda", dtype=torch.bfloat16)
    last = torch.randn(1 << 16, generator=rand(1), device="cuda").bfloat16()
    table[-1] = last
    table.requires_grad_()
    tokens = torch.full((33000,), 5, device="cuda")
    tokens[-1] = tokens[3] = 39999
    y = ops.embedding(tokens, table)
    assert torch.equal(y[-1], last) and torch.equal(y[3], last) and not y[32998].any()
    dy = torch.zeros_like(y)
    dy[-1], dy[3], dy[32998] = 1, 2, 4
    g, = torch.autograd.grad(y, table, dy)
    assert (g[-1] == 3).all() and (g[5] == 4).all() and not g[6:39999].any() and not g[:5].any()


def test_streams_and_graphs(ops):
    table = torch.randn(5003, 96, generator=rand(1), device="cuda").requires_grad_()
    tokens = some_tokens(2, 3000, 5003, "skewed")
    dy = torch.randn(3000, 96, generator=rand(3), device="cuda")
    side = torch.cuda.Stream()

    def both():
        y = ops.embedding(tokens, table, 2.0)
        return y.detach(), torch.autograd.grad(y, table, dy)[0]
    want = both()
    del want
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    tokens.copy_(some_tokens(5, 3000, 5003, "even"))
    dy.mul_(-1)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(torch.nan_to_num(a, 7.0), torch.nan_to_num(b, 7.0)) for a, b in zip(got, both()))
