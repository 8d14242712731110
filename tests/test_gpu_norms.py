"""The norms on the GPU against their definitions in float64.

Tolerances, with u = 2^-24 and `half` half a step of an output's type relative to
its value.  A mean of squares (or of products a u, relative to the mean of their
magnitudes) passes at most 16 additions in a thread, 5 in a warp, 16 of warps
and 4 roundings of its terms and of 1 / n: 41 u; r = 1 / sqrt(mean + eps) half of
that and 3 roundings: 24 u.  SiLU(z) is off by (8 + 3 |z|) u (exp2 and reciprocal
within 2 units, the exponent's two roundings of |z| log2 e): 38 u for |z| < 10,
its derivative twice that.  With K = 64 + 4 * 38 for all of these together an
output of magnitude `mag` (the same formula over absolute values) is off by at
most K u mag + half |value|; sums over rows add one rounding per row.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
K = 64 + 4 * 38
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
    from fhe_mamba_b200 import mamba_ops
    return mamba_ops


def close(got, want, mag, k=K, what=""):
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    half, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).smallest_normal
    err = k * U * mag
    worst = ((got.double() - want).abs() / (err + half * (want.abs() + err) + tiny)).max().item() if got.numel() else 0
    assert worst <= 1, f"{what}: {worst:.3g} of the tolerance"


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def norm_of(u, w, eps, groups=1):
    """y and r of rows u in float64."""
    r = (u.unflatten(-1, (groups, -1)).square().mean(-1, keepdim=True) + eps).rsqrt()
    r = r.expand(*r.shape[:-1], u.shape[-1] // groups).flatten(-2)
    return u * r * w, r


def mean_of(v, groups=1):
    m = v.unflatten(-1, (groups, -1)).mean(-1, keepdim=True)
    return m.expand(*m.shape[:-1], v.shape[-1] // groups).flatten(-2)


def grads_of(dy, u, r, w, groups=1):
    """Gradient of u and its magnitude, and the weight's per-row terms."""
    a, un = dy * w, u * r
    du = r * (a - un * mean_of(a * un, groups))
    mag = r * (a.abs() + un.abs() * mean_of((a * un).abs(), groups))
    return du, mag, dy * un


SHAPES = [(1, 1), (3, 7), (5, 8), (1, 768), (4, 768), (301, 768), (700, 1536), (13, 1001), (400, 333), (2, 16384), (3, 12296),
          (300, 4096), (310, 2560), (9, 1024), (333, 64), (299, 9000), (1000, 1), (77, 100), (130, 128), (65, 13), (5, 130)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, width", SHAPES)
def test_norm(ops, dtype, rows, width):
    for source in {dtype, torch.float32}:
        x = (3 * normal(1, rows, width)).to(source).requires_grad_()
        w = (1 + normal(2, width)).requires_grad_()
        y = ops.rms_norm(x, w, 1e-5, dtype)
        assert y.dtype == dtype
        want, r = norm_of(x.detach().double(), w.detach().double(), 1e-5)
        close(y.detach(), want, want.abs(), what="y")
        with torch.no_grad():
            assert torch.equal(ops.rms_norm(x, w, 1e-5, dtype), y)
        dy = normal(3, rows, width).to(dtype)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        du, mag, terms = grads_of(dy.double(), x.detach().double(), r, w.detach().double())
        close(dx, du, mag, what="dx")
        close(dw, terms.sum(0), terms.abs().sum(0), K + rows, "dw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, width", SHAPES)
@pytest.mark.parametrize("scale", [1.0, -0.3, "channels"])
def test_add_norm(ops, dtype, rows, width, scale):
    for stream in {dtype, torch.float32}:
        res = normal(1, rows, width).to(stream).requires_grad_()
        x = normal(2, rows, width).to(dtype).requires_grad_()
        w = (1 + normal(3, width)).requires_grad_()
        s = (0.5 + normal(4, width)).requires_grad_() if scale == "channels" else scale
        y, h = ops.add_rms_norm(res, x, w, 1e-5, s)
        assert y.dtype == dtype and h.dtype == stream
        s64 = s.detach().double() if scale == "channels" else s
        sum_ = res.detach().double() + s64 * x.detach().double()
        # the product's rounding and the sum's
        close(h.detach(), sum_, res.detach().double().abs() + (s64 * x.detach().double()).abs(), 2, "h")
        kept = h.detach().double()
        want, r = norm_of(kept, w.detach().double(), 1e-5)
        close(y.detach(), want, want.abs(), what="y")
        dy, dh = normal(5, rows, width).to(dtype), normal(6, rows, width).to(stream)
        leaves = [res, x, w] + ([s] if scale == "channels" else [])
        for followed, given, dh64 in (((y, h), (dy, dh), dh.double()), ((y,), (dy,), 0.0)):
            grads = torch.autograd.grad(followed, leaves, given, retain_graph=True)
            du, mag, terms = grads_of(dy.double(), kept, r, w.detach().double())
            du = du + dh64
            mag = mag + abs(dh64)
            close(grads[0], du, mag, what="dresidual")
            close(grads[1], du * s64, mag * abs(s64), what="dx")
            close(grads[2], terms.sum(0), terms.abs().sum(0), K + rows, "dw")
            if scale == "channels":
                t = x.detach().double()
                close(grads[3], (du * t).sum(0), (mag * t.abs()).sum(0), K + rows, "dscale")
        only = torch.autograd.grad(h, (res, x), dh)
        close(only[0], dh.double(), dh.double().abs(), what="dresidual of h alone")
        close(only[1], dh.double() * s64, (dh.double() * s64).abs(), what="dx of h alone")


GATED = [(1, 1, 1), (3, 7, 1), (999, 1, 1), (70, 104, 1), (31, 360, 3), (40, 39, 3), (4, 1536, 1), (301, 1536, 1), (300, 1536, 8), (20, 555 * 3, 3), (700, 192, 1), (2, 40960, 5),
         (299, 9000, 1), (33, 35, 5)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, width, groups", GATED)
def test_gated_norm(ops, dtype, rows, width, groups):
    for after in (0, 7, 24):  # the gate in its own memory, and a slice of rows whose stride does not or does align
        x = normal(1, rows, width).to(dtype).requires_grad_()
        wide = (2 * normal(2, rows, width + after)).clamp(-9.9, 9.9).to(dtype)
        z = wide[:, :width].detach().requires_grad_()
        w = (1 + normal(3, width)).requires_grad_()
        y = ops.gated_rms_norm(x, z, w, 1e-4, groups)
        x64, z64, w64 = x.detach().double(), z.detach().double(), w.detach().double()
        q = torch.sigmoid(z64)
        p = z64 * q
        v = x64 * p
        want, r = norm_of(v, w64, 1e-4, groups)
        close(y.detach(), want, want.abs(), what="y")
        dy = normal(4, rows, width).to(dtype)
        dx, dz, dw = torch.autograd.grad(y, (x, z, w), dy)
        dv, mag, terms = grads_of(dy.double(), v, r, w64, groups)
        close(dx, dv * p, mag * p.abs(), what="dx")
        close(dz, dv * x64 * (q + p * (1 - q)), mag * x64.abs() * (q + p.abs() * (1 - q)), what="dz")
        close(dw, terms.sum(0), terms.abs().sum(0), K + rows, "dw")


def test_strides_and_shapes(ops):
    """Any leading axes, rows apart or not evenly apart, unaligned starts, broadcast inputs, no rows at all.  How a row
    is loaded decides the order of its sum of squares: results are held to the module's bound, not to equal bits."""
    w = 1 + normal(1, 768)
    base = normal(2, 4, 6, 900).bfloat16()
    for x in (base[..., :768], base[..., 3:771], base.transpose(0, 1)[..., :768], base[1, 2, :768], base[:, 2, 100:868],
              base[:1, :, :768].expand(5, 6, 768), base[:0, :, :768]):
        want, _ = norm_of(x.double(), w.double(), 1e-5)
        close(ops.rms_norm(x, w), want, want.abs())
        y, h = ops.add_rms_norm(x.float(), x, w)
        assert torch.equal(h, 2 * x.float())
        want, _ = norm_of(h.double(), w.double(), 1e-5)
        close(y, want, want.abs())
        u = x.double() * x.double() * torch.sigmoid(x.double())
        want, _ = norm_of(u, w.double(), 1e-5)
        close(ops.gated_rms_norm(x, x, w), want, want.abs())
    one = base[:1, :1, :768].float().requires_grad_()
    y, h = ops.add_rms_norm(one.expand(4, 6, 768), base[..., :768], w)
    dy, dh = normal(3, 4, 6, 768).bfloat16(), normal(4, 4, 6, 768)
    whole = one.detach().expand(4, 6, 768).contiguous().requires_grad_()
    y2, h2 = ops.add_rms_norm(whole, base[..., :768], w)
    g, = torch.autograd.grad((y, h), one, (dy, dh))
    g2, = torch.autograd.grad((y2, h2), whole, (dy, dh))
    assert torch.equal(g, g2.sum((0, 1), keepdim=True))
    # a transposed innermost axis is copied
    t = normal(5, 768, 9).t()
    assert torch.equal(ops.rms_norm(t, w), ops.rms_norm(t.contiguous(), w))
    e = torch.empty(0, 768, device="cuda", requires_grad=True)
    wl = w.clone().requires_grad_()
    ge, gw = torch.autograd.grad(ops.rms_norm(e, wl), (e, wl), torch.empty(0, 768, device="cuda"))
    assert ge.shape == (0, 768) and not gw.any()


@pytest.mark.parametrize("width", [768, 1001, 16384])
def test_ranges(ops, width):
    """Rows of zeros, of numbers whose squares overflow or vanish, and infinities and NaN, which stay in their rows."""
    w = 1 + 0.1 * normal(1, width)
    x = normal(2, 6, width)
    for factor in (1e18, 1e30, 1e37):
        big = x * factor
        want, _ = norm_of(big.double(), w.double(), 1e-5)
        # r has at least 21 bits down to 2^-128
        close(ops.rms_norm(big, w), want, want.abs(), K + 8, f"{factor}")
    small = x * 1e-25
    want, _ = norm_of(small.double(), w.double(), 1e-5)
    close(ops.rms_norm(small, w), want, want.abs(), what="small")
    x[0] = 0
    x[2, 5] = math.inf
    x[4, 1] = math.nan
    y = ops.rms_norm(x, w)
    want, _ = norm_of(x.double(), w.double(), 1e-5)
    assert (y[0] == 0).all() and torch.isnan(y[4]).all()
    assert torch.isnan(y[2, 5]) and (y[2, :5] == 0).all() and (y[2, 6:] == 0).all()
    for i in (1, 3, 5):
        close(y[i], want[i], want[i].abs())
    y, h = ops.add_rms_norm(torch.zeros_like(x).half(), x.half(), w)
    assert torch.equal(h[1::2], x.half()[1::2]) and torch.isfinite(y[1::2]).all() and torch.isnan(y[4]).all()


def test_large_offsets(ops):
    """Rows past 2^31 elements, wide and narrow."""
    for rows, width in ((135000, 16384), (300_000_000, 8)):
        x = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16)
        g = torch.Generator(device="cuda").manual_seed(width)
        some = torch.randn(3, width, generator=g, device="cuda").bfloat16()
        at = torch.tensor([0, rows // 2 + 1, rows - 1], device="cuda")
        x[at] = some
        w = (1 + torch.randn(width, generator=g, device="cuda")).requires_grad_()
        small = some.clone().requires_grad_()
        want = ops.rms_norm(small, w)
        dw_want, dx_want = torch.autograd.grad(want, (w, small), some)
        x.requires_grad_()
        y = ops.rms_norm(x, w)
        assert torch.equal(y[at], want) and not y[1:9].any()
        dw, dx = torch.autograd.grad(y, (w, x), x.detach())
        assert torch.equal(dx[at], dx_want)
        # every other row adds an exact 0; three terms, added in whatever order, are off by 2 u of their magnitudes each way
        _, r = norm_of(some.double(), w.detach().double(), 1e-5)
        mag = (some.double() * some.double() * r).abs().sum(0)
        assert ((dw - dw_want).abs() <= 6 * U * mag).all()
        del x, y, dx
        torch.cuda.empty_cache()


def test_gradients_against_differences(ops):
    """Directional derivatives against central differences of the forward calls: the differences of steps of 2^-6 are
    off by the third-order term, below a hundredth of inputs of size 1, and by 2^-24 sqrt(n) / 2^-6 of the outputs."""
    rows, width = 8, 96
    g = lambda i: normal(i, rows, width)  # noqa: E731
    w, s = 1 + 0.2 * normal(9, width), 0.5 + 0.2 * normal(8, width)
    dy, dh = g(1), g(2)

    def check(f, tensors, outs):
        leaves = [t.clone().requires_grad_() for t in tensors]
        loss = lambda v: sum((o * d).sum().double() for o, d in zip(f(*v), outs))  # noqa: E731
        grads = torch.autograd.grad(loss(leaves), leaves)
        for i, t in enumerate(tensors):
            v = normal(20 + i, *t.shape)
            v = v + grads[i] / grads[i].norm() * v.norm()
            step = 2.0 ** -6
            at = [[u + (e * v if j == i else 0) for j, u in enumerate(tensors)] for e in (step, -step)]
            with torch.no_grad():
                num = ((loss(at[0]) - loss(at[1])) / (2 * step)).item()
            ana = (grads[i].double() * v.double()).sum().item()
            assert abs(num - ana) <= 0.02 * abs(ana), (i, num, ana)

    check(lambda r, x, w_, s_: ops.add_rms_norm(r, x, w_, 1e-5, s_), [g(3), g(4), w, s], (dy, dh))
    check(lambda x, z, w_: (ops.gated_rms_norm(x, z, w_, 1e-5, 3),), [g(5), g(6), w], (dy,))
    check(lambda x, w_: (ops.rms_norm(x, w_),), [g(7), w], (dy,))


def test_partial_gradients(ops):
    """Inputs that need no gradient leave the others' as they are."""
    r, x, w, s = normal(1, 40, 96), normal(2, 40, 96), 1 + normal(3, 96), 0.5 + normal(4, 96)
    dy, dh = normal(5, 40, 96), normal(6, 40, 96)
    for scale in (1.0, 0.5, s):
        every = [t.clone().requires_grad_() for t in (r, x, w)] + ([s.clone().requires_grad_()] if scale is s else [])
        want = torch.autograd.grad(ops.add_rms_norm(*every[:3], 1e-5, every[3] if scale is s else scale), every, (dy, dh))
        for i in range(len(every)):
            some = [t.detach().clone() for t in every]
            some[i].requires_grad_()
            outs = ops.add_rms_norm(*some[:3], 1e-5, some[3] if scale is s else scale)
            got = torch.autograd.grad([o for o in outs if o.requires_grad], some[i],
                                      [d for o, d in zip(outs, (dy, dh)) if o.requires_grad])[0]
            assert torch.equal(got, want[i]), i


def test_second_derivatives_are_refused(ops):
    """A graph of the backward pass may be asked for; using it raises, and no gradient comes out as if it were constant."""
    x, w = normal(1, 6, 32).requires_grad_(), (1 + normal(2, 32)).requires_grad_()
    table, tokens = normal(3, 9, 32).requires_grad_(), torch.tensor([1, 4], device="cuda")
    for y, leaf in ((ops.rms_norm(x, w), x), (ops.gated_rms_norm(x, x, w), w), (ops.embedding(tokens, table) * x[0], table)):
        once, = torch.autograd.grad(y.sin().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            once.sum().backward()


def test_one_leaf_twice_and_shared_gradients(ops):
    """A tensor that is stream and branch at once gets both gradients; leaves that share one do not share memory."""
    w, dy, dh = 1 + normal(1, 96), normal(2, 30, 96), normal(3, 30, 96)
    one = normal(4, 30, 96).requires_grad_()
    r, x = (one.detach().clone().requires_grad_() for _ in range(2))
    got, = torch.autograd.grad(ops.add_rms_norm(one, one, w), one, (dy, dh))
    a, b = torch.autograd.grad(ops.add_rms_norm(r, x, w), (r, x), (dy, dh))
    assert torch.equal(a, b) and torch.equal(got, a + b)
    torch.autograd.backward(ops.add_rms_norm(r, x, w), (dy, dh))
    r.grad.zero_()
    assert torch.equal(x.grad, a)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, width", [(700, 1536), (33, 1001), (500, 64), (4, 768)])
def test_outputs_over_inputs(ops, dtype, rows, width):
    """The C calls may write y and h over x, residual or gate."""
    from fhe_mamba_b200._lib import call
    w = 1 + normal(1, width)
    r, x, z = (normal(i, rows, width).to(dtype) for i in (2, 3, 4))
    for over in "xz":
        a, b = x.clone(), z.clone()
        want = ops.gated_rms_norm(a, b, w)
        values, _ = ops._norm_values(a, dtype, dtype, 1, 1e-5, 1.0, a, None, b, None, w, a if over == "x" else b, None, None)
        call("fhe_rms_norm", ops._norm_block(*values))
        assert torch.equal(a if over == "x" else b, want)
    a, b = x.clone(), r.clone()
    want = ops.add_rms_norm(b, a, w)
    values, _ = ops._norm_values(a, dtype, dtype, 1, 1e-5, 1.0, a, b, None, None, w, a, b, None)
    call("fhe_rms_norm", ops._norm_block(*values))
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_streams_and_graphs(ops):
    """Another stream than the default one, and a captured call replayed on new values."""
    x, r, w = normal(1, 50, 768).bfloat16(), normal(2, 50, 768), 1 + normal(3, 768)
    want = ops.add_rms_norm(r, x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.add_rms_norm(r, x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xi, ri, wi = x.clone().requires_grad_(), r.clone().requires_grad_(), w.clone().requires_grad_()
    dy, dh = normal(4, 50, 768).bfloat16(), normal(5, 50, 768)

    def both():
        return torch.autograd.grad(ops.add_rms_norm(ri, xi, wi), (ri, xi, wi), (dy, dh))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    with torch.no_grad():
        xi.copy_(xi + 1)
        ri.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    first = [c.clone() for c in captured]
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, captured))
    assert all(torch.equal(a, b) for a, b in zip(first, both()))
