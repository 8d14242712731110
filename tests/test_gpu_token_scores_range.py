"""Token scores over the whole range of finite logits and of upstream gradients, against 64 bits.

Tolerances, u = 2^-24, K = 64 + vocab / 64 roundings (a term's exponent, exponential and additions).  A sum of
exp(z - max) moves by K u times sum p (1 + |z - max|) <= K u (1 + H + log V) of itself, so a log-probability
lp is off by at most K u (1 + |lp| + log V), H <= log V among it.  The entropy's terms are p |lp| and p lp^2 u; their
sums are at most (1 + log V)^2.  An entry's gradient p (-G - g_e (lp + H)) carries p's and its bracket's errors.
"""
import math

import pytest
import torch

import mamba_plain as plain

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ALL = [torch.float32, torch.bfloat16, torch.float16]
WIDE = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from fhe_mamba_b200 import mamba_ops
    return mamba_ops


def rows_of(seed, r, v, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = 3 * torch.randn(r, v, generator=g, device="cuda")
    return z.to(dtype), torch.randint(0, v, (r,), generator=g, device="cuda")


def check(ops, z, t, k, ge=1.0, seed=0):
    r, v = z.shape
    z = z.detach().requires_grad_()
    got = ops.token_logprobs(z, t, k)
    zd = z.detach().double().requires_grad_()
    want = plain.logprobs(zd, t, k)
    K, lv = (64 + v / 64) * U, 1 + math.log(v)
    assert torch.equal(got.top_ids, want[3])
    for name, a, w in (("logprob", got.logprob, want[0]), ("top", got.top_logprobs, want[2])):
        same = (a.double() == w) | ((a.double() - w).abs() <= K * (w.abs() + lv))
        assert same.all(), (name, a[~same], w[~same])
    assert ((got.entropy.double() - want[1]).abs() <= K * lv ** 2).all(), (got.entropy, want[1])
    g = torch.Generator(device="cuda").manual_seed(seed)
    gl, gh = torch.randn(r, generator=g, device="cuda"), ge * torch.randn(r, generator=g, device="cuda").abs()
    gk = torch.randn(r, k, generator=g, device="cuda")
    outs = lambda o: [o[0], o[1]] + ([o[2]] if k else [])  # noqa: E731
    gs = [torch.where(torch.isfinite(o), q, 0.0) for o, q in zip(outs(want), (gl, gh, gk))]
    (da,) = torch.autograd.grad(outs(got), [z], [q.float() for q in gs])
    (dw,) = torch.autograd.grad(outs(want), [zd], [q.double() for q in gs])
    lp = torch.log_softmax(zd.detach(), -1)
    p = lp.exp()
    size = (gs[0].abs() + gs[2].abs().sum(-1) if k else gs[0].abs())[:, None].double()
    mag = p * (size + gh[:, None] * (lp.clamp(min=-200).abs() + lv))
    tiny = torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps
    lim = K * (lp.clamp(min=-200).abs() + lv) * mag + 2 * U * size * (dw != 0) + \
        torch.finfo(z.dtype).eps / 2 * dw.abs() + tiny + 2.0 ** -126 * (size + 300 * gh[:, None])
    bad = ~((da.double() - dw).abs() <= lim)
    assert not bad.any(), (bad.sum(), da[bad][:5], dw[bad][:5])


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("v", [3000, 50280])
@pytest.mark.parametrize("offset", [2e6, -2e6, 3e9, -3e9, 1e10, -1e10, 1e12, -1e12, 1e18, -1e18, 1e20, -1e20, 1e30, -1e30])
def test_rows_far_from_zero(ops, dtype, offset, v):
    """Whole rows around an offset of any size, their spread as the type holds it."""
    z, t = rows_of(1, 3, v, torch.float32)
    check(ops, (z + offset).to(dtype), t, 5)
    step = abs(offset) * torch.finfo(dtype).eps  # a few steps of the type apart
    check(ops, (offset + step * z.round()).to(dtype), t, 5)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("v", [700, 50280])
@pytest.mark.parametrize("mask", [-2e6, -3e9, -1e10, -1e12, -1e18, -1e20, -1e30, -3e38])
def test_masks_of_large_negative_numbers(ops, dtype, mask, v):
    """Entries masked by a large finite number beside ordinary ones: at the row's start, at its end, all but one."""
    z, t = rows_of(2, 4, v, dtype)
    z[0, : v - 50] = mask
    z[1, 60:] = mask
    z[2, :] = mask
    z[2, v // 2] = 1.25
    z[3, ::2] = mask
    t[0], t[1], t[2] = v - 7, 11, v // 2
    check(ops, z, t, 4)
    t[0], t[1], t[2], t[3] = 3, v - 1, 0, 2  # the masked entries' own scores
    check(ops, z, t, 4)


@pytest.mark.parametrize("dtype", WIDE)
def test_masks_of_several_sizes(ops, dtype):
    """Large numbers of different sizes in one row, ascending and descending, with and without an ordinary entry."""
    z, t = rows_of(3, 4, 40000, dtype)
    size = torch.logspace(3, 30, 40000, device="cuda").to(dtype)
    z[0], z[1] = -size, -size.flip(0)
    z[2] = -size
    z[2, 20000] = 0
    z[3] = size
    t[:] = torch.tensor([0, 39999, 20000, 39999], device="cuda")
    check(ops, z, t, 5)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("low", [-math.inf, "min"])
@pytest.mark.parametrize("ge", [1.0, 10.0, 65536.0])
def test_entropy_gradients_of_masked_rows(ops, dtype, low, ge):
    """Masked entries take no gradient however large the entropy's own is."""
    if dtype == torch.float16:
        ge = min(ge, 100.0)  # the gradients themselves fit float16
    z, t = rows_of(4, 3, 5003, dtype)
    z[:, 4800:] = torch.finfo(dtype).min if low == "min" else low
    z[1, ::2] = z[1, -1]
    t = t % 4800 | 1
    check(ops, z, t, 3, ge)
    odd = torch.zeros(3, 5004, dtype=dtype, device="cuda")[:, 1:]  # rows that 16-byte words do not fit
    odd.copy_(z)
    check(ops, odd, t, 3, ge)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_gradients_of_rows_without_scores(ops, dtype, value):
    """A row whose scores are not numbers has a gradient that is none either; the rows beside it keep theirs."""
    z, t = rows_of(5, 3, 5000, dtype)
    good = z.detach().clone().requires_grad_()
    z[1, 10] = value
    z.requires_grad_()
    got, want = (torch.autograd.grad(ops.token_logprobs(v, t).logprob.sum(), v)[0] for v in (z, good))
    assert got[1].isnan().all() and torch.equal(got[::2], want[::2])
