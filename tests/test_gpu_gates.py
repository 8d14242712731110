"""Gates of any size in the gated norm, against float64.

With u = 2^-24: a float32 SiLU(z) is off by at most 10 u whatever z is (exponential and reciprocal within 2 units,
4 and 2 u, the sum 1, the corrections of the exponent and the product 3).  As in the other tests of the norms, 64 u
stand for the sums, the root and the products, so with K = 64 + 4 * 10 an output of magnitude `mag` (the same formula over absolute values) is off by at most K u mag + half
|value|, half a step of its type.  A 16-bit gate may add (8 + 3 |z|) u, less than a quarter of half a step up to
|z| = 60.  Values below the type's normal numbers are off by its smallest one."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
K = 64 + 4 * 10


@pytest.fixture(scope="module")
def ops():
    from fhe_mamba_b200 import mamba_ops
    return mamba_ops


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def mean_of(v, groups):
    m = v.unflatten(-1, (groups, -1)).mean(-1, keepdim=True)
    return m.expand(*m.shape[:-1], v.shape[-1] // groups).flatten(-2)


def close(got, want, mag, k, what):
    half, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).smallest_normal
    err = k * U * mag
    assert torch.isfinite(got).all(), what
    worst = ((got.double() - want).abs() / (err + half * (want.abs() + err) + tiny)).max().item()
    assert worst <= 1, f"{what}: {worst:.3g} of the tolerance"


# rows through words, pairs and single elements, several warps, narrow rows
SIZES = [(40, 1536, 1), (300, 1536, 8), (40, 1002, 1), (40, 1001, 1), (3, 9000, 1), (70, 104, 1), (31, 39, 3), (600, 8, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, width, groups", SIZES)
def test_gates_far_from_zero(ops, dtype, rows, width, groups):
    x = normal(1, rows, width).to(dtype).requires_grad_()
    z = (25 * normal(2, rows, width)).clamp(-60, 60).to(dtype).requires_grad_()
    w = (1 + 0.1 * normal(3, width)).requires_grad_()
    y = ops.gated_rms_norm(x, z, w, 1e-4, groups)
    dy = normal(4, rows, width).to(dtype)
    dx, dz, dw = torch.autograd.grad(y, (x, z, w), dy)
    x, z, w, dy = x.detach().double(), z.detach().double(), w.detach().double(), dy.double()
    q = torch.sigmoid(z)
    p = z * q
    v = x * p
    r = torch.rsqrt(mean_of(v.square(), groups) + 1e-4)
    k = K if dtype == torch.float32 else K + 2 * (8 + 3 * 60)
    close(y.detach(), v * r * w, (v * r * w).abs(), k, "y")
    a, un = dy * w, v * r
    dv = r * (a - un * mean_of(a * un, groups))
    mag = r * (a.abs() + un.abs() * mean_of((a * un).abs(), groups))
    close(dx, dv * p, mag * p.abs(), k, "dx")
    close(dz, dv * x * (q + p * (1 - q)), mag * x.abs() * (q + p.abs() * (1 - q)), k, "dz")
    close(dw, (dy * un).sum(0), (dy * un).abs().sum(0), k + rows, "dw")


@pytest.mark.parametrize("rows, width, groups", SIZES)
def test_float32_gates_keep_their_bits(ops, rows, width, groups):
    """Down to z = -85, the last numbers whose SiLU is normal, a float32 output is off by 46 u: SiLU(z) by 10; the
    root by half of what the mean is (41, and twice 10 of its terms) and 3 roundings, 34; and two products."""
    x, z, w = normal(5, rows, width), (30 * normal(6, rows, width)).clamp(-85, 60), 1 + 0.1 * normal(7, width)
    y = ops.gated_rms_norm(x, z, w, 1e-4, groups)
    v = x.double() * z.double() * torch.sigmoid(z.double())
    want = v * torch.rsqrt(mean_of(v.square(), groups) + 1e-4) * w.double()
    close(y, want, want.abs(), 46, "y")


# the row or group that holds an infinity or a NaN, by layout: words, their groups, pairs, single elements, narrow rows
PLACES = [(8, 1536, 1), (9, 1536, 8), (5, 1002, 1), (5, 1001, 1), (7, 104, 1), (9, 39, 3), (40, 8, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, width, groups", PLACES)
def test_infinities_and_nan_stay_in_their_group(ops, dtype, rows, width, groups):
    x, w = normal(1, rows, width).to(dtype), 1 + 0.1 * normal(3, width)
    z, dy = normal(2, rows, width).to(dtype), normal(4, rows, width).to(dtype)
    x[x == 0] = 1
    z[z == 0] = 1

    def run(x, z):
        x, z = x.clone().requires_grad_(), z.clone().requires_grad_()
        y = ops.gated_rms_norm(x, z, w, 1e-4, groups)
        return [y.detach(), *torch.autograd.grad(y, (x, z), dy)]
    fine = run(x, z)
    each, at = width // groups, (rows // 2, width - 2 - width // 3)
    mine = torch.zeros(rows, width, dtype=torch.bool, device="cuda")
    mine[at[0], at[1] // each * each:(at[1] // each + 1) * each] = True
    here = torch.zeros_like(mine)
    here[at] = True
    inf, nan = float("inf"), float("nan")
    for where, value in (("z", inf), ("z", -inf), ("z", nan), ("x", inf), ("x", nan)):
        a, b = x.clone(), z.clone()
        (a if where == "x" else b)[at] = value
        got = run(a, b)
        for g, f in zip(got, fine):
            assert torch.equal(g[~mine], f[~mine]), (where, value)
        assert torch.isnan(got[0][at])
        if value == inf:  # SiLU(-inf) and NaN leave nothing of the group, an infinity divides it to 0
            assert (got[0][mine & ~here] == 0).all()
        else:
            assert torch.isnan(got[0][mine]).all()


@pytest.mark.parametrize("rows, width, groups", [(5, 1536, 1), (300, 1536, 8), (5, 1001, 1), (70, 104, 1), (31, 39, 3), (600, 8, 1),
                                                 (1000, 1, 1)])
def test_squares_past_float32(ops, rows, width, groups):
    """Some rows of products whose squares pass float32, among rows of ordinary ones: with and without a gate."""
    x, z, w = normal(1, rows, width), (3 * normal(2, rows, width)).clamp(-9, 9), 1 + 0.1 * normal(3, width)
    x[::3] *= 1e25
    x[1::5] *= 1e-3
    y = ops.gated_rms_norm(x, z, w, 1e-4, groups)
    v = x.double() * z.double() * torch.sigmoid(z.double())
    want = v * torch.rsqrt(mean_of(v.square(), groups) + 1e-4) * w.double()
    close(y, want, want.abs(), K + 8, "gate")  # the scaled root: 8 u more
    y = ops.rms_norm(x, w)
    want = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-5) * w.double()
    close(y, want, want.abs(), K + 8, "plain")
