"""The plaintext Mamba-2 operators on the GPU against their definitions in float64.

Tolerances.  Every output of the scan and the convolution is a sum of products
of the inputs (times decays in [0, 1]), so the same definition on the inputs'
absolute values, `mag`, bounds the sum of the terms' magnitudes.  A term passes
at most K roundings of relative size u = 2^-24: K = 6 per token carried (exp
within 2 ulp, multiply, add), one per summand of the inner products, heads,
tokens and segments, 32 besides.  The error is then at most K u mag, plus half
a step of the output's type, finfo.eps / 2 times the value.

With 16-bit activations rows of 64 tokens and more are multiplied on the tensor
cores, whose operands are rounded to the activations' type, half = finfo.eps / 2:
- a term of y (and of dx, dB, dC) has one rounded factor (the weighted product of
  c and b, or the carried state): half mag;
- a term of the fp32 state has a factor of three such terms (bfloat16, half^3) or
  of two (float16, half^2), and what is formed from states and such products (dw,
  dlog_decay, the carried state's gradient) at most three: 3 half^3 or 3 half^2 mag.
"""
import math

import pytest
import torch

import mamba_plain as plain

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
    from fhe_mamba_b200 import mamba_ops
    return mamba_ops


def close(got, want, mag, k, what="", factor=0.0):
    assert got.shape == want.shape, what
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal
    got = got.double()
    assert torch.isfinite(got).all(), what
    err = (k * U + factor) * mag
    tol = err + half * (want.abs() + err) + tiny
    worst = ((got - want).abs() / tol).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the tolerance"


def scan_inputs(seed, b, l, h, p, n, k, dtype, carried=True, resets=False, ragged=False, strided=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    wide = r(b, l, h * p + 2 * k * n).to(dtype)
    x, B, C = wide[..., :h * p], wide[..., h * p:h * p + k * n], wide[..., h * p + k * n:]
    if not strided:
        x, B, C = x.contiguous(), B.contiguous(), C.contiguous()
    write = torch.nn.functional.softplus(r(b, l, h) - 2)
    la = -torch.rand(h, generator=g, device="cuda") * 4 * write
    if resets:
        la[torch.rand(b, l, h, generator=g, device="cuda") < 0.1] = -math.inf
    d = dict(x=x.unflatten(-1, (h, p)), write=write, log_decay=la, B=B.unflatten(-1, (k, n)), C=C.unflatten(-1, (k, n)),
             D=r(h), initial_state=r(b, h, p, n) if carried else None, lengths=None)
    if ragged:
        d["lengths"] = torch.randint(0, l + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        d["lengths"][0] = l
        if b > 1:
            d["lengths"][1] = 0
    return d


def reference(i, dy=None, dfinal=None, absolute=False):
    """y, final state and the gradients in float64 (of the absolute values when asked)."""
    f = {k: v for k, v in i.items() if k != "lengths" and v is not None}
    f = {k: (v.double().abs() if absolute and k != "log_decay" else v.double()).detach().requires_grad_()
         for k, v in f.items()}
    y, s = plain.scan(f["x"], f["write"], f["log_decay"], f["B"], f["C"], f.get("D"), f.get("initial_state"), i["lengths"])
    if dy is None:
        return y.detach(), s.detach(), {}
    fix = (lambda v: v.double().abs()) if absolute else (lambda v: v.double())
    grads = torch.autograd.grad([y, s], list(f.values()), [fix(dy), fix(dfinal)], allow_unused=True, materialize_grads=True)
    return y.detach(), s.detach(), {k: torch.nan_to_num(v) for k, v in zip(f, grads)}


def rounded(i, dtype):
    """The relative size of the tensor cores' operand roundings in an output of `dtype`."""
    half = torch.finfo(i["x"].dtype).eps / 2
    if i["x"].dtype == torch.float32 or i["x"].shape[1] < 64:
        return 0.0
    return half if dtype == i["x"].dtype else 3 * half ** (3 if i["x"].dtype == torch.bfloat16 else 2)


def scan_k(i):
    b, l, h, p = i["x"].shape
    return 6 * l + i["B"].shape[3] + p + h + 32


def check_scan(ops, i, seed=0, backward=True):
    y, s = ops.ssm_scan(**i)
    wy, ws, _ = reference(i)
    my, ms, _ = reference(i, absolute=True)
    k = scan_k(i)
    close(y, wy, my, k, "y", rounded(i, y.dtype))
    close(s, ws, ms, k, "final state", rounded(i, s.dtype))
    if not backward:
        return
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    dy = torch.randn(y.shape, generator=g, device="cuda").to(y.dtype)
    ds = torch.randn(s.shape, generator=g, device="cuda")
    leaf = {n: v.detach().requires_grad_() for n, v in i.items() if n != "lengths" and v is not None}
    y, s = ops.ssm_scan(**leaf, lengths=i["lengths"])
    got = dict(zip(leaf, torch.autograd.grad([y, s], list(leaf.values()), [dy, ds])))
    _, _, want = reference(i, dy, ds)
    _, _, mag = reference(i, dy, ds, absolute=True)
    b, l, h, p = i["x"].shape
    # the gradient of log_decay is a running sum of alpha - beta with alpha <= gamma, beta <= gamma and
    # gamma = mag + beta: the terms that may have entered the sum are those of every later token
    beta = i["write"].double() * mag["write"]
    gamma = mag["log_decay"] + beta
    mag["log_decay"] = (2 * gamma).flip(1).cumsum(1).flip(1)
    for n in got:
        close(got[n], want[n], mag[n], 2 * k + (b * l if n == "D" else 0), "d" + n, rounded(i, got[n].dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b, l, h, p, n, k", [
    (1, 1, 1, 1, 1, 1), (2, 1, 4, 64, 128, 1), (2, 2, 3, 5, 7, 1), (1, 17, 2, 64, 128, 2), (3, 63, 4, 16, 32, 2),
    (2, 64, 2, 64, 64, 1), (1, 65, 2, 33, 100, 1), (2, 130, 3, 128, 256, 3), (1, 300, 24, 64, 128, 1),
    (1, 513, 2, 48, 128, 1),
])
def test_scan(ops, dtype, b, l, h, p, n, k):
    check_scan(ops, scan_inputs(l, b, l, h, p, n, k, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("carried, resets, ragged, strided", [
    (False, False, False, True), (True, True, False, False), (True, False, True, True), (False, True, True, False)])
def test_scan_masks(ops, dtype, carried, resets, ragged, strided):
    check_scan(ops, scan_inputs(3, 4, 150, 4, 64, 128, 2, dtype, carried, resets, ragged, strided))


def test_scan_without_skip(ops):
    i = scan_inputs(5, 2, 70, 2, 32, 64, 1, torch.float32)
    i["D"] = None
    check_scan(ops, i)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_odd_layouts(ops, dtype):
    """Strides and offsets that no vector load fits, a transposed gate, rows and heads expanded."""
    g = torch.Generator(device="cuda").manual_seed(2)
    b, l, h, p, n = 2, 77, 3, 10, 21
    wide = torch.randn(b, l, 1 + h * (p + 1) + 2 * n, generator=g, device="cuda").to(dtype)
    x = wide[..., 1:1 + h * (p + 1)].unflatten(-1, (h, p + 1))[..., :p]
    B = wide[..., 1 + h * (p + 1):1 + h * (p + 1) + n].unsqueeze(2)
    C = wide[:1, :, -n:].unsqueeze(2).expand(b, l, 1, n)
    w = torch.rand(h, b, l, generator=g, device="cuda").permute(1, 2, 0)
    la = -torch.rand(1, l, 1, generator=g, device="cuda").expand(b, l, h)
    check_scan(ops, dict(x=x, write=w, log_decay=la, B=B, C=C, D=torch.randn(h, generator=g, device="cuda"),
                         initial_state=None, lengths=None))


def test_scan_padding_is_not_read(ops):
    i = scan_inputs(7, 3, 90, 2, 64, 128, 1, torch.bfloat16, ragged=True, strided=False)
    y, s = ops.ssm_scan(**i)
    past = torch.arange(90, device="cuda") >= i["lengths"][:, None]
    for n in ("x", "B", "C", "write", "log_decay"):
        i[n] = i[n].clone()
        i[n][past] = math.nan
    y2, s2 = ops.ssm_scan(**i)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    assert (y2[past] == 0).all()
    leaf = {n: v.detach().requires_grad_() for n, v in i.items() if n != "lengths"}
    y, s = ops.ssm_scan(**leaf, lengths=i["lengths"])
    dy = torch.where(past[..., None, None], math.nan, 1.0).to(y.dtype) * torch.ones_like(y)
    for n, gr in zip(leaf, torch.autograd.grad([y, s], list(leaf.values()), [dy, torch.ones_like(s)])):
        assert torch.isfinite(gr).all(), n
        if n not in ("D", "initial_state"):
            assert (gr[past] == 0).all(), n


def test_lengths_are_clamped(ops):
    i = scan_inputs(8, 3, 40, 2, 16, 16, 1, torch.float32)
    y, s = ops.ssm_scan(**dict(i, lengths=torch.tensor([99, -5, 40], device="cuda", dtype=torch.int32)))
    y2, s2 = ops.ssm_scan(**dict(i, lengths=torch.tensor([40, 0, 40], device="cuda", dtype=torch.int32)))
    assert torch.equal(y, y2) and torch.equal(s, s2) and torch.equal(s[1], i["initial_state"][1])


def test_scan_float16_products_past_its_range(ops):
    """Products of B and C that float16 cannot hold, with outputs that it can: the fp32 walk takes over, forward and
    backward, so no operand's rounding is left."""
    i = scan_inputs(17, 2, 200, 2, 64, 128, 1, torch.float16, strided=False)
    i["B"], i["C"] = i["B"] * 200, i["C"] * 200
    i["write"] = i["write"] * 1e-5
    i["initial_state"] = i["initial_state"] * 1e-3
    assert (i["B"].float() @ i["C"].float().transpose(-1, -2)).abs().max() > 65504
    y, s = ops.ssm_scan(**i)
    wy, ws, _ = reference(i)
    my, ms, _ = reference(i, absolute=True)
    close(y, wy, my, scan_k(i), "y")
    close(s, ws, ms, scan_k(i), "state")
    check_scan(ops, i)


def test_scan_float16_small_factors(ops):
    """Weights and states near the bottom of float16's range lose nothing to it."""
    i = scan_inputs(18, 2, 300, 2, 64, 128, 1, torch.float16)
    i["write"], i["initial_state"], i["D"] = i["write"] * 1e-6, i["initial_state"] * 1e-4, None
    check_scan(ops, i)


@pytest.mark.parametrize("b, l", [(0, 5), (2, 0), (0, 0)])
def test_scan_empty(ops, b, l):
    i = scan_inputs(9, b, l, 2, 8, 16, 1, torch.float32)
    leaf = {n: v.detach().requires_grad_() for n, v in i.items() if n != "lengths"}
    y, s = ops.ssm_scan(**leaf)
    assert y.shape == (b, l, 2, 8) and torch.equal(s, i["initial_state"])
    got = dict(zip(leaf, torch.autograd.grad([y, s], list(leaf.values()), [torch.zeros_like(y), torch.ones_like(s)])))
    assert (got["D"] == 0).all() and (got["initial_state"] == 1).all()


def test_scan_zero_decay_forgets(ops):
    """A cleared state passes nothing on, and its log_decay has gradient exactly 0."""
    i = scan_inputs(10, 1, 200, 2, 64, 128, 1, torch.float32)
    i["log_decay"] = i["log_decay"].clone()
    i["log_decay"][:, 120] = -math.inf
    la = i["log_decay"].requires_grad_()
    y, s = ops.ssm_scan(**i)
    (dla,) = torch.autograd.grad(y.sum() + s.sum(), la)
    assert (dla[:, 120] == 0).all()
    cut = {n: v[:, 120:] if n not in ("D", "initial_state", "lengths") else None for n, v in i.items()}
    cut["D"], cut["lengths"], cut["initial_state"] = i["D"], None, None
    y2, s2 = ops.ssm_scan(**cut)
    my, ms, _ = reference(cut, absolute=True)
    close(y[:, 120:], y2.double(), my, 2 * scan_k(cut), "y")
    close(s, s2.double(), ms, 2 * scan_k(cut), "state")


@pytest.mark.parametrize("name", ["x", "write", "log_decay", "B", "C", "D", "initial_state"])
def test_scan_gradient_is_the_difference(ops, name):
    """<gradient, v> against the central difference along v.  f is linear in each argument alone, so the step
    is exact but for rounding (K u mag / step); along log_decay v moves one token by at most 1, so a term changes
    as exp(step) and the difference is off by at most step^2 / 6 e^step of mag."""
    i = scan_inputs(11, 2, 90, 4, 32, 64, 2, torch.float32, strided=False)
    g = torch.Generator(device="cuda").manual_seed(12)
    leaf = {n: v.detach().requires_grad_() for n, v in i.items() if n != "lengths"}
    y, s = ops.ssm_scan(**leaf)
    dy, ds = torch.randn(y.shape, generator=g, device="cuda"), torch.randn(s.shape, generator=g, device="cuda")
    (grad,) = torch.autograd.grad([y, s], [leaf[name]], [dy, ds])
    v = torch.randn(i[name].shape, generator=g, device="cuda").clamp(-1, 1)
    step = 1.0
    if name == "log_decay":
        v[:, :40] = 0
        v[:, 41:] = 0
        step = 2.0 ** -7
    f = lambda a: sum((o.double() * w.double()).sum() for o, w in zip(ops.ssm_scan(**dict(i, **{name: a})), (dy, ds)))  # noqa: E731
    num = (f(i[name] + step * v) - f(i[name] - step * v)) / (2 * step)
    ana = (grad.double() * v.double()).sum()
    big = dict(i, **{name: i[name].abs() + step * v.abs()}) if name != "log_decay" else i
    my, ms, _ = reference(big, absolute=True)
    total = ((my * dy.abs()).sum() + (ms * ds.abs()).sum()).item()
    tol = 2 * scan_k(i) * U * total * (1 + 1 / step) + (step ** 2 if name == "log_decay" else 0) * total
    assert abs(num - ana).item() <= tol


def test_scan_is_repeatable(ops):
    i = scan_inputs(13, 2, 600, 6, 64, 128, 1, torch.bfloat16)
    leaf = {n: v.detach().requires_grad_() for n, v in i.items() if n != "lengths" and v is not None}

    def once():
        y, s = ops.ssm_scan(**leaf)
        return (y, s) + torch.autograd.grad([y, s], list(leaf.values()), [torch.ones_like(y), torch.ones_like(s)])
    for a, b in zip(once(), once()):
        assert torch.equal(a, b)


def test_no_wait_ran_out(ops):
    import ctypes

    from fhe_mamba_b200 import _lib
    ops.ssm_scan(**scan_inputs(19, 2, 300, 4, 64, 128, 1, torch.bfloat16))
    torch.cuda.synchronize()
    n = ctypes.c_uint64(1)
    _lib.call("fhe_tc_timeouts", ctypes.byref(n))
    assert n.value == 0


def test_scan_on_a_long_row(ops):
    """Two rows of 9000 tokens against two of 4500 carried on: the same states and outputs, K u mag apart."""
    for dtype in DTYPES:
        i = scan_inputs(20, 2, 9000, 2, 32, 64, 1, dtype)
        y, s = ops.ssm_scan(**i)
        half = {n: (v[:, :4500] if n in ("x", "B", "C", "write", "log_decay") else v) for n, v in i.items()}
        y1, s1 = ops.ssm_scan(**half)
        half = {n: (v[:, 4500:] if n in ("x", "B", "C", "write", "log_decay") else v) for n, v in i.items()}
        y2, s2 = ops.ssm_scan(**dict(half, initial_state=s1))
        # decays of at most 4 per unit of write: contributions older than some 600 tokens are below u; a y is a sum
        # of at most that many terms of size max |x| |B| |C| w 64 <= the largest |y| a few times over
        big = y.float().abs().max().item()
        tol = 8 * (4000 * U + 2 * torch.finfo(dtype).eps) * big if dtype != torch.float32 else 8 * 4000 * U * big
        assert (torch.cat([y1, y2], 1).float() - y.float()).abs().max().item() <= tol
        assert (s2 - s).abs().max() <= 8 * 4000 * U * s.abs().max() + 3 * (torch.finfo(dtype).eps / 2) ** 2 * 64


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b, h, p, n, k", [(1, 1, 1, 1, 1), (3, 4, 64, 128, 1), (2, 6, 33, 100, 2), (5, 2, 128, 256, 1),
                                           (2, 3, 16, 16, 3), (2, 2, 20, 18, 1)])
def test_step(ops, dtype, b, h, p, n, k):
    i = scan_inputs(b, b, 1, h, p, n, k, dtype)
    one = {m: v[:, 0] for m, v in i.items() if m in ("x", "write", "log_decay", "B", "C")}
    wy, ws, _ = reference(i)
    my, ms, _ = reference(i, absolute=True)
    state = i["initial_state"].clone()
    y, new = ops.ssm_step(state, **one, D=i["D"], out=torch.empty_like(state))
    close(y, wy[:, 0], my[:, 0], scan_k(i), "y")
    close(new, ws, ms, scan_k(i), "state")
    assert torch.equal(state, i["initial_state"])
    y2, same = ops.ssm_step(state, **one, D=i["D"])
    assert same is state and torch.equal(state, new) and torch.equal(y, y2)


def test_steps_follow_the_scan(ops):
    i = scan_inputs(14, 2, 12, 4, 64, 128, 1, torch.float32)
    state = i["initial_state"].clone()
    wy, ws, _ = reference(i)
    my, ms, _ = reference(i, absolute=True)
    for t in range(12):
        y, _ = ops.ssm_step(state, *(i[n][:, t] for n in ("x", "write", "log_decay", "B", "C")), D=i["D"])
        close(y, wy[:, t], my[:, t], scan_k(i), f"y {t}")
    close(state, ws, ms, scan_k(i), "state")


def test_steps_over_a_saved_state_are_seen(ops):
    """A step that overwrites a state which a backward pass still needs makes that pass an error, as torch's own
    in-place operations do."""
    i = scan_inputs(4, 2, 5, 2, 16, 32, 1, torch.float32, carried=True)
    x = i["x"].requires_grad_()
    one = [i[n][:, 0].detach() for n in ("x", "write", "log_decay", "B", "C")]
    y, _ = ops.ssm_scan(**i)
    ops.ssm_step(i["initial_state"], *one)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)
    y, _ = ops.ssm_scan(**i)
    ops.ssm_step(i["initial_state"], *one, out=torch.empty_like(i["initial_state"]))
    torch.autograd.grad(y.sum(), x)
    x = torch.randn(2, 5, 32, device="cuda", requires_grad=True)
    w, state = torch.randn(32, 4, device="cuda"), torch.randn(2, 3, 32, device="cuda")
    y, _ = ops.causal_conv(x, w, initial_state=state)
    ops.causal_conv_step(state, x[:, 0].detach(), w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)


def test_step_refuses_overlap(ops):
    i = scan_inputs(15, 2, 1, 2, 8, 16, 1, torch.float32)
    buf = torch.zeros(5, 2, 8, 16, device="cuda")
    one = [i[n][:, 0] for n in ("x", "write", "log_decay", "B", "C")]
    with pytest.raises(ValueError, match="overlaps"):
        ops.ssm_step(buf[0:2], *one, out=buf[1:3])
    with pytest.raises(ValueError, match="contiguous"):
        ops.ssm_step(buf[::2][:2], *one)


# ---- convolution ------------------------------------------------------------------------------------


def conv_inputs(seed, b, l, c, k, dtype, carried=True, ragged=False, before=0, after=0, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    d = dict(x=r(b, l, before + c + after)[..., before:before + c], weight=r(c, k), bias=r(c) if bias else None,
             initial_state=r(b, k - 1, c) if carried else None, lengths=None)
    if ragged:
        d["lengths"] = torch.randint(0, l + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        d["lengths"][0] = min(l, 1)
        d["lengths"][-1] = 0
    return d


def check_conv(ops, i, activation, seed=0):
    """mag: the absolute sum; SiLU's slope is at most 1.1, its own 10 roundings are relative to its value, and its
    second derivative is at most 1/2 (the gradient's slope moves with the rounding of its argument)."""
    leaf = {n: v.detach().requires_grad_() for n, v in i.items() if n != "lengths" and v is not None}
    ref = {n: v.double().detach().requires_grad_() for n, v in leaf.items()}
    mag = {n: v.double().abs().detach().requires_grad_() for n, v in leaf.items()}
    silu = activation == "silu"
    y, s = ops.causal_conv(**leaf, lengths=i["lengths"], activation=activation)
    args = lambda d: (d["x"], d["weight"], d.get("bias"), d.get("initial_state"), i["lengths"])  # noqa: E731
    wy, ws = plain.conv(*args(ref), silu=silu)
    my, _ = plain.conv(*args(mag), silu=False)
    k = 32 + i["weight"].shape[1]
    close(y, wy.detach(), 1.1 * my.detach(), k, "y")
    assert torch.equal(s.double(), ws)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dy = torch.randn(y.shape, generator=g, device="cuda").to(y.dtype)
    ds = torch.randn(s.shape, generator=g, device="cuda").to(y.dtype)
    got = torch.autograd.grad([y, s], list(leaf.values()), [dy, ds])
    want = torch.autograd.grad([wy, ws], list(ref.values()), [dy.double(), ds.double()])
    _, ms = plain.conv(*args(mag), silu=False)
    scale = (1.1 + 0.5 * my.detach()) if silu else 1.0
    m = torch.autograd.grad([my, ms], list(mag.values()), [dy.double().abs() * scale, ds.double().abs()])
    b, l, _ = i["x"].shape
    for n, a, w, q in zip(leaf, got, want, m):
        close(a, w, q, k + (b * l if n in ("weight", "bias") else 0), "d" + n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b, l, c, k, silu", [
    (1, 1, 1, 1, True), (2, 1, 16, 4, True), (2, 3, 8, 4, False), (1, 7, 24, 8, True), (3, 63, 40, 2, True),
    (2, 65, 1001, 3, True), (2, 200, 1792, 4, True), (1, 130, 64, 5, False), (1, 64, 32, 6, True), (1, 33, 32, 7, True)])
def test_conv(ops, dtype, b, l, c, k, silu):
    check_conv(ops, conv_inputs(l, b, l, c, k, dtype), "silu" if silu else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("carried, ragged, before, after, bias", [
    (False, False, 1536, 24, True), (True, True, 8, 0, False), (False, True, 3, 2, True), (True, True, 0, 8, True)])
def test_conv_forms(ops, dtype, carried, ragged, before, after, bias):
    check_conv(ops, conv_inputs(1, 4, 100, 144, 4, dtype, carried, ragged, before, after, bias), "silu")


def test_conv_padding_is_not_read(ops):
    i = conv_inputs(2, 3, 50, 64, 4, torch.bfloat16, ragged=True)
    y, s = ops.causal_conv(**i)
    past = torch.arange(50, device="cuda") >= i["lengths"][:, None]
    x = i["x"].clone()
    x[past] = math.nan
    leaf = {n: v.detach().requires_grad_() for n, v in dict(i, x=x).items() if n != "lengths"}
    y2, s2 = ops.causal_conv(**leaf, lengths=i["lengths"])
    assert torch.equal(y, y2) and torch.equal(s, s2) and (y[past] == 0).all()
    dy = torch.where(past[..., None], math.nan, 1.0).to(y.dtype) * torch.ones_like(y)
    for n, g in zip(leaf, torch.autograd.grad([y2, s2], list(leaf.values()), [dy, torch.ones_like(s)])):
        assert torch.isfinite(g).all(), n


@pytest.mark.parametrize("b, l", [(0, 5), (2, 0)])
def test_conv_empty(ops, b, l):
    i = conv_inputs(3, b, l, 16, 4, torch.float32)
    leaf = {n: v.detach().requires_grad_() for n, v in i.items() if n != "lengths"}
    y, s = ops.causal_conv(**leaf)
    assert y.shape == (b, l, 16) and torch.equal(s, i["initial_state"])
    got = dict(zip(leaf, torch.autograd.grad([y, s], list(leaf.values()), [torch.zeros_like(y), torch.ones_like(s)])))
    assert (got["weight"] == 0).all() and (got["bias"] == 0).all() and (got["initial_state"] == 1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k, c", [(1, 8), (2, 9), (4, 1792), (8, 16)])
def test_conv_steps_follow_the_rows(ops, dtype, k, c):
    i = conv_inputs(4, 3, 9, c, k, dtype)
    y, s = ops.causal_conv(**i)
    state = i["initial_state"].clone()
    for t in range(9):
        out = torch.empty_like(state) if t % 2 else None
        got, state = ops.causal_conv_step(state, i["x"][:, t], i["weight"], i["bias"], out=out)
        assert torch.equal(got, y[:, t])
    assert torch.equal(state, s)


# ---- token scores -----------------------------------------------------------------------------------


def logits_of(seed, r, v, dtype, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = (spread * torch.randn(r, v, generator=g, device="cuda")).to(dtype)
    return z, torch.randint(0, v, (r,), generator=g, device="cuda")


def check_logprobs(ops, z, t, k, seed=0):
    """exp, log and the sums are within 32 roundings of terms relative to the value 1 + |z - max| (the exponent's
    rounding and __expf's 2 + 1.16 |x| ulp), and the sums of V terms add log2-depth plus per-thread chains below V / 64.
    A log-probability is a difference of numbers up to |z - max| + log V: the same bound."""
    z = z.detach().requires_grad_()
    got = ops.token_logprobs(z, t, k)
    zd = z.detach().double().requires_grad_()
    want = plain.logprobs(zd, t, k)
    assert torch.equal(got.top_ids, want[3])
    v = z.shape[1]
    finite = torch.where(torch.isinf(zd), 0.0, zd).detach()
    spread = (finite.max(-1).values - finite.min(-1).values + math.log(v) + 1)
    tol = (64 + v / 64) * U * spread
    for a, w, lim in ((got.logprob, want[0], tol), (got.entropy, want[1], tol * 2),
                      (got.top_logprobs, want[2], tol[:, None])):
        same = (a.double() == w) | ((a.double() - w).abs() <= lim)
        assert same.all(), (a, w)
    g = torch.Generator(device="cuda").manual_seed(seed)
    gl, ge = torch.randn(2, z.shape[0], generator=g, device="cuda").unbind(0)
    gk = torch.randn(z.shape[0], k, generator=g, device="cuda")
    live = torch.isfinite(want[1]) & torch.isfinite(want[0])
    rows = live & (zd.max(-1).values > -math.inf)
    outs = lambda o: [o[0][rows].double(), o[1][rows].double()] + ([o[2][rows].double()] if k else [])  # noqa: E731
    gs = [gl[rows].double(), ge[rows].double()] + ([gk[rows].double()] if k else [])
    gs = [torch.where(torch.isfinite(o), q, 0.0) for o, q in zip(outs(want), gs)]
    (da,) = torch.autograd.grad(outs(got), [z], gs)
    (dw,) = torch.autograd.grad(outs(want), [zd], gs)
    size = gl.abs() + ge.abs() * spread + gk.abs().sum(-1)
    prob = torch.nan_to_num(torch.softmax(zd.detach(), -1))
    mag = prob * size[:, None].double()
    mag = mag + (dw - 0).abs()
    lim = (64 + v / 64) * U * spread[:, None] * mag + torch.finfo(z.dtype).eps / 2 * dw.abs() + 1e-30 + \
        torch.finfo(z.dtype).smallest_normal
    assert ((da.double() - dw).abs() <= lim).all(), ((da.double() - dw).abs() / lim).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r, v, k", [(1, 1, 1), (1, 2, 2), (3, 7, 5), (4, 64, 64), (5, 257, 3), (2, 1003, 64),
                                     (3, 4099, 20), (2, 8192, 0), (2, 50280, 8), (1, 50280, 64), (2, 200001, 5)])
def test_logprobs(ops, dtype, r, v, k):
    z, t = logits_of(v, r, v, dtype)
    check_logprobs(ops, z, t, k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_logprobs_masks(ops, dtype):
    z, t = logits_of(1, 6, 3001, dtype)
    z[:, 2900:] = -math.inf          # a padded vocabulary
    z[1, :] = -math.inf              # one possible token
    z[1, 77] = 1.5
    t = t % 2900
    t[1] = 77
    t[2] = -1                        # not scored
    t[3] = 2950                      # an impossible token
    check_logprobs(ops, z, t, 6)
    z[4, :] = -math.inf              # nothing possible
    got = ops.token_logprobs(z, t, 6)
    assert got.logprob[4] == -math.inf and got.entropy[4] == 0 and (got.top_logprobs[4] == -math.inf).all()
    assert got.top_ids[4].tolist() == [0, 1, 2, 3, 4, 5]
    assert got.logprob[3] == -math.inf and got.logprob[2] == 0
    leaf = z.requires_grad_()
    o = ops.token_logprobs(leaf, t, 6)
    (d,) = torch.autograd.grad(o.entropy.sum(), leaf)
    assert torch.isfinite(d).all() and (d[4] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_logprobs_lowest_masks(ops, dtype):
    """Masks of the type's lowest number: impossible beside ordinary entries, uniform among themselves."""
    z, t = logits_of(4, 4, 2000, dtype)
    low = torch.finfo(dtype).min
    z[0, 100:] = low
    t[0] = 50
    z[1, :] = low
    z[2, :] = low
    z[2, 7] = -math.inf
    z[3, 5:] = -math.inf
    z[3, :5] = low
    t[2], t[3] = 9, 2
    check_logprobs(ops, z, t, 5)


def test_logprobs_far_from_zero(ops):
    """A common offset changes nothing but the logits' own rounding: scores and gradients keep their digits."""
    z, t = logits_of(6, 5, 3000, torch.float32)
    check_logprobs(ops, z + 1e5, t, 4)
    check_logprobs(ops, z * 1e3 - 1e6, t, 4)
    check_logprobs(ops, z * 1e36, t, 4)


def test_logprobs_ties_and_odd_rows(ops):
    z = torch.zeros(3, 9000, device="cuda")          # every entry equal: more candidates than are kept
    z[1, 5000:] = 1
    z[2] = torch.arange(9000, device="cuda") / 9000  # ascending: the largest come last
    t = torch.tensor([3, 6000, 8999], device="cuda")
    check_logprobs(ops, z, t, 64)
    z = torch.tensor([[-0.0, 0.0, -1.0, 0.0]], device="cuda")
    assert ops.token_logprobs(z, t[:1], 4).top_ids.tolist() == [[0, 1, 3, 2]]


def test_logprobs_not_numbers(ops):
    z, t = logits_of(2, 3, 500, torch.float32)
    z[0, 10] = math.nan
    z[1, 10] = math.inf
    t[2] = 500
    got = ops.token_logprobs(z, t, 2)
    assert got.logprob[:2].isnan().all() and got.entropy[:2].isnan().all() and got.logprob[2].isnan()
    assert got.top_ids[1, 0] == 10 and torch.equal(got.top_ids[0], torch.argsort(z[0].nan_to_num(-1e9), descending=True)[:2])
    z = torch.full((1, 3), math.nan, device="cuda")
    assert ops.token_logprobs(z, t[:1] * 0, 3).top_ids.tolist() == [[0, 1, 2]]


def test_logprobs_strided_and_empty(ops):
    z, t = logits_of(3, 4, 1000, torch.bfloat16)
    wide = torch.zeros(4, 1003, device="cuda", dtype=torch.bfloat16)
    wide[:, 1:1001] = z
    for a, b in zip(ops.token_logprobs(wide[:, 1:1001], t, 5), ops.token_logprobs(z, t, 5)):
        assert torch.equal(a, b) or (a.double() - b.double()).abs().max() < 1e-5
    e = ops.token_logprobs(z[:0], t[:0], 5)
    assert e.logprob.shape == (0,) and e.top_ids.shape == (0, 5)
    leaf = z[:0].requires_grad_()
    (g,) = torch.autograd.grad(ops.token_logprobs(leaf, t[:0]).logprob.sum(), leaf)
    assert g.shape == (0, 1000)


# ---- streams and graphs -----------------------------------------------------------------------------


def all_ops(ops, i, c, z, t):
    """Every operator with its gradient; the leaves are made anew by each call."""
    leaf = {n: v.detach().requires_grad_() for n, v in i.items() if n != "lengths"}
    y, s = ops.ssm_scan(**leaf, lengths=i["lengths"])
    cl = {n: v.detach().requires_grad_() for n, v in c.items() if n != "lengths"}
    v, f = ops.causal_conv(**cl, lengths=c["lengths"])
    zl = z.detach().requires_grad_()
    o = ops.token_logprobs(zl, t, 5)
    state = i["initial_state"].clone()
    step = ops.ssm_step(state, *(i[n][:, 0] for n in ("x", "write", "log_decay", "B", "C")))
    g = torch.autograd.grad([y, s, v, f, o.logprob, o.entropy], list(leaf.values()) + list(cl.values()) + [zl],
                            [torch.ones_like(q) for q in (y, s, v, f, o.logprob, o.entropy)])
    return [y, s, v, f, *o, *step, *g]


def stream_inputs():
    z, t = logits_of(5, 7, 5000, torch.float32)
    return scan_inputs(5, 2, 300, 4, 64, 128, 1, torch.bfloat16, ragged=True), conv_inputs(5, 2, 90, 64, 4, torch.float16, ragged=True), z, t


def test_another_stream(ops):
    a = stream_inputs()
    want = all_ops(ops, *a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = all_ops(ops, *a)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(got, want))


def test_captured_and_replayed(ops):
    """Two graphs of the same calls, replayed in turn on new inputs."""
    a, b = stream_inputs(), stream_inputs()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        all_ops(ops, *a)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for args in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = all_ops(ops, *args)
        graphs.append((g, out, args))
    for rep in range(2):
        for _, _, args in graphs:
            args[0]["x"].mul_(-0.5)
            args[2].add_(torch.randn_like(args[2]))
        for g, _, _ in graphs:
            g.replay()
        for _, out, args in graphs:
            want = all_ops(ops, *args)
            assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(out, want))


def test_backward_captured_after_an_eager_graph(ops):
    """The same leaves eagerly and then captured, once the eager graph is gone (torch ties a leaf's gradient to the
    stream of a graph that still lives, and a capture cannot wait for that stream)."""
    i = scan_inputs(6, 2, 100, 2, 64, 128, 1, torch.float32)
    leaf = {n: v.detach().requires_grad_() for n, v in i.items() if n != "lengths" and v is not None}

    def once():
        y, f = ops.ssm_scan(**leaf)
        return torch.autograd.grad([y, f], list(leaf.values()), [torch.ones_like(y), torch.ones_like(f)])
    want = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = once()
    g.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
