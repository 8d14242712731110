"""The state scan where ranges and masks are hard: 16-bit operands, small and large factors, values that are not
numbers, texts of different sizes in one row, waits that run out.  Against 64 bits, token by token.

Tolerances as in test_gpu_mamba_ops (K roundings of u = 2^-24 of the terms' magnitudes `mag`, half a step of the
output's type), with what an operand's rounding leaves, half = finfo.eps / 2 of the activations' type:
- outputs of that type (y, dx): an operand of two terms, half^2 mag; dB and dC no more;
- float32 outputs: three terms of bfloat16 or two of float16, 3 half^3 or 3 half^2 mag;
and, as an output's own last step can be a subnormal one, half the smallest subnormal of its type.  An operand's
terms below 2^-126 are lost to the tensor cores: 2^-116 for 128 of them times factors up to 8.
"""
import math

import pytest
import torch

from test_gpu_mamba_ops import DTYPES, U, reference, scan_inputs, scan_k

pytestmark = pytest.mark.gpu
HALVES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
    from fhe_mamba_b200 import mamba_ops
    return mamba_ops


def operand(i, dtype):
    """What the operands' roundings leave of a term in an output of `dtype`."""
    t = i["x"].dtype
    half = torch.finfo(t).eps / 2
    if t == torch.float32:
        return 0.0
    return half ** 2 if dtype == t or t == torch.float16 and dtype != torch.float32 else \
        3 * half ** (3 if t == torch.bfloat16 else 2)


def close(got, want, mag, k, what, factor):
    assert got.shape == want.shape, what
    f = torch.finfo(got.dtype)
    got = got.double()
    err = (k * U + factor) * mag
    tol = err + f.eps / 2 * (want.abs() + err) + f.smallest_normal * f.eps / 2 * (1 + 2.0 ** -20) + 2.0 ** -116
    past = want.abs() + tol > f.max  # what the type does not hold may be an infinity
    assert (torch.isfinite(got) | past & (got == want.sign() * math.inf)).all(), what
    worst = torch.where(torch.isfinite(got), (got - want).abs() / tol, 0.0).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the tolerance"


def log_decay_mag(i, mag):
    """Terms behind a token's gradient of log_decay: <dS, S> at the end of its 128 tokens and alpha, beta of those
    after it among them; a cleared state cuts the sum."""
    gamma = mag["log_decay"] + i["write"].double() * mag["write"]
    alive = torch.exp(i["log_decay"].double()) != 0
    out, l = torch.zeros_like(gamma), gamma.shape[1]
    acc = torch.zeros_like(gamma[:, 0])
    for t in reversed(range(l)):
        if t == l - 1 or t % 128 == 127:
            acc = gamma[:, t].clone()
        acc = acc + 2 * gamma[:, t]
        out[:, t] = acc
        acc = torch.where(alive[:, t], acc, 0.0)
    return out


def check(ops, i, dy=None, dfinal=None, names=None):
    """Forward, and the gradients of `names` (all if None) where dy and dfinal are given."""
    y, s = ops.ssm_scan(**i)
    wy, ws, _ = reference(i)
    my, ms, _ = reference(i, absolute=True)
    k = scan_k(i)
    close(y, wy, my, k, "y", operand(i, y.dtype))
    close(s, ws, ms, k, "final state", operand(i, s.dtype))
    if dy is None:
        return
    leaf = {n: v.detach().requires_grad_() for n, v in i.items() if n != "lengths" and v is not None}
    y, s = ops.ssm_scan(**leaf, lengths=i["lengths"])
    got = dict(zip(leaf, torch.autograd.grad([y, s], list(leaf.values()), [dy, dfinal])))
    _, _, want = reference(i, dy, dfinal)
    _, _, mag = reference(i, dy, dfinal, absolute=True)
    mag["log_decay"] = log_decay_mag(i, mag)
    b, l = i["x"].shape[:2]
    for n in names or got:
        close(got[n], want[n], mag[n], 2 * k + (b * l if n == "D" else 0), "d" + n, operand(i, got[n].dtype))


def upstream(i, seed, dy=1.0, dfinal=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, n = i["x"], i["B"].shape[3]
    return ((dy * torch.randn(x.shape, generator=g, device="cuda")).to(x.dtype),
            dfinal * torch.randn(x.shape[0], x.shape[2], x.shape[3], n, generator=g, device="cuda"))


def single(i, c=3):
    """Inputs whose inner products have one term each, so that an operand's rounding is not averaged away."""
    for n in ("B", "C"):
        v = torch.zeros_like(i[n])
        v[..., c] = i[n][..., c]
        i[n] = v
    return i


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("l", [64, 300])
@pytest.mark.parametrize("n", [8, 64, 128])
def test_outputs_hold_two_terms(ops, dtype, l, n):
    """y and dx are one product each (the state is cleared at every token), or the carried state alone: they are off
    by their own rounding and no operand's beside it."""
    i = single(scan_inputs(31, 2, l, 2, 64, n, 1, dtype, strided=False))
    i["D"] = None
    dy, ds = upstream(i, 1)
    check(ops, dict(i, log_decay=torch.full_like(i["write"], -math.inf), initial_state=None), dy, ds * 0)
    keep = i["log_decay"].clone()
    keep[:] = 0
    check(ops, dict(i, log_decay=keep, write=torch.zeros_like(keep)))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("l, p, n, k", [(64, 16, 32, 1), (130, 16, 16, 2), (129, 64, 128, 1), (300, 128, 128, 1),
                                        (200, 8, 104, 1), (257, 72, 40, 2)])
def test_tensor_core_sizes(ops, dtype, l, p, n, k):
    """Rows and columns that fill their tiles in part, with the 128 x 128 gradients."""
    i = scan_inputs(l, 2, l, 2, p, n, k, dtype, carried=True, ragged=l > 200, strided=False)
    check(ops, i, *upstream(i, 2))


def scaled(i, **by):
    return {n: v * by[n] if n in by else v for n, v in i.items()}


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dy, dfinal", [(0.0, 1e-4), (0.0, 1e-6), (0.0, 1e-8), (0.0, 1e-12), (1e-3, 0.0), (1e-4, 1e-5),
                                        (1e-5, 1e-9), (1.0, 1e-9), (300.0, 1e6)])
def test_small_upstream_gradients(ops, dtype, dy, dfinal):
    """Gradients of a mean over many entries, of a scaled loss: nothing falls below the operands' range."""
    i = scan_inputs(21, 2, 300, 2, 64, 128, 1, dtype, strided=False)
    check(ops, i, *upstream(i, 3, dy, dfinal))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("by", [dict(initial_state=1e-9, x=1e-4), dict(B=1e-3, C=1e-3), dict(B=1e-4, C=300.0),
                                dict(x=1e-5, write=1e-4), dict(write=1e-9), dict(initial_state=1e9, write=1e-3),
                                dict(initial_state=1e-30, write=1e-20, x=1e-3), dict(x=300.0, B=1e-3), dict(C=0.0),
                                dict(x=0.0), dict(write=0.0)])
def test_small_and_large_factors(ops, dtype, by):
    i = scan_inputs(22, 2, 300, 2, 64, 128, 1, dtype, strided=False)
    i["D"] = None
    out = by.get("C", 1.0)
    if "initial_state" in by and by["initial_state"] > 1:
        i["C"] = (i["C"] * 1e-3)
        out = 1e-3
        if dtype == torch.float16:
            by = dict(by, initial_state=1e4)  # y fits float16
    i = scaled(i, **by)
    assert out >= 0
    check(ops, i, *upstream(i, 4))


@pytest.mark.parametrize("dtype", HALVES)
def test_rows_of_different_sizes(ops, dtype):
    """Tokens, heads and channels whose sizes lie far apart in one call."""
    i = scan_inputs(23, 2, 300, 4, 64, 128, 2, dtype, strided=False)
    i["D"] = None
    i["x"] = i["x"] * torch.tensor([1, 1e-3, 30, 1e-2], device="cuda", dtype=dtype)[:, None]
    i["write"] = i["write"] * torch.logspace(0, -7, 300, device="cuda")[:, None]
    i["initial_state"] = i["initial_state"] * torch.tensor([1e-6, 1, 1e3, 1e-12], device="cuda")[:, None, None]
    i["C"] = i["C"] * torch.logspace(-3, 1, 300, device="cuda")[:, None, None].to(dtype)
    dy, ds = upstream(i, 5)
    check(ops, i, dy * torch.logspace(1, -3, 300, device="cuda")[:, None, None].to(dtype), ds * 1e-7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("name", ["x", "B", "C", "write", "log_decay"])
def test_nothing_reaches_earlier_tokens(ops, dtype, name, value):
    """A value that is not a number at token 200 leaves the tokens before it as they are (C's leaves all others)."""
    i = scan_inputs(24, 2, 300, 2, 64, 128, 1, dtype, strided=False)
    wy, _, _ = reference(i)
    my, _, _ = reference(i, absolute=True)
    i[name] = i[name].clone()
    i[name][1, 200] = value
    y, s = ops.ssm_scan(**i)
    k = scan_k(i)
    close(y[0], wy[0], my[0], k, "y of the other row", operand(i, y.dtype))
    close(y[1, :200], wy[1, :200], my[1, :200], k, "y", operand(i, y.dtype))
    assert not torch.isfinite(y[1, 200]).all()
    if name == "C":
        close(y[1, 201:], wy[1, 201:], my[1, 201:], k, "y", operand(i, y.dtype))
        assert torch.isfinite(s).all()
    else:
        assert not torch.isfinite(s[1]).all() and torch.isfinite(s[0]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_reaches_later_gradients(ops, dtype):
    """An upstream gradient that is not a number at token 40 leaves dx, dB of the tokens after it as they are."""
    i = scan_inputs(25, 1, 200, 2, 64, 128, 1, dtype, strided=False)
    dy, ds = upstream(i, 6)
    _, _, want = reference(i, dy, ds)
    _, _, mag = reference(i, dy, ds, absolute=True)
    dy[:, 40] = math.nan
    leaf = {n: v.detach().requires_grad_() for n, v in i.items() if n != "lengths"}
    got = dict(zip(leaf, torch.autograd.grad(ops.ssm_scan(**leaf), list(leaf.values()), [dy, ds])))
    for n in ("x", "B", "C", "write"):
        close(got[n][:, 41:], want[n][:, 41:], mag[n][:, 41:], 2 * scan_k(i), "d" + n, operand(i, got[n].dtype))
        assert got[n][:, 40].isnan().any()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("l, b", [(130, 2), (1100, 1)])
@pytest.mark.parametrize("bad", [False, True])
def test_state_in_place(ops, dtype, l, b, bad):
    """fhe_ssm_scan with final_state on initial_state's memory: the same outputs as beside it, also where the call is
    computed again."""
    import ctypes

    from fhe_mamba_b200 import _lib
    i = scan_inputs(28, b, l, 2, 64, 128, 1, dtype, strided=False)
    if bad:
        i["x"][0, 70, 1, 5] = math.inf
    y, s = ops.ssm_scan(**i)
    state, out = i["initial_state"].clone(), torch.empty_like(y)
    a = ops._scan_args(i["x"], i["write"], i["log_decay"], i["B"], i["C"], i["D"], state, None, out, state)
    ws = ops._workspace("fhe_ssm_scan_workspace", a, state.device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    _lib.call("fhe_ssm_scan", ctypes.byref(a))
    assert torch.equal(out.view(torch.int16), y.view(torch.int16)) and torch.equal(state.view(torch.int32), s.view(torch.int32))


WAITS = """
import ctypes, sys
sys.path.insert(0, {root!r})
sys.path.insert(0, {tests!r})
import torch
import test_gpu_scan_range as here
from fhe_mamba_b200 import _lib, mamba_ops as ops

def count():
    n = ctypes.c_uint64()
    _lib.call("fhe_tc_timeouts", ctypes.byref(n))
    return n.value

for dtype in here.HALVES:
    i = here.scan_inputs(29, 12, 130, 16, 64, 128, 1, dtype)  # 192 blocks: no state between segments
    long = here.scan_inputs(30, 1, 1100, 2, 64, 128, 1, dtype)
    leaf = i["x"].requires_grad_()
    before = count()
    here.check(ops, dict(i, x=leaf.detach()))
    assert count() == before
    _lib.call("fhe_scan_wait_limit", 0)
    here.check(ops, dict(i, x=leaf.detach()))
    assert count() > before
    y, s = ops.ssm_scan(**long)
    assert y[:, 1024:].isnan().all() and s.isnan().all()
    assert torch.autograd.grad(ops.ssm_scan(**i)[0].sum(), leaf)[0].isnan().any()
    _lib.call("fhe_scan_wait_limit", 1 << 20)
    before = count()
    here.check(ops, dict(i, x=leaf.detach()))
    here.check(ops, long)
    assert count() == before
print("done")
"""


def test_waits_that_run_out():
    """A wait that runs out (a limit of no polls) is counted and nothing is left unwritten: the outputs are computed
    again in float32, or NaN behind a state that was lost.  In a process of its own, whose count it moves."""
    import os
    import subprocess
    import sys
    tests = os.path.dirname(os.path.abspath(__file__))
    code = WAITS.format(root=os.path.dirname(tests), tests=tests)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("at", [1, 50, 127, 128, 199])
@pytest.mark.parametrize("size", [1e-4, 1e4])
def test_texts_of_different_sizes(ops, dtype, at, size):
    """A cleared state cuts the gradient of log_decay too: a text's is as exact as if it stood alone."""
    i = scan_inputs(26, 2, 200, 2, 32, 64, 1, dtype, carried=False, strided=False)
    i["D"] = None
    i["log_decay"] = i["log_decay"].clone()
    i["log_decay"][:, at] = -math.inf
    i["write"][:, at:] *= size
    dy, ds = upstream(i, 7)
    check(ops, i, dy, ds)
