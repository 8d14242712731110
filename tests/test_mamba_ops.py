"""The plaintext Mamba-2 operators on CPU: refused arguments, of the Python
functions and of the C entry points (none of them reaches a GPU)."""
import ctypes

import pytest
import torch

from fhe_mamba_b200 import _lib, mamba_ops as ops


def scan_inputs(b=2, l=5, h=4, p=8, n=16, k=2, dtype=torch.float32):
    return dict(x=torch.zeros(b, l, h, p, dtype=dtype), write=torch.zeros(b, l, h), log_decay=torch.zeros(b, l, h),
                B=torch.zeros(b, l, k, n, dtype=dtype), C=torch.zeros(b, l, k, n, dtype=dtype))


@pytest.mark.parametrize("change, message", [
    (dict(x=torch.zeros(2, 5, 4)), "batch, length, heads, head_dim"),
    (dict(x=torch.zeros(2, 5, 4, 8, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(x=torch.zeros(2, 5, 3, 8)), "multiple of groups"),
    (dict(x=torch.zeros(2, 5, 4, 129)), "head_dim"),
    (dict(B=torch.zeros(2, 5, 2, 257), C=torch.zeros(2, 5, 2, 257)), "d_state"),
    (dict(B=torch.zeros(2, 4, 2, 16)), "B must have shape"),
    (dict(C=torch.zeros(2, 5, 2, 8)), "C must have shape"),
    (dict(C=torch.zeros(2, 5, 2, 16, dtype=torch.bfloat16)), "C must be"),
    (dict(write=torch.zeros(2, 5, 4, dtype=torch.bfloat16)), "write must be"),
    (dict(log_decay=torch.zeros(2, 5)), "log_decay must have shape"),
    (dict(D=torch.zeros(3)), "D must have shape"),
    (dict(initial_state=torch.zeros(2, 4, 16, 8)), "initial_state must have shape"),
    (dict(initial_state=torch.zeros(2, 4, 8, 16, dtype=torch.bfloat16)), "initial_state must be"),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), "lengths must be"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths must have shape"),
    ({}, "CUDA tensors expected"),
])
def test_scan_refusals(change, message):
    with pytest.raises(ValueError, match=message):
        ops.ssm_scan(**dict(scan_inputs(), **change))


def test_step_refusals():
    i = {k: v[:, 0] for k, v in scan_inputs().items()}
    state = torch.zeros(2, 4, 8, 16)
    with pytest.raises(ValueError, match="without a length axis"):
        ops.ssm_step(state, **scan_inputs())
    with pytest.raises(ValueError, match="state must have shape"):
        ops.ssm_step(state[:1], **i)
    with pytest.raises(ValueError, match="no gradient"):
        ops.ssm_step(state, **dict(i, x=i["x"].requires_grad_()))
    i["x"].requires_grad_(False)
    with pytest.raises(ValueError, match="CUDA tensors expected"):
        ops.ssm_step(state, **i)
    c = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="without a length axis"):
        ops.causal_conv_step(torch.zeros(2, 3, 8), c[:, None], torch.zeros(8, 4))
    with pytest.raises(ValueError, match="state must have shape"):
        ops.causal_conv_step(torch.zeros(2, 2, 8), c, torch.zeros(8, 4))


@pytest.mark.parametrize("change, message", [
    (dict(x=torch.zeros(2, 8)), "batch, length, channels"),
    (dict(x=torch.zeros(2, 5, 8, dtype=torch.int32)), "float32, bfloat16 or float16"),
    (dict(weight=torch.zeros(8, 9)), "taps"),
    (dict(weight=torch.zeros(7, 4)), "weight must have shape"),
    (dict(weight=torch.zeros(8, 4, dtype=torch.float16)), "weight must be"),
    (dict(bias=torch.zeros(9)), "bias must have shape"),
    (dict(initial_state=torch.zeros(2, 4, 8)), "initial_state must have shape"),
    (dict(lengths=torch.zeros(2)), "lengths must be"),
    (dict(activation="gelu"), "activation"),
    ({}, "CUDA tensors expected"),
])
def test_conv_refusals(change, message):
    with pytest.raises(ValueError, match=message):
        ops.causal_conv(**dict(dict(x=torch.zeros(2, 5, 8), weight=torch.zeros(8, 4)), **change))


@pytest.mark.parametrize("change, message", [
    (dict(logits=torch.zeros(3)), "rows, vocab"),
    (dict(logits=torch.zeros(3, 7, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(logits=torch.zeros(3, 0)), "empty vocabulary"),
    (dict(targets=torch.zeros(2, dtype=torch.int64)), "targets must have shape"),
    (dict(targets=torch.zeros(3, dtype=torch.int32)), "targets must be"),
    (dict(top_k=8), "top_k"),
    (dict(top_k=-1), "top_k"),
    (dict(logits=torch.zeros(3, 100), top_k=65), "top_k"),
    ({}, "CUDA tensors expected"),
])
def test_logprob_refusals(change, message):
    with pytest.raises(ValueError, match=message):
        ops.token_logprobs(**dict(dict(logits=torch.zeros(3, 7), targets=torch.zeros(3, dtype=torch.int64)), **change))


def scan_struct(**kw):
    """A C argument block whose pointers are never followed: each call below is refused before."""
    s = dict(dtype=0, batch=1, length=4, heads=2, head_dim=8, d_state=16, groups=1, x=256, write=256, log_decay=256,
             b=256, c=256, y=256, final_state=256)
    s.update(kw)
    return _lib.SsmScanArgs(**s)


@pytest.mark.parametrize("kw, message", [
    (dict(dtype=7), "dtype"), (dict(heads=3, groups=2), "multiple of groups"), (dict(groups=0), "multiple of groups"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=200), "head_dim"), (dict(d_state=300), "d_state"),
    (dict(x=None), "null input"), (dict(y=None), "null output"), (dict(final_state=None), "null output"),
    (dict(batch=1 << 20, length=1 << 20), "below 2"), (dict(batch=1 << 8, heads=1 << 16), "below 2"),
    (dict(batch=1, heads=1 << 16, length=1 << 20), "below 2"),
    (dict(length=4096), "workspace too small"), (dict(length=4096, workspace=256 * 3 + 1, workspace_bytes=1 << 40), "aligned"),
])
def test_scan_c_refusals(kw, message):
    assert _lib.load().fhe_ssm_scan(ctypes.byref(scan_struct(**kw))) == _lib.FHE_ERR_INVALID
    assert message in _lib.last_error()


def test_backward_c_refusals():
    lib = _lib.load()
    g = _lib.SsmScanGradArgs(f=scan_struct())
    assert lib.fhe_ssm_scan_backward(ctypes.byref(g)) == _lib.FHE_ERR_INVALID
    assert "workspace too small" in _lib.last_error()
    n = ctypes.c_uint64()
    assert lib.fhe_ssm_scan_backward_workspace(ctypes.byref(g), ctypes.byref(n)) == 0 and n.value > 0
    c = _lib.CausalConvArgs(dtype=0, batch=1, length=4, channels=8, taps=9, x=256, y=256, weight=256)
    assert lib.fhe_causal_conv(ctypes.byref(c)) == _lib.FHE_ERR_INVALID and "taps" in _lib.last_error()
    c.taps = 4
    assert lib.fhe_causal_conv(ctypes.byref(c)) == _lib.FHE_ERR_INVALID and "final_state" in _lib.last_error()
    c.final_state = c.initial_state = 512
    assert lib.fhe_causal_conv(ctypes.byref(c)) == _lib.FHE_ERR_INVALID and "one token" in _lib.last_error()
    t = _lib.TokenLogprobsArgs(dtype=0, rows=1, vocab=10, top_k=11)
    assert lib.fhe_token_logprobs(ctypes.byref(t)) == _lib.FHE_ERR_INVALID and "top_k" in _lib.last_error()
    t.top_k = 0
    assert lib.fhe_token_logprobs(ctypes.byref(t)) == _lib.FHE_ERR_INVALID and "null" in _lib.last_error()
    for name in ("fhe_ssm_scan", "fhe_ssm_scan_backward", "fhe_causal_conv", "fhe_causal_conv_backward",
                 "fhe_token_logprobs", "fhe_token_logprobs_backward"):
        assert getattr(lib, name)(None) == _lib.FHE_ERR_INVALID and "null" in _lib.last_error()


def test_client_alternatives_refusals(tmp_path):
    import json

    from fhe_mamba_b200 import mamba2_decode
    out = tmp_path / "r.json"
    for extra in (["--client-alternatives", "3"], ["--client-alternatives", "65", "--autoregressive-client-loop", "1"]):
        assert mamba2_decode.main(["--input-chain", "missing", "--output-json", str(out)] + extra) == 2
        assert "--client-alternatives" in json.loads(out.read_text())["error"]
