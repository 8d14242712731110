"""The plaintext Mamba-2 operators as torch functions: the state recurrence
(``ssm_scan``, ``ssm_step``), the causal convolution (``causal_conv``,
``causal_conv_step``) and token scoring (``token_logprobs``).

They run on CUDA tensors through the C ABI (fhe_ssm_scan and the others in
include/fhe_b200.h), on the current stream of the tensors' device, and can be
captured into CUDA graphs; the scan, the convolution and the scores have
gradients (to capture a backward pass, hold no eager autograd graph of the same
leaves: torch would make the capture wait for that graph's stream, and refuses).
Activations are float32, bfloat16 or float16; gates, states and
scores are float32.  Arguments that do not fit raise ValueError before any GPU
work.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import call

_TYPES = {torch.float32: _lib.FHE_F32, torch.bfloat16: _lib.FHE_BF16, torch.float16: _lib.FHE_F16}
MAX_HEAD_DIM, MAX_STATE, MAX_TAPS, MAX_TOP = 128, 256, 8, 64


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _inner(t):
    """t with its innermost axis contiguous (itself if it is)."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _check_devices(op, first, *rest):
    _need(first.is_cuda, f"{op}: CUDA tensors expected")
    for t in rest:
        _need(t is None or t.device == first.device, f"{op}: tensors on different devices")


def _check(op, name, t, shape, dtype):
    _need(tuple(t.shape) == tuple(shape), f"{op}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    _need(t.dtype == dtype, f"{op}: {name} must be {dtype}, got {t.dtype}")


def _workspace(name, args, device):
    n = ctypes.c_uint64()
    call(name, ctypes.byref(args), ctypes.byref(n))
    return torch.empty(n.value, dtype=torch.uint8, device=device) if n.value else None


# the current stream's handle of a device index, without making a Stream object
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


# ---- state recurrence ---------------------------------------------------------------------------


def _scan_fits(x, write, log_decay, B, C, D, state, lengths):
    """Whether the arguments pass every test of ``_check_scan``, which names the one that fails."""
    if x.dim() != 4 or B.dim() != 4:
        return False
    b, l, h, p = x.shape
    k, n = B.shape[2:]
    t, d, f, gates = x.dtype, x.device, torch.float32, (b, l, h)
    return (t in _TYPES and x.is_cuda and k >= 1 and h >= 1 and h % k == 0 and 1 <= p <= MAX_HEAD_DIM
            and 1 <= n <= MAX_STATE and B.shape == C.shape == (b, l, k, n) and B.dtype == C.dtype == t
            and write.shape == log_decay.shape == gates and write.dtype == log_decay.dtype == f
            and B.device == C.device == write.device == log_decay.device == d
            and (D is None or (D.shape == (h,) and D.dtype == f and D.device == d))
            and (state is None or (state.shape == (b, h, p, n) and state.dtype == f and state.device == d))
            and (lengths is None or (lengths.shape == (b,) and lengths.dtype == torch.int32 and lengths.device == d)))


def _check_scan(op, x, write, log_decay, B, C, D, state, lengths, state_name="initial_state"):
    _need(x.dim() == 4, f"{op}: x must be [batch, length, heads, head_dim]")
    b, l, h, p = x.shape
    _need(x.dtype in _TYPES, f"{op}: x must be float32, bfloat16 or float16")
    _need(B.dim() == 4, f"{op}: B must be [batch, length, groups, d_state]")
    k, n = B.shape[2], B.shape[3]
    _need(k >= 1 and h >= 1 and h % k == 0, f"{op}: heads ({h}) must be a positive multiple of groups ({k})")
    _need(1 <= p <= MAX_HEAD_DIM, f"{op}: head_dim must be in [1, {MAX_HEAD_DIM}]")
    _need(1 <= n <= MAX_STATE, f"{op}: d_state must be in [1, {MAX_STATE}]")
    _check(op, "B", B, (b, l, k, n), x.dtype)
    _check(op, "C", C, (b, l, k, n), x.dtype)
    _check(op, "write", write, (b, l, h), torch.float32)
    _check(op, "log_decay", log_decay, (b, l, h), torch.float32)
    if D is not None:
        _check(op, "D", D, (h,), torch.float32)
    if state is not None:
        _check(op, state_name, state, (b, h, p, n), torch.float32)
    if lengths is not None:
        _check(op, "lengths", lengths, (b,), torch.int32)
    _check_devices(op, x, write, log_decay, B, C, D, state, lengths)


def _scan_args(x, write, log_decay, B, C, D, state, lengths, y, final):
    b, l, h, p = x.shape
    return _lib.SsmScanArgs(
        x.device.index, _TYPES[x.dtype], b, l, h, p, B.shape[3], B.shape[2],
        x.data_ptr(), x.stride()[:3], write.data_ptr(), write.stride(), log_decay.data_ptr(), log_decay.stride(),
        B.data_ptr(), B.stride()[:3], C.data_ptr(), C.stride()[:3],
        _ptr(D), _ptr(state), _ptr(lengths), _ptr(y), _ptr(final), None, 0, _stream_of(x.device.index))


def _scan_forward(x, write, log_decay, B, C, D, state, lengths, y, final):
    a = _scan_args(x, write, log_decay, B, C, D, state, lengths, y, final)
    if x.shape[1] >= 64:  # shorter rows need no workspace
        ws = _workspace("fhe_ssm_scan_workspace", a, x.device)
        if ws is not None:
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    call("fhe_ssm_scan", ctypes.byref(a))


def _run_scan(x, write, log_decay, B, C, D, state, lengths):
    b, _, h, p = x.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    final = torch.empty((b, h, p, B.shape[3]), dtype=torch.float32, device=x.device)
    _scan_forward(x, write, log_decay, B, C, D, state, lengths, y, final)
    return y, final


class _SsmScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, write, log_decay, B, C, D, state, lengths):
        y, final = _run_scan(x, write, log_decay, B, C, D, state, lengths)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, write, log_decay, B, C, D, state, lengths)
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        x, write, log_decay, B, C, D, state, lengths = ctx.saved_tensors
        b, l, h, p = x.shape
        k, n = B.shape[2], B.shape[3]
        dy = torch.zeros((b, l, h, p), dtype=x.dtype, device=x.device) if dy is None else dy.contiguous()
        dfinal = None if dfinal is None else dfinal.contiguous()
        new = lambda shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=x.device)  # noqa: E731
        dx, db, dc = new((b, l, h, p), x.dtype), new((b, l, k, n), x.dtype), new((b, l, k, n), x.dtype)
        dw, dla = new((b, l, h)), new((b, l, h))
        dd = new((h,)) if D is not None and ctx.needs_input_grad[5] else None
        ds = new((b, h, p, n)) if state is not None and ctx.needs_input_grad[6] else None
        g = _lib.SsmScanGradArgs(
            _scan_args(x, write, log_decay, B, C, D, state, lengths, None, None),
            dy.data_ptr(), _ptr(dfinal), dx.data_ptr(), dw.data_ptr(), dla.data_ptr(), db.data_ptr(), dc.data_ptr(),
            _ptr(dd), _ptr(ds), None, 0, _stream_of(x.device.index))
        ws = _workspace("fhe_ssm_scan_backward_workspace", g, x.device)
        if ws is not None:
            g.workspace, g.workspace_bytes = ws.data_ptr(), ws.numel()
        call("fhe_ssm_scan_backward", ctypes.byref(g))
        return dx, dw, dla, db, dc, dd, ds, None


def ssm_scan(x, write, log_decay, B, C, D=None, initial_state=None, lengths=None):
    """Mamba-2's recurrence over a padded batch of token rows:

        S_t = exp(log_decay_t) S_(t-1) + write_t x_t (x) B_t,   y_t = S_t C_t + D x_t

    x [batch, length, heads, head_dim]; write, log_decay [batch, length, heads]
    float32 (the layer's dt and A dt); B, C [batch, length, groups, d_state] in
    x's type, shared by heads/groups consecutive heads; D [heads];
    initial_state [batch, heads, head_dim, d_state] float32, zeros if None;
    lengths [batch] int32, full rows if None.  Returns (y, final_state).

    Tokens at or past a row's length are not read, leave the state and get
    y = 0 (a length is clamped to [0, length]).  log_decay = -inf clears the
    state before its token, so several texts may share a row.  x, B and C may
    be slices of one activation tensor (only the last axis must be contiguous,
    else it is copied).  Gradients reach every floating-point argument.

    Rows of 64 tokens and more in 16 bits run on the tensor cores, whose operands
    are split into two or three terms of that type: outputs of the type are off by
    their own rounding and 16 bits of each product, the final state and the gates'
    gradients keep 22 bits and more of every product (in float16 of those within
    2^-17 of the largest of 128 tokens, and 2^-39 of that of the others).  Where
    a product is not finite, y, dx, dB and dC are computed again in float32, so
    that a NaN or an infinity reaches the tokens that the formula says and no
    others; only log_decay's gradient, a running sum from the end of each 128
    tokens, may carry it to the others of those.  log_decay is at most 0, or at
    least the product of the decays of any run of tokens fits float32."""
    if not _scan_fits(x, write, log_decay, B, C, D, initial_state, lengths):
        _check_scan("ssm_scan", x, write, log_decay, B, C, D, initial_state, lengths)
    args = (_inner(x), write, log_decay, _inner(B), _inner(C), _dense(D), _dense(initial_state), _dense(lengths))
    if _wants_grad(x, write, log_decay, B, C, D, initial_state):
        return _SsmScan.apply(*args)
    return _run_scan(*args)


def _check_state_out(op, state, out):
    """Where a step writes the new state: over the old one if `out` is None."""
    _need(state.is_contiguous(), op + ": state and out must be contiguous")
    if out is None or out is state:
        return state
    if out.shape != state.shape or out.dtype != state.dtype:
        _check(op, "out", out, state.shape, state.dtype)
    _need(out.is_contiguous(), op + ": state and out must be contiguous")
    _need(out.device == state.device, op + ": tensors on different devices")
    _need(out.data_ptr() == state.data_ptr() or not _overlap(out, state), op + ": out overlaps part of state")
    return out


def ssm_step(state, x, write, log_decay, B, C, D=None, out=None):
    """One token of each sequence: ``ssm_scan`` without the length axis (x
    [batch, heads, head_dim], write and log_decay [batch, heads], B and C
    [batch, groups, d_state]).  The new state is written to `out` ([batch,
    heads, head_dim, d_state] float32, contiguous), or over `state` if None.
    Returns (y, new state)."""
    op = "ssm_step"
    _need(x.dim() == 3 and B.dim() == 3 and C.dim() == 3 and write.dim() == 2 and log_decay.dim() == 2,
          "ssm_step: one token of each sequence, without a length axis")
    if _wants_grad(state, x, write, log_decay, B, C, D, out):
        _need(False, f"{op} has no gradient (use ssm_scan)")
    b, h, p = x.shape
    k, n = B.shape[1:]
    t, d, f = x.dtype, x.device, torch.float32
    if not (t in _TYPES and x.is_cuda and k >= 1 and h >= 1 and h % k == 0 and 1 <= p <= MAX_HEAD_DIM
            and 1 <= n <= MAX_STATE and B.shape == C.shape == (b, k, n) and B.dtype == C.dtype == t
            and write.shape == log_decay.shape == (b, h) and write.dtype == log_decay.dtype == state.dtype == f
            and state.shape == (b, h, p, n) and B.device == C.device == write.device == log_decay.device == d
            and state.device == d and (D is None or (D.shape == (h,) and D.dtype == f and D.device == d))):
        _check_scan(op, *(v.unsqueeze(1) for v in (x, write, log_decay, B, C)), D, state, None, "state")
    out = _check_state_out(op, state, out)
    x, B, C, D = _inner(x), _inner(B), _inner(C), _dense(D)
    y = torch.empty(x.shape, dtype=t, device=d)
    gates = tuple((v.data_ptr(), (v.stride(0), 0, v.stride(1))) for v in (x, write, log_decay, B, C))
    (xp, xs), (wp, ws), (ap, as_), (bp, bs), (cp, cs) = gates
    a = _lib.SsmScanArgs(d.index, _TYPES[t], b, 1, h, p, n, k, xp, xs, wp, ws, ap, as_, bp, bs, cp, cs, _ptr(D),
                         state.data_ptr(), None, y.data_ptr(), out.data_ptr(), None, 0, _stream_of(d.index))
    call("fhe_ssm_scan", ctypes.byref(a))
    increment_version(out)  # a backward pass that saved the old state must not run on the new one
    return y, out


def _overlap(a, b):
    """Whether two contiguous tensors share memory."""
    a0, b0 = a.data_ptr(), b.data_ptr()
    return a0 < b0 + b.numel() * b.element_size() and b0 < a0 + a.numel() * a.element_size()


# ---- causal convolution -------------------------------------------------------------------------


def _conv_fits(x, weight, bias, state, lengths, activation):
    """Whether the arguments pass every test of ``_check_conv``."""
    if x.dim() != 3 or weight.dim() != 2:
        return False
    b, _, c = x.shape
    k, t, d = weight.shape[1], x.dtype, x.device
    return (t in _TYPES and x.is_cuda and c >= 1 and 1 <= k <= MAX_TAPS and weight.shape == (c, k)
            and weight.dtype == t and weight.device == d
            and (bias is None or (bias.shape == (c,) and bias.dtype == t and bias.device == d))
            and (state is None or (state.shape == (b, k - 1, c) and state.dtype == t and state.device == d))
            and (lengths is None or (lengths.shape == (b,) and lengths.dtype == torch.int32 and lengths.device == d))
            and (activation is None or activation == "silu"))


def _check_conv(op, x, weight, bias, state, lengths, activation, state_name="initial_state"):
    _need(x.dim() == 3, f"{op}: x must be [batch, length, channels]")
    b, _, c = x.shape
    _need(x.dtype in _TYPES, f"{op}: x must be float32, bfloat16 or float16")
    _need(c >= 1, f"{op}: channels must be positive")
    _need(weight.dim() == 2 and 1 <= weight.shape[1] <= MAX_TAPS, f"{op}: weight must be [channels, 1 to {MAX_TAPS} taps]")
    k = weight.shape[1]
    _check(op, "weight", weight, (c, k), x.dtype)
    if bias is not None:
        _check(op, "bias", bias, (c,), x.dtype)
    if state is not None:
        _check(op, state_name, state, (b, k - 1, c), x.dtype)
    if lengths is not None:
        _check(op, "lengths", lengths, (b,), torch.int32)
    _need(activation in (None, "silu"), f"{op}: activation must be None or 'silu'")
    _check_devices(op, x, weight, bias, state, lengths)


def _conv_args(x, weight, bias, state, lengths, silu, y, final):
    b, l, c = x.shape
    return _lib.CausalConvArgs(
        x.device.index, _TYPES[x.dtype], b, l, c, weight.shape[1], silu, 0, x.data_ptr(), x.stride()[:2],
        weight.data_ptr(), _ptr(bias), _ptr(state), _ptr(lengths), _ptr(y), _ptr(final), _stream_of(x.device.index))


def _run_conv(x, weight, bias, state, lengths, silu):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    final = torch.empty((x.shape[0], weight.shape[1] - 1, x.shape[2]), dtype=x.dtype, device=x.device)
    call("fhe_causal_conv", ctypes.byref(_conv_args(x, weight, bias, state, lengths, silu, y, final)))
    return y, final


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu):
        y, final = _run_conv(x, weight, bias, state, lengths, silu)
        ctx.set_materialize_grads(False)
        ctx.silu = silu
        ctx.save_for_backward(x, weight, bias, state, lengths)
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        x, weight, bias, state, lengths = ctx.saved_tensors
        b, l, c = x.shape
        dy = torch.zeros((b, l, c), dtype=x.dtype, device=x.device) if dy is None else dy.contiguous()
        dfinal = None if dfinal is None else dfinal.contiguous()
        dx = torch.empty((b, l, c), dtype=x.dtype, device=x.device)
        dw = torch.empty_like(weight)
        db = torch.empty_like(bias) if bias is not None else None
        ds = torch.empty_like(state) if state is not None and ctx.needs_input_grad[3] else None
        g = _lib.CausalConvGradArgs(
            _conv_args(x, weight, bias, state, lengths, ctx.silu, None, None), dy.data_ptr(), _ptr(dfinal),
            dx.data_ptr(), dw.data_ptr(), _ptr(db), _ptr(ds), None, 0, _stream_of(x.device.index))
        ws = _workspace("fhe_causal_conv_backward_workspace", g, x.device)
        if ws is not None:
            g.workspace, g.workspace_bytes = ws.data_ptr(), ws.numel()
        call("fhe_causal_conv_backward", ctypes.byref(g))
        return dx, dw, db, ds, None, None


def causal_conv(x, weight, bias=None, initial_state=None, lengths=None, activation="silu"):
    """Causal depthwise convolution over the tokens of a padded batch:

        y_t = act(bias + sum_i weight[:, i] row_(t+i)),   row = [initial_state; x]

    x [batch, length, channels] (a slice of a wider tensor will do); weight
    [channels, taps], the last tap on the present token; bias [channels];
    initial_state [batch, taps - 1, channels], the tokens before the row,
    oldest first, zeros if None; lengths [batch] int32; activation "silu" or
    None.  All in x's type.  Returns (y, final_state): y is 0 at and past a
    row's length, final_state is the window behind its last token.  Gradients
    reach every floating-point argument."""
    if not _conv_fits(x, weight, bias, initial_state, lengths, activation):
        _check_conv("causal_conv", x, weight, bias, initial_state, lengths, activation)
    args = (_inner(x), _dense(weight), _dense(bias), _dense(initial_state), _dense(lengths), activation == "silu")
    if _wants_grad(x, weight, bias, initial_state):
        return _CausalConv.apply(*args)
    return _run_conv(*args)


def causal_conv_step(state, x, weight, bias=None, activation="silu", out=None):
    """One token of each sequence: x [batch, channels], state [batch, taps - 1,
    channels].  The moved window is written to `out`, or over `state` if None.
    Returns (y, new state)."""
    op = "causal_conv_step"
    _need(x.dim() == 2, "causal_conv_step: one token of each sequence, without a length axis")
    if _wants_grad(state, x, weight, bias, out):
        _need(False, f"{op} has no gradient (use causal_conv)")
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    x = x.unsqueeze(1)
    if not _conv_fits(x, weight, bias, state, None, activation):
        _check_conv(op, x, weight, bias, state, None, activation, "state")
    out = _check_state_out(op, state, out)
    call("fhe_causal_conv", ctypes.byref(_conv_args(_inner(x), _dense(weight), _dense(bias), state, None,
                                                    activation == "silu", y, out)))
    increment_version(out)
    return y, out


# ---- token scores -------------------------------------------------------------------------------


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # [rows] float32
    entropy: torch.Tensor       # [rows] float32, in nats
    top_logprobs: torch.Tensor  # [rows, top_k] float32
    top_ids: torch.Tensor       # [rows, top_k] int64


def _logprob_args(logits, targets, top_k, logprob, entropy, top_logprobs, top_ids, norm):
    return _lib.TokenLogprobsArgs(
        logits.device.index, _TYPES[logits.dtype], logits.shape[0], logits.shape[1], top_k, 0, logits.data_ptr(),
        logits.stride(0), targets.data_ptr(), _ptr(logprob), _ptr(entropy), _ptr(top_logprobs), _ptr(top_ids),
        norm.data_ptr(), _stream_of(logits.device.index))


def _run_logprobs(logits, targets, top_k):
    r, d = logits.shape[0], logits.device
    logprob = torch.empty(r, dtype=torch.float32, device=d)
    entropy = torch.empty_like(logprob)
    norm = torch.empty((r, 2), dtype=torch.float32, device=d)
    top = torch.empty((r, top_k), dtype=torch.float32, device=d)
    ids = torch.empty((r, top_k), dtype=torch.int64, device=d)
    call("fhe_token_logprobs", ctypes.byref(_logprob_args(logits, targets, top_k, logprob, entropy, top, ids, norm)))
    return logprob, entropy, top, ids, norm


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k):
        logprob, entropy, top, ids, norm = _run_logprobs(logits, targets, top_k)
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        ctx.top_k = top_k
        ctx.save_for_backward(logits, targets, entropy, ids, norm)
        return logprob, entropy, top, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogprob, dentropy, dtop, _):
        logits, targets, entropy, ids, norm = ctx.saved_tensors
        dlogprob, dentropy, dtop = (None if g is None else g.contiguous() for g in (dlogprob, dentropy, dtop))
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        a = _lib.TokenLogprobsGradArgs(
            _logprob_args(logits, targets, ctx.top_k, None, entropy, None, ids, norm), _ptr(dlogprob),
            _ptr(dentropy), _ptr(dtop) if ctx.top_k else None, out.data_ptr(), _stream_of(logits.device.index))
        call("fhe_token_logprobs_backward", ctypes.byref(a))
        return out, None, None


def token_logprobs(logits, targets, top_k=0):
    """Scores of one token per row under softmax(logits): its log-probability,
    the row's entropy and its top_k (at most 64) most probable tokens, the
    lower index first among equals.

    logits [rows, vocab] float32, bfloat16 or float16; targets [rows] int64,
    negative for a row whose token is not scored (log-probability 0); a target
    past the vocabulary scores NaN.  Entries of -inf are impossible tokens.
    Returns a ``TokenLogprobs``; gradients of its floating-point parts reach
    the logits."""
    op, most = "token_logprobs", min(MAX_TOP, logits.shape[-1] if logits.dim() else 0)
    if not (logits.dim() == 2 and logits.dtype in _TYPES and targets.shape == logits.shape[:1]
            and targets.dtype == torch.int64 and 0 <= top_k <= most and most >= 1 and logits.is_cuda
            and targets.device == logits.device):
        _need(logits.dim() == 2 and logits.dtype in _TYPES,
              f"{op}: logits must be [rows, vocab] float32, bfloat16 or float16")
        _need(most >= 1, f"{op}: an empty vocabulary")
        _check(op, "targets", targets, (logits.shape[0],), torch.int64)
        _need(0 <= top_k <= most, f"{op}: top_k must be in [0, {most}]")
        _check_devices(op, logits, targets)
    logits, targets, top_k = _inner(logits), _dense(targets), int(top_k)
    if _wants_grad(logits):
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, top_k))
    return TokenLogprobs(*_run_logprobs(logits, targets, top_k)[:4])
