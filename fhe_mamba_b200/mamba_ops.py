"""The plaintext Mamba-2 operators as torch functions: the state recurrence
(``ssm_scan``, ``ssm_step``), the causal convolution (``causal_conv``,
``causal_conv_step``), the norms with their residual or gate (``rms_norm``,
``add_rms_norm``, ``gated_rms_norm``), the token embedding (``embedding``),
token scoring (``token_logprobs``) and beam search's selection and reordering of
states (``beam_select``, ``beam_reorder``).

They run on CUDA tensors through the C ABI (fhe_ssm_scan and the others in
include/fhe_b200.h), on the current stream of the tensors' device, and can be
captured into CUDA graphs; all but the steps and the beams have
gradients (to capture a backward pass, hold no eager autograd graph of the same
leaves: torch would make the capture wait for that graph's stream, and refuses).
Second and forward-mode derivatives are refused.
Activations are float32, bfloat16 or float16; gates, states, norm weights and
scores are float32.  Arguments that do not fit raise ValueError before any GPU
work.
"""
from __future__ import annotations

import ctypes
from array import array
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import call

_TYPES = {torch.float32: _lib.FHE_F32, torch.bfloat16: _lib.FHE_BF16, torch.float16: _lib.FHE_F16}
MAX_HEAD_DIM, MAX_STATE, MAX_TAPS, MAX_TOP, MAX_NORM_WIDTH = 128, 256, 8, 64, 16384
MAX_BEAMS = 64
_LARGEST = torch.finfo(torch.float32).max


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
    """Whether a backward pass may ask for gradients of these.  Tensors with a forward-mode derivative are refused:
    the outputs would have none."""
    if getattr(forward_ad, "_current_level", 0) >= 0:  # outside a dual level no tensor has one
        _need(all(t is None or forward_ad.unpack_dual(t).tangent is None for t in tensors),
              "the operators have no forward-mode derivatives")
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


# ---- norms --------------------------------------------------------------------------------------


def _rows(t):
    """t as [rows, width] with a contiguous innermost axis (a view where its strides allow one)."""
    return _inner(t if t.dim() == 2 else t.reshape(-1, t.shape[-1]))


def _check_norm(op, x, weight, eps, others, dtype, groups=1, scale=1.0):
    _need(x.dim() >= 1 and x.shape[-1] >= 1, f"{op}: x must be [..., width]")
    _need(x.dtype in _TYPES, f"{op}: x must be float32, bfloat16 or float16")
    width = x.shape[-1]
    _need(isinstance(groups, int) and groups >= 1 and width % groups == 0,
          f"{op}: width ({width}) must be a multiple of groups ({groups})")
    _need(width // groups <= MAX_NORM_WIDTH, f"{op}: at most {MAX_NORM_WIDTH} channels are normalised together")
    _check(op, "weight", weight, (width,), torch.float32)
    for name, t, types in others:
        _need(t.shape == x.shape, f"{op}: {name} must have shape {tuple(x.shape)}, got {tuple(t.shape)}")
        _need(t.dtype in types, f"{op}: {name} must be {' or '.join(str(v) for v in types)}, got {t.dtype}")
    _need(dtype == x.dtype or (x.dtype == torch.float32 and dtype in _TYPES),
          f"{op}: dtype must be x's, or a smaller one of a float32 x")
    _need(0 < eps <= _LARGEST, f"{op}: eps must be positive")
    if torch.is_tensor(scale):
        _check(op, "scale", scale, (width,), torch.float32)
    else:
        _need(abs(scale) <= _LARGEST, f"{op}: scale must be finite")
    _check_devices(op, x, weight, scale if torch.is_tensor(scale) else None, *(t for _, t, _ in others))


def _first_derivatives(backward):
    """``once_differentiable`` where a graph of the backward pass is asked for, else the function as it is."""
    guarded = once_differentiable(backward)

    def call_backward(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return call_backward


_norm_block, _norm_grad_block = _lib.packer(_lib.RmsNormArgs), _lib.packer(_lib.RmsNormGradArgs)


def _at(t):
    return 0 if t is None else t.data_ptr()


def _new(t, dtype):
    """An uninitialised contiguous tensor of t's shape."""
    if t.is_contiguous():
        return torch.empty_like(t) if t.dtype == dtype else torch.empty_like(t, dtype=dtype)
    return torch.empty(t.shape, dtype=dtype, device=t.device)


def _spaced(t):
    """t, or evenly spaced rows of it, and the distance between rows (None: None, 0)."""
    if t is None:
        return None, 0
    if t.is_contiguous():
        return t, t.shape[-1]
    t = _rows(t)
    return t, t.stride(0)


def _norm_values(like, stream, dtype, groups, eps, scale, x, residual, gate, channel_scale, weight, y, h, rstd):
    """The argument block's values; what is made here is to be kept until the call."""
    (x, xs), (residual, rs), (gate, gs) = _spaced(x), _spaced(residual), _spaced(gate)
    width, device = like.shape[-1], like.get_device()
    return (device, _TYPES[dtype], _TYPES[stream], like.numel() // width, width, groups, eps, scale, _at(x), xs,
            _at(residual), rs, _at(gate), gs, _at(channel_scale), weight.data_ptr(), _at(y), _at(h), _at(rstd),
            _stream_of(device)), (x, residual, gate)


def _run_norm(x, residual, gate, weight, channel_scale, eps, scale, groups, dtype, grad):
    y = _new(x, dtype)
    h = None if residual is None else _new(x, residual.dtype)
    stream = x.dtype if residual is None else residual.dtype
    rstd = torch.empty((x.numel() // x.shape[-1], groups), dtype=torch.float32, device=x.device) if grad else None
    values, kept = _norm_values(x, stream, dtype, groups, eps, scale, x, residual, gate, channel_scale, weight, y, h, rstd)
    call("fhe_rms_norm", _norm_block(*values))
    return y, h, rstd


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gate, weight, channel_scale, eps, scale, groups, dtype):
        y, h, rstd = _run_norm(x, residual, gate, weight, channel_scale, eps, scale, groups, dtype, True)
        ctx.set_materialize_grads(False)
        ctx.rest = eps, scale, groups, dtype, x.dtype
        ctx.save_for_backward(x if residual is None or channel_scale is not None else None, gate, weight,
                              channel_scale, h, rstd)
        return y if h is None else (y, h)

    @staticmethod
    @_first_derivatives
    def backward(ctx, dy, dh=None):
        x, gate, weight, channel_scale, h, rstd = ctx.saved_tensors
        eps, scale, groups, dtype, x_dtype = ctx.rest
        like, wants = x if h is None else h, ctx.needs_input_grad
        stream = like.dtype
        dy = torch.zeros(like.shape, dtype=dtype, device=like.device) if dy is None else dy.contiguous()
        dh = None if dh is None else dh.contiguous()
        # a branch added as it is has the stream's own gradient
        shared = h is not None and channel_scale is None and scale == 1.0 and x_dtype == stream
        dres = _new(like, stream) if h is not None and (wants[1] or (shared and wants[0])) else None
        dx = _new(like, x_dtype) if wants[0] and not shared else None
        dgate = _new(like, dtype) if gate is not None and wants[2] else None
        dw = torch.empty_like(weight) if wants[3] else None
        dcs = torch.empty_like(weight) if channel_scale is not None and wants[4] else None
        f, kept = _norm_values(like, stream, dtype, groups, eps, scale, x, h, gate, channel_scale, weight, None, h, rstd)
        outs = tuple(map(_at, (dy, dh, dx, dres, dgate, dw, dcs)))
        if dw is not None or dcs is not None:
            ws = _space("fhe_rms_norm_backward_workspace", _norm_grad_block(*f, *outs, 0, 0, 0), like.device)
            outs += ws.data_ptr(), ws.numel()
        else:
            outs += 0, 0
        call("fhe_rms_norm_backward", _norm_grad_block(*f, *outs, f[-1]))
        return dres if shared else dx, dres if wants[1] else None, dgate, dw, dcs, None, None, None, None


def _space(name, block, device):
    """The workspace that a packed argument block asks for."""
    n = ctypes.c_uint64()
    call(name, block, ctypes.byref(n))
    return torch.empty(n.value, dtype=torch.uint8, device=device)


def _norm_fits(x, weight, eps, dtype):
    """Whether the arguments that all norms share pass ``_check_norm``."""
    t, w = x.dtype, x.shape[-1] if x.dim() else 0
    return (x.is_cuda and t in _TYPES and 1 <= w <= MAX_NORM_WIDTH and weight.shape == (w,)
            and weight.dtype == torch.float32 and weight.get_device() == x.get_device() and 0 < eps <= _LARGEST
            and (dtype == t or (t == torch.float32 and dtype in _TYPES)))


def rms_norm(x, weight, eps=1e-5, dtype=None):
    """x / sqrt(mean(x^2) + eps) weight over the last axis.

    x [..., width] float32, bfloat16 or float16, width at most 16384; weight
    [width] float32.  The result has x's type, or the 16-bit `dtype` if x is
    float32.  Only the last axis must be contiguous and the others evenly spaced
    (a slice of wider rows will do), else x is copied.  Sums are float32; rows
    whose squares pass its range are scaled.  Gradients reach x and weight."""
    dtype = dtype or x.dtype
    if not _norm_fits(x, weight, eps, dtype):
        _check_norm("rms_norm", x, weight, eps, (), dtype)
    args = (x, None, None, _dense(weight), None, float(eps), 1.0, 1, dtype)
    if _wants_grad(x, weight):
        return _RmsNorm.apply(*args)
    return _run_norm(*args, False)[0]


def add_rms_norm(residual, x, weight, eps=1e-5, scale=1.0):
    """A residual stream's next value and its norm: h = residual + scale x, kept
    in residual's type, and y = h / sqrt(mean(h^2) + eps) weight in x's type, the
    norm of h as it is kept.

    residual [..., width] of x's type or float32; x and weight as in ``rms_norm``;
    scale a number, or [width] float32 for a factor of each channel.  Returns
    (y, h).  Gradients reach every tensor."""
    op = "add_rms_norm"
    t, r = x.dtype, residual.dtype
    channel_scale, factor = (_dense(scale), 1.0) if isinstance(scale, torch.Tensor) else (None, scale)
    if not (_norm_fits(x, weight, eps, t) and residual.shape == x.shape and (r == t or r == torch.float32)
            and residual.get_device() == x.get_device() and -_LARGEST <= factor <= _LARGEST
            and (channel_scale is None or (channel_scale.shape == weight.shape and channel_scale.dtype == torch.float32
                                           and channel_scale.get_device() == x.get_device()))):
        _check_norm(op, x, weight, eps, (("residual", residual, (t, torch.float32)),), t, scale=scale)
    args = (x, residual, None, _dense(weight), channel_scale, float(eps), float(factor), 1, x.dtype)
    if _wants_grad(x, residual, weight, channel_scale):
        return _RmsNorm.apply(*args)
    return _run_norm(*args, False)[:2]


def gated_rms_norm(x, gate, weight, eps=1e-5, groups=1):
    """The norm behind the recurrence: u = x SiLU(gate), then u / sqrt(mean(u^2) +
    eps) weight with the mean over each of `groups` equal parts of the last axis.

    x and gate [..., width] of one type, gate usually a slice of the layer's wider
    projection; weight [width] float32; a part has at most 16384 channels.
    Products x SiLU(gate) must fit float32.  Gradients reach every tensor."""
    if not (groups == 1 and _norm_fits(x, weight, eps, x.dtype) and gate.shape == x.shape and gate.dtype == x.dtype
            and gate.get_device() == x.get_device()):
        _check_norm("gated_rms_norm", x, weight, eps, (("gate", gate, (x.dtype,)),), x.dtype, groups)
    args = (x, None, gate, _dense(weight), None, float(eps), 1.0, groups, x.dtype)
    if _wants_grad(x, gate, weight):
        return _RmsNorm.apply(*args)
    return _run_norm(*args, False)[0]


# ---- embedding ----------------------------------------------------------------------------------


_embedding_block, _embedding_grad_block = _lib.packer(_lib.EmbeddingArgs), _lib.packer(_lib.EmbeddingGradArgs)


def _embedding_values(tokens, weight, scale, dtype, out):
    device = weight.get_device()
    return (device, _TYPES[weight.dtype], _TYPES[dtype], tokens.dtype == torch.int64, tokens.numel(), *weight.shape, scale,
            tokens.data_ptr(), weight.data_ptr(), weight.stride(0), _at(out), _stream_of(device))


def _run_embedding(tokens, weight, scale, dtype):
    out = torch.empty((*tokens.shape, weight.shape[1]), dtype=dtype, device=weight.device)
    call("fhe_embedding", _embedding_block(*_embedding_values(tokens, weight, scale, dtype, out)))
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, scale, dtype):
        ctx.rest = scale, dtype, weight.shape, weight.dtype
        ctx.save_for_backward(tokens)  # the table may change before the backward pass
        return _run_embedding(tokens, weight, scale, dtype)

    @staticmethod
    @_first_derivatives
    def backward(ctx, dout):
        tokens, = ctx.saved_tensors
        scale, dtype, shape, weight_dtype = ctx.rest
        dout, dw = dout.contiguous(), torch.empty(shape, dtype=weight_dtype, device=tokens.device)
        f = _embedding_values(tokens, dw, scale, dtype, None)
        outs = dout.data_ptr(), dw.data_ptr()
        ws = _space("fhe_embedding_backward_workspace", _embedding_grad_block(*f, *outs, 0, 0, 0), dw.device)
        call("fhe_embedding_backward", _embedding_grad_block(*f, *outs, ws.data_ptr(), ws.numel(), f[-1]))
        return dw, None, None, None


def embedding(tokens, weight, scale=1.0, dtype=None):
    """scale weight[tokens], rounded once.

    tokens [...] int64 or int32, negative for a position without a token (0, no
    gradient); a token past the vocabulary gives NaN and has no gradient.
    weight [vocab, width] float32, bfloat16 or float16; the result [..., width]
    has its type, or `dtype` float32.  The gradient is that of every row of
    weight, summed in float32 over the row's positions in their order."""
    op, dtype = "embedding", dtype or weight.dtype
    _need(tokens.dtype in (torch.int64, torch.int32), f"{op}: tokens must be int64 or int32, got {tokens.dtype}")
    _need(weight.dim() == 2 and weight.dtype in _TYPES and weight.shape[1] >= 1,
          f"{op}: weight must be [vocab, width] float32, bfloat16 or float16")
    _need(weight.shape[1] <= 1 << 20, f"{op}: width must be at most 2^20")
    _need(dtype in (weight.dtype, torch.float32), f"{op}: dtype must be weight's or float32")
    _need(abs(scale) <= _LARGEST, f"{op}: scale must be finite")
    _check_devices(op, weight, tokens)
    tokens, rows = _dense(tokens), _inner(weight)
    if _wants_grad(weight):
        return _Embedding.apply(rows, tokens, float(scale), dtype)
    return _run_embedding(tokens, rows, float(scale), dtype)


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


# ---- beam search --------------------------------------------------------------------------------


class BeamStep(NamedTuple):
    scores: torch.Tensor    # [batch, width] float32
    parents: torch.Tensor   # [batch, width] int64, beams
    tokens: torch.Tensor    # [batch, width] int64
    finished: torch.Tensor  # [batch, width] bool


def beam_select(logits, scores, finished=None, eos=None, width=None, keep_slots=False):
    """One step of beam search: for each batch item the `width` (default: the
    number of beams; at most 64) best of scores_i + log softmax(logits_i)_v over
    its beams i and tokens v, best first, the lower beam and then the lower token
    first among equals.

    logits [batch * beams, vocab] or [batch, beams, vocab] float32, bfloat16 or
    float16; scores [batch, beams] float32, -inf for a beam that does not count
    (all but the first of equal ones at the start); beams at most 64.  A beam of
    `finished` [batch, beams] bool goes on as it is, with the token `eos`.  Beams
    whose score is not finite or whose logits hold a NaN or +inf offer nothing:
    candidates of score -inf fill up what possible ones leave.  With keep_slots
    (width = beams) a beam's best child keeps its beam's place and the others
    take the free places in order, so that few states have to move.

    Returns a ``BeamStep``: scores, parents (beams), tokens, and which beams have
    ended.  Totals are compared in 64 bits where 32 do not tell them apart."""
    op = "beam_select"
    if not _select_fits(logits, scores, finished, eos, width, keep_slots):
        _check_select(op, logits, scores, finished, eos, width, keep_slots)
    if _wants_grad(logits, scores):
        _need(False, f"{op} has no gradient")
    (rows, stride), scores, finished = _spaced(logits), _dense(scores), _dense(finished)
    (b, k), v, device = scores.shape, logits.shape[-1], logits.get_device()
    width = k if width is None else width
    out = torch.empty((b, width), dtype=torch.float32, device=logits.device)
    parents = torch.empty_like(out, dtype=torch.int64)
    tokens, ended = torch.empty_like(parents), torch.empty_like(out, dtype=torch.bool)
    call("fhe_beam_select", _select_block(
        device, _TYPES[logits.dtype], b, k, v, width, bool(keep_slots), 0, rows.data_ptr(), stride, scores.data_ptr(),
        _at(finished), -1 if eos is None else int(eos), out.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
        ended.data_ptr(), _stream_of(device)))
    return BeamStep(out, parents, tokens, ended)


_select_block = _lib.packer(_lib.BeamSelectArgs)


def _select_fits(logits, scores, finished, eos, width, keep):
    """Whether the arguments pass every test of ``_check_select``."""
    if scores.dim() != 2 or logits.dim() not in (2, 3):
        return False
    (b, k), v, d = scores.shape, logits.shape[-1], logits.get_device()
    w = k if width is None else width
    return (1 <= k <= MAX_BEAMS and v >= 1 and (logits.shape[0] == b * k if logits.dim() == 2 else logits.shape[:2] == (b, k))
            and logits.is_cuda and logits.dtype in _TYPES and scores.dtype == torch.float32 and scores.get_device() == d
            and 1 <= w <= min(MAX_BEAMS, k * v) and (eos is None or 0 <= eos < v) and (not keep or w == k)
            and (finished is None or (eos is not None and finished.shape == (b, k) and finished.dtype == torch.bool
                                      and finished.get_device() == d)))


def _check_select(op, logits, scores, finished, eos, width, keep_slots):
    _need(scores.dim() == 2 and 1 <= scores.shape[1] <= MAX_BEAMS, f"{op}: scores must be [batch, 1 to {MAX_BEAMS} beams]")
    _need(scores.dtype == torch.float32, f"{op}: scores must be {torch.float32}, got {scores.dtype}")
    b, k = scores.shape
    _need(logits.dtype in _TYPES, f"{op}: logits must be float32, bfloat16 or float16")
    _need(logits.dim() in (2, 3) and logits.shape[:-1] in ((b * k,), (b, k)) and logits.shape[-1] >= 1,
          f"{op}: logits must be [batch * beams, vocab] or [batch, beams, vocab]")
    v, width = logits.shape[-1], k if width is None else width
    _need(1 <= width <= min(MAX_BEAMS, k * v), f"{op}: width must be in [1, {min(MAX_BEAMS, k * v)}]")
    _need(eos is None or 0 <= eos < v, f"{op}: eos must be a token")
    if finished is not None:
        _check(op, "finished", finished, (b, k), torch.bool)
        _need(eos is not None, f"{op}: finished beams need an eos")
    _need(not keep_slots or width == k, f"{op}: keep_slots needs a width of the number of beams")
    _check_devices(op, logits, scores, finished)


def beam_reorder(states, parents):
    """Moves the states of beams in place: row i of each batch item becomes what
    its row parents[:, i] was, in every tensor of `states`.

    parents [batch, beams] int64 (at most 64 beams); a parent outside the beams
    leaves its row.  states: contiguous tensors [batch * beams, ...] or [batch,
    beams, ...] of any types, no two of them on the same memory.  Rows that
    keep their place are neither read nor written."""
    op = "beam_reorder"
    _need(parents.dim() == 2 and 1 <= parents.shape[1] <= MAX_BEAMS, f"{op}: parents must be [batch, 1 to {MAX_BEAMS} beams]")
    _need(parents.dtype == torch.int64, f"{op}: parents must be {torch.int64}, got {parents.dtype}")
    (b, k), device = parents.shape, parents.get_device()
    _need(b <= 65535, f"{op}: batch must be at most 65535")
    rows, states = b * k, list(states)
    if not (device >= 0 and all([t.is_contiguous() and t.get_device() == device and t.dim() and t.size(0) == rows
                                 for t in states])):
        for t in states:
            _need(t.dim() >= 1 and (t.shape[0] == rows or t.shape[:2] == (b, k)),
                  f"{op}: states must be [batch * beams, ...] or [batch, beams, ...], got {tuple(t.shape)}")
            _need(t.is_contiguous(), f"{op}: states must be contiguous")
        _check_devices(op, parents, *states)
    parents = _dense(parents)  # a broadcast one spans more than it holds
    at, sizes = [t.data_ptr() for t in states], [t.nbytes for t in states]
    end = 0
    for p, n in sorted(zip([*at, parents.data_ptr()], [*sizes, parents.nbytes])):
        if p < end and n:
            _need(False, f"{op}: states share memory")
        end = p + n if n else end
    if _wants_grad(*states):
        _need(False, f"{op} has no gradient")
    if not rows:
        return
    at, sizes = array("Q", at), array("Q", [n // rows for n in sizes])
    call("fhe_beam_reorder", _reorder_block(device, b, k, len(states), at.buffer_info()[0], sizes.buffer_info()[0],
                                            parents.data_ptr(), _stream_of(device)))
    increment_version(states)


_reorder_block = _lib.packer(_lib.BeamReorderArgs)
