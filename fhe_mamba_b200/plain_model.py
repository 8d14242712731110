"""The plaintext Mamba-2 model over whole sequences on the GPU.

``Mamba2Model`` evaluates its layers token by token in float64 on the host, as
the reference for the encrypted loop.  ``PlainMamba2`` runs the same layers
with the exact nonlinearities (``exact_step``) over batches of sequences at
once: the in and out projections are library matrix products, everything else
the operators of ``mamba_ops``.  It scores long texts, prefills prompts of
different lengths, continues token by token from the carried states or by beam
search, and has gradients, so a model can be tuned before it is calibrated and
encrypted.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import mamba_ops as ops
from .mamba_ops import TokenLogprobs


def _operators_take(weight, eps):
    """Whether the norm operators take rows of this width with this eps."""
    f = torch.finfo(torch.float32)
    return weight.shape[0] <= ops.MAX_NORM_WIDTH and f.tiny <= eps <= f.max


def _rms(x, weight, eps):
    """The norm of float32 rows that the operators do not take."""
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight


class BeamTexts(NamedTuple):
    tokens: torch.Tensor   # [batch, beams, length] int64, best first; `eos` behind an end
    scores: torch.Tensor   # [batch, beams] float32, sums of log-probabilities
    lengths: torch.Tensor  # [batch, beams] int64, an end included


class PlainMamba2(torch.nn.Module):
    """`model`'s layers as parameters in `dtype` (activations and matrices; the
    norms, gates and states stay float32) on `device`.  The embedding is tied:
    it also gives the logits.  A negative input token counts from the
    vocabulary's end; past the vocabulary NaN comes out, before it the
    embedding is 0."""

    GATES = ("norm_w", "gn_w", "dt_bias", "a", "d")  # float32 whatever the dtype

    def __init__(self, model, device="cuda", dtype=torch.float32):
        super().__init__()
        if dtype not in ops._TYPES:
            raise ValueError("dtype must be float32, bfloat16 or float16")
        self.weights, self.dtype = model.layers, dtype
        put = lambda v, t: torch.nn.Parameter(torch.as_tensor(v).to(device=device, dtype=t))  # noqa: E731
        self.embedding = put(model.embedding, dtype)
        self.norm_f = put(model.norm_f, torch.float32)
        self.layers = torch.nn.ModuleList(
            torch.nn.ParameterDict({k: put(v, torch.float32 if k in self.GATES else dtype)
                                    for k, v in W.arrays.items()}) for W in model.layers)

    def initial_state(self, batch: int):
        """Zero (convolution window, recurrent state) of every layer."""
        d = self.embedding.device
        return [(torch.zeros(batch, W.conv_kernel - 1, W.conv_dim, dtype=self.dtype, device=d),
                 torch.zeros(batch, W.heads, W.head_dim, W.d_state, device=d)) for W in self.weights]

    def _norm(self, h, branch, weight, eps):
        """The norm of the residual stream with the last layer's output added (None: as it is), and that stream."""
        if not _operators_take(weight, eps):
            h = h if branch is None else h + branch.float()
            return _rms(h, weight, eps).to(self.dtype), h
        if branch is None:
            return ops.rms_norm(h, weight, eps, self.dtype), h
        return ops.add_rms_norm(h, branch, weight, eps)

    def _project(self, W, p, u):
        z, xbc, dt = (u @ p["w_in"].T).split([W.d_inner, W.conv_dim, W.heads], -1)
        write = torch.nn.functional.softplus(dt.float() + p["dt_bias"])
        return z, xbc, write, p["a"] * write

    def _parts(self, W, xa):
        x, B, C = xa.split([W.d_inner, W.d_state, W.d_state], -1)
        return x.unflatten(-1, (W.heads, W.head_dim)), B.unsqueeze(-2), C.unsqueeze(-2)

    def _finish(self, W, p, y, z):
        y, w = y.flatten(-2), p["gn_w"]
        if _operators_take(w, W.eps):
            return ops.gated_rms_norm(y, z, w, W.eps) @ p["w_out"].T
        return _rms(y.float() * torch.nn.functional.silu(z.float()), w, W.eps).to(self.dtype) @ p["w_out"].T

    def _embed(self, tokens):
        tokens = tokens.to(self.embedding.device)
        tokens = torch.add(tokens, tokens < 0, alpha=self.embedding.shape[0])  # an index from the end, as any tensor's
        return ops.embedding(tokens, self.embedding, dtype=torch.float32)

    def forward(self, tokens, state=None, lengths=None):
        """The normalised final hidden vectors [batch, length, d_model] of the
        token rows [batch, length] and the carried state behind each row's
        length (`lengths` int32 [batch], full rows if None)."""
        if tokens.dim() != 2:
            raise ValueError("tokens must be [batch, length]")
        state = state if state is not None else self.initial_state(tokens.shape[0])
        h, branch, new = self._embed(tokens), None, []
        for W, p, (window, s) in zip(self.weights, self.layers, state):
            u, h = self._norm(h, branch, p["norm_w"], W.eps)
            z, xbc, write, log_decay = self._project(W, p, u)
            xa, window = ops.causal_conv(xbc, p["conv_w"], p["conv_b"], initial_state=window, lengths=lengths)
            x, B, C = self._parts(W, xa)
            y, s = ops.ssm_scan(x, write, log_decay, B, C, D=p["d"], initial_state=s, lengths=lengths)
            branch = self._finish(W, p, y, z)
            new.append((window, s))
        return self._norm(h, branch, self.norm_f, self.weights[0].eps)[0], new

    @torch.no_grad()
    def step(self, tokens, state):
        """One token of each sequence ([batch]): its hidden vectors [batch,
        d_model].  `state` moves on in place."""
        h, branch = self._embed(tokens), None
        for W, p, (window, s) in zip(self.weights, self.layers, state):
            u, h = self._norm(h, branch, p["norm_w"], W.eps)
            z, xbc, write, log_decay = self._project(W, p, u)
            xa, _ = ops.causal_conv_step(window, xbc, p["conv_w"], p["conv_b"])
            x, B, C = self._parts(W, xa)
            y, _ = ops.ssm_step(s, x, write, log_decay, B, C, D=p["d"])
            branch = self._finish(W, p, y, z)
        return self._norm(h, branch, self.norm_f, self.weights[0].eps)[0]

    @torch.no_grad()
    def beam_search(self, tokens, beams, length, eos=None, lengths=None, length_penalty=0.0):
        """The `beams` best continuations of each prompt [batch, at least 1] by at
        most `length` tokens (``BeamTexts``): beam search over the sums of
        log-probabilities, a text ending with `eos` if that is given, ordered by
        score / text length ** length_penalty.  `lengths` int32 [batch] are those
        of padded prompts, at least 1."""
        if tokens.dim() != 2 or tokens.shape[1] < 1:
            raise ValueError("tokens must be [batch, at least 1]")
        if not (1 <= beams <= min(ops.MAX_BEAMS, self.embedding.shape[0]) and length >= 1):
            raise ValueError(f"beams must be in [1, {min(ops.MAX_BEAMS, self.embedding.shape[0])}], length at least 1")
        if lengths is not None and lengths.numel() and int(lengths.min()) < 1:
            raise ValueError("every prompt needs a token")
        b, d = tokens.shape[0], self.embedding.device
        hidden, state = self(tokens, lengths=lengths)
        last = torch.full((b,), tokens.shape[1] - 1, device=d) if lengths is None else \
            lengths.long().clamp(max=tokens.shape[1]) - 1
        logits = self.logits(hidden[torch.arange(b, device=d), last])
        state = [tuple(v.repeat_interleave(beams, 0) for v in pair) for pair in state]
        texts = torch.zeros(b, beams, length, dtype=torch.int64, device=d)
        moved = [texts, *(v for pair in state for v in pair)]
        found = ops.beam_select(logits, torch.zeros(b, 1, device=d), eos=eos, width=beams)
        for i in range(length):
            if i:
                found = ops.beam_select(self.logits(self.step(found.tokens.flatten(), state)), found.scores,
                                        found.finished if eos is not None else None, eos, keep_slots=True)
                ops.beam_reorder(moved, found.parents)
            texts[:, :, i] = found.tokens
            if eos is not None and bool(found.finished.all()):
                texts[:, :, i + 1:] = eos
                break
        n = torch.full((b, beams), length, device=d)
        if eos is not None:
            n = torch.minimum(n, (texts != eos).cumprod(-1).sum(-1) + 1)
        order = torch.sort(found.scores / n ** length_penalty, dim=1, descending=True, stable=True)[1]
        return BeamTexts(texts.gather(1, order[..., None].expand_as(texts)), found.scores.gather(1, order),
                         n.gather(1, order))

    def logits(self, hidden):
        return hidden @ self.embedding.T

    def score(self, tokens, state=None, lengths=None, top_k=0):
        """Each row's tokens 1.. under the model, given the tokens before them:
        a ``TokenLogprobs`` of [batch, length - 1] scores (log-probability 0 at
        and past a row's length)."""
        if tokens.dim() != 2 or tokens.shape[1] < 1:
            raise ValueError("tokens must be [batch, at least 1]")
        b, l = tokens.shape
        hidden, _ = self(tokens, state, lengths)
        targets = tokens[:, 1:].long()
        if lengths is not None:
            targets = targets.masked_fill(torch.arange(1, l, device=tokens.device) >= lengths[:, None], -1)
        out = ops.token_logprobs(self.logits(hidden[:, :-1]).flatten(0, 1), targets.flatten(), top_k)
        return TokenLogprobs(*(v.unflatten(0, (b, l - 1)) for v in out))

    def loss(self, tokens, lengths=None):
        """Mean negative log-probability of the scored tokens, 0 if there are none."""
        scores = self.score(tokens, lengths=lengths)
        n = max(tokens.shape[0] * (tokens.shape[1] - 1), 1) if lengths is None else \
            (lengths.long().clamp(0, tokens.shape[1]) - 1).clamp(min=0).sum().clamp(min=1)
        return -scores.logprob.sum() / n


def client_scores(logits, tokens, top_k, device=0):
    """The client's view of its selections: for each row of host logits the
    log-probability of the selected token, the entropy and the top_k
    alternatives as (token, log-probability) pairs."""
    z = torch.as_tensor(logits, dtype=torch.float32).to(torch.device("cuda", device))
    t = torch.as_tensor(tokens, dtype=torch.int64).to(z.device)
    s = ops.token_logprobs(z, t, min(top_k, z.shape[1]))
    return [{"token": int(tok), "logprob": lp, "entropy": h, "alternatives": list(zip(ids, lps))}
            for tok, lp, h, ids, lps in zip(tokens, s.logprob.tolist(), s.entropy.tolist(), s.top_ids.tolist(),
                                            s.top_logprobs.tolist())]
