"""Refused arguments of the operators around the layers (norms, embedding,
beams), of the Python functions and of the C entry points: none of them reaches
a GPU."""
import ctypes

import pytest
import torch

from fhe_mamba_b200 import _lib, mamba_ops as ops

F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64
z = torch.zeros


@pytest.mark.parametrize("args, message", [
    ((z(()), z(1)), "width"),
    ((z(2, 0), z(0)), "width"),
    ((z(2, 4, dtype=F64), z(4)), "float32, bfloat16 or float16"),
    ((z(2, 4), z(5)), "weight must have shape"),
    ((z(2, 4), z(4, dtype=BF16)), "weight must be"),
    ((z(1, 16385), z(16385)), "at most 16384"),
    ((z(2, 4), z(4), 0.0), "eps"),
    ((z(2, 4), z(4), float("nan")), "eps"),
    ((z(2, 4), z(4), 1e39), "eps"),
    ((z(2, 4), z(4), 1e-5, F64), "dtype"),
    ((z(2, 4, dtype=BF16), z(4), 1e-5, F32), "dtype"),
    ((z(2, 4), z(4)), "CUDA tensors expected"),
])
def test_norm_refusals(args, message):
    with pytest.raises(ValueError, match=message):
        ops.rms_norm(*args)


@pytest.mark.parametrize("args, message", [
    ((z(2, 5), z(2, 4), z(4)), "residual must have shape"),
    ((z(4), z(2, 4), z(4)), "residual must have shape"),
    ((z(2, 4, dtype=F16), z(2, 4, dtype=BF16), z(4)), "residual must be"),
    ((z(2, 4, dtype=F16), z(2, 4), z(4)), "residual must be"),
    ((z(2, 4), z(2, 4), z(4), 1e-5, z(5)), "scale must have shape"),
    ((z(2, 4), z(2, 4), z(4), 1e-5, z(())), "scale must have shape"),
    ((z(2, 4), z(2, 4), z(4), 1e-5, z(4, dtype=BF16)), "scale must be"),
    ((z(2, 4), z(2, 4), z(4), 1e-5, float("inf")), "scale must be finite"),
    ((z(2, 4), z(2, 4), z(4), 1e-5, -1e39), "scale must be finite"),
    ((z(2, 4), z(2, 4), z(4)), "CUDA tensors expected"),
])
def test_add_norm_refusals(args, message):
    with pytest.raises(ValueError, match=message):
        ops.add_rms_norm(*args)


@pytest.mark.parametrize("args, message", [
    ((z(2, 4), z(2, 5), z(4)), "gate must have shape"),
    ((z(2, 4), z(2, 4, dtype=BF16), z(4)), "gate must be"),
    ((z(2, 4), z(2, 4), z(4), 1e-5, 3), "multiple of groups"),
    ((z(2, 4), z(2, 4), z(4), 1e-5, 0), "multiple of groups"),
    ((z(1, 32770), z(1, 32770), z(32770), 1e-5, 2), "at most 16384"),
    ((z(2, 4), z(2, 4), z(4)), "CUDA tensors expected"),
])
def test_gated_norm_refusals(args, message):
    with pytest.raises(ValueError, match=message):
        ops.gated_rms_norm(*args)


def norm_struct(**kw):
    """A C argument block whose pointers are never followed: each call below is refused before."""
    s = dict(dtype=0, stream_dtype=0, rows=2, width=8, groups=1, eps=1e-5, scale=1.0, x=256, weight=256, y=256)
    s.update(kw)
    return _lib.RmsNormArgs(**s)


@pytest.mark.parametrize("kw, message", [
    (dict(dtype=7), "dtype"), (dict(dtype=1, stream_dtype=2), "stream_dtype"), (dict(gate=256, residual=256), "not both"),
    (dict(gate=256, groups=3), "multiple of groups"), (dict(gate=256, groups=0), "multiple of groups"),
    (dict(width=0), "multiple of groups"), (dict(groups=2), "groups need a gate"), (dict(width=16385), "16384"),
    (dict(eps=0.0), "eps"), (dict(channel_scale=256), "channel_scale needs"), (dict(scale=float("inf")), "scale"),
    (dict(rows=1 << 31), "too large"), (dict(gate=256, width=1 << 16, groups=1 << 16), "too large"),
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(weight=None), "null"), (dict(residual=256), "null"),
])
def test_norm_c_refusals(kw, message):
    lib = _lib.load()
    assert lib.fhe_rms_norm(ctypes.byref(norm_struct(**kw))) == _lib.FHE_ERR_INVALID
    assert message in _lib.last_error()


def test_norm_backward_c_refusals():
    lib = _lib.load()
    n = ctypes.c_uint64()

    def refused(message, f, **kw):
        g = _lib.RmsNormGradArgs(f=f, **kw)
        assert lib.fhe_rms_norm_backward(ctypes.byref(g)) == _lib.FHE_ERR_INVALID and message in _lib.last_error()
        return g
    refused("null", norm_struct(), dy=256, dx=256)
    refused("null", norm_struct(rstd=256), dx=256)
    refused("null", norm_struct(rstd=256, residual=256), dy=256, dx=256)
    refused("null", norm_struct(rstd=256, residual=256, h=256, channel_scale=256, x=None), dy=256, dx=256)
    refused("dgate", norm_struct(rstd=256), dy=256, dgate=256)
    refused("residual", norm_struct(rstd=256), dy=256, dresidual=256)
    refused("residual", norm_struct(rstd=256), dy=256, dh=256)
    refused("channel_scale", norm_struct(rstd=256), dy=256, dchannel_scale=256)
    g = refused("workspace too small", norm_struct(rstd=256), dy=256, dweight=256)
    assert lib.fhe_rms_norm_backward_workspace(ctypes.byref(g), ctypes.byref(n)) == 0 and n.value >= 32
    refused("aligned", norm_struct(rstd=256), dy=256, dweight=256, workspace=257, workspace_bytes=1 << 30)
    for name in ("fhe_rms_norm", "fhe_rms_norm_backward", "fhe_rms_norm_backward_workspace"):
        args = (None,) if name != "fhe_rms_norm_backward_workspace" else (None, None)
        assert getattr(lib, name)(*args) == _lib.FHE_ERR_INVALID and "null" in _lib.last_error()


I64 = torch.int64


@pytest.mark.parametrize("args, message", [
    ((z(3), z(5, 4)), "tokens must be"),
    ((z(3, dtype=torch.int16), z(5, 4)), "tokens must be"),
    ((z(3, dtype=I64), z(5)), "weight must be"),
    ((z(3, dtype=I64), z(5, 0)), "weight must be"),
    ((z(3, dtype=I64), z(5, 4, dtype=F64)), "weight must be"),
    ((z(3, dtype=I64), z(1, (1 << 20) + 1)), "width"),
    ((z(3, dtype=I64), z(5, 4), 1.0, BF16), "dtype"),
    ((z(3, dtype=I64), z(5, 4, dtype=F16), 1.0, BF16), "dtype"),
    ((z(3, dtype=I64), z(5, 4), float("nan")), "scale"),
    ((z(3, dtype=I64), z(5, 4), 1e39), "scale"),
    ((z(3, dtype=I64), z(5, 4)), "CUDA tensors expected"),
])
def test_embedding_refusals(args, message):
    with pytest.raises(ValueError, match=message):
        ops.embedding(*args)


@pytest.mark.parametrize("kw, message", [
    (dict(dtype=9), "dtype"), (dict(dtype=1, out_dtype=2), "out_dtype"), (dict(count=1 << 31), "2^31"),
    (dict(vocab=1 << 31), "2^31"), (dict(width=0), "width"), (dict(width=(1 << 20) + 1), "width"),
    (dict(scale=float("inf")), "scale"), (dict(ids=None), "null"), (dict(table=None), "null"), (dict(out=None), "null"),
])
def test_embedding_c_refusals(kw, message):
    lib = _lib.load()
    base = dict(dtype=0, out_dtype=0, count=4, vocab=5, width=8, scale=1.0, ids=256, table=256, table_stride=8, out=256)
    a = _lib.EmbeddingArgs(**{**base, **kw})
    assert lib.fhe_embedding(ctypes.byref(a)) == _lib.FHE_ERR_INVALID and message in _lib.last_error()


def test_embedding_backward_c_refusals():
    lib = _lib.load()
    f = _lib.EmbeddingArgs(dtype=0, out_dtype=0, count=4, vocab=5, width=8, scale=1.0, ids=256)
    for kw, message in ((dict(dtable=256), "null input"), (dict(dout=256), "null output"),
                        (dict(dout=256, dtable=256), "workspace too small"),
                        (dict(dout=256, dtable=256, workspace=257, workspace_bytes=1 << 30), "aligned")):
        g = _lib.EmbeddingGradArgs(f=f, **kw)
        assert lib.fhe_embedding_backward(ctypes.byref(g)) == _lib.FHE_ERR_INVALID and message in _lib.last_error()
    n = ctypes.c_uint64()
    assert lib.fhe_embedding_backward_workspace(ctypes.byref(g), ctypes.byref(n)) == 0 and n.value >= 32
    assert lib.fhe_embedding(None) == lib.fhe_embedding_backward(None) == _lib.FHE_ERR_INVALID


def select_args(**kw):
    return {**dict(logits=z(6, 9), scores=z(2, 3)), **kw}


@pytest.mark.parametrize("kw, message", [
    (dict(scores=z(6)), "scores must be"), (dict(scores=z(2, 65)), "scores must be"), (dict(scores=z(2, 0)), "scores must be"),
    (dict(scores=z(2, 3, dtype=F64)), "scores must be"), (dict(logits=z(6, 9, dtype=F64)), "logits must be float32"),
    (dict(logits=z(5, 9)), "logits must be"), (dict(logits=z(3, 2, 9)), "logits must be"), (dict(logits=z(6)), "logits must be"),
    (dict(logits=z(6, 0)), "logits must be"), (dict(width=0), "width"), (dict(width=28), "width"),
    (dict(logits=z(6, 99), width=65), "width"), (dict(eos=9), "eos must be a token"), (dict(eos=-1), "eos must be a token"),
    (dict(finished=z(2, 3, dtype=torch.bool)), "need an eos"), (dict(finished=z(2, 3), eos=0), "finished must be"),
    (dict(finished=z(6, dtype=torch.bool), eos=0), "finished must have shape"), (dict(keep_slots=True, width=2), "keep_slots"),
    ({}, "CUDA tensors expected"),
])
def test_select_refusals(kw, message):
    with pytest.raises(ValueError, match=message):
        ops.beam_select(**select_args(**kw))


@pytest.mark.parametrize("states, parents, message", [
    ([z(6, 4)], z(6, dtype=I64), "parents must be"), ([z(6, 4)], z(2, 65, dtype=I64), "parents must be"),
    ([z(6, 4)], z(2, 3, dtype=torch.int32), "parents must be"), ([z(5, 4)], z(2, 3, dtype=I64), "states must be"),
    ([z(3, 2, 4)], z(2, 3, dtype=I64), "states must be"), ([z(())], z(2, 3, dtype=I64), "states must be"),
    ([z(4, 6).t()], z(2, 3, dtype=I64), "contiguous"), ([z(6, 4)], z(2, 3, dtype=I64), "CUDA tensors expected"),
    ([z(65536, 1)], z(65536, 1, dtype=I64), "batch"),
])
def test_reorder_refusals(states, parents, message):
    with pytest.raises(ValueError, match=message):
        ops.beam_reorder(states, parents)


def test_reorder_shared_memory(monkeypatch):
    """One tensor twice, a view beside its base, and the parents among the states are refused (no GPU is asked)."""
    monkeypatch.setattr(ops, "_check_devices", lambda *a: None)
    t, parents = z(6, 4), z(2, 3, dtype=I64)
    for states in ([t, t], [t, z(6, 4), t.view(2, 3, 4)], [t, t.view(-1)[6:12]], [parents]):
        with pytest.raises(ValueError, match="share memory"):
            ops.beam_reorder(states, parents)


def test_beam_c_refusals():
    lib = _lib.load()
    base = dict(dtype=0, batch=2, beams=3, vocab=9, width=3, logits=256, logits_stride=9, scores=256, eos=-1, out_scores=256,
                parents=256, tokens=256)
    for kw, message in ((dict(dtype=5), "dtype"), (dict(beams=0), "beams"), (dict(beams=65), "beams"), (dict(vocab=0), "vocab"),
                        (dict(width=0), "width"), (dict(width=65), "width"), (dict(width=28), "width"),
                        (dict(batch=1 << 24), "batch"), (dict(eos=9), "eos"), (dict(finished=256), "eos"),
                        (dict(keep_slots=1, width=2), "keep_slots"), (dict(logits=None), "null"), (dict(tokens=None), "null")):
        a = _lib.BeamSelectArgs(**{**base, **kw})
        assert lib.fhe_beam_select(ctypes.byref(a)) == _lib.FHE_ERR_INVALID and message in _lib.last_error(), kw
    one, size = (ctypes.c_void_p * 1)(None), (ctypes.c_uint64 * 1)(8)
    for kw, message in ((dict(beams=65), "beams"), (dict(beams=0), "beams"), (dict(batch=65536), "batch"),
                        (dict(states=None), "null"), (dict(parents=None), "null"), ({}, "null state")):
        a = _lib.BeamReorderArgs(**{**dict(batch=2, beams=3, count=1, states=one, row_bytes=size, parents=256), **kw})
        assert lib.fhe_beam_reorder(ctypes.byref(a)) == _lib.FHE_ERR_INVALID and message in _lib.last_error(), kw
    assert lib.fhe_beam_select(None) == lib.fhe_beam_reorder(None) == _lib.FHE_ERR_INVALID


def test_sizes_past_their_fields():
    pack = _lib.packer(_lib.RmsNormArgs)
    fields = [0, 0, 0, 2, 8, 1, 1e-5, 1.0] + [0] * 12
    assert pack(*fields) == bytes(_lib.RmsNormArgs(rows=2, width=8, groups=1, eps=1e-5, scale=1.0))
    for place, value in ((3, 1 << 32), (4, -1), (0, 1 << 31)):
        with pytest.raises(ValueError, match="RmsNormArgs: a size is out of range"):
            pack(*fields[:place], value, *fields[place + 1:])
