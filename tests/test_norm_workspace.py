"""The workspace of the norms' gradients is the same wherever the arrays lie, so that it may be asked for before they do."""
import ctypes

import pytest

from fhe_mamba_b200 import _lib


def asked(dtype, stream, rows, width, groups, mode, at):
    """Bytes for arrays at addresses and strides that are multiples of `at` elements (none is followed)."""
    p = 4096 + 4 * at
    f = dict(dtype=dtype, stream_dtype=stream, rows=rows, width=width, groups=groups, eps=1e-5, scale=1.0, x=p,
             x_stride=width + at, weight=p, rstd=4096)
    if mode in ("add", "scaled"):
        f.update(residual=p, residual_stride=width + at, h=p)
    if mode == "scaled":
        f.update(channel_scale=p)
    if mode == "gate":
        f.update(gate=p, gate_stride=width + at)
    g = _lib.RmsNormGradArgs(f=_lib.RmsNormArgs(**f), dy=p, dx=p, dweight=4096)
    n = ctypes.c_uint64()
    assert _lib.load().fhe_rms_norm_backward_workspace(ctypes.byref(g), ctypes.byref(n)) == 0, _lib.last_error()
    return n.value


@pytest.mark.parametrize("mode", ["plain", "add", "scaled", "gate"])
@pytest.mark.parametrize("rows, width, groups", [(1, 8, 1), (300, 768, 1), (32768, 1536, 1), (5000, 1536, 8), (2000, 2560, 1),
                                                 (4000, 1024, 1), (700, 16384, 1), (90, 1002, 1), (5000, 1001, 1), (10 ** 6, 64, 1)])
def test_workspace_does_not_hang_on_alignment(mode, rows, width, groups):
    if groups > 1 and mode != "gate":
        groups = 1
    for dtype, stream in ((0, 0), (1, 0), (1, 1)):
        if mode == "gate":
            stream = dtype
        sizes = {asked(dtype, stream, rows, width, groups, mode, at) for at in (16, 8, 4, 2, 1)}
        assert len(sizes) == 1 and sizes.pop() >= width * 4
