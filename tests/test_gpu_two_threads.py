"""Calls of different sizes from two host threads at once, each on its own stream.

The most dynamic shared memory that a kernel may have is state of the whole
process: a call that sets its own size must not take it from another call.  The
threads repeat C calls whose argument blocks are made before, so that the calls
meet often."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
ROUNDS = 60000


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.fixture(scope="module")
def ops():
    from fhe_mamba_b200 import mamba_ops
    return mamba_ops


def side_by_side(monkeypatch, ops, calls):
    """Repeats each call's C calls in a thread of its own and checks what they leave."""
    from fhe_mamba_b200 import _lib
    lib, made = _lib.load(), []
    real = _lib.call
    for f in calls:
        seen, stream = [], torch.cuda.Stream()

        def record(name, *args):
            real(name, *args)
            if not name.endswith("workspace"):
                seen.append((getattr(lib, name), args))
        with monkeypatch.context() as m, torch.cuda.stream(stream):
            m.setattr(ops, "call", record)
            outs = f()
        stream.synchronize()
        made.append((seen, outs, [t.clone() for t in outs[0]]))  # outs keeps the blocks' tensors
    codes, gate = [], threading.Barrier(len(calls))

    def work(seen):
        gate.wait()
        for _ in range(ROUNDS):
            for fn, args in seen:
                code = fn(*args)
                if code:
                    codes.append((code, _lib.last_error()))
                    return
    threads = [threading.Thread(target=work, args=(seen,)) for seen, _, _ in made]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not codes, codes
    for seen, outs, want in made:
        assert seen and all(torch.equal(a, b) for a, b in zip(outs[0], want))


def test_reorder(ops, monkeypatch):
    def case(beams):
        def run():
            state = normal(beams, beams, 4)
            parents = torch.zeros(1, beams, dtype=torch.int64, device="cuda")
            at, sizes = ops.array("Q", [state.data_ptr()]), ops.array("Q", [16])
            ops.call("fhe_beam_reorder", ops._reorder_block(
                0, 1, beams, 1, at.buffer_info()[0], sizes.buffer_info()[0], parents.data_ptr(), ops._stream_of(0)))
            return (state,), parents, at, sizes
        return run
    side_by_side(monkeypatch, ops, [case(17), case(64)])


def test_select(ops, monkeypatch):
    def case(beams):
        def run():
            logits, scores = normal(beams, beams, 64), normal(beams + 1, 1, beams)
            return tuple(ops.beam_select(logits, scores, width=64)), logits, scores
        return run
    side_by_side(monkeypatch, ops, [case(40), case(64)])


def test_gated_norm(ops, monkeypatch):
    def case(rows, width):
        def run():
            x, z, w = normal(1, rows, width).bfloat16(), normal(2, rows, width).bfloat16(), 1 + normal(3, width)
            return (ops.gated_rms_norm(x, z, w),), x, z, w
        return run
    side_by_side(monkeypatch, ops, [case(300, 8192), case(2, 16384)])


def test_norm_gradients(ops, monkeypatch):
    def case(width, rows=300):
        def run():
            h, w = normal(1, rows, width), 1 + normal(4, width)
            x, dy = normal(2, rows, width).bfloat16(), normal(3, rows, width).bfloat16()
            rstd, dres, dw = normal(5, rows, 1).abs(), torch.empty_like(h), torch.empty_like(w)
            ws = torch.empty(16 << 20, dtype=torch.uint8, device="cuda")
            f, _ = ops._norm_values(h, torch.float32, torch.bfloat16, 1, 1e-5, 1.0, x, h, None, None, w, None, h, rstd)
            ops.call("fhe_rms_norm_backward", ops._norm_grad_block(
                *f, dy.data_ptr(), 0, 0, dres.data_ptr(), 0, dw.data_ptr(), 0, ws.data_ptr(), ws.numel(), f[-1]))
            return (dres, dw), h, w, x, dy, rstd, ws
        return run
    side_by_side(monkeypatch, ops, [case(1024), case(2560)])
