"""Beam search's selection and reordering on the GPU.

Parents, tokens and ends have to be those of the totals score + logit - log sum
exp in float64, also where float32 does not tell candidates apart.  A returned
score is that total rounded to float32, from a sum of exponentials off by at
most 2^-24 (2.2 (log2 of the vocabulary + 12) + 32) relative to itself (5.6e-6 up
to 2^17 tokens), and 8 2^-24 more for each time that a running shift moves: 8e-6
with five of them.  Moved rows are equal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
INF = math.inf
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
    from fhe_mamba_b200 import mamba_ops
    return mamba_ops


def rand(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def want_select(logits, scores, finished, eos, width, keep):
    """(scores, parents, tokens, finished) by the definition, on the host in float64."""
    b, k = scores.shape
    v = logits.shape[-1]
    z = logits.reshape(b, k, v).double().cpu()
    top = z.max(-1, keepdim=True).values
    lse = top[..., 0] + torch.log(torch.exp(z - top).sum(-1))
    s = scores.double().cpu()
    total = s[..., None] + z - lse[..., None]
    total[~(torch.isfinite(lse) & torch.isfinite(s))] = -INF
    done = finished.cpu() if finished is not None else torch.zeros(b, k, dtype=torch.bool)
    for i, j in done.nonzero().tolist():
        total[i, j] = -INF
        if math.isfinite(s[i, j]):
            total[i, j, eos] = s[i, j]
    outs = []
    for i in range(b):
        order = torch.sort(total[i].flatten(), descending=True, stable=True)[1][:width].tolist()
        picked = [(total[i].flatten()[o].item(), o // v, o % v) for o in order]
        if keep:
            places, rest = {}, []
            for p in picked:
                rest.append(p) if p[1] in places else places.__setitem__(p[1], p)
            for j in range(k):
                if j not in places:
                    places[j] = rest.pop(0)
            picked = [places[j] for j in range(k)]
        outs.append([(t, p, tok, bool(done[i, p]) or tok == eos) for t, p, tok in picked])
    return outs


def check(ops, logits, scores, finished=None, eos=None, width=None, keep=False):
    got = ops.beam_select(logits, scores, finished, eos, width, keep)
    want = want_select(logits, scores, finished, eos, width or scores.shape[1], keep)
    b, w = scores.shape[0], width or scores.shape[1]
    assert all(t.shape == (b, w) for t in got)
    assert got.scores.dtype == torch.float32 and got.parents.dtype == got.tokens.dtype == torch.int64
    values = [t.tolist() for t in got]
    for i in range(b):
        for j, (t, p, tok, end) in enumerate(want[i]):
            assert (values[1][i][j], values[2][i][j], values[3][i][j]) == (p, tok, end), (i, j)
            s = values[0][i][j]
            assert s == t if not math.isfinite(t) else abs(s - t) <= 8e-6 + 2.0 ** -24 * (abs(t) + 8e-6), (i, j, s, t)
    return got


# batch, beams, width, vocab
SIZES = [(1, 1, 1, 1), (1, 1, 5, 7), (2, 3, 3, 2), (1, 4, 4, 50280), (3, 4, 8, 50281), (64, 8, 8, 5003), (5, 10, 20, 1000),
         (2, 64, 64, 300), (1, 64, 64, 20000), (700, 2, 2, 257), (1, 1, 64, 131072), (9, 5, 5, 32001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch, beams, width, vocab", SIZES)
def test_select(ops, dtype, batch, beams, width, vocab):
    g = rand(vocab + beams)
    logits = (2.5 * torch.randn(batch * beams, vocab, generator=g, device="cuda")).to(dtype)
    scores = -12 + 1.5 * torch.randn(batch, beams, generator=g, device="cuda")
    check(ops, logits, scores, width=width)
    finished = torch.rand(batch, beams, generator=g, device="cuda") < 0.4
    check(ops, logits.view(batch, beams, vocab), scores, finished, vocab // 2, width)
    # masked tokens, beams that do not count, a beam with nothing but impossible tokens, one with a NaN or an infinity
    logits[torch.rand(logits.shape, generator=g, device="cuda") < 0.5] = -INF
    start = scores.clone()
    start[:, 1:] = -INF
    check(ops, logits, start, None, 0, width)
    logits[0] = -INF
    if batch * beams > 3:
        logits[1, vocab // 3] = math.nan
        logits[2, vocab - 1] = INF
        scores[-1, -1] = math.nan
        scores[-1, 0] = INF
    check(ops, logits, scores, None, None, width)
    check(ops, logits, scores, finished, 0, width)
    if width == beams:
        check(ops, logits, scores, finished, vocab - 1, width, True)
        check(ops, logits, scores, None, None, None, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [5, 777, 50280, 50283])
def test_ties(ops, dtype, vocab):
    """Equal logits, equal beams, and many entries of one value: the lower beam, then the lower token."""
    for value in (0.0, -3.0, 2.0 ** 15):
        check(ops, torch.full((8, vocab), value, device="cuda", dtype=dtype), torch.zeros(2, 4, device="cuda"))
    g = rand(vocab)
    row = torch.randn(vocab, generator=g, device="cuda").to(dtype)
    same = row.expand(12, vocab)
    check(ops, same, torch.zeros(3, 4, device="cuda"), width=min(20, 4 * vocab))
    apart = torch.zeros(3, 4, device="cuda")
    apart[:, 1] = torch.nextafter(apart[:, 1], apart[:, 1] + 1)  # larger by the least that there is
    apart[1] -= 7
    apart[1, 3] = torch.nextafter(apart[1, 3], apart[1, 3] + 1)
    check(ops, same, apart, width=min(20, 4 * vocab))
    # many lists of equal entries, of possible and of impossible ones
    wide = torch.zeros(2, 16, device="cuda")
    check(ops, row.expand(32, vocab), wide, width=min(64, 16 * vocab))
    wide[1, 3:] = -INF
    check(ops, torch.full((32, vocab), -1.0, device="cuda", dtype=dtype), wide, width=min(64, 16 * vocab))
    check(ops, torch.full((32, vocab), -INF, device="cuda", dtype=dtype), wide, width=min(64, 16 * vocab))
    few = (row * 2).round() / 2
    check(ops, few.expand(12, vocab), apart, width=min(16, 4 * vocab))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1001, 50280])
def test_candidates_closer_than_float32(ops, dtype, vocab):
    """Scores set so that the beams' best tokens have equal totals but for the scores' own roundings."""
    g = rand(vocab)
    b, k = 40, 4
    z = (3 * torch.randn(b, k, vocab, generator=g, device="cuda")).to(dtype)
    best = torch.log_softmax(z.double(), -1).max(-1).values
    scores = (best[:, :1] - best - 10).float()
    totals = (scores.double() + best).cpu()
    assert (totals - totals[:, :1]).abs().max() < 4e-6
    for width in (1, 2, 4, 7):
        check(ops, z, scores, width=width)
    check(ops, z, scores, keep=True)
    # the second best of each against the best of another
    second = torch.log_softmax(z.double(), -1).topk(2).values[..., 1]
    scores[:, 1] = (best[:, 0] + scores[:, 0] - second[:, 1]).float()
    check(ops, z, scores, width=8)


def test_large_and_shifted_logits(ops):
    """Logits far from zero, ascending rows (the shift moves on every turn) and rows of the largest numbers."""
    g = rand(5)
    z = torch.randn(8, 30011, generator=g, device="cuda")
    scores = torch.zeros(2, 4, device="cuda")
    for t in (z + 5000, z - 70000, z * 1e30, z.clamp(-1, 1) * 3e38, torch.sort(z * 5).values,
              torch.sort(z * 5, descending=True).values, z * 1e-6):
        check(ops, t, scores, width=6)
    check(ops, torch.sort(z * 30).values.half(), scores)


def test_strides_streams_and_graphs(ops):
    g = rand(6)
    wide = torch.randn(8, 1100, generator=g, device="cuda")
    scores = -torch.rand(4, 4, generator=g, device="cuda")
    for logits in (wide[:, 3:1003], wide[:, :1001], wide.t()[:1000].t(), wide[::2, 100:]):
        n = logits.shape[0] // 4
        check(ops, logits, scores[:n])
        check(ops, logits, scores.t()[:n])
        check(ops, logits, scores.t()[:, :n].t())
    logits = (3 * torch.randn(16, 5003, generator=g, device="cuda")).bfloat16()
    finished = torch.zeros(4, 4, dtype=torch.bool, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.beam_select(logits, scores, finished, 0)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, ops.beam_select(logits, scores, finished, 0)))
    state = torch.randn(16, 33, 7, generator=g, device="cuda")

    def step():
        out = ops.beam_select(logits, scores, finished, 0, keep_slots=True)
        ops.beam_reorder([state], out.parents)
        return out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    logits.copy_(logits.flip(0))
    finished[1, 2] = True
    before = state.clone()
    graph.replay()
    torch.cuda.synchronize()
    want = ops.beam_select(logits, scores, finished, 0, keep_slots=True)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    rows = (torch.arange(4, device="cuda")[:, None] * 4 + want.parents).flatten()
    assert torch.equal(state, before[rows])
    assert ops.beam_select(logits[:0], scores[:0]).tokens.shape == (0, 4)


@pytest.mark.parametrize("batch, beams", [(1, 1), (1, 2), (3, 4), (2, 8), (5, 9), (2, 16), (3, 17), (1, 64)])
def test_reorder(ops, batch, beams):
    """Permutations, cycles, copies and rows that stay, over tensors of odd sizes, types and alignments."""
    g = rand(beams)
    n = batch * beams
    storage = torch.randint(0, 255, (n * 1003 + 3,), generator=g, device="cuda", dtype=torch.uint8)
    ahead = storage[:3].clone()
    states = [torch.randn(n, 3, 1792, generator=g, device="cuda").bfloat16(), torch.randn(n, 24, 64, 16, generator=g, device="cuda"),
              torch.randn(batch, beams, 1001, generator=g, device="cuda").half(), storage[3:].view(n, 1003),
              torch.randint(0, 9, (n,), generator=g, device="cuda"), torch.rand(n, 5, generator=g, device="cuda") < 0.5,
              torch.randn(n, 4097, generator=g, device="cuda"), torch.empty(n, 0, device="cuda"),
              torch.randn(n, 1, generator=g, device="cuda").double()]
    states += [torch.randn(n, 5 + i, generator=g, device="cuda") for i in range(130)]
    shift = torch.arange(beams, device="cuda").roll(1).expand(batch, beams)
    for parents in (torch.randint(0, beams, (batch, beams), generator=g, device="cuda"), shift,
                    torch.arange(beams, device="cuda").expand(batch, beams), torch.zeros(batch, beams, dtype=torch.int64, device="cuda"),
                    torch.randint(-2, beams + 2, (batch, beams), generator=g, device="cuda")):
        before = [t.clone() for t in states]
        version = states[0]._version
        ops.beam_reorder(states, parents)
        own = torch.arange(beams, device="cuda")
        fine = torch.where((parents >= 0) & (parents < beams), parents, own)
        rows = (torch.arange(batch, device="cuda")[:, None] * beams + fine).flatten()
        for t, was in zip(states, before):
            if t.numel():
                assert torch.equal(t.view(n, -1), was.view(n, -1)[rows])
        assert states[0]._version > version
    assert torch.equal(storage[:3], ahead)
    ops.beam_reorder([], shift)


def test_reorder_broadcast_parents(ops):
    """Parents that are one row for every item, and a state right behind that row in memory."""
    flat = torch.zeros(4 + 400 * 4, dtype=torch.int64, device="cuda")
    flat[:4] = torch.tensor([1, 1, 0, 3], device="cuda")
    flat[4:] = torch.arange(400 * 4, device="cuda")
    state = flat[4:].view(1600, 1)
    ops.beam_reorder([state], flat[:4].expand(400, 4))
    want = (torch.arange(400, device="cuda")[:, None] * 4 + flat[:4]).view(1600, 1)
    assert torch.equal(state, want)


def test_reorder_large_offsets(ops):
    """Rows past 2^32 bytes."""
    state = torch.zeros(6, (1 << 30) + 8, dtype=torch.uint8, device="cuda")
    state[4, -5:] = torch.arange(1, 6, dtype=torch.uint8, device="cuda")
    ops.beam_reorder([state], torch.tensor([[0, 1, 2, 3, 4, 4]], device="cuda"))
    assert torch.equal(state[5, -5:], state[4, -5:]) and not state[5, :-5].any() and not state[3].any()
