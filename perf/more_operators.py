"""Workloads of the operators around the plaintext Mamba-2 layers: the norms
with their residual and gate, the token embedding, and beam search's selection
and reordering of states; forward, single-token and training forms.

A case is a dict of plain values.  ``prepare`` makes its inputs on the GPU,
``run`` is one pass (the framework's kernels when ``own`` is true, elementary
torch operations otherwise: in 32 bits, the selection's totals in 64, since
candidates next to each other differ by less than 32 bits hold) and ``exact``
the definition in 64 bits.

Sizes: the 24-layer model of the token loop (d_model 768, d_inner 1536, 24
heads of 64, state 128, convolution window 3 x 1792, in_proj width 3352,
vocabulary 50280) and odd neighbours of them.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5


def norm_case(op, name=None, **kw):
    # stream32: the residual stream is float32 whatever the activations; per_channel: a scale for each channel
    c = {"op": op, "dtype": "bf16", "rows": 1, "width": 768, "stream32": True, "per_channel": False}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def gated_case(op, name=None, **kw):
    # after: channels behind the gate's in the rows that it is a slice of
    c = {"op": op, "dtype": "bf16", "rows": 1, "width": 1536, "groups": 1, "after": 1816}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def embed_case(op, name=None, **kw):
    # zipf: natural text's frequencies, even ones otherwise; padded: share of positions without a token
    c = {"op": op, "dtype": "bf16", "tokens": 1, "vocab": 50280, "width": 768, "scale": 1.0, "out32": True,
         "zipf": True, "padded": 0.0}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def select_case(name=None, **kw):
    # done: share of finished beams; masked: the last tokens of the vocabulary are impossible; keep: survivors stay
    c = {"op": "select", "dtype": "fp32", "batch": 1, "beams": 4, "width": 4, "vocab": 50280, "masked": 0,
         "done": 0.0, "keep": True}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def reorder_case(name=None, **kw):
    c = {"op": "reorder", "dtype": "bf16", "batch": 2, "beams": 4, "survivors": 3, "layers": 24, "heads": 24,
         "head_dim": 64, "d_state": 128, "channels": 1792, "taps": 4}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the residual and norm of one decoded token of four sequences: latency
        norm_case("norm", "norm 4 rows", rows=4),
        # the same over a batch of long texts in a training pass
        norm_case("norm_train", "norm train 32768x768 bf16", rows=32768),
        # an odd width, the stream in 16 bits, a learned residual scale for each channel
        norm_case("norm_train", "norm train 1777x1001 fp16", dtype="fp16", rows=1777, width=1001, stream32=False,
                  per_channel=True),
        # the gated norm behind the recurrence, scoring long prompts in the calibration's accuracy, by groups of heads
        gated_case("gated", "gated 5000x1536 fp32", dtype="fp32", rows=5000, groups=8),
        # a training pass over a batch of long texts, the gate read out of the wide in_proj output
        gated_case("gated_train", "gated train 32768x1536 bf16", rows=32768),
        # the tokens of a batch of long texts in a training pass
        embed_case("embed_train", "embedding train 32768 bf16", tokens=32768),
        # a small batch in float32, a scaled embedding of odd width, a third of the positions padded
        embed_case("embed_train", "embedding train 4072 fp32", dtype="fp32", tokens=4072, vocab=5003, width=769,
                   scale=math.sqrt(769), zipf=False, padded=0.33),
        # one selection of a single request: latency
        select_case("select 1x4 fp32"),
        # a serving batch of wide beams, some of them finished, the vocabulary padded to a round size
        select_case("select 64x8 bf16", dtype="bf16", batch=64, beams=8, width=8, vocab=50304, masked=24, done=0.15),
        # moving the states of every layer after a selection: two requests of four beams
        reorder_case("reorder 2x4"),
        # a serving batch of sixteen requests of eight beams
        reorder_case("reorder 16x8", batch=16, beams=8, survivors=5),
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_train", "norm_train", "gated", "gated_train", "gated_train", "embed",
                     "embed_train", "embed_train", "select", "select", "select", "reorder", "reorder"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    half = 2 if dtype == "fp32" else 1
    if op in ("norm", "norm_train"):
        width = rng.choice([64, 333, 768, 768, 768, 1001, 1536, 2560, 8192, log_int(rng, 1, 16384)])
        return norm_case(op, dtype=dtype, rows=log_int(rng, 1, max(1, 32768 * 768 // (width * half))), width=width,
                         stream32=rng.random() < 0.6, per_channel=rng.random() < 0.3)
    if op in ("gated", "gated_train"):
        groups = rng.choice([1, 1, 1, 3, 5, 8])
        width = groups * rng.choice([64, 192, 555, 768, 1536, 1536, 1792, log_int(rng, 1, 2048)])
        return gated_case(op, dtype=dtype, rows=log_int(rng, 1, max(1, 32768 * 1536 // (width * half) // 2)),
                          width=width, groups=groups, after=rng.choice([0, 0, 24, 1816, 7]))
    if op in ("embed", "embed_train"):
        width = rng.choice([64, 500, 768, 768, 768, 769, 1536])
        vocab = rng.choice([211, 5003, 32000, 50280, 50280])
        return embed_case(op, dtype=dtype, width=width, vocab=vocab,
                          tokens=log_int(rng, 1, max(1, 32768 * 768 // (width * half))),
                          scale=rng.choice([1.0, math.sqrt(width), 0.3]), out32=rng.random() < 0.6,
                          zipf=rng.random() < 0.6, padded=rng.choice([0.0, 0.0, 0.1, 0.5]))
    if op == "select":
        batch = log_int(rng, 1, 64)
        beams = rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 10])
        vocab = rng.choice([256, 5003, 32000, 50280, 50280])
        while batch * beams > 512 // half:
            batch //= 2
        keep = rng.random() < 0.5
        return select_case(dtype=dtype, batch=batch, beams=beams, width=beams if keep else rng.choice(
            [beams, 2 * beams, 20]), vocab=vocab, masked=rng.choice([0, 0, 24]),
            done=rng.choice([0.0, 0.0, 0.2, 0.6]), keep=keep)
    beams = rng.randint(2, 10)
    batch = log_int(rng, 1, max(1, 100 // beams))
    return reorder_case(dtype=dtype, batch=batch, beams=beams, survivors=rng.randint(1, beams - 1),
                        layers=rng.randint(1, 24), heads=rng.choice([24, 24, 12, 5]), head_dim=rng.choice([64, 32]),
                        d_state=rng.choice([128, 64, 16]), channels=rng.choice([1792, 1792, 1001, 640]))


# ---- inputs -------------------------------------------------------------------------------------


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def uniform(g, lo, hi, *shape):
    return lo + (hi - lo) * torch.rand(*shape, generator=g, device="cuda")


def some_tokens(g, case):
    n, v = case["tokens"], case["vocab"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    if case["zipf"]:  # P(v) = log((v + 2) / (v + 1)) / log(vocab + 1)
        t = torch.exp(u * math.log(v + 1)).long() - 1
    else:
        t = (u * v).long()
    t.clamp_(0, v - 1)
    if case["padded"]:
        t[torch.rand(n, generator=g, device="cuda") < case["padded"]] = -1
    return t


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, op = TYPES[case["dtype"]], case["op"]
    s = {"case": case}
    if op in ("norm", "norm_train"):
        r, w = case["rows"], case["width"]
        stream = torch.float32 if case["stream32"] else t
        s["h"] = (normal(g, r, w) * uniform(g, 0.3, 4.0, w)).to(stream)  # channels of a stream differ in size
        s["x"] = (0.5 * normal(g, r, w)).to(t)
        s["weight"] = 1 + 0.1 * normal(g, w)
        s["scale"] = 0.5 + 0.1 * normal(g, w) if case["per_channel"] else 1.0
        if op == "norm_train":
            s["leaves"] = ["h", "x", "weight"] + (["scale"] if case["per_channel"] else [])
            s["grads"] = (normal(g, r, w).to(t), normal(g, r, w).to(stream))
    elif op in ("gated", "gated_train"):
        r, w = case["rows"], case["width"]
        s["x"] = (0.7 * normal(g, r, w)).to(t)
        s["z"] = normal(g, r, w + case["after"]).to(t)[:, :w]
        s["weight"] = 1 + 0.1 * normal(g, w)
        if op == "gated_train":
            s["leaves"] = ["x", "z", "weight"]
            s["grads"] = (normal(g, r, w).to(t),)
    elif op in ("embed", "embed_train"):
        s["tokens"] = some_tokens(g, case)
        s["table"] = (0.02 * normal(g, case["vocab"], case["width"])).to(t)
        if op == "embed_train":
            s["leaves"] = ["table"]
            s["grads"] = (normal(g, case["tokens"], case["width"]).to(torch.float32 if case["out32"] else t),)
    elif op == "select":
        b, k, v = case["batch"], case["beams"], case["vocab"]
        s["logits"] = (2.5 * normal(g, b * k, v)).to(t)
        if case["masked"]:
            s["logits"][:, v - case["masked"]:] = -math.inf
        s["scores"] = -12 + 1.5 * normal(g, b, k)
        s["finished"] = torch.rand(b, k, generator=g, device="cuda") < case["done"]
    else:
        b, k, live = case["batch"], case["beams"], case["survivors"]
        # survivors stay where they are, the other rows copy one of them each in turn
        order = torch.argsort(torch.rand(b, k, generator=g, device="cuda"), dim=1)
        alive, dead = order[:, :live], order[:, live:]
        s["parents"] = torch.empty_like(order)
        s["parents"].scatter_(1, alive, alive)
        s["parents"].scatter_(1, dead, alive[:, torch.arange(k - live, device="cuda") % live])
        s["states"] = []
        for _ in range(case["layers"]):
            s["states"].append(normal(g, b * k, case["taps"] - 1, case["channels"]).to(t))
            s["states"].append(normal(g, b * k, case["heads"], case["head_dim"], case["d_state"]))
    for i in s.get("leaves", ()):
        s[i] = s[i].detach().requires_grad_()
    return s


# ---- one pass -----------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from fhe_mamba_b200 import mamba_ops as ops
        add_norm, gated, embed, select, reorder = (ops.add_rms_norm, ops.gated_rms_norm, ops.embedding,
                                                   ops.beam_select, ops.beam_reorder)
    else:
        add_norm, gated, embed, select, reorder = plain_add_norm, plain_gated, plain_embed, plain_select, plain_reorder
    if op in ("norm", "norm_train"):
        outs = add_norm(s["h"], s["x"], s["weight"], eps=EPS, scale=s["scale"])
    elif op in ("gated", "gated_train"):
        outs = (gated(s["x"], s["z"], s["weight"], eps=EPS, groups=case["groups"]),)
    elif op in ("embed", "embed_train"):
        outs = (embed(s["tokens"], s["table"], scale=case["scale"], dtype=torch.float32 if case["out32"] else None),)
    elif op == "select":
        return tuple(select(s["logits"], s["scores"], finished=s["finished"], eos=0, width=case["width"],
                            keep_slots=case["keep"]))
    else:
        reorder(s["states"], s["parents"])
        return tuple(s["states"])
    outs = tuple(outs)
    if "leaves" not in s:
        return outs
    grads = torch.autograd.grad(outs, [s[i] for i in s["leaves"]], s["grads"])
    return tuple(o.detach() for o in outs) + tuple(grads)


def plain_add_norm(residual, x, weight, eps, scale):
    """h = residual + scale x, rounded to the stream's type, and h / sqrt(mean(h^2) + eps) * weight.  Gradients pass
    the rounding as they are."""
    h = residual.float() + scale * x.float()
    h = h + (h.to(residual.dtype).float() - h).detach()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight
    return y.to(x.dtype), h.to(residual.dtype)


def plain_gated(x, gate, weight, eps, groups):
    """x silu(gate), normalised over each group of channels, times weight."""
    z = gate.float()
    v = (x.float() * (z / (1 + torch.exp(-z)))).unflatten(-1, (groups, -1))
    y = (v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)).flatten(-2) * weight
    return y.to(x.dtype)


def plain_embed(tokens, table, scale, dtype):
    """Rows of the table times scale; 0 where there is no token."""
    rows = table.float()[tokens.clamp(min=0)] * scale
    return torch.where((tokens >= 0)[:, None], rows, 0.0).to(dtype or table.dtype)


def plain_select(logits, scores, finished, eos, width, keep_slots):
    """The `width` best of every beam's score plus its tokens' log-probabilities, the lower beam and then the
    lower token first among equals."""
    b, k = scores.shape
    v = logits.shape[1]
    z = logits.double().view(b, k, v)
    start = scores.double()[..., None]
    top = z.max(-1, keepdim=True).values
    lse = top + torch.log(torch.exp(z - top).sum(-1, keepdim=True))
    total = torch.where(torch.isfinite(lse) & torch.isfinite(start), start + z - lse, -math.inf)
    only = torch.full_like(total, -math.inf)
    only[..., eos] = scores.double()
    total = torch.where(finished[..., None], only, total).flatten(1)
    best, at = torch.sort(total, dim=-1, descending=True, stable=True)
    best, at = best[:, :width], at[:, :width]
    parents, tokens = at // v, at % v
    done = torch.gather(finished, 1, parents) | (tokens == eos)
    outs = (best.float(), parents, tokens, done)
    if not keep_slots:
        return outs
    # the best child of a beam takes its place, the others the free places in turn
    rank = torch.arange(k, device=parents.device)
    same = parents[:, :, None] == parents[:, None, :]
    first = ~(same & (rank[None, :] < rank[:, None])).any(-1)
    taken = (parents[:, None, :] == rank[None, :, None]).any(-1)
    free = torch.sort(taken.to(torch.uint8), dim=1, stable=True)[1]
    place = torch.where(first, parents, torch.gather(free, 1, (torch.cumsum(~first, 1) - 1).clamp(min=0)))
    return tuple(torch.empty_like(o).scatter_(1, place, o) for o in outs)


def plain_reorder(states, parents):
    """Row i of each batch item's beams becomes its row parents[i], in place."""
    b, k = parents.shape
    item = torch.arange(b, device=parents.device)[:, None]
    for v in states:
        rows = v.view(b, k, -1)
        rows.copy_(rows[item, parents])


# ---- what a pass cannot do without --------------------------------------------------------------


def distinct(case):
    """Expected number of different tokens."""
    v, n = case["vocab"], case["tokens"] * (1 - case["padded"])
    if not case["zipf"]:
        return v * -math.expm1(n * math.log1p(-1 / v)) if v > 1 else min(n, 1)
    i = torch.arange(v, dtype=torch.float64)
    p = torch.log((i + 2) / (i + 1)) / math.log(v + 1)
    return float((-torch.expm1(n * torch.log1p(-p.clamp(max=1 - 1e-9)))).sum())


def work(case):
    e, op = BYTES[case["dtype"]], case["op"]
    if op in ("norm", "norm_train"):
        r, w = case["rows"], case["width"]
        h = 4 if case["stream32"] else e
        total, flops = r * w * 2 * (h + e) + 4 * w, 6 * r * w
        if op == "norm_train":  # both outputs' gradients in, both inputs' out; x again for the scale's
            total += r * w * (2 * (h + e) + h + (e if case["per_channel"] else 0)) + 8 * w
            flops += 12 * r * w
        return {"bytes": total, "flops": flops}
    if op in ("gated", "gated_train"):
        r, w = case["rows"], case["width"]
        total, flops = 3 * r * w * e + 4 * w, 8 * r * w
        if op == "gated_train":
            total += 5 * r * w * e + 8 * w
            flops += 20 * r * w
        return {"bytes": total, "flops": flops}
    if op in ("embed", "embed_train"):
        n, w = case["tokens"], case["width"]
        out = 4 if case["out32"] else e
        total, flops = 8 * n + distinct(case) * w * e + n * w * out, n * w
        if op == "embed_train":
            total += 8 * n + n * (1 - case["padded"]) * w * out + case["vocab"] * w * e
            flops += n * w
        return {"bytes": total, "flops": flops}
    if op == "select":
        b, k, v = case["batch"], case["beams"], case["vocab"]
        live = b * k * (1 - case["done"])
        return {"bytes": live * v * e + b * k * 5 + b * case["width"] * 21, "flops": 4 * live * v}
    k, live = case["beams"], case["survivors"]
    row = case["layers"] * (case["heads"] * case["head_dim"] * case["d_state"] * 4 +
                            (case["taps"] - 1) * case["channels"] * e)
    moved = k - live
    return {"bytes": case["batch"] * (row * (moved + min(moved, live)) + 8 * k), "flops": 0}


# ---- the definition in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "reorder":
        return None  # rows moved as they are
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("norm", "norm_train"):
            return exact_norm(s)
        if case["op"] in ("gated", "gated_train"):
            return exact_gated(s)
        if case["op"] in ("embed", "embed_train"):
            return exact_embed(s)
        return exact_select(s)


def exact_norm(s):
    """The gradients by the formula, some rows at a time."""
    scale = s["scale"].double() if torch.is_tensor(s["scale"]) else s["scale"]
    w, n = s["weight"].double(), s["case"]["width"]
    parts, dw, ds = [], torch.zeros_like(w), torch.zeros_like(w)
    for i in range(0, s["case"]["rows"], 4096):
        at = slice(i, i + 4096)
        x = s["x"][at].double()
        whole = torch.addcmul(s["h"][at].double(), x, torch.as_tensor(scale, device=x.device, dtype=x.dtype))
        h = whole.to(s["h"].dtype).double()  # the norm is that of the stream as it is kept
        r = torch.rsqrt(torch.einsum("rw,rw->r", h, h) / n + EPS)[:, None]
        out = [r * h * w, whole]
        if "grads" in s:
            dy, dh = (v[at].double() for v in s["grads"])
            a = dy * w
            dh = dh + r * a - r ** 3 * h * (torch.einsum("rw,rw->r", a, h) / n)[:, None]
            dw += torch.einsum("rw,rw->w", dy, r * h)
            ds += torch.einsum("rw,rw->w", dh, x)
            out += [dh, dh * scale]
        parts.append(out)
    outs = tuple(torch.cat(v) for v in zip(*parts))
    if "grads" in s:
        outs += (dw,) + ((ds,) if s["case"]["per_channel"] else ())
    return outs


def exact_gated(s):
    w, k = s["weight"].double(), s["case"]["groups"]
    n = s["case"]["width"] // k
    parts, dw = [], torch.zeros_like(w)
    for i in range(0, s["case"]["rows"], 4096):
        x, z = (s[j][i:i + 4096].double() for j in ("x", "z"))
        q = torch.sigmoid(z)
        v = x * z * q
        spread = lambda u: u.repeat_interleave(n, 1)  # noqa: E731
        r = spread(torch.rsqrt(v.square().view(-1, k, n).mean(-1) + EPS))
        out = [v * r * w]
        if "grads" in s:
            dy = s["grads"][0][i:i + 4096].double()
            a = dy * w
            dv = r * a - r ** 3 * v * spread((a * v).view(-1, k, n).mean(-1))
            dw += (dy * v * r).sum(0)
            out += [dv * z * q, dv * x * (q + z * q * (1 - q))]
        parts.append(out)
    outs = tuple(torch.cat(v) for v in zip(*parts))
    return outs + ((dw,) if "grads" in s else ())


def exact_embed(s):
    case, t = s["case"], s["tokens"]
    used = t >= 0
    y = torch.zeros(case["tokens"], case["width"], device=t.device, dtype=torch.float64)
    y[used] = torch.index_select(s["table"].double(), 0, t[used]) * case["scale"]
    if case["op"] == "embed":
        return (y,)
    d = torch.zeros(case["vocab"], case["width"], device=t.device, dtype=torch.float64)
    d.index_add_(0, t[used], s["grads"][0][used].double())
    return y, d * case["scale"]


def exact_select(s):
    """Each batch item by itself: its few best tokens of each beam, put together and ordered on the host."""
    case = s["case"]
    b, k, v, width = (case[i] for i in ("batch", "beams", "vocab", "width"))
    scores, finished = s["scores"].double().tolist(), s["finished"].tolist()
    outs = []
    for i in range(b):
        found = []
        for j in range(k):
            if finished[i][j]:
                found.append((-scores[i][j], j, 0))
                found += [(math.inf, j, t) for t in range(1, min(v, width + 1))]
                continue
            z = s["logits"][i * k + j].double()
            lse = torch.logsumexp(z, 0).item()
            at = torch.sort(z, descending=True, stable=True)[1][:width]
            found += [(-(scores[i][j] + x - lse), j, t) for x, t in zip(z[at].tolist(), at.tolist())]
        found = sorted(found)[:width]
        if case["keep"]:
            places = [None] * k
            rest = []
            for c in found:
                if places[c[1]] is None:
                    places[c[1]] = c
                else:
                    rest.append(c)
            empty = [j for j in range(k) if places[j] is None]
            for j, c in zip(empty, rest):
                places[j] = c
            found = places
        outs.append(([-c[0] for c in found], [c[1] for c in found], [c[2] for c in found],
                     [finished[i][c[1]] or c[2] == 0 for c in found]))
    kinds = (torch.float64, torch.int64, torch.int64, torch.bool)
    return tuple(torch.tensor([o[i] for o in outs], dtype=d, device="cuda") for i, d in enumerate(kinds))
