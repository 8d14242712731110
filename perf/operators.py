"""Workloads of the plaintext Mamba-2 operators: the state scan, the causal
convolution and the token log-probabilities, each with its single-token form
or its gradients.

A case is a dict of plain values.  ``prepare`` makes its inputs on the GPU,
``run`` is one pass (the framework's kernels when ``own`` is true, elementary
torch operations in 32 bits otherwise) and ``exact`` the definition in 64 bits.

Sizes: the 24-layer model of the token loop (d_model 768, d_inner 1536, 24
heads of 64, state 128, one group, convolution over 1792 channels with 4 taps,
in_proj width 3352, vocabulary 50280, calibration of 8 sequences of 32 tokens)
and odd neighbours of them.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def scan_case(op, name=None, **kw):
    c = {"op": op, "dtype": "bf16", "batch": 1, "length": 1, "heads": 24, "head_dim": 64, "d_state": 128,
         "groups": 1, "ragged": False, "resets": False, "carried": True}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def conv_case(op, name=None, **kw):
    c = {"op": op, "dtype": "bf16", "batch": 1, "length": 1, "channels": 1792, "taps": 4, "before": 1536,
         "after": 24, "silu": True, "ragged": False, "carried": True}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def logprob_case(op, name=None, **kw):
    c = {"op": op, "dtype": "fp32", "rows": 1, "vocab": 50280, "top": 5, "padded": 0, "ignored": False}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one decoded token of four sequences beside the encrypted loop: latency
        scan_case("step", "step 4 sequences", batch=4),
        # one decoded token of a serving batch: the state is read and written once
        scan_case("step", "step 192 sequences", batch=192),
        # the calibration's own shape, 8 sequences of 32 tokens, in the accuracy it runs in
        scan_case("scan", "scan calibration fp32", dtype="fp32", batch=8, length=32, carried=False),
        # a batch of long prompts
        scan_case("scan", "scan 8x4096 bf16", batch=8, length=4096),
        # prompts of different lengths after a shared prefix, packed texts restarting inside a row
        scan_case("scan", "scan ragged 5x1777 fp16", dtype="fp16", batch=5, length=1777, ragged=True, resets=True),
        # one training pass over a batch of texts
        scan_case("scan_train", "scan train 4x2048 bf16", batch=4, length=2048, carried=False),
        # the same in the calibration's accuracy, an odd length and carried states
        scan_case("scan_train", "scan train 8x509 fp32", dtype="fp32", batch=8, length=509),
        # the convolution of a batch of long prompts, read out of the wide in_proj output
        conv_case("conv", "conv 8x4096 bf16", batch=8, length=4096),
        # its training pass at an odd length
        conv_case("conv_train", "conv train 8x1001 fp32", dtype="fp32", batch=8, length=1001),
        # the client's selection after one decrypted token
        logprob_case("logprobs", "logprobs 1 row fp32"),
        # scoring a prompt of 4095 tokens with its alternatives
        logprob_case("logprobs", "logprobs 4095 rows bf16", dtype="bf16", rows=4095, top=8),
        # a training loss over a batch, some tokens ignored, the vocabulary padded to a round size
        logprob_case("logprobs_train", "logprobs train 2048 rows bf16", dtype="bf16", rows=2048, vocab=50304,
                     padded=24, ignored=True, top=0),
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "scan_train", "scan_train", "conv", "conv_train", "logprobs",
                     "logprobs", "logprobs_train"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op in ("step", "scan", "scan_train"):
        groups = rng.choice([1, 1, 1, 2, 4])
        heads = groups * rng.randint(1, 24 // groups)
        head_dim = rng.choice([16, 32, 48, 64, 64, 64, 80, 128])
        d_state = rng.choice([16, 32, 64, 100, 128, 128, 128, 256])
        batch = log_int(rng, 1, 16)
        if op == "step":
            batch = log_int(rng, 1, 192)
            return scan_case(op, dtype=dtype, batch=batch, heads=heads, head_dim=head_dim, d_state=d_state,
                             groups=groups)
        most = 8 * 4096 if op == "scan" else 4 * 2048
        if dtype == "fp32" or d_state * head_dim > 8192:
            most //= 2
        length = log_int(rng, 1, min(4096, max(1, most // batch)))
        return scan_case(op, dtype=dtype, batch=batch, length=length, heads=heads, head_dim=head_dim,
                         d_state=d_state, groups=groups, ragged=rng.random() < 0.4, resets=rng.random() < 0.3,
                         carried=rng.random() < 0.5)
    if op in ("conv", "conv_train"):
        batch = log_int(rng, 1, 16)
        channels = rng.choice([144, 288, 640, 1001, 1792, 1792, 2304])
        most = 8 * 4096 if op == "conv" else 8 * 1001
        length = log_int(rng, 1, max(1, most * 1792 // (2304 * batch)))
        wide = rng.random() < 0.6
        return conv_case(op, dtype=dtype, batch=batch, length=length, channels=channels, taps=rng.randint(2, 4),
                         before=1536 if wide else 0, after=rng.choice([24, 7]) if wide else 0,
                         silu=rng.random() < 0.8, ragged=rng.random() < 0.4, carried=rng.random() < 0.5)
    rows = log_int(rng, 1, 4095 if op == "logprobs" else 2048)
    vocab = rng.choice([256, 1003, 8192, 32000, 50280, 50280, 50280])
    if dtype == "fp32":
        rows = max(1, rows // 2)
    return logprob_case(op, dtype=dtype, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 8, 20]),
                        padded=rng.choice([0, 0, 24]), ignored=rng.random() < 0.5)


# ---- inputs -------------------------------------------------------------------------------------


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def uniform(g, lo, hi, *shape):
    return lo + (hi - lo) * torch.rand(*shape, generator=g, device="cuda")


def silu(v):
    return v / (1 + torch.exp(-v))


def some_lengths(g, batch, length):
    """Lengths between none and all of a row, both among them where the batch has room."""
    n = torch.randint(0, length + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    n[0] = length
    if batch > 2:
        n[1] = 0
    return n


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]
    s = {"case": case}
    train = case["op"].endswith("train")
    if case["op"] in ("step", "scan", "scan_train"):
        b, l, h, p, n, k = (case[i] for i in ("batch", "length", "heads", "head_dim", "d_state", "groups"))
        # x, B and C are slices of one activated convolution output, as the layer holds them
        xa = silu(normal(g, b, l, h * p + 2 * k * n)).to(t)
        dt_bias = torch.log(torch.expm1(uniform(g, 0.001, 0.1, h)))
        write = torch.nn.functional.softplus(0.5 * normal(g, b, l, h) + dt_bias)
        log_decay = -uniform(g, 1.0, 16.0, h) * write
        if case["resets"]:
            log_decay[torch.rand(b, l, 1, generator=g, device="cuda").expand(b, l, h) < 0.004] = -math.inf
        s["x"] = xa[..., :h * p].unflatten(-1, (h, p))
        s["B"] = xa[..., h * p:h * p + k * n].unflatten(-1, (k, n))
        s["C"] = xa[..., h * p + k * n:].unflatten(-1, (k, n))
        s["write"], s["log_decay"] = write, log_decay
        s["D"] = 1 + 0.1 * normal(g, h)
        s["state"] = uniform(g, -1, 1, b, h, p, n) if case["carried"] else None
        s["lengths"] = some_lengths(g, b, l) if case["ragged"] else None
        if case["op"] == "step":
            for i in ("x", "B", "C", "write", "log_decay"):
                s[i] = s[i][:, 0]
            s["next"] = torch.empty_like(s["state"])
        if train:
            s["leaves"] = ["x", "write", "log_decay", "B", "C", "D"] + (["state"] if case["carried"] else [])
            s["grads"] = (normal(g, b, l, h, p).to(t), 0.1 * normal(g, b, h, p, n))
    elif case["op"] in ("conv", "conv_train"):
        b, l, c, k = (case[i] for i in ("batch", "length", "channels", "taps"))
        wide = normal(g, b, l, case["before"] + c + case["after"]).to(t)
        s["x"] = wide[..., case["before"]:case["before"] + c]
        s["weight"] = (0.2 * normal(g, c, k)).to(t)
        s["bias"] = (0.02 * normal(g, c)).to(t)
        s["state"] = normal(g, b, k - 1, c).to(t) if case["carried"] else None
        s["lengths"] = some_lengths(g, b, l) if case["ragged"] else None
        if train:
            s["leaves"] = ["x", "weight", "bias"] + (["state"] if case["carried"] else [])
            s["grads"] = (normal(g, b, l, c).to(t), normal(g, b, k - 1, c).to(t))
    else:
        r, v = case["rows"], case["vocab"]
        logits = (2.5 * normal(g, r, v)).to(t)
        if case["padded"]:
            logits[:, v - case["padded"]:] = -math.inf
        s["logits"] = logits
        s["targets"] = torch.randint(0, v - case["padded"], (r,), generator=g, device="cuda")
        if case["ignored"]:
            s["targets"][torch.rand(r, generator=g, device="cuda") < 0.2] = -1
        if train:
            s["leaves"] = ["logits"]
            s["grads"] = (normal(g, r), 0.1 * normal(g, r)) + ((0.1 * normal(g, r, case["top"]),) if case["top"]
                                                               else ())
    for i in s.get("leaves", ()):
        s[i] = s[i].detach().requires_grad_()
    return s


# ---- one pass -----------------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        from fhe_mamba_b200 import mamba_ops as ops
        scan, step, conv, logprobs = ops.ssm_scan, ops.ssm_step, ops.causal_conv, ops.token_logprobs
    else:
        scan, step, conv, logprobs = plain_scan, plain_step, plain_conv, plain_logprobs
    if op == "step":
        return step(s["state"], s["x"], s["write"], s["log_decay"], s["B"], s["C"], D=s["D"], out=s["next"])
    if op in ("scan", "scan_train"):
        outs = scan(s["x"], s["write"], s["log_decay"], s["B"], s["C"], D=s["D"], initial_state=s["state"],
                    lengths=s["lengths"])
    elif op in ("conv", "conv_train"):
        outs = conv(s["x"], s["weight"], s["bias"], initial_state=s["state"], lengths=s["lengths"],
                    activation="silu" if s["case"]["silu"] else None)
    else:
        outs = logprobs(s["logits"], s["targets"], top_k=s["case"]["top"])
    outs = tuple(outs)
    if "leaves" not in s:
        return outs
    followed = [o for o in outs if o.is_floating_point() and o.numel()]
    grads = torch.autograd.grad(followed, [s[i] for i in s["leaves"]], [g for g in s["grads"] if g.numel()])
    return tuple(o.detach() for o in outs) + tuple(grads)


def plain_step(state, x, write, log_decay, B, C, D, out):
    """S' = exp(log_decay) S + write x (x) B and y = S' C + D x for one token of each sequence."""
    h, k = x.shape[1], B.shape[1]
    xf = x.float()
    bf, cf = (v.float().repeat_interleave(h // k, dim=1) for v in (B, C))
    torch.add(torch.exp(log_decay)[..., None, None] * state,
              (write[..., None] * xf)[..., None] * bf[:, :, None, :], out=out)
    y = (out * cf[:, :, None, :]).sum(-1) + D[:, None] * xf
    return y.to(x.dtype), out


def plain_scan(x, write, log_decay, B, C, D, initial_state, lengths, chunk=64):
    """The recurrence of ``plain_step`` over every token, 64 tokens at a time: within a chunk the
    decays between two tokens multiply the products of C and B, across chunks the state carries on."""
    b, l, h, p = x.shape
    k, n = B.shape[2], B.shape[3]
    xf = x.float()
    bf, cf = B.float(), C.float()
    w, la = write, log_decay
    if lengths is not None:
        inside = torch.arange(l, device=x.device) < lengths[:, None]
        w = torch.where(inside[..., None], w, 0.0)
        la = torch.where(inside[..., None], la, 0.0)
    s = initial_state if initial_state is not None else x.new_zeros(b, h, p, n, dtype=torch.float32)
    ys = []
    for i in range(0, l, chunk):
        j = min(l, i + chunk)
        q = j - i
        at = la[:, i:j].transpose(1, 2)  # [b, h, q]
        wt = w[:, i:j].transpose(1, 2)
        xt = xf[:, i:j].transpose(1, 2)  # [b, h, q, p]
        bt = bf[:, i:j].transpose(1, 2).repeat_interleave(h // k, dim=1)  # [b, h, q, n]
        ct = cf[:, i:j].transpose(1, 2).repeat_interleave(h // k, dim=1)
        ones = torch.ones(q, q, device=x.device, dtype=torch.bool)
        steps = torch.where(ones.tril(-1), at[..., :, None], 0.0)  # log decay of token t where t > s
        between = torch.where(ones.tril(), torch.exp(torch.cumsum(steps.double(), -2)), 0.0).float()
        since = torch.exp(torch.cumsum(at.double(), -1)).float()  # from the chunk's start to t
        m = (ct @ bt.transpose(-1, -2)) * between * wt[..., None, :]
        ys.append((m @ xt + since[..., None] * (ct @ s.transpose(-1, -2))).transpose(1, 2))
        to_end = between[..., -1, :] * wt
        s = since[..., -1, None, None] * s + (xt * to_end[..., None]).transpose(-1, -2) @ bt
    y = torch.cat(ys, 1) + D[:, None] * xf
    if lengths is not None:
        y = torch.where(inside[..., None, None], y, 0.0)
    return y.to(x.dtype), s


def plain_conv(x, weight, bias, initial_state, lengths, activation):
    """y_t = act(bias + sum_i weight_i x_(t - taps + 1 + i)) per channel; the state is the window before the row."""
    b, l, c = x.shape
    k = weight.shape[1]
    before = initial_state.float() if initial_state is not None else x.new_zeros(b, k - 1, c, dtype=torch.float32)
    row = torch.cat([before, x.float()], 1)
    wf = weight.float()
    y = bias.float() + sum(wf[:, i] * row[:, i:i + l] for i in range(k))
    if activation == "silu":
        y = y * (1 / (1 + torch.exp(-y)))
    if lengths is None:
        return y.to(x.dtype), row[:, l:].to(x.dtype)
    y = torch.where((torch.arange(l, device=x.device) < lengths[:, None])[..., None], y, 0.0)
    last = lengths[:, None].long() + torch.arange(k - 1, device=x.device)
    return y.to(x.dtype), torch.gather(row, 1, last[..., None].expand(b, k - 1, c)).to(x.dtype)


def plain_logprobs(logits, targets, top_k):
    """log softmax at the targets (0 for an ignored target), the entropy and the top_k largest with their
    log-probabilities, the lower index first among equals."""
    z = logits.float()
    top = z.max(-1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    lp = z - top - torch.log(total)
    prob = e / total
    entropy = -(prob * torch.where(prob > 0, lp, 0.0)).sum(-1)
    at = torch.gather(lp, 1, targets.clamp(min=0)[:, None])[:, 0]
    logprob = torch.where(targets >= 0, at, 0.0)
    ids = torch.sort(z.detach(), dim=-1, descending=True, stable=True).indices[:, :top_k] if top_k else \
        targets.new_zeros(targets.shape[0], 0)
    return logprob, entropy, torch.gather(lp, 1, ids), ids


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] in ("step", "scan", "scan_train"):
        b, l, h, p, n, k = (case[i] for i in ("batch", "length", "heads", "head_dim", "d_state", "groups"))
        acts = b * l * (h * p + 2 * k * n) * e + 2 * b * l * h * 4  # x, B, C, write, log_decay
        y = b * l * h * p * e
        states = b * h * p * n * 4
        total = acts + y + states * (2 if case["carried"] or case["op"] == "step" else 1)
        flops = 5 * b * l * h * p * n  # decay, write and add to the state; multiply and add into y
        if case["op"] == "scan_train":
            total += y + acts + states * (2 if case["carried"] else 1)
            flops += 12 * b * l * h * p * n
        return {"bytes": total, "flops": flops}
    if case["op"] in ("conv", "conv_train"):
        b, l, c, k = (case[i] for i in ("batch", "length", "channels", "taps"))
        row = b * l * c * e
        state = b * (k - 1) * c * e
        total = 2 * row + state * (2 if case["carried"] else 1) + c * (k + 1) * e
        flops = b * l * c * (2 * k + 4)
        if case["op"] == "conv_train":
            total += 2 * row + state * (2 if case["carried"] else 1) + c * (k + 1) * e
            flops *= 3
        return {"bytes": total, "flops": flops}
    r, v, top = case["rows"], case["vocab"], case["top"]
    total = r * v * e + r * (8 + 4 + 4 + 12 * top)
    flops = 5 * r * v
    if case["op"] == "logprobs_train":
        total += r * v * e + r * (8 + 4 * top)
        flops *= 2
    return {"bytes": total, "flops": flops}


# ---- the definition in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("step", "scan", "scan_train"):
            return exact_scan(s)
        if case["op"] in ("conv", "conv_train"):
            return exact_conv(s)
        return exact_logprobs(s)


def exact_scan(s):
    """Token by token; the gradients walk back over states kept for each block of tokens."""
    case = s["case"]
    b, l, h, p, n, k = (case[i] for i in ("batch", "length", "heads", "head_dim", "d_state", "groups"))
    shape = {"x": (b, l, h, p), "B": (b, l, k, n), "C": (b, l, k, n), "write": (b, l, h), "log_decay": (b, l, h)}
    x, B, C, w, la = (s[i].double().reshape(shape[i]) for i in ("x", "B", "C", "write", "log_decay"))
    a = torch.exp(la)
    D = s["D"].double()
    live = torch.ones(b, l, 1, device="cuda", dtype=torch.float64)
    if s.get("lengths") is not None:
        live = (torch.arange(l, device="cuda") < s["lengths"][:, None]).double()[..., None]
    w, a = w * live, a * live + (1 - live)
    st = s["state"].double() if s["state"] is not None else torch.zeros(b, h, p, n, device="cuda",
                                                                       dtype=torch.float64)
    each = h // k

    def advance(st, t):
        add = (w[:, t, :, None] * x[:, t])[..., None] * B[:, t].repeat_interleave(each, 1)[:, :, None]
        return a[:, t, :, None, None] * st + add

    y = torch.empty(b, l, h, p, device="cuda", dtype=torch.float64)
    block, kept = 32, []
    for t in range(l):
        if t % block == 0:
            kept.append(st)
        st = advance(st, t)
        y[:, t] = torch.matmul(st, C[:, t].repeat_interleave(each, 1)[..., None])[..., 0]
    y = (y + D[:, None] * x) * live[..., None]
    if case["op"] == "step":
        return y[:, 0], st
    if case["op"] == "scan":
        return y, st
    dy = s["grads"][0].double() * live[..., None]
    ds = s["grads"][1].double()
    dx, dw, dla = torch.empty_like(x), torch.empty_like(w), torch.empty_like(la)
    dB, dC = torch.empty_like(B), torch.empty_like(C)
    for i in reversed(range(len(kept))):
        first, last = i * block, min(l, (i + 1) * block)
        run_ = [kept[i]]
        for t in range(first, last):
            run_.append(advance(run_[-1], t))
        for t in reversed(range(first, last)):
            Bt, Ct = (v[:, t].repeat_interleave(each, 1) for v in (B, C))
            now, prev = run_[t - first + 1], run_[t - first]
            ds = ds + dy[:, t][..., None] * Ct[:, :, None]
            dC[:, t] = torch.einsum("bhpn,bhp->bhn", now, dy[:, t]).reshape(b, k, each, n).sum(2)
            bx = torch.einsum("bhpn,bhn->bhp", ds, Bt)
            dx[:, t] = w[:, t, :, None] * bx
            dw[:, t] = (bx * x[:, t]).sum(-1)
            dB[:, t] = (w[:, t, :, None] * torch.einsum("bhpn,bhp->bhn", ds, x[:, t])).reshape(b, k, each, n).sum(2)
            dla[:, t] = a[:, t] * (ds * prev).sum((-1, -2))
            ds = a[:, t, :, None, None] * ds
    dx = dx + D[:, None] * dy
    dD = (dy * x).sum((0, 1, 3))
    outs = (y, st, dx, dw * live, dla * live, dB, dC, dD)
    return outs + ((ds,) if s["state"] is not None else ())


def exact_conv(s):
    """Every output as one gathered window times its taps; gradients by scattering the windows back."""
    case = s["case"]
    b, l, c, k = (case[i] for i in ("batch", "length", "channels", "taps"))
    before = s["state"].double() if s["state"] is not None else torch.zeros(b, k - 1, c, device="cuda",
                                                                           dtype=torch.float64)
    row = torch.cat([before, s["x"].double()], 1)
    w, bias = s["weight"].double(), s["bias"].double()
    n = s["lengths"].long() if s["lengths"] is not None else torch.full((b,), l, device="cuda")
    live = (torch.arange(l, device="cuda") < n[:, None]).double()[..., None]
    pre = torch.einsum("blck,ck->blc", row.unfold(1, k, 1), w) + bias
    gate = torch.sigmoid(pre) if case["silu"] else torch.ones_like(pre)
    y = (pre * gate if case["silu"] else pre) * live
    ends = n[:, None] + torch.arange(k - 1, device="cuda")
    rows = torch.arange(b, device="cuda")[:, None]
    outs = (y, row[rows, ends])
    if case["op"] == "conv":
        return outs
    slope = gate * (1 + pre * (1 - gate)) if case["silu"] else gate
    dpre = s["grads"][0].double() * slope * live
    drow = torch.zeros_like(row)
    for i in range(k):
        drow[:, i:i + l] += dpre * w[:, i]
    drow.index_put_((rows, ends), s["grads"][1].double(), accumulate=True)
    dw = torch.stack([(dpre * row[:, i:i + l]).sum((0, 1)) for i in range(k)], -1)
    outs += (drow[:, k - 1:], dw, dpre.sum((0, 1)))
    return outs + ((drow[:, :k - 1],) if s["state"] is not None else ())


def exact_logprobs(s):
    case = s["case"]
    r, top = case["rows"], case["top"]
    parts = []
    for i in range(0, r, 512):
        z = s["logits"][i:i + 512].double()
        t = s["targets"][i:i + 512]
        lp = torch.log_softmax(z, -1)
        prob = torch.exp(lp)
        plp = torch.where(prob > 0, prob * lp, 0.0)
        entropy = -plp.sum(-1)
        used = t >= 0
        logprob = torch.where(used, lp[torch.arange(len(t), device="cuda"), t.clamp(min=0)], 0.0)
        ids = torch.sort(z, dim=-1, descending=True, stable=True)[1][:, :top]
        out = [logprob, entropy, lp.gather(1, ids), ids]
        if case["op"] == "logprobs_train":
            gl = s["grads"][0][i:i + 512].double() * used
            ge = s["grads"][1][i:i + 512].double()
            d = -prob * gl[:, None] - ge[:, None] * (plp + prob * entropy[:, None])
            d[torch.arange(len(t), device="cuda"), t.clamp(min=0)] += gl
            if top:
                gk = s["grads"][2][i:i + 512].double()
                d -= prob * gk.sum(-1, keepdim=True)
                d.scatter_add_(1, ids, gk)
            out.append(d)
        parts.append(out)
    return tuple(torch.cat(v) for v in zip(*parts))
