"""The plaintext Mamba-2 operators from their definitions in float64, token by
token, with autograd gradients: what the GPU tests compare with."""
import torch


def scan(x, write, log_decay, B, C, D=None, state=None, lengths=None):
    b, l, h, p = x.shape
    k, n = B.shape[2], B.shape[3]
    s = state if state is not None else x.new_zeros(b, h, p, n)
    ys = []
    for t in range(l):
        Bt, Ct = (v[:, t].repeat_interleave(h // k, 1) for v in (B, C))
        new = torch.exp(log_decay[:, t])[..., None, None] * s + \
            (write[:, t][..., None] * x[:, t])[..., None] * Bt[:, :, None]
        y = (new * Ct[:, :, None]).sum(-1)
        if D is not None:
            y = y + D[:, None] * x[:, t]
        if lengths is not None:
            live = (t < lengths)[:, None, None]
            y = torch.where(live, y, 0.0)
            new = torch.where(live[..., None], new, s)
        ys.append(y)
        s = new
    return (torch.stack(ys, 1) if l else x.new_zeros(b, 0, h, p)), s


def conv(x, weight, bias=None, state=None, lengths=None, silu=True):
    b, l, c = x.shape
    k = weight.shape[1]
    row = torch.cat([state if state is not None else x.new_zeros(b, k - 1, c), x], 1)
    y = sum(weight[:, i] * row[:, i:i + l] for i in range(k))
    if bias is not None:
        y = y + bias
    if silu:
        y = y * torch.sigmoid(y)
    n = lengths.long() if lengths is not None else torch.full((b,), l, device=x.device)
    y = torch.where((torch.arange(l, device=x.device) < n[:, None])[..., None], y, 0.0)
    last = n[:, None] + torch.arange(k - 1, device=x.device)
    return y, torch.gather(row, 1, last[..., None].expand(b, k - 1, c))


def logprobs(z, targets, top_k=0):
    """NaN and +inf free logits; rows of -inf alone give log-probabilities -inf and entropy 0."""
    m = z.max(-1, keepdim=True).values
    m = torch.where(m == -torch.inf, 0.0, m)
    e = torch.exp(z - m)
    total = e.sum(-1, keepdim=True)
    lp = torch.where(total > 0, z - m - torch.log(total), -torch.inf)
    prob = torch.where(total > 0, e / total.clamp(min=1e-300), 0.0)
    entropy = -torch.where(prob > 0, prob * torch.where(prob > 0, lp, 0.0), 0.0).sum(-1)
    at = torch.gather(lp, 1, targets.clamp(0, z.shape[1] - 1)[:, None])[:, 0]
    logprob = torch.where(targets >= 0, at, 0.0)
    ids = torch.sort(z.detach(), dim=-1, descending=True, stable=True).indices[:, :top_k]
    return logprob, entropy, torch.gather(lp, 1, ids), ids
