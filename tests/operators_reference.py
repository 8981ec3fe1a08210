"""Head norms with rotation, attention and token log probabilities in 64 bits, from their formulas, gradients by autograd: what
the tests hold the CUDA operators against."""
import torch


def norm_rotate(x, weight, cos, sin, positions, layout, eps):
    """x [B, T, heads, D] in 64 bits."""
    y = x / ((x * x).mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        y = y * weight
    half = 0 if cos is None else cos.shape[1]
    if half == 0:
        return y
    B, T = x.shape[:2]
    at = torch.arange(T, device=x.device).expand(B, T) if positions is None else positions.long()
    keep = (at < 0)[:, :, None, None]
    at = at.clamp(min=0)
    beyond = (at >= cos.shape[0])[:, :, None, None]
    at = at.clamp(max=cos.shape[0] - 1)
    c = torch.where(beyond, torch.nan, torch.where(keep, 1.0, cos.double()[at][:, :, None]))
    s = torch.where(keep, 0.0, sin.double()[at][:, :, None])
    i = torch.arange(half, device=x.device)
    one, two = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    out = y.clone()
    out[..., one] = y[..., one] * c - y[..., two] * s
    out[..., two] = y[..., two] * c + y[..., one] * s
    return out


def visible(B, Tq, Tk, causal, prefix, documents, query_documents, device):
    place = torch.arange(Tk - Tq, Tk, device=device)[:, None]
    key = torch.arange(Tk, device=device)[None, :]
    seen = torch.ones(B, Tq, Tk, dtype=torch.bool, device=device)
    if causal:
        ahead = key <= place
        seen = seen & (ahead if prefix is None else ahead | (key < prefix[:, None, None]))
    if documents is not None:
        dq = query_documents if query_documents is not None else documents[:, Tk - Tq:]
        seen = seen & (dq[:, :, None] == documents[:, None, :]) & (dq[:, :, None] >= 0)
    return seen


def attention(q, k, v, scale=None, cap=0.0, slopes=None, causal=False, prefix=None, documents=None, query_documents=None):
    """q [B, Tq, H, D], k and v [B, Tk, G, D] in 64 bits."""
    B, Tq, H, D = q.shape
    Tk, G = k.shape[1:3]
    if documents is not None:  # padding may hold anything
        dq = query_documents if query_documents is not None else documents[:, Tk - Tq:]
        q = torch.where((dq >= 0)[:, :, None, None], q, 0.0)
        k = torch.where((documents >= 0)[:, :, None, None], k, 0.0)
        v = torch.where((documents >= 0)[:, :, None, None], v, 0.0)
    k, v = k.repeat_interleave(H // G, dim=2), v.repeat_interleave(H // G, dim=2)
    s = torch.einsum("bihd,bjhd->bhij", q, k) * (D ** -0.5 if scale is None else scale)
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        place = torch.arange(Tk - Tq, Tk, device=q.device)[:, None]
        s = s - slopes.double()[:, None, None] * (place - torch.arange(Tk, device=q.device)).abs()
    seen = visible(B, Tq, Tk, causal, prefix, documents, query_documents, q.device)[:, None]
    some = seen.any(-1, keepdim=True)
    p = torch.softmax(torch.where(some, s.masked_fill(~seen, -torch.inf), 0.0), dim=-1)
    return torch.einsum("bhij,bjhd->bihd", torch.where(some, p, 0.0), v)


def token_logprobs(x, targets, top, ignore_index=-100):
    """x [N, C] in 64 bits."""
    logs = torch.log_softmax(x, dim=1)
    given = targets != ignore_index
    logp = torch.where(given, logs.gather(1, targets.clamp(min=0)[:, None])[:, 0], 0.0)
    p = logs.exp()
    entropy = -torch.where(p > 0, p * logs.masked_fill(p == 0, 0.0), 0.0).sum(1)
    order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top]
    return logp, entropy, logs.gather(1, order), order
