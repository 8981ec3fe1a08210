"""The attention half of a transformer block and the answers of a classifier or token predictor, as cases that can be timed.

  norm_rotate     queries and keys of every head divided by their root mean square, weighted, and rotated by their positions
  attention       softmax attention with shared key heads, capped scores, a bias by distance, document, causal and prefix masks
  token_logprobs  log probability of a given class in each row of logits, the row's entropy and its most probable classes

`own` is set by the program that times them: true runs the framework's operators, false the same formulas in elementary
PyTorch operations in 32 bits (64 for probabilities next to one).  `exact` states them once more in 64 bits, gradients written out."""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one image of 197 tokens (ViT-S/16 at 224 pixels) in evaluation: a call's latency
        dict(name="norm_vit_s_b1", kind="norm", dtype="fp32", b=1, t=197, h=6, g=6, d=64, rot=64, layout="half", grid=True, train=False),
        # ViT-S training, batch 64, in the network's own fp32; the class token is not rotated
        dict(name="norm_vit_s_train_b64", kind="norm", dtype="fp32", b=64, t=197, h=6, g=6, d=64, rot=64, layout="half", grid=True, train=True),
        # long rows with shared key heads, half of each head rotated in neighbouring pairs
        dict(name="norm_bf16_8192_train", kind="norm", dtype="bf16", b=4, t=8192, h=32, g=8, d=128, rot=64, layout="interleaved", grid=False, train=True),
        # one image in evaluation: latency
        dict(name="attn_vit_s_b1", kind="attn", dtype="bf16", b=1, tq=197, tk=197, h=6, g=6, d=64, cap=30.0, slopes=False, causal=False, prefix=0, docs=0, train=False),
        # ViT-S training, batch 64, exact fp32 scores as the network has them
        dict(name="attn_vit_s_train_b64", kind="attn", dtype="fp32", b=64, tq=197, tk=197, h=6, g=6, d=64, cap=0.0, slopes=False, causal=False, prefix=0, docs=0, train=True),
        # images of many resolutions packed into rows, with padding behind the last one; capped scores
        dict(name="attn_packed_train", kind="attn", dtype="bf16", b=4, tq=4097, tk=4097, h=6, g=6, d=64, cap=50.0, slopes=False, causal=False, prefix=0, docs=11, train=True),
        # token prediction with a prefix that sees itself, shared key heads, bias by distance
        dict(name="attn_prefix_4096_train", kind="attn", dtype="bf16", b=2, tq=4096, tk=4096, h=16, g=4, d=128, cap=0.0, slopes=True, causal=True, prefix=500, docs=0, train=True),
        # the class token alone as query over a long row of patches
        dict(name="attn_one_query_16385", kind="attn", dtype="bf16", b=16, tq=1, tk=16385, h=16, g=4, d=64, cap=0.0, slopes=False, causal=False, prefix=0, docs=0, train=False),
        # long evaluation
        dict(name="attn_fp16_8192", kind="attn", dtype="fp16", b=1, tq=8192, tk=8192, h=16, g=16, d=128, cap=0.0, slopes=False, causal=True, prefix=0, docs=0, train=False),
        # loss and confidence of a 1000-way classifier at batch 64: latency
        dict(name="logp_64x1000_train", kind="logp", dtype="fp32", n=64, c=1000, top=5, train=True),
        # a batch of tokens over an odd number of classes
        dict(name="logp_8192x32001_train", kind="logp", dtype="bf16", n=8192, c=32001, top=5, train=True),
        # few rows, many classes: the answers of a predictor
        dict(name="logp_5x128257", kind="logp", dtype="bf16", n=5, c=128257, top=20, train=False),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(["norm", "attn", "attn", "attn", "logp"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    train = rng.random() < 0.6
    while True:
        g = rng.choice([1, 2, 3, 4, 6, 8])
        h = g * rng.choice([1, 1, 2, 4])
        d = rng.choice([32, 64, 64, 64, 80, 96, 128, 128])
        if kind == "norm":
            case = dict(kind=kind, dtype=dtype, b=_log_uniform(rng, 1, 64), t=_log_uniform(rng, 1, 16384), h=h, g=g, d=d,
                        rot=rng.choice([d, d, d // 2]), layout=rng.choice(["half", "interleaved"]), grid=rng.random() < 0.3, train=train)
            if case["b"] * case["t"] * (h + g) * d >= 500 and work(case)["bytes"] <= 1.3e9:
                return case
        elif kind == "attn":
            tk = _log_uniform(rng, 2 if train else 1, 16384)  # (over one key the gradients of q and k are zero)
            form = rng.choice(["same", "same", "same", "few"])
            tq = tk if form == "same" else min(tk, rng.choice([1, 1, 1, 2, 5, 16]))
            causal = rng.random() < 0.5
            case = dict(kind=kind, dtype=dtype, b=_log_uniform(rng, 1, 64), tq=tq, tk=tk, h=h, g=g, d=d,
                        cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3, causal=causal,
                        prefix=rng.randrange(0, tk) if causal and rng.random() < 0.4 else 0,
                        docs=rng.choice([0, 0, 3, 17]) if tq == tk and tk >= 32 else 0, train=train)
            scores = case["b"] * h * tq * tk
            most = 1.5e8 if dtype == "fp32" else 5e8
            if 1e4 <= scores * d and scores <= most and work(case)["flops"] <= 4.8e11 and work(case)["bytes"] <= 1.3e9:
                return case
        else:
            case = dict(kind=kind, dtype=dtype, n=_log_uniform(rng, 1, 16384), c=_log_uniform(rng, 2, 200000), top=rng.choice([0, 1, 5, 20]),
                        train=train)
            case["top"] = min(case["top"], case["c"])
            if 500 <= case["n"] * case["c"] <= 1.6e8:
                return case


# ---- states ---------------------------------------------------------------------------------------------------------
def _document_lengths(case):
    """Lengths of the documents of one row and, behind them, padding: the same for every seed, so that the work is."""
    rng = random.Random(case["docs"] * 100003 + case["tk"])
    total = case["tk"] - case["tk"] // 50  # the last two per cent are padding
    cuts = sorted(rng.sample(range(1, total), min(case["docs"], total) - 1)) if total > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _rotary_tables(length, rot, dev):
    """cos and sin of position * 10000^(-2i/rot), in 64 bits before they are rounded: what a program makes once."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    angle = torch.arange(length, dtype=torch.float64, device=dev)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def randn(*shape, kind=dtype):
        return torch.randn(*shape, generator=gen, device=dev).to(kind)

    state = dict(case=case)
    if case["kind"] == "norm":
        b, t, h, g, d = (case[k] for k in ("b", "t", "h", "g", "d"))
        # views of one projection's output, as a network has them
        rows = randn(b, t, h + 2 * g, d)
        q, k = rows[:, :, :h], rows[:, :, h:h + g]
        qw, kw = 1 + 0.1 * randn(d, kind=torch.float32), 1 + 0.1 * randn(d, kind=torch.float32)
        cos, sin = _rotary_tables(t, case["rot"], dev)
        # patches by their place, the class token in front of them without one
        positions = (torch.arange(t, device=dev, dtype=torch.int32) - 1).expand(b, t).contiguous() if case["grid"] else None
        state.update(q=q, k=k, qw=qw, kw=kw, cos=cos, sin=sin, positions=positions)
        if case["train"]:
            state.update(gq=randn(b, t, h, d), gk=randn(b, t, g, d))
            for name in ("q", "k", "qw", "kw"):
                state[name] = state[name].detach().requires_grad_(True)
    elif case["kind"] == "attn":
        b, tq, tk, h, g, d = (case[k] for k in ("b", "tq", "tk", "h", "g", "d"))
        if tq == tk:
            rows = randn(b, tk, h + 2 * g, d)
            q, k, v = rows[:, :, :h], rows[:, :, h:h + g], rows[:, :, h + g:]
        else:
            q, k, v = randn(b, tq, h, d), randn(b, tk, g, d), randn(b, tk, g, d)
        state.update(q=q, k=k, v=v)
        state["slopes"] = 2.0 ** (-8.0 * torch.arange(1, h + 1, device=dev, dtype=torch.float32) / h) if case["slopes"] else None
        state["prefix"] = None
        if case["prefix"]:  # rows of a batch have prefixes of their own
            state["prefix"] = (case["prefix"] - torch.arange(b, device=dev, dtype=torch.int32) % 7).clamp_(min=0)
        state["documents"] = None
        if case["docs"]:
            lengths = _document_lengths(case)
            ids = torch.repeat_interleave(torch.arange(len(lengths), dtype=torch.int32), torch.tensor(lengths))
            ids = torch.cat([ids, torch.full((tk - ids.numel(),), -1, dtype=torch.int32)])
            state["documents"] = ids.to(dev).expand(b, tk).contiguous()
        if case["train"]:
            state["g"] = randn(b, tq, h, d)
            for name in ("q", "k", "v"):
                state[name] = state[name].detach().requires_grad_(True)
    else:
        n, c = case["n"], case["c"]
        # one class in each row stands out, as a trained network answers
        logits = torch.randn(n, c, generator=gen, device=dev)
        best = torch.randint(0, c, (n,), generator=gen, device=dev)
        logits[torch.arange(n, device=dev), best] += 8
        targets = torch.where(torch.rand(n, generator=gen, device=dev) < 0.7, best, torch.randint(0, c, (n,), generator=gen, device=dev))
        targets[torch.rand(n, generator=gen, device=dev) < 0.05] = -100  # rows without an answer
        state.update(logits=(2 * logits).to(dtype), targets=targets)
        if case["train"]:
            state["logits"].requires_grad_(True)
            state.update(g_logp=-torch.ones(n, device=dev) / n, g_entropy=0.01 * randn(n, kind=torch.float32) / n)
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _plain_norm_rotate(x, weight, cos, sin, positions, layout):
    half = cos.shape[1]
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6) * weight
    if positions is None:
        c, s = cos[None, :x.shape[1], None], sin[None, :x.shape[1], None]
    else:
        at, moved = positions.clamp(min=0).long(), (positions >= 0)[:, :, None, None]
        c, s = torch.where(moved, cos[at][:, :, None], 1.0), torch.where(moved, sin[at][:, :, None], 0.0)
    if layout == "half":
        a, b = y[..., :half], y[..., half:2 * half]
        return torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * half:]], dim=-1)
    a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2), y[..., 2 * half:]], dim=-1)


def _visible(case, state, dev):
    """[B or 1, 1, Tq, Tk] truth values, or None where everything is seen; the last query stands at the last key."""
    tq, tk = case["tq"], case["tk"]
    at, key = torch.arange(tk - tq, tk, device=dev)[:, None], torch.arange(tk, device=dev)
    seen = None
    if case["causal"]:
        seen = (key <= at)[None, None]
        if state["prefix"] is not None:
            seen = seen | (key < state["prefix"][:, None])[:, None, None]
    if state["documents"] is not None:
        ids = state["documents"]
        same = ((ids[:, :, None] == ids[:, None, :]) & (ids[:, :, None] >= 0))[:, None]
        seen = same if seen is None else seen & same
    return seen


def _plain_attention(case, state, q, k, v):
    b, tq, h, d = q.shape
    tk, g = k.shape[1], k.shape[2]
    q = q.float().permute(0, 2, 1, 3).reshape(b, g, h // g * tq, d)
    k, v = k.float().permute(0, 2, 1, 3), v.float().permute(0, 2, 1, 3)
    s = ((q @ k.transpose(-1, -2)) * (d ** -0.5)).view(b, h, tq, tk)
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    if state["slopes"] is not None:
        away = (torch.arange(tk - tq, tk, device=q.device)[:, None] - torch.arange(tk, device=q.device)).abs().float()
        s = s - state["slopes"][:, None, None] * away
    seen = _visible(case, state, q.device)
    if seen is not None:
        s = torch.where(seen, s, -torch.inf)
    top = s.detach().amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = p.view(b, g, h // g * tq, tk) @ v
    return o.view(b, h, tq, d).permute(0, 2, 1, 3).contiguous()


def _top_keys(x):
    """Values and places as one whole number that orders by value, then by the lower place."""
    bits = (x + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    return bits * (1 << 32) + ((1 << 32) - 1 - torch.arange(x.shape[1], device=x.device))


def _plain_logprobs(logits, targets, top):
    # in 64 bits: where one class has nearly all of the probability, the entropy and the gradient are what is left beside it
    x = logits.double()
    most = x.detach().amax(dim=1, keepdim=True)
    logs = (x - most) - (x - most).exp().sum(dim=1, keepdim=True).log()
    given = targets >= 0
    logp = torch.where(given, logs.gather(1, targets.clamp(min=0)[:, None])[:, 0], 0.0)
    entropy = -(logs.exp() * logs).sum(dim=1)
    keys = torch.topk(_top_keys(logits.detach().float()), top, dim=1)[0]
    at = (1 << 32) - 1 - (keys & 0xFFFFFFFF)
    return logp.float(), entropy.float(), logs.detach().gather(1, at).float(), at


# ---- one pass -------------------------------------------------------------------------------------------------------
def _operators():
    package = os.path.join(os.getcwd(), "appmult-aware-retraining_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import lutgemm_attention
    import lutgemm_loss
    return lutgemm_attention, lutgemm_loss


def run(state):
    case, train = state["case"], state["case"]["train"]
    dtype = _TYPES[case["dtype"]]
    if own:
        attention_ops, loss_ops = _operators()
    with torch.set_grad_enabled(train):
        if case["kind"] == "norm":
            q, k, qw, kw, cos, sin, positions = (state[n] for n in ("q", "k", "qw", "kw", "cos", "sin", "positions"))
            if own:
                yq, yk = attention_ops.norm_rotate(q, k, qw, kw, cos, sin, positions=positions, layout=case["layout"])
            else:
                yq = _plain_norm_rotate(q, qw, cos, sin, positions, case["layout"]).to(dtype)
                yk = _plain_norm_rotate(k, kw, cos, sin, positions, case["layout"]).to(dtype)
            out = {"q": yq.detach(), "k": yk.detach()}
            if train:
                grads = torch.autograd.grad((yq, yk), (q, k, qw, kw), (state["gq"], state["gk"]))
                out.update(zip(("grad_q", "grad_k", "grad_q_weight", "grad_k_weight"), grads))
            return out
        if case["kind"] == "attn":
            q, k, v = state["q"], state["k"], state["v"]
            if own:
                y = attention_ops.attention(q, k, v, cap=case["cap"], slopes=state["slopes"], causal=case["causal"],
                                            prefix=state["prefix"], documents=state["documents"])
            else:
                y = _plain_attention(case, state, q, k, v).to(dtype)
            out = {"out": y.detach()}
            if train:
                out.update(zip(("grad_q", "grad_k", "grad_v"), torch.autograd.grad(y, (q, k, v), state["g"])))
            return out
        logits, targets = state["logits"], state["targets"]
        if own:
            logp, entropy, top, at = loss_ops.token_logprobs(logits, targets, top=case["top"])
        else:
            logp, entropy, top, at = _plain_logprobs(logits, targets, case["top"])
        out = {"logp": logp.detach(), "entropy": entropy.detach(), "top_logp": top, "top_index": at}
        if train:
            out["grad"] = torch.autograd.grad((logp, entropy), logits, (state["g_logp"], state["g_entropy"]))[0]
        return out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def _pairs(case):
    """Query-key pairs that the masks leave, per head and row of the batch."""
    tq, tk = case["tq"], case["tk"]
    first = tk - tq
    if case["docs"]:
        lengths, start, total = _document_lengths(case), 0, 0
        for n in lengths:
            if not case["causal"]:
                total += n * n
            else:  # the causal half, and what of the prefix lies behind a query
                reach = min(max(case["prefix"] - start, 0), n)
                total += n * (n + 1) // 2 + reach * (reach - 1) // 2
            start += n
        return total
    if not case["causal"]:
        return tq * tk
    total = sum(range(first + 1, tk + 1))
    behind = max(0, min(case["prefix"], tk) - first - 1)
    return total + behind * (behind + 1) // 2


def work(case):
    size = _SIZE[case["dtype"]]
    if case["kind"] == "norm":
        values = case["b"] * case["t"] * (case["h"] + case["g"]) * case["d"]
        # x once in, y once out; in training their gradients too
        return {"bytes": float(values * size * (4 if case["train"] else 2)), "flops": float(values * (16 if case["train"] else 6))}
    if case["kind"] == "attn":
        rows, keys = case["b"] * case["tq"] * case["h"] * case["d"], case["b"] * case["tk"] * case["g"] * case["d"]
        # q, k, v in and the result out; in training its gradient in, and three gradients out.  Products of queries and keys
        # and of probabilities and values; the backward pass has five more of the same size
        return {"bytes": float(size * (2 * rows + 2 * keys) * (2 if case["train"] else 1)),
                "flops": (14.0 if case["train"] else 4.0) * case["d"] * case["h"] * case["b"] * _pairs(case)}
    values = case["n"] * case["c"]
    return {"bytes": float(values * size * (2 if case["train"] else 1)), "flops": float(values * (10 if case["train"] else 6))}


# ---- in 64 bits -----------------------------------------------------------------------------------------------------
def _turn(x, cos, sin, layout, back):
    """Rotates pairs of the last axis by the angles, or back."""
    half = cos.shape[-1]
    i = torch.arange(half, device=x.device)
    one, two = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    y = x.clone()
    sign = -1.0 if back else 1.0
    y[..., one] = x[..., one] * cos - sign * x[..., two] * sin
    y[..., two] = x[..., two] * cos + sign * x[..., one] * sin
    return y


def _exact_norm(case, s):
    out = {}
    b, t = case["b"], case["t"]
    at = torch.arange(t, device="cuda").expand(b, t) if s["positions"] is None else s["positions"].long()
    cos, sin = s["cos"].double()[at.clamp(min=0)], s["sin"].double()[at.clamp(min=0)]
    cos[at < 0], sin[at < 0] = 1.0, 0.0
    cos, sin = cos[:, :, None], sin[:, :, None]
    for name in ("q", "k"):
        x, w = s[name].detach().double(), s[name + "w"].detach().double()
        r = 1 / ((x ** 2).sum(-1, keepdim=True) / case["d"] + 1e-6).sqrt()
        unit = x * r
        out[name] = _turn(unit * w, cos, sin, case["layout"], False)
        if case["train"]:
            g = _turn(s["g" + name].double(), cos, sin, case["layout"], True)
            out["grad_%s_weight" % name] = (g * unit).sum((0, 1, 2))
            g = g * w
            out["grad_" + name] = r * (g - unit * (g * unit).sum(-1, keepdim=True) / case["d"])
    return out


def _exact_attention(case, s):
    """One head at a time."""
    b, tq, tk, h, g, d = (case[k] for k in ("b", "tq", "tk", "h", "g", "d"))
    r, cap, scale = h // g, case["cap"], 1 / math.sqrt(d)
    dev = torch.device("cuda")
    place, key = torch.arange(tq, device=dev)[:, None] + tk - tq, torch.arange(tk, device=dev)[None, :]
    away = (place - key).abs().double()
    out = {"out": torch.zeros(b, tq, h, d, dtype=torch.float64, device=dev)}
    if case["train"]:
        out.update({"grad_q": torch.zeros_like(out["out"]), "grad_k": torch.zeros(b, tk, g, d, dtype=torch.float64, device=dev)})
        out["grad_v"] = torch.zeros_like(out["grad_k"])
    step = max(1, int(2e8 // (tq * tk)))  # rows of the batch at a time: 1.6 GB of scores
    for first in range(0, b, step):
        rows = slice(first, first + step)
        hidden = torch.zeros(min(step, b - first), tq, tk, dtype=torch.bool, device=dev)
        if case["causal"]:
            hidden |= key > place
            if s["prefix"] is not None:
                hidden &= key >= s["prefix"][rows, None, None]
        if s["documents"] is not None:
            ids = s["documents"][rows]
            hidden |= (ids[:, place[:, 0], None] != ids[:, None]) | (ids < 0)[:, None]
        for head in range(h):
            q, k, v = (s[n].detach()[rows, :, i].double() for n, i in (("q", head), ("k", head // r), ("v", head // r)))
            score = torch.einsum("bid,bjd->bij", q, k) * scale
            bent = cap * torch.tanh(score / cap) if cap else score
            logit = bent - s["slopes"][head].double() * away if s["slopes"] is not None else bent
            p = torch.softmax(logit.masked_fill(hidden, -math.inf), dim=-1).nan_to_num(0.0)  # rows that see nothing
            del logit
            out["out"][rows, :, head] = torch.einsum("bij,bjd->bid", p, v)
            if not case["train"]:
                continue
            go = s["g"][rows, :, head].double()
            gp = torch.einsum("bid,bjd->bij", go, v)
            out["grad_v"][rows, :, head // r] += torch.einsum("bij,bid->bjd", p, go)
            gs = p * (gp - (p * gp).sum(-1, keepdim=True))
            if cap:
                gs = gs * (1 - (bent / cap) ** 2)
            gs = gs * scale
            out["grad_q"][rows, :, head] = torch.einsum("bij,bjd->bid", gs, k)
            out["grad_k"][rows, :, head // r] += torch.einsum("bij,bid->bjd", gs, q)
    return out


def _exact_logprobs(case, s):
    x = s["logits"].detach().double()
    logs = torch.log_softmax(x, dim=1)
    p = logs.exp()
    given = s["targets"] >= 0
    where = s["targets"].clamp(min=0)[:, None]
    entropy = -(p * logs).sum(1)
    order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :case["top"]]
    out = {"logp": logs.gather(1, where)[:, 0] * given, "entropy": entropy, "top_logp": logs.gather(1, order), "top_index": order}
    if case["train"]:
        gl, ge = (s["g_logp"].double() * given)[:, None], s["g_entropy"].double()[:, None]
        hot = torch.zeros_like(p).scatter_(1, where, 1.0)
        out["grad"] = gl * (hot - p) - ge * p * (logs + entropy[:, None])
    return out


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "attn": _exact_attention, "logp": _exact_logprobs}[case["kind"]](case, state)
