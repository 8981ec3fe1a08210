"""Where head norms, attention and log probabilities meet the ends of their types' ranges, rows that are not there, and derivatives
that they do not have; on a GPU."""
import pytest
import torch

import operators_reference as R
from test_gpu_operators import DTYPES, IDS, attention_bounds, close, gen, ops, randn, rounding

pytestmark = pytest.mark.gpu


def logprobs(*args, **kw):
    import lutgemm_loss
    return lutgemm_loss.token_logprobs(*args, **kw)


def check_logprobs(x, targets, top, g_logp, g_entropy):
    """Results and gradients against 64 bits.  Classes farther than 745 below a row's largest have no probability in 64 bits and none in
    32; the others are `spread` apart at most.  Their distances to the largest are exact to f = 2^-24 of themselves, exponentials to
    (spread + 4) f (of a rounded product), sums of positive terms, in runs and trees of at most 512, to 600 f, the logarithm to 4 f."""
    x = x.detach().requires_grad_(True)
    logp, entropy, top_logp, top_index = logprobs(x, targets, top)
    both = torch.autograd.grad((logp, entropy), x, (g_logp, g_entropy), retain_graph=True)[0]
    only = torch.autograd.grad(logp, x, g_logp)[0]
    xd, f, u = x.detach().double(), 2.0 ** -24, rounding(x.dtype)
    want = R.token_logprobs(xd, targets, top)
    assert torch.equal(top_index, want[3])
    m = xd.amax(1)
    near = xd >= m[:, None] - 745
    spread = m - xd.masked_fill(~near, torch.inf).amin(1)
    rel = (2 * spread + 650) * f
    others = (torch.logsumexp(xd, 1) - m).clamp(max=1.0)  # (L is off by at most rel * min(L, 1))
    e_logp = 4 * f * (want[0].abs() + spread + 1) + rel * others
    close(logp, want[0], e_logp, "logp")
    close(entropy, want[1], (rel + 8 * f) * (want[1] + torch.logsumexp(xd, 1) - m) + 1e-30, "entropy")
    close(top_logp, want[2], 4 * f * (want[2].abs() + spread[:, None] + 1) + (rel * others)[:, None], "top_logp")
    logs, p = torch.log_softmax(xd, 1), torch.softmax(xd, 1)
    hot = torch.zeros_like(p).scatter_(1, targets.clamp(min=0)[:, None], 1.0)
    gl, ge = torch.where(targets == -100, 0.0, g_logp.double())[:, None], g_entropy.double()[:, None]
    rest = torch.where(hot > 0, -torch.expm1(logs), -p)
    tail = torch.where(p > 0, p * (logs.masked_fill(p == 0, 0.0) + want[1][:, None]), 0.0)
    per = rel[:, None] + 8 * f  # of a probability
    e = gl.abs() * (rest.abs() + hot * p) * per
    # (below 2^-126 fp32 probabilities are nothing)
    e_both = e + ge.abs() * (tail.abs() * per + p * 8 * f * (spread[:, None] + 1 + want[1][:, None])) + ge.abs() * 2.0 ** -126 * 100
    tiny = (2.0 ** -25 if x.dtype is torch.float16 else 0.0) + 2.0 ** -126 * (1 + gl.abs())
    close(only, gl * rest, u * (gl * rest).abs() + e + tiny, "gradient of logp alone")
    close(both, gl * rest - ge * tail, u * (gl * rest - ge * tail).abs() + e_both + tiny, "gradient")


# rows masked with the type's lowest value, which is not infinite: (rows, classes, which ones are left)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("N,C,left", [(64, 64, "half"), (9, 40, "three"), (700, 1000, "half"), (5, 5000, "half"), (3, 32001, "three"),
                                      (2500, 1024, "three"), (1, 128257, "start"), (2, 200003, "end"), (3, 100001, "three")])
def test_logits_masked_with_the_lowest_value(N, C, left, dtype):
    g = gen(N + C)
    x = (2 * randn(g, N, C)).to(dtype)
    if left == "half":
        keep = torch.rand(N, C, generator=g, device="cuda") < 0.5
    else:
        keep = torch.zeros(N, C, dtype=torch.bool, device="cuda")
        if left == "three":
            keep.scatter_(1, torch.randint(0, C, (N, 3), generator=g, device="cuda"), True)
        elif left == "start":  # whole parts of the row are masked
            keep[:, :100] = True
        else:
            keep[:, -100:] = True
    keep[:, C // 3] = keep[:, C // 3] | ~keep.any(1)
    x = torch.where(keep, x, torch.finfo(dtype).min)
    targets = x.float().argmax(1)
    targets[1::2] = torch.randint(0, C, (N,), generator=g, device="cuda")[1::2]  # (masked ones among them)
    targets[2::5] = -100
    check_logprobs(x, targets, min(3, C), randn(g, N), randn(g, N))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("C", [33, 40000])
def test_large_gradients_of_entropies_beside_classes_without_probability(C, dtype):
    g = gen(C)
    x = (2 * randn(g, 6, C)).to(dtype)
    x[torch.rand(6, C, generator=g, device="cuda") < 0.3] = -torch.inf
    x = x.requires_grad_(True)
    entropy = logprobs(x, torch.zeros(6, dtype=torch.int64, device="cuda"))[1]
    one = torch.autograd.grad(entropy, x, torch.ones(6, device="cuda"), retain_graph=True)[0]
    # (a gradient is a product of g_entropy, so a power of two beyond it changes exponents alone; fp16 has no room for them)
    many = torch.autograd.grad(entropy, x, torch.full((6,), 2.0 ** 40, device="cuda"))[0]
    hidden = x.detach() == -torch.inf
    assert not many[hidden].any()
    if dtype is not torch.float16:
        assert torch.equal(many, one * 2.0 ** 40)


# (B, T, H, G, D, rot, layout, type): groups of lanes without a head in the last turn, heads that do not fill a turn, loads that run ahead
@pytest.mark.parametrize("B,T,H,G,D,rot,layout,dtype", [
    (1, 197, 6, 6, 64, 64, "half", torch.float32), (1, 1, 1, 1, 8, 8, "half", torch.float32), (3, 33, 8, 2, 128, 64, "interleaved", torch.bfloat16),
    (2, 1031, 5, 3, 64, 32, "half", torch.float16), (1, 13, 3, 1, 254, 254, "half", torch.float32), (2, 65, 4, 1, 80, 40, "half", torch.bfloat16),
    (2, 8195, 17, 5, 128, 64, "interleaved", torch.bfloat16), (1, 20011, 7, 8, 80, 40, "half", torch.float32),
    (3, 5003, 21, 3, 128, 128, "half", torch.float16)])
def test_norms_without_eps(B, T, H, G, D, rot, layout, dtype):
    g = gen(B + T + D)
    q, k = (randn(g, B, T, n, D, dtype=dtype).requires_grad_(True) for n in (H, G))
    qw, kw = ((1 + 0.2 * randn(g, D)).requires_grad_(True) for _ in range(2))
    cos, sin = ops().rotary_tables(T, rot, device="cuda")
    go = [randn(g, B, T, n, D, dtype=dtype) for n in (H, G)]
    y = ops().norm_rotate(q, k, qw, kw, cos, sin, layout=layout, eps=0.0)
    grads = torch.autograd.grad(y, (q, k, qw, kw), go)
    u, f = rounding(dtype), 2.0 ** -24
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        xd, wd = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
        want = R.norm_rotate(xd, wd, cos, sin, None, layout, 0.0)
        wx, ww = torch.autograd.grad(want, (xd, wd), go[i].double())
        want, xd, god = want.detach(), xd.detach(), go[i].double()
        # D/2 + 12 roundings of fp32 for a value, each of at most the largest of its head, and one of the type
        close(y[i].detach(), want, u * want.abs() + (D + 24) * f * want.abs().amax(-1, keepdim=True), "y")
        r = 1 / xd.square().mean(-1, keepdim=True).sqrt()
        unit, most = xd * r, god.abs().amax(-1, keepdim=True) * 2 * wd.detach().abs().max()
        close(grads[i], wx, u * wx.abs() + (D + 24) * f * r * most * (1 + unit.abs().amax(-1, keepdim=True) ** 2), "grad_x")
        n = B * T * x.shape[2]
        terms = (2 * god.abs().amax(-1, keepdim=True) * unit.abs()).sum((0, 1, 2))
        close(grads[2 + i], ww, (min(n, 4096) + D + 24) * f * terms, "grad_w")


def test_forward_mode_derivatives_are_refused():
    """There are none, and a result without its tangent would be taken for one whose derivative is zero."""
    import torch.autograd.forward_ad as forward_mode
    g = gen(31)
    q, k, v, w = randn(g, 1, 5, 2, 16), randn(g, 1, 5, 2, 16), randn(g, 1, 5, 2, 16), torch.ones(16, device="cuda")
    cos, sin = ops().rotary_tables(5, 16, device="cuda")
    x, t, slopes = randn(g, 5, 9), torch.arange(5, device="cuda"), torch.ones(2, device="cuda")
    norm = dict(q=q, k=k, q_weight=w, k_weight=w, cos=cos, sin=sin)
    attention = dict(q=q, k=k, v=v, slopes=slopes)
    plain = [ops().norm_rotate(**norm)[0], ops().attention(**attention), logprobs(x, t)[0]]
    learned = q.clone().requires_grad_(True)
    with forward_mode.dual_level():
        def dual(y):
            return forward_mode.make_dual(y, torch.ones_like(y))
        for grads in (torch.enable_grad, torch.no_grad):
            with grads():
                for name in norm:
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        ops().norm_rotate(**{**norm, name: dual(norm[name])})
                for name in attention:
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        ops().attention(**{**attention, name: dual(attention[name])})
                with pytest.raises(RuntimeError, match="forward-mode"):
                    ops().attention(dual(q), k[:, :0], v[:, :0])  # nothing to see
                with pytest.raises(RuntimeError, match="forward-mode"):
                    logprobs(dual(x), t)
                # tensors without a tangent, and a primal, are as they were
                same = [ops().norm_rotate(**norm)[0], ops().attention(**attention), logprobs(forward_mode.unpack_dual(dual(x)).primal, t)[0]]
                assert all(torch.equal(a, b) for a, b in zip(same, plain))
        # a gradient that carries a tangent
        go = dual(q.clone())
        for y, leaf, grad in ((ops().norm_rotate(learned, k)[0], learned, go), (ops().attention(learned, k, v), learned, go),
                              (logprobs(learned.view(10, 16), torch.zeros(10, dtype=torch.int64, device="cuda"))[0], learned,
                               dual(torch.ones(10, device="cuda")))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, grad)


def test_losses_leave_out_ignored_labels():
    """The fused loss is F.cross_entropy, whose mean is over the labels that are not -100; so are the figures of an evaluation."""
    import copy
    import torch.nn.functional as F
    from lutgemm_dp import OverlappedGradReducer
    from lutgemm_train import evaluate_top, train_step
    torch.manual_seed(5)
    model = torch.nn.Linear(20, 30).cuda()
    other, exact = copy.deepcopy(model), copy.deepcopy(model).double()
    g = gen(32)
    x, y = randn(g, 64, 20), torch.randint(0, 30, (64,), generator=g, device="cuda")
    f = 2.0 ** -24
    for ignored in (0, 21, 63):
        y[:ignored] = -100
        want = F.cross_entropy(exact(x.double()), y)
        wants = torch.autograd.grad(want, list(exact.parameters()))
        for net, fused in ((model, True), (other, False)):
            opt = torch.optim.SGD(net.parameters(), lr=0.0)
            loss = train_step(net, opt, OverlappedGradReducer(net.parameters()), x, y, fused_loss=fused)
            # logits: 21 roundings of at most 20 terms of up to 1; log probabilities of 30 classes of spread below 16 and a mean of
            # 64: 1000 roundings are far more than any term of the loss or of a gradient (at most 64 times 5) has seen
            assert abs(loss.item() - want.item()) <= 1000 * f * (1 + want.item())
            for p, w in zip(net.parameters(), wants):
                assert (p.grad - w).abs().max().item() <= 1000 * f * 5
        found = evaluate_top(model, [(x, y), (x[:7], y[:7])], top=3)
        xs, ys = torch.cat([x, x[:7]]), torch.cat([y, y[:7]])
        logits, ys = exact(xs.double())[ys != -100], ys[ys != -100]
        p = torch.softmax(logits, 1)
        best = logits.topk(3, 1)[1] == ys[:, None]
        for name, value in (("top1", best[:, 0].double().mean()), ("top3", best.sum(1).double().mean()), ("nll", F.cross_entropy(logits, ys)),
                            ("entropy", -(p * p.log()).sum(1).mean())):
            assert abs(found[name] - value.item()) <= 1000 * f * (1 + value.item()), name
    y[:] = -100
    assert evaluate_top(model, [(x, y)], top=3) == dict(top1=0.0, top3=0.0, nll=0.0, entropy=0.0)


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
def test_biases_by_distance_beyond_24_bits_of_place(dtype):
    """Places of 2^24 and more are no longer whole numbers of fp32; distances of near keys have to be."""
    g, T, n = gen(34), 2 ** 24 + 333, 2048
    k, v = (torch.zeros(1, T, 1, 8, dtype=dtype, device="cuda") for _ in range(2))
    for x in (k, v):
        x[:, -n:] = randn(g, 1, n, 1, 8, dtype=dtype)
    q, go = randn(g, 1, 5, 1, 8, dtype=dtype), randn(g, 1, 5, 1, 8, dtype=dtype)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    slopes = torch.tensor([0.7], device="cuda")  # (2048 places away nothing is left: exp(-1400))
    out = ops().attention(*leaves, slopes=slopes)
    got = [out.detach(), *torch.autograd.grad(out, leaves, go)]
    case = [q, k.detach()[:, -n:], v.detach()[:, -n:]]
    want, tol = attention_bounds(*case, go, dict(slopes=slopes), dtype)
    tiny = 0.0 if dtype is not torch.float16 else 2.0 ** -24 * 40  # (as in test_attention: subnormal results and probabilities)
    for name, x, w, t in zip(("out", "grad_q", "grad_k", "grad_v"), got, want, tol):
        if x.shape[1] == T:
            assert not x[:, :-n].any(), name
            x = x[:, -n:]
        close(x, w, t + tiny, name)


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("D", [64, 72])
def test_attention_beside_the_largest_values_of_a_type(D, dtype):
    """Another document's values of +-finfo.max in the same tile are finite, and a probability of zero hides them."""
    g = gen(35 + D)
    ids = torch.zeros(1, 70, dtype=torch.int32, device="cuda")
    ids[:, 31:50] = 1
    other, kw = ids[0] == 1, dict(documents=ids, cap=20.0)
    near = [randn(g, 1, 70, 2, D, dtype=dtype) for _ in range(4)]
    for x in near[1:]:
        x[:, other] = 0.0
    want, tol = attention_bounds(*near, kw, dtype)
    for filler in (torch.finfo(dtype).max, torch.finfo(dtype).min):
        xs = [x.clone() for x in near]
        for x in xs[1:]:
            x[:, other] = filler
        leaves = [x.requires_grad_(True) for x in xs[:3]]
        out = ops().attention(*leaves, **kw)
        got = [out.detach(), *torch.autograd.grad(out, leaves, xs[3])]
        for name, x, w, t in zip(("out", "grad_q", "grad_k", "grad_v"), got, want, tol):
            close(x[:, ~other], w[:, ~other], t[:, ~other], name)


def test_attention_of_the_largest_fp32_values():
    """Beyond the largest bf16 value, where a first plane of 16 bits would round to infinity."""
    g = gen(36)
    q, k = randn(g, 1, 5, 1, 64), randn(g, 1, 1, 1, 64)
    v = torch.full((1, 1, 1, 64), torch.finfo(torch.float32).max, device="cuda")
    v[..., ::2] *= -1 + 2.0 ** -9
    # one key: its probability is one, whose products with three planes and sum are off by a rounding each, 2^-22 in all
    out = ops().attention(q, k, v).double()
    want = v.double().expand(1, 5, 1, 64)
    assert ((out - want).abs() <= 2.0 ** -22 * want.abs()).all()


def score_gradients(q, k, v, go, **kw):
    """p, p (gp - delta) and gp in 64 bits, [B, H, Tq, Tk]; heads of their own, no cap, no bias."""
    qd, kd, vd, god = (x.detach().double() for x in (q, k, v, go))
    seen = R.visible(q.shape[0], q.shape[1], k.shape[1], kw.get("causal", False), None, kw.get("documents"), None, q.device)[:, None]
    s = torch.einsum("bihd,bjhd->bhij", qd, kd) * q.shape[3] ** -0.5
    p = torch.softmax(s.masked_fill(~seen, -torch.inf), -1)
    gp = torch.einsum("bihd,bjhd->bhij", god, vd)
    return p, p * (gp - (p * gp).sum(-1, keepdim=True)), gp


# gradients of very different sizes, or values that are large: one row's beside the others', one document's, all of them tiny
@pytest.mark.parametrize("form", ["one row", "causal", "tiny", "large values", "document"])
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_score_gradients_of_uneven_rows(form, D):
    """dS = p (gp - delta) is rounded to fp16, in units that keep it normal: by row for grad_q, by block of keys for grad_k."""
    g, T, H = gen(33 + D), 4096 if form != "large values" else 50, 1
    q, k, v = (randn(g, 1, T, H, D, dtype=torch.float16).requires_grad_(True) for _ in range(3))
    go = randn(g, 1, T, H, D)
    kw = {}
    big = slice(T // 2, T // 2 + 1)
    if form in ("one row", "causal"):
        go[:, big] *= 2.0 ** 13
        kw = dict(causal=form == "causal")
    elif form == "document":  # (the last tile of the first document holds rows of the second)
        ids = torch.zeros(1, T, dtype=torch.int32, device="cuda")
        ids[:, 1000:] = 1
        go[:, 1000:] *= 2.0 ** 12
        kw = dict(documents=ids)
        big = slice(1000, T)
    elif form == "tiny":
        go[:, :T // 2] *= 2.0 ** -9
        big = slice(T // 2, T)
    else:
        sign = 1.0 - 2.0 * (torch.arange(T, device="cuda") % 2)
        with torch.no_grad():
            q.mul_(2.0)  # (rows have a few probable keys)
            v[..., :16] = 60000.0 * sign[:, None, None]  # gp is beyond fp16, in units of the largest gradient too
        go[..., :16] = 2.0
        go *= 2.0 ** -11
    go = go.half()
    got = torch.autograd.grad(ops().attention(q, k, v, **kw), (q, k, v), go)
    qd, kd, vd = (x.detach().double().requires_grad_(True) for x in (q, k, v))
    wants = torch.autograd.grad(R.attention(qd, kd, vd, **kw), (qd, kd, vd), go.double())
    p, gs, gp = score_gradients(q, k, v, go, **kw)
    u, f, scale = 2.0 ** -11, 2.0 ** -24, D ** -0.5
    # a term: its rounding u, the relative error of p (scores of up to 2^6 by exp2 and sums of T terms), gp and delta by D products of
    # fp32; delta besides by the errors of out, whose probabilities were rounded, and sums of T products, each of 2 f or less
    most = torch.einsum("bihd,bjhd->bhij", go.double().abs(), vd.detach().abs())
    off = (u + (2 * D + T + 64) * 2 * f)
    e = gs.abs() * off + p * ((D + 8) * f * most + (p * most).sum(-1, keepdim=True) * off)
    # what lies below fp16's normal range is off by 2^-25 units; a row's unit is at most 2^-14 of a bound of its terms, sqrt of the two
    # sums of squares and delta, and a block of keys' the largest of its rows'
    length = go.double().square().sum(-1).sqrt().transpose(1, 2)  # [B, H, T]
    longest = vd.detach().square().sum(-1).sqrt().amax(1)[..., None]
    bound = (length * longest + (p * gp).sum(-1).abs()) * 2.0 ** -39

    def check(name, got, want, terms, least, with_, spec, rows):
        tol = torch.einsum(spec, terms + least, with_.detach().abs()) * scale + u * want.abs() + 2.0 ** -25
        close(got[:, rows], want[:, rows], tol[:, rows], name)
    everything = slice(0, T)
    check("grad_q", got[0], wants[0], e, bound[..., None] * p.gt(0), kd, "bhij,bjhd->bihd", everything)
    check("grad_k", got[1], wants[1], e, bound.amax(-1)[..., None, None] * p.gt(0), qd, "bhij,bihd->bjhd", everything)


# (B, Tq, Tk, H): keys in one part, keys split over blocks and joined
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("B,Tq,Tk,H", [(2, 100, 100, 4), (32, 1, 1024, 4)])
def test_gradients_use_the_unrounded_result(B, Tq, Tk, H, dtype):
    """Two equal keys share a query's probability, and their values are neighbours in the operands' type: the result lies between them.
    A score's gradient p (gp - delta) is then the difference of near values, and delta from the rounded result would be off by as much."""
    D, g = 64, gen(37 + Tk)
    k, v = (randn(g, B, Tk // 2, H, D) for _ in range(2))
    k = (8 * k / k.norm(dim=-1, keepdim=True)).to(dtype).repeat_interleave(2, dim=1)
    v = torch.where(v.abs() < 2.0 ** -6, 1.0, v).to(dtype).repeat_interleave(2, dim=1)
    v[:, 1::2] = (v[:, 1::2].contiguous().view(torch.int16) + 1).view(dtype)
    at = 2 * torch.randint(0, Tk // 2, (B, Tq, H), generator=g, device="cuda")
    q = (3 * k.gather(1, at[..., None].expand(B, Tq, H, D))).requires_grad_(True)
    go = randn(g, B, Tq, H, D, dtype=dtype)
    got = torch.autograd.grad(ops().attention(q, k, v), q, go)[0]
    qd, kd, vd, god = (x.detach().double() for x in (q, k, v, go))
    qd.requires_grad_(True)
    want = R.attention(qd, kd, vd)
    grad = torch.autograd.grad(want, qd, god)[0]
    want, u, f, scale = want.detach(), rounding(dtype), 2.0 ** -24, D ** -0.5
    s = torch.einsum("bihd,bjhd->bhij", qd.detach(), kd) * scale
    p = torch.softmax(s, -1)
    peak = p > 0.25
    rest = p.masked_fill(peak, 0.0)
    # both keys are more than 8 above everything else in log 2, so their P are relative to themselves: one up to f |s| log2 e, which is
    # rounded away; the sum of unrounded P keeps it
    assert (peak.sum(-1) == 2).all() and (rest.amax(-1) < p.amax(-1) * 2.0 ** -8).all()
    most = torch.einsum("bihd,bjhd->bhij", qd.detach().abs(), kd.abs()) * scale
    off = (D + 8) * f * most + 16 * f * s.abs() + 60 * f
    # out: errors of the other probabilities, relative to themselves, by any two values; of the sum; of a part's sums of products (256
    # keys at most, cut off or rounded) and the joining of parts; the rest of the rounding is itself rounded, by u^2
    both = rest * (off + off.amax(-1, keepdim=True) + u)
    assert vd.abs().max() <= 8
    e_out = 16 * both.sum(-1)[..., None].transpose(1, 2) + want.abs() * u * u + want.abs() * f * (
        2 * (min(Tk, 256) + 64) + 16 + 2 * s.abs().amax(-1)[..., None].transpose(1, 2)) + (2.0 ** -25 if dtype is torch.float16 else 0.0)
    gp = torch.einsum("bihd,bjhd->bhij", god, vd)
    gp_most = torch.einsum("bihd,bjhd->bhij", god.abs(), vd.abs())
    delta = (p * gp).sum(-1, keepdim=True)
    e_delta = torch.einsum("bihd,bihd->bhi", god.abs(), e_out + D * f * want.abs())[..., None]
    gs = p * (gp - delta)
    e_gs = gs.abs() * (off + off.amax(-1, keepdim=True) + u + 8 * f + 2 * (Tk + 64) * f) + p * ((D + 8) * f * gp_most + e_delta)
    if dtype is torch.float16:  # dS below fp16's normal range: 2^-25 of a unit, which is at most 2^-14 of |grad_o| |v| + |delta|
        bound = god.norm(dim=-1).transpose(1, 2) * vd.norm(dim=-1).amax(1)[..., None] + delta[..., 0].abs()
        e_gs = e_gs + 2.0 ** -39 * bound[..., None]
    tol = torch.einsum("bhij,bjhd->bihd", e_gs, kd.abs()) * scale + u * grad.abs() + (2.0 ** -25 if dtype is torch.float16 else 0.0)
    # delta from the rounded result would not pass
    rounded = torch.einsum("bihd,bihd->bhi", god, want.to(dtype).double())[..., None]
    planted = grad - torch.einsum("bhij,bjhd->bihd", p * (rounded - delta), kd) * scale
    assert ((planted - grad).abs() > 2 * tol).any()
    close(got, grad, tol, "grad_q")
