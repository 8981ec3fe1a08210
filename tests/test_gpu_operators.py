"""Head norms with rotation, attention and token log probabilities against their formulas in 64 bits, on a GPU.

Tolerances count roundings.  u = finfo(type).eps / 2 is the most a value is off when it is rounded to a type; every operator rounds
its results once, and attention of 16-bit operands rounds probabilities and score gradients to the operands' type on the way
(each an error of u of the term it stands in).  Sums are fp32: n terms are off by at most n * 2^-24 of the sum of their magnitudes."""
import pytest
import torch

import operators_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


def ops():
    import lutgemm_attention
    return lutgemm_attention


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def rounding(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, tol, what):
    """|got - want| <= tol elementwise, equal where want is not finite; tol: a number or a tensor."""
    got = got.double()
    assert got.shape == want.shape, what
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)]), what
    over = torch.where(odd, torch.zeros_like(want), (got - want).abs() - tol)
    assert over.max().item() <= 0 if over.numel() else True, f"{what}: {over.max().item():.3g} beyond the tolerance at {over.argmax().item()}"


# ---- norm_rotate -----------------------------------------------------------------------------------------------------------
# (B, T, H, G, D, rot, layout, with positions)
NORM = [
    (1, 1, 1, 1, 2, 2, "half", False), (2, 7, 6, 6, 64, 64, "half", True), (1, 197, 6, 6, 64, 64, "half", True),
    (3, 33, 8, 2, 128, 64, "interleaved", False), (2, 65, 4, 1, 80, 40, "half", True), (2, 9, 3, 3, 96, 48, "interleaved", True),
    (1, 5, 2, 2, 256, 256, "half", False), (1, 5, 2, 1, 256, 130, "interleaved", False), (2, 11, 5, 5, 30, 6, "half", False),
    (2, 3, 2, 2, 64, 0, "half", False), (2, 1031, 12, 4, 64, 32, "half", True), (1, 4099, 16, 4, 128, 128, "interleaved", False),
    (1, 13, 3, 1, 254, 254, "half", False),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,T,H,G,D,rot,layout,place", NORM)
def test_norm_rotate(B, T, H, G, D, rot, layout, place, dtype):
    g = gen(B * 1000 + T + D)
    rows = randn(g, B, T, H + 2 * G + 1, D, dtype=dtype)
    q, k = rows[:, :, :H].detach().requires_grad_(True), rows[:, :, H:H + G].detach().requires_grad_(True)
    qw, kw = (1 + 0.2 * randn(g, D)).requires_grad_(True), (1 + 0.2 * randn(g, D)).requires_grad_(True)
    cos, sin = ops().rotary_tables(T + 3, rot, device="cuda") if rot else (None, None)
    positions = torch.randint(-1, T + 3, (B, T), generator=g, device="cuda", dtype=torch.int32) if place else None
    gq, gk = randn(g, B, T, H, D, dtype=dtype), randn(g, B, T, G, D, dtype=dtype)
    yq, yk = ops().norm_rotate(q, k, qw, kw, cos, sin, positions, layout)
    grads = torch.autograd.grad((yq, yk), (q, k, qw, kw), (gq, gk))
    u, f = rounding(dtype), 2.0 ** -24
    for x, w, y, go, gx, gw in ((q, qw, yq, gq, grads[0], grads[2]), (k, kw, yk, gk, grads[1], grads[3])):
        xd, wd = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
        want = R.norm_rotate(xd, wd, cos, sin, positions, layout, 1e-6)
        wx, ww = torch.autograd.grad(want, (xd, wd), go.double())
        assert y.dtype is dtype and y.is_contiguous() and gx.dtype is dtype
        want = want.detach()
        # a value is a turned pair of two products of three factors: D/2 + 12 roundings of fp32, and one of the type
        pair = want.abs().amax(-1, keepdim=True)
        close(y, want, u * want.abs() + (D + 24) * f * pair + 1e-30, "y")
        # grad_x: r * (g w - n mean(g w n)): terms as large as r * max|g w n^2|
        r = 1 / (xd.detach().square().mean(-1, keepdim=True) + 1e-6).sqrt()
        size = r * (go.double().abs().amax(-1, keepdim=True) * 1.5 * 2) * (1 + (xd.detach() * r).abs().amax(-1, keepdim=True) ** 2)
        close(gx, wx, u * wx.abs() + (D + 24) * f * size, "grad_x")
        n = B * T * x.shape[2]
        unit = xd.detach() * r
        terms = (go.double().abs().amax(-1, keepdim=True) * 1.5 * unit.abs()).sum((0, 1, 2))
        close(gw, ww, (min(n, 4096) + D + 24) * f * terms + 1e-30, "grad_w")


def test_norm_rotate_positions_beyond_the_table_and_other_forms():
    g = gen(1)
    q, k = randn(g, 2, 5, 2, 8), randn(g, 2, 5, 1, 8)
    cos, sin = ops().rotary_tables(5, 4, device="cuda")
    positions = torch.tensor([[0, 1, 5, -7, 4], [2 ** 40, 3, 2, 1, -1]], device="cuda")
    yq, yk = ops().norm_rotate(q, k, None, None, cos, sin, positions)
    for y, x in ((yq, q), (yk, k)):
        want = R.norm_rotate(x.double(), None, cos, sin, positions, "half", 1e-6)
        assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.isnan(y[0, 2, :, :4]).all() and torch.isfinite(y[0, 2, :, 4:]).all()
        close(y, want, 40 * 2.0 ** -24 * 3, "y")
    # 16-bit weights come back in their type, frozen ones not at all
    w = torch.ones(8, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    q.requires_grad_(True)
    yq, yk = ops().norm_rotate(q, k, w, torch.ones(8, device="cuda"), cos, sin)
    (yq.sum() + yk.sum()).backward()
    assert w.grad.dtype is torch.bfloat16 and q.grad.shape == q.shape
    # strides that allow no vectors, an expanded operand, a gradient in another order
    base = randn(g, 2, 5, 3, 9)
    odd = base[..., 1:]
    yq, _ = ops().norm_rotate(odd, k, None, None, cos, sin)
    close(yq, R.norm_rotate(odd.double(), None, cos, sin, None, "half", 1e-6), 40 * 2.0 ** -24 * 3, "unaligned")
    wide = randn(g, 1, 5, 1, 8).expand(2, 5, 4, 8)
    yq, _ = ops().norm_rotate(wide, k, None, None, cos, sin)
    close(yq, R.norm_rotate(wide.double(), None, cos, sin, None, "half", 1e-6), 40 * 2.0 ** -24 * 3, "expanded")
    x = randn(g, 2, 5, 2, 8).requires_grad_(True)
    yq, yk = ops().norm_rotate(x, k, None, None, cos, sin)
    go = randn(g, 2, 5, 8, 2).transpose(2, 3)
    got = torch.autograd.grad(yq, x, go)[0]
    xd = x.detach().double().requires_grad_(True)
    want = torch.autograd.grad(R.norm_rotate(xd, None, cos, sin, None, "half", 1e-6), xd, go.double())[0]
    close(got, want, 40 * 2.0 ** -24 * 20, "transposed gradient")
    # nothing to do
    empty, _ = ops().norm_rotate(torch.empty(0, 3, 2, 8, device="cuda"), torch.empty(0, 3, 1, 8, device="cuda"), None, None, cos, sin)
    assert empty.shape == (0, 3, 2, 8)


def test_norm_rotate_gradient_against_differences():
    g = gen(5)
    q, k = randn(g, 1, 3, 2, 16), randn(g, 1, 3, 1, 16)
    w = 1 + 0.1 * randn(g, 16)
    cos, sin = ops().rotary_tables(3, 16, device="cuda")
    go, step = randn(g, 1, 3, 2, 16), randn(g, 1, 3, 2, 16)
    x = q.clone().requires_grad_(True)
    grad = torch.autograd.grad(ops().norm_rotate(x, k, w, w, cos, sin)[0], x, go)[0]
    h = 2.0 ** -7

    def value(t):
        return (ops().norm_rotate(q + t * step, k, w, w, cos, sin)[0].double() * go.double()).sum().item()
    slope = (value(h) - value(-h)) / (2 * h)
    # central difference: h^2/6 of the third derivative (of order 50 for sums of 96 terms of order one), and 2^-24 * 100 / h of rounding
    assert abs(slope - (grad.double() * step.double()).sum().item()) <= h * h / 6 * 500 + 2.0 ** -24 * 100 / h


@pytest.mark.parametrize("change,match", [
    (dict(q="cpu"), "CUDAtensor"), (dict(q="int"), "of type"), (dict(k="half"), "of type"), (dict(q="3d"), "B, T, heads, D"),
    (dict(k="short"), "expected"), (dict(layout="rows"), "layout"), (dict(sin=None), "belong together"), (dict(cos="long"), "at most"),
    (dict(cos="few"), "positions"), (dict(w="short"), "expected"), (dict(w="int"), "of type"), (dict(positions="float"), "of type"),
    (dict(positions="short"), "expected"), (dict(q="odd"), "even size"), (dict(q="wide"), "even size")])
def test_norm_rotate_refuses(change, match):
    g = gen(2)
    q, k, w = randn(g, 2, 5, 2, 8), randn(g, 2, 5, 1, 8), torch.ones(8, device="cuda")
    cos, sin = ops().rotary_tables(5, 8, device="cuda")
    positions, layout = None, "half"
    kind = change.get("q")
    q = {"cpu": lambda: q.cpu(), "int": lambda: q.int(), "3d": lambda: q[0], "odd": lambda: q[..., :7], "wide": lambda: randn(g, 2, 5, 2, 300)}.get(kind, lambda: q)()
    if kind in ("odd", "wide"):
        k = k[..., :7] if kind == "odd" else randn(g, 2, 5, 1, 300)
        w = None
    k = {"half": lambda: k.half(), "short": lambda: k[:, :4]}.get(change.get("k"), lambda: k)()
    if "layout" in change:
        layout = change["layout"]
    if "sin" in change:
        sin = None
    if change.get("cos") == "long":
        cos, sin = ops().rotary_tables(5, 10, device="cuda")
    if change.get("cos") == "few":
        cos, sin = cos[:4], sin[:4]
    if "w" in change:
        w = w[:4] if change["w"] == "short" else w.int()
    if "positions" in change:
        positions = torch.zeros(2, 5, device="cuda") if change["positions"] == "float" else torch.zeros(2, 4, device="cuda", dtype=torch.int32)
    with pytest.raises((RuntimeError, ValueError), match=match):
        ops().norm_rotate(q, k, w, None, cos, sin, positions, layout)


# ---- attention ---------------------------------------------------------------------------------------------------------------
def documents_of(kind, B, T, g):
    if kind is None:
        return None
    if kind == "sorted":  # runs, padding behind the last
        ids = torch.sort(torch.randint(0, max(2, T // 20), (B, T), generator=g, device="cuda"), dim=1)[0].int()
        ids[:, T - T // 7 - 1:] = -1
        return ids
    if kind == "mixed":  # ids in no order, padding in between
        return torch.randint(-1, 3, (B, T), generator=g, device="cuda", dtype=torch.int32)
    if kind == "none":  # nothing but padding in the first row
        ids = torch.zeros(B, T, device="cuda", dtype=torch.int32)
        ids[0] = -5
        return ids
    raise ValueError(kind)


# (B, Tq, Tk, H, G, D, keywords)
ATTENTION = [
    (1, 1, 1, 1, 1, 8, {}), (2, 197, 197, 6, 6, 64, {}), (1, 197, 197, 6, 6, 64, dict(cap=30.0)), (2, 64, 64, 4, 4, 64, {}),
    (1, 128, 128, 2, 2, 128, dict(causal=True)), (2, 129, 129, 4, 2, 64, dict(causal=True)), (1, 333, 333, 6, 2, 96, dict(causal=True, slopes=True)),
    (3, 65, 65, 3, 1, 80, dict(slopes=True)), (2, 257, 257, 4, 1, 64, dict(causal=True, prefix=True)),
    (2, 300, 300, 2, 2, 64, dict(docs="sorted")), (2, 300, 300, 4, 2, 32, dict(docs="sorted", causal=True, cap=20.0)),
    (2, 130, 130, 2, 1, 64, dict(docs="mixed")), (2, 130, 130, 2, 1, 128, dict(docs="mixed", causal=True, prefix=True, slopes=True, cap=5.0)),
    (2, 70, 70, 2, 2, 64, dict(docs="none")), (2, 1, 333, 8, 2, 64, {}), (1, 1, 1000, 16, 4, 128, dict(slopes=True)),
    (2, 1, 77, 6, 6, 64, dict(docs="sorted", query_docs=True)), (2, 5, 400, 4, 4, 64, dict(causal=True)), (1, 16, 777, 8, 1, 72, dict(causal=True, cap=50.0)),
    (2, 100, 60, 2, 2, 64, dict(causal=True)), (2, 40, 300, 2, 1, 64, dict(causal=True, prefix=True, docs="sorted")), (1, 700, 700, 2, 2, 64, dict(docs="sorted")),
    (1, 2, 2, 2, 1, 16, dict(causal=True)), (1, 513, 513, 1, 1, 120, dict(causal=True, prefix=True)), (1, 300, 9, 4, 4, 64, {}),
    (1, 1, 5000, 4, 2, 64, dict(docs="mixed", query_docs=True)), (4, 3, 2500, 4, 4, 64, dict(cap=30.0, causal=True)),
]


def attention_case(B, Tq, Tk, H, G, D, kw, dtype, seed=0):
    kw = dict(kw)
    g = gen(seed + 7 * Tq + Tk + D)
    rows = randn(g, B, Tk, 3 * G, D, dtype=dtype)
    q = randn(g, B, Tq, H, D, dtype=dtype)
    k, v = rows[:, :, G:2 * G], rows[:, :, 2 * G:]  # views of one tensor
    docs = documents_of(kw.pop("docs", None), B, Tk, g)
    if kw.pop("query_docs", False):
        kw["query_documents"] = torch.randint(0, 2, (B, Tq), generator=g, device="cuda", dtype=torch.int32)
    if docs is not None:
        kw["documents"] = docs
    if kw.pop("slopes", False):
        kw["slopes"] = torch.rand(H, generator=g, device="cuda") * 0.2
    if kw.pop("prefix", False):
        kw["prefix"] = torch.randint(0, Tk + 5, (B,), generator=g, device="cuda", dtype=torch.int32)
    return [x.detach().requires_grad_(True) for x in (q, k, v)], kw, randn(g, B, Tq, H, D, dtype=dtype)


def attention_bounds(q, k, v, go, kw, dtype):
    """Results and gradients in 64 bits and how far each element may be off.

    16-bit operands: a probability is off by at most u of itself, so an output by u * sum p|v|, and then by u of itself.  grad_v sums
    such probabilities: u * sum p|go|.  A score gradient p (gp - delta) scale is rounded (u of itself), its p not being rounded
    before; delta is the sum of go * out with out rounded: off by u * sum |go||out|.  grad_q and grad_k sum these times k and q.
    fp32: the same formulas with u = 2^-24 and, for the sums of D or T terms, the exponential of scores of up to 64 and their
    products, a factor: scores off by (D + 8) 2^-24 of sum |q||k| scale, which p multiplies."""
    u, f = rounding(dtype), 2.0 ** -24
    qd, kd, vd = (x.detach().double().requires_grad_(True) for x in (q, k, v))
    want = R.attention(qd, kd, vd, **kw)
    grads = torch.autograd.grad(want, (qd, kd, vd), go.double())
    qd, kd, vd, want, god = qd.detach(), kd.detach(), vd.detach(), want.detach(), go.double()
    B, Tq, H, D = q.shape
    Tk, G = k.shape[1:3]
    documents, cap, slopes = kw.get("documents"), kw.get("cap", 0.0), kw.get("slopes")
    seen = R.visible(B, Tq, Tk, kw.get("causal", False), kw.get("prefix"), documents, kw.get("query_documents"), q.device)[:, None]
    if documents is not None:
        dq = kw.get("query_documents")
        dq = documents[:, Tk - Tq:] if dq is None else dq
        qd, god = (torch.where((dq >= 0)[:, :, None, None], x, 0.0) for x in (qd, god))
        kd, vd = (torch.where((documents >= 0)[:, :, None, None], x, 0.0) for x in (kd, vd))
    ke, ve = kd.repeat_interleave(H // G, 2), vd.repeat_interleave(H // G, 2)
    scale = kw.get("scale", D ** -0.5)
    s = torch.einsum("bihd,bjhd->bhij", qd, ke) * scale
    most = torch.einsum("bihd,bjhd->bhij", qd.abs(), ke.abs()) * abs(scale)
    bend = torch.ones_like(s)
    if cap:
        t = torch.tanh(s / cap)
        bend = 1 - t * t
        s = cap * t
    if slopes is not None:
        s = s - slopes.double()[:, None, None] * (torch.arange(Tk - Tq, Tk, device=q.device)[:, None] - torch.arange(Tk, device=q.device)).abs()
    some = seen.any(-1, keepdim=True)
    p = torch.softmax(torch.where(some, s.masked_fill(~seen, -torch.inf), 0.0), -1) * some * seen
    # relative error of p: of its score (products, cap, bias, scaling), of exp2 and of the sum of a row
    off = (D + 8) * f * most + 8 * f * s.abs().clamp(max=1e4) + (f * 16 * cap if cap else 0) + 8 * f + (Tk ** 0.5 + 40) * f
    off = off + (p * off).sum(-1, keepdim=True)
    half = 0.0 if dtype is torch.float32 else u
    sums = 2 * (Tk + 64) * f  # accumulation of a row's products in fp32, rounded or cut off
    e_out = torch.einsum("bhij,bjhd->bihd", p * (off + half + sums), ve.abs()) + u * want.abs()
    gp = torch.einsum("bihd,bjhd->bhij", god, ve)
    gp_most = torch.einsum("bihd,bjhd->bhij", god.abs(), ve.abs())
    delta = (p * gp).sum(-1, keepdim=True)
    e_delta = torch.einsum("bihd,bihd->bhi", god.abs(), e_out + D * f * want.abs())[..., None]
    gs = p * (gp - delta)
    e_gs = gs.abs() * (off + half + 8 * f) + p * ((D + 8) * f * gp_most + e_delta)
    if cap:  # the derivative of the cap, computed from a rounded tanh
        e_gs = e_gs * bend + gs.abs() * (8 * f + 2 * (D + 8) * f * most / cap)
    rows = 2 * (Tq * (H // G) + 64) * f
    e_gs, gs = e_gs * abs(scale), gs * bend * scale

    def shared(x):  # sum over the heads of a group
        return x.view(B, Tk, G, H // G, D).sum(3)
    e_q = torch.einsum("bhij,bjhd->bihd", e_gs + sums * gs.abs(), ke.abs()) + u * grads[0].abs()
    e_k = shared(torch.einsum("bhij,bihd->bjhd", e_gs + rows * gs.abs(), qd.abs())) + u * grads[1].abs()
    e_v = shared(torch.einsum("bhij,bihd->bjhd", p * (off + half + rows), god.abs())) + u * grads[2].abs()
    return [want, *grads], [e_out + 1e-30, e_q + 1e-30, e_k + 1e-30, e_v + 1e-30]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,Tq,Tk,H,G,D,kw", ATTENTION)
def test_attention(B, Tq, Tk, H, G, D, kw, dtype):
    (q, k, v), kw, go = attention_case(B, Tq, Tk, H, G, D, kw, dtype)
    out = ops().attention(q, k, v, **kw)
    got = [out.detach(), *torch.autograd.grad(out, (q, k, v), go)]
    want, tol = attention_bounds(q, k, v, go, kw, dtype)
    assert out.dtype is dtype and out.is_contiguous()
    tiny = 0.0 if dtype is not torch.float16 else 2.0 ** -24  # (subnormal fp16 results and probabilities)
    for name, x, w, t in zip(("out", "grad_q", "grad_k", "grad_v"), got, want, tol):
        close(x, w, t + tiny * 40, name)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_attention_padding_may_hold_anything(dtype):
    (q, k, v), kw, go = attention_case(2, 150, 150, 4, 2, 64, dict(docs="sorted", cap=30.0), dtype)
    out = ops().attention(q, k, v, **kw)
    plain = [out.detach(), *torch.autograd.grad(out, (q, k, v), go)]
    pad = kw["documents"] < 0
    assert pad.any()
    bad = []
    for x, filler in ((q, float("nan")), (k, float("inf")), (v, float("nan"))):
        y = x.detach().clone()
        y[pad] = filler
        bad.append(y.requires_grad_(True))
    gbad = go.clone()
    gbad[pad] = float("inf")
    out = ops().attention(*bad, **kw)
    for name, x, y in zip(("out", "grad_q", "grad_k", "grad_v"), [out.detach(), *torch.autograd.grad(out, bad, gbad)], plain):
        assert torch.equal(x, y), name
        assert (x[pad] == 0).all(), name


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_attention_repeats_its_bits_and_runs_on_other_streams_and_in_graphs(dtype):
    (q, k, v), kw, go = attention_case(2, 260, 260, 8, 2, 64, dict(causal=True, prefix=True, slopes=True), dtype)

    def both():
        out = ops().attention(q, k, v, **kw)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), go)]
    first = both()
    for x, y in zip(both(), first):
        assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(other, first):
        assert torch.equal(x, y)
    # forward passes captured and replayed on new inputs
    one = q.detach()[:, -1:].contiguous()
    static, static_one = q.detach().clone(), one.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        ops().attention(static, k, v, **kw), ops().attention(static_one, k, v, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y, y_one = ops().attention(static, k, v, **kw), ops().attention(static_one, k, v, **kw)
    static.copy_(q.detach().flip(0))
    static_one.copy_(one.flip(0))
    graph.replay()
    with torch.no_grad():
        assert torch.equal(y, ops().attention(static, k, v, **kw)) and torch.equal(y_one, ops().attention(static_one, k, v, **kw))


def test_attention_strides_and_empty_problems():
    g = gen(3)
    # heads before tokens, unaligned rows, expanded batch
    for dtype in DTYPES:
        base = [randn(g, 2, 4, 70, 64, dtype=dtype) for _ in range(3)]
        q, k, v = (x.transpose(1, 2) for x in base)
        same = ops().attention(*(x.contiguous() for x in (q, k, v)), causal=True)
        assert torch.equal(ops().attention(q, k, v, causal=True), same)
        odd = randn(g, 2, 70, 4, 65, dtype=dtype)[..., 1:]
        assert torch.equal(ops().attention(odd, k, v), ops().attention(odd.contiguous(), k, v))
        assert torch.equal(ops().attention(q, odd, odd), ops().attention(q, odd.contiguous(), odd.contiguous()))
        wide = k[:1].expand(2, 70, 4, 64)
        assert torch.equal(ops().attention(q, wide, wide), ops().attention(q, wide.contiguous(), wide.contiguous()))
    for B, Tq, Tk in ((0, 3, 3), (2, 0, 3), (2, 3, 0)):
        q = randn(g, B, Tq, 2, 64).requires_grad_(True)
        k, v = randn(g, B, Tk, 1, 64).requires_grad_(True), randn(g, B, Tk, 1, 64)
        out = ops().attention(q, k, v)
        gq, gk = torch.autograd.grad(out, (q, k), torch.ones_like(out))
        assert out.shape == q.shape and not out.any() and gq.shape == q.shape and not gq.any() and gk.shape == k.shape and not gk.any()


def test_attention_gradient_against_differences():
    (q, k, v), kw, go = attention_case(1, 40, 40, 2, 1, 16, dict(causal=True, slopes=True, cap=4.0), torch.float32)
    out = ops().attention(q, k, v, **kw)
    grads = torch.autograd.grad(out, (q, k, v), go)
    g, h = gen(9), 2.0 ** -6
    for i in range(3):
        step = randn(g, *(q, k, v)[i].shape)
        step /= step.norm()

        def value(t):
            args = [x.detach() + (t * step if j == i else 0) for j, x in enumerate((q, k, v))]
            return (ops().attention(*args, **kw).double() * go.double()).sum().item()
        slope = (value(h) - value(-h)) / (2 * h)
        # h^2/6 of a third derivative of order |go| |v| ~ 40 * 4 along a unit step, 2^-24 * 1280 values / h of rounding
        assert abs(slope - (grads[i].double() * step.double()).sum().item()) <= h * h / 6 * 160 + 2.0 ** -24 * 1280 / h


@pytest.mark.parametrize("change,match", [
    (dict(q=lambda x: x.cpu()), "CUDAtensor"), (dict(k=lambda x: x.half()), "of type"), (dict(v=lambda x: x[:, :4]), "must both be"),
    (dict(q=lambda x: x[0]), "B, T, heads, D"), (dict(q=lambda x: x[:, :, :3]), "multiple of the"), (dict(cap=-1.0), "negative"),
    (dict(cap=float("inf")), "negative"), (dict(scale=float("nan")), "finite"), (dict(slopes=torch.ones(3)), "slopes"),
    (dict(prefix=torch.ones(2, dtype=torch.int32)), "causal"), (dict(documents=torch.ones(2, 9)), "documents"),
    (dict(query_documents=torch.ones(2, 9, dtype=torch.int32)), "belong to documents"),
    (dict(causal=True, prefix=torch.ones(2, dtype=torch.int64)), "prefix"), (dict(documents=torch.ones(2, 8, dtype=torch.int32)), "documents")])
def test_attention_refuses(change, match):
    g = gen(4)
    x = dict(q=randn(g, 2, 9, 4, 16), k=randn(g, 2, 9, 2, 16), v=randn(g, 2, 9, 2, 16))
    kw = {}
    for name, f in change.items():
        if name in x:
            x[name] = f(x[name])
        else:
            kw[name] = f.cuda() if isinstance(f, torch.Tensor) else f
    with pytest.raises((RuntimeError, ValueError), match=match):
        ops().attention(x["q"], x["k"], x["v"], **kw)


def test_attention_refuses_head_sizes_and_learned_slopes():
    g = gen(4)
    for d in (4, 12, 136):
        x = randn(g, 1, 3, 2, d)
        with pytest.raises(RuntimeError, match="multiple of 8"):
            ops().attention(x, x, x)
    x = randn(g, 1, 3, 2, 8)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops().attention(x, x, x, slopes=torch.ones(2, device="cuda", requires_grad=True))
    with pytest.raises(RuntimeError, match="query_documents"):
        ops().attention(randn(g, 1, 4, 2, 8), x, x, documents=torch.zeros(1, 3, device="cuda", dtype=torch.int32))


# ---- token_logprobs ------------------------------------------------------------------------------------------------------------
LOGP = [(1, 1, 1), (1, 2, 2), (3, 7, 7), (64, 10, 5), (64, 1000, 5), (5, 513, 32), (37, 4097, 20), (2, 32001, 5), (300, 2049, 0), (3, 128257, 32),
        (1, 200003, 1), (700, 511, 3), (5, 40, 32), (1, 4500, 32)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("N,C,top", LOGP)
def test_token_logprobs(N, C, top, dtype):
    import lutgemm_loss
    g = gen(N + C)
    x = (2 * randn(g, N, C)).to(dtype)
    x[torch.arange(N, device="cuda"), torch.randint(0, C, (N,), generator=g, device="cuda")] += 9
    if C > 3:
        x[torch.rand(N, C, generator=g, device="cuda") < 0.05] = -torch.inf
    x = x.requires_grad_(True)
    targets = torch.randint(0, C, (N,), generator=g, device="cuda")
    targets[::5] = x.detach()[::5].float().argmax(1)
    targets[1::7] = -100
    logp, entropy, top_logp, top_index = lutgemm_loss.token_logprobs(x, targets, top)
    g_logp, g_entropy = randn(g, N), randn(g, N)
    grad = torch.autograd.grad((logp, entropy), x, (g_logp, g_entropy), retain_graph=True)[0]
    only = torch.autograd.grad(logp, x, g_logp)[0]
    xd = x.detach().double()
    want = R.token_logprobs(xd, targets, top)
    assert torch.equal(top_index, want[3])
    f, u = 2.0 ** -24, rounding(dtype)
    spread = (xd.amax(1) - xd.masked_fill(xd == -torch.inf, torch.inf).amin(1))
    # distances to the largest logit up to `spread` are exact to f of themselves, their exponentials to (spread + 4) f (ex2 of a
    # rounded product), sums of C positive terms (in runs and trees of at most 512) to 600 f, the logarithm to 4 f
    rel = (2 * spread + 650) * f
    others = torch.logsumexp(xd, 1) - xd.amax(1)  # log1p of what is beside the largest
    e_logp = 4 * f * (want[0].abs() + spread) + rel * others.clamp(max=1.0) + 1e-30
    hit = targets == xd.argmax(1)
    e_logp = torch.where(hit, 4 * f * want[0].abs() + rel * others.clamp(max=1.0), e_logp)
    close(logp, want[0], e_logp + 1e-30, "logp")
    close(entropy, want[1], (rel + 8 * f) * (want[1] + others) + 1e-30, "entropy")
    close(top_logp, want[2], (4 * f * (spread + 1) + rel * others.clamp(max=1.0))[:, None] + 1e-30, "top_logp")
    p = torch.softmax(xd, 1)
    logs = torch.log_softmax(xd, 1)
    hot = torch.zeros_like(p).scatter_(1, targets.clamp(min=0)[:, None], 1.0)
    gl = torch.where(targets == -100, 0.0, g_logp.double())[:, None]
    rest = torch.where(hot > 0, -torch.expm1(logs), -p)
    ge = g_entropy.double()[:, None]
    tail = torch.where(p > 0, p * (logs.masked_fill(p == 0, 0.0) + want[1][:, None]), 0.0)
    tiny = 2.0 ** -25 if dtype is torch.float16 else 1e-37  # (subnormal results)
    e = gl.abs() * (rest.abs() * (rel[:, None] + 8 * f)) + ge.abs() * (tail.abs() * (rel[:, None] + 8 * f) + p * 8 * f * (spread[:, None] + 1 + want[1][:, None]))
    # (1 - p of a given class that is not the largest: fp32 off by its exponent, all of it relative to p)
    e = e + gl.abs() * hot * (rel[:, None] + 8 * f) * p * (~hit)[:, None]
    close(grad, gl * rest - ge * tail, u * (gl * rest - ge * tail).abs() + e + tiny, "grad")
    close(only, gl * rest, u * (gl * rest).abs() + e + tiny, "grad of logp alone")


@pytest.mark.parametrize("C", [5, 600, 9001, 70001])
def test_token_logprobs_ties_and_odd_rows(C):
    import lutgemm_loss
    top = min(C, 32)
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(8, C, device="cuda")
    x[1] = -inf                      # nothing has probability
    x[2, 0] = nan
    x[3, C // 2] = inf
    x[4] = torch.arange(C, device="cuda") % 2 * 3.0   # ties of two values
    x[5] = -inf
    x[5, C - 1] = 2.0                # one class alone
    x[6, ::2] = -0.0                 # zeros of both signs are equal
    x[7] = torch.finfo(torch.float32).min
    targets = torch.full((8,), C - 1, device="cuda")
    x.requires_grad_(True)
    logp, entropy, top_logp, top_index = lutgemm_loss.token_logprobs(x, targets, top)
    grad = torch.autograd.grad(logp.sum() + entropy.sum(), x)[0]
    flat = torch.arange(top, device="cuda")
    for r in (0, 1, 6, 7):
        assert torch.equal(top_index[r], flat), r
    log_c = torch.log(torch.tensor(float(C), dtype=torch.float64)).item()
    for r in (0, 6, 7):
        assert abs(logp[r].item() + log_c) <= 1e-5 and abs(entropy[r].item() - log_c) <= 1e-5
    assert logp[1].item() == -inf and entropy[1].item() == 0 and not grad[1].any() and (top_logp[1] == -inf).all()
    for r in (2, 3):
        assert torch.isnan(logp[r]) and torch.isnan(entropy[r])
    assert torch.isnan(grad[2]).all()
    assert top_index[2, 0] == 0 and top_index[3, 0] == C // 2
    odd = torch.arange(1, C, 2, device="cuda")
    want = torch.cat([odd, torch.arange(0, C, 2, device="cuda")])[:top]
    assert torch.equal(top_index[4], want)
    assert logp[5].item() == 0 and entropy[5].item() == 0 and top_index[5, 0] == C - 1 and not grad[5].any()


def test_token_logprobs_shapes_strides_and_targets():
    import lutgemm_loss
    g = gen(8)
    x = randn(g, 3, 4, 50)
    t = torch.randint(0, 50, (3, 4), generator=g, device="cuda")
    logp, entropy, top_logp, top_index = lutgemm_loss.token_logprobs(x, t, 3)
    assert logp.shape == entropy.shape == (3, 4) and top_logp.shape == top_index.shape == (3, 4, 3)
    flat = lutgemm_loss.token_logprobs(x.view(12, 50), t.view(12), 3)
    assert torch.equal(flat[0], logp.view(12)) and torch.equal(flat[3], top_index.view(12, 3))
    one = lutgemm_loss.token_logprobs(x[0, 0], t[0, 0], 2)
    assert one[0].shape == () and one[3].shape == (2,) and torch.equal(one[0], logp[0, 0])
    wide = randn(g, 12, 131)
    part = lutgemm_loss.token_logprobs(wide[:, 3:53], t.view(12), 4)  # rows of a wider matrix, unaligned
    again = lutgemm_loss.token_logprobs(wide[:, 3:53].contiguous(), t.view(12), 4)
    close(part[0], again[0].double(), 1e-5, "logp of a slice")
    assert torch.equal(part[3], again[3])
    turned = randn(g, 50, 12).t()
    assert torch.equal(lutgemm_loss.token_logprobs(turned, t.view(12), 4)[0], lutgemm_loss.token_logprobs(turned.contiguous(), t.view(12), 4)[0])
    # a gradient for rows that lie on other boundaries than the result's
    sliced = wide[:, 3:53].detach().requires_grad_(True)
    gr = torch.autograd.grad(lutgemm_loss.token_logprobs(sliced, t.view(12))[0].sum(), sliced)[0]
    p = torch.softmax(sliced.detach().double(), 1)
    close(gr, torch.nn.functional.one_hot(t.view(12), 50) - p, 1e-5, "gradient of a slice")
    # targets that are no class, and another number for rows without one
    bad = torch.tensor([50, -1, -100, 7, 2 ** 40, -2 ** 40], device="cuda")
    y = x.view(12, 50)[:6].clone().requires_grad_(True)
    logp = lutgemm_loss.token_logprobs(y, bad)[0]
    assert torch.equal(torch.isnan(logp).cpu(), torch.tensor([1, 1, 0, 0, 1, 1]).bool()) and logp[2] == 0
    gr = torch.autograd.grad(logp.sum(), y)[0]
    assert torch.isnan(gr[0]).all() and not gr[2].any() and torch.isfinite(gr[3]).all()
    assert lutgemm_loss.token_logprobs(y.detach(), bad, ignore_index=7)[0][3] == 0
    empty = lutgemm_loss.token_logprobs(torch.empty(0, 5, device="cuda", requires_grad=True), torch.empty(0, dtype=torch.int64, device="cuda"), 2)
    assert empty[0].shape == (0,) and empty[3].shape == (0, 2)


@pytest.mark.parametrize("args,error", [
    ((lambda x, t: (x.cpu(), t)), "CUDAtensor"), ((lambda x, t: (x.double(), t)), "of type"), ((lambda x, t: (x, t.int())), "int64"),
    ((lambda x, t: (x, t[:3])), "expected"), ((lambda x, t: (x, t, 11)), "top"), ((lambda x, t: (x, t, -1)), "top"),
    ((lambda x, t: (x[:, :0], t)), "classes"), ((lambda x, t: (x, t.cpu())), "int64")])
def test_token_logprobs_refuses(args, error):
    import lutgemm_loss
    x, t = torch.zeros(4, 10, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises((RuntimeError, ValueError), match=error):
        lutgemm_loss.token_logprobs(*args(x, t))
