"""Head norms, attention and log probabilities as programs call them: some inputs learned and others not, several streams at once,
passes captured into graphs, offsets beyond 32 bits, the most rows, one tensor in several places."""
import pytest
import torch

import operators_reference as R
from test_gpu_operators import DTYPES, IDS, attention_bounds, attention_case, close, gen, ops, randn, rounding

pytestmark = pytest.mark.gpu


def logprobs(*args, **kw):
    import lutgemm_loss
    return lutgemm_loss.token_logprobs(*args, **kw)


def check_attention(case, kw, dtype):
    (q, k, v), kw, go = case
    out = ops().attention(q, k, v, **kw)
    got = [out.detach(), *torch.autograd.grad(out, (q, k, v), go)]
    want, tol = attention_bounds(q, k, v, go, kw, dtype)
    tiny = 0.0 if dtype is not torch.float16 else 2.0 ** -24
    for name, x, w, t in zip(("out", "grad_q", "grad_k", "grad_v"), got, want, tol):
        close(x, w, t + tiny * 40, name)


# heads of queries to one of keys that do not divide a tile of 64, and a whole tile of them
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,Tq,Tk,H,G,D,kw", [
    (2, 90, 90, 3, 1, 64, dict(docs="sorted")), (1, 90, 90, 6, 2, 128, dict(docs="mixed", causal=True)), (1, 40, 40, 33, 1, 64, dict(causal=True, cap=20.0)),
    (1, 11, 70, 64, 1, 64, dict(slopes=True)), (2, 9, 50, 10, 2, 32, dict(docs="sorted", causal=True, prefix=True)), (1, 3, 700, 7, 1, 128, {})])
def test_attention_of_odd_groups_of_heads(B, Tq, Tk, H, G, D, kw, dtype):
    check_attention(attention_case(B, Tq, Tk, H, G, D, kw, dtype), kw, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("scale,sign", [(0.0, 0.0), (-0.2, 0.0), (0.3, -1.0), (-0.1, 1.0)])
def test_attention_scales_and_slopes_of_either_sign(scale, sign, dtype):
    (q, k, v), kw, go = attention_case(1, 100, 140, 2, 1, 64, dict(causal=True, scale=scale, **(dict(slopes=True) if sign else {})), dtype)
    if sign:
        kw["slopes"] = kw["slopes"] * sign
    check_attention(((q, k, v), kw, go), kw, dtype)


def test_learned_inputs_alone():
    g = gen(21)
    q, k, w = randn(g, 2, 5, 3, 16), randn(g, 2, 5, 2, 16), 1 + 0.1 * randn(g, 16)
    cos, sin = ops().rotary_tables(5, 8, device="cuda")
    gq, gk = randn(g, 2, 5, 3, 16), randn(g, 2, 5, 2, 16)

    def grads(fn, leaves, others):  # of the leaves alone, and of all inputs in 64 bits
        leaf = {n: x.detach().clone().requires_grad_(True) for n, x in leaves.items()}
        yq, yk = fn(**leaf, **others)
        return torch.autograd.grad((yq * gq.to(yq.dtype)).sum() + (yk * gk.to(yk.dtype)).sum(), list(leaf.values()), allow_unused=True)

    def plain(q, k, q_weight=None, k_weight=None):
        q, k = q.double(), k.double()
        return (R.norm_rotate(q, None if q_weight is None else q_weight.double(), cos, sin, None, "half", 1e-6),
                R.norm_rotate(k, None if k_weight is None else k_weight.double(), cos, sin, None, "half", 1e-6))

    def own(q, k, q_weight=None, k_weight=None):
        return ops().norm_rotate(q, k, q_weight, k_weight, cos, sin)
    everything = dict(q=q, k=k, q_weight=w, k_weight=w + 0.1)
    for learned in (("k_weight",), ("q_weight",), ("k", "q_weight"), ("q", "k_weight")):
        for given in (("q", "k") + learned, tuple(everything)):
            leaves = {n: everything[n] for n in learned}
            others = {n: everything[n] for n in everything if n in given and n not in learned}
            for x, y, n in zip(grads(own, leaves, others), grads(plain, leaves, others), learned):
                # sums of 30 products of values up to 5, each off by some roundings
                close(x, y.double(), 30 * 25 * 16 * 2.0 ** -24, n)


def test_one_tensor_in_several_places():
    g = gen(22)
    for dtype in DTYPES:
        x = randn(g, 2, 70, 2, 64, dtype=dtype).requires_grad_(True)
        go = randn(g, 2, 70, 2, 64, dtype=dtype)
        three = [x.detach().clone().requires_grad_(True) for _ in range(3)]
        one, apart = ops().attention(x, x, x, causal=True), ops().attention(*three, causal=True)
        assert torch.equal(one, apart)
        parts = [y.double() for y in torch.autograd.grad(apart, three, go)]
        sums = torch.autograd.grad(one, x, go)[0]
        # (the library adds two and then the third, each sum rounded)
        close(sums, sum(parts), 2 * 1.01 * rounding(dtype) * sum(y.abs() for y in parts), "gradient of all three")


def test_gradients_of_sums():  # expanded from one value
    g = gen(23)
    for dtype in DTYPES:
        q, k = (randn(g, 2, 9, 2, 16, dtype=dtype).requires_grad_(True) for _ in range(2))
        cos, sin = ops().rotary_tables(9, 16, device="cuda")
        for fn in (lambda: ops().norm_rotate(q, k, cos=cos, sin=sin)[0], lambda: ops().attention(q, k, k)):
            y = fn()
            assert torch.equal(torch.autograd.grad(y.sum(), q)[0], torch.autograd.grad(fn(), q, torch.ones_like(y))[0])
        x, t = randn(g, 7, 20, dtype=dtype).requires_grad_(True), torch.arange(7, device="cuda")
        assert torch.equal(torch.autograd.grad(logprobs(x, t)[1].sum(), x)[0],
                           torch.autograd.grad(logprobs(x, t)[1], x, torch.ones(7, device="cuda"))[0])


def test_refusals_of_gradients():
    g = gen(24)
    q, k = (randn(g, 1, 5, 2, 16).requires_grad_(True) for _ in range(2))
    x, t = randn(g, 5, 9).requires_grad_(True), torch.arange(5, device="cuda")
    cos, sin = ops().rotary_tables(5, 16, device="cuda")
    for y, leaf in ((ops().norm_rotate(q, k)[0], q), (ops().attention(q, k, k), q), (logprobs(x, t)[0], x)):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y.sum(), leaf, create_graph=True)
    learned = cos.clone().requires_grad_(True)
    slopes = torch.ones(2, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops().norm_rotate(q, k, cos=learned, sin=sin)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops().attention(q, k, k, slopes=slopes)
    with torch.no_grad():
        assert torch.equal(ops().norm_rotate(q, k, cos=learned, sin=sin)[0], ops().norm_rotate(q, k, cos=cos, sin=sin)[0])
        assert torch.equal(ops().attention(q, k, k, slopes=slopes), ops().attention(q, k, k, slopes=slopes.detach()))


# (B, T, H, G, D, keywords): partial tiles, several rounds, each way of handing tiles from warp to warp
REPEATED = [(2, 197, 6, 6, 64, {}), (2, 197, 6, 6, 64, dict(cap=30.0)), (1, 1000, 4, 4, 64, dict(slopes=True)), (1, 1000, 4, 2, 128, dict(causal=True)),
            (2, 260, 3, 1, 96, dict(docs="sorted", cap=10.0)), (1, 900, 6, 2, 64, dict(docs="sorted", causal=True))]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,T,H,G,D,kw", REPEATED)
def test_attention_repeats_its_bits_over_many_calls(B, T, H, G, D, kw, dtype):
    (q, k, v), kw, go = attention_case(B, T, T, H, G, D, kw, dtype)
    first = None
    for _ in range(20):
        out = ops().attention(q, k, v, **kw)
        now = [out.detach(), *torch.autograd.grad(out, (q, k, v), go)]
        first = first or now
        assert all(torch.equal(x, y) for x, y in zip(now, first))


def test_streams_at_once():
    cases = [attention_case(2, T, T, H, G, D, kw, dtype) for T, H, G, D, kw, dtype in (
        (400, 6, 6, 64, {}, torch.bfloat16), (300, 6, 6, 64, {}, torch.float32), (500, 4, 2, 128, dict(causal=True), torch.float16),
        (350, 4, 4, 64, dict(cap=20.0), torch.bfloat16))]
    cos, sin = ops().rotary_tables(500, 64, device="cuda")
    targets = torch.arange(800, device="cuda") % 384

    def work(case):
        (q, k, v), kw, go = case
        a, b = ops().norm_rotate(q, k, cos=cos[:, :q.shape[3] // 2], sin=sin[:, :q.shape[3] // 2])
        out = ops().attention(a, b, v, **kw)
        logits = out.reshape(-1, out.shape[2] * out.shape[3])
        logp = logprobs(logits, targets.repeat(2)[:logits.shape[0]] % logits.shape[1], 3)
        return [out.detach(), *(x.detach() for x in logp), *torch.autograd.grad((out, logp[0].sum()), (q, k, v), (go, torch.ones((), device="cuda")))]
    alone = [work(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    results = [[] for _ in cases]
    for _ in range(6):
        for s, c, r in zip(streams, cases, results):
            with torch.cuda.stream(s):
                r.append(work(c))
    torch.cuda.synchronize()
    for r, a in zip(results, alone):
        for now in r:
            assert all(torch.equal(x, y) for x, y in zip(now, a))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_passes_captured_and_replayed(dtype):
    """Forward and backward of all three, two graphs replayed in turn on inputs that change."""
    g = gen(25)
    cos, sin = ops().rotary_tables(150, 32, device="cuda")
    targets = torch.randint(0, 128, (300,), generator=g, device="cuda")
    ids = torch.arange(150, device="cuda", dtype=torch.int32).expand(2, 150) // 40

    def step(q, k, v, w):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v, w)]
        a, b = ops().norm_rotate(leaves[0], leaves[1], leaves[3], None, cos, sin)
        out = ops().attention(a, b, leaves[2], causal=True, documents=ids)
        logp, entropy, _, at = logprobs(out.reshape(300, 128), targets, 2)
        return [out.detach(), at, *torch.autograd.grad(logp.mean() + entropy.mean(), leaves)]

    def fresh():
        return [randn(g, 2, 150, 2, 64, dtype=dtype) for _ in range(3)] + [1 + 0.1 * randn(g, 64)]
    statics, graphs, results = [fresh() for _ in range(2)], [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*statics[0])
    torch.cuda.current_stream().wait_stream(side)
    for static in statics:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step(*static))
        graphs.append(graph)
    for _ in range(2):
        inputs = [fresh() for _ in range(2)]
        for static, new in zip(statics, inputs):
            for x, y in zip(static, new):
                x.copy_(y)
        for graph in graphs:
            graph.replay()
        for result, new in zip(results, inputs):
            assert all(torch.equal(x, y) for x, y in zip(result, step(*new)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_offsets_beyond_32_bits(dtype):
    """Tokens 2^22 elements apart: the last of 600 lies 2.5 * 10^9 elements behind the first."""
    g = gen(26)
    pitch, T = 1 << 22, 600
    room = torch.empty(pitch * T, dtype=dtype, device="cuda")

    def far(x):  # [1, T, heads, D] with its tokens `pitch` apart
        y = room.as_strided(x.shape, (pitch * T, pitch, x.shape[3], 1), far.at)
        far.at += x[0, 0].numel()
        return y.copy_(x)
    for D in (64, 128):
        far.at = 0
        near = [randn(g, 1, T, heads, D, dtype=dtype) for heads in (4, 2, 2)]
        away = [far(x) for x in near]
        go = randn(g, 1, T, 4, D, dtype=dtype)
        away_go = far(go)
        results = []
        for xs, grad in ((near, go), (away, away_go)):
            q, k, v = (x.detach().requires_grad_(True) for x in xs)
            a, b = ops().norm_rotate(q, k)
            out = ops().attention(q, k, v, causal=True)
            with torch.no_grad():
                one = ops().attention(q[:, -1:], k, v)
            results.append([a.detach(), b.detach(), one, out.detach(), *torch.autograd.grad((out, a), (q, k, v), (grad, grad))])
        for x, y in zip(*results):
            assert torch.equal(x, y)
    rows = randn(g, T, 1000, dtype=dtype)
    wide = room.as_strided((T, 1000), (pitch, 1), 0)
    wide.copy_(rows)
    targets = torch.arange(T, device="cuda")
    results = []
    for x in (rows, wide):
        x = x.detach().requires_grad_(True)
        logp, entropy, top, at = logprobs(x, targets, 4)
        results.append([logp.detach(), entropy.detach(), top, at, torch.autograd.grad(logp.sum() + entropy.sum(), x)[0]])
    for x, y in zip(*results):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("D", [8, 72])
def test_the_most_rows_of_a_batch(dtype, D):
    case = attention_case(65535, 1, 2, 1, 1, D, dict(docs="none"), dtype)
    check_attention(case, case[1], dtype)
    x = torch.empty(65536, 1, 1, D, dtype=dtype, device="cuda")
    with pytest.raises(RuntimeError, match="too many"):
        ops().attention(x, x, x)


# enough rows that loads run ahead through shared memory: heads that do not fill a group's turn, lanes without a vector, a last round
# that not every group has
@pytest.mark.parametrize("B,T,H,G,D,rot,layout,place,dtype", [
    (2, 8195, 17, 5, 128, 64, "interleaved", False, torch.bfloat16), (3, 5003, 21, 3, 128, 128, "half", True, torch.float16),
    (1, 20011, 8, 8, 80, 40, "half", True, torch.float32), (2, 9001, 7, 3, 128, 0, "half", False, torch.float32),
    (1, 40003, 13, 3, 48, 16, "interleaved", True, torch.bfloat16), (1, 16001, 40, 1, 64, 64, "half", False, torch.float16)])
def test_norm_rotate_of_many_rows(B, T, H, G, D, rot, layout, place, dtype):
    import test_gpu_operators
    test_gpu_operators.test_norm_rotate(B, T, H, G, D, rot, layout, place, dtype)
