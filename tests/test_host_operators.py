"""Host code of the head norms, attention and log probabilities without a GPU: what their entry points refuse and ask for, and that
nothing is launched before a refusal.  (The stand-in runtime has no tensor maps, so attention that needs them ends there.)"""
import ctypes
import math
import random

import pytest

import host_dispatch as H

F32, BF16, F16 = 0, 1, 2
E_CUDA = -3


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return H.Library(H.build(tmp_path_factory.mktemp("host")))


def at(n):
    return ctypes.c_void_p((1 << 40) + n)


def norm(lib, name="lutgemm_norm_rotate", dtype=BF16, B=2, T=5, H_=4, G=2, D=64, rot=64, eps=1e-6, table=5, cos=at(0), pos=None, q=at(0),
         dqw=at(0), scratch=at(0), scratch_bytes=1 << 40):
    s = [H.Size(1)] * 3
    side = [at(0), at(0), cos, at(0), table, pos, at(0), at(0)]
    shape = [dtype, B, T, H_, G, D, rot, 0, eps]
    if name == "lutgemm_norm_rotate":
        return lib.call(name, q, *s, at(0), *s, *side, *shape, None)
    return lib.call(name, at(0), *s, at(0), *s, q, *s, at(0), *s, *side, dqw, at(0), *shape, scratch, H.Size(scratch_bytes), None)


@pytest.mark.parametrize("name", ["lutgemm_norm_rotate", "lutgemm_norm_rotate_backward"])
@pytest.mark.parametrize("bad,status", [
    (dict(q=None), H.E_BADARG), (dict(dtype=3), H.E_BADARG), (dict(B=0), H.E_BADARG), (dict(G=0), H.E_BADARG), (dict(D=63, rot=62), H.E_BADARG),
    (dict(rot=63), H.E_BADARG), (dict(rot=66), H.E_BADARG), (dict(D=258), H.E_TOOLARGE), (dict(table=4), H.E_BADARG), (dict(cos=None), H.E_BADARG),
    (dict(eps=-1.0), H.E_BADARG), (dict(eps=float("nan")), H.E_BADARG), (dict(B=1 << 15, T=1 << 15, table=1 << 15), H.E_TOOLARGE)])
def test_norm_refuses_before_it_launches(lib, name, bad, status):
    assert norm(lib, name, **bad) == (status, [])


def test_norm_scratch(lib):
    need = lib.query("lutgemm_norm_rotate_backward_scratch_bytes", 64)
    name = "lutgemm_norm_rotate_backward"
    assert norm(lib, name, scratch_bytes=need - 1) == (H.E_SCRATCH, [])
    assert norm(lib, name, scratch=None) == (H.E_BADARG, [])
    rc, calls = norm(lib, name, scratch_bytes=need)
    assert rc == H.OK and [c[0] for c in calls] == ["norm_rotate_kernel", "norm_weight_sums_kernel"]
    assert norm(lib, pos=at(0), table=1)[0] == H.OK and norm(lib, rot=0, cos=None, table=0)[0] == H.OK
    # blocks never have more sums than the scratch buffer has room for
    rng = random.Random(0)
    for _ in range(200):
        D = 2 * rng.randint(1, 128)
        B, T, h, g = rng.randint(1, 64), int(math.exp(rng.uniform(0, 9))), rng.randint(1, 64), rng.randint(1, 64)
        if B * T * (h + g) >= 1 << 31:
            continue
        rc, calls = norm(lib, name, dtype=rng.randint(0, 2), B=B, T=T, H_=h, G=g, D=D, rot=0, scratch_bytes=1 << 40)
        assert rc == H.OK and calls[0][1] * D * 4 <= lib.query("lutgemm_norm_rotate_backward_scratch_bytes", D)


def attention(lib, backward=False, dtype=BF16, B=2, Tq=100, Tk=100, H_=4, G=2, D=64, scale=0.125, cap=0.0, doc_q=None, doc_k=None, stride=64,
              q=at(0), out=at(0), rest=at(0), scratch=at(0), scratch_bytes=1 << 40):
    s = [H.Size(stride)] * 3
    masks = [scale, cap, None, 0, None, doc_q, H.Size(Tq), doc_k, H.Size(Tk)]
    shape = [dtype, B, Tq, Tk, H_, G, D]
    tail = [*masks, scratch, H.Size(scratch_bytes), None]
    operands = [q, *s, at(0), *s, at(0), *s]
    if backward:
        return lib.call("lutgemm_attention_backward", at(0), *s, *operands, out, rest, at(0), at(0), at(0), at(0), *shape, *tail)
    return lib.call("lutgemm_attention", *operands, out, rest, at(0), *shape, *tail)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("bad,status", [
    (dict(q=None), H.E_BADARG), (dict(out=None), H.E_BADARG), (dict(dtype=5), H.E_BADARG), (dict(B=0), H.E_BADARG), (dict(Tk=0), H.E_BADARG),
    (dict(H_=5), H.E_BADARG), (dict(D=60), H.E_BADARG), (dict(D=136), H.E_TOOLARGE), (dict(H_=130, G=2), H.E_TOOLARGE),
    (dict(B=70000), H.E_TOOLARGE), (dict(cap=-1.0), H.E_BADARG), (dict(cap=float("inf")), H.E_BADARG), (dict(scale=float("nan")), H.E_BADARG),
    (dict(doc_q=at(0)), H.E_BADARG), (dict(q=at(8)), H.E_BADARG), (dict(stride=60), H.E_BADARG), (dict(stride=0), H.E_BADARG),
    (dict(out=at(8)), H.E_BADARG), (dict(Tq=1 << 30, H_=128, G=2), H.E_TOOLARGE)])
def test_attention_refuses_before_it_launches(lib, backward, bad, status):
    assert attention(lib, backward, **bad) == (status, [])


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attention_scratch(lib, backward, dtype):
    rng = random.Random(dtype + 10 * backward)
    name = "lutgemm_attention_backward_scratch_bytes" if backward else "lutgemm_attention_scratch_bytes"
    for _ in range(100):
        G = rng.randint(1, 8)
        shape = dict(B=rng.randint(1, 32), Tq=int(math.exp(rng.uniform(0, 8))), Tk=int(math.exp(rng.uniform(0, 10))), H_=G * rng.choice([1, 2, 3, 5, 8]),
                     G=G, D=8 * rng.randint(1, 16))
        docs = dict(doc_q=at(0), doc_k=at(0)) if rng.random() < 0.5 else {}
        need = lib.query(name, dtype, shape["B"], shape["Tq"], shape["Tk"], shape["H_"], G, shape["D"], int(bool(docs)))
        rc, _ = attention(lib, backward, dtype=dtype, scratch_bytes=need, **shape, **docs)
        assert rc == (H.OK if dtype == F32 and shape["D"] > 64 else E_CUDA), shape  # (as far as the tensor maps)
        if need:
            assert attention(lib, backward, dtype=dtype, scratch_bytes=need - 1, **shape, **docs) == (H.E_SCRATCH, [])
            assert attention(lib, backward, dtype=dtype, scratch=None, scratch_bytes=need, **shape, **docs) == (H.E_BADARG, [])
            assert attention(lib, backward, dtype=dtype, scratch=at(8), scratch_bytes=need, **shape, **docs) == (H.E_BADARG, [])
    if backward and dtype != F32:
        assert attention(lib, True, dtype=dtype, rest=None) == (H.E_BADARG, [])
    # fp32 operands may lie anywhere
    assert attention(lib, backward, dtype=F32, D=72, stride=7, q=at(4))[0] == H.OK


def logprobs(lib, dtype=BF16, N=100, C=1000, top=5, logits=at(0), top_logp=at(0), scratch=at(0), scratch_bytes=1 << 40):
    return lib.call("lutgemm_token_logprobs", logits, dtype, H.Size(C), H.Size(N), C, at(0), H.Size(0), top, at(0), at(0), at(0), top_logp, at(0),
                    scratch, H.Size(scratch_bytes), None)


@pytest.mark.parametrize("bad,status", [
    (dict(logits=None), H.E_BADARG), (dict(dtype=-1), H.E_BADARG), (dict(N=0), H.E_BADARG), (dict(C=0), H.E_BADARG), (dict(top=-1), H.E_BADARG),
    (dict(top=33), H.E_TOOLARGE), (dict(C=4), H.E_BADARG), (dict(top_logp=None), H.E_BADARG), (dict(N=1 << 31), H.E_TOOLARGE),
    (dict(N=3, C=100000, scratch_bytes=100), H.E_SCRATCH), (dict(N=3, C=100000, scratch=None), H.E_BADARG)])
def test_logprobs_refuse_before_they_launch(lib, bad, status):
    assert logprobs(lib, **bad) == (status, [])


def test_logprobs_scratch_and_gradient(lib):
    rng = random.Random(1)
    for _ in range(200):
        N, C = int(math.exp(rng.uniform(0, 10))), int(math.exp(rng.uniform(0.7, 14)))
        top, dtype = min(C, rng.randint(0, 32)), rng.randint(0, 2)
        need = lib.query("lutgemm_token_logprobs_scratch_bytes", H.Size(N), C, top)
        rc, calls = logprobs(lib, dtype, N, C, top, scratch_bytes=need)
        assert rc == H.OK and len(calls) == (2 if need else 1)
        if need:
            assert logprobs(lib, dtype, N, C, top, scratch_bytes=need - 1) == (H.E_SCRATCH, [])
        rc, calls = lib.call("lutgemm_token_logprobs_backward", at(0), dtype, H.Size(C), H.Size(N), C, at(0), H.Size(0), at(0), at(0), None, at(0), None)
        assert rc == H.OK and len(calls) == 1
    assert lib.call("lutgemm_token_logprobs_backward", at(0), 0, H.Size(5), H.Size(0), 5, at(0), H.Size(0), at(0), at(0), None, at(0), None) == (H.E_BADARG, [])


def test_operators_need_a_gpu():
    import torch
    import lutgemm_attention
    import lutgemm_loss
    x = torch.zeros(1, 2, 2, 8)
    for call in (lambda: lutgemm_attention.attention(x, x, x), lambda: lutgemm_attention.norm_rotate(x, x),
                 lambda: lutgemm_loss.token_logprobs(x[0, 0], torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDAtensor"):
            call()


def test_rotary_tables():
    """Angles of far positions are computed in 64 bits; rows and columns of an image turn a half of the pairs each."""
    import torch
    import lutgemm_attention
    cos, sin = lutgemm_attention.rotary_tables(1 << 17, 8, scale=4.0)
    for at_, i in ((0, 0), (131071, 0), (131071, 3), (77777, 1)):
        angle = at_ / 4.0 * 10000.0 ** (-2 * i / 8)
        assert abs(cos[at_, i].item() - math.cos(angle)) <= 2.0 ** -24 and abs(sin[at_, i].item() - math.sin(angle)) <= 2.0 ** -24
    cos, sin = lutgemm_attention.rotary_tables_2d(3, 5, 16)
    assert cos.shape == (15, 8) and cos.dtype is torch.float32
    for r in range(3):
        for c in range(5):
            for i in range(4):
                rate = 100.0 ** (-4 * i / 16)
                assert abs(sin[5 * r + c, i].item() - math.sin(r * rate)) <= 2.0 ** -24
                assert abs(cos[5 * r + c, 4 + i].item() - math.cos(c * rate)) <= 2.0 ** -24
    with pytest.raises(ValueError):
        lutgemm_attention.rotary_tables(4, 3)
    with pytest.raises(ValueError):
        lutgemm_attention.rotary_tables_2d(4, 4, 6)


def test_logprobs_refuse_rows_beyond_their_indices(lib):
    most = 1 << 27
    assert logprobs(lib, N=1, C=most)[0] == H.OK and logprobs(lib, N=1, C=most + 1) == (H.E_TOOLARGE, [])
