"""What a transformer block computes between its projections, exact while the projections are approximate: norm of every head of
queries and keys with the rotation by position (`norm_rotate`), and softmax attention (`attention`).  `lutgemm_models.ViT` runs
on them with `attention="fused"`.

Operands are CUDA tensors [B, T, heads, D] in fp32, bf16 or fp16, read by their strides (views of one projection's output need
no copy; the last axis has to be contiguous), sums and statistics are fp32, results are contiguous and rounded once.  Calls run
on the current stream of the operands' device and keep nothing; there is no fallback without the CUDA library."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

import approx_ops

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # LUTGEMM_F32, LUTGEMM_BF16, LUTGEMM_F16


def _check_heads(x: torch.Tensor, name: str, like: torch.Tensor = None) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not x.is_cuda:
        raise RuntimeError(f"{name} must be a CUDAtensor")
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"{name} must be of type torch.float32, torch.bfloat16 or torch.float16")
    if x.dim() != 4:
        raise RuntimeError(f"{name} must be [B, T, heads, D], got {tuple(x.shape)}")
    if like is not None and (x.dtype is not like.dtype or x.get_device() != like.get_device()):
        raise RuntimeError(f"{name} must be of type {like.dtype} on {like.device}")


def _check_side(x: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, like: torch.Tensor) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if x.dtype is not dtype:
        raise RuntimeError(f"{name} must be of type {dtype}")
    if x.get_device() != like.get_device():
        raise RuntimeError(f"{name} must be on {like.device}")
    if tuple(x.shape) != shape:
        raise RuntimeError(f"{name} has shape {tuple(x.shape)}, expected {shape}")


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as the kernels read it: by the strides of its first three axes."""
    return x if x.stride(3) == 1 or x.shape[3] == 1 else x.contiguous()


def _vectors(x: torch.Tensor) -> torch.Tensor:
    """The same where 16-bit operands are read by bulk copies of eight values and more: a copy of one that lies differently or repeats
    itself."""
    if x.dtype is torch.float32:
        return _rows(x)
    sb, st, sh, sd = x.stride()
    if sd == 1 and sb and st and sh and not ((sb | st | sh) & 7 or x.data_ptr() & 15):
        return x
    B, T, heads, D = x.shape
    if (sd != 1 and D > 1) or x.data_ptr() & 15 or any(n > 1 and (s & 7 or not s) for n, s in ((B, sb), (T, st), (heads, sh))):
        return x.clone(memory_format=torch.contiguous_format)
    return x


def _at(x: torch.Tensor):
    return (x.data_ptr(), *x.stride()[:3])


def rotary_tables(length: int, rot: int, base: float = 10000.0, scale: float = 1.0, device=None):
    """cos and sin [length, rot / 2] in fp32 of the angles (position / scale) * base^(-2i / rot), computed in 64 bits (far positions
    lose their angle in 32).  `scale` above one fits longer rows into the angles that a network has seen."""
    if rot < 0 or rot % 2:
        raise ValueError(f"rot must be even, got {rot}")
    rates = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    angles = torch.outer(torch.arange(length, dtype=torch.float64) / scale, rates)
    return angles.cos().float().to(device), angles.sin().float().to(device)


def rotary_tables_2d(height: int, width: int, rot: int, base: float = 100.0, device=None):
    """The same for the patches of an image in row order: the first half of the pairs turn by a patch's row, the others by its
    column.  [height * width, rot / 2]."""
    if rot < 0 or rot % 4:
        raise ValueError(f"rot must be a multiple of 4, got {rot}")
    rates = base ** (-torch.arange(0, rot, 4, dtype=torch.float64) / max(rot, 1))
    rows = torch.arange(height, dtype=torch.float64).repeat_interleave(width)
    columns = torch.arange(width, dtype=torch.float64).repeat(height)
    angles = torch.cat([torch.outer(rows, rates), torch.outer(columns, rates)], dim=1)
    return angles.cos().float().to(device), angles.sin().float().to(device)


def _norm_rotate_forward(q, k, qw, kw, cos, sin, positions, interleaved, eps):
    B, T, H, D = q.shape
    G, dev = k.shape[2], q.device
    qo = torch.empty((B, T, H, D), dtype=q.dtype, device=dev)
    ko = torch.empty((B, T, G, D), dtype=q.dtype, device=dev)
    if B * T:
        with approx_ops._guard(dev):
            rc = approx_ops.library().lutgemm_norm_rotate(
                *_at(q), *_at(k), qw.data_ptr() if qw is not None else None, kw.data_ptr() if kw is not None else None, cos.data_ptr(),
                sin.data_ptr(), cos.shape[0], positions.data_ptr() if positions is not None else None, qo.data_ptr(), ko.data_ptr(),
                _DTYPES[q.dtype], B, T, H, G, D, 2 * cos.shape[1], interleaved, eps, approx_ops._stream_ptr(dev))
        approx_ops._check(rc, "norm_rotate")
    return qo, ko


class _NormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, cos, sin, positions, interleaved, eps):
        B, T, H, D = q.shape
        ctx.cfg = (B, T, H, k.shape[2], D, 2 * cos.shape[1], interleaved, eps)
        ctx.save_for_backward(q, k, qw, kw, cos, sin, positions)
        return _norm_rotate_forward(q, k, qw, kw, cos, sin, positions, interleaved, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, qw, kw, cos, sin, positions = ctx.saved_tensors
        B, T, H, G, D, rot, interleaved, eps = ctx.cfg
        dq = torch.empty((B, T, H, D), dtype=q.dtype, device=q.device)
        dk = torch.empty((B, T, G, D), dtype=q.dtype, device=q.device)
        dqw = torch.empty_like(qw) if qw is not None and ctx.needs_input_grad[2] else None
        dkw = torch.empty_like(kw) if kw is not None and ctx.needs_input_grad[3] else None
        if B * T == 0:
            return (dq, dk, dqw.zero_() if dqw is not None else None, dkw.zero_() if dkw is not None else None) + (None,) * 5
        gq, gk = _rows(gq), _rows(gk)
        lib = approx_ops.library()
        with approx_ops._guard(q.device):
            nbytes = 0
            if dqw is not None or dkw is not None:
                nbytes = approx_ops._scratch_bytes("lutgemm_norm_rotate_backward_scratch_bytes", q.get_device(), D)
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
            rc = lib.lutgemm_norm_rotate_backward(
                *_at(gq), *_at(gk), *_at(q), *_at(k), qw.data_ptr() if qw is not None else None,
                kw.data_ptr() if kw is not None else None, cos.data_ptr(), sin.data_ptr(), cos.shape[0],
                positions.data_ptr() if positions is not None else None, dq.data_ptr(), dk.data_ptr(),
                dqw.data_ptr() if dqw is not None else None, dkw.data_ptr() if dkw is not None else None, _DTYPES[q.dtype], B, T, H, G,
                D, rot, interleaved, eps, scratch.data_ptr() if nbytes else None, nbytes, approx_ops._stream_ptr(q.device))
        approx_ops._check(rc, "norm_rotate (backward)")
        return dq, dk, dqw, dkw, None, None, None, None, None


def norm_rotate(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor = None, k_weight: torch.Tensor = None,
                cos: torch.Tensor = None, sin: torch.Tensor = None, positions: torch.Tensor = None, layout: str = "half",
                eps: float = 1e-6):
    """(q, k) with every head divided by its root mean square (of D values, plus eps), times the weights [D] (None: 1), and the
    first `2 * cos.shape[1]` values of it turned by the token's angles: pairs (i, i + half) in the "half" layout, (2i, 2i + 1) in
    the "interleaved" one.  Without tables nothing is turned.

    q [B, T, H, D], k [B, T, G, D], D even and at most 256; cos, sin: fp32 tables by position (`rotary_tables`); positions: int32 or
    int64 [B, T] (default 0 .. T-1): a negative one leaves its token unturned (a class token), one beyond the table makes the
    token's turned values NaN.  Gradients for q, k and the weights."""
    _check_heads(q, "q")
    _check_heads(k, "k", q)
    B, T, H, D = q.shape
    if k.shape[0] != B or k.shape[1] != T or k.shape[3] != D:
        raise RuntimeError(f"k has shape {tuple(k.shape)}, expected {(B, T, 'heads', D)}")
    if H == 0 or k.shape[2] == 0 or D == 0 or D % 2 or D > 256:
        raise RuntimeError(f"heads must be at least one of an even size up to 256, got {H} and {k.shape[2]} of {D}")
    if layout not in ("half", "interleaved"):
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    if (cos is None) != (sin is None):
        raise RuntimeError("cos and sin belong together")
    if cos is None:
        cos = sin = torch.empty((T, 0), dtype=torch.float32, device=q.device)
        positions = None
    if cos.dim() != 2 or 2 * cos.shape[1] > D:
        raise RuntimeError(f"cos must be [positions, at most {D // 2}], got {tuple(cos.shape)}")
    for x, name in ((cos, "cos"), (sin, "sin")):
        _check_side(x, name, torch.float32, tuple(cos.shape), q)
    if positions is None:
        if cos.shape[0] < T:
            raise RuntimeError(f"cos and sin have {cos.shape[0]} positions, the rows {T}")
    else:
        if positions.dtype is torch.int64:
            # (beyond 32 bits is beyond any table)
            positions = positions.clamp(-1, 0x7FFFFFFF).to(torch.int32)
        _check_side(positions, "positions", torch.int32, (B, T), q)
        positions = positions.contiguous()
    weights = []
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            _check_side(w, name, w.dtype if w.dtype in _DTYPES else torch.float32, (D,), q)
            w = w.float().contiguous()
        weights.append(w)
    args = (_rows(q), _rows(k), weights[0], weights[1], cos.contiguous(), sin.contiguous(), positions, layout == "interleaved", float(eps))
    # (without a backward pass the call through autograd would be a fifth of its time)
    wanted = torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in args[:4])
    return _NormRotate.apply(*args) if wanted else _norm_rotate_forward(*args)


def _masks(scale, cap, slopes, causal, prefix, doc_q, doc_k):
    """The arguments of the library's calls that say who sees whom."""
    return (scale, cap, slopes.data_ptr() if slopes is not None else None, causal, prefix.data_ptr() if prefix is not None else None,
            *((doc_q.data_ptr(), doc_q.stride(0), doc_k.data_ptr(), doc_k.stride(0)) if doc_q is not None else (None, 0, None, 0)))


def _attention_forward(training, q, k, v, scale, cap, slopes, causal, prefix, doc_q, doc_k):
    """(out, rest, lse); rest, which the backward pass of 16-bit operands wants: what the rounding of out leaves."""
    B, Tq, H, D = q.shape
    Tk, G, dev = k.shape[1], k.shape[2], q.device
    out = torch.empty((B, Tq, H, D), dtype=q.dtype, device=dev)
    lse = torch.empty((B, G, Tq * H // G), dtype=torch.float32, device=dev)
    rest = torch.empty_like(out) if training and q.dtype is not torch.float32 else None
    dtype = _DTYPES[q.dtype]
    with approx_ops._guard(dev):
        nbytes = approx_ops._scratch_bytes("lutgemm_attention_scratch_bytes", dev.index, dtype, B, Tq, Tk, H, G, D, doc_k is not None)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        rc = approx_ops.library().lutgemm_attention(
            *_at(q), *_at(k), *_at(v), out.data_ptr(), rest.data_ptr() if rest is not None else None, lse.data_ptr(), dtype, B, Tq, Tk,
            H, G, D, *_masks(scale, cap, slopes, causal, prefix, doc_q, doc_k), scratch.data_ptr() if nbytes else None, nbytes,
            approx_ops._stream_ptr(dev))
    approx_ops._check(rc, "attention")
    return out, rest, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, cap, slopes, causal, prefix, doc_q, doc_k):
        out, rest, lse = _attention_forward(True, q, k, v, scale, cap, slopes, causal, prefix, doc_q, doc_k)
        ctx.save_for_backward(q, k, v, out, rest, lse, slopes, prefix, doc_q, doc_k)
        ctx.cfg = (scale, cap, causal)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        q, k, v, out, rest, lse, slopes, prefix, doc_q, doc_k = ctx.saved_tensors
        scale, cap, causal = ctx.cfg
        B, Tq, H, D = q.shape
        Tk, G = k.shape[1], k.shape[2]
        go = _vectors(go)
        dq = torch.empty((B, Tq, H, D), dtype=q.dtype, device=q.device)
        dk = torch.empty((B, Tk, G, D), dtype=q.dtype, device=q.device)
        dv = torch.empty((B, Tk, G, D), dtype=q.dtype, device=q.device)
        lib, dtype = approx_ops.library(), _DTYPES[q.dtype]
        with approx_ops._guard(q.device):
            nbytes = approx_ops._scratch_bytes("lutgemm_attention_backward_scratch_bytes", q.get_device(), dtype, B, Tq, Tk, H, G, D,
                                               doc_k is not None)
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            rc = lib.lutgemm_attention_backward(*_at(go), *_at(q), *_at(k), *_at(v), out.data_ptr(),
                                                rest.data_ptr() if rest is not None else None, lse.data_ptr(), dq.data_ptr(),
                                                dk.data_ptr(), dv.data_ptr(), dtype, B, Tq, Tk, H, G, D,
                                                *_masks(scale, cap, slopes, causal, prefix, doc_q, doc_k), scratch.data_ptr(), nbytes,
                                                approx_ops._stream_ptr(q.device))
        approx_ops._check(rc, "attention (backward)")
        return dq, dk, dv, None, None, None, None, None, None, None


class _Empty(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v):
        ctx.like = [x.shape for x in (q, k, v)]
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device)

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        return tuple(torch.zeros(s, dtype=go.dtype, device=go.device) for s in ctx.like)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float = None, cap: float = 0.0, slopes: torch.Tensor = None,
              causal: bool = False, prefix: torch.Tensor = None, documents: torch.Tensor = None,
              query_documents: torch.Tensor = None) -> torch.Tensor:
    """Softmax attention, [B, Tq, H, D]: q [B, Tq, H, D], k and v [B, Tk, G, D], G a divisor of H (query head h reads key head
    h / (H/G), at most 64 read one), D a multiple of 8 up to 128.

    scale      of the scores q.k, by default D^-0.5
    cap        above zero: scores s become cap * tanh(s / cap)
    slopes     fp32 [H]: scores fall by slopes[h] per place of distance
    causal     queries see keys up to their own place; the last query stands at the last key
    prefix     int32 [B], with `causal`: the first prefix[b] keys are seen by all queries
    documents  int32 [B, Tk]: tokens see tokens of their own id; ids below zero are padding, whose q, k and v may hold anything.
               Queries have the ids of their places, or `query_documents` [B, Tq]

    A query that sees nothing gives zeros and no gradient.  Values that some query of the same row of the batch sees have to be
    finite (a probability of zero does not hide an infinity from its neighbours); padding need not be.  Gradients for q, k and v;
    they do not depend on the order in which the GPU runs."""
    _check_heads(q, "q")
    _check_heads(k, "k", q)
    _check_heads(v, "v", q)
    B, Tq, H, D = q.shape
    Tk, G = k.shape[1], k.shape[2]
    if tuple(k.shape) != (B, Tk, G, D) or k.shape != v.shape:
        raise RuntimeError(f"k and v must both be {(B, 'Tk', 'heads', D)}, got {tuple(k.shape)} and {tuple(v.shape)}")
    if G == 0 or H == 0 or H % G or H // G > 64:
        raise RuntimeError(f"q's {H} heads must be a multiple of the {G} heads of k and v, at most 64 to one")
    if D == 0 or D % 8 or D > 128:
        raise RuntimeError(f"the size of a head must be a multiple of 8 up to 128, got {D}")
    cap = float(cap)
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 <= cap < float("inf") or scale != scale or abs(scale) == float("inf"):
        raise ValueError(f"cap must not be negative, cap and scale must be finite, got {cap} and {scale}")
    if slopes is not None:
        _check_side(slopes, "slopes", torch.float32, (H,), q)
        if slopes.requires_grad:
            raise RuntimeError("slopes have no gradient")
        slopes = slopes.contiguous()
    if prefix is not None:
        if not causal:
            raise RuntimeError("prefix belongs to causal attention")
        _check_side(prefix, "prefix", torch.int32, (B,), q)
        prefix = prefix.contiguous()
    if query_documents is not None and documents is None:
        raise RuntimeError("query_documents belong to documents")
    if documents is not None:
        _check_side(documents, "documents", torch.int32, (B, Tk), q)
        documents = documents if documents.stride(1) == 1 or Tk <= 1 else documents.contiguous()
        if query_documents is None:
            if Tq > Tk:
                raise RuntimeError("more queries than keys need query_documents")
            query_documents = documents[:, Tk - Tq:]
        else:
            _check_side(query_documents, "query_documents", torch.int32, (B, Tq), q)
            query_documents = query_documents if query_documents.stride(1) == 1 or Tq <= 1 else query_documents.contiguous()
    if B * Tq == 0 or Tk == 0:  # nothing to see: zeros, whose gradients are zeros
        return _Empty.apply(q, k, v)
    args = (_vectors(q), _vectors(k), _vectors(v), scale, cap, slopes, bool(causal), prefix, query_documents, documents)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attention.apply(*args)
    return _attention_forward(False, *args)[0]
