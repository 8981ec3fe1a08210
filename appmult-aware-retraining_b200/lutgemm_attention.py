"""What a transformer block computes between its projections, exact while the projections are approximate: norm of every head of
queries and keys with the rotation by position (`norm_rotate`), and softmax attention (`attention`).  `lutgemm_models.ViT` runs
on them with `attention="fused"`.

Operands are CUDA tensors [B, T, heads, D] in fp32, bf16 or fp16, read by their strides (views of one projection's output need
no copy; the last axis has to be contiguous), sums and statistics are fp32, results are contiguous and rounded once.  Calls run
on the current stream of the operands' device and keep nothing; second derivatives and forward-mode ones are refused, and there is no
fallback without the CUDA library."""
from __future__ import annotations

import torch

import approx_ops


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


def norm_rotate(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor = None, k_weight: torch.Tensor = None,
                cos: torch.Tensor = None, sin: torch.Tensor = None, positions: torch.Tensor = None, layout: str = "half",
                eps: float = 1e-6):
    """(q, k) with every head divided by its root mean square (of D values, plus eps), times the weights [D] (None: 1), and the
    first `2 * cos.shape[1]` values of it turned by the token's angles: pairs (i, i + half) in the "half" layout, (2i, 2i + 1) in
    the "interleaved" one.  Without tables nothing is turned.

    q [B, T, H, D], k [B, T, G, D], D even and at most 256; cos, sin: fp32 tables by position (`rotary_tables`); positions: int32 or
    int64 [B, T] (default 0 .. T-1): a negative one leaves its token unturned (a class token), one beyond the table makes the
    token's turned values NaN.  Gradients for q, k and the weights."""
    return approx_ops.torch_operators().norm_rotate(q, k, q_weight, k_weight, cos, sin, positions, layout, eps)


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

    A query that sees nothing gives zeros and no gradient.  All values but padding have to be finite, those that no query sees among
    them (a probability of zero does not hide an infinity from its neighbours).  Gradients for q, k and v; they do not depend on the
    order in which the GPU runs.  Of fp16 operands, the gradients of scores lose bits below 2^-28 of the largest that |grad_o| |v|
    allows: in their row for q, in all rows that see the same block of 128 keys for k."""
    return approx_ops.torch_operators().attention(q, k, v, scale, cap, slopes, causal, prefix, documents, query_documents)
