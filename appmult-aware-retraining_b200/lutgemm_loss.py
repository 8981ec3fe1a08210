"""Log probabilities, entropy and most probable classes of rows of logits in one pass over them (`token_logprobs`), with the
gradient of the first two: the loss of `lutgemm_train.train_step` with `fused_loss=True` and the answers that
`lutgemm_train.evaluate` counts beyond the first.  CUDA logits in fp32, bf16 or fp16; there is no fallback without the library."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

import approx_ops
from lutgemm_attention import _DTYPES


def _logprobs_forward(logits, targets, top, ignore_index):
    """(logp, entropy, top_logp, top_index, stats); stats are for the backward pass."""
    N, C = logits.shape
    dev = logits.device
    logp = torch.empty(N, dtype=torch.float32, device=dev)
    entropy = torch.empty(N, dtype=torch.float32, device=dev)
    stats = torch.empty((N, 3), dtype=torch.float32, device=dev)
    top_logp = torch.empty((N, top), dtype=torch.float32, device=dev)
    top_index = torch.empty((N, top), dtype=torch.int64, device=dev)
    if N:
        with approx_ops._guard(dev):
            nbytes = approx_ops._scratch_bytes("lutgemm_token_logprobs_scratch_bytes", dev.index, N, C, top)
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
            rc = approx_ops.library().lutgemm_token_logprobs(
                logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0), N, C, targets.data_ptr(), ignore_index, top, logp.data_ptr(),
                entropy.data_ptr(), stats.data_ptr(), top_logp.data_ptr(), top_index.data_ptr(), scratch.data_ptr() if nbytes else None,
                nbytes, approx_ops._stream_ptr(dev))
        approx_ops._check(rc, "token_logprobs")
    return logp, entropy, top_logp, top_index, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, ignore_index):
        logp, entropy, top_logp, top_index, stats = _logprobs_forward(logits, targets, top, ignore_index)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_logp, top_index)
        ctx.save_for_backward(logits, targets, stats)
        ctx.ignore_index = ignore_index
        return logp, entropy, top_logp, top_index

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logp, g_entropy, _, __):
        logits, targets, stats = ctx.saved_tensors
        N, C = logits.shape
        if g_logp is None and g_entropy is None:
            return None, None, None, None
        grad = torch.empty((N, C), dtype=logits.dtype, device=logits.device)
        if N:
            g_logp = g_logp.contiguous() if g_logp is not None else None
            g_entropy = g_entropy.contiguous() if g_entropy is not None else None
            lib = approx_ops.library()
            with approx_ops._guard(logits.device):
                rc = lib.lutgemm_token_logprobs_backward(logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0), N, C,
                                                         targets.data_ptr(), ctx.ignore_index, stats.data_ptr(),
                                                         g_logp.data_ptr() if g_logp is not None else None,
                                                         g_entropy.data_ptr() if g_entropy is not None else None, grad.data_ptr(),
                                                         approx_ops._stream_ptr(logits.device))
            approx_ops._check(rc, "token_logprobs (backward)")
        return grad, None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0, ignore_index: int = -100):
    """(logp, entropy, top_logp, top_index) of the rows of logits [..., C]: the log probability of targets [...] (int64 classes), the
    entropy of the row's distribution, both fp32 [...], and the log probabilities and classes of its `top` (0 to 32) most
    probable classes [..., top], the lower class first among equals.

    Rows whose target is `ignore_index` have logp 0 and no gradient through it; a target that is no class gives NaN.  Logits of
    -inf are classes without probability; a row of nothing else has logp -inf, entropy 0 and no gradient.  Gradients of logp and
    entropy reach the logits; the answers have none."""
    if not isinstance(logits, torch.Tensor) or not isinstance(targets, torch.Tensor):
        raise TypeError("logits and targets must be torch.Tensors")
    if not logits.is_cuda:
        raise RuntimeError("logits must be a CUDAtensor")
    if logits.dtype not in _DTYPES:
        raise RuntimeError("logits must be of type torch.float32, torch.bfloat16 or torch.float16")
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise RuntimeError(f"logits must be [..., classes], got {tuple(logits.shape)}")
    if targets.dtype is not torch.int64 or targets.get_device() != logits.get_device():
        raise RuntimeError(f"targets must be of type torch.int64 on {logits.device}")
    if targets.shape != logits.shape[:-1]:
        raise RuntimeError(f"targets have shape {tuple(targets.shape)}, expected {tuple(logits.shape[:-1])}")
    C = logits.shape[-1]
    top = int(top)
    if not 0 <= top <= min(32, C):
        raise ValueError(f"top must lie between 0 and {min(32, C)}, got {top}")
    lead = targets.shape
    x = logits if logits.dim() == 2 else logits.reshape(-1, C)
    if x.stride(1) != 1 and C > 1:
        x = x.contiguous()
    t = targets.reshape(-1).contiguous()
    if x.requires_grad and torch.is_grad_enabled():
        out = _TokenLogprobs.apply(x, t, top, int(ignore_index))
    else:
        out = _logprobs_forward(x, t, top, int(ignore_index))[:4]
    if logits.dim() == 2:
        return out
    return out[0].view(lead), out[1].view(lead), out[2].view(*lead, top), out[3].view(*lead, top)
