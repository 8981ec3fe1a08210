"""Log probabilities, entropy and most probable classes of rows of logits in one pass over them (`token_logprobs`), with the
gradient of the first two: the loss of `lutgemm_train.train_step` with `fused_loss=True` and the answers that
`lutgemm_train.evaluate` counts beyond the first.  CUDA logits in fp32, bf16 or fp16; there is no fallback without the library."""
from __future__ import annotations

import torch

import approx_ops


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0, ignore_index: int = -100):
    """(logp, entropy, top_logp, top_index) of the rows of logits [..., C]: the log probability of targets [...] (int64 classes), the
    entropy of the row's distribution, both fp32 [...], and the log probabilities and classes of its `top` (0 to 32) most
    probable classes [..., top], the lower class first among equals.

    Rows whose target is `ignore_index` have logp 0 and no gradient through it; a target that is no class gives NaN.  Logits of
    -inf are classes without probability; a row of nothing else has logp -inf, entropy 0 and no gradient.  Gradients of logp and
    entropy reach the logits; the answers have none."""
    return approx_ops.torch_operators().token_logprobs(logits, targets, top, ignore_index)
