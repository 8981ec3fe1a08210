"""Data-parallel AppMult-aware training launcher (one process per GPU, NCCL):

    python -m torch.distributed.run --nproc-per-node N --master-addr 127.0.0.1 lutgemm_train.py \\
        [--lut-file FILE] [--bits 7] [--batch 256] [--steps 100] [--lr 0.01] [--ste] [--conv-impl fused]
        [--model vit_s --attention fused [--qk-norm] [--rotary] [--logit-cap 30] [--class-query]] [--fused-loss]

What the reference's single-GPU loop does per step (micronet+/app_train.py:23-36: forward, cross-entropy,
backward, optimizer step) with the batch sharded over the ranks and the parameter gradients averaged by
bucketed all-reduce.  Without --lut-file the benchmark's synthetic multiplier is used; data is synthetic
(N(0,1) images of the CIFAR shape, uniform labels) because no dataset ships with this repository - plug a
DataLoader with a DistributedSampler into `batches` for real data.  Observer statistics (activation /
weight ranges) stay per rank, like the per-GPU batch-norm statistics."""
from __future__ import annotations

import argparse
import os
import time

import torch
import torch.distributed as dist
import torch.nn.functional as F

import self_ops
from lutgemm_dp import OverlappedGradReducer
from lutgemm_layers import prepare
from lutgemm_loss import token_logprobs
from lutgemm_luts import synthetic_multiplier, window_difference_gradients
from lutgemm_models import MODELS


def install_tables(device, bits: int, lut_file: str | None) -> None:
    if lut_file:
        self_ops.init_lookup_tables(device, lut_file, bits)
    else:
        fp = synthetic_multiplier(bits, seed=0)
        ga, gb = window_difference_gradients(fp, max(1, (1 << bits) // 16))
        self_ops.set_lookup_tables(device, fp, ga, gb, bits)


def build(device, bits: int, conv_impl: str = "layer", use_ste: bool = False, lr: float = 0.01, model_name: str = "resnet18",
          **model_options):
    """`model_options` go to the network's constructor (`lutgemm_models.ViT`: attention, qk_norm, rotary, logit_cap, class_query)."""
    torch.manual_seed(0)  # identical initial weights on every rank
    ctor, _, classes = MODELS[model_name]
    model = ctor(classes, **model_options).to(device)
    prepare(model, a_bits=bits, w_bits=bits, use_ste_gradient=use_ste, conv_impl=conv_impl)
    model = model.to(memory_format=torch.channels_last).train()
    opt = torch.optim.SGD(model.parameters(), lr=lr, momentum=0.9)
    return model, opt


def train_step(model, opt, reducer, images, labels, fused_loss: bool = False):
    """One step: forward, cross-entropy, backward with the bucketed gradient all-reduce launched from hooks
    while backward runs (`reducer`: an OverlappedGradReducer over the model's parameters), optimizer step.  `fused_loss`: the
    cross-entropy by `lutgemm_loss.token_logprobs` instead of PyTorch, the mean over the labels that are not -100 too."""
    reducer.zero_grad()
    logits = model(images)
    if fused_loss:
        loss = -token_logprobs(logits, labels)[0].sum() / (labels != -100).sum()
    else:
        loss = F.cross_entropy(logits, labels)
    loss.backward()
    reducer.finish()
    opt.step()
    return loss


@torch.no_grad()
def evaluate(model, batches):
    """Top-1 accuracy over (images, labels) batches, without building autograd graphs (the reference's test loop
    runs with gradients enabled, micronet+/app_train.py:39-85); observers are frozen by eval()."""
    was_training = model.training
    model.eval()
    correct = total = 0
    for images, labels in batches:
        correct += int((model(images).argmax(dim=1) == labels).sum())
        total += labels.numel()
    model.train(was_training)
    return correct / max(1, total)


@torch.no_grad()
def evaluate_top(model, batches, top: int = 5):
    """Over (images, labels) batches: top-1 and top-`top` accuracy, mean negative log probability of the labels and mean entropy of
    the answers, in one pass over the logits (`lutgemm_loss.token_logprobs`); one read by the host, at the end.  Images whose label is
    -100 do not count; without any that does, all four are zero."""
    was_training = model.training
    model.eval()
    sums = None
    for images, labels in batches:
        logp, entropy, _, answers = token_logprobs(model(images), labels, top=top)
        hits, given = answers == labels[:, None], labels != -100
        batch = torch.stack([hits[:, 0].sum(), hits.sum(), -logp.double().sum(), torch.where(given, entropy, 0.0).double().sum(),
                             given.sum()])
        sums = batch if sums is None else sums + batch
    model.train(was_training)
    names = ("top1", f"top{top}" if top > 1 else "top1", "nll", "entropy")
    return dict(zip(names, (sums[:4] / sums[4].clamp(min=1)).tolist() if sums is not None else (0.0,) * 4))


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--model", choices=sorted(MODELS), default="resnet18")
    ap.add_argument("--lut-file", default=None)
    ap.add_argument("--bits", type=int, default=7, choices=[4, 6, 7, 8])
    ap.add_argument("--batch", type=int, default=256, help="per-GPU batch")
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--lr", type=float, default=0.01)
    ap.add_argument("--ste", action="store_true", help="straight-through backward instead of the gradient tables")
    ap.add_argument("--conv-impl", choices=["layer", "fused", "unfold"], default="layer")
    ap.add_argument("--attention", choices=["library", "fused"], default="library", help="vit_s: exact attention of PyTorch or of this package")
    ap.add_argument("--qk-norm", action="store_true", help="vit_s, fused attention: norms of queries and keys")
    ap.add_argument("--rotary", action="store_true", help="vit_s, --qk-norm: positions as rotations")
    ap.add_argument("--logit-cap", type=float, default=0.0, help="vit_s, fused attention: cap of the attention logits (0: none)")
    ap.add_argument("--class-query", action="store_true", help="vit_s, fused attention: the last block for the class token alone")
    ap.add_argument("--fused-loss", action="store_true", help="loss, and answers beyond the first in evaluation, by this package's kernels")
    ap.add_argument("--eval-batches", type=int, default=0, help="synthetic batches to evaluate after training")
    args = ap.parse_args()
    options = dict(attention=args.attention, qk_norm=args.qk_norm, rotary=args.rotary, logit_cap=args.logit_cap,
                   class_query=args.class_query)
    if args.model != "vit_s":
        if args.attention != "library" or args.qk_norm or args.rotary or args.logit_cap or args.class_query:
            ap.error("--attention, --qk-norm, --rotary, --logit-cap and --class-query belong to --model vit_s")
        options = {}
    rank, world = int(os.environ.get("RANK", "0")), int(os.environ.get("WORLD_SIZE", "1"))
    device = torch.device(f"cuda:{int(os.environ.get('LOCAL_RANK', '0'))}")
    torch.cuda.set_device(device)
    if world > 1:
        dist.init_process_group("nccl", device_id=device)
    install_tables(device, args.bits, args.lut_file)
    model, opt = build(device, args.bits, args.conv_impl, args.ste, args.lr, args.model, **options)
    _, image_shape, classes = MODELS[args.model]
    reducer = OverlappedGradReducer(model.parameters())
    g = torch.Generator().manual_seed(100 + rank)
    t0 = time.time()
    for step in range(args.steps):
        images = torch.randn(args.batch, *image_shape, generator=g).pin_memory().to(device, non_blocking=True)
        labels = torch.randint(0, classes, (args.batch,), generator=g).pin_memory().to(device, non_blocking=True)
        loss = train_step(model, opt, reducer, images, labels, args.fused_loss)
        if rank == 0 and (step % 10 == 0 or step == args.steps - 1):
            print(f"step {step:4d}  loss {loss.item():.4f}  {world * args.batch * (step + 1) / (time.time() - t0):.0f} img/s",
                  flush=True)
    if args.eval_batches:
        data = [(torch.randn(args.batch, *image_shape, generator=g).to(device),
                 torch.randint(0, classes, (args.batch,), generator=g).to(device)) for _ in range(args.eval_batches)]
        if args.fused_loss:
            found = evaluate_top(model, data)
            if rank == 0:
                print(f"evaluation on {args.eval_batches} synthetic batches: " + ", ".join(f"{k} {v:.4f}" for k, v in found.items()),
                      flush=True)
        acc = evaluate(model, data)
        if rank == 0:
            print(f"eval accuracy on {args.eval_batches} synthetic batches: {acc:.4f}", flush=True)
    if world > 1:
        dist.destroy_process_group()


if __name__ == "__main__":
    main()
