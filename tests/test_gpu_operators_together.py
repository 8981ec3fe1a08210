"""Head norms, rotations, attention and log probabilities as networks and the training command use them, on a GPU."""
import subprocess
import sys

import pytest
import torch
import torch.nn.functional as F

import operators_reference as R

pytestmark = pytest.mark.gpu


def small_vit(**kw):
    from lutgemm_models import ViT
    torch.manual_seed(3)
    return ViT(image=48, patch=8, dim=64, depth=2, heads=2, mlp=128, num_classes=10, **kw).cuda()


def batch(n=4, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, 3, 48, 48, generator=g, device="cuda"), torch.randint(0, 10, (n,), generator=g, device="cuda")


def test_fused_attention_is_the_library_s_up_to_rounding():
    """The same network with either attention and either loss: fp32 all through, so results differ by the order of fp32 sums
    (a few hundred terms per sum, 30 layers of operations: 2^-24 * 300 * 30 = 5e-4 of the largest is far above what may differ)."""
    a, b = small_vit(), small_vit(attention="fused")
    b.load_state_dict(a.state_dict())
    x, y = batch()
    from lutgemm_loss import token_logprobs
    la, lb = a(x), b(x)
    assert (la - lb).abs().max() <= 5e-4 * la.abs().max()
    F.cross_entropy(la, y).backward()
    (-token_logprobs(lb, y)[0].mean()).backward()
    for (name, p), q in zip(a.named_parameters(), b.parameters()):
        assert (p.grad - q.grad).abs().max() <= 5e-4 * p.grad.abs().max() + 1e-7, name


def reference_vit(model, x, documents):
    """The fused network's forward pass from formulas in 64 bits; `model` in 64 bits."""
    x = model.patch_embed(x).flatten(2).transpose(1, 2)
    x = torch.cat([model.cls.expand(x.shape[0], -1, -1), x], dim=1) + model.pos
    place = model.place.expand(x.shape[0], -1) if model.rotary else None
    for block in model.blocks:
        B, T, D = x.shape
        q, k, v = block.qkv(block.norm1(x)).view(B, T, 3, block.heads, D // block.heads).unbind(2)
        if block.q_norm is not None:
            cos, sin = (model.cos, model.sin) if model.rotary else (None, None)
            q = R.norm_rotate(q, block.q_norm, cos, sin, place, "half", 1e-6)
            k = R.norm_rotate(k, block.k_norm, cos, sin, place, "half", 1e-6)
        asked = None
        if block.class_query:
            q, x, asked = q[:, :1], x[:, :1], documents[:, :1] if documents is not None else None
        a = R.attention(q, k, v, cap=block.logit_cap, documents=documents, query_documents=asked)
        x = x + block.proj(a.reshape(B, -1, D))
        x = x + block.fc2(F.gelu(block.fc1(block.norm2(x))))
    return model.head(model.norm(x)[:, 0])


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("options", [dict(qk_norm=True), dict(qk_norm=True, rotary=True, logit_cap=5.0), dict(class_query=True),
                                     dict(qk_norm=True, rotary=True, logit_cap=20.0, class_query=True)])
def test_network_with_all_of_them_against_64_bits(options, masked):
    model = small_vit(attention="fused", **options)
    x, y = batch()
    documents = None
    if masked:  # the last patches of some images are not there
        documents = torch.zeros(4, 37, dtype=torch.int32, device="cuda")
        documents[1, 20:] = -1
        documents[3, 1:] = -1
    from lutgemm_loss import token_logprobs
    logits = model(x, documents)
    loss = -token_logprobs(logits, y)[0].mean()
    grads = torch.autograd.grad(loss, list(model.parameters()), allow_unused=True)
    import copy
    exact = copy.deepcopy(model).double()
    want = reference_vit(exact, x.double(), documents)
    wants = torch.autograd.grad(F.cross_entropy(want, y), list(exact.parameters()), allow_unused=True)
    # 2^-24 per operation, a few hundred terms per sum, 30 layers of operations
    assert (logits - want).abs().max() <= 5e-4 * want.abs().max()
    for (name, _), g, w in zip(model.named_parameters(), grads, wants):
        assert (g is None) == (w is None), name
        if w is not None:
            assert (g - w).abs().max() <= 5e-4 * w.abs().max() + 1e-7, name


def test_training_step_with_approximate_linears():
    """A step of the training loop on the approximate layers: everything is reached, gradients arrive and parameters move."""
    from lutgemm_dp import OverlappedGradReducer
    from lutgemm_layers import prepare
    from lutgemm_train import evaluate, evaluate_top, install_tables, train_step
    install_tables(torch.device("cuda"), 7, None)
    model = small_vit(attention="fused", qk_norm=True, rotary=True, logit_cap=30.0, class_query=True)
    prepare(model, conv_impl="layer")
    model.train()
    opt = torch.optim.SGD(model.parameters(), lr=0.01)
    reducer = OverlappedGradReducer(model.parameters())
    x, y = batch(8)
    before = [p.detach().clone() for p in model.parameters()]
    loss = train_step(model, opt, reducer, x, y, fused_loss=True)
    assert torch.isfinite(loss)
    assert all(torch.isfinite(p).all() for p in model.parameters())
    assert all((p != q).any() for (n, p), q in zip(model.named_parameters(), before) if "norm" in n or "qkv.weight" in n)
    found = evaluate_top(model, [(x, y), (x, y)], top=3)
    assert abs(found["top1"] - evaluate(model, [(x, y)])) < 1e-9 and found["top1"] <= found["top3"] <= 1 and found["nll"] > 0
    with torch.no_grad():
        model.eval()
        logits = model(x).double()
    assert abs(found["nll"] - F.cross_entropy(logits, y).item()) <= 1e-5 * found["nll"]
    p = torch.softmax(logits, 1)
    assert abs(found["entropy"] + (p * p.log()).sum(1).mean().item()) <= 1e-5


def test_options_refused():
    from lutgemm_models import ViT
    for kw in (dict(attention="other"), dict(qk_norm=True), dict(logit_cap=5.0), dict(class_query=True), dict(attention="fused", rotary=True)):
        with pytest.raises(ValueError):
            ViT(image=16, patch=8, dim=32, depth=1, heads=2, mlp=32, num_classes=3, **kw)
    model = small_vit()
    with pytest.raises(ValueError, match="fused"):
        model(batch()[0], torch.zeros(4, 37, dtype=torch.int32, device="cuda"))


def test_training_command(tmp_path):
    import os
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "appmult-aware-retraining_b200")
    run = subprocess.run([sys.executable, "lutgemm_train.py", "--model", "vit_s", "--attention", "fused", "--qk-norm", "--rotary", "--logit-cap",
                          "30", "--class-query", "--fused-loss", "--batch", "2", "--steps", "2", "--eval-batches", "1"],
                         cwd=package, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    assert "step    1" in run.stdout and "top5" in run.stdout
    run = subprocess.run([sys.executable, "lutgemm_train.py", "--model", "resnet18", "--attention", "fused"], cwd=package, capture_output=True,
                         text=True, timeout=300)
    assert run.returncode == 2 and "vit_s" in run.stderr
