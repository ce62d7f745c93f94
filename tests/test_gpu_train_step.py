"""A training step on the package's own operators: the classifier's loss, the budget, the balance of the gates, the AdamW step - against
the same step put together from torch's operators in float32 and float64."""
import copy

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def _deit(dev, classes=7, **kw):
    from vtpack_amd.models.dge.deit_dge import VisionTransformer
    from vtpack_amd.synthetic import set_synthetic_router
    torch.manual_seed(0)
    m = VisionTransformer(img_size=64, patch_size=8, embed_dim=64, depth=2, num_heads=1, mlp_ratio=2, num_classes=classes,
                          split_sizes=[4, 2, 1], **kw)
    return set_synthetic_router(m, 2).to(dev).train()


def _batch(dev, classes=7, n=5):
    from vtpack_amd.synthetic import synthetic_images
    return synthetic_images(n, 64, seed=1).to(dev), torch.randint(0, classes, (n,), generator=torch.Generator().manual_seed(3)).to(dev)


@pytest.mark.parametrize("kw", [{}, {"distilled": True}, {"representation_size": 48}])
@pytest.mark.parametrize("mode", ["train", "eval"])
def test_loss_of_a_model(dev, kw, mode):
    m = _deit(dev, **kw).train(mode == "train")
    images, target = _batch(dev)
    torch.manual_seed(5)
    loss = m(images, target, label_smoothing=0.1)
    torch.manual_seed(5)                                  # the gates are sampled
    with torch.no_grad():
        feats = m.forward_features(images)
        logits = (feats[0] if "distilled" in kw else feats) @ m.head.weight.t() + m.head.bias
    want = F.cross_entropy(logits.double(), target, label_smoothing=0.1)
    assert abs(float(loss.detach()) - float(want)) <= 1e-5 * float(want)
    loss.backward()
    assert float(m.head.weight.grad.abs().max()) > 0
    if mode == "train":                                   # (the fused blocks of eval mode have no gradients)
        assert float(m.patch_embed.proj.weight.grad.abs().max()) > 0


def test_loss_of_a_pyramid(dev):
    from vtpack_amd.models.dge.pvt_dge import PyramidVisionTransformer
    torch.manual_seed(0)
    m = PyramidVisionTransformer(img_size=128, patch_size=4, num_classes=9, embed_dims=[64, 64, 64, 64], num_heads=[1, 1, 1, 1], mlp_ratios=[2] * 4,
                                 depths=[1, 1, 1, 1], sr_ratios=[8, 4, 2, 1], split_sizes=[[4, 2, 1]] * 4, qkv_bias=True).to(dev).eval()
    images = torch.randn(3, 3, 128, 128, generator=torch.Generator().manual_seed(0)).to(dev)
    target = torch.tensor([1, -100, 8], device=dev)
    with torch.no_grad():
        rows = m.loss(images, target, reduction="none")
        logits = m(images)
    want = F.cross_entropy(logits.double(), target, reduction="none")
    assert float((rows.double() - want).abs().max()) <= 1e-4 and float(rows[1]) == 0


@pytest.mark.parametrize("state_bits", [32, 8])
def test_a_step_is_the_step_of_its_parts(dev, state_bits):
    """Two steps; loss, gradients and weights against torch's operators on a copy with the same gate samples."""
    from vtpack_amd import harness
    from vtpack_amd.optim import AdamW
    ours = _deit(dev)
    theirs = copy.deepcopy(ours)
    images, target = _batch(dev)
    how = dict(dge_enable=True, dge_budget=0.4, dge_lr_scale=2.0)
    opt = AdamW(harness.weight_decay_groups(ours, 0.05), lr=1e-3, state_bits=state_bits)
    ref = torch.optim.AdamW(harness.weight_decay_groups(theirs, 0.05), lr=1e-3)
    assert len(opt.param_groups) == 2 and opt.param_groups[1]["weight_decay"] == 0.0
    for k in range(2):
        torch.manual_seed(11 + k)
        out = harness.train_step(ours, images, target, opt, label_smoothing=0.1, balance_scale=0.3, clip_grad=1.0, **how)
        torch.manual_seed(11 + k)
        logits = theirs(images)
        loss_cls = F.cross_entropy(logits, target, label_smoothing=0.1)
        loss_dge, ratio, _ = harness.budget_loss(theirs, images, 0.4, 2.0)
        balance = 0
        for blk in theirs.blocks:
            p, hard = blk.dge.states["gate_logits"].softmax(-1).reshape(-1, 3), blk.dge.states["gate"].detach().reshape(-1, 3)
            balance = balance + 3 * (hard.mean(0) * p.mean(0)).sum() / 2
        ref.zero_grad()
        (loss_cls + loss_dge + 0.3 * balance).backward()
        norm = torch.nn.utils.clip_grad_norm_(theirs.parameters(), 1.0)
        ref.step()
        for name, want in (("loss_cls", loss_cls), ("loss_dge", loss_dge), ("dge_ratio", ratio), ("loss_balance", balance), ("grad_norm", norm)):
            assert abs(float(out[name]) - float(want)) <= 2e-4 * abs(float(want)) + 1e-7, name
        assert out["gate_counts"].shape == (2, 3) and out["gate_counts"].sum(1).tolist() == [20, 20]
        for (name, p), q in zip(ours.named_parameters(), theirs.parameters()):
            if q.grad is None:
                assert p.grad is None
                continue
            # chains of fp32 products on both sides
            assert float((p.grad - q.grad).norm()) <= 1e-3 * float(q.grad.norm()) + 1e-7, name
        if k == 0:
            # the first step moves a weight by lr times the sign of its gradient: the same where the gradient is not next to zero
            for (name, p), q in zip(ours.named_parameters(), theirs.parameters()):
                if q.grad is not None:
                    clear = q.grad.abs() > 1e-2 * q.grad.abs().max()
                    assert float((p - q)[clear].abs().max()) <= 2e-5, name


def test_an_epoch(dev):
    from vtpack_amd import harness
    from vtpack_amd.optim import AdamW
    m = _deit(dev)
    batches = list(harness.synthetic_loader(3, 4, 64, num_classes=7, seed=3))
    opt = AdamW(harness.weight_decay_groups(m, 0.05), lr=1e-3, state_bits=8)
    before = m.head.weight.detach().clone()
    stats = harness.train_one_epoch(batches, m, opt, dev, label_smoothing=0.1, dge_enable=True, dge_budget=0.5, balance_scale=0.01)
    assert set(stats) == {"loss", "loss_cls", "loss_dge", "dge_ratio", "loss_balance", "lr"} and stats["lr"] == 1e-3
    assert m.training and not torch.equal(before, m.head.weight) and 1.0 <= stats["loss_balance"] <= 3.0
    # the fused path sees the weights as they are now (its copies of them are made anew)
    m.eval()
    with torch.no_grad():
        fused, plain = m(batches[0][0].to(dev)), m.set_fused(False)(batches[0][0].to(dev))
    assert float((fused - plain).norm()) <= 1e-4 * float(plain.norm())


def test_through_a_wrapper(dev):
    """A DistributedDataParallel-style wrapper sees the training pass as its own forward."""
    from vtpack_amd import harness
    from vtpack_amd.optim import AdamW

    class Wrapper(torch.nn.Module):
        def __init__(self, module):
            super().__init__()
            self.module, self.calls = module, 0

        def forward(self, *a, **k):
            self.calls += 1
            return self.module(*a, **k)

    w = Wrapper(_deit(dev))
    out = harness.train_step(w, *_batch(dev), AdamW(w.parameters()), dge_enable=True, balance_scale=1.0)
    assert w.calls == 1 and torch.isfinite(out["loss"])


def test_refusals(dev):
    from vtpack_amd import harness
    from vtpack_amd.optim import AdamW
    m = _deit(dev)
    images, target = _batch(dev)
    with pytest.raises(RuntimeError, match="training mode"):
        harness.train_step(m.eval(), images, target, AdamW(m.parameters()))
    with pytest.raises(RuntimeError, match="training mode"):
        m.blocks[0].dge.balance()
    m.train()
    with pytest.raises(TypeError, match="float32"):
        harness.train_step(m.bfloat16(), images.bfloat16(), target, AdamW(m.parameters()))
    with pytest.raises(ValueError, match="DynamicGrainedEncoder"):
        harness.balance_loss(torch.nn.Linear(3, 3))


@pytest.mark.parametrize("fused", [True, False])
def test_an_evaluation_leaves_nothing_of_the_training_pass(dev, fused):
    """The balance is that of a training pass: behind an evaluation there is none, the pass's graph is given up and the model can be
    copied."""
    m = _deit(dev)
    images, target = _batch(dev)
    m(images, target).backward()
    assert all(blk.dge.balance()[1].sum() > 0 for blk in m.blocks)
    m.eval().set_fused(fused)
    with torch.no_grad():
        m(images)
    for blk in m.blocks:
        assert "gate_logits" not in blk.dge.states
    if not fused:                                         # (a fused pass leaves values that are worked out when they are read)
        copy.deepcopy(m)
    m.train()
    for blk in m.blocks:
        with pytest.raises(RuntimeError, match="training mode"):
            blk.dge.balance()
    m(images, target)
    assert all(blk.dge.balance()[1].sum() > 0 for blk in m.blocks)


def test_an_epoch_ends_before_a_loss_that_is_not_finite_moves_anything(dev):
    from vtpack_amd import harness
    from vtpack_amd.optim import AdamW
    m = _deit(dev)
    batches = list(harness.synthetic_loader(1, 4, 64, num_classes=7, seed=3))
    opt = AdamW(harness.weight_decay_groups(m, 0.05), lr=1e-3, state_bits=8)
    harness.train_one_epoch(batches, m, opt, dev)
    with torch.no_grad():
        m.head.bias[2] = float("nan")

    def everything():
        tensors = [p.detach() for p in m.parameters()] + [t for p in m.parameters() for t in opt.state.get(p, {}).values() if torch.is_tensor(t)]
        return [t.contiguous().view(-1).view(torch.uint8).clone() for t in tensors], [g["step"] for g in opt.param_groups]

    tensors, steps = everything()
    with pytest.raises(FloatingPointError, match="nan"):
        harness.train_one_epoch(batches, m, opt, dev)
    now, after = everything()
    assert steps == after == [1] * len(steps) and all(torch.equal(a, b) for a, b in zip(tensors, now))
    # a step by itself looks when it is asked to
    images, target = (t.to(dev) for t in batches[0])
    with pytest.raises(FloatingPointError):
        harness.train_step(m, images, target, opt, finite=True)
    assert all(torch.equal(a, b) for a, b in zip(tensors, everything()[0]))
