"""Preference, policy and distillation training through the streamed trainer: its
log-probabilities and gradients against the same model held whole, with the losses
written in plain torch.

The streamed and the whole forward run the same kernels on the same bytes, so their
logits are equal and log-probabilities are held to the bound derived in
test_losses_gpu.py. LoRA gradients go through bf16 gradients of the logits, 2^-9 of
each entry and independent of one another, and through the same bf16 backward on both
sides; 2e-2 of their RMS is the bar of the cross-entropy step (test_trainer_gpu.py),
whose gradient is rounded alike."""
import pytest
import torch

from lema_b200 import ops
from lema_b200.llama import LlamaBlock, LlamaShape, apply_lora
from lema_b200.moe import MixtralShape
from lema_b200.objectives import IGNORE, Distill, Policy, Preference, next_targets
from lema_b200.trainer import StreamedLoraTrainer

pytestmark = pytest.mark.gpu

SMALL = LlamaShape(hidden=256, heads=4, kv_heads=4, intermediate=688, vocab=512, layers=3)
U = 2.0 ** -24


def _trainer(dev, batch=4, seq=48, **kw):
    tr = StreamedLoraTrainer(SMALL, dev, batch=batch, seq=seq, seed=3, **{"lr": 0.0, **kw})
    g = torch.Generator(device=dev).manual_seed(5)
    with torch.no_grad():  # adapters that change the model
        for layer in tr.lora:
            for _, b in layer.values():
                b.copy_(torch.randn(b.shape, device=dev, generator=g) * 0.05)
    return tr


def _batch(dev, batch=4, seq=48, vocab=SMALL.vocab):
    g = torch.Generator(device=dev).manual_seed(7)
    ids = torch.randint(0, vocab, (batch, seq), device=dev, generator=g)
    labels = ids.clone()
    labels[:, :seq // 4] = IGNORE         # a prompt
    labels[1, -9:] = IGNORE               # padding
    return ids, labels


def _whole(tr, ids, adapters=True):
    """Logits of the same weights held whole, with autograd, and the LoRA leaves."""
    h = tr.embed(ids)
    leaves = []
    for b in range(tr.L):
        blk = LlamaBlock(tr.shape, quantized=True, device=tr.device)
        buf = tr.ws.ram[b].to(tr.device)
        for name in ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"):
            blk.base_projection(name).bind(tr.ws._view(buf, name + ".wq"),
                                           tr.ws._view(buf, name + ".sw"))
        blk.input_layernorm.weight.data = tr.ws._view(buf, "input_layernorm")
        blk.post_attention_layernorm.weight.data = tr.ws._view(buf, "post_attention_layernorm")
        blk.build_fused_weights()
        params = {n: (torch.nn.Parameter(a.detach().clone()),
                      torch.nn.Parameter(bb.detach().clone()))
                  for n, (a, bb) in tr.lora[b].items()}
        if adapters:
            apply_lora(blk, 16, 32.0, params=params)
        leaves.append(params)
        h = blk(h, tr.cos, tr.sin)
    return tr.head(h), leaves


def _logps(logits, targets):
    lsm = torch.log_softmax(logits.double(), -1)
    lp = lsm.gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    return torch.where(targets == IGNORE, 0.0, lp)


def _step_grads(tr, ids, labels, objective):
    """One step with the optimizer and the clipping held off: (loss, LoRA gradients)."""
    tr.opt.zero_grad(set_to_none=True)
    seen = {}
    step, clip = tr.opt.step, torch.nn.utils.clip_grad_norm_

    def grab():
        seen["g"] = [{n: (a.grad.clone(), b.grad.clone()) for n, (a, b) in layer.items()}
                     for layer in tr.lora]
    tr.opt.step = grab
    torch.nn.utils.clip_grad_norm_ = lambda params, max_norm: None
    try:
        loss = tr.train_step(ids, labels, objective=objective)
    finally:
        tr.opt.step, torch.nn.utils.clip_grad_norm_ = step, clip
    return loss, seen["g"]


def _compare(got, leaves):
    for layer, want in zip(got, leaves):
        for n, pair in layer.items():
            for g, p in zip(pair, want[n]):
                w = p.grad.float()
                rel = (g.float() - w).pow(2).mean().sqrt() / (w.pow(2).mean().sqrt() + 1e-30)
                assert rel <= 2e-2, (n, rel.item())


def _bound(lp):
    return (40 + 2.1 * 9 + 1) * U + U * lp.abs()


def test_scores(cuda_device):
    tr = _trainer(cuda_device)
    ids, labels = _batch(cuda_device)
    t = next_targets(labels)
    for adapters in (True, False):
        lp = tr.token_logprobs(ids, labels, adapters=adapters)
        with torch.no_grad():
            want = _logps(_whole(tr, ids, adapters)[0], t)
        assert lp.shape == ids.shape and lp.dtype == torch.float32
        assert ((lp.double() - want).abs() <= _bound(want)).all()
        assert (lp[t == IGNORE] == 0).all() and (lp[:, -1] == 0).all()
    with_, without = (tr.token_logprobs(ids, labels, adapters=a) for a in (True, False))
    assert (with_ - without).abs().max() > 1e-2
    # a training step after it runs with the adapters
    a = _step_grads(tr, ids, labels, None)[0]
    b = _step_grads(tr, ids, labels, None)[0]
    assert torch.equal(a, b)
    tr.close()


def test_preference_step(cuda_device):
    tr = _trainer(cuda_device)
    ids, labels = _batch(cuda_device)
    t = next_targets(labels)
    ref = tr.token_logprobs(ids, labels, adapters=False)
    obj = Preference(ref, beta=0.3, label_smoothing=0.1)
    loss, grads = _step_grads(tr, ids, labels, obj)
    logits, leaves = _whole(tr, ids)
    R = 0.3 * (_logps(logits, t) - ref.double()).sum(1)
    h = R[:2] - R[2:]
    sp = torch.nn.functional.softplus
    want = (0.9 * sp(-h) + 0.1 * sp(h)).mean()
    want.backward()
    n = (t != IGNORE).sum().item()
    slack = 0.3 * n * _bound(torch.tensor(12.0)).item()
    assert abs(loss.item() - want.item()) <= slack + 2 * U * abs(want.item())
    assert ((obj.rewards.double() - R.detach()).abs() <= slack + U * R.detach().abs()).all()
    _compare(grads, leaves)
    tr.close()


def test_policy_step_and_accumulation(cuda_device):
    tr = _trainer(cuda_device)
    ids, labels = _batch(cuda_device)
    t = next_targets(labels)
    old = tr.token_logprobs(ids, labels)
    ref = tr.token_logprobs(ids, labels, adapters=False)
    g = torch.Generator(device=cuda_device).manual_seed(9)
    adv = torch.randn(4, device=cuda_device, generator=g)
    obj = Policy(adv, old, ref, kl_coef=0.2, reduction="sequence")
    loss, grads = _step_grads(tr, ids, labels, obj)
    logits, leaves = _whole(tr, ids)
    lp = _logps(logits, t)
    keep = (t != IGNORE).double()
    d = ref.double() - lp
    per = -torch.exp(lp - old.double()) * adv.double()[:, None] + 0.2 * (torch.exp(d) - 1 - d)
    want = ((per * keep).sum(1) / keep.sum(1)).mean()
    want.backward()
    tol = (adv.abs().max().item() + 0.2) * 8 * _bound(torch.tensor(12.0)).item() + 1e-7
    assert abs(loss.item() - want.item()) <= tol
    # the model has not moved since, but another kernel added its sums up: both are within the
    # bound of the truth
    assert ((obj.logps - old).abs() <= 2 * _bound(old)).all()
    _compare(grads, leaves)
    # two accumulated micro-steps of half the gradient each
    tr2 = _trainer(cuda_device, grad_accum=2)
    tr2.opt.zero_grad(set_to_none=True)
    tr2.train_step(ids, labels, objective=obj)
    half = [{n: (a.grad.clone(), b.grad.clone()) for n, (a, b) in layer.items()}
            for layer in tr2.lora]
    for l1, l2 in zip(grads, half):
        for n in l1:
            for a, b in zip(l1[n], l2[n]):
                rel = (a.float() - 2 * b.float()).pow(2).mean().sqrt() / a.float().pow(2).mean().sqrt()
                assert rel <= 2e-2
    tr.close()
    tr2.close()


def test_distill_step(cuda_device):
    tr = _trainer(cuda_device)
    ids, labels = _batch(cuda_device)
    t = next_targets(labels)
    with torch.no_grad():
        teacher = _whole(tr, ids, adapters=False)[0].float()
    val, idx = torch.topk(teacher, 24, -1)
    loss, grads = _step_grads(tr, ids, labels, Distill(idx, val, temperature=2.0))
    logits, leaves = _whole(tr, ids)
    lt = torch.log_softmax(val.double() / 2, -1)
    lq = torch.log_softmax(logits.double() / 2, -1).gather(-1, idx)
    keep = (t != IGNORE).double()
    want = 4 * ((lt.exp() * (lt - lq)).sum(-1) * keep).sum() / keep.sum()
    want.backward()
    assert abs(loss.item() - want.item()) <= 4 * (100 + 2.1 * 9) * U + 2 * U * abs(want.item())
    _compare(grads, leaves)
    tr.close()


def test_one_after_another(cuda_device):
    """Reference scores, a preference step, a policy step, a distillation step and a plain
    step on one trainer, with the optimizer: finite, and the adapters move."""
    shape = MixtralShape(hidden=256, heads=4, kv_heads=2, intermediate=512, vocab=512, layers=2,
                         experts=4, top_k=2)
    tr = StreamedLoraTrainer(shape, cuda_device, batch=4, seq=32, seed=1, lr=1e-3)
    ids, labels = _batch(cuda_device, 4, 32)
    ref = tr.token_logprobs(ids, labels, adapters=False)
    assert torch.equal(ref, tr.token_logprobs(ids, labels))   # B starts at zero
    before = [p.detach().clone() for p in tr.params]
    teacher = torch.randn(4, 32, 8, device=cuda_device)
    for obj in (Preference(ref), Policy(torch.ones(4, device=cuda_device), ref, ref, kl_coef=0.1),
                Distill(torch.randint(0, 512, (4, 32, 8), device=cuda_device), teacher), None):
        loss = tr.train_step(ids, labels, objective=obj)
        assert torch.isfinite(loss)
    assert any(not torch.equal(a, b) for a, b in zip(before, tr.params))
    assert not torch.equal(ref, tr.token_logprobs(ids, labels))
    assert torch.equal(ref, tr.token_logprobs(ids, labels, adapters=False))
    tr.check_device_errors()
    tr.close()


def test_bad_label_stops_training(cuda_device):
    """A target outside the vocabulary is found by the device error watch, as any failure of
    a kernel is."""
    from lema_b200._native import LemaError
    tr = _trainer(cuda_device)
    ids, labels = _batch(cuda_device)
    labels[0, -1] = SMALL.vocab + 3
    lp = tr.token_logprobs(ids, labels)
    torch.cuda.synchronize()
    assert lp.isnan().sum() == 1
    with pytest.raises(LemaError, match="outside the vocabulary"):
        tr.train_step(ids)
    tr.train_step(ids)
    tr.close()


def test_scores_of_shorter_sequences(cuda_device):
    """Sequences shorter than the trainer's and other batches, through the fused blocks and (an
    adapter on o_proj) the others: the bits of a trainer built for that length, which runs the
    same kernels on the same bytes. Longer ones are refused and the trainer goes on."""
    for targets in (("q_proj", "v_proj"), ("q_proj", "o_proj")):
        tr = _trainer(cuda_device, targets=targets)
        ids, labels = _batch(cuda_device)
        want = tr.token_logprobs(ids, labels)
        for b, s in ((4, 31), (1, 48), (3, 1)):
            one = _trainer(cuda_device, batch=b, seq=s, targets=targets)
            got = tr.token_logprobs(ids[:b, :s], labels[:b, :s])
            assert got.shape == (b, s)
            assert torch.equal(got, one.token_logprobs(ids[:b, :s], labels[:b, :s]))
            one.close()
        for bad in (torch.cat([ids, ids], 1), torch.cat([ids, ids[:, :1]], 1), ids[:, :0], ids[0]):
            with pytest.raises(ValueError, match="ids"):
                tr.token_logprobs(bad)
        assert torch.equal(want, tr.token_logprobs(ids, labels))
        tr.close()


def test_reference_scores_and_full_fine_tuning(cuda_device):
    """The reference is scored before the first full fine-tuning step, of an accumulated
    one too, and refused behind it; scores with the adapters go on."""
    tr = _trainer(cuda_device, full_ft_layers=(1,), lr=1e-3, grad_accum=2)
    ids, labels = _batch(cuda_device)
    ref = tr.token_logprobs(ids, labels, adapters=False)
    tr.train_step(ids, labels, objective=Preference(ref))
    assert torch.equal(ref, tr.token_logprobs(ids, labels, adapters=False))
    before = tr.token_logprobs(ids, labels)
    tr.train_step(ids, labels, objective=Preference(ref))
    with pytest.raises(RuntimeError, match="full fine-tuning"):
        tr.token_logprobs(ids, labels, adapters=False)
    assert not torch.equal(before, tr.token_logprobs(ids, labels))
    tr.train_step(ids, labels, objective=Preference(ref))
    tr.check_device_errors()
    tr.close()
