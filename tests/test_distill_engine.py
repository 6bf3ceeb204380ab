"""Distillation through the LM head and the training engine."""

import math

import pytest
import torch

import vocab_oracle as oracle
from libra_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U16 = 2.0 ** -8


def _head(device, R, H, V, seed=0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(R, H, generator=g).bfloat16().to(device)
    w = (torch.randn(V, H, generator=g) * 0.15).bfloat16().to(device)
    t = (h.float() @ w.float().t() + torch.randn(R, V, generator=g).to(device)).double()
    top = torch.log_softmax(t, 1).topk(12, 1)
    return h, w, top.indices, top.values.float()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("with_targets", [False, True])
@pytest.mark.parametrize("main_grad", [False, True])
@pytest.mark.parametrize("R,H,V", [(1, 64, 256), (37, 128, 1000), (300, 64, 2048)])
def test_lm_head_distill_against_the_oracle(device, with_targets, main_grad, R, H, V, monkeypatch):
    monkeypatch.setattr(ops, "LOGPROB_CHUNK_ROWS", 128)
    h, w, ids, lps = _head(device, R, H, V)
    if R > 2:
        ids[2] = -1
    gen = torch.Generator().manual_seed(5)
    g = torch.randn(R, generator=gen).to(device)
    g_lp = torch.randn(R, generator=gen).to(device) if with_targets else None
    targets = torch.randint(0, V, (R,), generator=gen).to(device) if with_targets else None
    hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    start = torch.randn(V, H, generator=gen).to(device)
    if main_grad and device == "cuda":
        ww.main_grad = start.clone()
    out = ops.lm_head_distill(hh, ww, ids, lps, divergence="js", beta=0.3, temperature=0.9, targets=targets)
    loss, logp = out if with_targets else (out, None)
    total = (loss * g).sum() + (0 if logp is None else (logp * g_lp).sum())
    total.backward()
    # the operator's own logits, so that their rounding is not in question
    logits = ops.gemm(h, w) if device == "cuda" else h.float() @ w.float().t()
    wl, wp, d = oracle.distill(logits, ids.cpu(), lps.cpu(), "js", 0.3, "bucket", 0.9, targets, g, g_lp)
    assert float((loss.detach().double().cpu() - wl).abs().max()) < 1e-5
    if with_targets:
        assert float((logp.detach().double().cpu() - wp).abs().max()) < 1e-5
    W, X = w.double().cpu(), h.double().cpu()
    # each logit's gradient is off by at most half a step of bf16 and the fp32 limits of distill_loss (far below); the
    # products accumulate in fp32, and dh is rounded to bf16 once
    dh, dw = d @ W, d.t() @ X
    lim_h = (1.1 * U16 * d.abs() + 1e-6) @ W.abs() + 1.1 * U16 * dh.abs()
    assert bool(((hh.grad.double().cpu() - dh).abs() <= lim_h).all())
    got = ww.grad
    lim_w = (2.2 * U16 * d.abs() + 1e-6).t() @ X.abs()  # one more rounding: of the rows scaled by g
    if main_grad and device == "cuda":
        assert got is None
        got = ww.main_grad - start
        lim_w = lim_w + 4 * 2.0 ** -24 * start.abs().double().cpu()
    else:
        lim_w = lim_w + 1.1 * U16 * dw.abs()
    assert bool(((got.double().cpu() - dw).abs() <= lim_w).all())


@pytest.mark.parametrize("device", DEVICES)
def test_lm_head_top_logprobs_is_the_teachers_table(device, monkeypatch):
    monkeypatch.setattr(ops, "LOGPROB_CHUNK_ROWS", 16)
    h, w, _, _ = _head(device, 37, 64, 512)
    ids, lps = ops.lm_head_top_logprobs(h, w, 9, 1.2)
    wi, wl, _ = oracle.top(ops.linear(h, w), 9, 1.2)
    assert torch.equal(ids.cpu(), wi) and float((lps.double().cpu() - wl).abs().max()) < 1e-5
    with pytest.raises(ValueError, match="k must"):
        ops.lm_head_top_logprobs(h, w, 0)


@pytest.mark.parametrize("device", DEVICES)
def test_lm_head_distill_refusals(device):
    h, w, ids, lps = _head(device, 4, 64, 256)
    with pytest.raises(ValueError, match="K"):
        ops.lm_head_distill(h, w, ids[:2], lps[:2])
    with pytest.raises(ValueError, match="lm_head_distill"):
        ops.lm_head_distill(h, w[:, :32], ids, lps)
    with pytest.raises(ValueError, match="divergence"):
        ops.lm_head_distill(h, w, ids, lps, divergence="none")
    if device == "cuda":
        hh = h.clone().requires_grad_(True)
        loss = ops.lm_head_distill(hh, w, ids, lps).sum()
        loss.backward(retain_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            loss.backward()
        with torch.no_grad():
            assert float((ops.lm_head_distill(h, w, ids, lps).sum() - loss.detach()).abs()) < 1e-4


def _engine(device, **kw):
    from libra_b200.engine.train_engine import B200TrainEngine

    eng = B200TrainEngine("tiny" if device == "cpu" else "tiny-gpu", device=device, learning_rate=1e-3,
                          micro_batch_size=2, max_tokens_per_micro_batch=64, **kw)
    eng.initialize()
    return eng


def _trajectories(vocab, n=4):
    g = torch.Generator().manual_seed(2)
    out = []
    for i in range(n):
        L = 12 + 5 * i
        mask = torch.ones(1, L, dtype=torch.long)
        mask[0, :4] = 0
        out.append({"input_ids": torch.randint(0, vocab, (1, L), generator=g), "loss_mask": mask,
                    "rewards": torch.tensor([float(i % 2)]), "advantages": torch.tensor([[1.0 if i % 2 else -1.0]])})
    return out


@pytest.mark.parametrize("device", DEVICES)
def test_teacher_tables_and_distill_update(device):
    teacher, student = _engine(device, seed=1), _engine(device, seed=7)
    trajs = _trajectories(student.cfg.vocab_size)
    teacher.score_teacher(trajs, 6)
    for t in trajs:
        L = t["input_ids"].numel()
        assert t["teacher_ids"].shape == t["teacher_logprobs"].shape == (1, L, 6)
        assert bool((t["teacher_ids"][0, :4] == -1).all()) and bool((t["teacher_ids"][0, 4:] >= 0).all())
        assert bool((t["teacher_logprobs"][0, 4:].diff(dim=1) <= 0).all())
    # the update's loss is the weighted divergence of the student's own logits from the tables
    w = student.loss_weights(trajs)
    want = 0.0
    from libra_b200.models.qwen3 import pack_sequences

    for t, wt in zip(trajs, w):
        with torch.no_grad():
            logits = student.model.logits(pack_sequences([t["input_ids"].reshape(-1)]).to(student.device))
        rows = torch.arange(3, t["input_ids"].numel() - 1)
        loss, _, _ = oracle.distill(logits[rows].float(), t["teacher_ids"][0, rows + 1],
                                    t["teacher_logprobs"][0, rows + 1], "forward", 0.5, "bucket", 1.0)
        want += wt * float(loss.sum())
    before = student.flat_param.clone()
    stats = student.distill_update(trajs)
    # bf16 activations of another batch composition on the GPU: a rounding of the logits (2^-8 of values near 1)
    assert abs(stats["distill_loss"] - want) < (1e-4 if device == "cpu" else 2e-2) * max(1.0, abs(want))
    assert stats["loss"] == stats["distill_loss"] and stats["grad_norm"] > 0 and stats["n_samples"] == 0
    assert not torch.equal(before, student.flat_param)
    with pytest.raises(ValueError, match="teacher_ids"):
        student.distill_update(_trajectories(student.cfg.vocab_size))


@pytest.mark.parametrize("device", DEVICES)
def test_grpo_update_with_the_distillation_term(device):
    teacher = _engine(device, seed=1)
    plain, zero, both = _engine(device, seed=7), _engine(device, seed=7, distill_coef=0.0), \
        _engine(device, seed=7, distill_coef=0.5, distill_divergence="reverse")
    trajs = _trajectories(plain.cfg.vocab_size)
    plain.recompute_logprobs(trajs)
    a = plain.grpo_update(trajs)
    ga = plain.flat_grad.clone()
    teacher.score_teacher(trajs[:3], 5)  # the last trajectory stays without a teacher
    b = zero.grpo_update(trajs)
    assert b["loss"] == a["loss"] and "distill_loss" not in b
    # the same work; on the GPU the backward's atomics sum in another order, which may turn a rounding of an
    # intermediate bf16 gradient (half a step at most)
    assert float((ga - zero.flat_grad).norm() / ga.norm()) <= (0.0 if device == "cpu" else U16)
    c = both.grpo_update(trajs)
    assert c["distill_loss"] > 0 and abs(c["loss"] - (a["loss"] + 0.5 * c["distill_loss"])) < 2e-3
    # gradients add up: GRPO's and half the distillation's, which an engine of the same weights computes alone
    alone = _engine(device, seed=7, distill_divergence="reverse")
    packed = alone.pack(trajs, False, alone.loss_weights(trajs))
    alone.flat_grad.zero_()
    acc, kd = torch.zeros(3, device=alone.device), torch.zeros(1, device=alone.device)
    alone._loss_backward(alone.to_device(packed), acc, kd)
    assert abs(float(kd) - c["distill_loss"]) < 1e-2 * max(1.0, c["distill_loss"])
    # three gradients of bf16 parameters and activations, each rounded to bf16 (half a step) on its way
    want = ga + 0.5 * alone.flat_grad
    assert float((both.flat_grad - want).norm() / want.norm()) < 4 * U16


def test_hybrid_payload_carries_the_distillation_term():
    teacher = _engine("cpu", seed=1)
    kw = dict(seed=7, distill_coef=0.5)
    core, hybrid = _engine("cpu", **kw), _engine("cpu", **kw)
    trajs = _trajectories(core.cfg.vocab_size)
    core.recompute_logprobs(trajs)
    teacher.score_teacher(trajs, 5)
    core.grpo_update(trajs)
    hybrid.compute_gradient_payload(trajs, replica_id="h", target_core_id="c", step=0, membership_epoch=0)
    assert torch.equal(core.flat_grad, hybrid.flat_grad)


def test_engine_refuses_distillation_across_ranks():
    from libra_b200.engine.train_engine import B200TrainEngine

    for kw in (dict(tp_size=2), dict(pp_size=2)):
        with pytest.raises(ValueError, match="distill_coef"):
            B200TrainEngine("tiny", device="cpu", distill_coef=0.1, **kw)
    with pytest.raises(ValueError, match="negative"):
        B200TrainEngine("tiny", device="cpu", distill_coef=-0.1)
    with pytest.raises(ValueError, match="distill_divergence"):
        B200TrainEngine("tiny", device="cpu", distill_divergence="kl")
