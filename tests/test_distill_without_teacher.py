"""A distillation weight without teacher tables has nothing to act on, and says so."""

import logging

import pytest

from test_distill_engine import _engine, _trajectories


def _warnings(caplog):
    return [r for r in caplog.records if r.levelno >= logging.WARNING and "teacher" in r.getMessage()]


@pytest.mark.parametrize("through", ["grpo_update", "compute_gradient_payload"])
def test_distill_coef_without_teacher_tables_warns_once(through, caplog):
    eng = _engine("cpu", seed=7, distill_coef=0.5)
    trajs = _trajectories(eng.cfg.vocab_size)
    eng.recompute_logprobs(trajs)

    def update():
        if through == "grpo_update":
            assert "distill_loss" not in eng.grpo_update(trajs)
        else:
            eng.compute_gradient_payload(trajs, replica_id="h", target_core_id="c", step=0, membership_epoch=0)

    with caplog.at_level(logging.WARNING):
        update()
        assert len(_warnings(caplog)) == 1
        update()
        assert len(_warnings(caplog)) == 1


def test_no_warning_with_tables_or_without_the_weight(caplog):
    eng = _engine("cpu", seed=7, distill_coef=0.5)
    plain = _engine("cpu", seed=7)
    trajs = _trajectories(eng.cfg.vocab_size)
    eng.recompute_logprobs(trajs)
    with caplog.at_level(logging.WARNING):
        plain.grpo_update(trajs)
        plain.score_teacher(trajs[:1], 4)
        assert eng.grpo_update(trajs)["distill_loss"] > 0
        assert not _warnings(caplog)


def test_no_warning_for_a_rank_without_trajectories(caplog):
    eng = _engine("cpu", seed=7, distill_coef=0.5)
    with caplog.at_level(logging.WARNING):
        assert eng.prepare_update([]) == []
    assert not _warnings(caplog)
