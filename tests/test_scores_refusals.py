"""Refusals of the operators over rows of logits that need no GPU: forward-mode tangents, and teacher lists of
other than two dimensions."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from dsv41_rocm import distill, distillation_loss, logit_scores, scores


def test_logits_with_a_tangent_are_refused():
    x = torch.zeros(2, 10)
    ids, lq = torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1)
    with fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            logit_scores(dual)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            distillation_loss(dual, ids, lq)
        # (a detached one has none: the next check refuses it)
        with pytest.raises(ValueError, match="on the GPU"):
            logit_scores(dual.detach())


def test_upstream_gradients_with_a_tangent_are_refused():
    x, ids, lq, g = torch.zeros(2, 10), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1), torch.ones(2)
    stats = torch.zeros(2, 7, dtype=torch.float64)
    with fwad.dual_level():
        dual = fwad.make_dual(g, torch.ones_like(g))
        for own in ((dual, None, None), (None, dual, None), (g, g, dual[:, None])):
            with pytest.raises(NotImplementedError, match="gradients carry a forward-mode"):
                scores.scores_backward(x, ids[:, 0], ids, 1.0, stats[:, :4], *own)
        with pytest.raises(NotImplementedError, match="gradients carry a forward-mode"):
            distill.distillation_backward(x, ids, lq, 1.0, stats, dual)


def test_the_teachers_log_probs_lose_both_kinds_of_derivatives(monkeypatch):
    monkeypatch.setattr(distill, "rows_of_logits", lambda logits, temperature: logits)
    x, ids, lq = torch.zeros(2, 10), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1)
    with fwad.dual_level():
        for t in (fwad.make_dual(lq, torch.ones_like(lq)), lq.clone().requires_grad_()):
            got = distill.prepare(x, ids, t, 1.0, "rest")[2]
            assert not got.requires_grad and fwad.unpack_dual(got).tangent is None


def test_lists_of_other_dimensions_are_refused_by_name(monkeypatch):
    monkeypatch.setattr(distill, "rows_of_logits", lambda logits, temperature: logits)
    x, ids, lq = torch.zeros(2, 10), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1)
    for i, q in ((torch.tensor(3), lq), (ids, torch.tensor(0.5)), (torch.tensor(3), torch.tensor(0.5)), (ids[:, 0], lq[:, 0]),
                 (ids[None], lq[None])):
        with pytest.raises(ValueError, match="must have shape \\[rows, entries\\]"):
            distill.prepare(x, i, q, 1.0, "rest")
    # the sizes are checked behind the shapes
    with pytest.raises(NotImplementedError, match="2\\^31"):
        distill.prepare(x[:1], ids[:1].expand(1, 2 ** 31), lq[:1].expand(1, 2 ** 31), 1.0, "rest")
