"""Forward-mode tangents: the operators over rows of logits have no rule for them, so logits that carry one are
refused, in the functions and in the torch.library ops; a teacher's tensors are constants."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from dsv41_rocm import distillation_loss, logit_scores

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def inputs():
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(3, 500, generator=g)
    lq, ids = torch.log_softmax(logits, 1).topk(8, 1)
    return logits.to(DEV), ids.to(DEV), lq.to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_logits_with_a_tangent_are_refused(dtype, requires_grad):
    logits, ids, lq = inputs()
    logits = logits.to(dtype).requires_grad_(requires_grad)
    targets = ids[:, 0].contiguous()
    with fwad.dual_level():
        dual = fwad.make_dual(logits, torch.ones_like(logits))
        for call in (lambda: logit_scores(dual, targets, top_k=3), lambda: logit_scores(dual, check=False),
                     lambda: distillation_loss(dual, ids, lq), lambda: distillation_loss(dual, ids, lq, check=False),
                     lambda: torch.ops.dsv41_rocm.logit_scores(dual, targets, 3, 1.0),
                     lambda: torch.ops.dsv41_rocm.distillation_loss(dual, ids, lq, 1.0, "rest")):
            with pytest.raises(NotImplementedError, match="forward"):
                call()
        # a detached tensor has none
        assert torch.equal(logit_scores(dual.detach()).entropy, logit_scores(logits.detach()).entropy)
    if not requires_grad:
        with pytest.raises(NotImplementedError, match="forward"):
            torch.func.jvp(lambda x: distillation_loss(x, ids, lq), (logits,), (torch.ones_like(logits),))


def test_a_teacher_with_a_tangent_is_constant():
    logits, ids, lq = inputs()
    want = distillation_loss(logits, ids, lq, tail="rest")
    with fwad.dual_level():
        dual = fwad.make_dual(lq, torch.ones_like(lq))
        for leaf in (logits, logits.clone().requires_grad_()):
            loss = distillation_loss(leaf, ids, dual, tail="rest")
            assert torch.equal(loss.detach(), want) and fwad.unpack_dual(loss).tangent is None


def test_upstream_gradients_with_a_tangent_are_refused():
    logits, ids, lq = inputs()
    leaf = logits.requires_grad_()
    with fwad.dual_level():
        weight = fwad.make_dual(torch.ones(3, device=DEV), torch.ones(3, device=DEV))
        for out in (logit_scores(leaf, ids[:, 0]).log_probs, logit_scores(leaf).entropy, distillation_loss(leaf, ids, lq),
                    torch.ops.dsv41_rocm.distillation_loss(leaf, ids, lq, 1.0, "rest")[0],
                    torch.ops.dsv41_rocm.logit_scores(leaf, None, 2, 1.0)[4][:, 0]):
            with pytest.raises(NotImplementedError, match="gradients carry a forward-mode"):
                torch.autograd.grad(out, leaf, weight)
