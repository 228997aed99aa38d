"""torch.ops.dsv41_rocm.logit_scores and distillation_loss: the functions' values and gradients, and
shapes under a fake device."""

import pytest
import torch

from dsv41_rocm import distillation_loss, logit_scores

OPS = torch.ops.dsv41_rocm


def _inputs(device):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 3001, generator=g)
    lq, ids = torch.log_softmax(x + 0.5 * torch.randn(6, 3001, generator=g), 1).topk(9, 1)
    return x.to(device), torch.randint(0, 3001, (6,), generator=g).to(device), ids.to(device), lq.to(device)


@pytest.mark.gpu
def test_scores_op():
    x, t, _, _ = _inputs("cuda")
    g = torch.rand(6, device="cuda")
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    s = logit_scores(a, t, top_k=5, temperature=0.7)
    lp, rank, entropy, ids, top, status, _ = OPS.logit_scores(b, t, 5, 0.7)
    for u, v in ((s.log_probs, lp), (s.ranks, rank), (s.entropy, entropy), (s.top_ids, ids), (s.top_log_probs, top)):
        assert torch.equal(u, v)
    assert int(status.max()) == 0
    up = [g, 2 * g, g[:, None].expand(6, 5)]
    (ga,) = torch.autograd.grad([s.log_probs, s.entropy, s.top_log_probs], a, up)
    (gb,) = torch.autograd.grad([lp, entropy, top], b, up)
    assert torch.equal(ga, gb)
    lp, rank, entropy, ids, top, _, _ = OPS.logit_scores(x.half(), None, 0, 1.0)
    assert lp.shape == rank.shape == (0,) and ids.shape == (6, 0)
    c = x.half().requires_grad_()
    (gc,) = torch.autograd.grad(OPS.logit_scores(c, None, 0, 1.0)[2], c, g)
    assert gc.dtype == torch.float16 and float(gc.abs().max()) > 0
    with pytest.raises(RuntimeError, match="differentiated again"):
        b = x.clone().requires_grad_()
        (gb,) = torch.autograd.grad(OPS.logit_scores(b, t, 0, 1.0)[0].sum(), b, create_graph=True)
        gb.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("tail", ["renormalize", "rest"])
def test_distillation_op(tail):
    x, _, ids, lq = _inputs("cuda")
    g = torch.rand(6, device="cuda")
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    u = distillation_loss(a, ids, lq, temperature=0.7, tail=tail)
    v, status, _ = OPS.distillation_loss(b, ids, lq, 0.7, tail)
    assert torch.equal(u, v) and int(status.max()) == 0
    assert torch.equal(torch.autograd.grad(u, a, g)[0], torch.autograd.grad(v, b, g)[0])


def test_fake_shapes():
    with torch.device("meta"):
        x, t, ids, lq = torch.empty(6, 50), torch.empty(6, dtype=torch.int64), torch.empty(6, 3, dtype=torch.int64), torch.empty(6, 3)
        out = OPS.logit_scores(x, t, 4, 1.0)
        assert [tuple(o.shape) for o in out] == [(6,), (6,), (6,), (6, 4), (6, 4), (6,), (6, 4)]
        assert [o.dtype for o in out[:6]] == [torch.float32, torch.int64, torch.float32, torch.int64, torch.float32, torch.int32]
        assert OPS.logit_scores(x, None, 0, 1.0)[0].shape == (0,)
        loss, status, stats = OPS.distillation_loss(x, ids, lq, 1.0, "rest")
        assert loss.shape == status.shape == (6,) and stats.shape == (6, 7) and stats.dtype == torch.float64


def test_host_tensors_are_refused():
    with pytest.raises(NotImplementedError):
        OPS.logit_scores(torch.zeros(2, 5), None, 0, 1.0)
    with pytest.raises(NotImplementedError):
        OPS.distillation_loss(torch.zeros(2, 5), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1), 1.0, "rest")
