"""distillation_loss against lists of values of any size: tail="renormalize" takes the softmax of a list, so a
teacher's logits do as well as its log-probs, masks of a finite value among them.

Tolerances as in test_gpu_distill.py; the list's own terms are formed in 64 bits."""

import math

import pytest
import torch

from dsv41_rocm import distillation_loss

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
H = 2.0 ** -24


@pytest.mark.parametrize("base", [0.0, -1e6, 1e6, -1e9, 1e15, -1e17, -1e20, -1e30, 1e38, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("rows,V,k", [(3, 900, 7), (2, 30000, 600), (700, 9000, 5)])
def test_lists_far_from_zero(rows, V, k, base):
    print(f"case: distillation_loss {rows} x {V} k {k} base {base}", flush=True)
    g = torch.Generator().manual_seed(k)
    x = torch.randn(rows, V, generator=g)
    ids = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(rows)])
    # whole steps of the base, of 1 where it is small: lists that differ by some entries, or by none
    lq = (base + torch.randn(rows, k, generator=g)).float()
    lq = lq.clamp_min(torch.finfo(torch.float32).min)
    leaf = x.to(DEV).requires_grad_()
    loss = distillation_loss(leaf, ids.to(DEV), lq.to(DEV))
    up = torch.linspace(1, 2, rows)
    (grad,) = torch.autograd.grad(loss, leaf, up.to(DEV))
    q, logq = torch.softmax(lq.double(), 1), torch.log_softmax(lq.double(), 1)
    logp = torch.log_softmax(x.double(), 1)
    want = torch.where(q > 0, q * (logq - logp.gather(1, ids)), 0.0).sum(1)
    slope = logp.exp().scatter_add(1, ids, -q) * up.double()[:, None]
    n = 32 + V / 512 + 16
    off = (loss.detach().cpu().double() - want).abs()
    assert bool((off <= H * (2.1 * n + 4 + 2 * want.abs())).all()), (off.max(), want[:3])
    # p is off by n and its exponent's roundings (at most 9 nats below the row's largest), the result by half a step
    bound = logp.exp() * up.double()[:, None] * H * (n + 16 + 4 * 9) + slope.abs() * H * 1.01 + 1e-38
    off = (grad.cpu().double() - slope).abs()
    assert bool((off <= bound).all()), (off.max(), (off / bound).max())
