"""distillation_loss where logits lie far apart: finite masks of any size beside normal logits, a rest of the
vocabulary that consists of such masks, and a rest many hundreds of nats below the list.

The plain implementation is in 64 bits and in logarithms throughout.  Tolerances as in
test_gpu_distill.py: a sum over exponentials is off by n 2^-24 relative, n = 32 + V / 512 + 16; the loss by that for
Q log S and once more for the rest's logarithm, and by the rounding of the result.  Of the gradient outside
the list, Q p_i takes two such sums and rest w_i (w: p outside the list by itself) one, each with
the exponent's three roundings, 2^-24 of its size; the result is rounded once to the logits' dtype."""

import math

import pytest
import torch

from dsv41_rocm import distillation_loss

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
H = 2.0 ** -24


def plain(x, ids, lq, T, tail):
    """fp64 on the CPU: (loss, d loss / dx, what its tolerance counts)."""
    # the call takes its temperature in fp32: 0.3 as 0.3 (1 + 4e-8), two thirds of the 2^-24 that a rounded -q / T may be off by
    T = torch.tensor(T, dtype=torch.float32).item()
    z, ids, lq = x.detach().cpu().double() / T, ids.cpu(), lq.cpu().double()
    named = torch.zeros_like(z, dtype=torch.bool).scatter_(1, ids, True)
    # (differences first: logits of -1e12 in 64 bits have steps of 1e-4, which a logarithm added to them would drown in)
    top = z.amax(1, keepdim=True)
    logp, p = torch.log_softmax(z - top, 1), torch.softmax(z - top, 1)
    outside = z.masked_fill(named, -math.inf)
    near = outside - outside.amax(1, keepdim=True)
    w = torch.softmax(near, 1)
    log_rest = (outside.amax(1, keepdim=True) - top) + torch.logsumexp(near, 1, keepdim=True) - torch.logsumexp(z - top, 1, keepdim=True)
    if tail == "renormalize":
        lq = lq - torch.logsumexp(lq, 1, keepdim=True)
    q = lq.exp()
    loss = (q * (lq - logp.gather(1, ids))).sum(1)
    total = q.sum(1, keepdim=True)
    rest = torch.zeros_like(total)
    if tail == "rest":
        rest = 1 - total
        loss = loss + (rest * (rest.log() - log_rest))[:, 0]
        total = total + rest
    far = near.clamp(-800, 0).abs()
    grad = (total * p - rest * w).scatter(1, ids, total * p.gather(1, ids) - q)
    weight = 2 * total * p + rest * w
    return loss, grad / T, weight * (1 + far) / T


def compare(logits, ids, lq, T, tail, g=None):
    print(f"case: distillation_loss {tuple(logits.shape)} {logits.dtype} T {T} {tail}", flush=True)
    rows, V = logits.shape
    g = torch.linspace(1, 2, rows) if g is None else g
    leaf = logits.detach().requires_grad_()
    loss = distillation_loss(leaf, ids, lq, temperature=T, tail=tail)
    (grad,) = torch.autograd.grad(loss, leaf, g.to(DEV))
    want, slope, weight = plain(logits.float(), ids, lq, T, tail)
    n = 32 + V / 512 + 16
    d = (loss.detach().cpu().double() - want).abs()
    tol = H * (2.1 * n + 4 + 2 * want.abs())
    assert bool((d <= tol).all()), (loss, want)
    slope, weight = slope * g.double()[:, None], weight * g.double()[:, None]
    bound = weight * H * (n + 20) + slope.abs() * torch.finfo(logits.dtype).eps / 2 * 1.01 + 1e-37
    d = (grad.cpu().double() - slope).abs()
    assert bool((d <= bound).all()), (d.max(), (d / bound).max())
    assert torch.equal(distillation_loss(logits, ids, lq, temperature=T, tail=tail), loss.detach())


def teacher(rows, V, k, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(rows)])
    lq = torch.log_softmax(torch.randn(rows, k, generator=g), 1) + math.log(0.9)
    return ids, lq.float()


FILLS = [-1e4, -1e7, -2e7, -1e9, -1e10, -1e12, -1e20, -1e30, "lowest"]


def value_of(fill, dtype):
    return torch.finfo(dtype).min if fill == "lowest" else fill


@pytest.mark.parametrize("tail", ["renormalize", "rest"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fill", FILLS)
@pytest.mark.parametrize("V", [9003, 40001])  # one slice a row, several
def test_finite_masks_beside_normal_logits(V, fill, dtype, tail):
    # nine tenths of the tokens are masked: whole runs of them at the row's begin and end and within, and others
    # here and there; in some rows the list's tokens, too, but for one
    rows, k = 4, 12
    g = torch.Generator().manual_seed(V)
    x = 3 * torch.randn(rows, V, generator=g)
    gone = torch.rand(rows, V, generator=g) < 0.6
    gone[:, :V // 2] = True
    gone[:, V - V // 4:] = True
    gone[1, :16] = False
    ids, lq = teacher(rows, V, k, V + 1)
    gone[:2].scatter_(1, ids[:2], False)
    gone[2:].scatter_(1, ids[2:, :1], False)
    # (masked tokens of the list are masked for the teacher, too)
    lq[2:] = torch.where(gone[2:].gather(1, ids[2:]), torch.tensor(-1e38), lq[2:])
    x = x.masked_fill(gone, value_of(fill, dtype)).to(dtype).to(DEV)
    for T in (0.3, 0.5, 1.0, 2.0):
        compare(x[:2], ids[:2].to(DEV), lq[:2].to(DEV), T, tail)
    # a teacher's -1e38 has no probability: the entry counts for nothing but its place outside the rest
    there = lq[2:] > -1e30
    entries = lq[2:].masked_fill(~there, -math.inf).to(DEV)
    for T in (0.3, 0.5, 1.0, 2.0):
        loss = distillation_loss(x[2:], ids[2:].to(DEV), entries, temperature=T, tail=tail)
        masked = x[2:].float().masked_fill(gone[2:].to(DEV), -math.inf)
        want = distillation_loss(masked, ids[2:].to(DEV), entries, temperature=T, tail=tail)
        # the masks' probabilities are zero in 64 bits, too, from -1e4 on
        assert float((loss - want).abs().max()) <= H * (4.2 * (48 + V / 512) + 8 + 4 * float(want.abs().max()))


@pytest.mark.parametrize("tail", ["renormalize", "rest"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fill", FILLS[:-1])
@pytest.mark.parametrize("V", [9003, 40001])
def test_a_rest_of_finite_masks(V, fill, dtype, tail):
    # the student leaves the rest nothing but such masks: a divergence as large as their distance
    rows, k = 3, 12
    ids, lq = teacher(rows, V, k, V + 2)
    x = torch.full((rows, V), value_of(fill, dtype))
    x.scatter_(1, ids, torch.randn(rows, k, generator=torch.Generator().manual_seed(3)))
    for T in (0.3, 0.5, 1.0, 2.0):
        compare(x.to(dtype).to(DEV), ids.to(DEV), lq.to(DEV), T, tail)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_rest_at_the_lowest_value_is_masked(dtype):
    # the lowest value of the logits' type is as good as -inf where all of the rest has it: no mass for the teacher's
    V, k = 9003, 12
    ids, lq = (t.to(DEV) for t in teacher(3, V, k, 5))
    x = torch.full((3, V), torch.finfo(dtype).min, device=DEV)
    x = x.scatter(1, ids, torch.randn(3, k, device=DEV)).to(dtype)
    with pytest.raises(ValueError, match="non-finite"):
        distillation_loss(x, ids, lq, tail="rest")
    leaf = x.requires_grad_()
    loss = distillation_loss(leaf, ids, lq, tail="rest", check=False)
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    assert bool((loss == math.inf).all()) and bool(grad.isfinite().all())
    compare(x.detach(), ids, lq, 1.0, "renormalize")


@pytest.mark.parametrize("tail", ["renormalize", "rest"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [3000, 40001])
def test_a_rest_whose_mass_64_bits_do_not_hold(V, dtype, tail):
    # 740, 800, 2000 and 20000 nats below the list at this temperature
    T, k = 0.05, 6
    ids, lq = teacher(4, V, k, V + 3)
    g = torch.Generator().manual_seed(4)
    x = 0.05 * torch.randn(4, V, generator=g)
    x.scatter_(1, ids, torch.tensor([[37.0], [40.0], [100.0], [1000.0]]) + 0.05 * torch.randn(4, k, generator=g))
    x = x.to(dtype)
    compare(x.to(DEV), ids.to(DEV), lq.to(DEV), T, tail)


def test_logits_beyond_what_a_product_with_the_scale_holds():
    # the largest logits, of both signs, and a scale that takes their product out of fp32
    V, k = 9003, 8
    ids, lq = teacher(4, V, k, 9)
    g = torch.Generator().manual_seed(6)
    x = torch.randn(4, V, generator=g)
    x[0] += 3e38 * (torch.rand(V, generator=g) < 0.5)
    x[1] = 2e7 + 2 * torch.randint(-4, 5, (V,), generator=g)
    x[2] = -2e7 + 2 * torch.randint(-4, 5, (V,), generator=g)
    x[3, V // 2:] -= 1.1629e7  # (powers of two around -2^24)
    for tail in ("renormalize", "rest"):
        for T in (1.0, 0.7):
            compare(x[1:].to(DEV), ids[1:].to(DEV), lq[1:].to(DEV), T, tail)
    # (a row whose list lies 3e38 below its rest, or beside it)
    for tail in ("renormalize", "rest"):
        for T in (1.0, 1e30):
            loss = distillation_loss(x[:1].to(DEV), ids[:1].to(DEV), lq[:1].to(DEV), temperature=T, tail=tail, check=False)
            assert not bool(loss.isnan().any())


@pytest.mark.parametrize("tail", ["renormalize", "rest"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("base", [100.0, -5e3, -3e5, 3e5, 2e6, -5e6])
@pytest.mark.parametrize("V", [9003, 40001])
def test_logits_that_rise_far_from_zero(V, base, dtype, tail):
    # every thread raises its reference again and again, where half a step of the reference is up to 1 / 2
    rows, k = 3, 12
    ids, lq = teacher(rows, V, k, V + 4)
    step = 2.0 ** -6 if dtype == torch.float32 else abs(base) * 2.0 ** -8
    x = torch.linspace(-8, 0, V).expand(rows, V) * max(1.0, 8 * step) + torch.randn(rows, V, generator=torch.Generator().manual_seed(8))
    x = (x + base).to(dtype)
    for T in (0.7, 1.0, 2.0):
        compare(x.to(DEV), ids.to(DEV), lq.to(DEV), T * max(1.0, step), tail)


@pytest.mark.parametrize("tail", ["renormalize", "rest"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,k", [(40, 12), (9003, 12), (9003, 600), (40001, 12), (40001, 700)])
def test_rows_beyond_the_reference(V, k, dtype, tail):
    # rows that lie beyond 2^24 powers of two, whose list is above, below and among the rest, and ties with it
    ids, lq = teacher(6, V, k, V + 5)
    g = torch.Generator().manual_seed(9)
    unit = 2.0 if dtype == torch.float32 else 2.0 ** 17  # steps of the type there
    x = torch.randint(-6, 1, (6, V), generator=g).float() * unit
    x[1].scatter_(0, ids[1], unit * torch.randint(1, 4, (k,), generator=g).float())
    x[2].scatter_(0, ids[2], -unit * torch.randint(7, 9, (k,), generator=g).float())
    x[3].scatter_(0, ids[3], 0.0)
    x[4, V // 3:] -= 2.0 ** 26  # parts of the row, and with it slices of it, far from the others
    x[5, :V // 2] += 2.0 ** 26
    for base in (2.0 ** 25, -(2.0 ** 25), -(2.0 ** 25) - 2.0 ** 30):
        for T in (1.0, 2.0 * unit):
            compare((x + base).to(dtype).to(DEV), ids.to(DEV), lq.to(DEV), T, tail)


@pytest.mark.parametrize("tail", ["renormalize", "rest"])
@pytest.mark.parametrize("V", [9003, 40001])
@pytest.mark.parametrize("base", [-1e9, 3e7])
def test_no_distribution_beyond_the_reference(V, base, tail):
    # a NaN or +inf is found in a row whose rest lies there, and a row of masked tokens beside it
    k = 12
    ids, lq = teacher(5, V, k, V + 6)
    x = torch.full((5, V), base)
    x.scatter_(1, ids, torch.randn(5, k, generator=torch.Generator().manual_seed(3)))
    spare = (~torch.zeros(5, V, dtype=torch.bool).scatter_(1, ids, True)).nonzero()
    for row, value in ((1, math.nan), (2, math.inf)):
        at = spare[spare[:, 0] == row][:, 1]
        x[row, at[len(at) // 2]] = value
    x[3] = -math.inf
    ids, lq = ids.to(DEV), lq.to(DEV)
    with pytest.raises(ValueError, match="non-finite"):
        distillation_loss(x.to(DEV), ids, lq, tail=tail)
    leaf = x.to(DEV).requires_grad_()
    loss = distillation_loss(leaf, ids, lq, tail=tail, check=False)
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    assert loss.isfinite().tolist() == [True, False, False, False, True]
    assert bool(loss[1:4].isnan().all()) and bool(grad[1:4].isnan().any(1).all()) and bool(grad[[0, 4]].isfinite().all())
    keep = [0, 4]
    compare(x[keep].to(DEV), ids[keep], lq[keep], 1.0, tail)
