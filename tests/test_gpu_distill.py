"""distillation_loss and its gradient against a plain implementation in 64 bits, over dtypes, both
tails, ragged and empty lists, masks, cuts and refusals, and a teacher-to-student step.

Tolerances.  The list's terms are formed in 64 bits, so what is off is S: by the terms outside the list,
2^-24 relative times 32 + V / 512 + 16 (the exponents' roundings, an exponential's, a thread's additions), and
the loss by that much of Q, of q_rest for log p_rest, and the rounding of the result."""

import math

import pytest
import torch

from dsv41_rocm import distillation_loss, logit_scores

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
H = 2.0 ** -24


def plain(x, ids, lq, T, tail):
    """fp64 on the CPU: (loss, d loss / dx, p)."""
    x, ids, lq = x.detach().cpu().double(), ids.cpu(), lq.cpu().double()
    V = x.shape[1]
    there = ids >= 0
    logp = torch.log_softmax(x / T, 1)
    p = logp.exp()
    slot = torch.where(there, ids, V)
    lq = lq.masked_fill(~there, -math.inf)
    if tail == "renormalize":
        lq = lq - torch.where(there.any(1, keepdim=True), torch.logsumexp(lq, 1, keepdim=True), 0.0)
    q = lq.exp()
    lp = torch.cat([logp, torch.zeros(len(x), 1)], 1).gather(1, slot)
    loss = torch.where(q > 0, q * (lq - lp), torch.zeros_like(q)).sum(1)
    total = q.sum(1)
    factor = total.clone()
    named = torch.zeros(len(x), V + 1).double().scatter_(1, slot, 1.0)[:, :V]
    if tail == "rest":
        rest = 1 - total
        rest[rest < 2.0 ** -20] = 0.0
        p_rest = (p * (1 - named)).sum(1)
        loss = loss + torch.where(rest > 0, rest * (rest.log() - p_rest.log()), torch.zeros_like(rest))
        total = total + rest
        factor = torch.where(p_rest > 0, total - rest / p_rest, total)
    dense_q = torch.zeros(len(x), V + 1).double().scatter_(1, slot, q)[:, :V]
    grad = torch.where(named > 0, total[:, None] * p - dense_q, factor[:, None] * p) / T
    empty = ~there.any(1)
    loss[empty], grad[empty] = 0.0, 0.0
    return loss, grad, p, factor


def make(rows, V, k, dtype, seed, ragged=False, pad=0, shift=0, scale=3.0, T=1.0):
    g = torch.Generator().manual_seed(seed)
    width = V + pad
    buf = torch.full((rows * width + shift,), float("nan"))
    view = buf[shift:shift + rows * width].view(rows, width)[:, :V]
    view.copy_(scale * torch.randn(rows, V, generator=g))
    teacher = torch.log_softmax((view + torch.randn(rows, V, generator=g)).double() / T, 1)
    lq, ids = teacher.topk(k, 1)
    lq = lq.float()
    if ragged:
        keep = torch.rand(rows, k, generator=g) < 0.6
        keep[0] = False
        ids = ids.masked_fill(~keep, -1)
        lq = lq.masked_fill(~keep, math.nan)
    dev = buf.to(dtype).to(DEV)
    return dev[shift:shift + rows * width].view(rows, width)[:, :V], ids.to(DEV), lq.to(DEV)


def compare(logits, ids, lq, T, tail, g=None):
    print(f"case: distillation_loss {tuple(logits.shape)} {logits.dtype} k {ids.shape[1]} T {T} {tail}", flush=True)
    rows, V = logits.shape
    leaf = logits.detach().requires_grad_()
    loss = distillation_loss(leaf, ids, lq, temperature=T, tail=tail)
    g = torch.linspace(-1, 2, rows) if g is None else g
    (grad,) = torch.autograd.grad(loss, leaf, g.to(DEV))
    torch.cuda.synchronize()
    want, slope, p, factor = plain(logits.float(), ids, lq, T, tail)
    n = 32 + V / 512 + 16
    got = loss.detach().cpu().double()
    tol = H * (2.1 * n + 4 + 2 * want.abs())
    same = (got == want) | ((got - want).abs() <= tol)
    assert bool(same.all()), ((got - want).abs().max(), tol)
    slope = slope * g.double()[:, None]
    # p is off by n and its exponent's roundings, others' factor by 2 n more of q_rest / p_rest
    weight = (p * (1 + 2 * factor.abs()[:, None] + 2 * (factor - 1).abs()[:, None]) + slope.abs()) * g.double().abs()[:, None] / T
    weight = weight + (p + H) * 1.1 * g.double().abs()[:, None] / T
    exponent = torch.where(p > 0, p.log(), torch.zeros_like(p)).abs() + math.log(V)
    bound = weight * H * (n + 16 + 4 * exponent) + slope.abs() * torch.finfo(logits.dtype).eps / 2 * 1.01 + 1e-38
    d = (grad.cpu().double() - slope).abs()
    assert bool((d <= bound).all()), (d.max(), (d / bound).max())
    # without a gradient the loss is the same
    assert torch.equal(distillation_loss(logits, ids, lq, temperature=T, tail=tail), loss.detach())
    return loss.detach(), grad


@pytest.mark.parametrize("tail", ["renormalize", "rest"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,k,ragged,pad,shift", [
    (1, 2, 1, False, 0, 0), (3, 9, 4, True, 1, 1), (4, 33, 33, True, 0, 0), (5, 1000, 1, False, 0, 0),
    (3, 4099, 64, True, 5, 3), (2, 8200, 600, False, 0, 0), (1, 129280, 16, False, 0, 1), (3, 151851, 100, True, 85, 0),
    (1200, 2051, 12, True, 0, 0)])
def test_matches_plain(rows, V, k, ragged, pad, shift, dtype, tail):
    logits, ids, lq = make(rows, V, k, dtype, V + k, ragged, pad, shift, T=0.8)
    compare(logits, ids, lq, 0.8, tail)


@pytest.mark.parametrize("T", [0.05, 20.0])
@pytest.mark.parametrize("tail", ["renormalize", "rest"])
def test_temperatures(T, tail):
    logits, ids, lq = make(4, 3001, 20, torch.float32, 5, T=T)
    compare(logits, ids, lq, T, tail)


def test_vocabularies_above_one_slice():
    for rows, V in ((2, 163841), (1100, 170000)):
        g = torch.Generator(device=DEV).manual_seed(V)
        logits = torch.randn(rows, V, generator=g, device=DEV).to(torch.bfloat16)
        lq, ids = torch.log_softmax(logits.float() + 0.5 * torch.randn(rows, V, generator=g, device=DEV), 1).topk(20, 1)
        print(f"case: distillation_loss {rows} x {V}", flush=True)
        leaf = logits.requires_grad_()
        loss = distillation_loss(leaf, ids, lq, tail="rest")
        (grad,) = torch.autograd.grad(loss.sum(), leaf)
        few = [0, rows - 1]
        want, slope, _, _ = plain(logits[few].float(), ids[few], lq[few], 1.0, "rest")
        assert float((loss.detach()[few].cpu().double() - want).abs().max()) <= H * 2.1 * (48 + V / 512)
        assert float((grad[few].cpu().double() - slope).norm() / slope.norm()) <= 2.0 ** -8


def test_student_far_more_certain_than_its_rest():
    # p_rest of 1e-9: formed by subtraction from 1 it would be lost
    V, k = 5000, 8
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, V, generator=g)
    x[:, :k] += 33.0
    lq = torch.log_softmax(torch.randn(2, k, generator=g), 1) + math.log(0.999)
    ids = torch.arange(k).expand(2, k)
    loss, grad = compare(x.to(DEV), ids.to(DEV), lq.to(DEV), 1.0, "rest")
    assert float(loss.min()) > 0


@pytest.mark.parametrize("tail", ["renormalize", "rest"])
def test_rest_far_below_the_list(tail):
    # 200 and 600 nats below: p_rest is no fp32 number, but the loss and the gradient are
    V, k = 3000, 6
    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, V, generator=g)
    x[0, :k] += 200.0
    x[1, :k] += 600.0
    x[2, :k] += 95.0
    lq = torch.log_softmax(torch.randn(3, k, generator=g), 1) + math.log(0.9)
    ids = torch.arange(k).expand(3, k)
    loss, grad = compare(x.to(DEV), ids.to(DEV), lq.to(DEV), 1.0, tail, g=torch.tensor([1.0, 1.0, 2.0 ** 16]))
    if tail == "rest":
        assert abs(float(grad[0, k:].sum()) + 0.1) < 1e-5 and abs(float(grad[1, k:].sum()) + 0.1) < 1e-5
    else:
        # e^-95 is below 2^-126, and 2^16 times that is above it
        assert float(grad[2, k:].min()) > 0.0


def test_confident_teacher_has_no_rest():
    # log-probs whose mass rounds to 1 (or to just above it): the rest is none, the loss finite
    V, k = 300, 5
    x = torch.randn(3, V, generator=torch.Generator().manual_seed(1))
    x[2, k:] = -math.inf  # the student leaves the rest nothing either
    lq = torch.tensor([[0.0, -30, -40, -50, -60], [math.log(0.2)] * 5, [math.log(0.2)] * 5])
    ids = torch.arange(k).expand(3, k)
    compare(x.to(DEV), ids.to(DEV), lq.to(DEV), 1.0, "rest")


@pytest.mark.parametrize("tail", ["renormalize", "rest"])
def test_masks_and_lowest_values(tail):
    V, k = 6000, 10
    logits, ids, lq = make(4, V, k, torch.float32, 6)
    x, ids, lq = logits.clone(), ids.clone(), lq.clone()
    x[0] = torch.finfo(torch.float32).min
    x[1, 3000:] = -math.inf
    ids[1], lq[1] = torch.arange(k, device=DEV), math.log(0.05)
    x[2, ids[2, 3]], lq[2, 3] = -math.inf, -math.inf  # masked by both: nothing
    lq[3, 4:] = -math.inf
    compare(x, ids, lq, 1.0, tail)


def test_empty_lists_read_nothing():
    V = 9000
    logits, ids, lq = make(6, V, 7, torch.float32, 8)
    x, ids = logits.clone(), ids.clone()
    x[1], x[4] = math.nan, math.inf
    ids[1], ids[4] = -1, -5
    leaf = x.requires_grad_()
    for tail in ("renormalize", "rest"):
        loss = distillation_loss(leaf, ids, lq, tail=tail)
        (grad,) = torch.autograd.grad(loss.sum(), leaf)
        assert float(loss[1]) == 0.0 == float(loss[4]) and bool(grad.isfinite().all())
        assert float(grad[1].abs().max()) == 0.0 == float(grad[4].abs().max()) and float(grad[0].abs().max()) > 0
    none = distillation_loss(leaf, ids[:, :0], lq[:, :0])
    (grad,) = torch.autograd.grad(none.sum(), leaf)
    assert float(none.abs().max()) == 0.0 == float(grad.abs().max())
    assert distillation_loss(x[:0].detach(), ids[:0], lq[:0]).shape == (0,)


def test_zero_gradients_write_zeros():
    logits, ids, lq = make(3, 5000, 4, torch.bfloat16, 2)
    leaf = logits.detach().requires_grad_()
    loss = distillation_loss(leaf, ids, lq)
    (grad,) = torch.autograd.grad(loss, leaf, torch.tensor([0.0, 1.0, 0.0], device=DEV))
    assert float(grad[0].abs().max()) == 0.0 == float(grad[2].abs().max()) and float(grad[1].abs().max()) > 0


@pytest.mark.parametrize("rows", [5, 1300])
def test_refused_rows(rows):
    V, k = 9000, 6
    logits, ids, lq = make(rows, V, k, torch.float32, 4)
    want = distillation_loss(logits, ids, lq, tail="rest")

    def case(match, tail="rest", row=2, **changes):
        x, i, l = logits.clone(), ids.clone(), lq.clone()
        for name, (col, value) in changes.items():
            {"x": x, "i": i, "l": l}[name][row, col] = value
        with pytest.raises(ValueError, match=match):
            distillation_loss(x, i, l, tail=tail)
        leaf = x.requires_grad_()
        loss = distillation_loss(leaf, i, l, tail=tail, check=False)
        assert not bool(loss[row].isfinite())
        if tail == "rest":
            others = [r for r in (0, 1, 3, rows - 1) if r != row]
            assert torch.equal(loss[others], want[others])
        (grad,) = torch.autograd.grad(loss.sum(), leaf)
        assert bool(grad[0].isfinite().all())
        return loss[row], grad[row]

    case("outside the model vocabulary", i=(3, V))
    case("outside the model vocabulary", i=(0, 1 << 40))
    loss, grad = case("non-finite", x=([i for i in range(V) if i not in ids[2].tolist()], torch.finfo(torch.float32).min))
    assert float(loss) == math.inf and bool(grad.isfinite().all())
    for tail in ("rest", "renormalize"):
        case("names a token twice", tail, i=(3, ids[2, 1].item()))
        case("do not form", tail, l=(2, math.nan))
        case("do not form", tail, l=(2, math.inf))
        case("non-finite", tail, x=(17, math.nan))
        case("non-finite", tail, x=(17, math.inf))
        loss, grad = case("non-finite", tail, x=(ids[2, 0].item(), -math.inf))
        assert float(loss) == math.inf and bool(grad.isfinite().all())
        case("non-finite", tail, x=(slice(None), -math.inf))
    case("do not form", l=(slice(None), 0.0))  # mass 6
    case("do not form", "renormalize", l=(slice(None), -math.inf))


def test_refused_arguments():
    logits, ids, lq = make(3, 100, 4, torch.float32, 1)
    with pytest.raises(ValueError, match="tail"):
        distillation_loss(logits, ids, lq, tail="drop")
    with pytest.raises(ValueError, match="shape"):
        distillation_loss(logits, ids[:2], lq)
    with pytest.raises(ValueError, match="shape"):
        distillation_loss(logits, ids[:, 0], lq)
    with pytest.raises(ValueError, match="per teacher ID"):
        distillation_loss(logits, ids, lq[:, :3])
    with pytest.raises(ValueError, match="integers"):
        distillation_loss(logits, ids.float(), lq)
    with pytest.raises(ValueError, match="on the GPU"):
        distillation_loss(logits.cpu(), ids, lq)
    for T in (0.0, math.nan, 1e31):
        with pytest.raises(ValueError, match="temperature"):
            distillation_loss(logits, ids, lq, temperature=T)
    with pytest.raises(NotImplementedError, match="2\\^21"):
        distillation_loss(torch.zeros(1, (1 << 21) + 1, device=DEV), ids[:1], lq[:1])


def test_sizes_past_32_bits_are_refused():
    one, ids, lq = torch.zeros(1, 1, device=DEV), torch.zeros(1, 1, dtype=torch.int64, device=DEV), torch.zeros(1, 1, device=DEV)
    n = 2 ** 32 + 1
    for x, i, q in ((one.expand(n, 1), ids.expand(n, 1), lq.expand(n, 1)), (one.expand(1, n), ids, lq),
                    (one, ids.expand(1, n), lq.expand(1, n))):
        with pytest.raises(NotImplementedError, match="2\\^31"):
            distillation_loss(x, i, q)


def test_layouts():
    logits, ids, lq = make(12, 800, 6, torch.float32, 9)
    want = distillation_loss(logits, ids, lq, tail="rest")
    wide_ids, wide_lq = ids.repeat_interleave(2, 1)[:, ::2], lq.repeat_interleave(2, 1)[:, ::2]
    assert torch.equal(distillation_loss(logits.t().contiguous().t(), wide_ids, wide_lq, tail="rest"), want)
    assert torch.equal(distillation_loss(logits, ids.int().cpu(), lq.cpu(), tail="rest"), want)
    one = logits[:1]
    many = distillation_loss(one.expand(12, 800), ids, lq, tail="rest")
    assert torch.equal(many, distillation_loss(one.repeat(12, 1), ids, lq, tail="rest"))
    leaf = one.clone().requires_grad_()
    (a,) = torch.autograd.grad(distillation_loss(leaf.expand(12, 800), ids, lq, tail="rest").sum(), leaf)
    (b,) = torch.autograd.grad(distillation_loss(leaf.repeat(12, 1), ids, lq, tail="rest").sum(), leaf)
    assert float((a - b).abs().max()) <= 12 * H
    half = logits.half().requires_grad_()
    (g,) = torch.autograd.grad(distillation_loss(half, ids, lq).sum(), half)
    assert g.dtype == torch.float16


def test_the_teacher_is_constant_and_no_second_derivatives():
    logits, ids, lq = make(3, 500, 4, torch.float32, 9)
    leaf, lq = logits.detach().clone().requires_grad_(), lq.requires_grad_()
    loss = distillation_loss(leaf, ids, lq)
    grad, none = torch.autograd.grad(loss.sum(), (leaf, lq), create_graph=True, allow_unused=True)
    assert none is None
    with pytest.raises(RuntimeError, match="differentiated again"):
        grad.sum().backward()


@pytest.mark.parametrize("tail", ["renormalize", "rest"])
def test_gradient_against_differences(tail):
    V, k, T = 60, 5, 0.7
    logits, ids, lq = make(2, V, k, torch.float32, 10, T=T)
    x = logits.cpu().double()
    v = torch.randn(2, V, generator=torch.Generator().manual_seed(1)).double()
    value = lambda x: plain(x, ids, lq, T, tail)[0].sum()
    slope = (value(x + 1e-6 * v) - value(x - 1e-6 * v)) / 2e-6
    assert abs(float((plain(x, ids, lq, T, tail)[1] * v).sum() - slope)) < 1e-7
    leaf = logits.detach().requires_grad_()
    (got,) = torch.autograd.grad(distillation_loss(leaf, ids, lq, temperature=T, tail=tail).sum(), leaf)
    assert abs(float((got.cpu().double() * v).sum() - slope)) < 1e-5


@pytest.mark.parametrize("tail", ["renormalize", "rest"])
def test_teacher_to_student(tail):
    # the operators in the order of use: a teacher's list, the student's loss through its head, a padded batch
    B, L, Hd, V, K, T = 2, 9, 64, 5003, 24, 1.5
    g = torch.Generator().manual_seed(20)
    hidden = torch.randn(B, L, Hd, generator=g).to(torch.bfloat16).to(DEV).requires_grad_()
    weight = (0.3 * torch.randn(V, Hd, generator=g)).to(torch.bfloat16).to(DEV).requires_grad_()
    teacher = (3 * torch.randn(B, L, V, generator=g)).to(DEV)
    mask = torch.ones(B, L, dtype=torch.bool, device=DEV)
    mask[1, 5:] = False
    s = logit_scores(teacher.view(-1, V), top_k=K, temperature=T)
    ids = s.top_ids.masked_fill(~mask.view(-1, 1), -1)
    logits = torch.nn.functional.linear(hidden, weight)
    loss = distillation_loss(logits.view(-1, V), ids, s.top_log_probs, temperature=T, tail=tail)
    want, slope, _, _ = plain(logits.detach().float().view(-1, V), ids, s.top_log_probs, T, tail)
    assert float((loss.detach().cpu().double() - want).abs().max()) <= H * (2.1 * 60 + 40)
    assert float(loss.view(B, L)[~mask].abs().max()) == 0.0
    scale = T * T / float(mask.sum())
    dh, dw = torch.autograd.grad(loss.sum() * scale, (hidden, weight))
    # bf16 logit gradients, then bf16 products: half a step each, and the products' fp32 sums
    dl = slope * scale
    want_h = dl @ weight.detach().cpu().double()
    want_w = dl.t() @ hidden.detach().cpu().double().view(-1, Hd)
    assert float((dh.cpu().double().view(-1, Hd) - want_h).norm() / want_h.norm()) <= 2.0 ** -7
    assert float((dw.cpu().double() - want_w).norm() / want_w.norm()) <= 2.0 ** -7


def test_a_student_equal_to_its_teacher_has_no_divergence():
    V, K = 7000, 50
    x = (3 * torch.randn(4, V, generator=torch.Generator().manual_seed(2))).to(DEV)
    s = logit_scores(x, top_k=K, temperature=0.7)
    leaf = x.requires_grad_()
    loss = distillation_loss(leaf, s.top_ids, s.top_log_probs, temperature=0.7, tail="rest")
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    assert float(loss.abs().max()) <= H * 2.1 * (48 + V / 512) and float(grad.abs().max()) <= H * 2 * (64 + V / 512) / 0.7


def test_streams_graphs_and_repeats():
    rows, V, k = 9, 30000, 20
    batches = [make(rows, V, k, torch.bfloat16, 40 + i, ragged=True) for i in range(3)]
    x, ids, lq = (t.clone() for t in batches[0])
    g = torch.rand(rows, device=DEV)

    def step(x, ids, lq):
        leaf = x.detach().requires_grad_()
        loss = distillation_loss(leaf, ids, lq, tail="rest", check=False)
        return loss.detach(), torch.autograd.grad(loss, leaf, g)[0]

    want = [step(*b) for b in batches]
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        again = step(*batches[1])
    torch.cuda.current_stream(DEV).wait_stream(side)
    for a, b in zip(again, want[1]):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, ids, lq)
        with pytest.raises(RuntimeError, match="check=False"):
            distillation_loss(x, ids, lq)
    for i in (0, 1, 2, 1):
        for a, b in zip((x, ids, lq), batches[i]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)
        distillation_loss(batches[0][0], batches[0][1], batches[0][2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tail", ["renormalize", "rest"])
def test_lists_longer_than_the_threads_over_slices(tail, dtype):
    # more entries than a workgroup has threads, some of them none, of rows that are cut
    logits, ids, lq = make(3, 30000, 1100, dtype, 81, ragged=True, pad=3, shift=1)
    compare(logits, ids, lq, 1.0, tail)
    # as many entries as tokens, and more with the empty ones
    logits, ids, lq = make(2, 700, 700, dtype, 82)
    ids = torch.cat([ids.new_full((2, 50), -7), ids], 1)
    lq = torch.cat([lq.new_full((2, 50), math.inf), lq], 1)
    compare(logits, ids, lq, 1.0, tail)


def test_offsets_above_32_bits():
    rows, V = 15000, 151936
    logits = torch.zeros(rows, V, dtype=torch.bfloat16, device=DEV)
    logits[-1, 100000], logits[-1, 7] = 9.0, 8.0
    ids = torch.tensor([[100000, 151935]], device=DEV).expand(rows, 2)
    lq = torch.log(torch.tensor([[0.5, 0.25]], device=DEV)).expand(rows, 2)
    print("case: distillation_loss 15000 x 151936 bf16", flush=True)
    leaf = logits.requires_grad_()
    loss = distillation_loss(leaf, ids, lq, tail="rest")
    g = torch.zeros(rows, device=DEV)
    g[-1] = 1.0
    (grad,) = torch.autograd.grad(loss, leaf, g)
    few = [0, rows - 1]
    want, slope, _, _ = plain(logits.detach()[few].float(), ids[few], lq[few], 1.0, "rest")
    assert float((loss.detach()[few].cpu().double() - want).abs().max()) <= H * 2.1 * (48 + V / 512) + 4 * H * 12
    assert float((grad[-1].cpu().double() - slope[1]).norm() / slope[1].norm()) <= 2.0 ** -8
    assert float(grad[-2].abs().max()) == 0.0 and float(grad[0].abs().max()) == 0.0


def test_two_streams_at_once():
    batches = [make(15, 30000 + 500 * i, 70, torch.float32, 90 + i, ragged=True) for i in range(4)]

    def step(x, ids, lq):
        leaf = x.detach().requires_grad_()
        loss = distillation_loss(leaf, ids, lq, tail="rest", check=False)
        return loss.detach(), torch.autograd.grad(loss.sum(), leaf)[0]

    want = [step(*b) for b in batches]
    sides = [torch.cuda.Stream(DEV) for _ in range(2)]
    for s in sides:
        s.wait_stream(torch.cuda.current_stream(DEV))
    got = []
    for turn in range(3):
        for i, b in enumerate(batches):
            with torch.cuda.stream(sides[i % 2]):
                got.append((i, step(*b)))
    torch.cuda.synchronize()
    for i, out in got:
        for a, b in zip(out, want[i]):
            assert torch.equal(a, b)


def test_what_was_saved_is_not_changed_unseen():
    logits, ids, lq = make(3, 2000, 9, torch.float32, 95)
    for change in (lambda ids, lq: ids.fill_(-1), lambda ids, lq: lq.zero_()):
        leaf, i, q = logits.clone().requires_grad_(), ids.clone(), lq.clone()
        loss = distillation_loss(leaf, i, q)
        change(i, q)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", [(2, 33003), (40, 40001), (3, 5), (1, 151851)])
def test_listed_tokens_at_the_ends_of_slices_and_chunks(rows, V, dtype):
    # wherever the gradient's slices of whole 32 elements end, their first and last tokens are listed in some
    # row, and so are the few behind the last 16 bytes
    logits, _, _ = make(rows, V, 1, dtype, V + 5, pad=1, shift=1)
    edges = [i for n in range(1, 41) for b in (-(-(-(-V // n)) // 32) * 32,) for j in range(1, n) for i in (j * b - 1, j * b)]
    edges = sorted({i for i in edges if 0 <= i < V} | set(range(max(0, V - 9), V)) | {0})
    k = min(len(edges), 500)
    g = torch.Generator().manual_seed(3)
    ids = torch.stack([torch.tensor(edges)[torch.randperm(len(edges), generator=g)[:k]] for _ in range(rows)])
    lq = torch.log_softmax(torch.randn(rows, k, generator=g), 1) - 0.1
    ids, lq = ids.to(DEV), lq.to(DEV)
    if k == V:
        # the teacher's rest, 1 - exp(-0.1), has no token left to go to: q (log q - log 0) is infinite
        assert bool(plain(logits.float(), ids, lq, 1.0, "rest")[0].isinf().all())
        with pytest.raises(ValueError, match="non-finite"):
            distillation_loss(logits, ids, lq, tail="rest")
        compare(logits, ids, lq, 1.0, "renormalize")
        return
    compare(logits, ids, lq, 1.0, "rest")
