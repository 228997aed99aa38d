"""logit_scores against a plain implementation in 64 bits: log-probs, ranks, entropy, top alternatives
and the gradient, over dtypes, strides, masks, ties and lengths that the kernels treat differently.

Tolerances.  A term 2^((x - r) c) of the sums is off by the rounding of a difference, of a product (2
halves of 2^-23 relative to the exponent) and of the exponential (2^-23): weighted by the terms, the
exponents' mean is below log2 V <= 21, so S is off by less than 2^-24 (2 ln2 21 + 2) < 32 * 2^-24, and by
one half of 2^-23 for each of the n <= V / 512 + 16 additions of a thread.  A log-prob adds its own rounding.
An entropy is log S minus a mean of exponents that are off by as much each."""

import math

import pytest
import torch

import dsv41_rocm
from dsv41_rocm import logit_scores

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
H = 2.0 ** -24


def plain(x, targets, k, T):
    """fp64 on the CPU: dict of the outputs, with stable orders."""
    x = x.detach().cpu().double()
    logp = torch.log_softmax(x / T, 1)
    p = logp.exp()
    out = {"p": p, "logp": logp, "entropy": torch.special.entr(p).sum(1)}
    order = torch.sort(x + 0.0, dim=1, descending=True, stable=True)[1]
    top = order[:, :k]
    lp = logp.gather(1, top)
    out["top_ids"], out["top_log_probs"] = top.masked_fill(lp == -math.inf, -1), lp
    if targets is not None:
        t = targets.cpu()
        out["log_probs"] = logp.gather(1, t[:, None])[:, 0]
        out["ranks"] = 1 + (order == t[:, None]).int().argmax(1)
    return out


def terms(V):
    return 32 + V / 512 + 16


def close(got, want, tol, what):
    got = got.detach().cpu().double()
    # a value past fp32's range, as of a token at the type's lowest value, is an infinity in fp32
    want = torch.where(want.float().isinf(), want.float().double(), want)
    same = (got == want) | ((got - want).abs() <= tol)
    assert bool(same.all()), (what, (got - want).abs()[~same].max(), got[~same][:4], want[~same][:4])


def check(logits, targets, k, T, **kw):
    print(f"case: logit_scores {tuple(logits.shape)} {logits.dtype} strides {logits.stride()} k {k} T {T}", flush=True)
    s = logit_scores(logits, targets, top_k=k, temperature=T, **kw)
    torch.cuda.synchronize()
    V = logits.shape[1]
    ref = plain(logits.float(), targets, k, T)
    n = terms(V)
    close(s.entropy, ref["entropy"], H * (n + 16) * (2 + math.log(V)), "entropy")
    if targets is not None:
        close(s.log_probs, ref["log_probs"], H * (n + ref["log_probs"].abs()), "log_probs")
        assert torch.equal(s.ranks.cpu(), ref["ranks"])
    else:
        assert s.log_probs is None and s.ranks is None
    assert s.top_ids.dtype == torch.int64 and s.top_ids.shape == (logits.shape[0], k)
    assert torch.equal(s.top_ids.cpu(), ref["top_ids"])
    close(s.top_log_probs, ref["top_log_probs"], H * (n + ref["top_log_probs"].abs()), "top_log_probs")
    return s, ref


def make(rows, V, dtype, seed, scale=3.0, pad=0, shift=0):
    """Logits whose rows begin at any element: a view of a padded, shifted buffer."""
    g = torch.Generator().manual_seed(seed)
    width = V + pad
    buf = torch.full((rows * width + shift,), float("nan"))
    view = buf[shift:shift + rows * width].view(rows, width)[:, :V]
    view.copy_(scale * torch.randn(rows, V, generator=g))
    t = torch.randint(0, V, (rows,), generator=g)
    dev = buf.to(dtype).to(DEV)
    return dev[shift:shift + rows * width].view(rows, width)[:, :V], t.to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,k,pad,shift", [
    (1, 1, 1, 0, 0), (3, 2, 2, 0, 0), (2, 7, 3, 1, 1), (5, 31, 31, 0, 3), (4, 33, 5, 0, 0), (3, 257, 20, 7, 1),
    (2, 1000, 64, 0, 5), (7, 4099, 0, 0, 0), (3, 4099, 100, 13, 2), (2, 8192, 1024, 0, 0), (1, 16385, 1, 0, 1),
    (2, 20001, 300, 3, 0), (1, 129280, 5, 0, 0), (3, 151851, 20, 85, 0), (2, 151936, 1000, 0, 0)])
def test_matches_plain(rows, V, k, pad, shift, dtype):
    logits, t = make(rows, V, dtype, 7 * V + k, pad=pad, shift=shift)
    check(logits, t, k, 0.7)


@pytest.mark.parametrize("T", [1.0, 0.05, 30.0, 1e-30, 1e30])
def test_temperatures(T):
    logits, t = make(4, 5000, torch.float32, 3)
    check(logits, t, 8, T)


def test_one_workgroup_a_row_and_no_targets():
    # enough rows that none is cut
    logits, t = make(1100, 3000, torch.bfloat16, 5)
    check(logits, None, 50, 1.0)
    check(logits, t, 0, 1.0)


def test_vocabularies_above_one_slice():
    # a slice holds at most 163840 elements, so these rows are cut however many there are
    for rows, V in ((2, 163841), (1100, 170000), (1, (1 << 21))):
        g = torch.Generator(device=DEV).manual_seed(V)
        logits = torch.randn(rows, V, generator=g, device=DEV).to(torch.bfloat16)
        t = torch.randint(0, V, (rows,), generator=g, device=DEV)
        print(f"case: logit_scores {rows} x {V}", flush=True)
        s = logit_scores(logits, t, top_k=33)
        few = torch.tensor(sorted({0, rows // 2, rows - 1}), device=DEV)
        ref = plain(logits[few].float(), t[few], 33, 1.0)
        assert torch.equal(s.top_ids[few].cpu(), ref["top_ids"]) and torch.equal(s.ranks[few].cpu(), ref["ranks"])
        n = terms(V)
        close(s.log_probs[few], ref["log_probs"], H * (n + ref["log_probs"].abs()), "log_probs")
        close(s.entropy[few], ref["entropy"], H * (n + 16) * (2 + math.log(V)), "entropy")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [1, 40, 700])
def test_ties_go_to_the_lowest_index(dtype, k):
    V = 30011
    g = torch.Generator().manual_seed(k)
    flat = torch.zeros(1, V)
    levels = torch.randint(0, 3, (1, V), generator=g).float()
    signs = torch.where(torch.rand(1, V, generator=g) < 0.5, 0.0, -0.0)
    ascending = (torch.arange(V) // 50).float()[None]
    descending = -ascending
    late = torch.where(torch.arange(V) >= V - 45, 1.0, 0.0)[None]
    x = torch.cat([flat, levels, signs, ascending, descending, late])
    t = torch.tensor([V - 1, 5, 17, 0, 29000, V - 2], device=DEV)
    check(x.to(dtype).to(DEV), t, k, 1.0)
    # the same without cuts
    check(x.to(dtype).to(DEV).repeat(200, 1), t.repeat(200), k, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks(dtype):
    V, k = 9001, 30
    g = torch.Generator().manual_seed(11)
    x = 2 * torch.randn(7, V, generator=g)
    x[0, torch.randperm(V, generator=g)[: V - 5]] = -math.inf  # fewer tokens than alternatives
    x[1, 1:] = -math.inf  # one token
    x[2, : V - 1] = -math.inf
    x[3, ::2] = -math.inf
    x[4] = torch.finfo(dtype).min  # nothing but the lowest value: uniform
    x[5, 3:] = torch.finfo(dtype).min
    x[6, :5000] = -math.inf
    x = x.to(dtype).to(DEV)
    t = torch.tensor([int(x[0].argmax()), 0, V - 1, 1, 77, 4000, 10], device=DEV)
    s, _ = check(x, t, k, 0.8)
    assert int((s.top_ids[0] >= 0).sum()) == 5 and float(s.log_probs[6]) == -math.inf
    assert float(s.log_probs[1]) == 0.0 and float(s.entropy[1]) == 0.0


@pytest.mark.parametrize("rows", [6, 1500])
def test_rows_without_a_distribution(rows):
    V = 20000
    logits, t = make(rows, V, torch.float32, 2)
    logits = logits.clone()
    logits[1, 17] = math.nan
    logits[2, 19999] = math.inf
    logits[3] = -math.inf
    good = logits.clone()
    good[1:4] = 0
    want = logit_scores(good, t, top_k=9)
    with pytest.raises(ValueError, match="without a distribution"):
        logit_scores(logits, t, top_k=9)
    s = logit_scores(logits, t, top_k=9, check=False)
    bad = torch.tensor([1, 2, 3], device=DEV)
    assert bool(s.log_probs[bad].isnan().all()) and bool(s.entropy[bad].isnan().all())
    assert bool((s.ranks[bad] == 0).all()) and bool((s.top_ids[bad] == -1).all()) and bool(s.top_log_probs[bad].isnan().all())
    rest = torch.tensor([r for r in range(rows) if r not in (1, 2, 3)], device=DEV)
    for a, b in zip((s.log_probs, s.ranks, s.entropy, s.top_ids, s.top_log_probs),
                    (want.log_probs, want.ranks, want.entropy, want.top_ids, want.top_log_probs)):
        assert torch.equal(a[rest], b[rest])


def test_refusals():
    logits, t = make(4, 100, torch.float32, 1)
    for bad in (t.clone().fill_(100), t.clone().fill_(-1)):
        with pytest.raises(ValueError, match="outside the model vocabulary"):
            logit_scores(logits, bad)
        s = logit_scores(logits, bad, check=False)
        assert bool(s.log_probs.isnan().all()) and bool((s.ranks == 0).all()) and bool(s.entropy.isfinite().all())
    with pytest.raises(ValueError, match="one target"):
        logit_scores(logits, t[:3])
    with pytest.raises(ValueError, match="integers"):
        logit_scores(logits, t.float())
    for k in (-1, 101, True, 2.0):
        with pytest.raises(ValueError, match="top_k"):
            logit_scores(logits, top_k=k)
    wide = torch.zeros(1, 2000, device=DEV)
    with pytest.raises(NotImplementedError, match="1024"):
        logit_scores(wide, top_k=1025)
    for T in (0.0, -1.0, math.nan, math.inf, 1e-31, 1e31):
        with pytest.raises(ValueError, match="temperature"):
            logit_scores(logits, temperature=T)
    with pytest.raises(ValueError, match="shape"):
        logit_scores(logits[0])
    with pytest.raises(NotImplementedError, match="2\\^21"):
        logit_scores(torch.zeros(1, (1 << 21) + 1, device=DEV))
    with pytest.raises(ValueError, match="on the GPU"):
        logit_scores(logits.cpu())


def test_sizes_past_32_bits_are_refused():
    # (views of one element: a wrapped size would pass for a small batch)
    one = torch.zeros(1, 1, device=DEV)
    for shape in ((2 ** 32 + 1, 1), (1, 2 ** 32 + 5), (2 ** 31, 1)):
        with pytest.raises(NotImplementedError, match="2\\^31"):
            logit_scores(one.expand(shape))
        with pytest.raises(NotImplementedError, match="2\\^31"):
            torch.ops.dsv41_rocm.logit_scores(one.expand(shape), None, 0, 1.0)


def test_empty_batch_and_other_layouts():
    s = logit_scores(torch.empty(0, 50, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV), top_k=3)
    assert s.log_probs.shape == (0,) and s.top_ids.shape == (0, 3)
    x, t = make(40, 500, torch.float32, 9)
    check(x.t().contiguous().t(), t, 7, 1.0)           # columns first
    check(x[:, ::2], t // 2, 7, 1.0)                     # every second column
    check(x[:1].expand(40, 500), t, 7, 1.0)            # one row, broadcast
    check(x.to(torch.float16), t, 7, 1.0)
    check(x.double(), t.int(), 7, 1.0)
    check(x.as_strided((3, 500), (100, 1)), t[:3], 7, 1.0)  # overlapping rows
    check(x[::3], t[::3], 7, 1.0)
    check(x, t.cpu(), 7, 1.0)


def test_offsets_above_32_bits():
    rows, V = 15000, 151936
    logits = torch.zeros(rows, V, dtype=torch.bfloat16, device=DEV)
    logits[-1, 100000], logits[-1, 7] = 9.0, 8.0
    t = torch.full((rows,), 7, device=DEV)
    print("case: logit_scores 15000 x 151936 bf16", flush=True)
    leaf = logits.requires_grad_()
    s = logit_scores(leaf, t, top_k=2)
    assert s.top_ids[-1].tolist() == [100000, 7] and int(s.ranks[-1]) == 2 and s.top_ids[0].tolist() == [0, 1]
    g = torch.zeros(rows, device=DEV)
    g[-1] = 1.0
    (grad,) = torch.autograd.grad(s.log_probs, leaf, g)
    p = torch.softmax(logits[-1].detach().double(), 0)
    want = (torch.nn.functional.one_hot(t[-1], V).double() - p).bfloat16()
    assert float((grad[-1].double() - want.double()).abs().max()) <= 2.0 ** -8 and float(grad[-2].abs().max()) == 0.0
    assert abs(float(grad[-1, 100000].double() / want[100000].double()) - 1) <= 2.0 ** -7


# ------------------------------------------------------------------------------------ gradients
def plain_grad(ref, targets, T, g_lp, g_h, g_top):
    p, logp, h = ref["p"], ref["logp"], ref["entropy"]
    c = torch.zeros_like(p)
    if targets is not None:
        c.scatter_add_(1, targets.cpu()[:, None], g_lp.cpu().double()[:, None])
    ids = ref["top_ids"]
    if ids.shape[1]:
        c.scatter_add_(1, ids.clamp_min(0), g_top.cpu().double().masked_fill(ids < 0, 0.0))
    g_h = g_h.cpu().double()[:, None]
    grad = (c - c.sum(1, keepdim=True) * p + g_h * (torch.special.entr(p) - p * h[:, None])) / T
    # the size of what was added up, for the tolerance
    safe = torch.where(p > 0, logp, torch.zeros_like(p)).abs()
    size = (p * (c.abs().sum(1, keepdim=True) + g_h.abs() * (safe + h[:, None] + math.log(p.shape[1]))) + c.abs()) / T
    return grad, size


def grad_tolerance(size, grad, dtype, ref, T, V):
    # p is off by 2^-24 (terms + 2 |exponent| ln 2 ...): the exponent's two roundings and c's own
    exponent = torch.where(ref["p"] > 0, ref["logp"], torch.zeros_like(ref["p"])).abs() + math.log(V)
    return size * H * (terms(V) + 16 + 4 * exponent) + grad.abs() * torch.finfo(dtype).eps / 2 * 1.01 + 1e-38


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,k,pad", [(1, 1, 1, 0), (3, 37, 5, 0), (2, 4099, 0, 0), (4, 8200, 64, 3), (1, 129280, 20, 0),
                                          (1100, 2001, 3, 0)])
def test_gradient(rows, V, k, pad, dtype):
    T = 0.6
    logits, t = make(rows, V, dtype, V + 1, pad=pad)
    t[0] = int(logits[0].float().argmax())  # a target that is among the alternatives
    g = torch.Generator().manual_seed(4)
    g_lp, g_h, g_top = torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn(rows, k, generator=g)
    leaf = logits.detach().requires_grad_()
    s, ref = check(leaf, t, k, T)
    outs, gs = [s.log_probs, s.entropy], [g_lp.to(DEV), g_h.to(DEV)]
    if k:
        outs, gs = outs + [s.top_log_probs], gs + [g_top.to(DEV)]
    (got,) = torch.autograd.grad(outs, leaf, gs)
    assert got.dtype == dtype and got.shape == logits.shape
    want, size = plain_grad(ref, t, T, g_lp, g_h, g_top)
    close(got, want, grad_tolerance(size, want, dtype, ref, T, V), "gradient")


def test_gradient_parts_and_zero_rows():
    rows, V, k = 5, 6000, 4
    logits, t = make(rows, V, torch.float32, 8)
    leaf = logits.detach().requires_grad_()
    g = torch.tensor([0.0, 1.0, 0.0, -2.0, 0.5], device=DEV)
    zero, none = torch.zeros(rows), torch.zeros(rows, k)
    for name in ("log_probs", "entropy", "top"):
        s, ref = check(leaf, t if name == "log_probs" else None, k, 1.3)
        out = s.top_log_probs if name == "top" else getattr(s, name)
        up = g[:, None].expand(rows, k) if name == "top" else g
        (got,) = torch.autograd.grad(out, leaf, up)
        want, size = plain_grad(ref, t if name == "log_probs" else None, 1.3, g.cpu() if name == "log_probs" else zero,
                                g.cpu() if name == "entropy" else zero, up.cpu() if name == "top" else none)
        close(got, want, grad_tolerance(size, want, torch.float32, ref, 1.3, V), name)
        assert float(got[0].abs().max()) == 0.0 and float(got[2].abs().max()) == 0.0
    # a row without a distribution has no gradient either, unless nothing flows into it
    x = logits.clone()
    x[0], x[1, 5] = -math.inf, math.nan
    leaf = x.requires_grad_()
    s = logit_scores(leaf, t, check=False)
    (got,) = torch.autograd.grad(s.log_probs, leaf, g)
    assert float(got[0].abs().max()) == 0.0 and bool(got[1].isnan().all()) and bool(got[2:].isfinite().all())


def test_gradient_of_masked_tokens_and_missing_alternatives():
    V, k = 5000, 8
    logits, t = make(3, V, torch.float32, 21)
    x = logits.clone()
    x[0, 3:] = -math.inf
    x[1, ::3] = -math.inf
    t = torch.tensor([1, 1, 4], device=DEV)
    leaf = x.requires_grad_()
    s, ref = check(leaf, t, k, 1.0)
    g = torch.Generator().manual_seed(1)
    g_lp, g_h, g_top = torch.randn(3, generator=g), torch.randn(3, generator=g), torch.randn(3, k, generator=g)
    (got,) = torch.autograd.grad([s.log_probs, s.entropy, s.top_log_probs], leaf, [g_lp.to(DEV), g_h.to(DEV), g_top.to(DEV)])
    want, size = plain_grad(ref, t, 1.0, g_lp, g_h, g_top)
    close(got, want, grad_tolerance(size, want, torch.float32, ref, 1.0, V), "gradient")
    assert float(got[0, 3:].abs().max()) == 0.0 and float(got[1, ::3].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_of_probabilities_below_the_smallest_normal_number(dtype):
    V = 2048
    x = torch.full((1, V), -92.0)
    x[0, 5] = 0.0
    leaf = x.to(dtype).to(DEV).requires_grad_()
    s = logit_scores(leaf, torch.tensor([5], device=DEV))
    (got,) = torch.autograd.grad(s.log_probs, leaf, torch.tensor([2.0 ** 20], device=DEV))
    want = -math.exp(float(leaf[0, 7].detach())) * 2.0 ** 20  # (the other tokens change S by less than 1e-36)
    assert 0 < -want < 2.0 ** -104 and abs(float(got[0, 7]) / want - 1) <= 2.0 ** -8


def test_gradient_against_differences():
    # the plain gradient itself, by central differences in 64 bits
    V, k, T = 50, 6, 0.9
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, V, generator=g).double()
    t = torch.tensor([3, 40])
    g_lp, g_h, g_top = torch.randn(2, generator=g), torch.randn(2, generator=g), torch.randn(2, k, generator=g)

    def value(x):
        r = plain(x, t, k, T)
        return (r["log_probs"] * g_lp).sum() + (r["entropy"] * g_h).sum() + (r["top_log_probs"] * g_top).sum()

    want, _ = plain_grad(plain(x, t, k, T), t, T, g_lp, g_h, g_top)
    v = torch.randn(2, V, generator=g).double()
    slope = (value(x + 1e-6 * v) - value(x - 1e-6 * v)) / 2e-6
    assert abs(float(slope - (want * v).sum())) < 1e-7
    leaf = x.float().to(DEV).requires_grad_()
    s = logit_scores(leaf, t.to(DEV), top_k=k, temperature=T)
    (got,) = torch.autograd.grad([s.log_probs, s.entropy, s.top_log_probs], leaf, [g_lp.to(DEV), g_h.to(DEV), g_top.to(DEV)])
    assert abs(float((got.cpu().double() * v).sum() - slope)) < 1e-5


def test_gradients_through_broadcast_rows_views_and_a_head():
    V, T = 700, 1.0
    g = torch.Generator().manual_seed(6)
    row = torch.randn(1, V, generator=g).to(DEV).requires_grad_()
    t = torch.randint(0, V, (6,), generator=g).to(DEV)
    (got,) = torch.autograd.grad(logit_scores(row.expand(6, V), t).log_probs.sum(), row)
    (want,) = torch.autograd.grad(torch.log_softmax(row.double(), 1).expand(6, V).gather(1, t[:, None]).sum(), row)
    assert float((got - want).abs().max()) <= 6 * H * 100
    # a transposed leaf, and second derivatives refused
    leaf = torch.randn(V, 4, generator=g).to(DEV).requires_grad_()
    s = logit_scores(leaf.t(), t[:4])
    (got,) = torch.autograd.grad(s.log_probs.sum(), leaf, create_graph=True)
    (want,) = torch.autograd.grad(torch.log_softmax(leaf.t().double(), 1).gather(1, t[:4, None]).sum(), leaf)
    assert float((got.detach() - want).abs().max()) <= H * 100
    with pytest.raises(RuntimeError, match="differentiated again"):
        got.sum().backward()


# ------------------------------------------------------------------------- streams and graphs
def test_another_stream():
    logits, t = make(64, 30000, torch.float32, 12)
    want = logit_scores(logits, t, top_k=12)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        s = logit_scores(logits, t, top_k=12)
        u = logit_scores(logits, t, top_k=12, check=False)
    torch.cuda.current_stream(DEV).wait_stream(side)
    for a in (s, u):
        assert torch.equal(a.top_ids, want.top_ids) and torch.equal(a.log_probs, want.log_probs)
        assert torch.equal(a.entropy, want.entropy) and torch.equal(a.ranks, want.ranks)


def test_captured_and_replayed():
    rows, V, k = 5, 40000, 15
    batches = [make(rows, V, torch.bfloat16, 30 + i) for i in range(3)]
    x, t = batches[0][0].clone(), batches[0][1].clone()
    g = torch.ones(rows, device=DEV)

    def step(x, t):
        leaf = x.detach().requires_grad_()
        s = logit_scores(leaf, t, top_k=k, check=False)
        (grad,) = torch.autograd.grad([s.log_probs, s.entropy], leaf, [g, g])
        return s.log_probs, s.ranks, s.entropy, s.top_ids, s.top_log_probs, grad

    want = [step(*b) for b in batches]
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        step(x, t)
    torch.cuda.current_stream(DEV).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, t)
        with pytest.raises(RuntimeError, match="check=False"):
            logit_scores(x, t)
    for i in (0, 1, 2, 1):
        x.copy_(batches[i][0])
        t.copy_(batches[i][1])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)
        dsv41_rocm.sample(batches[0][0], greedy=True)


def test_the_same_call_twice_is_bit_for_bit_the_same():
    logits, t = make(300, 50000, torch.float32, 14)
    a, b = (logit_scores(logits, t, top_k=200) for _ in range(2))
    for name in ("log_probs", "ranks", "entropy", "top_ids", "top_log_probs"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name


def test_agrees_with_the_sampler():
    # greedy's token is rank 1 and the first alternative; its log-prob is the sampler's
    logits, _ = make(32, 129280, torch.bfloat16, 15)
    r = dsv41_rocm.sample(logits, greedy=True, temperature=0.9)
    s = logit_scores(logits, r.ids, top_k=4, temperature=0.9)
    assert torch.equal(s.top_ids[:, 0], r.ids) and bool((s.ranks == 1).all())
    assert float((s.log_probs - r.logprobs).abs().max()) <= 1e-4
    assert torch.equal(s.log_probs, s.top_log_probs[:, 0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,k", [(2, 3000, 700), (1, 6000, 1024), (600, 5000, 600), (2, 9000, 513), (1, 40000, 1024)])
def test_many_alternatives_of_few_tokens(rows, V, k, dtype):
    # more alternatives than groups of 32 tokens, or not far from it; and values that crowd together
    logits, t = make(rows, V, dtype, V + k, scale=1.0)
    check(logits, t, k, 1.0)
    g = torch.Generator().manual_seed(k)
    near = (5 + 0.01 * torch.rand(rows, V, generator=g)).to(dtype).to(DEV)
    near[0, V // 2] = 900.0
    check(near, t, k, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [5, 64, 400])
def test_top_tokens_that_lie_together(dtype, k):
    # all of one thread's share, all of one slice, all of one group, every 512th chunk
    V = 65536
    g = torch.Generator().manual_seed(k)
    x = torch.randn(4, V, generator=g)
    x[0, torch.arange(0, V, 4096)] += 50
    x[1, 30000:31000] += 50
    x[2, 64:96] += 50
    vec = 4 if dtype == torch.float32 else 8
    x[3, (torch.arange(V) // vec) % 512 == 7] += 50
    t = torch.tensor([4096, 30500, 70, 7 * vec], device=DEV)
    check(x.to(dtype).to(DEV), t, k, 1.0)
    check(x.to(dtype).to(DEV).repeat(150, 1), t.repeat(150), k, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ranks_of_every_token(dtype):
    # ties within the target's chunk, before and behind it, zeros of both signs, masked targets, and
    # the neighbours of each value
    V = 1037
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-3, 4, (1, V), generator=g).float() * 0.5
    x[0, torch.randperm(V, generator=g)[:200]] = -0.0
    x[0, torch.randperm(V, generator=g)[:150]] = -math.inf
    x[0, 100:103] = torch.tensor([torch.finfo(dtype).tiny, -torch.finfo(dtype).tiny, torch.finfo(dtype).min])
    x[0, 103:105] = torch.tensor([1.5 + 2 * torch.finfo(dtype).eps, 1.5 - 2 * torch.finfo(dtype).eps])
    rows = x.to(dtype).expand(V, V).contiguous().to(DEV)
    check(rows, torch.arange(V, device=DEV), 0, 1.0)
    # and in slices: the same row, long
    long = torch.cat([x] * 30, 1).to(dtype).to(DEV)
    t = torch.randint(0, long.shape[1], (40,), generator=g).to(DEV)
    check(long.expand(40, -1), t, 3, 1.0)


@pytest.mark.parametrize("rows,V,k", [(2, 9000, 1024), (3, 40000, 700)])
def test_gradient_of_more_alternatives_than_threads(rows, V, k):
    T = 0.6
    logits, t = make(rows, V, torch.float32, V + k)
    order = logits.argsort(1, descending=True)
    t[0], t[1] = order[0, 600], order[1, 3]  # among the alternatives, in a thread's second and first
    g = torch.Generator().manual_seed(5)
    g_lp, g_h, g_top = torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn(rows, k, generator=g)
    leaf = logits.detach().requires_grad_()
    s, ref = check(leaf, t, k, T)
    (got,) = torch.autograd.grad([s.log_probs, s.entropy, s.top_log_probs], leaf, [g_lp.to(DEV), g_h.to(DEV), g_top.to(DEV)])
    want, size = plain_grad(ref, t, T, g_lp, g_h, g_top)
    # the sum of k gradients in fp64 of fp32 values adds nothing; a scaled sum's rounding is in `size`
    close(got, want, grad_tolerance(size, want, torch.float32, ref, T, V), "gradient")


def test_two_streams_and_two_threads_at_once():
    import threading

    batches = [make(20 + i, 30000 + 1000 * i, torch.bfloat16, 60 + i) for i in range(4)]

    def step(x, t, check):
        leaf = x.detach().requires_grad_()
        s = logit_scores(leaf, t, top_k=40, check=check)
        (grad,) = torch.autograd.grad(s.log_probs.sum() + s.top_log_probs.sum(), leaf)
        return s.log_probs.detach(), s.ranks, s.entropy.detach(), s.top_ids, s.top_log_probs.detach(), grad

    want = [step(*b, True) for b in batches]
    # unchecked calls in turn on two streams, with nothing between them
    sides = [torch.cuda.Stream(DEV) for _ in range(2)]
    for s in sides:
        s.wait_stream(torch.cuda.current_stream(DEV))
    got = []
    for turn in range(3):
        for i, b in enumerate(batches):
            with torch.cuda.stream(sides[i % 2]):
                got.append((i, step(*b, False)))
    torch.cuda.synchronize()
    # checked calls from two threads, each on its own stream
    failed = []

    def work(n):
        try:
            with torch.cuda.stream(sides[n]):
                for turn in range(3):
                    for i in (n, 2 + n):
                        out = step(*batches[i], True)
                        sides[n].synchronize()
                        got.append((i, out))
        except Exception as e:  # shown by the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    torch.cuda.synchronize()
    assert not failed and len(got) == 24
    for i, out in got:
        for a, b in zip(out, want[i]):
            assert torch.equal(a, b)


def test_two_graphs_replayed_at_once():
    batches = [make(6, 50000, torch.float32, 70 + i) for i in range(2)]
    want = [logit_scores(*b, top_k=300) for b in batches]
    graphs, outs = [], []
    for b in batches:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(logit_scores(*b, top_k=300, check=False))
        graphs.append(graph)
    sides = [torch.cuda.Stream(DEV) for _ in range(2)]
    for turn in range(4):
        for s, graph, out in zip(sides, graphs, outs):
            for t in (out.entropy, out.top_log_probs, out.log_probs):
                t.zero_()
            s.wait_stream(torch.cuda.current_stream(DEV))
        for s, graph in zip(sides, graphs):
            with torch.cuda.stream(s):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            for name in ("log_probs", "ranks", "entropy", "top_ids", "top_log_probs"):
                assert torch.equal(getattr(out, name), getattr(w, name)), name


def test_what_was_saved_is_not_changed_unseen():
    logits, t = make(3, 2000, torch.float32, 5)
    for change in (lambda leaf, t, s: t.zero_(), lambda leaf, t, s: s.top_ids.zero_()):
        leaf, t2 = logits.clone().requires_grad_(), t.clone()
        s = logit_scores(leaf, t2, top_k=4)
        change(leaf, t2, s)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            s.log_probs.sum().backward()
    # outputs that nothing saves may be edited, and targets of any integer type or shape given
    leaf = logits.clone().requires_grad_()
    s = logit_scores(leaf, t.to(torch.int16).view(3, 1), top_k=4)
    s.ranks.zero_()
    (got,) = torch.autograd.grad((s.log_probs * 2.0).sum(), leaf)
    leaf2 = logits.clone().requires_grad_()
    (want,) = torch.autograd.grad(logit_scores(leaf2, t).log_probs.sum(), leaf2)
    assert torch.equal(got, 2.0 * want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [33003, 8192, 16385])
def test_gradient_of_targets_at_the_ends_of_slices_and_chunks(V, dtype):
    # a row for each place where a slice of whole 32 elements may end, and for the last elements
    edges = [i for n in range(1, 9) for b in (-(-(-(-V // n)) // 32) * 32,) for j in range(1, n) for i in (j * b - 1, j * b)]
    edges = sorted({i for i in edges if 0 <= i < V} | set(range(V - 9, V)) | {0, 2047, 2048, 4095, 4096})
    rows, T = len(edges), 1.0
    logits, _ = make(rows, V, dtype, V + 9, pad=1, shift=1)
    t = torch.tensor(edges, device=DEV)
    g = torch.Generator().manual_seed(6)
    g_lp, g_h, g_top = torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.zeros(rows, 0)
    leaf = logits.detach().requires_grad_()
    s, ref = check(leaf, t, 0, T)
    (got,) = torch.autograd.grad([s.log_probs, s.entropy], leaf, [g_lp.to(DEV), g_h.to(DEV)])
    want, size = plain_grad(ref, t, T, g_lp, g_h, g_top)
    close(got, want, grad_tolerance(size, want, dtype, ref, T, V), "gradient")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", range(0, 70, 3))
def test_rows_that_begin_anywhere_in_a_line(shift, dtype):
    # rows of an odd stride, cut into slices whose ends lie inside 16 bytes; few values, so that most
    # comparisons are ties, masked tokens at the slices' ends, and masked targets; NaN around the rows
    rows, V, k = 6, 25003, 30
    g = torch.Generator().manual_seed(shift)
    x = torch.randint(0, 4, (rows, V), generator=g).float()
    x[torch.rand(rows, V, generator=g) < 0.3] = -math.inf
    for n in range(1, 5):
        b = -(-(-(-V // n)) // 32) * 32
        for j in range(1, n):
            x[0::2, j * b - 3:j * b + 5] = -math.inf
    t = torch.randint(0, V, (rows,), generator=g)
    t[0], t[1], t[2] = V - 1, 0, V // 2
    x[0, V - 1] = x[2, V // 2] = -math.inf
    x[1, 0] = 0.0
    buf = torch.full((rows * (V + 2) + shift,), math.nan, dtype=dtype)
    view = buf[shift:].view(rows, V + 2)
    view[:, :V] = x.to(dtype)
    logits = buf.to(DEV)[shift:].view(rows, V + 2)[:, :V]
    assert logits.data_ptr() % 128 == shift * buf.element_size() % 128
    leaf = logits.detach().requires_grad_()
    s, ref = check(leaf, t.to(DEV), k, 1.0)
    up = torch.zeros(rows)
    up[3:] = 1.0  # (the rows with masked targets aside)
    (got,) = torch.autograd.grad([s.log_probs, s.entropy], leaf, [up.to(DEV), up.to(DEV)])
    ref["top_ids"] = ref["top_ids"][:, :0]
    want, size = plain_grad(ref, t, 1.0, up, up, torch.zeros(rows, 0))
    want = torch.where((x == -math.inf) & (torch.arange(V) != t[:, None]), torch.zeros_like(want), want)
    got, want, size = got[3:], want[3:], size[3:]
    ref = {key: value[3:] for key, value in ref.items()}
    close(got, want, grad_tolerance(size, want, dtype, ref, 1.0, V), "gradient")
