"""process_logits against plain 64-bit arithmetic and against the sampler's own penalties: biases, penalties
with knobs for each row, token masks, in place and not, and the gradient."""

import math

import pytest
import torch

from dsv41_rocm import logit_scores, process_logits, sample

pytestmark = pytest.mark.gpu

DEV = "cuda"
INF = math.inf


def _mask_words(allowed):
    """int32 words of a bool [m, V]."""
    m, V = allowed.shape
    W = (V + 31) // 32
    bits = torch.zeros(m, W * 32, dtype=torch.int64)
    bits[:, :V] = allowed.cpu().long()
    words = (bits.reshape(m, W, 32) << torch.arange(32)).sum(2)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).int()


def _inputs(rows, V, dtype, hist=0, bias=0, masks=None, knobs="rows", seed=0, pad=0):
    """CPU tensors of a call."""
    g = torch.Generator().manual_seed(1000 * rows + V + seed)
    x = (3 * torch.randn(rows, V + pad, generator=g)).to(dtype)[:, :V]
    a = {}
    if hist:
        h = torch.randint(0, V, (rows, hist), generator=g)
        h = torch.where(torch.rand(rows, hist, generator=g) < 0.4, h % max(1, V // 50), h)  # repeated ones
        h[torch.rand(rows, hist, generator=g) < 0.1] = -1
        a["history"] = h
        a["history_lens"] = torch.randint(0, hist + 1, (rows,), generator=g).int()
        a["history_lens"][0] = hist
        a["history_prompt_lens"] = torch.randint(0, hist + 2, (rows,), generator=g).int()
        if knobs == "rows":
            a["repetition_penalty"] = torch.rand(rows, generator=g) + 0.6
            a["presence_penalty"] = torch.randn(rows, generator=g)
            a["frequency_penalty"] = torch.randn(rows, generator=g)
            a["repetition_penalty"][rows // 2] = 1.0
            a["presence_penalty"][rows // 2] = a["frequency_penalty"][rows // 2] = 0.0
        else:
            a.update(knobs)
    if bias:
        ids = torch.randint(-1, V, (rows, bias), generator=g)
        ids[:, bias // 2] = ids[:, 0]  # an id named twice
        a["bias_ids"] = ids
        a["bias"] = 4 * torch.randn(rows, bias, generator=g)
        a["bias"][0, 0] = -INF
    if masks:
        allowed = torch.rand(masks, V, generator=g) < 0.4
        allowed[:, V - 1] = True
        a["token_mask"] = _mask_words(allowed)
        a["mask_rows"] = torch.randint(-1, masks, (rows,), generator=g).int()
        a["fill"] = -8192.0 if seed % 2 else -INF
    return x, a


def _unpack(words, V):
    bits = (words.long()[:, :, None] >> torch.arange(32)) & 1
    return bits.reshape(words.shape[0], -1)[:, :V].bool()


def _plain(x, a, g=None):
    """(result, its bound, gradient, its bound) in 64 bits, element by element.

    Bound: with u = 2^-24, the kernel rounds x + b, the product or quotient by rp, freq c, and two
    differences; each rounding is at most u times its own value, and the factor (at most f = max(rp, 1 / rp)) carries
    what came before.  The values are at most A f, |freq c|, A f + |freq c| and A f + |freq c| + |pres| with
    A = |x + b|: in all u (A f + A f + |freq c| + (A f + |freq c|) + (A f + |freq c| + |pres|)), and a half more for
    the terms of second order; then half a step of the type."""
    rows, V = x.shape
    half = torch.finfo(x.dtype).eps / 2
    u = 2.0 ** -24
    y = x.double().clone()
    bound = torch.zeros_like(y)
    grad = None if g is None else g.double().clone()
    for r in range(rows):
        if "bias" in a:
            ids, b = a["bias_ids"][r], a["bias"][r].double()
            last = {int(i): float(v) for i, v in zip(ids, b) if 0 <= int(i) < V}
            for i, v in last.items():
                y[r, i] += v
                bound[r, i] = u * abs(float(y[r, i]))
        if "history" in a:
            n = min(max(int(a["history_lens"][r]), 0), a["history"].shape[1]) if "history_lens" in a else a["history"].shape[1]
            prompt = int(a["history_prompt_lens"][r]) if "history_prompt_lens" in a else 0
            knob = lambda k, d: float(a[k][r]) if isinstance(a.get(k), torch.Tensor) else torch.tensor(a.get(k, d), dtype=torch.float32).item()
            rp, pres, freq = knob("repetition_penalty", 1.0), knob("presence_penalty", 0.0), knob("frequency_penalty", 0.0)
            h = a["history"][r, :n]
            ok = (h >= 0) & (h < V)
            seen = torch.zeros(V, dtype=torch.bool)
            seen[h[ok]] = True
            count = torch.bincount(h[prompt:][ok[prompt:]], minlength=V).double()
            one = torch.ones(V, dtype=torch.float64)
            factor = torch.where(seen, torch.where(y[r] > 0, one / rp, one * rp), one)
            A = y[r].abs().nan_to_num(posinf=0) * max(rp, 1 / rp)
            fc = (freq * count).abs()
            bound[r] = torch.where(seen, 1.5 * u * (4 * A + 3 * fc + abs(pres)), bound[r])
            y[r] = y[r] * factor - freq * count - pres * (count > 0)
            if g is not None:
                grad[r] *= factor
        if "token_mask" in a:
            m = int(a["mask_rows"][r]) if "mask_rows" in a else (0 if a["token_mask"].shape[0] == 1 else r)
            if m >= 0:
                out = ~_unpack(a["token_mask"][m:m + 1], V)[0]
                fill = torch.tensor(a.get("fill", -INF)).to(x.dtype).double()
                y[r] = torch.where(out, fill, y[r])
                bound[r] = torch.where(out, 0.0, bound[r])
                if g is not None:
                    grad[r] = torch.where(out, 0.0, grad[r])
    if x.dtype == torch.bfloat16:
        bound = bound + half * (y.abs().nan_to_num(posinf=0) + bound)
    gbound = None if g is None else (1.5 * u + (half if x.dtype == torch.bfloat16 else 0)) * grad.abs() * 1.01
    return y, bound, grad, gbound


def _to(a, dev=DEV):
    return {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in a.items()}


def _close(got, want, bound):
    got = got.double().cpu()
    same = got == want
    assert bool((same | ((got - want).abs() <= bound)).all()), float(((got - want).abs() - bound)[~same].max())


SHAPES = [(1, 1), (3, 31), (2, 33), (2, 8191), (1, 8192), (3, 8193), (5, 20001), (40, 1000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("hist,bias,masks", [(0, 0, 0), (50, 0, 0), (0, 5, 0), (0, 0, 2), (700, 9, 3)])
def test_against_64_bits(rows, V, dtype, hist, bias, masks):
    for seed, pad in ((0, 0), (1, 3)):
        x, a = _inputs(rows, V, dtype, hist, bias, masks, seed=seed, pad=pad)
        want, bound, _, _ = _plain(x, a)
        d = torch.empty(rows, V + pad, dtype=dtype, device=DEV)[:, :V].copy_(x)
        before = d.clone()
        got = process_logits(d, **_to(a))
        _close(got, want, bound)
        assert torch.equal(d, before) and got.dtype == dtype
        # in place, and into rows further apart, bit for bit the same; nothing behind the rows is touched
        wide = torch.full((rows, V + 9), 7.0, dtype=dtype, device=DEV)
        assert process_logits(d, **_to(a), out=wide[:, 1:V + 1]).data_ptr() == wide[:, 1:].data_ptr()
        assert torch.equal(wide[:, 1:V + 1].nan_to_num(), got.nan_to_num())
        assert bool((wide[:, 0] == 7).all()) and bool((wide[:, V + 1:] == 7).all())
        wide = torch.full((rows, V + 9), 7.0, dtype=dtype, device=DEV)
        wide[:, 1:V + 1] = d
        own = wide[:, 1:V + 1]
        process_logits(own, **_to(a), out=own)
        assert torch.equal(own.nan_to_num(), got.nan_to_num())
        assert bool((wide[:, 0] == 7).all()) and bool((wide[:, V + 1:] == 7).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("hist,bias,masks", [(0, 0, 0), (50, 0, 0), (0, 5, 0), (0, 0, 2), (700, 9, 3)])
def test_gradient_against_the_formula(rows, V, dtype, hist, bias, masks):
    x, a = _inputs(rows, V, dtype, hist, bias, masks, pad=1)
    g = torch.randn(rows, V + 2, generator=torch.Generator().manual_seed(5)).to(dtype)[:, 1:V + 1]
    _, _, want, bound = _plain(x, a, g)
    leaf = x.to(DEV).requires_grad_()
    y = process_logits(leaf, **_to(a))
    with torch.no_grad():
        assert torch.equal(y.nan_to_num(), process_logits(leaf, **_to(a)).nan_to_num())
    gd = torch.empty(rows, V + 2, dtype=dtype, device=DEV)[:, 1:V + 1].copy_(g)
    (grad,) = torch.autograd.grad(y, leaf, gd)
    _close(grad, want, bound)
    # a gradient that is one number everywhere (stride 0) is that number's
    y = process_logits(leaf, **_to(a))
    (one,) = torch.autograd.grad(y, leaf, torch.ones((), dtype=dtype, device=DEV).expand(rows, V))
    _, _, want, bound = _plain(x, a, torch.ones(rows, V, dtype=dtype))
    _close(one, want, bound)


def test_gradient_against_differences():
    # piecewise linear in x: away from x + b = 0 a difference quotient is the slope up to the rounding of its
    # two values, each off by 8e-6 at most for |value| < 32 (bound of _plain), over a step of 1/4
    x, a = _inputs(4, 300, torch.float32, 80, 6, 2, seed=1)
    step = 0.125
    leaf = x.to(DEV).requires_grad_()
    (grad,) = torch.autograd.grad(process_logits(leaf, **_to(a)).sum(), leaf)
    with torch.no_grad():
        up, down = process_logits(leaf + step, **_to(a)), process_logits(leaf - step, **_to(a))
    quotient = (up - down).double().cpu() / (2 * step)
    b = torch.zeros_like(x)
    for r in range(4):
        for i, v in zip(a["bias_ids"][r].tolist(), a["bias"][r].tolist()):
            if i >= 0:
                b[r, i] = v
    steady = ((x + b).abs() > step) & torch.isfinite(b)
    value = torch.maximum(up.abs(), down.abs()).double().cpu()
    plain = value > 4000  # filled
    err = (grad.double().cpu() - quotient).abs()
    assert float(torch.where(steady & ~plain, err, 0.0).max()) < 2 * 8e-6 / (2 * step) + 1e-6
    assert float(torch.where(plain, grad.double().cpu().abs(), 0.0).max()) == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("greedy", [True, False])
def test_penalties_are_the_samplers(dtype, greedy):
    # top-k draws are exact in the processed logits, so the sampler draws the same from rows that were
    # processed before it; bf16 rows are widened first, as the sampler widens them
    knobs = dict(repetition_penalty=1.3, presence_penalty=0.4, frequency_penalty=-0.2)
    x, a = _inputs(64, 5000, dtype, 300, knobs=knobs)
    u = torch.rand(64, generator=torch.Generator().manual_seed(1)).to(DEV)
    a = _to(a)
    d = x.to(DEV)
    draw = dict(temperature=0.7, top_k=40, uniforms=u, greedy=greedy)
    want = sample(d, **a, **draw)
    got = sample(process_logits(d.float(), **a), **draw)
    assert torch.equal(got.ids, want.ids) and torch.equal(got.logprobs, want.logprobs) and torch.equal(got.kept, want.kept)
    # one knob of the batch, and the same knob row by row
    rows = {k: torch.full((64,), v, device=DEV) for k, v in knobs.items()}
    assert torch.equal(process_logits(d, **a), process_logits(d, **{**a, **rows}))


def test_decode_step_together():
    # mask, bias and penalties, then the draw: only allowed tokens come out, and the log-prob is the processed row's
    x, a = _inputs(96, 20001, torch.float32, 200, 12, 7, seed=1)
    a["bias"][0, 0] = -50.0
    u = torch.rand(96, generator=torch.Generator().manual_seed(2)).to(DEV)
    y = process_logits(x.to(DEV), **_to(a))
    s = sample(y, temperature=0.8, uniforms=u)
    allowed = _unpack(a["token_mask"], 20001)
    for r in range(96):
        m = int(a["mask_rows"][r])
        assert m < 0 or bool(allowed[m, int(s.ids[r])])
    z = (y.double() / 0.8).log_softmax(1).gather(1, s.ids[:, None])[:, 0]
    assert float((z - s.logprobs.double()).abs().max()) < 1e-4  # the sampler's stated accuracy


def test_learner_scores_under_the_processed_distribution():
    x, a = _inputs(12, 4001, torch.float32, 100, 6, 3)
    a["bias"][0, 0] = 2.0
    t = torch.full((12,), 4000)  # allowed by every mask
    leaf = x.to(DEV).requires_grad_()
    s = logit_scores(process_logits(leaf, **_to(a)), t.to(DEV), temperature=0.9)
    g = torch.randn(12, generator=torch.Generator().manual_seed(3))
    (grad,) = torch.autograd.grad(s.log_probs, leaf, g.to(DEV))
    y, _, _, _ = _plain(x, a)
    p = (y / 0.9).softmax(1)
    up = g.double()[:, None] * (torch.nn.functional.one_hot(t, 4001) - p) / 0.9
    _, _, want, _ = _plain(x, a, up)
    lp = (y / 0.9).log_softmax(1)[:, 4000]
    assert float((s.log_probs.double().cpu() - lp).abs().max()) < 1e-5
    # |g| / T times a probability off by 1e-6 or so, times a factor up to 1 / 0.6
    assert float((grad.double().cpu() - want).abs().max()) < 1e-5


def test_statuses_and_what_a_bad_row_holds():
    x, a = _inputs(4, 300, torch.float32, 20, 4, 2)
    a["bias"][0, 0] = 0.0
    a = _to(a)
    d = x.to(DEV)
    good = process_logits(d, **a)

    def bad(message, row, nan, **change):
        b = {**a, **change}
        with pytest.raises(ValueError, match=message):
            process_logits(d, **b)
        got = process_logits(d, **b, check=False)
        others = [r for r in range(4) if r != row]
        assert torch.equal(got[others], good[others])
        assert bool(got[row].isnan().all()) == nan
        own = d.clone()
        process_logits(own, **b, check=False, out=own)
        assert torch.equal(own.nan_to_num(9e9), got.nan_to_num(9e9))

    def at(name, row, value, col=None):
        t = a[name].clone()
        t[(row,) if col is None else (row, col)] = value
        return {name: t}

    live = 1 if a["repetition_penalty"][1] != 1 else 2
    for value in (0.0, -1.0, INF, math.nan):
        bad("repetition penalties must be", live, True, **at("repetition_penalty", live, value))
    bad("the other penalties finite", live, True, **at("presence_penalty", live, INF))
    bad("the other penalties finite", live, True, **at("frequency_penalty", live, math.nan))
    bad("mask_rows names a mask", 3, True, **at("mask_rows", 3, 2))
    bad("history token ID", 0, False, **{**at("history", 0, 300, 0), **at("history_lens", 0, 20)})
    bad("biased token ID", 2, False, **at("bias_ids", 2, 1 << 40, 1))
    empty = a["token_mask"].clone()
    empty[1] = 0
    empty[1, -1] = ~((1 << 300 % 32) - 1)  # only bits past the vocabulary
    b = {**a, "token_mask": empty, "mask_rows": torch.tensor([0, 1, -1, 0], dtype=torch.int32, device=DEV)}
    with pytest.raises(ValueError, match="leaves a row without tokens"):
        process_logits(d, **b)
    got = process_logits(d, **b, check=False)
    assert bool((got[1] == a["fill"]).all())
    # a gradient of such rows: NaN for bad knobs, zeros for a mask without tokens
    leaf = d.clone().requires_grad_()
    (grad,) = torch.autograd.grad(process_logits(leaf, **b, check=False), leaf, torch.ones_like(d))
    assert bool((grad[1] == 0).all())


def test_special_values():
    x = torch.tensor([[INF, -INF, math.nan, 0.0, -0.0, 3.0, 1e38, -1e38]], device=DEV)
    h = torch.arange(8, device=DEV)[None]
    got = process_logits(x, history=h, repetition_penalty=2.0)
    want = torch.tensor([[INF, -INF, math.nan, 0.0, -0.0, 1.5, 5e37, -2e38]], device=DEV)
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    # what a mask leaves out is gone, a NaN or an infinity too, and its gradient is 0 even where the one from above is NaN
    mask = torch.tensor([0b11111000], dtype=torch.int32, device=DEV)
    leaf = x.clone().requires_grad_()
    y = process_logits(leaf, token_mask=mask, fill=torch.finfo(torch.float32).min)
    assert y[0, :3].tolist() == [torch.finfo(torch.float32).min] * 3 and torch.equal(y[0, 3:], x[0, 3:])
    (grad,) = torch.autograd.grad(y, leaf, torch.full_like(x, math.nan))
    assert grad[0, :3].tolist() == [0.0] * 3 and bool(grad[0, 3:].isnan().all())
    # at x + b = 0 the slope is the penalty's of numbers that are not positive, as the forward multiplies there
    leaf = torch.tensor([[0.0, -0.0, 1.0, -1.0]], device=DEV, requires_grad=True)
    y = process_logits(leaf, history=h[:, :4], repetition_penalty=2.0, bias_ids=torch.tensor([2], device=DEV),
                       bias=torch.tensor([-1.0], device=DEV))
    (grad,) = torch.autograd.grad(y.sum(), leaf)
    assert grad.tolist() == [[2.0, 2.0, 2.0, 2.0]]


def test_shared_lists_rows_and_masks():
    x, a = _inputs(6, 900, torch.bfloat16, 0, 7, 1, seed=1)
    del a["mask_rows"]
    ids, b = a["bias_ids"][0], torch.randn(7)
    one = process_logits(x.to(DEV), bias_ids=ids.to(DEV), bias=b.to(DEV), token_mask=a["token_mask"][0].to(DEV), fill=-5.0)
    each = process_logits(x.to(DEV), bias_ids=ids.expand(6, 7).to(DEV), bias=b.expand(6, 7).to(DEV),
                          token_mask=a["token_mask"].to(DEV).expand(6, -1), fill=-5.0)
    assert torch.equal(one, each)
    # rows that are all the same one, processed differently
    row = x[:1].to(DEV).expand(6, 900)
    h = torch.arange(6, device=DEV)[:, None]
    got = process_logits(row, history=h, presence_penalty=1.0)
    want = row.float() - (torch.arange(900, device=DEV) == h).float()
    assert torch.equal(got, want.bfloat16())
    # a history whose rows are the same, in another integer type
    got = process_logits(x.to(DEV), history=h[:1].int().expand(6, 1), frequency_penalty=1.0)
    assert torch.equal(got[:, 1:], x.to(DEV)[:, 1:]) and torch.equal(got[:, 0], (x[:, 0].float() - 1).bfloat16().to(DEV))


def test_no_rows_and_no_history():
    x = torch.zeros(0, 50, device=DEV)
    assert process_logits(x, token_mask=torch.zeros(1, 2, dtype=torch.int32, device=DEV)).shape == (0, 50)
    x = torch.randn(2, 50, device=DEV)
    h = torch.zeros(2, 0, dtype=torch.int64, device=DEV)
    assert torch.equal(process_logits(x, history=h, repetition_penalty=2.0), x)
    h = torch.zeros(2, 4, dtype=torch.int64, device=DEV)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert torch.equal(process_logits(x, history=h, history_lens=lens, repetition_penalty=2.0), x)
    assert torch.equal(process_logits(x), x)
    half = x.half()
    assert process_logits(half).dtype == torch.float32


def test_longest_lists():
    # 4095 biases, and one token 524287 times
    V = 9000
    x = torch.randn(1, V, device=DEV)
    ids = torch.arange(4095, device=DEV) * 2
    b = torch.randn(4095, device=DEV)
    got = process_logits(x, bias_ids=ids, bias=b)
    want = x.clone()
    want[0, ids] += b
    assert torch.equal(got, want)
    h = torch.full((1, 524287), 8999, device=DEV)
    got = process_logits(x, history=h, frequency_penalty=1.0)
    want = x.clone()
    want[0, 8999] = x[0, 8999] - 524287.0
    assert torch.equal(got, want)


def test_captured_and_on_other_streams():
    x, a = _inputs(50, 8200, torch.float32, 90, 5, 4)
    a = _to(a)
    d = x.to(DEV)
    out = torch.empty_like(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        process_logits(d, **a, out=out, check=False)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        process_logits(d, **a, out=out, check=False)
    for k in range(3):
        d.copy_(torch.randn(d.shape, generator=torch.Generator(device=DEV).manual_seed(k), device=DEV))
        a["history"].random_(0, 8200)
        want = process_logits(d, **a, check=False)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.nan_to_num(), want.nan_to_num())
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            process_logits(d, **a)


def test_refusals_on_the_gpu():
    x = torch.zeros(2, 40, device=DEV, requires_grad=True)
    d = x.detach()
    with pytest.raises(ValueError, match="no gradient"):
        process_logits(x, out=torch.empty_like(d))
    for out in (torch.empty(2, 41, device=DEV), torch.empty(2, 40, device=DEV).bfloat16(), torch.empty(2, 40),
                torch.empty(40, 2, device=DEV).t(), torch.empty(1, 40, device=DEV).expand(2, 40)):
        with pytest.raises(ValueError, match="out must"):
            process_logits(d, out=out)
    big = torch.zeros(3, 40, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        process_logits(big[:2], out=big[1:])
    with pytest.raises(NotImplementedError, match="bias has no gradient"):
        process_logits(d, bias_ids=torch.zeros(1, dtype=torch.int64), bias=torch.zeros(1, requires_grad=True))
    y = process_logits(x, history=torch.zeros(2, 1, dtype=torch.int64, device=DEV), repetition_penalty=2.0)
    (grad,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(grad.sum(), x)
    # a list that was written between the two passes is refused, as autograd refuses its own saved tensors
    h = torch.zeros(2, 1, dtype=torch.int64, device=DEV)
    y = process_logits(x, history=h, repetition_penalty=2.0)
    h.fill_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    # so is a tensor that a call wrote through out
    z = torch.zeros(2, 40, device=DEV, requires_grad=True)
    w = torch.ones(2, 40, device=DEV)
    loss = (z * w).sum()
    with torch.no_grad():
        process_logits(d, out=w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("rows,V,hist,bias,masks", [(1100, 300, 60, 9, 5), (530, 20001, 700, 64, 0), (1030, 16385, 16383, 0, 3),
                                                    (1030, 5000, 16384, 3, 0), (1030, 5000, 40, 65, 2)])
def test_many_bf16_rows_are_those_of_few(rows, V, hist, bias, masks):
    # large batches of bf16 rows keep what the lists say in words of 16 bits, where those hold it; small ones in 32
    x, a = _inputs(rows, V, torch.bfloat16, hist, bias, masks, pad=3)
    a["history"][0] = V - 1  # one token as often as the list is long
    a["history_prompt_lens"][0] = 0
    a["history"][1] = 7
    a["history_prompt_lens"][1] = hist
    a, d = _to(a), x.to(DEV)
    up = torch.randn(rows, V, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).bfloat16()

    def part(take):
        return {k: v[take] if isinstance(v, torch.Tensor) and k != "token_mask" else v for k, v in a.items()}

    def both(take):
        leaf = d[take].detach().requires_grad_()
        y = process_logits(leaf, **part(take))
        own = d[take].clone()
        process_logits(own, **part(take), out=own)
        assert torch.equal(own, y)
        return y.detach(), torch.autograd.grad(y, leaf, up[take])[0]

    whole = both(slice(None))
    for r in range(0, rows, 50):
        take = slice(r, min(rows, r + 50))
        for u, v in zip(whole, both(take)):
            assert torch.equal(u[take], v)
    few = [0, 1, 2, rows // 2, rows - 1]
    small = {k: v[few].cpu() if isinstance(v, torch.Tensor) and k != "token_mask" else v.cpu() if isinstance(v, torch.Tensor) else v
             for k, v in a.items()}
    want, bound, grad, gbound = _plain(x[few], small, up[few].cpu())
    _close(whole[0][few], want, bound)
    _close(whole[1][few], grad, gbound)


def test_longest_lists_of_bf16_rows():
    V = 9000
    x = torch.randn(1, V, device=DEV).bfloat16()
    ids = torch.arange(4095, device=DEV) * 2
    b = torch.randn(4095, device=DEV)
    want = x.float()
    want[0, ids] += b
    assert torch.equal(process_logits(x, bias_ids=ids, bias=b), want.bfloat16())
    h = torch.full((1, 524287), 8999, device=DEV)
    want = x.float()
    want[0, 8999] = want[0, 8999] - 524287.0
    assert torch.equal(process_logits(x, history=h, frequency_penalty=1.0), want.bfloat16())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hist", [None, 0])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("rows", [4, 1030])
def test_penalties_of_rows_without_a_history(dtype, hist, masked, rows):
    # looked at all the same: the row of an invalid one holds NaN, its gradient too, and a checked call raises
    V = 8200
    g = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.randn(rows, V, generator=g, device=DEV).to(dtype)
    a = {} if hist is None else {"history": torch.zeros(rows, 0, dtype=torch.int64, device=DEV)}
    if masked:
        a["token_mask"] = torch.full((1, (V + 31) // 32), 0x55555555, dtype=torch.int32, device=DEV)
        a["fill"] = -5.0
    want = process_logits(x, **a)
    up = torch.randn(rows, V, generator=g, device=DEV).to(dtype)
    slope = torch.where(torch.arange(V, device=DEV) % 2 == 0, up, 0.0) if masked else up
    for name, value in (("repetition_penalty", 0.0), ("repetition_penalty", INF), ("presence_penalty", math.nan),
                        ("frequency_penalty", -INF)):
        knob = torch.rand(rows, generator=g, device=DEV) + 0.5
        assert torch.equal(process_logits(x, **a, **{name: knob}), want)
        knob[rows - 2] = value
        with pytest.raises(ValueError, match="repetition penalties must be finite and positive, the other penalties finite"):
            process_logits(x, **a, **{name: knob})
        leaf = x.clone().requires_grad_()
        y = process_logits(leaf, **a, **{name: knob}, check=False)
        (grad,) = torch.autograd.grad(y, leaf, up)
        own = x.clone()
        process_logits(own, **a, **{name: knob}, check=False, out=own)
        good = torch.arange(rows, device=DEV) != rows - 2
        for got, right in ((y.detach(), want), (own, want), (grad, slope)):
            assert bool(got[rows - 2].isnan().all()) and torch.equal(got[good], right[good])


def test_an_out_that_is_no_tensor_is_refused():
    x = torch.zeros(2, 40, device=DEV)
    for logits in (x, x.clone().requires_grad_()):
        for bad in (3, [x], "out"):
            with pytest.raises(ValueError, match="out must have the shape"):
                process_logits(logits, out=bad)
