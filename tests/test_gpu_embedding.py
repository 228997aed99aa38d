"""token_embedding and its gradient against 64-bit sums."""

import math

import pytest
import torch

from dsv41_rocm import selected_log_probs, token_embedding, token_embedding_backward

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _ids(kind, n, V, g):
    if kind == "random":
        ids = torch.randint(0, V, (n,), generator=g)
    elif kind == "one":
        ids = torch.full((n,), V - 1)
    elif kind == "falling":
        ids = (V - 1 - torch.arange(n) // 3) % V
    elif kind == "zipf":
        ids = (torch.exp(torch.rand(n, generator=g) * math.log(V)) - 1).long().clamp_(0, V - 1)
    else:
        ids = torch.full((n,), -1)
    if kind in ("random", "zipf"):
        ids[torch.rand(n, generator=g) < 0.1] = -1
    return ids


def _plain(ids, grad, V, scale):
    """(sums, their bound before the last rounding): fp32 sums of m terms in sequence, and of partial sums, are off by
    (m - 1) 2^-24 sum |g| at most whatever the order, the product by the scale by 2^-24 more (and the scale itself by
    as much, where it is no fp32 number)."""
    ok = (ids >= 0) & (ids < V)
    g = grad.double()[ok]
    out = torch.zeros(V, g.shape[1], dtype=torch.float64).index_add_(0, ids[ok], g)
    size = torch.zeros_like(out).index_add_(0, ids[ok], g.abs())
    m = torch.bincount(ids[ok], minlength=V)[:, None].double()
    return out * scale, size * abs(scale) * (m + 2) * 2.0 ** -24


CASES = [(1, 1, 1), (1, 8, 511), (31, 5, 512), (32, 64, 513), (33, 127, 100), (64, 1030, 2000), (65, 8, 7), (1000, 130, 1500),
         (3000, 33, 40), (257, 2048, 5000)]


@pytest.mark.parametrize("tg,to", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                   (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("kind", ["random", "one", "falling", "zipf", "padding"])
@pytest.mark.parametrize("n,h,V", CASES)
def test_gradient(n, h, V, kind, tg, to):
    g = torch.Generator().manual_seed(n + h + V)
    ids = _ids(kind, n, V, g)
    grad = torch.randn(n, h, generator=g).to(tg)
    scale = 1.0 if n % 2 else 0.37
    want, bound = _plain(ids, grad, V, scale)
    half = torch.finfo(to).eps / 2
    got = token_embedding_backward(grad.to(DEV), ids.to(DEV), V, scale=scale, dtype=to)
    assert got.dtype == to and got.shape == (V, h)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound + half * (want.abs() + bound)).all()), float((err - bound - half * want.abs()).max())
    assert torch.equal(got, token_embedding_backward(grad.to(DEV), ids.to(DEV), V, scale=scale, dtype=to))
    # onto what is there, in a matrix of rows further apart: absent rows and what lies between keep their bits
    base = torch.randn(V, h + 3, generator=g).to(to)
    onto = base.to(DEV)
    view = onto[:, 1:h + 1]
    assert token_embedding_backward(grad.to(DEV), ids.to(DEV), scale=scale, out=view) is view
    total = base[:, 1:h + 1].double() + want
    err = (view.double().cpu() - total).abs()
    assert bool((err <= bound + (2.0 ** -24 + half) * (total.abs() + bound) * 1.001).all())
    there = torch.zeros(V, dtype=torch.bool)
    there[ids[ids >= 0]] = True
    assert torch.equal(onto.cpu()[~there], base[~there])
    assert torch.equal(onto.cpu()[:, 0], base[:, 0]) and torch.equal(onto.cpu()[:, h + 1:], base[:, h + 1:])


@pytest.mark.parametrize("n,h,V", [(4000, 9, 140000), (2500, 20, 131072), (6000, 8, 70000), (5000, 4, 300)])
@pytest.mark.parametrize("kind", ["zipf", "few", "two"])
def test_gradient_of_ids_close_together(n, h, V, kind):
    # most of the batch in one range of ids: many of them among 64 neighbours, few, and two in turn; integers, so exact
    g = torch.Generator().manual_seed(n)
    if kind == "zipf":
        ids = _ids("zipf", n, V, g)
    elif kind == "few":
        ids = torch.randint(0, 5, (n,), generator=g) * 7 + V - 40
    else:
        ids = torch.arange(n) % 2 * 3 + 100
    grad = torch.randint(-8, 9, (n, h), generator=g).float()
    want = torch.zeros(V, h).index_add_(0, ids.clamp_min(0), torch.where((ids >= 0)[:, None], grad, 0.0))
    assert torch.equal(token_embedding_backward(grad.to(DEV), ids.to(DEV), V).cpu(), want)
    onto = torch.ones(V, h, dtype=torch.float32, device=DEV)
    token_embedding_backward(grad.to(DEV), ids.to(DEV), out=onto)
    assert torch.equal(onto.cpu(), want + 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,h,V", CASES)
def test_rows(n, h, V, dtype):
    g = torch.Generator().manual_seed(n + h + V)
    ids = _ids("random", n, V, g)
    table = torch.randn(V, h + 5, generator=g).to(dtype)
    for scale in (1.0, math.sqrt(h) + 0.1):
        got = token_embedding(ids.to(DEV), table.to(DEV)[:, 3:h + 3], scale=scale).cpu()
        # one fp32 product, rounded once
        s = torch.tensor(scale, dtype=torch.float32)
        want = (table[ids.clamp_min(0), 3:h + 3].float() * s).to(dtype).masked_fill(ids[:, None] < 0, 0.0)
        assert got.dtype == dtype and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autograd(dtype):
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(-1, 60, (4, 25), generator=g)
    table = torch.randn(60, 48, generator=g).to(dtype)
    up = torch.randn(4, 25, 48, generator=g).to(dtype)
    leaf = table.to(DEV).requires_grad_()
    out = token_embedding(ids.to(DEV), leaf, scale=2.5)
    assert out.shape == (4, 25, 48) and out.dtype == dtype
    (got,) = torch.autograd.grad(out, leaf, up.to(DEV))
    want, bound = _plain(ids.reshape(-1), up.reshape(-1, 48), 60, 2.5)
    half = torch.finfo(dtype).eps / 2
    assert bool(((got.double().cpu() - want).abs() <= bound + half * (want.abs() + bound)).all())
    # an upstream gradient that is one row everywhere
    out = token_embedding(ids.to(DEV), leaf)
    (got,) = torch.autograd.grad(out, leaf, torch.ones(48, dtype=dtype, device=DEV).expand(4, 25, 48))
    count = torch.bincount(ids[ids >= 0], minlength=60).double()
    assert torch.equal(got.double().cpu(), count[:, None].expand(60, 48))


def test_gradient_against_differences():
    # linear in the table: a step of 1 in one element moves the sum of the results by scale times its count,
    # exactly in fp32 for these numbers
    ids = torch.tensor([3, 1, 3, -1, 3, 0], device=DEV)
    table = torch.zeros(5, 4, device=DEV, requires_grad=True)
    (grad,) = torch.autograd.grad(token_embedding(ids, table, scale=0.5).sum(), table)
    for v in range(5):
        step = torch.zeros(5, 4, device=DEV)
        step[v, 2] = 1.0
        with torch.no_grad():
            moved = token_embedding(ids, table + step, scale=0.5).sum()
        assert float(moved) == float(grad[v, 2])


def test_ids_outside_the_vocabulary():
    table = torch.randn(10, 16, device=DEV, requires_grad=True)
    ids = torch.tensor([2, 10, -5, 1 << 40, 9], device=DEV)
    with pytest.raises(ValueError, match="token ID is outside the model vocabulary"):
        token_embedding(ids, table)
    out = token_embedding(ids, table, check=False)
    assert out.isnan().all(1).tolist() == [False, True, False, True, False]
    assert bool((out[2] == 0).all()) and torch.equal(out[[0, 4]], table.detach()[[2, 9]])
    (grad,) = torch.autograd.grad(out, table, torch.ones_like(out))
    assert grad[:, 0].tolist() == [0, 0, 1, 0, 0, 0, 0, 0, 0, 1]


@pytest.mark.parametrize("n", [1, 63, 1024, 1025, 5000, 300001])
@pytest.mark.parametrize("train", [False, True])
def test_one_id_outside_among_many(n, train):
    # the check looks at every id, wherever it lies and however the ids are aligned; the next call is sound again
    table = torch.randn(50, 4, device=DEV, requires_grad=train)
    g = torch.Generator(DEV).manual_seed(n)
    ids = torch.randint(-3, 50, (n + 1,), generator=g, device=DEV)
    for shift in (0, 1):
        mine = ids[shift:shift + n].clone() if shift == 0 else ids[shift:]
        assert token_embedding(mine, table).shape == (n, 4)
        for at in {0, n // 2, n - 1}:
            good = int(mine[at])
            for bad in (50, 1 << 40):
                mine[at] = bad
                with pytest.raises(ValueError, match="token ID is outside the model vocabulary"):
                    token_embedding(mine, table)
            mine[at] = good
    want = torch.where((mine >= 0)[:, None], table.detach()[mine.clamp_min(0)], 0.0)
    assert torch.equal(token_embedding(mine, table).detach(), want)


def test_checked_behind_work_that_takes_long():
    # the answer comes long after the host begins to look for it, on a stream of its own too
    table = torch.randn(60, 32, device=DEV, requires_grad=True)
    ids = torch.randint(0, 60, (100,), device=DEV)
    bad = ids.clone()
    bad[57] = 60
    a = torch.rand(4096, 4096, device=DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            for _ in range(8):
                b = a @ a
            rows = token_embedding(ids, table)
            for _ in range(8):
                b = a @ a
            with pytest.raises(ValueError, match="token ID is outside the model vocabulary"):
                token_embedding(bad, table)
            (grad,) = torch.autograd.grad(rows.sum(), table)
        torch.cuda.synchronize()
        assert torch.equal(rows.detach(), table.detach()[ids])
        assert torch.equal(grad, torch.bincount(ids, minlength=60).float()[:, None].expand(60, 32))
        del b


def test_no_tokens():
    table = torch.randn(10, 16, device=DEV, requires_grad=True)
    ids = torch.zeros(3, 0, dtype=torch.int64, device=DEV)
    out = token_embedding(ids, table)
    assert out.shape == (3, 0, 16)
    (grad,) = torch.autograd.grad(out.sum(), table)
    assert bool((grad == 0).all())
    onto = torch.ones(10, 16, device=DEV)
    token_embedding_backward(out.detach(), ids, out=onto)
    assert bool((onto == 1).all())


def test_tied_table_together():
    # embedding, a head of the same table, and the sum of the two gradients: autograd's, and by hand with out
    g = torch.Generator().manual_seed(8)
    table = (0.3 * torch.randn(400, 64, generator=g)).bfloat16()
    ids, targets = torch.randint(0, 400, (50,), generator=g), torch.randint(0, 400, (50,), generator=g)
    leaf = table.to(DEV).requires_grad_()
    x = token_embedding(ids.to(DEV), leaf, scale=8.0)
    lp, _, _ = selected_log_probs(x, leaf, targets.to(DEV))
    (grad,) = torch.autograd.grad(lp.sum(), leaf)
    # the same with 64-bit log-probs of the bf16 rows that the head saw
    ref = table.double().requires_grad_()
    rows = (ref[ids] * 8.0)
    rows = rows + (rows.detach().bfloat16().double() - rows.detach())
    want, = torch.autograd.grad((rows @ ref.t()).log_softmax(1).gather(1, targets[:, None]).sum(), ref)
    # the head's logit gradient, dx, dw and this one are rounded to bf16 on the way
    assert float((grad.double().cpu() - want).norm() / want.norm()) < 4 * 2.0 ** -8
    head = torch.zeros(400, 64, dtype=torch.float32, device=DEV)
    up = torch.randn(50, 64, generator=g).bfloat16()
    base = torch.randn(400, 64, generator=g)
    head.copy_(base)
    token_embedding_backward(up.to(DEV), ids.to(DEV), scale=8.0, out=head)
    part, bound = _plain(ids, up, 400, 8.0)
    assert bool(((head.double().cpu() - base - part).abs() <= bound + 2.0 ** -23 * (base.abs() + part.abs())).all())


def test_captured():
    g = torch.Generator(device=DEV).manual_seed(1)
    n, h, V = 700, 96, 1300
    ids = torch.randint(0, V, (n,), generator=g, device=DEV)
    grad = torch.randn(n, h, generator=g, device=DEV)
    onto = torch.zeros(V, h, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token_embedding_backward(grad, ids, V)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dense = token_embedding_backward(grad, ids, V)
        token_embedding_backward(grad, ids, out=onto)
    for k in range(3):
        ids.copy_(torch.randint(-1, V // (k + 1), (n,), generator=g, device=DEV))
        grad.copy_(torch.randn(n, h, generator=g, device=DEV))
        want = token_embedding_backward(grad, ids, V)
        onto.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dense, want) and torch.equal(onto, want)


def test_refusals_on_the_gpu():
    table = torch.randn(10, 16, device=DEV)
    ids = torch.zeros(3, dtype=torch.int64, device=DEV)
    grad = torch.randn(3, 16, device=DEV)
    with pytest.raises(ValueError, match="fp32 or bf16"):
        token_embedding(ids, table.half())
    with pytest.raises(ValueError, match="integers"):
        token_embedding(ids.float(), table)
    with pytest.raises(ValueError, match="scale must be finite"):
        token_embedding(ids, table, scale=math.inf)
    with pytest.raises(ValueError, match="grad must have"):
        token_embedding_backward(grad[:2], ids, 10)
    with pytest.raises(ValueError, match="vocabulary_size"):
        token_embedding_backward(grad, ids)
    with pytest.raises(ValueError, match="another vocabulary_size"):
        token_embedding_backward(grad, ids, 9, out=table)
    with pytest.raises(ValueError, match="do not overlap"):
        token_embedding_backward(grad, ids, out=table[:1].expand(10, 16))
    with pytest.raises(NotImplementedError, match="detach"):
        token_embedding_backward(grad, ids, out=table.clone().requires_grad_())
    leaf = table.clone().requires_grad_()
    out = token_embedding(ids, leaf)
    up = torch.ones_like(out, requires_grad=True)
    (dw,) = torch.autograd.grad(out, leaf, up, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(dw.sum(), up)
