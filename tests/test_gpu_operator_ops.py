"""torch.ops.dsv41_rocm.process_logits, head_logits and token_embedding: the functions' values and gradients, shapes
under a fake device, forward-mode tangents, saved tensors that move, and captured training steps."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from dsv41_rocm import head_logits, process_logits, quantize_head, token_embedding, token_embedding_backward

OPS = torch.ops.dsv41_rocm
DEV = "cuda"


def _process_inputs(device=DEV):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 3001, generator=g)
    a = dict(history=torch.randint(0, 3001, (6, 90), generator=g)[:, ::2], history_lens=torch.randint(0, 46, (6,), generator=g),
             history_prompt_lens=torch.randint(0, 20, (6,), generator=g), repetition_penalty=torch.rand(6, generator=g) + 0.7,
             presence_penalty=torch.rand(6, generator=g), frequency_penalty=torch.rand(6, generator=g),
             bias_ids=torch.randint(0, 3001, (6, 4), generator=g), bias=torch.randn(6, 4, generator=g),
             token_mask=torch.randint(-2 ** 31, 2 ** 31 - 1, (3, 200), generator=g, dtype=torch.int64).int()[:, :94],
             mask_rows=torch.tensor([0, -1, 2, 1, 1, -1]))
    return x.to(device), {k: v.to(device) for k, v in a.items()}


def _op(x, a, fill=-5.0):
    return OPS.process_logits(x, a["history"], a["history_lens"], a["history_prompt_lens"], 1.0, 0.0, 0.0,
                              a["repetition_penalty"], a["presence_penalty"], a["frequency_penalty"], a["bias_ids"], a["bias"],
                              a["token_mask"], a["mask_rows"], fill)


@pytest.mark.gpu
def test_process_op():
    x, a = _process_inputs()
    g = torch.randn(6, 3001, device=DEV)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        u, v = x.to(dtype).requires_grad_(), x.to(dtype).requires_grad_()
        want = process_logits(u, **a, fill=-5.0)
        got, status = _op(v, a)
        assert torch.equal(got, want) and int(status.max()) == 0
        (gu,), (gv,) = torch.autograd.grad(want, u, g.to(want.dtype)), torch.autograd.grad(got, v, g.to(got.dtype))
        assert torch.equal(gu, gv) and gv.dtype == dtype
    got, _ = OPS.process_logits(x, a["history"], None, None, 1.5, 0.25, 0.125, None, None, None, None, None, None, None, 0.0)
    assert torch.equal(got, process_logits(x, history=a["history"], repetition_penalty=1.5, presence_penalty=0.25,
                                           frequency_penalty=0.125))
    v = x.clone().requires_grad_()
    (gv,) = torch.autograd.grad(_op(v, a)[0].sum(), v, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        gv.sum().backward()


@pytest.mark.gpu
def test_head_op():
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(5, 200, generator=g).bfloat16().to(DEV), torch.randn(70, 200, generator=g).bfloat16().to(DEV)
    head = quantize_head(w)
    for dtype in (torch.float32, torch.bfloat16):
        got, status = OPS.head_logits(x, head.tiles, head.scales, 70, dtype)
        assert torch.equal(got, head_logits(x, head, dtype=dtype)) and int(status.max()) == 0


@pytest.mark.gpu
def test_embedding_op():
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(-1, 50, (3, 7), generator=g).to(DEV)
    w = torch.randn(50, 24, generator=g).to(DEV)
    up = torch.randn(3, 7, 24, generator=g).to(DEV)
    u, v = w.clone().requires_grad_(), w.clone().requires_grad_()
    want = token_embedding(ids, u, scale=3.0)
    got, status = OPS.token_embedding(ids, v, 3.0)
    assert torch.equal(got, want) and int(status.max()) == 0
    assert torch.equal(torch.autograd.grad(want, u, up)[0], torch.autograd.grad(got, v, up)[0])


def test_fake_shapes():
    with torch.device("meta"):
        x = torch.empty(6, 50)
        out, status = OPS.process_logits(x.bfloat16(), None, None, None, 1.0, 0.0, 0.0, None, None, None, None, None, None, None, 0.0)
        assert out.shape == (6, 50) and out.dtype == torch.bfloat16 and status.shape == (6,) and status.dtype == torch.int32
        out, status = OPS.head_logits(x, torch.empty(64 * 128, dtype=torch.int8), torch.empty(60), 60, torch.bfloat16)
        assert out.shape == (6, 60) and out.stride() == (64, 1) and out.dtype == torch.bfloat16 and status.shape == (6,)
        out, status = OPS.token_embedding(torch.empty(2, 3, dtype=torch.int64), x, 1.0)
        assert out.shape == (2, 3, 50) and status.shape == (6,)


def test_host_tensors_are_refused():
    x = torch.zeros(2, 5)
    with pytest.raises(NotImplementedError):
        OPS.process_logits(x, None, None, None, 1.0, 0.0, 0.0, None, None, None, None, None, None, None, 0.0)
    with pytest.raises(NotImplementedError):
        OPS.head_logits(x, torch.zeros(1, dtype=torch.int8), torch.zeros(5), 5, torch.float32)
    with pytest.raises(NotImplementedError):
        OPS.token_embedding(torch.zeros(2, dtype=torch.int64), x, 1.0)


@pytest.mark.gpu
def test_tangents_are_refused():
    x, a = _process_inputs()
    w = torch.randn(50, 24, device=DEV)
    ids = torch.zeros(3, dtype=torch.int64, device=DEV)
    with fwad.dual_level():
        dual, table = fwad.make_dual(x, torch.ones_like(x)), fwad.make_dual(w, torch.ones_like(w))
        for call in (lambda: process_logits(dual, **a), lambda: _op(dual, a), lambda: token_embedding(ids, table),
                     lambda: OPS.token_embedding(ids, table, 1.0), lambda: quantize_head(table),
                     lambda: head_logits(table, quantize_head(w)),
                     lambda: token_embedding_backward(fwad.make_dual(w[:3], w[:3]), ids, 50),
                     lambda: process_logits(x, bias_ids=a["bias_ids"], bias=fwad.make_dual(a["bias"], a["bias"]))):
            with pytest.raises(NotImplementedError, match="forward"):
                call()


@pytest.mark.gpu
def test_saved_tensors_that_move():
    # saved on the host and brought back, at other places and strides
    x, a = _process_inputs()
    leaf = x.requires_grad_()
    up = torch.randn(6, 3001, device=DEV)
    (want,) = torch.autograd.grad(process_logits(leaf, **a), leaf, up)
    with torch.autograd.graph.save_on_cpu():
        y = process_logits(leaf, **a)
        w = torch.randn(50, 24, device=DEV, requires_grad=True)
        ids = torch.arange(40, device=DEV)
        rows = token_embedding(ids, w)
    junk = [torch.full((6, 90), 1 << 20, dtype=torch.int64, device=DEV) for _ in range(8)]  # over memory that came free
    (got,) = torch.autograd.grad(y, leaf, up)
    assert torch.equal(got, want) and len(junk) == 8
    (dw,) = torch.autograd.grad(rows.sum(), w)
    assert dw[:, 0].tolist() == [1.0] * 40 + [0.0] * 10


@pytest.mark.gpu
def test_captured_training_step():
    x, a = _process_inputs()
    x = x.requires_grad_()
    table = torch.randn(80, 48, device=DEV, requires_grad=True)
    ids = torch.randint(-1, 80, (33,), device=DEV)
    up, ug = torch.randn(6, 3001, device=DEV), torch.randn(33, 48, device=DEV)

    def step():
        y = process_logits(x, **a, check=False)
        r = token_embedding(ids, table, scale=2.0, check=False)
        return (y, r, *torch.autograd.grad([y, r], [x, table], [up, ug]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        g = torch.Generator(device=DEV).manual_seed(k)
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
            table.copy_(torch.randn(table.shape, generator=g, device=DEV))
            up.copy_(torch.randn(up.shape, generator=g, device=DEV))
            ids.copy_(torch.randint(-1, 80 >> k, ids.shape, generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        for u, v in zip(got, want):
            assert torch.equal(u.detach().nan_to_num(), v.detach().nan_to_num())


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    x, a = _process_inputs()
    g = torch.Generator(device=DEV).manual_seed(4)
    w = torch.randn(5000, 256, generator=g, device=DEV).bfloat16()
    h = torch.randn(40, 256, generator=g, device=DEV).bfloat16()
    head = quantize_head(w)
    ids = torch.randint(0, 5000, (900,), generator=g, device=DEV)
    up = torch.randn(900, 256, generator=g, device=DEV).bfloat16()
    calls = (lambda: process_logits(x, **a, check=False), lambda: head_logits(h, head, check=False),
             lambda: token_embedding_backward(up, ids, 5000))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for k in range(6):
        for i, c in enumerate(calls):
            with torch.cuda.stream(streams[(i + k) % 3]):
                outs.append((i, c()))
    torch.cuda.synchronize()
    for i, o in outs:
        assert torch.equal(o.nan_to_num(), want[i].nan_to_num())


CONSTANTS = ["repetition_penalties", "presence_penalties", "frequency_penalties", "bias"]


def _op_of(x, **named):
    a = dict(history=torch.zeros(2, 4, dtype=torch.int64), bias_ids=torch.zeros(3, dtype=torch.int64), bias=torch.zeros(3))
    a = {k: v.to(x.device) for k, v in a.items()} | named
    return OPS.process_logits(x, a["history"], None, None, 1.0, 0.0, 0.0, *(a.get(k) for k in CONSTANTS[:3]), a["bias_ids"], a["bias"],
                              None, None, 0.0)


def _refuses_gradients_of_constants(device):
    # process_logits refuses them too: the op has no gradient to give
    x = torch.zeros(2, 40, device=device)
    for name in CONSTANTS:
        t = torch.ones(3 if name == "bias" else 2, device=device, requires_grad=True)
        for logits in (x, x.clone().requires_grad_()):
            with pytest.raises(NotImplementedError, match=f"{name} has no gradient"):
                _op_of(logits, **{name: t})
            assert _op_of(logits, **{name: t.detach()})[0].requires_grad == logits.requires_grad
            with torch.no_grad():
                assert not _op_of(logits, **{name: t})[0].requires_grad


def test_gradients_of_constants_are_refused_in_tracing():
    _refuses_gradients_of_constants("meta")


@pytest.mark.gpu
def test_gradients_of_constants_are_refused():
    _refuses_gradients_of_constants(DEV)
