"""The 8-bit head against integer arithmetic: quantized rows, their exact products, the two scales."""

import math

import pytest
import torch

from dsv41_rocm import Int8Head, head_logits, process_logits, quantize_head, sample

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _quantized(x):
    """(integers as fp64, fp32 scales) of bf16 rows on the CPU, by exact rational comparison in 64 bits: 127 x is
    exact, and its quotient by the maximum is a half exactly or clearly not."""
    x = x.double()
    top = x.abs().amax(1, keepdim=True)
    q = torch.round(127 * x / torch.where(top > 0, top, 1.0))
    return q, (top[:, 0].float() / 127.0)


def _want(x, w, t, dtype):
    """fp32 products in the kernels' order of the exact sums: bit for bit what they give."""
    q, s = _quantized(x)
    sums = q @ w.double().t()  # below 2^53
    return ((sums.float() * s[:, None]) * t).to(dtype)


def _inputs(n, h, v, seed=0):
    g = torch.Generator().manual_seed(n + 7 * h + 31 * v + seed)
    x = (torch.randn(n, h, generator=g) * torch.exp(torch.randn(h, generator=g))).bfloat16()
    w = (0.1 * torch.randn(v, h, generator=g)).bfloat16()
    return x, w


SIZES = [(1, 1, 1), (1, 127, 63), (2, 128, 64), (15, 129, 65), (16, 64, 1000), (17, 300, 100), (33, 2048, 130),
         (49, 255, 200), (64, 1024, 257), (65, 1024, 257), (100, 130, 255), (255, 256, 256), (256, 128, 513), (257, 384, 1000),
         (600, 513, 700)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,h,v", SIZES)
def test_exact(n, h, v, dtype):
    x, w = _inputs(n, h, v)
    head = quantize_head(w.to(DEV))
    q, t = _quantized(w)
    assert torch.equal(head.integers().cpu().double(), q) and torch.equal(head.scales.cpu(), t)
    again = Int8Head.from_quantized(head.integers(), head.scales)
    assert torch.equal(again.tiles, head.tiles) and (again.vocab, again.hidden) == (v, h)
    want = _want(x, q, t, dtype)
    got = head_logits(x.to(DEV), head, dtype=dtype)
    assert got.dtype == dtype and got.shape == (n, v)
    assert torch.equal(got.cpu(), want)
    # into rows of any alignment; nothing beside them is touched
    for pad in (1, 4):
        wide = torch.full((n, v + 2 * pad), 7.0, dtype=dtype, device=DEV)
        head_logits(x.to(DEV), head, out=wide[:, pad:pad + v])
        assert torch.equal(wide[:, pad:pad + v].cpu(), want)
        assert bool((wide[:, :pad] == 7).all()) and bool((wide[:, pad + v:] == 7).all())
    # hidden states at a stride
    big = torch.full((n, h + 3), 9.0, dtype=torch.bfloat16, device=DEV)
    big[:, 1:h + 1] = x.to(DEV)
    assert torch.equal(head_logits(big[:, 1:h + 1], head, dtype=dtype).cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [33, 48, 49, 64])
@pytest.mark.parametrize("h,v", [(4100, 32827), (4100, 65536), (4000, 32827), (4100, 32768)])
def test_many_groups(n, h, v, dtype):
    # two groups of 64 rows a workgroup, three in one of them, or a part of one at the end
    _many_rows(n, h, v, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,h,v", [(257, 128, 33000), (300, 129, 33000), (320, 300, 65536), (305, 513, 65537), (321, 257, 33000),
                                   (640, 256, 32500), (590, 384, 40001)])
def test_tiles_of_tokens(n, h, v, dtype):
    # rows for many workgroups, where the widest tiles of tokens are taken: full and cut ones, one stage and several
    _many_rows(n, h, v, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,h,v", [(17, 100, 70001), (64, 128, 65600), (65, 128, 70001), (128, 129, 70001), (100, 300, 140000),
                                   (40, 400, 140001), (128, 513, 20000), (70, 257, 64), (20, 130, 70)])
def test_rings(n, h, v, dtype):
    # runs of groups that make several blocks of rows, whole and not, of one stage, two and more
    _many_rows(n, h, v, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,h", [(1, 1), (1, 8), (2, 136), (3, 2040), (4, 2048), (5, 2048), (4, 2047), (4, 2056), (2, 7168), (1, 16385),
                                 (3, 700), (16, 2048), (4, 128)])
def test_tokens_quantized_by_the_product(n, h, dtype):
    # few short tokens are quantized in the product's own launch: full ones, cut ones, one too many, too long, of odd lengths
    _many_rows(n, h, 33000 + n, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,h,v", [(17, 64, 70001), (40, 128, 70001), (64, 100, 200), (65, 128, 70001), (128, 127, 140001)])
def test_scales_that_come_from_memory(n, h, v, dtype):
    # rows of one stage: the call before leaves another head's scales where this one's come to, and they come late, as no
    # cache holds them
    g = torch.Generator(DEV).manual_seed(n + h + v)
    x = _inputs(n, h, 1)[0]
    q, s = _quantized(x)
    w = torch.randint(-127, 128, (v, h), generator=g, dtype=torch.int8, device=DEV)
    sums = torch.cat([q.to(DEV) @ part.double().t() for part in w.split(8192)], 1).float() * s.to(DEV)[:, None]
    scales = [torch.rand(v, generator=g, device=DEV) + k for k in (1, 100)]
    heads = [Int8Head.from_quantized(w, t) for t in scales]
    x = x.to(DEV)
    junk = torch.empty(1 << 30, dtype=torch.int8, device=DEV)
    outs = []
    for k in (0, 1, 0):
        junk.fill_(k)
        outs.append((k, head_logits(x, heads[k], dtype=dtype, check=False)))
    for k, got in outs:
        assert torch.equal(got, (sums * scales[k]).to(dtype))


def _many_rows(n, h, v, dtype):
    x = _inputs(n, h, 1)[0]
    w = torch.randint(-127, 128, (v, h), generator=torch.Generator(DEV).manual_seed(n + h + v), dtype=torch.int8, device=DEV)
    t = torch.rand(v, generator=torch.Generator(DEV).manual_seed(n), device=DEV)
    q, s = _quantized(x)
    sums = torch.cat([q.to(DEV) @ part.double().t() for part in w.split(8192)], 1)  # integers below 2^53
    want = ((sums.float() * s.to(DEV)[:, None]) * t).to(dtype)
    wide = torch.full((n, v + 16), 7.0, dtype=dtype, device=DEV)
    head_logits(x.to(DEV), Int8Head.from_quantized(w, t), out=wide[:, 8:8 + v])
    assert torch.equal(wide[:, 8:8 + v], want)
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + v:] == 7).all())


def test_ties_and_borders():
    # against a maximum of 254, odd numbers are ties, and go to the even integer
    x = torch.arange(-254.0, 255.0).bfloat16()[None]
    head = Int8Head.from_quantized(torch.eye(509, dtype=torch.int8, device=DEV), torch.ones(509, device=DEV))
    got = head_logits(x.to(DEV), head)[0].cpu()
    want = torch.round(x[0].double() / 2).float() * (torch.tensor(254.0) / 127)
    assert torch.equal(got, want)


@pytest.mark.parametrize("scale", [2.0**-133, 2.0**-126, 2.0**-101, 2.0**-100, 2.0**-99, 2.0**-7, 2.0**92, 2.0**93, 2.0**120])
def test_every_quotient(scale):
    # every mantissa of the largest against every mantissa, at every exponent that is not far below a half of a step
    a = torch.arange(128, 256, dtype=torch.float64)
    x = torch.cat([a * 2.0**-s for s in range(10)] + [torch.zeros(1, dtype=torch.float64)])
    rows = torch.where(x[None, :] <= a[:, None], x[None, :], 0.0).repeat(1, 2)
    rows[:, x.numel():] *= -1
    rows[:, x.numel() - 1] = a
    rows = (rows * scale).bfloat16()  # (exact but for the subnormal ones, which are rounded before both sides see them)
    q, s = _quantized(rows)
    head = quantize_head(rows.to(DEV))
    assert torch.equal(head.integers().cpu().double(), q) and torch.equal(head.scales.cpu(), s)
    eye = Int8Head.from_quantized(torch.eye(rows.shape[1], dtype=torch.int8, device=DEV), torch.ones(rows.shape[1], device=DEV))
    want = q.float() * s[:, None]
    for n in (2, 16, 128):  # quantized by the product, and before it
        assert torch.equal(torch.cat([head_logits(part, eye) for part in rows.to(DEV).split(n)]).cpu(), want)


@pytest.mark.parametrize("n", [3, 70])
@pytest.mark.parametrize("top", [1e-38, 1e-40, 3e38, 1.0])
def test_magnitudes(n, top):
    # subnormal and enormous rows, and a row of zeros
    x, w = _inputs(n, 200, 90)
    x = (x.double() / x.double().abs().amax() * top).bfloat16()
    x[1] = 0
    q, t = _quantized(w)
    got = head_logits(x.to(DEV), quantize_head(w.to(DEV))).cpu()
    want = _want(x, q, t, torch.float32)
    assert bool((got[1] == 0).all())
    assert torch.equal(got, want)


@pytest.mark.parametrize("n", [2, 70])
def test_largest_sums(n):
    h = 133120
    x = torch.full((n, h), 3.0, dtype=torch.bfloat16, device=DEV)
    x[1] = -3.0
    w = torch.full((70, h), 127, dtype=torch.int8, device=DEV)
    got = head_logits(x, Int8Head.from_quantized(w, torch.ones(70, device=DEV)))
    want = float(torch.tensor(float(h * 127 * 127)) * (torch.tensor(3.0) / 127))
    assert bool((got[0] == want).all()) and bool((got[1] == -want).all())
    with pytest.raises(NotImplementedError, match="overflow"):
        head_logits(torch.zeros(1, h + 1, device=DEV), Int8Head.from_quantized(w[:, :1].expand(70, h + 1), torch.ones(70, device=DEV)))


@pytest.mark.parametrize("n", [2, 70, 200])
def test_largest_sums_of_the_lowest_integer(n):
    # 127 times -128, as often as 32 bits hold, in either sign: 132104 * 127 * 128 = 2^31 - 1024
    h = 132104
    x = torch.full((n, h), 127.0, dtype=torch.bfloat16, device=DEV)
    x[1] = -127.0
    w = torch.full((70, h), -128, dtype=torch.int8, device=DEV)
    got = head_logits(x, Int8Head.from_quantized(w, torch.ones(70, device=DEV)))
    want = float(2 ** 31 - 1024)
    assert bool((got[0] == -want).all()) and bool((got[1] == want).all())
    wide = torch.full((3, h + 1), 127, dtype=torch.int8, device=DEV)
    Int8Head.from_quantized(wide, torch.ones(3, device=DEV))
    wide[2, h] = -128
    with pytest.raises(NotImplementedError, match="-128"):
        Int8Head.from_quantized(wide, torch.ones(3, device=DEV))


def test_accuracy_against_the_bf16_head():
    # rounding to 127 steps: each factor is off by half a step of its row's maximum at most, so a logit by
    # (|x|_1 max|w| + |w|_1 max|x|) / 254 and a quarter of a step's product a column
    x, w = _inputs(40, 2048, 300)
    got = head_logits(x.to(DEV), quantize_head(w.to(DEV))).double().cpu()
    x, w = x.double(), w.double()
    mx, mw = x.abs().amax(1, keepdim=True), w.abs().amax(1)
    bound = (x.abs().sum(1, keepdim=True) * mw + w.abs().sum(1) * mx) / 254 + 2048 * mx * mw / 254 ** 2
    assert bool(((got - x @ w.t()).abs() <= bound * 1.0001).all())


@pytest.mark.parametrize("n", [4, 100])
def test_rows_that_are_not_finite(n):
    x, w = _inputs(n, 300, 100)
    x, w = x.to(DEV), w.to(DEV)
    head = quantize_head(w)
    good = head_logits(x, head)
    for value in (math.nan, math.inf, -math.inf):
        y = x.clone()
        y[2, 299] = value
        with pytest.raises(ValueError, match="non-finite"):
            head_logits(y, head)
        got = head_logits(y, head, check=False)
        keep = [r for r in range(n) if r != 2]
        assert bool(got[2].isnan().all()) and torch.equal(got[keep], good[keep])
        b = w.clone()
        b[7, 0] = value
        with pytest.raises(ValueError, match="non-finite"):
            quantize_head(b)
        got = head_logits(x, quantize_head(b, check=False))
        assert bool(got[:, 7].isnan().all()) and torch.equal(got[:, 8:], good[:, 8:])


def test_rows_do_not_depend_on_their_batch():
    x, w = _inputs(300, 500, 700)
    head = quantize_head(w.to(DEV))
    x = x.to(DEV)
    whole = head_logits(x, head)
    for n in (1, 16, 40, 64, 65, 128):
        assert torch.equal(head_logits(x[5:5 + n], head), whole[5:5 + n])


def test_decode_step_together():
    # hidden states to a token through the head, a mask and the draw
    x, w = _inputs(24, 512, 5003)
    logits = head_logits(x.to(DEV), quantize_head(w.to(DEV)), dtype=torch.bfloat16)
    mask = torch.zeros(1, (5003 + 31) // 32, dtype=torch.int32, device=DEV)
    mask[0, 3] = 0b1010
    process_logits(logits, token_mask=mask, fill=-8192.0, out=logits)
    s = sample(logits, uniforms=torch.rand(24, generator=torch.Generator().manual_seed(1)))
    assert set(s.ids.tolist()) <= {97, 99}


def test_captured_with_own_workspaces():
    x, w = _inputs(20, 700, 900)
    head = quantize_head(w.to(DEV))
    a, b = x.to(DEV), torch.zeros_like(x, device=DEV)
    oa, ob = torch.empty(20, 900, device=DEV), torch.empty(20, 900, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        head_logits(a, head, out=oa, check=False)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        head_logits(a, head, out=oa, check=False)
    with torch.cuda.graph(gb):
        head_logits(b, head, out=ob, check=False)
    for k in range(3):
        a.copy_(torch.randn(20, 700, generator=torch.Generator(device=DEV).manual_seed(k), device=DEV))
        b.copy_(torch.randn(20, 700, generator=torch.Generator(device=DEV).manual_seed(10 + k), device=DEV))
        want = head_logits(a, head), head_logits(b, head)
        oa.fill_(1.0)
        ob.fill_(1.0)
        ga.replay()
        gb.replay()
        torch.cuda.synchronize()
        assert torch.equal(oa, want[0]) and torch.equal(ob, want[1])


def test_refusals_on_the_gpu():
    x, w = _inputs(3, 200, 50)
    head = quantize_head(w.to(DEV))
    d = x.to(DEV)
    assert head_logits(d[:0], head).shape == (0, 50)
    with pytest.raises(ValueError, match="hidden must be"):
        head_logits(d[:, :199], head)
    with pytest.raises(ValueError, match="float32 or torch.bfloat16"):
        head_logits(d, head, dtype=torch.float16)
    with pytest.raises(NotImplementedError, match="no gradient"):
        head_logits(d.float().requires_grad_(), head)
    with torch.no_grad():
        head_logits(d.float().requires_grad_(), head)
    with pytest.raises(NotImplementedError, match="no gradient"):
        quantize_head(w.to(DEV).requires_grad_())
    with pytest.raises(ValueError, match="layout"):
        head_logits(d, Int8Head(head.tiles[:-1], head.scales, 50, 200))
    with pytest.raises(ValueError, match="layout"):
        head_logits(d, Int8Head(head.tiles, head.scales.double(), 50, 200))
    with pytest.raises(ValueError, match="out must"):
        head_logits(d, head, out=torch.empty(3, 51, device=DEV))
    with pytest.raises(ValueError, match="do not overlap"):
        head_logits(d, head, out=torch.empty(1, 50, device=DEV).expand(3, 50))
    with pytest.raises(ValueError, match="one value per row"):
        Int8Head.from_quantized(torch.zeros(3, 4, dtype=torch.int8, device=DEV), torch.ones(4, device=DEV))


@pytest.mark.parametrize("n", [3, 40, 200])
def test_out_beside_what_is_read(n):
    # an out over the hidden states or the head is refused; columns beside them in the same buffer are not
    x, w = _inputs(n, 128, 64)
    head = quantize_head(w.to(DEV))
    want = head_logits(x.to(DEV), head, dtype=torch.bfloat16)
    both = torch.empty(n, 128 + 64, dtype=torch.bfloat16, device=DEV)
    both[:, :128] = x.to(DEV)
    hidden = both[:, :128]
    for out in (both[:, 64:128], both[:, :64], both.view(-1)[100:100 + 64 * n].view(n, 64)):
        with pytest.raises(ValueError, match="out overlaps"):
            head_logits(hidden, head, out=out)
    scales = torch.ones(64 * n + 64, device=DEV)
    with pytest.raises(ValueError, match="out overlaps"):
        head_logits(hidden, Int8Head(head.tiles, scales[:64], 64, 128), out=scales[60:60 + 64 * n].view(n, 64))
    tiles = torch.zeros(8192 + 256 * n, dtype=torch.int8, device=DEV)
    with pytest.raises(ValueError, match="out overlaps"):
        head_logits(hidden, Int8Head(tiles[:8192], head.scales, 64, 128), out=tiles[4096:4096 + 256 * n].view(torch.float32).view(n, 64))
    head_logits(hidden, head, out=both[:, 128:])
    assert torch.equal(both[:, 128:], want) and torch.equal(both[:, :128].cpu(), x)


def test_heads_and_outs_of_other_types_are_refused():
    x, w = _inputs(3, 200, 50)
    head = quantize_head(w.to(DEV))
    for bad in (w.to(DEV), None, (head.tiles, head.scales)):
        with pytest.raises(ValueError, match="Int8Head"):
            head_logits(x.to(DEV), bad)
    for bad in (3, [x]):
        with pytest.raises(ValueError, match="out must be"):
            head_logits(x.to(DEV), head, out=bad)
