"""Timed cases of the operators at a model's vocabulary: penalties, biases and token masks on rows of
logits with their gradient, logits from an 8-bit head, and the embedding of tokens with its gradient.

``listed()`` are fixed cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare(case,
seed)`` the inputs, ``run(state)`` one pass (elementary torch operations, or the package's calls
where ``own`` is set), ``work(case)`` what a pass cannot do without and ``exact(case, seed)`` its
outputs in 64 bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
FILL = -8192.0  # a token that is out for a sampler that takes finite logits only: of no mass at temperatures up to 200


def _process(rows, vocab, dtype, history=0, bias=0, masks=0.0, prompt=False, inplace=False, train=False, stride=None):
    return {"kind": "process", "rows": rows, "vocab": vocab, "stride": stride or vocab, "dtype": dtype,
            "history": history, "bias": bias, "masks": masks, "prompt": prompt, "inplace": inplace, "train": train}


def _head(rows, hidden, vocab, dtype):
    return {"kind": "head", "rows": rows, "hidden": hidden, "vocab": vocab, "dtype": dtype}


def _embed(tokens, hidden, vocab, dtype, train, scale=1.0, padding=0.0):
    return {"kind": "embed", "tokens": tokens, "hidden": hidden, "vocab": vocab, "dtype": dtype, "train": train,
            "scale": scale, "padding": padding}


def listed():
    return [
        # one response's decoding step: penalties over what it has said so far, and a few biased tokens
        {"name": "process_1", **_process(1, 129280, "f32", history=256, bias=8)},
        # a serving batch, half of whose requests follow a grammar; logits a view of a head padded to 128
        {"name": "process_48_grammar", **_process(48, 151851, "bf16", history=512, bias=16, masks=0.5, prompt=True,
                                                  stride=151936)},
        # constrained decoding of a whole batch, written over its own logits
        {"name": "process_256_mask_inplace", **_process(256, 151936, "bf16", masks=1.0, inplace=True)},
        # a learner's rows under the processing that its tokens were sampled with, and the gradient
        {"name": "process_500_grad", **_process(500, 151851, "bf16", history=2048, masks=0.3, prompt=True, train=True)},
        # rollouts with long ragged histories, the largest
        {"name": "process_2048", **_process(2048, 151936, "f32", history=4096)},
        # one decoded token
        {"name": "head_1", **_head(1, 7168, 129280, "f32")},
        # a decode batch, odd vocabulary
        {"name": "head_48", **_head(48, 2048, 151851, "bf16")},
        # a short prompt whose every position is scored
        {"name": "head_300", **_head(300, 7168, 129280, "f32")},
        # a microbatch of a teacher or a rollout engine's scoring pass, the largest
        {"name": "head_4096", **_head(4096, 2048, 151936, "bf16")},
        # a decode batch's tokens
        {"name": "embed_48", **_embed(48, 7168, 129280, "bf16", False)},
        # one response of a fp32 model, scaled by sqrt(hidden) as tied tables are
        {"name": "embed_1000_grad", **_embed(1000, 2048, 151851, "f32", True, scale=math.sqrt(2048))},
        # a padded microbatch of the learner, the largest
        {"name": "embed_16384_grad", **_embed(16384, 7168, 129280, "bf16", True, padding=0.1)},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["process", "head", "embed"])
    dtype = rng.choice(["f32", "bf16"])
    vocab = rng.choice([129280, 151936, 151851, _log_int(rng, 8192, 151936), _log_int(rng, 8192, 151936)])
    size = 4 if dtype == "f32" else 2
    if kind == "process":
        train = rng.random() < 0.35
        most = 2048 * 151936 * 8 // (vocab * size * (4 if train else 2))
        rows = _log_int(rng, 1, min(2048, most))
        stride = (vocab + 127) // 128 * 128 if rng.random() < 0.5 else vocab
        history = rng.choice([0, _log_int(rng, 1, 4096), _log_int(rng, 64, 4096)])
        bias = rng.choice([0, 0, _log_int(rng, 1, 300)])
        masks = rng.choice([0.0, 0.5, 1.0, round(rng.random(), 2)]) if history or bias else rng.choice([0.5, 1.0, 1.0])
        inplace = not train and masks == 1.0 and not history and not bias and rng.random() < 0.5
        return _process(rows, vocab, dtype, history, bias, masks, rng.random() < 0.5, inplace, train, stride)
    if kind == "head":
        hidden = rng.choice([7168, 2048, _log_int(rng, 256, 7168)])
        most = 4096 * 2048 * 151936 // (hidden * vocab)
        return _head(_log_int(rng, 1, min(4096, most)), hidden, vocab, dtype)
    hidden = rng.choice([7168, 2048, _log_int(rng, 64, 7168)])
    train = rng.random() < 0.7
    room = (129280 + 3 * 16384) * 7168 * 2 // (size * hidden) - (vocab if train else 0)
    if room < 1:
        dtype, room = "bf16", (129280 + 3 * 16384) * 7168 // hidden - vocab
    return _embed(_log_int(rng, 1, max(1, min(16384, room // 3))), hidden, vocab, dtype, train,
                  rng.choice([1.0, math.sqrt(hidden), round(rng.uniform(0.1, 12.0), 3)]), rng.choice([0.0, 0.1, 0.5]))


# ------------------------------------------------------------------------------------- inputs
def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _zipf_ids(shape, vocab, g):
    """Token ids with Zipf frequencies, the frequent ones spread over the vocabulary."""
    u = torch.rand(shape, generator=g, device=DEV, dtype=torch.float64)
    rank = (torch.exp(u * math.log(vocab)) - 1).long().clamp_(0, vocab - 1)
    return (rank * 7919 + 13) % vocab


def _prepare_process(case, g, state):
    rows, V = case["rows"], case["vocab"]
    full = torch.zeros(rows, case["stride"], dtype=_dtype(case), device=DEV)
    for r in range(0, rows, 512):
        e = min(rows, r + 512)
        full[r:e, :V] = 3.0 * torch.randn(e - r, V, generator=g, device=DEV)
    logits = full[:, :V]
    args = {}
    if case["history"]:
        L = case["history"]
        # half of what was said are frequent words, said again and again
        often = _zipf_ids((rows, L), V, g)
        seldom = torch.randint(0, V, (rows, L), generator=g, device=DEV)
        args["history"] = torch.where(torch.rand(rows, L, generator=g, device=DEV) < 0.5, often, seldom)
        args["history_lens"] = torch.randint((L + 1) // 2, L + 1, (rows,), generator=g, device=DEV, dtype=torch.int32)
        if case["prompt"]:
            share = torch.rand(rows, generator=g, device=DEV)
            args["history_prompt_lens"] = (share * args["history_lens"]).int()
        # every request comes with knobs of its own, some of them neutral
        pick = torch.randint(0, 3, (rows,), generator=g, device=DEV)
        knob = lambda values: torch.tensor(values, device=DEV)[pick]
        args["repetition_penalty"] = knob([1.05, 1.0, 1.2])
        args["presence_penalty"] = knob([0.0, 0.5, 0.3])
        args["frequency_penalty"] = knob([0.1, 0.2, 0.0])
    if case["bias"]:
        k = case["bias"]
        # distinct tokens of every row; some requests have fewer
        step = torch.randint(1, V // k + 1, (rows, 1), generator=g, device=DEV)
        start = torch.randint(0, V, (rows, 1), generator=g, device=DEV)
        ids = (start + step * torch.arange(k, device=DEV)) % V
        few = torch.randint(0, k + 1, (rows, 1), generator=g, device=DEV)
        args["bias_ids"] = torch.where(torch.arange(k, device=DEV) < few, ids, -1)
        args["bias"] = 4.0 * torch.randn(rows, k, generator=g, device=DEV)
    if case["masks"]:
        # a grammar's states: most allow a few tokens, some all but a few; requests without one have no mask
        n = max(1, int(round(rows * case["masks"])))
        W = (V + 31) // 32
        words = torch.zeros(n, W, dtype=torch.int32, device=DEV)
        share = torch.tensor([0.002, 0.02, 0.5, 0.99], device=DEV)[torch.arange(n, device=DEV) % 4]
        for bit in range(32):
            on = torch.rand(n, W, generator=g, device=DEV) < share[:, None]
            words |= on.int() * (1 << bit if bit < 31 else -(1 << 31))
        words[:, 0] |= 1
        args["token_mask"] = words
        where = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
        where[torch.randperm(rows, generator=g, device=DEV)[:n]] = torch.arange(n, dtype=torch.int32, device=DEV)
        args["mask_rows"] = where
        args["fill"] = FILL if case["inplace"] else -math.inf
    state["args"] = args
    state["logits"] = logits.requires_grad_(case["train"])
    if case["train"]:
        state["g"] = (torch.randn(rows, V, generator=g, device=DEV) / rows).to(_dtype(case))


def _prepare_head(case, g, state):
    rows, H, V = case["rows"], case["hidden"], case["vocab"]
    # hidden states with a few channels that stand out, as norms leave them
    gain = torch.exp(0.5 * torch.randn(H, generator=g, device=DEV))
    state["x"] = (torch.randn(rows, H, generator=g, device=DEV) * gain).bfloat16()
    w = torch.empty(V, H, dtype=torch.int8, device=DEV)
    scales = torch.empty(V, device=DEV)
    for s in range(0, V, 16384):
        e = min(V, s + 16384)
        part = (0.02 * torch.randn(e - s, H, generator=g, device=DEV)).bfloat16().float()
        top = part.abs().amax(1)
        w[s:e] = torch.round(127 * part / top[:, None]).to(torch.int8)
        scales[s:e] = top / 127
    state["w"], state["scales"] = w, scales
    if own:
        # the head in the package's layout, kept for as long as the weights are
        state["head"] = _calls().Int8Head.from_quantized(w, scales)


def _prepare_embed(case, g, state):
    n, H, V = case["tokens"], case["hidden"], case["vocab"]
    table = torch.empty(V, H, dtype=_dtype(case), device=DEV)
    for s in range(0, V, 16384):
        e = min(V, s + 16384)
        table[s:e] = 0.02 * torch.randn(e - s, H, generator=g, device=DEV)
    ids = _zipf_ids((n,), V, g)
    if case["padding"]:
        # the padding behind a batch's shorter sequences
        ids = ids.masked_fill(torch.rand(n, generator=g, device=DEV) < case["padding"], -1)
    state["ids"], state["table"] = ids, table.requires_grad_(case["train"])
    if case["train"]:
        state["g"] = (torch.randn(n, H, generator=g, device=DEV) / n).to(_dtype(case))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    state = {"case": case}
    {"process": _prepare_process, "head": _prepare_head, "embed": _prepare_embed}[case["kind"]](case, g, state)
    return state


# --------------------------------------------------------------------------------------- pass
def _allowed(token_mask, mask_rows, V):
    at = torch.arange(V, device=token_mask.device)
    bits = (token_mask[:, at // 32] >> (at % 32)) & 1
    return (bits[mask_rows.clamp_min(0).long()] != 0) | (mask_rows < 0)[:, None]


def _plain_process(case, logits, args, g):
    rows, V = logits.shape
    if case["inplace"]:
        return {"logits": logits.masked_fill_(~_allowed(args["token_mask"], args["mask_rows"], V), args["fill"])}
    x = logits.float()
    if case["bias"]:
        ids = args["bias_ids"]
        b = torch.zeros(rows, V + 1, device=x.device)
        b.scatter_(1, torch.where(ids >= 0, ids, V), args["bias"])
        x = x + b[:, :V]
    factor = None
    if case["history"]:
        h = args["history"]
        at = torch.arange(h.shape[1], device=x.device)[None, :]
        there = at < args["history_lens"][:, None]
        said = there & (at >= args["history_prompt_lens"][:, None]) if case["prompt"] else there
        count = torch.zeros(rows, V + 1, device=x.device)
        count.scatter_add_(1, torch.where(said, h, V), torch.ones_like(h, dtype=torch.float32))
        count = count[:, :V]
        seen = torch.zeros(rows, V + 1, dtype=torch.bool, device=x.device)
        seen = seen.scatter_(1, torch.where(there, h, V), True)[:, :V]
        rp = args["repetition_penalty"][:, None]
        if case["train"]:
            one = torch.ones_like(rp)
            factor = torch.where(seen, torch.where(x > 0, one / rp, rp), one)
        x = torch.where(seen, torch.where(x > 0, x / rp, x * rp), x)
        x = x - args["frequency_penalty"][:, None] * count
        x = torch.where(count > 0, x - args["presence_penalty"][:, None], x)
    allowed = None
    if case["masks"]:
        allowed = _allowed(args["token_mask"], args["mask_rows"], V)
        x = x.masked_fill(~allowed, args["fill"])
    out = {"logits": x.to(logits.dtype)}
    if case["train"]:
        grad = g.float()
        if factor is not None:
            grad = grad * factor
        if allowed is not None:
            grad = grad.masked_fill(~allowed, 0.0)
        out["grad"] = grad.to(logits.dtype)
    return out


def _plain_head(case, x, w, scales):
    x = x.float()
    top = x.abs().amax(1, keepdim=True)
    q = torch.round(127 * x / torch.where(top > 0, top, torch.ones_like(top)))
    return {"logits": ((q @ w.float().t()) * (top / 127) * scales).to(_dtype(case))}


def _plain_embed(case, ids, table, g):
    V = table.shape[0]
    there = (ids >= 0)[:, None]
    rows = table[ids.clamp_min(0)].float() * case["scale"]
    out = {"rows": torch.where(there, rows, torch.zeros_like(rows)).to(table.dtype)}
    if case["train"]:
        grad = torch.zeros(V + 1, table.shape[1], device=table.device)
        grad.index_add_(0, torch.where(ids >= 0, ids, V), g.float())
        out["grad"] = (grad[:V] * case["scale"]).to(table.dtype)
    return out


def _calls():
    if "dsv41_rocm" not in sys.modules:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "tiny-dsv41_amd"))
        import dsv41_rocm  # noqa: F401
    return sys.modules["dsv41_rocm"]


def _run_own(state):
    case, calls = state["case"], _calls()
    if case["kind"] == "process":
        # the sampler behind it looks at the rows, and a grammar at its own states: no check here
        y = calls.process_logits(state["logits"], **state["args"], out=state["logits"] if case["inplace"] else None,
                                 check=False)
        out = {"logits": y}
        if case["train"]:
            (out["grad"],) = torch.autograd.grad(y, (state["logits"],), (state["g"],))
        return out
    if case["kind"] == "head":
        if "head" not in state:
            state["head"] = calls.Int8Head.from_quantized(state["w"], state["scales"])
        return {"logits": calls.head_logits(state["x"], state["head"], dtype=_dtype(case), check=False)}
    # a learner checks its batch's ids, a decoding loop has them from the sampler
    rows = calls.token_embedding(state["ids"], state["table"], scale=case["scale"], check=case["train"])
    out = {"rows": rows}
    if case["train"]:
        (out["grad"],) = torch.autograd.grad(rows, (state["table"],), (state["g"],))
    return out


def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    with torch.no_grad():
        if case["kind"] == "process":
            return _plain_process(case, state["logits"], state["args"], state.get("g"))
        if case["kind"] == "head":
            return _plain_head(case, state["x"], state["w"], state["scales"])
        return _plain_embed(case, state["ids"], state["table"], state.get("g"))


# -------------------------------------------------------------------------- what a pass needs
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "process":
        rows, V = case["rows"], case["vocab"]
        masks = max(1, int(round(rows * case["masks"]))) if case["masks"] else 0
        moved = masks * ((V + 31) // 32) * 4 + (rows * 4 if masks else 0)
        if case["inplace"]:
            # what is masked is written: 0.622 of the tokens of a grammar's state, on average
            return {"bytes": moved + int(masks * V * size * 0.622), "flops": masks * V}
        moved += rows * V * size * (4 if case["train"] else 2)
        if case["history"]:
            moved += rows * (case["history"] * 6 + 20)  # three quarters of the entries, 8 bytes each
        moved += rows * case["bias"] * 12
        return {"bytes": moved, "flops": rows * V * (2 if case["train"] else 1)}
    if case["kind"] == "head":
        n, H, V = case["rows"], case["hidden"], case["vocab"]
        return {"bytes": V * H + 4 * V + n * H * 2 + n * V * size, "flops": 2 * n * H * V}
    n, H, V = case["tokens"], case["hidden"], case["vocab"]
    moved = n * 8 + 2 * n * H * size
    flops = n * H
    if case["train"]:
        moved += n * H * size + V * H * size
        flops += 2 * n * H
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------------ 64-bit results
def _exact_process(case, state):
    rows, V = case["rows"], case["vocab"]
    args, x = state["args"], state["logits"].detach()
    allowed = torch.ones(rows, V, dtype=torch.bool, device=x.device)
    if case["masks"]:
        shifts = torch.arange(32, device=x.device, dtype=torch.int64)
        states = ((args["token_mask"].long()[:, :, None] >> shifts) & 1).reshape(args["token_mask"].shape[0], -1)[:, :V]
        has = torch.nonzero(args["mask_rows"] >= 0)[:, 0]
        allowed[has] = states[args["mask_rows"][has].long()].bool()
    parts, grads = [], []
    for r in range(0, rows, 128):
        take = slice(r, min(rows, r + 128))
        y = x[take].double()
        n = y.shape[0]
        slope = torch.ones_like(y)
        if case["bias"]:
            row, col = torch.nonzero(args["bias_ids"][take] >= 0, as_tuple=True)
            y[row, args["bias_ids"][take][row, col]] += args["bias"][take][row, col].double()
        if case["history"]:
            at = torch.arange(case["history"], device=x.device)[None, :].expand(n, -1)
            row, col = torch.nonzero(at < args["history_lens"][take][:, None], as_tuple=True)
            token = args["history"][take][row, col]
            rp = args["repetition_penalty"][take].double()[:, None].expand_as(y)
            listed_ = torch.zeros_like(y).index_put_((row, token), torch.ones((), dtype=torch.float64, device=x.device))
            slope = torch.where(listed_ > 0, torch.where(y > 0, 1.0 / rp, rp), slope)
            y = y * slope
            if case["prompt"]:
                late = col >= args["history_prompt_lens"][take][row]
                row, token = row[late], token[late]
            count = torch.bincount(row * V + token, minlength=n * V).reshape(n, V)
            y -= args["frequency_penalty"][take].double()[:, None] * count
            y -= args["presence_penalty"][take].double()[:, None] * (count > 0)
        y[~allowed[take]] = args.get("fill", 0.0)
        parts.append(y)
        if case["train"]:
            grads.append(torch.where(allowed[take], state["g"][take].double() * slope, 0.0))
    out = {"logits": torch.cat(parts)}
    if case["train"]:
        out["grad"] = torch.cat(grads)
    return out


def _exact_head(case, state):
    x = state["x"].double()
    top = x.abs().max(1).values
    # a quotient of values of 15 and 8 bits is a half or at least 2^-9 away from one
    q = torch.round(x * 127 / torch.where(top > 0, top, 1.0)[:, None])
    out = torch.empty(case["rows"], case["vocab"], dtype=torch.float64, device=x.device)
    for s in range(0, case["vocab"], 16384):
        w = state["w"][s:s + 16384].double() * state["scales"][s:s + 16384].double()[:, None]
        out[:, s:s + 16384] = (q * (top / 127)[:, None]) @ w.t()
    return {"logits": out}


def _exact_embed(case, state):
    ids, table = state["ids"], state["table"].detach()
    rows = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=ids.device)
    at = torch.nonzero(ids >= 0)[:, 0]
    rows[at] = table[ids[at]].double() * case["scale"]
    out = {"rows": rows}
    if case["train"]:
        # every token's gradients summed by themselves, in the order of the batch
        order = at[torch.argsort(ids[at], stable=True)]
        names, lengths = torch.unique_consecutive(ids[order], return_counts=True)
        grad = torch.zeros(case["vocab"], case["hidden"], dtype=torch.float64, device=ids.device)
        if len(at):
            total = torch.cumsum(state["g"][order].double(), 0)
            last = torch.cumsum(lengths, 0) - 1
            ends = total[last]
            grad[names] = (ends - torch.cat([torch.zeros_like(ends[:1]), ends[:-1]])) * case["scale"]
        out["grad"] = grad
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"process": _exact_process, "head": _exact_head, "embed": _exact_embed}[case["kind"]](case, state)
