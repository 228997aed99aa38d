"""Timed cases of the operators over rows of logits: the scores of given tokens with entropy and top
alternatives, and distillation from a teacher's top tokens, each with its backward pass.

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
REST_FLOOR = 2.0 ** -20  # a teacher's rest mass below this is none


def _scores(rows, vocab, dtype, top_k, targets=True, masked=False, train=False, stride=None, temperature=1.0):
    return {"kind": "scores", "rows": rows, "vocab": vocab, "stride": stride or vocab, "dtype": dtype, "top_k": top_k,
            "targets": targets, "masked": masked, "train": train, "temperature": temperature}


def _distill(rows, vocab, dtype, top_k, tail, train=True, ragged=False, stride=None, temperature=1.0):
    return {"kind": "distill", "rows": rows, "vocab": vocab, "stride": stride or vocab, "dtype": dtype, "top_k": top_k,
            "tail": tail, "ragged": ragged, "train": train, "temperature": temperature}


def listed():
    return [
        # one decoded token's log-prob with the five alternatives that a serving API returns
        {"name": "decode_1_top5", **_scores(1, 129280, "f32", 5, temperature=0.7)},
        # a decode batch with twenty alternatives, logits a view of a head padded to a multiple of 128
        {"name": "decode_48_top20", **_scores(48, 151851, "bf16", 20, stride=151936)},
        # a few rows under grammar masks, some of which leave fewer tokens than alternatives
        {"name": "constrained_8_top20", **_scores(8, 129280, "f32", 20, masked=True, temperature=0.8)},
        # the log-probs, ranks and entropies of a prompt's own tokens
        {"name": "prompt_1000", **_scores(1000, 129280, "bf16", 0)},
        # wide lists of one response, kept as a teacher's record
        {"name": "teacher_300_top512", **_scores(300, 151936, "bf16", 512, targets=False)},
        # a teacher's pass over a microbatch, no targets
        {"name": "teacher_4096_top64", **_scores(4096, 151936, "f32", 64, targets=False)},
        # a policy's log-probs with an entropy bonus, from logits of an odd vocabulary, and their gradient
        {"name": "policy_1000_grad", **_scores(1000, 151851, "bf16", 0, train=True)},
        # the smallest training call: a few tokens of one response
        {"name": "distill_8_top16", **_distill(8, 129280, "f32", 16, "rest")},
        # one response against a teacher's lists, whose rest of the mass is a bucket of its own
        {"name": "distill_331_top64", **_distill(331, 129280, "bf16", 64, "rest")},
        # a padded batch against lists of ragged lengths, renormalized, fp32 logits of an odd vocabulary
        {"name": "distill_1000_top100", **_distill(1000, 151851, "f32", 100, "renormalize", ragged=True, temperature=2.0)},
        # a microbatch of the learner, the largest
        {"name": "distill_4096_top64", **_distill(4096, 151936, "bf16", 64, "rest", ragged=True)},
        # the divergence of a validation set, without gradients
        {"name": "distill_eval_512_top256", **_distill(512, 151936, "f32", 256, "rest", train=False)},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["scores", "scores", "distill", "distill"])
    dtype = rng.choice(["f32", "bf16"])
    vocab = rng.choice([129280, 151936, _log_int(rng, 8192, 151936), _log_int(rng, 8192, 151936)])
    train = rng.random() < (0.4 if kind == "scores" else 0.75)
    most = 4096 * 151936 * 4 // (vocab * (4 if dtype == "f32" else 2) * (2 if train else 1))
    rows = _log_int(rng, 1, min(4096, most))
    stride = (vocab + 127) // 128 * 128 if rng.random() < 0.5 else vocab
    temperature = rng.choice([1.0, 0.6, 2.0, round(rng.uniform(0.3, 3.0), 3)])
    if kind == "scores":
        top_k = rng.choice([0, 1, 5, 20, _log_int(rng, 1, 512)])
        return _scores(rows, vocab, dtype, top_k, targets=train or rng.random() < 0.7, masked=rng.random() < 0.2,
                       train=train, stride=stride, temperature=temperature)
    return _distill(rows, vocab, dtype, _log_int(rng, 1, 512), rng.choice(["renormalize", "rest"]), train=train,
                    ragged=rng.random() < 0.5, stride=stride, temperature=temperature)


# ------------------------------------------------------------------------------------- inputs
def _zipf_logits(case, g):
    """Next-token logits with a Zipf-like head, N(0, 1) - 1.1 log(rank), ranks in an order of each row's own."""
    V, rows = case["vocab"], case["rows"]
    order = torch.randperm(V, generator=g, device=DEV)
    shift = torch.randint(0, V, (rows,), generator=g, device=DEV)
    bias = -1.1 * torch.log((order + 1).float())
    ids = torch.arange(V, device=DEV)
    out = torch.zeros(rows, case["stride"], dtype=torch.float32, device=DEV)
    for r in range(0, rows, 512):
        e = min(rows, r + 512)
        out[r:e, :V] = torch.randn(e - r, V, generator=g, device=DEV) + bias[(ids[None, :] + shift[r:e, None]) % V]
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows, V, k = case["rows"], case["vocab"], case["top_k"]
    dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    full = _zipf_logits(case, g)
    state = {"case": case}
    if case["kind"] == "scores":
        if case["masked"]:
            # one row in four keeps a handful of tokens, the others the tokens of a random class
            keep = torch.rand(rows, V, generator=g, device=DEV) < 0.1
            few = torch.arange(rows, device=DEV) % 4 == 1
            keep[few] = torch.rand(int(few.sum()), V, generator=g, device=DEV) < 8.0 / V
            keep.scatter_(1, full[:, :V].argmax(1, keepdim=True), True)
            full[:, :V].masked_fill_(~keep, -math.inf)
        logits = full.to(dtype)[:, :V]
        if case["targets"]:
            # sampled tokens, so mostly likely ones
            noise = -torch.log(-torch.log(torch.rand(rows, V, generator=g, device=DEV)))
            state["targets"] = (full[:, :V] / case["temperature"] + noise).argmax(1)
        else:
            state["targets"] = None
        if case["train"]:
            state["g_lp"] = torch.randn(rows, generator=g, device=DEV) / rows
            state["g_entropy"] = torch.full((rows,), -0.01 / rows, device=DEV)
            state["g_top"] = torch.randn(rows, k, generator=g, device=DEV) / (rows * max(k, 1))
    else:
        teacher = (full[:, :V] + 0.7 * torch.randn(rows, V, generator=g, device=DEV)) / case["temperature"]
        top, ids = teacher.topk(k, dim=1)
        lq = top - teacher.logsumexp(1, keepdim=True)
        if case["ragged"]:
            # lists cut at a nucleus (-1: no entry), and rows of padding, which have none
            length = torch.randint(1, k + 1, (rows, 1), generator=g, device=DEV)
            length[torch.rand(rows, 1, generator=g, device=DEV) < 0.1] = 0
            gone = torch.arange(k, device=DEV)[None, :] >= length
            ids, lq = ids.masked_fill(gone, -1), lq.masked_fill(gone, 0.0)
        state["ids"], state["lq"] = ids.contiguous(), lq.contiguous()
        logits = full.to(dtype)[:, :V]
        state["g"] = torch.rand(rows, generator=g, device=DEV) / rows
    state["logits"] = logits.requires_grad_(case["train"])
    return state


# --------------------------------------------------------------------------------------- pass
def _plain_scores(case, x, targets, g_lp, g_entropy, g_top):
    T, k, V = case["temperature"], case["top_k"], case["vocab"]
    x32 = x.float()
    z = x32 / T
    d = z - z.amax(1, keepdim=True)
    e = torch.exp(d)
    S = e.sum(1, keepdim=True)
    lp = d - torch.log(S)
    p = e / S
    plogp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    entropy = -plogp.sum(1)
    out = {"entropy": entropy}
    at = torch.arange(V, device=x.device)
    if targets is not None:
        out["log_probs"] = lp.gather(1, targets[:, None])[:, 0]
        xt = x32.gather(1, targets[:, None])
        before = (x32 > xt) | ((x32 == xt) & (at[None, :] < targets[:, None]))
        out["ranks"] = 1 + before.sum(1)
    if k:
        bits = (x32 + 0.0).view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64) * (1 << 32) + (V - 1 - at)
        best = key.topk(k, dim=1).values
        ids = V - 1 - best % (1 << 32)
        top = lp.gather(1, ids)
        none = torch.isinf(top)
        out["top_ids"], out["top_log_probs"] = ids.masked_fill(none, -1), top
    if case["train"]:
        grad = -g_entropy[:, None] * (plogp + p * entropy[:, None]) - g_lp[:, None] * p
        grad.scatter_add_(1, targets[:, None], g_lp[:, None])
        if k:
            gk = g_top.masked_fill(none, 0.0)
            grad -= gk.sum(1, keepdim=True) * p
            grad.scatter_add_(1, ids, gk)
        out["grad"] = (grad / T).to(x.dtype)
    return out


def _plain_distill(case, x, ids, lq, g):
    T, V = case["temperature"], case["vocab"]
    valid = ids >= 0
    some = valid.any(1)
    at = ids.clamp_min(0)
    x32 = x.float()
    top = x32.amax(1, keepdim=True)
    # a divergence is what is left of sums that nearly cancel, so the listed tokens' terms are formed in 64
    # bits; the mass of the tokens outside the list is summed by itself
    d_at = (x32.gather(1, at).double() - top) / T
    named = torch.zeros(x.shape[0], V + 1, dtype=torch.bool, device=x.device)
    named.scatter_(1, torch.where(valid, ids, V), True)
    e = torch.exp((x32 - top) / T)
    S_rest = torch.where(named[:, :V], torch.zeros_like(e), e).sum(1, keepdim=True, dtype=torch.float64)
    e_at = torch.where(valid, torch.exp(d_at), torch.zeros_like(d_at))
    S = S_rest + e_at.sum(1, keepdim=True)
    lp = d_at - torch.log(S)
    lq = lq.double().masked_fill(~valid, -math.inf)
    if case["tail"] == "renormalize":
        lq = lq - torch.logsumexp(lq, 1, keepdim=True)
    q = torch.where(valid, torch.exp(lq), torch.zeros_like(lq))
    loss = torch.where(q > 0, q * (lq - lp), torch.zeros_like(q)).sum(1)
    total, others = torch.ones_like(S), torch.ones_like(S)
    if case["tail"] == "rest":
        mass = q.sum(1, keepdim=True)
        rest = 1 - mass
        rest = torch.where(rest < REST_FLOOR, torch.zeros_like(rest), rest)
        p_rest = S_rest / S
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - torch.log(p_rest)), torch.zeros_like(rest))[:, 0]
        total = mass + rest
        others = torch.where(p_rest > 0, total - rest / p_rest, total)
    out = {"loss": torch.where(some, loss, torch.zeros_like(loss)).float()}
    if case["train"]:
        weight = torch.where(some, g, torch.zeros_like(g))[:, None] / T
        grad = torch.cat([e * (others * weight / S).float(), torch.zeros_like(weight)], 1)
        grad.scatter_(1, torch.where(valid, ids, V), ((total * e_at / S - q) * weight).float())
        out["grad"] = grad[:, :V].to(x.dtype)
    return out


def _calls():
    if "dsv41_rocm" not in sys.modules:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "tiny-dsv41_amd"))
        import dsv41_rocm  # noqa: F401
    return sys.modules["dsv41_rocm"]


def _own_scores(case, state):
    logits = state["logits"]
    # logits that a token was sampled from were checked there; a learner and a teacher check here
    s = _calls().logit_scores(logits, state["targets"], top_k=case["top_k"], temperature=case["temperature"],
                              check=case["train"] or state["targets"] is None)
    out = {"entropy": s.entropy}
    outputs, grads = [s.entropy], [state.get("g_entropy")]
    if state["targets"] is not None:
        out["log_probs"], out["ranks"] = s.log_probs, s.ranks
        outputs.append(s.log_probs)
        grads.append(state.get("g_lp"))
    if case["top_k"]:
        out["top_ids"], out["top_log_probs"] = s.top_ids, s.top_log_probs
        outputs.append(s.top_log_probs)
        grads.append(state.get("g_top"))
    if case["train"]:
        (out["grad"],) = torch.autograd.grad(outputs, (logits,), grads)
    return out


def _own_distill(case, state):
    loss = _calls().distillation_loss(state["logits"], state["ids"], state["lq"], temperature=case["temperature"],
                                      tail=case["tail"])
    out = {"loss": loss}
    if case["train"]:
        (out["grad"],) = torch.autograd.grad(loss, (state["logits"],), state["g"])
    return out


def run(state):
    case = state["case"]
    if own:
        return _own_scores(case, state) if case["kind"] == "scores" else _own_distill(case, state)
    with torch.no_grad():
        if case["kind"] == "scores":
            return _plain_scores(case, state["logits"], state["targets"], state.get("g_lp"), state.get("g_entropy"),
                                 state.get("g_top"))
        return _plain_distill(case, state["logits"], state["ids"], state["lq"], state["g"])


# -------------------------------------------------------------------------- what a pass needs
def work(case):
    rows, V, k = case["rows"], case["vocab"], case["top_k"]
    size = 4 if case["dtype"] == "f32" else 2
    moved = rows * V * size * (2 if case["train"] else 1)
    if case["kind"] == "scores":
        moved += rows * (4 + 12 * k) + (rows * (8 + 4 + 8) if case["targets"] else 0)
        moved += rows * (8 + 4 * k) if case["train"] else 0
        flops = 6  # difference, scale, exponential, two sums, comparison
    else:
        moved += rows * (12 * k + 4) + (rows * 4 if case["train"] else 0)
        flops = 4
    return {"bytes": moved, "flops": rows * V * (flops + (5 if case["train"] else 0))}


# ------------------------------------------------------------------------------ 64-bit results
def exact(case, seed):
    state = prepare(case, seed)
    T, V, k = case["temperature"], case["vocab"], case["top_k"]
    parts = []
    for r in range(0, case["rows"], 256):
        take = slice(r, min(case["rows"], r + 256))
        x = state["logits"].detach()[take].double()
        logp = torch.log_softmax(x / T, 1)
        p = logp.exp()
        part = {}
        if case["kind"] == "scores":
            h = torch.special.entr(p).sum(1)
            part["entropy"] = h
            if state["targets"] is not None:
                t = state["targets"][take][:, None]
                part["log_probs"] = logp.gather(1, t)[:, 0]
            if k:
                part["top_log_probs"], where = logp.topk(k, 1)
            if case["train"]:
                # the loss as a function of logp: sum_i c_i logp_i + g_entropy * H; d logp_i / dz_j = [i = j] - p_j
                c = torch.zeros_like(p).scatter_add_(1, t, state["g_lp"][take][:, None].double())
                if k:
                    # alternatives that tie are told apart by the lowest index
                    stable = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
                    gk = state["g_top"][take].double().masked_fill(part["top_log_probs"] == -math.inf, 0.0)
                    c.scatter_add_(1, stable, gk)
                grad = c - c.sum(1, keepdim=True) * p
                grad += state["g_entropy"][take][:, None].double() * (torch.special.entr(p) - p * h[:, None])
                part["grad"] = grad / T
        else:
            ids, lq = state["ids"][take], state["lq"][take].double()
            # the teacher as a row of its own over the vocabulary: q where it names a token, 0 elsewhere
            there = ids >= 0
            q = torch.zeros(x.shape[0], V + 1, dtype=torch.float64, device=x.device)
            q.scatter_(1, torch.where(there, ids, V), torch.where(there, lq.exp(), 0.0))
            named = torch.zeros_like(q).scatter_(1, torch.where(there, ids, V), 1.0)[:, :V]
            q = q[:, :V]
            empty = ~there.any(1)
            if case["tail"] == "renormalize":
                q = q / q.sum(1, keepdim=True)
                q[empty] = 0.0
                loss = (-torch.special.entr(q) - torch.special.xlogy(q, 1.0) - q * logp).sum(1)
                grad = p - q
            else:
                rest = 1 - q.sum(1)
                rest[rest < REST_FLOOR] = 0.0
                outside = p * (1 - named)
                p_rest = outside.sum(1)
                loss = (-torch.special.entr(q) - q * logp).sum(1) - torch.special.entr(rest)
                loss = loss - torch.special.xlogy(rest, p_rest)
                share = torch.where(p_rest > 0, rest / p_rest, torch.zeros_like(rest))
                grad = (q.sum(1) + rest)[:, None] * p - q - outside * share[:, None]
            loss[empty], grad[empty] = 0.0, 0.0
            part["loss"] = loss
            if case["train"]:
                part["grad"] = grad * state["g"][take][:, None].double() / T
        parts.append(part)
    out = {name: torch.cat([q[name] for q in parts]) for name in parts[0]}
    if case["kind"] == "scores":
        if state["targets"] is not None:
            out["ranks"] = None
        if k:
            out["top_ids"] = None
    return out
