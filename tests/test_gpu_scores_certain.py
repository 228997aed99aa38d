"""logit_scores of a token far above all the others, whose log-prob is what a sum has beside its 1.

Tolerance.  In a slice of n elements the thread that holds the token adds n / 512 terms to two fp32 sums, one of
which holds the 1: n / 1024 additions, and up to 4 more in whole chunks, half a step of 2^-23 each.  The other
terms, in sums of their own size, are off relative to themselves by their exponents' roundings (three of
2^-24 |d|, |d| = 26 powers of two), an exponential's and n / 1024 additions; the result is rounded once."""

import math

import pytest
import torch

from dsv41_rocm import logit_scores

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
H = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,n", [(600, 151936, 151936), (1100, 5001, 5001), (1, 151936, 151936 // 4), (40, 129280, 129280 // 2)])
def test_log_prob_of_a_likely_token(rows, V, n, dtype):
    print(f"case: logit_scores {rows} x {V} {dtype}", flush=True)
    x = torch.full((rows, V), -18.0, dtype=dtype, device=DEV)
    # met first, last and between, by the first and the last threads
    at = torch.tensor([0, V - 1, V // 2, 7, 4095, 4096, V - 9, 511 * 8], device=DEV)
    t = at[torch.arange(rows, device=DEV) % len(at)] % V
    x.scatter_(1, t[:, None], 0.0)
    s = logit_scores(x, t, top_k=1)
    rest = (V - 1) * math.exp(-18.0)
    want = -math.log1p(rest)
    tol = (n / 1024 + 4) * H + rest * H * (3 * 26 + 4 + n / 1024) - want * H
    off = float((s.log_probs.double() - want).abs().max())
    assert off <= tol, (off, tol)
    # relative to the log-prob: 4e-3 in the longest row, 0.02 beside a rest of 8e-5
    assert off / -want <= (4e-3 if V > 100000 else 0.02)
    assert torch.equal(s.top_log_probs[:, 0], s.log_probs) and bool((s.ranks == 1).all())
    entropy = math.log1p(rest) + 18.0 * rest / (1 + rest)
    assert float((s.entropy.double() - entropy).abs().max()) <= tol + 18.0 * rest * H * (3 * 26 + 8 + n / 1024) + entropy * H
