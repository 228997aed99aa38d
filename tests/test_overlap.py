"""Whether an `out` meets what a call reads: against the bytes that the two tensors really have."""

import random

import pytest
import torch

from dsv41_rocm.scores import overlap


def _bytes(t, base):
    at = torch.zeros(0, dtype=torch.int64)
    if t.numel():
        first = torch.zeros((), dtype=torch.int64)
        for n, step in zip(t.shape, t.stride()):
            first = first[..., None] + torch.arange(n) * step
        at = (first.reshape(-1, 1) * t.element_size() + torch.arange(t.element_size())).reshape(-1) + t.data_ptr() - base
    return set(at.tolist())


@pytest.mark.parametrize("seed", range(400))
def test_rows_as_far_apart(seed):
    r = random.Random(seed)
    step = r.randint(1, 12)
    buffer = torch.zeros(600)
    both = []
    for _ in range(2):
        rows, width, at = r.randint(0, 6), r.randint(1, step), r.randint(0, 80)
        both.append(buffer[at:].as_strided((rows, width), (step, 1), storage_offset=at))
    a, b = both
    want = bool(_bytes(a, buffer.data_ptr()) & _bytes(b, buffer.data_ptr()))
    assert overlap(a, b) == overlap(b, a) == want
    # the same memory as twice as many bf16 elements
    half = buffer.view(torch.bfloat16)[2 * b.storage_offset():].as_strided((b.shape[0], 2 * b.shape[1]), (2 * step, 1),
                                                                         storage_offset=2 * b.storage_offset())
    assert overlap(a, half) == overlap(half, a) == want


def test_other_strides_are_told_by_their_ends():
    x = torch.zeros(20, 30)
    assert overlap(x, x) and overlap(x[:, :10], x.view(-1)[15:16]) and overlap(x[:, ::2], x[:, 1::2])
    assert not overlap(x[:10], x[10:]) and not overlap(x[:, :10], x[:, 10:]) and not overlap(x[:0], x)
    assert not overlap(x, torch.zeros(20, 30)) and overlap(x[:1].expand(4, 30), x[:1])
    assert overlap(x[:, :10], x[:, 9:]) and overlap(x[:5, :10], x.view(-1)[29:149].view(4, 30)[:, :2])
