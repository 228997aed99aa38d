"""What ring_kernel's waits leave in flight (csrc/ring_rule.h): a wave's loads in the kernel's order, which come back in the
order they were issued, followed as far as the waits say."""

import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    """(stages in LDS, stage_wait, scales_wait)"""
    path = tmp_path_factory.mktemp("ring")
    src, exe = path / "rule.cpp", path / "rule"
    src.write_text('#include <stdio.h>\n#include <stdlib.h>\n#include "ring_rule.h"\nint main(int, char** a) {\n'
                   'printf("%d %d %d", dsv41::RING, dsv41::stage_wait(atoi(a[2])), dsv41::scales_wait(atoi(a[1]), atoi(a[2]))); }\n')
    subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "tiny-dsv41_amd" / "csrc"), "-o", str(exe), str(src)], check=True)

    def ask(stages, loads):
        out = subprocess.run([str(exe), str(stages), str(loads)], check=True, capture_output=True, text=True).stdout
        return tuple(int(v) for v in out.split())

    return ask


@pytest.mark.parametrize("stages", [1, 2, 3, 4, 7, 16])
@pytest.mark.parametrize("tokens,loads", [(64, 5), (128, 6)])
@pytest.mark.parametrize("stores", [0, 1, 64])
def test_what_is_read_has_come(rule, stages, tokens, loads, stores):
    ring, stage_wait, scales_wait = rule(stages, loads)
    queue = []  # what may be in flight, oldest first

    def wait(n):
        del queue[:max(0, len(queue) - n)]

    blocks, at = 4, 0
    for s in range(ring - 1):
        queue += [("stage", s)] * loads
    for b in range(blocks):
        for k in range(stages):
            wait(stage_wait)
            assert ("stage", at) not in queue
            if k == 0:
                queue.append(("scales", b))
            queue += [("stage", at + ring - 1)] * loads
            at += 1
        if scales_wait >= 0:
            wait(scales_wait)
        assert ("scales", b) not in queue, f"{tokens} tokens: scales are read ahead of their load"
        queue += [("store", b)] * stores  # of the block's logits, in the same count
