"""The scratch words of the routing plan of many picks as a model: histograms, a flag for an id out of range, the running counts that take the histograms' place. One scratch
serves calls of any size, so whatever a longer call leaves must not be a later call's flag. The places are those that the source states."""
import os
import re

import numpy as np
import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cudapp_b200", "csrc", "moe_route.cu")


def places():
    """flag(chunks, experts) and the first histogram's word, as the kernels have them"""
    with open(SOURCE) as f:
        text = f.read()
    names = {k: int(v) for k, v in re.findall(r"(PLAN_\w+) = (\d+)", text)}
    flag = re.sub(r"\(size_t\)", "", re.search(r"atomicOr\(scratch \+ ([^,]+), 1u\)", text).group(1))
    hist = re.search(r"scratch\[(?:(\w+) \+ )?\(size_t\)blockIdx\.x \* experts \+ e\] = smem\[e\]", text).group(1)
    return lambda chunks, experts: eval(flag, {}, dict(names, chunks=chunks, experts=experts)), names[hist] if hist else 0


def plan(scratch, ids, experts, flag, hist):
    """-> (refused, the running counts) of one call"""
    chunks = (len(ids) + 1023) // 1024
    at = flag(chunks, experts)
    for c in range(chunks):
        part = ids[c * 1024:(c + 1) * 1024]
        if (part >= experts).any():
            scratch[at] |= 1
        scratch[hist + c * experts:hist + (c + 1) * experts] = np.bincount(part[part < experts], minlength=experts)
    refused = scratch[at] != 0
    scratch[at] = 0
    run = np.zeros(experts, np.int64)
    for c in range(chunks):
        mine = scratch[hist + c * experts:hist + (c + 1) * experts].copy()
        scratch[hist + c * experts:hist + (c + 1) * experts] = run
        run += mine
    return bool(refused), run


@pytest.mark.parametrize("sizes", [(4096, 1500, 2048, 600, 513, 4096), (4096, 600, 1024), (512, 4096, 512, 4095, 514), (3000, 4096, 3000, 3000, 4096)])
@pytest.mark.parametrize("experts", [1, 8, 128, 257])
def test_a_plan_does_not_depend_on_the_calls_before_it(sizes, experts):
    flag, hist = places()
    rng = np.random.default_rng(experts)
    most = (max(sizes) * 8 + 1023) // 1024
    scratch = np.zeros(most * experts + 1, np.int64)                       # what the layers allocate
    for i, tokens in enumerate(sizes):
        ids = rng.integers(0, experts, tokens * 8)
        chunks = (len(ids) + 1023) // 1024
        assert flag(chunks, experts) < len(scratch) and hist + chunks * experts <= len(scratch)
        refused, counts = plan(scratch, ids, experts, flag, hist)
        assert not refused, "the call of %d tokens is refused after %s" % (tokens, sizes[:i])
        assert np.array_equal(counts, np.bincount(ids, minlength=experts))
        bad = ids.copy(); bad[rng.integers(len(bad))] = experts
        assert plan(scratch, bad, experts, flag, hist)[0]


def test_a_flag_behind_the_calls_own_histograms_is_caught():
    scratch, rng = np.zeros(32 * 128 + 1, np.int64), np.random.default_rng(0)
    seen = [plan(scratch, rng.integers(0, 128, tokens * 8), 128, lambda chunks, experts: chunks * experts, 0)[0] for tokens in (4096, 1500)]
    assert seen == [False, True]
