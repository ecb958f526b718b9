"""CPU checks of the attention operators: what their sources and their Python objects have to keep, whatever a GPU does with it."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tokspur-public_b200", "csrc")


def source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_refills_stand_behind_the_reads_of_what_they_overwrite():
    """A bulk copy writes shared memory through the asynchronous proxy. A warp barrier alone does not keep it behind loads whose values nobody has used, so
    every lane fences between its reads of a stage and the barrier in front of the copy (tree_attention_kernel, whose warps refill their own rings) or the
    arrival that lets another warp copy (the tile warps of tree_mma_kernel)."""
    assert "fence.proxy.async" in re.search(r"void fence_async_smem\(\) \{([^}]*)\}", source("tsp_tree_attn.cuh")).group(1)
    narrow = source("tsp_tree_attn.cu")
    refill = re.search(r"auto pass = \[&\]\(\) \{(.*?)\n\s*\};", narrow, re.S).group(1)
    assert re.search(r"fence_async_smem\(\);\s*__syncwarp\(\);.*issue\(stage\)", refill, re.S)
    assert narrow.count("issue(") == 2                      # the ring's first filling and the refill: no third way to a copy
    wide = source("tsp_tree_mma.cu")
    releases = [m.start() for m in re.finditer(r"mbar_arrive\(&sm\.code_empty\[st\]\)", wide)]
    assert len(releases) == 2                               # tiles of keys, tiles of values
    for at in releases:
        assert re.search(r"fence_async_smem\(\);\s*__syncwarp\(\);\s*if \(lane == 0\) \{[^}]*$", wide[:at]), wide[at - 200:at]
