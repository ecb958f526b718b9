"""CPU checks of the attention operators: what their sources and their Python objects have to keep, whatever a GPU does with it."""
import os
import re

import pytest

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


def test_norm_shuffles_are_reached_by_whole_warps():
    """turn_rows: eight dims a lane, so that a warp holds 32 / (dim / 8) heads and may hold the last query heads beside the first key heads, of which one side may have
    no norm. The sum of squares goes round the whole warp, so the warp decides as a whole whether it is formed."""
    for dim in (64, 128):
        lanes = dim // 8
        mixed = [(hq, hk) for hq in range(1, 9) for hk in range(1, 9) if any(len({h >= hq for h in range(w, min(w + 32 // lanes, hq + hk))}) == 2
                                                                            for w in range(0, hq + hk, 32 // lanes))]
        assert (7, 2) in mixed                              # such calls exist
    body = re.search(r"__device__ __forceinline__ void turn_rows\(.*?\n\}\n", source("tsp_kv.cu"), re.S).group(0)
    before = body[:body.index("__shfl_xor_sync")]
    branch = re.findall(r"if \((\w+)\) \{", before)[-1]
    declared = re.search(r"const bool %s = ([^;]*);" % branch, body)
    assert declared and declared.group(1).startswith("__any_sync(0xffffffffu, "), branch      # one answer for the warp


def test_the_check_answers_what_the_call_would():
    """tsp_tree_attention_check, without a device: refusals of arguments come before anything that needs one."""
    import ctypes as C
    from test_attention_host import Call
    from tokspur_public_b200 import capi

    def check(c):
        return capi.lib().tsp_tree_attention_check(C.byref(c.cache), C.byref(c.batch), c.q, c.qs, c.mask, c.q_heads, c.max_rows, c.scale, c.out, c.os, c.dtype, c.scratch,
                                                   c.scratch_bytes)
    for change in (dict(q_heads=33), dict(max_rows=0), dict(max_rows=65), dict(scale=float("inf")), dict(mask=(1 << 26) + 4), dict(scratch=(6 << 40) + 8), dict(scratch_bytes=0),
                   dict(out=1 << 40), dict(out=1 << 32), dict(out=(4 << 40) + 4), dict(scratch=1 << 40), dict(scratch=4 << 40), dict(scratch=1 << 32), dict(os=16368), dict(q=None)):
        c = Call()
        vars(c).update(change)
        assert check(c) == capi.E_ARG == c.attend(), change


def test_wide_tiles_are_left_where_their_registers_do_not_fit(tmp_path):
    """The rule that chooses a kernel, compiled on its own: another register count of the wide kernel sends its calls to the narrow one, and refuses none."""
    import subprocess
    main = tmp_path / "rule.cpp"
    main.write_text('#include <initializer_list>\n#include "tsp_tree_rule.h"\n'
                    'using tsp::wide_tiles;\n'
                    'int main() {\n'
                    '    for (unsigned dim : {64u, 128u}) {\n'
                    '        if (!wide_tiles(dim, true, 49, 128) || wide_tiles(dim, true, 48, 128) || wide_tiles(dim, false, 4096, 128)) return 1;\n'
                    '        for (int regs : {96, 120, 126, 127, 129, 168}) if (wide_tiles(dim, true, 4096, regs)) return 2;\n'
                    '    }\n'
                    '    return wide_tiles(256, true, 4096, 128) ? 3 : 0;\n'
                    '}\n')
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, "-o", str(tmp_path / "rule"), str(main)], check=True)
    assert subprocess.run([str(tmp_path / "rule")]).returncode == 0
    calls = source("tsp_tree_attn.cu")
    assert re.search(r"tree_mma_registers\(p, registers\)\) return rc;\s*if \(wide_tiles\(D, f16, rows, registers\)\) return launch_tree_mma\(p, st\);", calls)
    assert "numRegs" not in re.search(r"static int launch_tree_mma_t\(.*?\n\}\n", source("tsp_tree_mma.cu"), re.S).group(0)     # nothing refused there


def objects(rows=3, heads=2, dim=64):
    """Cache, batch and rows in host memory: what is wrong with a tensor is said before anybody asks for a device."""
    import torch
    from tokspur_public_b200 import attention as A
    cache = A.KvCache(torch.zeros(4, A.page_bytes("q8_0", 16, heads, dim), dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.int32), 16, heads, dim, "q8_0")
    batch = A.KvBatch(torch.tensor([0, rows], dtype=torch.int32), torch.zeros(1, dtype=torch.int32), rows)
    return A, torch, cache, batch, torch.zeros(rows, heads, dim), torch.zeros(rows, dtype=torch.int32)


def test_a_workspace_or_error_word_without_memory_of_its_own_is_refused():
    """numel() of an expanded tensor says nothing of the memory behind it, and the library writes as much as it was told."""
    A, torch, cache, batch, x, _ = objects()
    size = 1 << 24
    for scratch in (torch.zeros(1, dtype=torch.uint8).expand(size), torch.zeros(2 * size, dtype=torch.uint8)[::2], torch.zeros(size, dtype=torch.float32)):
        with pytest.raises(ValueError, match="scratch"):
            A.tree_attention(cache, batch, x, x.clone(), None, 3, 1.0, scratch, None)
    for error in (torch.zeros(1, dtype=torch.uint8), torch.zeros(0, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="error word: one int32"):
            A.kv_cache_append(cache, batch, x, x, error)


def test_positions_and_rows_that_are_left_out():
    """What the C entry accepts (no positions where nothing is rotated) goes through to it, here as far as the missing device; what it does not is a ValueError."""
    A, torch, cache, batch, x, words = objects()
    still, turned = A.QkNormRope(64, 0, "halves", None), A.QkNormRope(64, 64, "halves", torch.ones(32))
    for call in (lambda: A.qk_norm_rope(still, x, None, None, x, None, None), lambda: A.qk_norm_rope_append(still, cache, batch, x, x, x, None, x, None)):
        with pytest.raises(ValueError, match="tensors in host memory"):
            call()
    for call in (lambda: A.qk_norm_rope(turned, x, None, None, x, None, None), lambda: A.qk_norm_rope_append(turned, cache, batch, x, x, x, None, x, None)):
        with pytest.raises(ValueError, match="positions: 3 dense values"):
            call()
    for rows in ((None, None, None, None), (x, None, None, None), (None, x, None, None), (x, x, x, None)):
        with pytest.raises(ValueError, match="rows of queries, keys or both"):
            A.qk_norm_rope(still, rows[0], rows[1], None, rows[2], rows[3], None)


def test_a_page_table_that_is_part_of_a_wider_one_is_refused():
    A, torch, cache, batch, x, _ = objects()
    wide = torch.zeros(2, 8, dtype=torch.int32)
    with pytest.raises(ValueError, match="not next to one another"):
        A.KvCache(cache.pages, wide[:, :4], 16, 2, 64, "q8_0")
    assert A.KvCache(cache.pages, wide[:1, :4], 16, 2, 64, "q8_0").struct.table_stride == 4      # one row of it has no next


def test_outputs_over_the_arrays_of_the_step_are_refused():
    """Blocks look sequences, pages and tree words up while others write: output rows, pages and workspaces lie apart from them."""
    from test_attention_host import Call
    from tokspur_public_b200 import capi
    row = 32 * 128 * 4                                 # bytes of a query row

    def place(entry, field, at):
        c = Call()
        target, _, name = field.partition("__")
        setattr(getattr(c, target) if name else c, name or target, at)
        return getattr(c, entry)()
    out, pages, scratch, kout = 4 << 40, 1 << 32, 6 << 40, 5 << 40
    step = ["batch__d_row_offsets", "batch__d_lengths", "cache__d_page_table"]
    turn = ["positions", "turn__d_q_norm", "turn__d_k_norm", "turn__d_inv_freq"]
    for entry, fields, written in (("norm", turn, [out, out + 31 * row, kout]), ("fused", turn + step, [out, out + 31 * row + 256, pages, pages + 15 * Call().cache.page_stride_bytes]),
                                   ("append", step, [pages]), ("read", step, [2 << 40, 3 << 40]), ("keep", step + ["accepted", "counts"], [pages + 64]),
                                   ("attend", step + ["mask"], [out, scratch, scratch + (1 << 30) - 16])):
        for field in fields:
            for at in written:
                assert place(entry, field, at) == capi.E_ARG, (entry, field, hex(at))
                assert "overlap" in capi.last_error()
    # an array between two rows, or behind the last, is nobody's (without a device the call ends there)
    import torch
    if not torch.cuda.is_available():
        c = Call()
        c.os, c.batch.d_lengths, c.mask = row + 512, out + row, out + 32 * (row + 512) - 512 + 8
        assert c.attend() == capi.E_CUDA, capi.last_error()
        c.batch.d_lengths = out + row + 500            # reaches into the second
        assert c.attend() == capi.E_ARG
