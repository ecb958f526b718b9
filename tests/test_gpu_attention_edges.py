"""The attention operators where buffers, scales and sizes meet their edges, against 64-bit restatements (attention_ref.py). Tolerances are those of
test_gpu_attention.py, derived there."""
import numpy as np
import pytest

import attention_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention import U16, U32, Step, check_turned, dev, error_word, make_cache  # noqa: E402
from tokspur_public_b200 import attention as A  # noqa: E402
from tokspur_public_b200 import capi  # noqa: E402


@pytest.mark.parametrize("type_,dim,group,dtype", [("q8_0", 128, 4, "f16"), ("q8_0", 128, 4, "f32"), ("f16", 256, 8, "f32"), ("f16", 64, 8, "f16"), ("q8_0", 128, 32, "f16")])
def test_many_refills_give_the_same_bits(type_, dim, group, dtype):
    """Rings that go round dozens of times in every warp, 200 calls: a stage that is refilled under its reader shows as another result."""
    s = Step(41, type_, dim, 64, 4, group, [2, 1], [9000, 7000], dtype, False)
    cache, scratch, err, q = make_cache(s.p), A.tree_attention_scratch(), error_word(), dev(s.q)
    want, code = s.run(cache, scratch)
    assert code == 0
    s.check(want)
    outs = [torch.empty_like(want) for _ in range(20)]
    differing = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(10):
        for out in outs:
            A.tree_attention(cache, s.batch, q, out, None, s.most, s.scale, scratch, err)
        for out in outs:
            differing += (out != want).sum()
    assert int(differing) == 0 and int(err) == 0
