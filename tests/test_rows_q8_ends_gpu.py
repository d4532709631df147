"""What calls over 8-bit kept rows hold to at the ends of their ranges: weights far below a row's largest, scales that are
no numbers, codes half-way between two, rows of a block in any order, several launches and several host threads."""
import numpy as np
import pytest
import torch

from tests import q8_model as M
from tests.test_rows_q8_gpu import attend_case, bf16, inv_freq, make, np64, paged
from tests.util import dev_u32

pytestmark = pytest.mark.gpu
FAR = 0xFFFFFFFF


@pytest.mark.parametrize("width,heads", [(64, 16), (128, 16), (128, 3), (256, 8)])
@pytest.mark.parametrize("weight", [20.5, 5.5, 1.5])
def test_many_small_weights_beside_one_large_one_that_adds_nothing(width, heads, weight):
    """The first key has nearly all of the weight and the value zero; the others, `weight` * 2^-24 of it each, make up the
    output.  Rows enough that one worker takes a whole row: a run of its own, where the others' weights stand beside the
    first one's.  Scores are 0 and one number; so what counts is the weights' rounding to f16: half a step, 2^-11, and
    2^-32 of the largest weight (2^7 in a run's own units) where that is subnormal, for each key; the sum's own error
    (8193 terms, 2^-24 each) is below 2^-11 as well.  bf16: half a step."""
    from tessera_b200 import ops
    rng = np.random.default_rng(30)
    n, rows = 8193, 1300
    kv, kept, _ = attend_case(rng, (heads, 1, width, 64, 64, "dense"), [n])
    kv.k.zero_()
    kv.k_scale.fill_(1.0)
    kv.v_scale.fill_(1.0)
    kv.k[0, 0, 0, 7] = 127
    kv.v.copy_(torch.from_numpy(rng.integers(40, 128, tuple(kv.v.shape)).astype(np.int8)))
    kv.v[0, 0, 0] = 0
    store = M.Store(kv, "dense", kept.scalar)
    q = torch.zeros((rows, heads, width), dtype=torch.bfloat16, device="cuda")
    q[:, :, 7] = 1.0
    scale = (24 - np.log2(weight)) * np.log(2.0) / 127
    at = dev_u32([0] * rows)
    # (positions that are not neighbours, so that every row is a tile)
    pos = [n - 1 if r % 2 == 0 else n - 5 for r in range(rows)]
    got = np64(ops.attend_rows_q8(q, kv, at, dev_u32(pos), kept, n, scale=scale))
    for r in (0, 1):
        want, a, top, keys = M.attend_keys(store, np64(q[0]), 0, 0, range(pos[r] + 1), np.float32(scale).astype(np.float64))
        largest = 1 / (1 + (keys - 1) * weight * 2.0 ** -24)
        tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -10 * a + keys * 2.0 ** -32 * largest * top
        off = np.abs(got[r::2] - want)
        assert np.all(off <= tol), (off / np.abs(want)).max()
