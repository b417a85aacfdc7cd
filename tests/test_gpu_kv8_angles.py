"""Rotation on the way to the 8-bit cache at angles of any size."""
import numpy as np
import pytest
import torch

import _kv8 as ref
from test_gpu_kv8 import Pools, do_append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("most", [1.0, 2.0e4, 7.0e8])
def test_angles_past_32_bits_of_quarter_turns(llmk, dim, most):
    """inv_freq up to `most` at positions around 10^5: angles of up to 10^5, 2 10^9 (just below 2^31
    quarter turns) and 7 10^13, of either sign. Codes are those of the 64-bit value; q one rounding
    to fp16 of products in fp32 (cosine and sine 2^-22, two products and a sum)."""
    heads, n_kv, rows = 3, 2, 40
    rng = np.random.default_rng(dim)
    inv = (most * rng.uniform(-1, 1, dim // 2)).astype(np.float32)
    lens, starts = np.array([100000 + rows]), np.array([0, rows])
    tables = np.zeros((1, 6256), np.int32)
    tables[0, 6250:6253] = [2, 0, 1]
    pools = Pools(3, n_kv, dim)
    qkv = rng.standard_normal((rows, (heads + 2 * n_kv) * dim)).astype(np.float16)
    got = do_append(llmk, pools, qkv, tables, starts, lens, inv, (heads, n_kv, dim))
    want = ref.append(pools.k, pools.v, qkv, tables, starts, lens, inv, heads, n_kv, dim)
    x = np.abs(qkv[:, :heads * dim].astype(np.float64)).reshape(rows, heads, 2, dim // 2)
    size = np.repeat(x.sum(2)[:, :, None], 2, 2).reshape(want.shape)
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 2.0 ** -21 * size
    assert (np.abs(got.astype(np.float64) - want) <= tol).all()
    written = np.arange(48) < rows
    for side, c in enumerate((pools.k, pools.v)):
        assert np.array_equal(pools.scale(side), c.scale)
        a, b = (y[[2, 0, 1]].transpose(0, 2, 1, 3).reshape(48, -1)[written]
                for y in (pools.codes(side), c.codes))
        assert np.array_equal(a, b)
