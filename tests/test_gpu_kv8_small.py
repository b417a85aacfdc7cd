"""Attention over the 8-bit cache where fp16 has only subnormals: keys under the least scale, and queries."""
import numpy as np
import pytest

from test_gpu_kv8 import attention_case, check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", [(8, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("counts", [[1, 3, 2], [20, 30, 9], [20, 300, 9]])
def test_subnormal_keys_and_queries(llmk, layout, counts):
    """Keys of at most 2^-15 under queries of up to 60000, then queries of at most 2^-15 over keys of up to
    57344: scores of some units, all of which are lost where subnormals count as zero."""
    q, pools, tables, starts, lens = attention_case(91, layout, [50, 420, 77], counts)
    rng = np.random.default_rng(92)
    pools.k.codes[:] = rng.integers(0, 0x39, pools.k.codes.shape) | (
        rng.integers(0, 2, pools.k.codes.shape) << 7)  # -1 .. 1
    pools.k.scale[:] = 2.0 ** -15
    pools.upload()
    q[:] = rng.uniform(-60000, 60000, q.shape)
    got = check_attention(llmk, q, pools, tables, starts, lens)
    q[:] = 0
    even = check_attention(llmk, q, pools, tables, starts, lens)
    assert np.abs(got - even).max() > 2.0 ** -8 * np.abs(even).max()
    pools.k.codes[:] = (rng.integers(0x60, 0x7F, pools.k.codes.shape)  # 32 .. 448
                        | (rng.integers(0, 2, pools.k.codes.shape) << 7))
    pools.k.scale[:] = 2.0 ** 7
    pools.upload()
    q[:] = rng.integers(-512, 513, q.shape) * 2.0 ** -24
    got = check_attention(llmk, q, pools, tables, starts, lens)
    assert np.abs(got - even).max() > 2.0 ** -8 * np.abs(even).max()
