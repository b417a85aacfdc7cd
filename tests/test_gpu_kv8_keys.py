"""Keys of the 8-bit cache are those of the 64-bit definition, code for code, however they came in: prompts
that begin and end inside pages, rows over refused ones, single rows, tokens rounded again. And the sizes
of the attention's workspace."""
import numpy as np
import pytest

import _kv8 as ref
from test_gpu_kv8 import LAYOUTS, Pools, do_append, inv_freq, one_nan, rows_case, tables_for


def append_both(llmk, pools, qkv, tables, starts, lens, layout):
    """One append on both sides; every code and scale of both pools, a NaN's sign aside."""
    heads, n_kv, dim = layout
    inv = inv_freq(llmk, dim)
    do_append(llmk, pools, qkv, tables, starts, lens, inv, layout)
    ref.append(pools.k, pools.v, qkv, tables, starts, lens, inv, heads, n_kv, dim)
    for side, c in enumerate((pools.k, pools.v)):
        assert np.array_equal(pools.scale(side), c.scale, equal_nan=True)
        assert np.array_equal(one_nan(pools.codes(side)), one_nan(c.codes))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS)
def test_steps_of_a_serving_loop(llmk, layout):
    """Ragged prompts, further chunks from inside pages, then forty steps of one to six rows each of
    which the first few of the next step's take the places of up to five; sizes that swing over 10^4,
    so that scales grow over tokens held and new pages begin small."""
    heads, n_kv, dim = layout
    rng = np.random.default_rng(7 * heads + dim)
    n, widest = 6, 24
    tables, pages = tables_for(rng, np.full(n, widest))
    pools = Pools(pages, n_kv, dim)
    lens = np.zeros(n, int)
    for counts in ([37, 0, 16, 1, 90, 47], [30, 5, 33, 18, 1, 64]):
        lens = lens + counts
        starts = np.r_[0, np.cumsum(counts)]
        qkv = rows_case(rng, n_kv, heads, dim, int(starts[-1]) + 1, pad=8)
        append_both(llmk, pools, qkv, tables, starts, lens, layout)
    for turn in range(40):
        counts = rng.integers(1, 7, n)
        lens = np.maximum(lens - rng.integers(0, 6, n), 0) + counts
        starts = np.r_[0, np.cumsum(counts)]
        qkv = rows_case(rng, n_kv, heads, dim, int(starts[-1]), spread=1.5).astype(np.float64)
        qkv = np.clip(qkv * 10.0 ** rng.uniform(-2, 2), -60000, 60000).astype(np.float16)
        append_both(llmk, pools, qkv, tables, starts, lens, layout)
    assert lens.max() <= widest * ref.PAGE


@pytest.mark.gpu
@pytest.mark.parametrize("layout", [(32, 8, 64), (4, 2, 128)])
def test_single_rows_of_a_batch(llmk, layout):
    """row_starts None: 200 sequences at lengths of their own, 20 tokens each, growing and shrinking."""
    heads, n_kv, dim = layout
    rng = np.random.default_rng(dim)
    n = 200
    tables, pages = tables_for(rng, np.full(n, 4))
    pools = Pools(pages, n_kv, dim)
    for c in (pools.k, pools.v):  # tokens in front
        c.codes[:] = rng.integers(0, 127, c.codes.shape)
        c.scale[:] = 2.0 ** rng.integers(-12, -6, c.scale.shape)
    pools.upload()
    lens = rng.integers(0, 40, n)
    for size in np.r_[1.0, 10.0 ** rng.uniform(-3, 3, 19)]:
        lens = lens + 1
        qkv = (rows_case(rng, n_kv, heads, dim, n, 0.3) * size).astype(np.float16)
        append_both(llmk, pools, qkv, tables, None, lens, layout)


@pytest.mark.parametrize("dim", [64, 128])
def test_workspace_floats(llmk, dim):
    """131072 columns of partial results, each with a maximum and a sum, and notes of 8 words, two for
    each of 2048 workers."""
    assert llmk.kv8_attention_workspace_floats(dim) == 131072 * (dim + 2) + 2 * 2048 * 8
    assert llmk.kv8_attention_workspace_floats(dim + 1) == 0
