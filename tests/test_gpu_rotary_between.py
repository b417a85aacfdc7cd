"""q and k whose heads lie between one another's: what turns of one is what the other leaves."""
import numpy as np
import pytest
import torch

import _unlike as ref
from test_gpu_rotary import positions, tables, to

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dim,rotary,n", [(64, 32, 9), (128, 48, 40), (20, 6, 5)])
def test_heads_between_heads(llmk, pairs, dim, rotary, n):
    rng = np.random.default_rng([dim, n])
    inv, t, s = tables(rng, n, rotary, 2)
    pos, heads, ld, second = positions(rng, n), 3, 4 * dim + 8, dim // 2
    x = rng.standard_normal((n, ld)).astype(np.float16)
    d = to(x, np.float16)
    llmk.rotary_apply(d, ld, d[:, second:], ld, to(pos, np.int32), to(inv, np.float32), to(t, np.int32),
                      to(s, np.float32), n, heads, heads, dim, rotary, int(pairs))
    got, left = d.cpu().numpy().astype(np.float64), np.ones((n, ld), bool)
    for at in (0, second):
        cols = at + np.arange(heads)[:, None] * dim + np.arange(rotary)
        want, bound = ref.rotate(x[:, cols], pos, inv, t, s, rotary, pairs)
        assert (np.abs(got[:, cols] - want) <= bound).all()
        left[:, cols.reshape(-1)] = False
    assert np.array_equal(d.cpu().numpy().view(np.uint16)[left], x.view(np.uint16)[left])
    with pytest.raises(llmk.LlmkError):
        llmk.rotary_apply(d, ld, d[:, rotary - 1:], ld, to(pos, np.int32), to(inv, np.float32), None, None, n, heads, heads,
                          dim, rotary, int(pairs))
    torch.cuda.synchronize()
