"""Attention over contexts that one worker walks from end to end: the sums of weights that grow to
10^5 terms. Scores and weights are such that the result is known without a sum over positions."""
import numpy as np
import pytest
import torch

import _kv8 as ref
from test_gpu_kv8 import DEV, PAGE, dev, i32

pytestmark = pytest.mark.gpu

LOW = 128  # positions in front, all a worker's first step: the maximum that weights stay relative to


def flat_cache(dim, positions, rows):
    """One sequence, one kv head. The first LOW positions score 0, the others q[0] / sqrt(dim); V is 0
    but for one page, well behind LOW, that every row sees, whose rows are all the same."""
    pages = (positions + PAGE - 1) // PAGE
    k, v = ref.Cache(pages, 1, dim, 0, 1.0), ref.Cache(pages, 1, dim, 0, 1.0)
    k.codes[LOW // PAGE:, :, :, 0] = 0x38  # 1
    some = (positions - rows) // PAGE - 1
    v.codes[some] = 0x70 + np.arange(dim) % 15  # 128 .. 448, as 15 significands and exponents
    v.scale[some] = 2.0 ** 7
    tables = np.arange(pages, dtype=np.int32)[None]
    return [dev(x) if x.dtype != np.uint8 else dev(x).view(torch.float8_e4m3fn)
            for x in (k.codes, k.scale, v.codes, v.scale)], i32(tables), v.rows(tables[0], np.array(
                [some * PAGE]))[0, 0]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows,max_rows", [(1, 1), (6, 6), (40, 40), (40, 2000)])
@pytest.mark.parametrize("positions", [65536 + 5, 131072 + 9])
def test_sums_of_many_equal_weights(llmk, dim, rows, max_rows, positions):
    """No workspace: a sequence stays whole. All but the first positions weigh the same, up to 2^7.9
    of the reference maximum (below the 2^8 at which it gives way), and 16 of them have values.

    Off by: a weight, its two parts 2^-15 (their first 8 bits cut off, the rest rounded to 8); the
    weights' common error leaves the quotient but for the LOW positions' share of less than 2^-9,
    exponents of up to 8 off by 2^-20 and the exponential by 2^-22: less than 2^-27; the sum of
    the weights and the quotient 2^-20; one rounding, half a step of fp16."""
    heads = 4
    # q[0] / sqrt(dim) in log2 units; equal terms of these sizes leave remainders that add up where
    # each is added by itself
    sizes = np.array([7.902, 7.727, 6.988, 7.8])
    q = np.zeros((rows, heads, dim), np.float16)
    q[:, :, 0] = sizes * np.log(2.0) * np.sqrt(dim)
    pools, tables, value = flat_cache(dim, positions, rows)
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device=DEV)
    llmk.kv8_attention(dev(q), *pools, tables, i32([0, rows]), i32([positions]), out, None, rows, 1,
                       max_rows, tables.shape[1], PAGE, heads, 1, dim)
    torch.cuda.synchronize()
    got = out.cpu().numpy().astype(np.float64)
    weight = np.exp(q[:, :, 0].astype(np.float64) / np.sqrt(dim))
    seen = positions - rows + 1 + np.arange(rows)[:, None]
    share = PAGE * weight / (LOW + (seen - LOW) * weight)
    want = share[:, :, None] * value
    half_step = np.spacing(np.abs(want).astype(np.float16)).astype(np.float64) / 2
    off = np.abs(got - want) - half_step
    tol = (2.0 ** -15 + 2.0 ** -20 + 2.0 ** -27) * np.abs(want)
    assert (off <= tol).all(), (np.log2((off / np.abs(want)).max()), (off > tol).mean())
