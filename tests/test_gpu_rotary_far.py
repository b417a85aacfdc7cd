"""Rotations of rows, and into pages, whose bytes lie past 2^32 and whose elements past 2^31."""
import numpy as np
import pytest
import torch

import _unlike as ref
from test_gpu_rotary import tables, to

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 32), (80, 20)])
def test_far_rows(llmk, pairs, dim, rotary):
    rng = np.random.default_rng([dim, rotary])
    n, ld, heads, kv = 40000, 65536, 3, 2
    inv, _, _ = tables(rng, n, rotary, 1)
    pos = rng.integers(0, 5000, n)
    width, last = (heads + kv) * dim, 3
    x = torch.zeros(n, ld, dtype=torch.float16, device=DEV)
    rows = rng.standard_normal((last, width)).astype(np.float16)
    x[-last:, -width:] = to(rows, np.float16)
    llmk.rotary_apply(x[:, -width:], ld, x[:, ld - kv * dim:], ld, to(pos, np.int32), to(inv, np.float32), None, None, n,
                      heads, kv, dim, rotary, int(pairs))
    want, bound = ref.rotate(rows.reshape(last, -1, dim), pos[-last:], inv, None, None, rotary, pairs)
    got = x[-last:, -width:].cpu().numpy().reshape(want.shape).astype(np.float64)
    assert (np.abs(got - want) <= bound).all()
    x[-last:, -width:] = 0
    assert not x.any()


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dim,rotary", [(256, 128), (240, 60)])
def test_far_rows_into_far_pages(llmk, pairs, dim, rotary):
    rng = np.random.default_rng([dim, rotary])
    n, ld, heads, kv, page = 40000, 65536, 2, 8, 16
    num_pages, last = 70000, 3
    inv, _, _ = tables(rng, n, rotary, 1)
    pos = rng.integers(0, 2 * page, n)
    width = (heads + 2 * kv) * dim
    x = torch.zeros(n, ld, dtype=torch.float16, device=DEV)
    rows = rng.standard_normal((last, width)).astype(np.float16)
    x[-last:, -width:] = to(rows, np.float16)
    table = np.full((n, 2), -1)
    table[-last:] = num_pages - 1 - np.arange(2 * last).reshape(last, 2)
    kp = torch.zeros((num_pages, page, kv, dim), dtype=torch.float16, device=DEV)
    vp, q = torch.zeros_like(kp), torch.zeros((n, heads, dim), dtype=torch.float16, device=DEV)
    llmk.qkv_rotary_scatter(x[:, -width:], ld, q, kp, vp, to(table, np.int32), to(pos, np.int32), to(inv, np.float32), None,
                            None, n, 2, page, heads, kv, dim, rotary, int(pairs))
    y = rows.reshape(last, -1, dim)
    want, bound = ref.rotate(y[:, :heads + kv], pos[-last:], inv, None, None, rotary, pairs)
    bound[..., rotary:] = 0
    assert (np.abs(q[-last:].cpu().numpy().astype(np.float64) - want[:, :heads]) <= bound[:, :heads]).all()
    for r in range(last):
        at = int(table[n - last + r, pos[n - last + r] // page]), int(pos[n - last + r] % page)
        got = kp[at].cpu().numpy().astype(np.float64)
        assert (np.abs(got - want[r, heads:]) <= bound[r, heads:]).all()
        assert np.array_equal(vp[at].cpu().numpy().view(np.uint16), y[r, heads + kv:].view(np.uint16))
        kp[at], vp[at] = 0, 0
    assert not kp.any() and not vp.any() and not q[:-last].any()
