"""Adapters in every way that a call's sizes choose among (test_lora_plan.py checks that they do): what a block keeps from
one tile to the next, sums of many parts of in_features, adapters that change inside a block's run of tiles."""
import numpy as np
import pytest

from _lora_variants import SIZES, Sizes
from test_gpu_lora import Case, ids_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("at", range(len(SIZES)), ids=["-".join(map(str, s)) for s in SIZES])
def test_every_way(llmk, at):
    s = Sizes(at)
    ids = ids_of(s.rng, s.n, s.adapters, 0.1 if s.n > 3 else 0.0)
    ranks = None if at % 3 == 0 else s.rng.integers(1, s.rank + 1, s.adapters)
    c = Case(s.rng, ids, s.rows, s.adapters, s.rank, s.inner, s.ends, ranks=ranks, scales=at % 4 > 0)
    assert c.n_rows == s.n_rows
    c.check(llmk)


@pytest.mark.parametrize("at", [i for i, s in enumerate(SIZES) if s[0] * s[1] > 100 and s[3] <= 64])
def test_every_way_of_one_adapter_in_turn(llmk, at):
    """Tiles of adapters of unlike ranks side by side, of which some are 0: sums are exact."""
    s = Sizes(at)
    if s.rows is None:
        s.rows = np.ones(s.n, np.int64)
    ids = np.arange(s.n) % s.adapters
    ranks = s.rng.permutation(np.arange(s.adapters) * (s.rank + 1) // s.adapters)
    c = Case(s.rng, ids, s.rows, s.adapters, s.rank, min(s.inner, 2056), s.ends, ranks=ranks, whole=True)
    h = 32 * min(s.inner, 2056)
    c.b[np.abs(c.b) > 1] = 1  # sums of at most 64 values of 2^16.01 by 1, below 2^24 with y
    assert h * s.rank + 2000 < 2 ** 24 and h < 2 ** 21
    c.check(llmk, exact=True)
