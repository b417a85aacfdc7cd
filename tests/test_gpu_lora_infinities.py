"""Adapters whose weights hold infinities and NaN: the definition's infinities, with their signs, and its NaN, where
they belong and nowhere else."""
import numpy as np
import pytest

from test_gpu_lora import Case

pytestmark = pytest.mark.gpu


def check(llmk, c):
    y = c.upload(llmk)
    c.call(llmk, y, check_indices=True)
    got = y.cpu().numpy()[:, :c.ends[-1]].astype(np.float64)
    with np.errstate(all="ignore"):
        want, bound = c.want()
        want16 = want.astype(np.float16)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        inf = np.isinf(want)
        assert np.array_equal(got[inf], want[inf])
        fin = np.isfinite(want16) & ~inf
        assert (np.abs(got - want) <= bound)[fin].all()
    return inf.sum(), np.isnan(want).sum(), fin.sum()


@pytest.mark.parametrize("rank,inner,ends,rows", [
    (16, 256, (64, 128), 1), (8, 2048, (2048,), 3), (32, 512, (1024,), 20), (24, 64, (40, 96), 7),   # one launch
    (16, 16392, (48,), 1), (32, 8192, (520,), 40), (16, 1024, (8192, 16384), 700),                   # two
    (64, 256, (136,), 5), (48, 4104, (1000,), 33), (128, 512, (264,), 20), (72, 8192, (64, 128), 3),
    (256, 1024, (512,), 18), (136, 2048, (72, 328), 50)])
def test_infinities_of_b(llmk, rank, inner, ends, rows):
    """One in a column is the result's, two of opposite signs or a value of 0 against them are NaN."""
    rng = np.random.default_rng([rank, inner, rows])
    c = Case(rng, [0, 1, 0], [rows, rows, rows], 2, rank, inner, ends)
    out = ends[-1]
    c.b[0, 3, 5], c.b[0, 17, 0], c.b[0, out - 1, rank - 1] = np.inf, -np.inf, np.inf
    c.b[0, 30, 1], c.b[0, 30, 6] = np.inf, -np.inf
    c.b[1, 12, 2], c.b[1, 13, 7] = np.nan, -np.inf
    c.x[2 * rows, :inner] = 0  # every value between the products is 0
    inf, nan, fin = check(llmk, c)
    assert inf >= 3 * (2 * rows - 1) and nan > rows and fin > 0


@pytest.mark.parametrize("rank,inner,rows", [(16, 256, 1), (32, 512, 20), (64, 256, 5), (128, 512, 20), (256, 1024, 18)])
def test_infinities_of_a(llmk, rank, inner, rows):
    """A rank's value is infinite for every row: so are its part's columns, but those with a weight of 0 for it."""
    rng = np.random.default_rng([rank, inner, rows, 1])
    c = Case(rng, [0, 1, 0], [rows, rows, rows], 2, rank, inner, (64, 128))
    c.a[0, 1, 4, 9] = -np.inf
    c.b[0, 70, 4], c.b[0, 90, 4] = 0, np.inf
    inf, nan, fin = check(llmk, c)
    assert inf >= 2 * rows * 60 and nan >= 2 * rows and fin >= 2 * rows * 64
