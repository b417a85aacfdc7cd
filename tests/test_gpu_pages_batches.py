"""Forks of large and of lopsided batches: thousands of children, one prompt's samples, caches of thousands of pages,
pages that run out."""
import numpy as np
import pytest
import torch

import _unlike as ref
from test_gpu_pages import check_fork

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_old,n_new", [(1200, 4096), (1200, 4097), (3000, 6000), (9000, 4500), (2, 12000)])
@pytest.mark.parametrize("spare", [0, 900, 30000])
def test_thousands_of_children(llmk, n_old, n_new, spare):
    """Past 4096 children the begins of their wanted pages are kept in the workspace."""
    rng = np.random.default_rng([n_old, n_new, spare])
    tables, lens, refs, num_pages = ref.batch(rng, n_old, 4, 90, 16, 7, spare=spare)
    parents = rng.integers(-1, n_old, n_new)
    reserve = rng.integers(0, 40, n_new) if spare != 900 else np.ones(n_new)
    want = check_fork(llmk, tables, lens, parents, reserve, refs, 16, num_pages)
    assert want[4][0] > 0 and (spare < 30000 or want[4][1] == 0)


@pytest.mark.parametrize("n,spare", [(4098, 0), (4098, 20000), (6000, 3000)])
def test_thousands_cut_inside_a_page_that_they_share(llmk, n, spare):
    rng = np.random.default_rng([n, spare])
    page, num_pages = 4, 3 * (n // 3) + spare
    order, tables, refs = rng.permutation(num_pages), np.full((n, 5), -1), np.zeros(num_pages, np.int64)
    for s in range(n):  # three share three pages, and are cut behind the first, in the second or in the third
        tables[s, :3] = order[3 * (s // 3):3 * (s // 3) + 3]
        refs[tables[s, :3]] += 1
    want = check_fork(llmk, tables, np.repeat(rng.integers(3, 12, n // 3), 3), rng.integers(0, n, n), np.full(n, 2), refs,
                      page, num_pages)
    pairs = want[3][want[3][:, 0] >= 0]
    assert not np.isin(pairs[:, 1], pairs[:, 0]).any() and (spare == 0 or len(pairs) > n // 4)


@pytest.mark.parametrize("samples", [1, 2, 8, 63, 64, 65, 256, 1000])
@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 1000, 8191])
def test_samples_of_one_prompt(llmk, samples, length):
    """All share the prompt's whole pages; the page that it ends inside is the first one's, the others copy it."""
    rng = np.random.default_rng([samples, length])
    num_pages, held = 512 + 2 * samples + 9, -(-length // 16)
    tables, refs = np.full((1, 520), -1), np.zeros(num_pages, np.int64)
    tables[0, :held] = rng.permutation(num_pages)[:held]
    refs[tables[0, :held]] = 1
    want = check_fork(llmk, tables, np.array([length]), np.zeros(samples), np.ones(samples), refs, 16, num_pages)
    assert want[4][1] == 0
    assert (want[3][:, 0] >= 0).sum() == (samples - 1 if length % 16 else 0)
    assert all(want[2][p] == samples for p in tables[0, :length // 16])


@pytest.mark.parametrize("free", [0, 1, 5, 40, 200])
@pytest.mark.parametrize("n", [12, 300])
def test_pages_run_out_in_a_large_cache(llmk, n, free):
    """16000 pages, most of which others hold; what is free goes to the first children, in order."""
    rng = np.random.default_rng([n, free])
    tables, lens, mine, pages = ref.batch(rng, n, 3, 300, 16, 21)
    num_pages, refs = 16000 + pages, np.ones(16000 + pages, np.int64)
    names = rng.permutation(num_pages)
    tables = np.where(tables >= 0, names[tables], -1)
    refs[names[:pages]] = mine
    refs[names[pages:pages + free]] = 0
    parents = np.sort(rng.integers(0, n, n + 40))
    want = check_fork(llmk, tables, lens, parents, np.full(n + 40, 200), refs, 16, num_pages)
    assert want[4][1] > 0 or free == 200


@pytest.mark.parametrize("bytes_of_a_page", [16, 20])
def test_many_pairs_in_many_pools(llmk, bytes_of_a_page):
    """Pairs and pools whose blocks are counted before the first launch, as one might not take its own."""
    n, num_pages, n_pools = 900000, 2000, 130
    pools = [torch.randint(-9, 9, (num_pages, bytes_of_a_page // 4), dtype=torch.int32, device="cuda") for _ in range(n_pools)]
    before = [p.clone() for p in pools]
    pairs = torch.full((n, 2), -1, dtype=torch.int32, device="cuda")
    for i, pair in ((0, (3, 7)), (n // 2, (1999, 0)), (n - 1, (5, 1200))):
        pairs[i] = torch.tensor(pair)
    llmk.kv_copy_pages(pools, pairs, None, n, num_pages)
    for p, b in zip(pools, before):
        b[7], b[0], b[1200] = b[3].clone(), b[1999].clone(), b[5].clone()
        assert torch.equal(p, b)
