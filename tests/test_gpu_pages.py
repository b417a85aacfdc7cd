"""Copies, forks and compaction of cache pages on the GPU against their definitions in plain loops."""
import numpy as np
import pytest
import torch

import _unlike as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def guarded(n):
    """n ints with 16 more behind that nobody may write."""
    return torch.full((n + 16,), -77, dtype=torch.int32, device=DEV)


def left(*tensors):
    for t in tensors:
        assert (t[-16:] == -77).all(), "write past the end"


# ---------------------------------------------------------------------------------------------
# copies
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("sizes", [(16384,), (16,), (4, 8, 12), (16384, 4100, 32, 16), (20,) * 70, (16400,) * 65,
                                   (4096, 4096), (1048576,)])
@pytest.mark.parametrize("n", [0, 1, 5, 40])
def test_copies(llmk, sizes, n):
    rng = np.random.default_rng([len(sizes), sizes[0], n])
    num_pages = 2 * n + 3
    pools = [torch.randint(-100, 100, (num_pages, b // 4), dtype=torch.int32, device=DEV) for b in sizes]
    before = [p.clone() for p in pools]
    order = rng.permutation(num_pages)
    pairs = np.stack([order[:n], order[n:2 * n]], 1).astype(np.int64)
    gone = np.zeros(n, bool)
    if n >= 5:  # pairs that copy nothing
        for i, bad in zip(range(5), ((-1, -1), (pairs[1, 0], num_pages), (-5, pairs[2, 1]), (3, 3),
                                     (2 ** 31 - 1, 0))):
            pairs[i], gone[i] = bad, True
    for count in (None, n, n - 2, 0, -3, n + 9):
        for p, b in zip(pools, before):
            p.copy_(b)
        llmk.kv_copy_pages(pools, i32(pairs.reshape(-1)) if n else i32([0, 0]), None if count is None else i32([count]),
                           n, num_pages, check_indices=True)
        m = n if count is None else max(0, min(n, count))
        on = np.flatnonzero(~gone[:m])
        src = torch.from_numpy(pairs[on, 0]).to(DEV)
        dst = torch.from_numpy(pairs[on, 1]).to(DEV)
        for p, b in zip(pools, before):
            want = b.clone()
            want[dst] = b[src]
            assert torch.equal(p, want)


@pytest.mark.parametrize("sizes", [(16384,), (32, 4100, 4096, 32, 16), (20,) * 3])
@pytest.mark.parametrize("n", [511, 512, 1300])
def test_many_copies(llmk, sizes, n):
    test_copies(llmk, sizes, n)


def test_copies_of_any_type_and_address(llmk):
    """Pools of other types, and one that begins between 16-byte addresses."""
    flat = torch.arange(4096, device=DEV, dtype=torch.int32)
    pools = [torch.randn(6, 2, 16, 64, device=DEV).to(torch.float8_e4m3fn), torch.randn(6, 2, device=DEV),
             torch.randn(6, 16, 1, 8, device=DEV).half(), flat[1:1 + 6 * 100].view(6, 100)]
    want = [p.clone() for p in pools]
    llmk.kv_copy_pages(pools, i32([[0, 3], [5, 1]]), None, 2, 6)
    for p, w in zip(pools, want):
        b = w.view(torch.uint8)
        b[3], b[1] = b[0].clone(), b[5].clone()
        assert torch.equal(p.view(torch.uint8), b)
    assert flat[0] == 0 and flat[601] == 601


def test_a_copy_past_32_bits(llmk):
    """Page numbers whose bytes lie past 2^32."""
    page, num_pages = 1 << 20, 4200
    pool = torch.zeros((num_pages, page // 4), dtype=torch.int32, device=DEV)
    pool[4150] = torch.arange(page // 4, device=DEV, dtype=torch.int32)
    pool[3] = 5
    llmk.kv_copy_pages([pool], i32([[4150, 7], [3, 4199]]), None, 2, num_pages)
    assert torch.equal(pool[7], pool[4150]) and (pool[4199] == 5).all()
    assert pool[[0, 8, 4198, 4149]].abs().sum() == 0


def test_copies_refused(llmk):
    pool, pairs = torch.zeros(8, 4, device=DEV), i32([[0, 1], [2, 3]])
    llmk.kv_copy_pages([pool], pairs, None, 2, 8, check_indices=True)
    for bad in (dict(pools=[pool[:7]]), dict(pools=[pool[:, ::2]]), dict(pools=[pool.cpu()]),
                dict(copies=pairs.long()), dict(n=3), dict(pages=0), dict(n=-1),
                dict(copies=i32([[0, 1], [2, 1]])), dict(copies=i32([[0, 1], [1, 3]])),
                dict(pools=[torch.zeros(8, 3, dtype=torch.int8, device=DEV)])):
        a = dict(pools=[pool], copies=pairs, count=None, n=2, pages=8) | bad
        with pytest.raises(llmk.LlmkError):
            llmk.kv_copy_pages(*a.values(), check_indices=True)


# ---------------------------------------------------------------------------------------------
# forks
# ---------------------------------------------------------------------------------------------
class Fork:
    def __init__(self, llmk, n_old, n_new, max_pages, page, num_pages):
        self.llmk, self.sizes = llmk, (n_old, n_new, max_pages, page, num_pages)
        self.new, self.lens = guarded(n_new * max_pages), guarded(n_new)
        self.copies, self.counts = guarded(2 * n_new), guarded(2)
        self.ws = guarded(llmk.kv_fork_workspace_ints(n_old, n_new, max_pages, num_pages))

    def __call__(self, tables, lens, parents, reserve, refs, check=False):
        self.llmk.kv_fork(tables, lens, parents, reserve, refs, self.new, self.lens, self.copies, self.counts,
                          self.ws, *self.sizes, check_indices=check)

    def results(self, refs):
        left(self.new, self.lens, self.copies, self.counts, self.ws)
        n_new, max_pages = self.sizes[1:3]
        return (self.new[:-16].view(n_new, max_pages), self.lens[:-16], refs, self.copies[:-16].view(n_new, 2),
                self.counts[:-16])


def check_fork(llmk, tables, lens, parents, reserve, refs, page, num_pages):
    n_old, max_pages = tables.shape
    n_new = len(parents)
    want = ref.fork(tables, lens, parents, reserve, refs, n_new, max_pages, page, num_pages)
    f, dev = Fork(llmk, n_old, n_new, max_pages, page, num_pages), i32(refs)
    f(i32(tables.reshape(-1)), i32(lens), i32(parents), i32(reserve), dev, check=True)
    for got, w, name in zip(f.results(dev), want, ("tables", "lens", "refs", "copies", "counts")):
        assert np.array_equal(got.cpu().numpy(), w), name
    return want


@pytest.mark.parametrize("seed", range(40))
def test_forks(llmk, seed):
    rng = np.random.default_rng(seed)
    page, max_pages = int(rng.choice([1, 3, 16, 64])), int(rng.integers(1, 40))
    n_old, n_new = int(rng.integers(1, 70)), int(rng.integers(1, 70))
    tables, lens, refs, num_pages = ref.batch(rng, n_old, 4, page * max_pages, page, max_pages,
                                              spare=int(rng.choice([0, 3, 60, 3000])))
    # lengths past what is held or below 0; entries behind the held pages that are none
    lens = np.where(rng.random(n_old) < 0.1, rng.choice([-3, 2 ** 31 - 1], n_old), lens)
    tables = np.where((tables < 0) & (rng.random(tables.shape) < 0.3), num_pages + 5, tables).astype(np.int32)
    parents = rng.integers(-1, n_old + 1, n_new)
    reserve = None if seed % 3 == 0 else rng.integers(-5, page * max_pages + 3, n_new) // int(rng.integers(1, 9))
    if seed % 5 == 0:  # sequences cut back into pages that others hold
        lens = (lens * rng.random(n_old)).astype(np.int64).clip(-3, page * max_pages)
    check_fork(llmk, tables, lens, parents, reserve, refs, page, num_pages)


@pytest.mark.parametrize("n_old,n_new", [(0, 5), (5, 0), (0, 0), (1, 300), (300, 1), (1024, 1024), (1500, 1100)])
def test_batches_of_unlike_sizes(llmk, n_old, n_new):
    rng = np.random.default_rng([n_old, n_new])
    tables, lens, refs, num_pages = ref.batch(rng, n_old, 5, 90, 16, 7, spare=2 * n_new + 5)
    parents = rng.integers(0, n_old, n_new) if n_old else np.full(n_new, -1)
    check_fork(llmk, tables.reshape(n_old, 7), lens, parents, np.full(n_new, 1), refs, 16, num_pages)


@pytest.mark.parametrize("max_pages", [255, 256, 257, 1000, 8192])
def test_wide_tables(llmk, max_pages):
    rng = np.random.default_rng(max_pages)
    tables, lens, refs, num_pages = ref.batch(rng, 6, 2, 16 * max_pages, 16, max_pages, spare=2 * max_pages)
    check_fork(llmk, tables, lens, np.array([0, 0, 3, 5, 5, 5, -1]), np.array([0, 40, 1, 0, 9, 17, 16 * max_pages]),
               refs, 16, num_pages)


@pytest.mark.parametrize("max_pages", [63, 64, 65, 128, 129, 300, 512, 513, 1025])
def test_wide_tables_of_many(llmk, max_pages):
    rng = np.random.default_rng(max_pages)
    tables, lens, refs, num_pages = ref.batch(rng, 70, 3, 16 * max_pages, 16, max_pages, spare=600)
    reserve = np.where(rng.random(70) < 0.1, rng.integers(0, 16 * max_pages, 70), 1)
    check_fork(llmk, tables, lens, rng.integers(-1, 70, 70), reserve, refs, 16, num_pages)
    lens = (lens * rng.random(70)).astype(np.int64)  # cut back into pages that others hold
    check_fork(llmk, tables, lens, rng.integers(-1, 70, 70), np.full(70, 20), refs, 16, num_pages)


def test_free_pages_far_behind(llmk):
    """A nearly full cache: the free pages lie at its end, some are freed by the call itself."""
    num_pages, n = 70000, 8
    rng = np.random.default_rng(5)
    refs = np.ones(num_pages, np.int64)
    tables = np.full((n, 20), -1)
    names = rng.permutation(num_pages)
    for s in range(n):
        tables[s, :10] = names[10 * s:10 * s + 10]
    free = np.setdiff1d(np.arange(num_pages - 6, num_pages), tables[tables >= 0])
    refs[free] = 0
    want = check_fork(llmk, tables.astype(np.int32), np.full(n, 10 * 16 - 3), np.array([0, 0, 0, 1, 1, 5, 5, 5, 5, 5]),
                      np.full(10, 20), refs, 16, num_pages)
    assert want[4][0] > 10


def test_no_pages_left(llmk):
    tables = np.array([[0, 1, -1, -1], [2, 3, 4, -1]])
    for refs, gives in (([1] * 5, 0), ([1] * 5 + [0], 1)):
        want = check_fork(llmk, tables.astype(np.int32), np.array([20, 40]), np.array([0, 0, 1, 1]),
                          np.array([1, 30, 1, 1]), np.array(refs), 16, len(refs))
        assert want[4][0] == gives and want[4][1] > 0


@pytest.mark.parametrize("n,spare", [(2, 0), (2, 9), (40, 0), (40, 300), (3000, 1), (3000, 9000)])
def test_sequences_cut_inside_a_page_that_they_share(llmk, n, spare):
    """All let go of the page that their children copy: it is free afterwards, and no copy's destination."""
    rng = np.random.default_rng([n, spare])
    page, num_pages = 4, 3 * (n // 2) + spare
    order, tables, refs = rng.permutation(num_pages), np.full((n, 5), -1), np.zeros(num_pages, np.int64)
    for s in range(n):  # pairs share three pages, and are cut behind the first, in the second or in the third
        tables[s, :3] = order[3 * (s // 2):3 * (s // 2) + 3]
        refs[tables[s, :3]] += 1
    lens = np.repeat(rng.integers(3, 12, n // 2), 2)
    parents = rng.integers(0, n, n)
    want = check_fork(llmk, tables, lens, parents, np.full(n, 2), refs, page, num_pages)
    pairs = want[3][want[3][:, 0] >= 0]
    assert not np.isin(pairs[:, 1], pairs[:, 0]).any() and len(set(pairs[:, 1])) == len(pairs)
    assert (want[2] >= 0).all()
    assert spare < n or len(pairs) > n // 4
    # what the children hold is what their parents held
    pool = torch.randint(-99, 99, (num_pages, page), dtype=torch.int32, device=DEV)
    before = pool.cpu().numpy()
    llmk.kv_copy_pages([pool], i32(want[3].reshape(-1)), None, n, num_pages, check_indices=True)
    after = pool.cpu().numpy()
    for c in range(n):
        held = ref.held(want[0][c], num_pages)
        tokens = min(int(lens[parents[c]]), len(held) * page)
        assert np.array_equal(after[held].reshape(-1)[:tokens], before[tables[parents[c], :3]].reshape(-1)[:tokens])


def test_a_search_captured_and_replayed(llmk):
    """Two graphs (the batch goes to and fro between two sets of arrays) run a search of many steps, whose
    pages hold what each beam wrote: nobody's tokens are lost or changed by others."""
    rng = np.random.default_rng(9)
    n, max_pages, page = 12, 8, 4
    num_pages = n * max_pages
    refs = i32(np.zeros(num_pages))
    pools = [torch.full((num_pages, page), -1, dtype=torch.int32, device=DEV),
             torch.full((num_pages, page, 3), -1.0, dtype=torch.float32, device=DEV)]
    f = [Fork(llmk, n, n, max_pages, page, num_pages) for _ in range(2)]
    parents = i32(np.full(n, -1))
    reserve = i32(np.ones(n))
    f[1].new[:-16] = -1
    f[1].lens[:-16] = 0

    def step(a, b):
        b(a.new, a.lens, parents, reserve, refs)
        llmk.kv_copy_pages(pools, b.copies, None, n, num_pages)
    graphs = []
    saved = refs.clone()
    for a, b in ((f[1], f[0]), (f[0], f[1])):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(a, b)
        graphs.append(g)
    assert torch.equal(refs, saved)
    texts = [[] for _ in range(n)]
    for t in range(page * max_pages - 1):
        ps = np.sort(rng.integers(0, n, n)) if t else np.full(n, -1)
        if t % 5 == 4:
            ps[int(rng.integers(0, n))] = -1  # one leaves, another begins
        parents.copy_(i32(ps))
        graphs[t % 2].replay()
        torch.cuda.synchronize()
        now = f[t % 2]
        assert now.counts[1] == 0
        texts = [list(texts[p]) if p >= 0 else [] for p in ps]
        tables, lens = now.new[:-16].view(n, max_pages).cpu().numpy(), now.lens[:-16].cpu().numpy()
        assert [len(x) for x in texts] == lens.tolist()
        for c in range(n):  # each writes a token of its own
            at = lens[c]
            pools[0][tables[c, at // page], at % page] = 1000 * t + c
            pools[1][tables[c, at // page], at % page] = float(1000 * t + c)
            texts[c].append(1000 * t + c)
        now.lens[:-16] += 1
        ids, values = pools[0].cpu().numpy(), pools[1].cpu().numpy()
        for c in range(n):
            got = np.concatenate([ids[p] for p in tables[c] if p >= 0])[:len(texts[c])]
            assert got.tolist() == texts[c]
            got = np.concatenate([values[p][:, 2] for p in tables[c] if p >= 0])[:len(texts[c])]
            assert got.tolist() == texts[c]


def test_fork_refused(llmk):
    i = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731

    def call(**kw):
        a = dict(tables=i(8) - 1, lens=i(2), parents=i(2), reserve=None, refs=i(9), new=i(8), new_lens=i(2),
                 copies=i(4), counts=i(2), ws=i(64), n_old=2, n_new=2, max_pages=4, page=16, pages=9) | kw
        llmk.kv_fork(*a.values(), check_indices=True)
    call()
    same = i(8) - 1
    for bad in (dict(tables=i(7)), dict(lens=i(1)), dict(parents=i(1)), dict(refs=i(8)), dict(new=i(7)),
                dict(copies=i(3)), dict(counts=i(1)), dict(ws=i(2)), dict(parents=i(2).long()), dict(page=0),
                dict(n_old=-1), dict(tables=i(8)), dict(tables=same, new=same), dict(reserve=i(1))):
        with pytest.raises(llmk.LlmkError):
            call(**bad)


# ---------------------------------------------------------------------------------------------
# compaction
# ---------------------------------------------------------------------------------------------
def check_compact(llmk, tables, refs, in_place):
    num_pages, (n, max_pages) = len(refs), tables.shape
    new, new_refs, pairs, counts = ref.compact(tables, refs)
    dt, dr = guarded(n * max_pages), guarded(num_pages)
    dt[:-16], dr[:-16] = i32(tables.reshape(-1)), i32(refs)
    ot, orf = (dt, dr) if in_place else (guarded(n * max_pages), guarded(num_pages))
    copies, got = guarded(2 * (num_pages // 2)), guarded(2)
    ws = guarded(llmk.kv_compact_workspace_ints(num_pages))
    llmk.kv_compact(dt, dr, ot, orf, copies, got, ws, n, max_pages, num_pages)
    left(dt, dr, ot, orf, copies, got, ws)
    assert np.array_equal(ot[:-16].cpu().numpy().reshape(n, max_pages), new)
    assert np.array_equal(orf[:-16].cpu().numpy(), new_refs)
    assert np.array_equal(got[:2].cpu().numpy(), counts)
    c = copies[:-16].cpu().numpy().reshape(-1, 2)
    assert [tuple(p) for p in c[:len(pairs)]] == pairs and (c[len(pairs):] == -1).all()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seed", range(15))
def test_compaction(llmk, seed, in_place):
    rng = np.random.default_rng(seed)
    tables, _, refs, num_pages = ref.batch(rng, int(rng.integers(1, 40)), 3, int(rng.choice([5, 60, 900])), 16, 57,
                                           spare=int(rng.choice([0, 1, 50, 5000, 20000])))
    tables[tables < 0] = rng.choice([-1, -9, num_pages, 2 ** 31 - 1], int((tables < 0).sum()))
    check_compact(llmk, tables, refs, in_place)


@pytest.mark.parametrize("num_pages", [1, 2, 3, 255, 256, 257, 4095, 4096, 4097, 8192, 50001, 300000])
@pytest.mark.parametrize("share", [0.0, 0.1, 0.5, 0.97, 1.0])
def test_pools_of_many_sizes(llmk, num_pages, share):
    rng = np.random.default_rng([num_pages, int(100 * share)])
    refs = np.where(rng.random(num_pages) < share, rng.integers(1, 5, num_pages), 0)
    tables = rng.integers(-1, num_pages, (3, 70)).astype(np.int32)
    check_compact(llmk, tables, refs, num_pages % 2 == 0)
    check_compact(llmk, tables[:0], refs, False)


def test_compaction_moves_what_sequences_hold(llmk):
    """Through the copies: every sequence's pages hold what they did, captured and replayed."""
    rng = np.random.default_rng(4)
    tables, _, refs, num_pages = ref.batch(rng, 20, 3, 300, 16, 20, spare=400)
    dt, dr = i32(tables.reshape(-1)), i32(refs)
    ot, orf = torch.empty_like(dt), torch.empty_like(dr)
    copies, counts = i32(np.zeros(num_pages // 2 * 2)), i32([0, 0])
    ws = i32(np.zeros(llmk.kv_compact_workspace_ints(num_pages)))
    pool = torch.randn(num_pages, 16, 2, 8, device=DEV)

    def step():
        llmk.kv_compact(dt, dr, ot, orf, copies, counts, ws, 20, 20, num_pages)
        llmk.kv_copy_pages([pool], copies, counts, num_pages // 2, num_pages)
    g = torch.cuda.CUDAGraph()
    before = pool.clone()
    with torch.cuda.graph(g):
        step()
    for replay in range(3):
        pool.copy_(before)
        g.replay()
        torch.cuda.synchronize()
        new, old = ot.view(20, 20).long(), dt.view(20, 20).long()
        held = old >= 0
        assert torch.equal(pool[new[held]], before[old[held]])
        assert int(new.max()) < int(counts[1]) == int((dr > 0).sum())
        ws.random_()


def test_compaction_refused(llmk):
    i = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
    for bad in (dict(tables=i(7)), dict(refs=i(8)), dict(new=i(7)), dict(new_refs=i(8)), dict(copies=i(7)),
                dict(counts=i(1)), dict(ws=i(8)), dict(n=-1), dict(pages=0), dict(refs=i(9).float())):
        a = dict(tables=i(8), refs=i(9), new=i(8), new_refs=i(9), copies=i(8), counts=i(2), ws=i(99), n=2,
                 max_pages=4, pages=9) | bad
        with pytest.raises(llmk.LlmkError):
            llmk.kv_compact(*a.values())
