"""The 8-bit KV cache on the GPU (append with rotation, read-back, attention) against its definition
in 64 bits, at the sizes, lengths and values where it can go wrong."""
import numpy as np
import pytest
import torch

import _kv8 as ref
from _helpers import ROPE

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 16

LAYOUTS = [(32, 8, 64), (32, 8, 128), (5, 5, 64), (28, 4, 128), (12, 2, 64), (32, 1, 128),
           (3, 1, 64)]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def i32(a):
    return None if a is None else dev(np.asarray(a, np.int32))


def inv_freq(llmk, dim):
    return np.array(llmk.compute_rope_inv_freq(dim, *ROPE.values()), np.float32)


def tables_for(rng, need, extra=2):
    """Block tables of the given page counts from a shuffled pool; unused entries name page 0."""
    need = np.asarray(need)
    order = rng.permutation(int(need.sum()) + extra).astype(np.int32)
    t, at = np.zeros((need.size, max(1, int(need.max(initial=1)))), np.int32), 0
    for s, n in enumerate(need):
        t[s, :n] = order[at:at + n]
        at += n
    return t, order.size


class Pools:
    """A cache on the GPU beside its restatement."""

    def __init__(self, num_pages, n_kv, dim):
        self.k, self.v = ref.Cache(num_pages, n_kv, dim), ref.Cache(num_pages, n_kv, dim)
        self.upload()

    def upload(self):
        self.gpu = []
        for c in (self.k, self.v):
            self.gpu += [dev(c.codes).view(torch.float8_e4m3fn), dev(c.scale)]

    def codes(self, side):
        return self.gpu[2 * side].view(torch.uint8).cpu().numpy()

    def scale(self, side):
        return self.gpu[2 * side + 1].cpu().numpy()


def random_cache(rng, num_pages, n_kv, dim, size=1.0):
    p = Pools(num_pages, n_kv, dim)
    for c in (p.k, p.v):
        c.codes[:] = rng.integers(0, 256, c.codes.shape)
        c.codes[(c.codes & 127) == 127] = 0
        c.codes[(c.codes & 127) > 0x58] &= 0xDF  # mostly middle magnitudes, as real blocks have
        c.scale[:] = 2.0 ** rng.integers(-9, -5, c.scale.shape) * size
    p.upload()
    return p


def do_append(llmk, pools, qkv, tables, starts, lens, inv, layout, stream=None, ld=None):
    heads, n_kv, dim = layout
    q = torch.full((qkv.shape[0], heads, dim), 7.0, dtype=torch.float16, device=DEV)
    llmk.kv8_append(dev(qkv), qkv.shape[1], q, *pools.gpu, i32(tables), i32(starts), i32(lens),
                    dev(inv), qkv.shape[0], tables.shape[0], tables.shape[1], PAGE, heads, n_kv,
                    dim, stream)
    torch.cuda.synchronize()
    return q.cpu().numpy()


def one_nan(codes):
    """The codes with one NaN for both: its sign is nobody's."""
    return np.where((codes & 127) == 127, 127, codes)


def check_append(llmk, pools, qkv, tables, starts, lens, layout):
    """One append on both sides. V is exact; K's codes are those of the 64-bit value or, where that
    lies within what fp32 may be off of the middle between two, the neighbour's."""
    heads, n_kv, dim = layout
    inv = inv_freq(llmk, dim)
    got = do_append(llmk, pools, qkv, tables, starts, lens, inv, layout).astype(np.float64)
    want = ref.append(pools.k, pools.v, qkv, tables, starts, lens, inv, heads, n_kv, dim)
    x = np.abs(qkv[:, :heads * dim].astype(np.float64)).reshape(-1, heads, 2, dim // 2)
    size = np.repeat(x.sum(2)[:, :, None], 2, 2).reshape(want.shape)
    none = np.isnan(want).all((1, 2)) if starts is not None else np.zeros(len(want), bool)
    assert (got[none] == 7.0).all(), "a row of no sequence was written"
    # one rounding to fp16; cosine and sine to 2^-22, two products and a sum in fp32
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 2.0 ** -21 * size
    assert (np.abs(got - want)[~none] <= tol[~none]).all()
    assert np.array_equal(one_nan(pools.codes(1)), one_nan(pools.v.codes))
    assert np.array_equal(pools.scale(1), pools.v.scale, equal_nan=True)
    assert np.array_equal(pools.scale(0), pools.k.scale, equal_nan=True)
    a, b = one_nan(pools.codes(0)), one_nan(pools.k.codes)
    if not np.array_equal(a, b):
        d = np.abs(a.astype(int) - b.astype(int))
        assert d.max() == 1 and (d > 0).mean() < 1e-4, ((d > 0).sum(), d.max())
        pools.k.codes = a.copy()  # go on from there


def rows_case(rng, n_kv, heads, dim, n_rows, spread=1.0, pad=0):
    x = rng.standard_normal((n_rows, heads + 2 * n_kv, dim)) * np.exp(
        spread * rng.standard_normal((n_rows, heads + 2 * n_kv, 1)))
    out = np.full((n_rows, (heads + 2 * n_kv) * dim + pad), np.nan, np.float16)
    out[:, :x[0].size] = x.reshape(n_rows, -1)
    return out


@pytest.mark.parametrize("layout", LAYOUTS)
def test_append_a_prompt_then_drafts_then_single_tokens(llmk, layout):
    """Ragged prompts (one of no rows, one that fills its pages exactly), then up to five rows over
    the last ones of before (refused drafts), then one row each without row_starts, each behind the
    other: pages end inside a call, scales grow and stay, ld is wider than a row."""
    heads, n_kv, dim = layout
    rng = np.random.default_rng(heads * dim + n_kv)
    counts = np.array([37, 0, 16, 1, 130])
    tables, pages = tables_for(rng, [4, 1, 3, 2, 10])
    pools = Pools(pages, n_kv, dim)
    lens = counts.copy()
    qkv = rows_case(rng, n_kv, heads, dim, int(counts.sum()) + 2, pad=24)  # two rows of nobody
    check_append(llmk, pools, qkv, tables, np.r_[0, np.cumsum(counts)], lens, layout)
    for back, counts in ((0, [3, 5, 1, 2, 5]), (2, [4, 5, 2, 3, 1]), (1, [2, 2, 2, 2, 2])):
        counts = np.array(counts)
        lens = np.maximum(lens - back, 0) + counts
        qkv = rows_case(rng, n_kv, heads, dim, int(counts.sum()), pad=8)
        check_append(llmk, pools, qkv, tables, np.r_[0, np.cumsum(counts)], lens, layout)
    for size in (0.1, 30.0, 3.0):
        lens = lens + 1
        qkv = rows_case(rng, n_kv, heads, dim, 5)
        check_append(llmk, pools, (qkv * size).astype(np.float16), tables, None, lens, layout)


def test_append_every_fp16_as_a_value(llmk):
    """All 65536 bit patterns as V, subnormals, infinities and NaN among them: the codes and scales
    of the definition, and what is read back is the code's value exactly."""
    layout = heads, n_kv, dim = 1, 1, 64
    bits = np.random.default_rng(3).permutation(65536).astype(np.uint16)
    bits[:1024] = np.sort(bits[:1024])  # some blocks of near magnitudes
    bits[-4096:] &= 0x83FF  # some of subnormals alone
    qkv = np.zeros((1024, 192), np.float16)
    qkv[:, 128:] = bits.view(np.float16).reshape(1024, 64)
    tables, pages = tables_for(np.random.default_rng(4), [64])
    pools = Pools(pages, n_kv, dim)
    check_append(llmk, pools, qkv, tables, np.array([0, 1024]), np.array([1024]), layout)
    k, v = do_gather(llmk, pools, tables, np.array([0, 1024]), np.array([1024]), 1024)
    want = ref.gather(pools.v, tables, np.array([0, 1024]), np.array([1024]), 1024)
    assert np.array_equal(v.astype(np.float64), want, equal_nan=True)
    assert not k.any()


def test_append_one_token_at_a_time_with_growing_and_shrinking_sizes(llmk):
    """A page filled token by token: each larger one rounds what is held again, smaller ones leave
    the scale; the next page begins with its own. Zeros alone give the least scale; magnitudes past
    57344 are held as that."""
    layout = heads, n_kv, dim = 4, 2, 64
    rng = np.random.default_rng(11)
    tables, pages = tables_for(rng, [3, 3])
    pools = Pools(pages, n_kv, dim)
    sizes = [1e-3, 1.0, 0.0, 1e-6, 60.0, 5.0, 900.0, 1e-2] * 5
    for n, size in enumerate(sizes):
        qkv = (rng.standard_normal((2, 8 * dim)) * size).astype(np.float16)
        if n == 30:
            qkv[1, -dim:] = 65504.0
        check_append(llmk, pools, qkv, tables, None, np.array([n + 1, n + 1]), layout)


def test_append_to_places_that_do_not_exist(llmk):
    """Rows in front of position 0 and past the table: nothing is written there, and their q is
    zero; a sequence of length 0 and one of no rows among them."""
    layout = heads, n_kv, dim = 4, 1, 128
    rng = np.random.default_rng(12)
    tables, pages = tables_for(rng, [2, 2, 2, 2])
    pools = random_cache(rng, pages, n_kv, dim)  # tokens in front of the rows
    starts, lens = np.array([0, 5, 8, 8, 28]), np.array([2, 0, 7, 40])
    check_append(llmk, pools, rows_case(rng, n_kv, heads, dim, 30), tables, starts, lens, layout)
    check_append(llmk, pools, rows_case(rng, n_kv, heads, dim, 4), tables, None,
                 np.array([0, -3, 33, 32]), layout)


@pytest.mark.parametrize("dim", [64, 128])
def test_append_at_far_positions(llmk, dim):
    """Angles of 10^5 and more keep their fraction."""
    layout = heads, n_kv, dim = 2, 1, dim
    rng = np.random.default_rng(13)
    tables = np.zeros((3, 8192), np.int32)
    at = np.array([131072, 100003, 65537])
    tables[np.arange(3), (at - 1) // PAGE] = [1, 2, 3]
    pools = Pools(4, n_kv, dim)
    for c in (pools.k, pools.v):
        c.scale[:] = 2.0 ** -9
    pools.upload()
    check_append(llmk, pools, rows_case(rng, n_kv, heads, dim, 3, 0.0), tables, None, at, layout)


def test_append_of_many_sequences_with_and_without_rows(llmk):
    """5000 sequences, most without rows: the search for a row's sequence takes several steps."""
    layout = heads, n_kv, dim = 1, 1, 64
    rng = np.random.default_rng(14)
    counts = (rng.random(5000) < 0.2).astype(int) * rng.integers(1, 4, 5000)
    lens = counts + rng.integers(0, 30, 5000)
    tables, pages = tables_for(rng, np.full(5000, 3))
    pools = Pools(pages, n_kv, dim)
    for c in (pools.k, pools.v):
        c.codes[:] = 0x21
        c.scale[:] = 2.0 ** -8
    pools.upload()
    check_append(llmk, pools, rows_case(rng, n_kv, heads, dim, int(counts.sum()) + 3), tables,
                 np.r_[0, np.cumsum(counts)], lens, layout)


def do_gather(llmk, pools, tables, starts, lens, n_rows):
    n_kv, dim = pools.k.codes.shape[1], pools.k.codes.shape[3]
    k = torch.full((n_rows, n_kv, dim), float("inf"), dtype=torch.float16, device=DEV)
    v = k.clone()
    llmk.kv8_gather(*pools.gpu, i32(tables), i32(starts), i32(lens), k, v, n_rows, tables.shape[0],
                    tables.shape[1], PAGE, n_kv, dim)
    torch.cuda.synchronize()
    return k.cpu().numpy(), v.cpu().numpy()


@pytest.mark.parametrize("n_kv,dim", [(8, 64), (1, 64), (3, 128)])
def test_gather_is_exact(llmk, n_kv, dim):
    """Whole sequences and their ends, from inside pages; sequences of no rows, rows of nobody,
    positions that do not exist; every scale."""
    rng = np.random.default_rng(21)
    counts = np.array([0, 1, 70, 33, 5, 0, 200])
    lens = np.array([9, 1, 70, 50, 3, 0, 215])
    tables, pages = tables_for(rng, (lens + 15) // 16)
    pools = random_cache(rng, pages, n_kv, dim)
    for c in (pools.k, pools.v):
        c.scale[:] = 2.0 ** rng.integers(-15, 8, c.scale.shape)
        c.codes[:] = rng.integers(0, 256, c.codes.shape)
    pools.upload()
    n_rows = int(counts.sum()) + 5
    for starts, lens, n in ((np.r_[0, np.cumsum(counts)], lens, n_rows),
                            (None, np.array([9, 1, 70, 0, -2, 17, 500]), 7)):
        for got, c in zip(do_gather(llmk, pools, tables, starts, lens, n), (pools.k, pools.v)):
            assert np.array_equal(got.astype(np.float64), ref.gather(c, tables, starts, lens, n),
                                  equal_nan=True)


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def do_attention(llmk, q, pools, tables, starts, lens, workspace=True, max_rows=None, out=None):
    n_rows, heads, dim = q.shape
    if out is None:
        out = torch.full(q.shape, 7.0, dtype=torch.float16, device=DEV)
    ws = None
    if workspace:
        ws = torch.full((llmk.kv8_attention_workspace_floats(dim) + 4,), float("nan"), device=DEV)
        ws[-4:] = 5.0
    counts = [1] if starts is None else np.diff(starts)
    llmk.kv8_attention(q if isinstance(q, torch.Tensor) else dev(q), *pools.gpu, i32(tables),
                       i32(starts), i32(lens), out, ws, n_rows, tables.shape[0],
                       max(counts) if max_rows is None else max_rows, tables.shape[1], PAGE, heads,
                       pools.k.codes.shape[1], dim)
    torch.cuda.synchronize()
    assert ws is None or bool((ws[-4:] == 5.0).all()), "a write past the workspace"
    return out.cpu().numpy()


def check_attention(llmk, q, pools, tables, starts, lens, **how):
    got = do_attention(llmk, q, pools, tables, starts, lens, **how).astype(np.float64)
    want, bound = ref.attention(q, pools.k, pools.v, tables, starts, lens)
    nobody = np.isinf(want)
    assert (got[nobody] == 7.0).all(), "a row of no sequence was written"
    assert np.array_equal(np.isnan(got), np.isnan(want))
    some = ~nobody & ~np.isnan(want)
    off = np.abs(got - want)[some] / np.maximum(bound[some], 2.0 ** -60)  # exact where it is 0
    assert off.size == 0 or off.max() <= 1.0, (off.max(), (off > 1).sum(), off.size)
    return got


def attention_case(seed, layout, lens, counts=None, slack=0, size=1.0):
    """q, cache, tables: pages that nobody owns, and slots behind a sequence's end, hold NaN."""
    heads, n_kv, dim = layout
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens)
    tables, pages = tables_for(rng, (np.maximum(lens, 0) + 15) // 16)
    pools = random_cache(rng, pages, n_kv, dim, size)
    used = set()
    for s, n in enumerate(lens):
        used |= set(tables[s, :max(0, n + 15) // 16])
        if n > 0 and n % 16:
            for c in (pools.k, pools.v):
                c.codes[tables[s, n // 16], :, n % 16:] = 0x7F
    for page in set(range(pages)) - used:
        for c in (pools.k, pools.v):
            c.codes[page] = 0xFF
            c.scale[page] = np.nan
    pools.upload()
    starts = None if counts is None else np.r_[0, np.cumsum(counts)]
    n_rows = (lens.size if counts is None else int(np.sum(counts))) + slack
    q = rng.standard_normal((n_rows, heads, dim)).astype(np.float16)
    return q, pools, tables, starts, lens


EDGES = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 257, 300]


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_attention_of_one_row_a_sequence(llmk, layout, workspace):
    """Lengths around every edge of pages and steps; a sequence of length 0 gives zeros."""
    case = attention_case(31, layout, [0] + EDGES + [0])
    check_attention(llmk, *case, workspace=workspace)


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_attention_of_a_few_rows_a_sequence(llmk, layout, workspace):
    """Drafted rows, ragged, sequences without rows, more rows than positions (the first see
    nothing: zeros), rows of nobody."""
    counts = [1, 5, 0, 2, 9, 3, 5, 4]
    lens = [300, 70, 33, 17, 9, 2, 64, 131]
    case = attention_case(32, layout, lens, counts, slack=2)
    check_attention(llmk, *case, workspace=workspace)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("counts,lens", [([150], [150]), ([70, 1, 33, 1], [200, 90, 33, 300]),
                                         ([65, 0, 40], [64, 5, 300])])
def test_attention_of_prompts(llmk, layout, counts, lens):
    """Prompts with and without a cached prefix, single rows beside them, a prompt that claims a row
    more than it has positions; with and without a workspace."""
    case = attention_case(33, layout, lens, counts, slack=1)
    for workspace in (True, False):
        check_attention(llmk, *case, workspace=workspace)


def test_attention_of_few_long_sequences(llmk):
    """Contexts that many blocks share."""
    case = attention_case(34, (8, 2, 64), [20011, 5, 7777])
    check_attention(llmk, *case)
    case = attention_case(35, (4, 1, 128), [9001, 700], [5, 3])
    check_attention(llmk, *case)


def test_attention_more_rows_than_announced(llmk):
    """max_rows only chooses kernels."""
    case = attention_case(36, (8, 2, 64), [90, 40], [60, 2])
    a = check_attention(llmk, *case, max_rows=1)
    b = check_attention(llmk, *case, max_rows=60)
    c = check_attention(llmk, *case, max_rows=1000000)
    assert np.abs(a - b).max() < 0.1 and np.abs(a - c).max() < 0.1


@pytest.mark.parametrize("layout", [(32, 8, 64), (6, 2, 128)])
def test_attention_passes_over_nan_that_a_row_does_not_see(llmk, layout):
    """A cached NaN (K or V) reaches exactly the rows that see its position, and in V only its dim;
    a NaN in q its own row and head."""
    q, pools, tables, starts, lens = attention_case(37, layout, [40, 64, 200], [6, 20, 130])
    pools.v.codes[tables[0, 2], 0, 5, 3] = 0x7F   # position 37 of 40: rows 3 .. 5 of 6 see it
    pools.v.codes[tables[1, 3], 1, 9, :] = 0xFF   # position 57 of 64
    pools.k.codes[tables[2, 10], 1, 7, 60] = 0x7F  # position 167 of 200
    pools.v.codes[tables[2, 5], 0, 0, 9] = 0x7F   # position 80
    pools.v.codes[tables[2, 2], 0, 15, 10] = 0x7F  # position 47: in front of all its rows
    pools.upload()
    q[3, 1, 5] = np.nan
    q[8, 0, 0] = np.inf
    for workspace in (True, False):
        check_attention(llmk, q, pools, tables, starts, lens, workspace=workspace)


def test_attention_scores_of_any_size(llmk):
    """Scores from 2^-20 to 2^24 and more: the largest weight stays 1, nothing overflows. Past 2^24
    fp32 scores are whole numbers apart, so the cache is made such that a row's largest score is
    alone by far, or that all its scores are equal."""
    heads, n_kv, dim = layout = (4, 1, 64)
    for size in (2.0 ** -4, 16.0):
        case = attention_case(38, layout, [50, 333], [1, 40], size=size)
        check_attention(llmk, *case)
    q, pools, tables, starts, lens = attention_case(39, layout, [50, 333], [1, 40])
    pools.k.codes[:] = 0x7E  # 448
    pools.k.scale[:] = 2.0 ** 7
    pools.upload()
    q[:] = 60000.0
    got = check_attention(llmk, q, pools, tables, starts, lens)
    assert np.isfinite(got).all()
    q[:] = -60000.0
    check_attention(llmk, q, pools, tables, starts, lens)
    pools.k.codes[tables[1, 3], :, 4] = 0xFE  # -448: with q < 0 the only large score
    pools.upload()
    got = check_attention(llmk, q, pools, tables, starts, lens)
    value = pools.v.rows(tables[1], np.array([52]))[0, 0]
    assert np.array_equal(got[1:], np.broadcast_to(value, got[1:].shape))


def test_attention_keeps_small_weights(llmk):
    """Many weights of 2^-20 and less of the largest add up: one near position against 4000 far
    ones, whose values are large."""
    heads, n_kv, dim = layout = (4, 1, 64)
    q, pools, tables, starts, lens = attention_case(40, layout, [4001, 4001], [1, 40])
    q[:] = 0
    q[:, :, 0] = 8.0
    pools.k.codes[:] = 0
    pools.k.scale[:] = 1.0
    pools.k.codes[:, :, :, 0] = 0xD4  # -12: score -12
    for s in range(2):
        pools.k.codes[tables[s, 0], :, 0, 0] = 0x30  # 0.5
    pools.v.scale[:] = 1.0
    pools.v.codes[:] = 0x70  # 128
    for s in range(2):
        pools.v.codes[tables[s, 0], :, 0, :] = 0
    pools.upload()
    check_attention(llmk, q, pools, tables, starts, lens)


@pytest.mark.parametrize("layout", [(32, 8, 64), (8, 2, 128)])
def test_attention_and_cache_past_32_bit_offsets(llmk, layout):
    """Pages whose bytes lie past 2^31 of the pools (the pools are not filled: only theirs are
    read and written)."""
    heads, n_kv, dim = layout
    pages = 2 ** 31 // (n_kv * PAGE * dim) + 9
    k = torch.empty((pages, n_kv, PAGE, dim), dtype=torch.float8_e4m3fn, device=DEV)
    v = torch.empty_like(k)
    ks = torch.empty((pages, n_kv), dtype=torch.float32, device=DEV)
    gpu = [k, ks, v, torch.empty_like(ks)]
    rng = np.random.default_rng(41)
    tables = np.array([[pages - 1, pages - 3, pages - 2]], np.int32)
    small = Pools(3, n_kv, dim)
    where = np.array([[0, 1, 2]], np.int32)
    qkv = rows_case(rng, n_kv, heads, dim, 40, 0.2)
    inv = inv_freq(llmk, dim)
    starts, lens = np.array([0, 40]), np.array([40])
    outs = []
    for pools, t in ((small.gpu, where), (gpu, tables)):
        q = torch.empty((40, heads, dim), dtype=torch.float16, device=DEV)
        batch = (i32(t), i32(starts), i32(lens))
        llmk.kv8_append(dev(qkv), qkv.shape[1], q, *pools, *batch, dev(inv), 40, 1, 3, PAGE, heads,
                        n_kv, dim)
        out, kk, vv = torch.empty_like(q), *(torch.empty((40, n_kv, dim), dtype=torch.float16,
                                                         device=DEV) for _ in range(2))
        llmk.kv8_attention(q, *pools, *batch, out, None, 40, 1, 40, 3, PAGE, heads, n_kv, dim)
        one = torch.empty_like(q[:1])
        llmk.kv8_attention(q[-1:].contiguous(), *pools, batch[0], None, batch[2], one, None, 1, 1,
                           1, 3, PAGE, heads, n_kv, dim)
        llmk.kv8_gather(*pools, *batch, kk, vv, 40, 1, 3, PAGE, n_kv, dim)
        outs.append([x.cpu() for x in (q, out, one, kk, vv)])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
def test_streams_and_graphs(llmk):
    """Append, attention and read-back on a stream of their own, captured and replayed with other
    lengths and rows between replays, against eager calls on another cache."""
    layout = heads, n_kv, dim = 8, 2, 64
    rng = np.random.default_rng(51)
    n, widest = 6, 40
    tables = rng.permutation(n * widest).astype(np.int32).reshape(n, widest)
    inv = dev(inv_freq(llmk, dim))
    counts = np.array([3, 1, 5, 2, 4, 1])
    starts = i32(np.r_[0, np.cumsum(counts)])
    n_rows = int(counts.sum())
    stream = torch.cuda.Stream()
    sides = []
    for _ in range(2):
        sides.append(dict(
            pools=Pools(n * widest, n_kv, dim).gpu, tables=i32(tables), lens=i32(counts),
            qkv=torch.zeros((n_rows, 12 * dim), dtype=torch.float16, device=DEV),
            q=torch.zeros((n_rows, heads, dim), dtype=torch.float16, device=DEV),
            out=torch.zeros((n_rows, heads, dim), dtype=torch.float16, device=DEV),
            k=torch.zeros((n_rows, n_kv, dim), dtype=torch.float16, device=DEV),
            v=torch.zeros((n_rows, n_kv, dim), dtype=torch.float16, device=DEV),
            ws=torch.zeros(llmk.kv8_attention_workspace_floats(dim), device=DEV)))

    def step(s):
        batch = (s["tables"], starts, s["lens"])
        llmk.kv8_append(s["qkv"], 12 * dim, s["q"], *s["pools"], *batch, inv, n_rows, n, widest,
                        PAGE, heads, n_kv, dim)
        llmk.kv8_attention(s["q"], *s["pools"], *batch, s["out"], s["ws"], n_rows, n, 5, widest,
                           PAGE, heads, n_kv, dim)
        llmk.kv8_gather(*s["pools"], *batch, s["k"], s["v"], n_rows, n, widest, PAGE, n_kv, dim)

    with torch.cuda.stream(stream):
        step(sides[1])  # warm
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(sides[1])
    lens = counts.copy()
    for turn in range(6):
        x = rng.standard_normal((n_rows, 12 * dim)).astype(np.float16)
        for s in sides:
            s["qkv"].copy_(dev(x))
            s["lens"].copy_(i32(lens))
        step(sides[0])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for key in ("q", "out", "k", "v"):
            assert torch.equal(sides[0][key], sides[1][key]), (turn, key)
        lens = lens + counts - np.minimum(counts, turn % 3)


def test_python_refusals(llmk):
    layout = heads, n_kv, dim = 4, 1, 64
    rng = np.random.default_rng(61)
    tables, pages = tables_for(rng, [2, 2])
    pools = random_cache(rng, pages, n_kv, dim)
    qkv = dev(rows_case(rng, n_kv, heads, dim, 2))
    q = torch.zeros((2, heads, dim), dtype=torch.float16, device=DEV)
    inv, lens = dev(inv_freq(llmk, dim)), i32([5, 20])

    def call(**kw):
        a = dict(qkv=qkv, q_out=q, k_pool=pools.gpu[0], k_scale=pools.gpu[1], v_pool=pools.gpu[2],
                 v_scale=pools.gpu[3], block_tables=i32(tables), row_starts=None, seq_lens=lens,
                 inv_freq=inv, n_rows=2, n_seqs=2, max_pages=2, page_size=16, n_heads=heads,
                 n_kv_heads=n_kv, head_dim=dim, ld=6 * dim, check_indices=True) | kw
        llmk.kv8_append(**a)

    call()
    shared = tables.copy()
    shared[1, 1] = shared[0, 0]
    for bad, text in ((dict(k_pool=pools.gpu[0].view(torch.uint8)), "float8"),
                      (dict(v_scale=pools.gpu[3][:-1]), "num_pages"),
                      (dict(seq_lens=i32([5, 33])), "seq_lens"),
                      (dict(block_tables=i32([[0, 0], [0, pages]])), "block_tables"),
                      (dict(block_tables=i32(shared)), "same page"),
                      (dict(row_starts=i32([0, 2, 1])), "row_starts"),
                      (dict(row_starts=i32([1, 1, 2])), "row_starts"),
                      (dict(inv_freq=inv.cpu()), "CUDA"),
                      (dict(ld=5 * dim), "ld"),
                      (dict(n_rows=3), "elements")):
        with pytest.raises(llmk.LlmkError, match=text):
            call(**bad)
