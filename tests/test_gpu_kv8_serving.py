"""The operators of the 8-bit cache as a serving loop runs them, one behind the other, and attention's
launches for long prompts."""
import numpy as np
import pytest
import torch

import _kv8 as ref
from test_gpu_kv8 import (DEV, PAGE, Pools, attention_case, check_attention, dev, do_append, do_attention,
                          i32, inv_freq)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------
# long prompts: blocks of 256 columns (rows x heads of a group), for more than 1024
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("layout", [(8, 2, 64), (7, 1, 64), (8, 2, 128), (5, 1, 128)])
def test_attention_of_long_prompts(llmk, layout, workspace):
    """Prompts with and without a cached prefix beside single rows and none; a tile's and a step's
    edges, a prompt that claims more rows than it has positions; rows of nobody."""
    case = attention_case(71, layout, [700, 90, 5, 255, 257, 30], [300, 1, 0, 257, 64, 33], slack=2)
    check_attention(llmk, *case, workspace=workspace)


@pytest.mark.parametrize("dim", [64, 128])
def test_long_prompts_pass_over_nan_that_a_row_does_not_see(llmk, dim):
    q, pools, tables, starts, lens = attention_case(72, (8, 2, dim), [64, 420], [20, 300])
    pools.v.codes[tables[0, 3], 1, 9, :] = 0xFF    # position 57 of 64
    pools.k.codes[tables[1, 20], 1, 7, 60] = 0x7F  # position 327 of 420
    pools.v.codes[tables[1, 12], 0, 0, 9] = 0x7F   # position 192
    pools.v.codes[tables[1, 2], 0, 15, 10] = 0x7F  # position 47: in front of all its rows
    pools.v.codes[tables[1, 26], 0, 3, 11] = 0xFF  # position 419: the last row's alone
    pools.upload()
    q[25, 1, 5] = np.nan
    q[28, 0, 0] = np.inf
    for workspace in (True, False):
        check_attention(llmk, q, pools, tables, starts, lens, workspace=workspace)


def test_long_prompts_among_hundreds_of_sequences(llmk):
    """More sequences than a block has threads, most of one row or none."""
    rng = np.random.default_rng(73)
    counts = rng.integers(0, 2, 700)
    counts[[3, 411, 699]] = 300, 150, 40
    lens = counts + rng.integers(0, 30, 700)
    case = attention_case(74, (4, 1, 64), lens, counts, slack=1)
    check_attention(llmk, *case)


@pytest.mark.parametrize("n", [64, 65, 200, 256, 257, 600])
def test_batches_of_many_sequences(llmk, n):
    """Shares are found by lanes up to 256 sequences and by threads past them: single rows, a few, and
    a few beside more."""
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 150, n)
    check_attention(llmk, *attention_case(77, (4, 1, 64), lens))
    counts = np.minimum(rng.integers(0, 5, n), lens)
    check_attention(llmk, *attention_case(78, (4, 1, 128), lens, counts, slack=1))
    counts[rng.integers(0, n, 5)] = 20
    check_attention(llmk, *attention_case(79, (4, 1, 64), lens, counts))


@pytest.mark.parametrize("longest", [90, 250, 700])
def test_more_units_than_simds_under_narrow_tables(llmk, longest):
    """2400 pairs of a sequence and a kv head: whole, shared among two waves a SIMD, among one."""
    lens = np.random.default_rng(longest).integers(0, 60, 300)
    lens[7] = longest
    check_attention(llmk, *attention_case(81, (8, 8, 64), lens))


def test_a_prompt_of_more_tiles_than_a_wave_counts(llmk):
    """One sequence of 67200 columns; some of its rows against the definition."""
    heads, rows = 32, 2100
    q, pools, tables, starts, lens = attention_case(80, (heads, 1, 64), [rows], [rows])
    got = do_attention(llmk, q, pools, tables, starts, lens).astype(np.float64)
    some = np.array([0, 1, 7, 8, 1000, 2040, 2047, 2048, 2098, 2099])
    want, bound = ref.attention(q[some], pools.k, pools.v, np.repeat(tables, some.size, 0), None,
                                some + 1)
    assert (np.abs(got[some] - want) <= np.maximum(bound, 2.0 ** -60)).all()
    assert np.isfinite(got).all()


def test_long_prompts_with_scores_of_any_size(llmk):
    """Scores past 2^30, all equal or one alone, and a maximum that grows by steps of less and of more
    than what a running one lets pass."""
    q, pools, tables, starts, lens = attention_case(75, (4, 1, 64), [600], [300])
    for sign in (1.0, -1.0):
        pools.k.codes[:] = 0x7E
        pools.k.scale[:] = 2.0 ** 7
        pools.upload()
        q[:] = 60000.0 * sign
        check_attention(llmk, q, pools, tables, starts, lens)
    pools.k.codes[:] = 0
    pools.k.scale[:] = 1.0
    for page in range(38):  # scores 0, 4, 8 .. log2 units, and a step down behind each third page
        pools.k.codes[tables[0, page], :, :, 0] = ref.encode(np.full(
            (1, PAGE), (page - (page % 3 == 2) * 2) * 0.7))
    pools.upload()
    for size in (1.0, 4.0, 30.0):
        q[:] = 0
        q[:, :, 0] = size
        check_attention(llmk, q, pools, tables, starts, lens)


@pytest.mark.parametrize("n_kv", [257, 512])
def test_more_kv_heads_than_wide_blocks(llmk, n_kv):
    """max_rows announces a long prompt where a launch has fewer such blocks than kv heads."""
    case = attention_case(76, (n_kv, n_kv, 64), [37, 20], [3, 2])
    check_attention(llmk, *case, max_rows=2000)


@pytest.mark.parametrize("n_kv,dim", [(8, 64), (4, 128)])
def test_keys_are_the_nearest_to_the_definition(llmk, n_kv, dim):
    """Two million rotated keys, at near and far positions: every code that of the 64-bit value."""
    rng = np.random.default_rng(82)
    for first in (0, 120000):
        rows = 4000
        lens = np.array([first + rows])
        tables = np.zeros((1, (first + rows + 15) // 16), np.int32)
        tables[0, first // 16:] = rng.permutation(rows // 16)
        pools = Pools(rows // 16, n_kv, dim)
        qkv = (rng.standard_normal((rows, (1 + 2 * n_kv) * dim))
               * np.exp(rng.standard_normal((rows, 1)))).astype(np.float16)
        inv = inv_freq(llmk, dim)
        starts = np.array([0, rows])
        do_append(llmk, pools, qkv, tables, starts, lens, inv, (1, n_kv, dim))
        ref.append(pools.k, pools.v, qkv, tables, starts, lens, inv, 1, n_kv, dim)
        for side, c in enumerate((pools.k, pools.v)):
            assert np.array_equal(pools.scale(side), c.scale)
            assert np.array_equal(pools.codes(side), c.codes)


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
class Loop:
    """Some sequences served from tables of tokens: qkv of a token's row, logits by a projection of
    the attention's output."""
    heads, n_kv, dim, vocab, n, widest = 8, 2, 64, 1003, 4, 9

    def __init__(self, llmk, seed, rows):
        rng = np.random.default_rng(seed)
        self.llmk, self.rng = llmk, rng
        self.embed = rng.standard_normal((self.vocab, 12 * self.dim)).astype(np.float16)
        self.head = (rng.standard_normal((self.vocab, 512)) * 0.4).astype(np.float16)
        self.tables = rng.permutation(self.n * self.widest).astype(np.int32).reshape(self.n, -1)
        self.pools = Pools(self.n * self.widest, self.n_kv, self.dim)
        self.on_gpu = i32(self.tables)
        self.blas = llmk.Blas()
        self.inv = dev(inv_freq(llmk, self.dim))
        self.ws = torch.zeros(llmk.kv8_attention_workspace_floats(self.dim), device=DEV)
        self.vs = torch.zeros(llmk.verify_drafts_workspace_floats(rows, self.n, self.vocab),
                              device=DEV)
        half = dict(dtype=torch.float16, device=DEV)
        self.qkv = torch.zeros((rows, 12 * self.dim), **half)
        self.q = torch.zeros((rows, self.heads, self.dim), **half)
        self.out = torch.zeros((rows, self.heads, self.dim), **half)
        self.logits = torch.zeros((rows, self.vocab), **half)
        self.guess = torch.zeros((rows, self.vocab), **half)
        whole = dict(dtype=torch.int32, device=DEV)
        self.lens, self.n_accepted = (torch.zeros(self.n, **whole) for _ in range(2))
        self.drafts, self.tokens = (torch.zeros(rows, **whole) for _ in range(2))
        self.u, self.u2 = torch.zeros(rows, device=DEV), torch.zeros(self.n, device=DEV)
        self.t, self.w = dev(np.array([1.0, 0.7, 0.0, 1.5], np.float32)), dev(self.head)

    def step(self, starts, n_rows, max_rows):
        """The rows into the cache, over it, to logits, to tokens."""
        L, batch = self.llmk, (self.on_gpu, starts, self.lens)
        L.kv8_append(self.qkv, 12 * self.dim, self.q, *self.pools.gpu, *batch, self.inv, n_rows,
                     self.n, self.widest, PAGE, self.heads, self.n_kv, self.dim)
        L.kv8_attention(self.q, *self.pools.gpu, *batch, self.out, self.ws, n_rows, self.n, max_rows,
                        self.widest, PAGE, self.heads, self.n_kv, self.dim)
        L.linear(self.blas, self.out, self.w, self.logits, n_rows, 512, self.vocab)
        L.verify_drafts(self.logits, self.guess, self.drafts, starts, self.t, self.u, self.u2,
                        self.n_accepted, self.tokens, self.vs, n_rows, self.n, self.vocab)

    def give(self, tokens, starts, lens):
        """The rows' inputs: random numbers, and draft logits that are near the target's where the last
        step had some."""
        n_rows = len(tokens)
        self.qkv[:n_rows] = dev(self.embed[tokens])
        self.lens.copy_(i32(lens))
        noise = dev((self.rng.standard_normal((n_rows, self.vocab)) * 0.5).astype(np.float16))
        self.guess[:n_rows] = self.logits[:n_rows] + noise
        drafts = np.zeros(n_rows, np.int32)
        for s in range(self.n):  # a row's draft is the next row's token
            drafts[starts[s]:starts[s + 1] - 1] = tokens[starts[s] + 1:starts[s + 1]]
        self.drafts[:n_rows] = dev(drafts)
        self.u[:n_rows] = dev(self.rng.random(n_rows, dtype=np.float32) * 0.3)
        self.u2.copy_(dev(self.rng.random(self.n, dtype=np.float32)))


def test_prompts_then_drafts_step_by_step(llmk):
    """Prompts, then steps of drafted tokens of which some are refused: their places in the cache are
    taken by the next step's rows. Every operator's result against the definition, from the inputs
    that it got."""
    prompt = np.array([40, 17, 1, 33])
    loop = Loop(llmk, 81, 2 * int(prompt.sum()))
    rng, layout = loop.rng, (loop.heads, loop.n_kv, loop.dim)
    held = np.zeros(loop.n, np.int64)
    pending = [list(rng.integers(0, loop.vocab, n)) for n in prompt]
    refused = 0
    for turn in range(7):
        starts = np.r_[0, np.cumsum([len(p) for p in pending])]
        n_rows, tokens = int(starts[-1]), np.array(sum(pending, []))
        lens = held + np.diff(starts)
        loop.give(tokens, starts, lens)
        loop.step(i32(starts), n_rows, int(np.diff(starts).max()))
        torch.cuda.synchronize()
        # the cache
        qkv = loop.embed[tokens]
        want = ref.append(loop.pools.k, loop.pools.v, qkv, loop.tables, starts, lens,
                          loop.inv.cpu().numpy(), *layout)
        size = np.abs(qkv[:, :512].astype(np.float64)).reshape(n_rows, 8, 2, 32).sum(2)
        tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 2.0 ** -21 * np.concatenate([size, size], -1)
        q = loop.q[:n_rows].cpu().numpy()
        assert (np.abs(q - want) <= tol).all()
        for side, c in enumerate((loop.pools.k, loop.pools.v)):
            used = ~np.isnan(c.scale)
            assert np.array_equal(loop.pools.scale(side)[used], c.scale[used])
            a, b = loop.pools.codes(side), c.codes
            differ = (a != b) & used[:, :, None, None]
            # K is rotated in fp32: a value at the middle between two codes may take the other
            assert not differ.any() or (side == 0 and differ.mean() < 1e-4 and np.abs(
                a[differ].astype(int) - b[differ]).max() == 1)
            c.codes[:] = a
        # the attention, of the q that it got
        out = loop.out[:n_rows].cpu().numpy().astype(np.float64)
        want, bound = ref.attention(q, loop.pools.k, loop.pools.v, loop.tables, starts, lens)
        assert (np.abs(out - want) <= np.maximum(bound, 2.0 ** -60)).all()
        # the logits: one rounding to fp16 of sums of 512 products in fp32
        logits, out = loop.logits[:n_rows].cpu().numpy(), out.reshape(n_rows, 512)
        want = out @ loop.head.astype(np.float64).T
        tol = 2.0 ** -11 * np.abs(want) + 512 * 2.0 ** -24 * (
            np.abs(out) @ np.abs(loop.head.astype(np.float64)).T) + 2.0 ** -25
        assert (np.abs(logits - want) <= tol).all()
        # the tokens
        accepted, chosen = ref.verify(
            logits, loop.guess[:n_rows].cpu().numpy(), loop.drafts.cpu().numpy()[:n_rows], starts,
            loop.t.cpu().numpy(), loop.u.cpu().numpy()[:n_rows], loop.u2.cpu().numpy(), loop.n)
        assert np.array_equal(loop.n_accepted.cpu().numpy(), accepted)
        assert np.array_equal(loop.tokens[:n_rows].cpu().numpy(), chosen)
        # on: what stands is held, the new token is the next step's first row, drafts behind it
        for s in range(loop.n):
            rows = len(pending[s])
            if turn == 0:  # a prompt is no draft: all of it stands, the last row's logits count
                stand, token = rows, int(logits[starts[s + 1] - 1].argmax())
            else:
                stand, token = 1 + int(accepted[s]), int(chosen[starts[s] + accepted[s]])
                refused += rows - stand
            held[s] += stand
            # half of the drafts are what the model itself would say, so that some stand
            likely = np.argsort(-logits[starts[s + 1] - 1])[:2]
            drafts = [int(likely[i % 2]) if rng.random() < 0.7 else int(rng.integers(loop.vocab))
                      for i in range(int(rng.integers(0, 5)))]
            pending[s] = [token] + drafts
    assert refused > 0


def test_two_graphs_with_one_workspace(llmk):
    """A prompt's step and a step of drafts, captured apart with the same workspaces and replayed in
    turn with other inputs, against eager calls with their own."""
    a, b = Loop(llmk, 82, 80), Loop(llmk, 82, 80)
    shapes = [np.array([0, 40, 50, 51, 75]), np.array([0, 3, 4, 9, 11])]
    on_gpu = [i32(x) for x in shapes]
    for loop in (a, b):
        loop.give(np.zeros(75, np.int64), shapes[0], np.diff(shapes[0]))
    graphs, stream = [], torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for x, g in zip(shapes, on_gpu):
            b.step(g, int(x[-1]), int(np.diff(x).max()))
    stream.synchronize()
    for x, g in zip(shapes, on_gpu):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            b.step(g, int(x[-1]), int(np.diff(x).max()))
        graphs.append(graph)
    for loop in (a, b):  # what the warm steps left
        for x in loop.pools.gpu:
            x.view(torch.uint8).zero_()
        loop.logits.zero_()
        loop.rng = np.random.default_rng(83)
    held = np.zeros(4, np.int64)
    for turn in range(8):
        which = 0 if turn == 0 else 1 if turn % 3 else 0
        x = shapes[which]
        if held.max() + 40 > 9 * PAGE:
            held[:] = 0
        lens, n_rows = held + np.diff(x), int(x[-1])
        tokens = np.random.default_rng(90 + turn).integers(0, a.vocab, n_rows)
        for loop in (a, b):
            loop.give(tokens, x, lens)
        a.step(on_gpu[which], n_rows, int(np.diff(x).max()))
        torch.cuda.synchronize()
        graphs[which].replay()
        torch.cuda.synchronize()
        for key in ("q", "out", "logits", "tokens", "n_accepted"):
            p, r = getattr(a, key), getattr(b, key)
            assert torch.equal(p[:n_rows], r[:n_rows]), (turn, key)
        held = held + np.diff(x) - (np.diff(x) > 1)
    del graphs  # in front of the projections' handle


def test_two_streams_at_once(llmk):
    """Two batches on streams of their own, each with a workspace and a cache of its own."""
    cases = [attention_case(84, (8, 2, 64), [5000, 300], [1, 4]),
             attention_case(85, (8, 2, 64), [2500, 900, 70], [300, 1, 9])]
    runs = []
    for q, pools, tables, starts, lens in cases:
        runs.append(dict(q=dev(q), pools=pools.gpu, batch=(i32(tables), i32(starts), i32(lens)),
                         shape=(q.shape[0], tables.shape[0], int(np.diff(starts).max()),
                                tables.shape[1]),
                         ws=torch.zeros(llmk.kv8_attention_workspace_floats(64), device=DEV),
                         out=[torch.zeros_like(dev(q)) for _ in range(8)],
                         stream=torch.cuda.Stream()))
    torch.cuda.synchronize()

    def go(r, out, stream):
        llmk.kv8_attention(r["q"], *r["pools"], *r["batch"], out, r["ws"], *r["shape"], PAGE, 8, 2,
                           64, stream)
    for r in runs:
        go(r, r["out"][0], None)
        torch.cuda.synchronize()
    for i in range(1, 8):
        for r in runs:
            go(r, r["out"][i], r["stream"])
    torch.cuda.synchronize()
    for r in runs:
        for out in r["out"][1:]:
            assert torch.equal(out, r["out"][0])
