"""Verification of drafted tokens on the GPU against its definition in 64 bits."""
import numpy as np
import pytest
import torch

import _kv8 as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def at_offset(a, by):
    """a on the GPU, its first element `by` elements behind an aligned address."""
    t = torch.empty(a.size + 8, dtype=torch.float16, device=DEV)
    t[by:by + a.size] = dev(a).reshape(-1)
    return t[by:by + a.size].view(a.shape)


def run(llmk, logits, draft_logits, drafts, starts, temperature, accept_u, sample_u, n_seqs,
        offsets=(0, 0)):
    n_rows, vocab = logits.shape
    ws = torch.full((llmk.verify_drafts_workspace_floats(n_rows, n_seqs, vocab) + 4,),
                    float("nan"), device=DEV)
    ws[-4:] = 5.0
    n_accepted = torch.full((n_seqs,), -9, dtype=torch.int32, device=DEV)
    tokens = torch.full((n_rows,), -7, dtype=torch.int32, device=DEV)
    llmk.verify_drafts(
        at_offset(logits, offsets[0]),
        None if draft_logits is None else at_offset(draft_logits, offsets[1]), dev(drafts),
        dev(starts), dev(temperature), dev(accept_u), dev(sample_u), n_accepted, tokens, ws, n_rows,
        n_seqs, vocab)
    torch.cuda.synchronize()
    assert bool((ws[-4:] == 5.0).all()), "a write past the workspace"
    return n_accepted.cpu().numpy(), tokens.cpu().numpy()


def case(seed, counts, vocab, drafted, slack=0, std=2.5, noise=0.5, temperature=None):
    rng = np.random.default_rng(seed)
    n_rows, n = int(np.sum(counts)) + slack, len(counts)
    logits = (rng.standard_normal((n_rows, vocab)) * std).astype(np.float16)
    hot = rng.integers(0, vocab, (n_rows, 4))
    np.put_along_axis(logits, hot, (rng.standard_normal((n_rows, 4)) + 8).astype(np.float16), 1)
    q = (logits + noise * rng.standard_normal((n_rows, vocab))).astype(np.float16)
    t = (0.5 + rng.random(n)).astype(np.float32) if temperature is None else temperature
    drafts = np.zeros(n_rows, np.int32)
    for r in range(n_rows):
        p = ref.softmax(q[r], 1.0)
        drafts[r] = rng.choice(vocab, p=p)
    starts = np.r_[0, np.cumsum(counts)].astype(np.int32)
    return (logits, q if drafted else None, drafts, starts, t,
            rng.random(n_rows, dtype=np.float32), rng.random(n, dtype=np.float32), n)


def check(llmk, c, offsets=(0, 0)):
    got, want = run(llmk, *c, offsets=offsets), ref.verify(*c)
    assert np.array_equal(got[0], want[0]), (got[0], want[0])
    assert np.array_equal(got[1], want[1]), (got[1], want[1])
    return got


@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 1001, 8185, 8192, 8193, 20000, 32001])
def test_drafts_against_the_definition(llmk, vocab, drafted):
    """Ragged rows, sequences of one row (no drafts) and of none, rows of nobody; vocabularies around
    the edges of vectors and chunks."""
    check(llmk, case(vocab, [1, 5, 0, 3, 2, 9, 1, 4], vocab, drafted, slack=2))


@pytest.mark.parametrize("offsets", [(1, 1), (3, 0), (0, 5), (7, 2)])
def test_logits_at_any_alignment(llmk, offsets):
    for vocab in (1000, 8191):
        check(llmk, case(vocab, [3, 2, 4], vocab, True), offsets)
        check(llmk, case(vocab, [3, 2, 4], vocab, False), offsets)


@pytest.mark.parametrize("std", [0.0, 0.5, 6.0])
def test_flat_and_peaked_rows(llmk, std):
    """Flat rows put a border every 10^-5 of the random number's range."""
    for seed in range(3):
        check(llmk, case(seed, [2, 3, 1, 4], 50001, seed % 2 == 0, std=std))


def test_sampling_without_drafts(llmk):
    """row_starts None: one row a sequence, a token each; temperature None is 1."""
    logits, _, _, _, _, _, u, _ = case(5, [1] * 20, 3001, False)
    c = (logits, None, None, None, None, None, u, 20)
    accepted, tokens = check(llmk, c)
    assert not accepted.any() and (tokens >= 0).all()


def test_greedy(llmk):
    """Temperatures that are 0, negative or NaN: argmax, the lowest of equals, drafts that are it."""
    t = np.array([0.0, -1.0, np.nan, 0.0, 1.0, 0.0], np.float32)
    c = list(case(6, [4, 4, 3, 2, 4, 1], 9000, True, temperature=t))
    logits, drafts = c[0], c[2]
    logits[2, [17, 4000, 8999]] = 60.0
    best = logits.astype(np.float32).argmax(1)
    for r in (0, 1, 2, 4, 8, 9):
        drafts[r] = best[r]
    accepted, tokens = check(llmk, c)
    assert accepted[0] == 3 and tokens[2] == 17
    c[1] = None
    check(llmk, c)


def test_random_numbers_at_their_ends(llmk):
    """0 accepts whatever has probability and draws the first place that has any weight; the largest
    float below 1 draws near the end, and 1 (outside the range) the last place with any."""
    for u in (0.0, np.nextafter(np.float32(1), np.float32(0)), 1.0):
        c = list(case(7, [3, 1, 2, 5], 9001, True))
        c[0][:, :50] = -np.inf
        c[0][:, 8500:] = -np.inf
        c[5][:] = u
        c[6][:] = u
        got = run(llmk, *c)
        if u < 1:
            want = ref.verify(*c)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        assert ((got[1] >= 50) & (got[1] < 8500) | (got[1] == -1) | (got[1] == c[2])).all()


def test_masked_infinite_and_nan_logits(llmk):
    """-inf and NaN have no probability, +inf shares all of it; rows of nothing give -1 and refuse
    their drafts; draft rows of nothing leave p."""
    c = list(case(8, [3, 3, 2, 2, 4], 10007, True))
    logits, q, drafts = c[0], c[1], c[2]
    logits[:, ::3] = -np.inf
    logits[:, 1::5] = np.nan
    logits[1, [5, 9999]] = np.inf
    logits[4] = -np.inf
    logits[6] = np.nan
    q[2] = -np.inf
    q[8] = -np.inf
    q[10, 4:9000] = np.nan
    drafts[10] = 10000
    check(llmk, c)
    c[4] = np.array([0.0, 0.0, 0.0, 0.0, 1.0], np.float32)
    check(llmk, c)
    c[1] = None
    check(llmk, c)


def test_drafts_outside_the_vocabulary_are_refused(llmk):
    c = list(case(9, [4, 3, 2], 5000, True))
    c[2][[0, 4, 7]] = [-1, 5000, 2 ** 31 - 1]
    c[5][:] = 0.0
    accepted, _ = check(llmk, c)
    assert list(accepted) == [0, 0, 0]
    c[1] = None
    check(llmk, c)


def test_a_certain_draft_that_is_all_there_is(llmk):
    """Refusing the only token with probability draws it after all; refusing one of two draws the
    other, however small it is."""
    c = list(case(10, [2, 2], 20000, False, temperature=np.array([1.0, 1.0], np.float32)))
    c[0][:] = -np.inf
    c[0][0, 777] = 3.0
    c[2][0] = 777
    c[0][2, 9000] = 30.0
    c[0][2, 19999] = -30.0
    c[2][2] = 9000
    c[0][[1, 3], 1] = 0.0
    c[5][:] = 1.0  # not below any probability
    accepted, tokens = check(llmk, c)
    assert list(accepted) == [0, 0] and tokens[0] == 777 and tokens[2] == 19999


def test_equal_distributions_accept_every_draft(llmk):
    c = list(case(11, [5, 4, 6], 30000, True, noise=0.0))
    accepted, _ = check(llmk, c)
    assert list(accepted) == [4, 3, 5]


def test_extreme_temperatures(llmk):
    t = np.array([1e-3, 1e-30, 100.0, 3e38, np.inf, 1e-45], np.float32)
    check(llmk, case(12, [3] * 6, 4000, True, temperature=t))
    check(llmk, case(12, [3] * 6, 4000, False, temperature=t))


def test_many_rows_of_one_sequence_and_many_sequences(llmk):
    check(llmk, case(13, [70], 700, True, noise=0.05))
    rng = np.random.default_rng(14)
    check(llmk, case(14, rng.integers(0, 4, 700), 33, True))


@pytest.mark.parametrize("drafted", [True, False])
def test_vocabularies_of_more_pieces_than_a_wave_has_lanes(llmk, drafted):
    """Tokens in the first pieces, behind the 64th, and the row's last; weights in a few places only."""
    vocab = 300001
    c = list(case(22, [2, 1, 3, 2, 1], vocab, drafted, std=1.0))
    for u in (0.0, 0.5, 0.97, np.nextafter(np.float32(1.0), np.float32(0.0))):
        c[6] = np.full(5, u, np.float32)
        check(llmk, c)
    c[0][:] = -np.inf
    c[0][:, [70000, 290000, 300000]] = np.array([1.0, 0.5, 2.0], np.float16)
    if drafted:
        c[1][:, [70000, 290000, 300000]] = np.array([9.0, 9.0, 8.0], np.float16)
    for u in (0.0, 0.4, 0.999):
        c[6] = np.full(5, u, np.float32)
        check(llmk, c)


def test_no_rows(llmk):
    """Sequences without a row in the call: nothing but zeros, and no workspace needed."""
    n_accepted = torch.full((5,), -9, dtype=torch.int32, device=DEV)
    none = torch.empty(0, dtype=torch.float16, device=DEV)
    llmk.verify_drafts(none, None, none.int(), torch.zeros(6, dtype=torch.int32, device=DEV), None,
                       none.float(), torch.zeros(5, device=DEV), n_accepted, none.int(),
                       none.float(), 0, 5, 100)
    torch.cuda.synchronize()
    assert not n_accepted.any()


def test_drafts_next_to_the_border(llmk):
    """Random numbers a few roundings of fp32 from p / q, on either side, over long rows: the
    comparison is that of 64 bits."""
    n, vocab = 12, 70001
    c = list(case(21, [2] * n, vocab, True, std=1.0))
    for drafted in (True, False):
        if not drafted:
            c[1] = None
        for s in range(n):
            r, d = 2 * s, int(c[2][2 * s])
            p = ref.softmax(c[0][r], float(c[4][s]))[d]
            q = ref.softmax(c[1][r], float(c[4][s]))[d] if drafted else 1.0
            if p >= q:  # the draft's probability is to be the smaller one
                c[2][r] = d = int((ref.softmax(c[0][r], 1.0) - (
                    ref.softmax(c[1][r], 1.0) if drafted else 1.0)).argmin())
                p = ref.softmax(c[0][r], float(c[4][s]))[d]
                q = ref.softmax(c[1][r], float(c[4][s]))[d] if drafted else 1.0
            u = np.float32(min(p / q, 0.999))
            for _ in range(abs(s - 6)):
                u = np.nextafter(u, np.float32(s > 6))
            c[5][r] = u
        check(llmk, c)


def test_graph_replays_with_other_numbers(llmk):
    """Captured once, replayed with other logits, numbers and rows, eager work in between."""
    a = case(15, [3, 1, 4, 2], 9000, True)
    n_rows, vocab = a[0].shape
    state = [dev(x) for x in a[:7]]
    ws = torch.zeros(llmk.verify_drafts_workspace_floats(n_rows, 4, vocab), device=DEV)
    n_accepted = torch.zeros(4, dtype=torch.int32, device=DEV)
    tokens = torch.zeros(n_rows, dtype=torch.int32, device=DEV)

    def step():
        llmk.verify_drafts(*state, n_accepted, tokens, ws, n_rows, 4, vocab)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for seed, counts in ((16, [1, 2, 3, 4]), (17, [4, 0, 5, 1]), (18, [3, 1, 4, 2]),
                         (19, [10, 0, 0, 0])):
        b = case(seed, counts, vocab, True)
        for x, y in zip(state, b):
            x.copy_(dev(y))
        tokens.fill_(-7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = ref.verify(*b)
        assert np.array_equal(n_accepted.cpu().numpy(), want[0]), seed
        assert np.array_equal(tokens.cpu().numpy(), want[1]), seed


def test_python_refusals(llmk):
    c = case(20, [2, 2], 100, True)
    args = [dev(x) for x in c[:7]]
    n_accepted = torch.zeros(2, dtype=torch.int32, device=DEV)
    tokens = torch.zeros(4, dtype=torch.int32, device=DEV)
    ws = torch.zeros(llmk.verify_drafts_workspace_floats(4, 2, 100), device=DEV)
    names = ("logits", "draft_logits", "drafts", "row_starts", "temperature", "accept_u",
             "sample_u")

    def call(n_rows=4, ws=ws, **kw):
        a = dict(zip(names, args)) | kw
        llmk.verify_drafts(*a.values(), n_accepted, tokens, ws, n_rows, 2, 100, check_indices=True)

    call()
    for bad, text in ((dict(n_rows=5), "elements"), (dict(ws=ws[:-1]), "workspace"),
                      (dict(drafts=args[2].long()), "int32"), (dict(drafts=None), "status"),
                      (dict(row_starts=None), "status"),
                      (dict(row_starts=dev(np.array([0, 3, 2], np.int32))), "row_starts"),
                      (dict(sample_u=args[6].cpu()), "CUDA")):
        with pytest.raises(llmk.LlmkError, match=text):
            call(**bad)
