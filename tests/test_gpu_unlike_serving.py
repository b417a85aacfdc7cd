"""Adapters, rotary layouts and shared pages together, as a server's step uses them: a beam search whose requests
have adapters and position scalings of their own, over one paged cache."""
import numpy as np
import pytest
import torch

import _unlike as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
HEADS, KV, DIM, ROT, PAGE, MAX_PAGES = 8, 2, 64, 32, 16, 4
HIDDEN, ENDS = 256, (HEADS * DIM, (HEADS + KV) * DIM, (HEADS + 2 * KV) * DIM)
OUT, ADAPTERS, RANK, BEAMS = ENDS[-1], 3, 16, 10


def half(rng, *shape, std=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float16)).to(DEV)


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


class Server:
    """What a server holds: weights, adapters, scalings, the pools, two sets of a batch's arrays."""

    def __init__(self, llmk, rng):
        self.llmk, self.blas = llmk, llmk.Blas()
        self.w = half(rng, OUT, HIDDEN, std=HIDDEN ** -0.5)
        self.a = half(rng, ADAPTERS, 3, RANK, HIDDEN, std=HIDDEN ** -0.5)
        self.b = half(rng, ADAPTERS, OUT, RANK, std=0.2)
        self.ranks, self.scales = i32([16, 8, 11]), torch.tensor([1.0, 2.0, -0.5], device=DEV)
        tables = [llmk.compute_rotary_inv_freq(k, ROT, 10000.0, 4.0, 16.0) for k in
                  (llmk.ROTARY_PLAIN, llmk.ROTARY_LINEAR, llmk.ROTARY_YARN)]
        self.inv = torch.tensor([t[0] for t in tables], device=DEV)
        self.turn = torch.tensor([t[1] for t in tables], device=DEV)
        self.num_pages = BEAMS * MAX_PAGES
        self.refs = i32(np.zeros(self.num_pages))
        self.k = torch.full((self.num_pages, PAGE, KV, DIM), float("nan"), dtype=torch.float16, device=DEV)
        self.v = self.k.clone()
        self.tables = [i32(np.full((BEAMS, MAX_PAGES), -1)) for _ in range(2)]
        self.lens = [i32(np.zeros(BEAMS)) for _ in range(2)]
        self.parents, self.one = i32(np.full(BEAMS, -1)), i32(np.ones(BEAMS))
        self.copies, self.counts = i32(np.zeros((BEAMS, 2))), i32([0, 0])
        self.fork_ws = i32(np.zeros(llmk.kv_fork_workspace_ints(BEAMS, BEAMS, MAX_PAGES, self.num_pages)))
        self.lora_ws = torch.empty(llmk.lora_add_workspace_floats(BEAMS, BEAMS, ADAPTERS, RANK, HIDDEN, 3),
                                   device=DEV)
        self.att_ws = torch.empty(llmk.attention_decode_fast_workspace_floats(BEAMS, HEADS, 2), device=DEV)
        self.x = half(rng, BEAMS, HIDDEN)
        self.ids, self.base = i32(np.zeros(BEAMS)), torch.empty(BEAMS, OUT, dtype=torch.float16, device=DEV)
        self.qkv = torch.empty_like(self.base)
        self.q = torch.empty(BEAMS, HEADS, DIM, dtype=torch.float16, device=DEV)
        self.out = torch.empty_like(self.q)

    def step(self, now):
        """The children take over, then each writes its token's row and attends."""
        L, old, new = self.llmk, self.tables[1 - now], self.tables[now]
        L.kv_fork(old, self.lens[1 - now], self.parents, self.one, self.refs, new, self.lens[now], self.copies,
                  self.counts, self.fork_ws, BEAMS, BEAMS, MAX_PAGES, PAGE, self.num_pages)
        L.kv_copy_pages([self.k, self.v], self.copies, None, BEAMS, self.num_pages)
        L.linear(self.blas, self.x, self.w, self.base, BEAMS, HIDDEN, OUT)
        self.qkv.copy_(self.base)
        L.lora_add(self.x, HIDDEN, self.a, self.b, self.ranks, self.scales, self.ids, None, self.qkv, OUT, ENDS,
                   self.lora_ws, BEAMS, BEAMS, ADAPTERS, RANK, HIDDEN)
        L.qkv_rotary_scatter(self.qkv, OUT, self.q, self.k, self.v, new, self.lens[now], self.inv, self.ids,
                             self.turn, BEAMS, MAX_PAGES, PAGE, HEADS, KV, DIM, ROT, L.ROTARY_PAIRS)
        self.lens[now] += 1
        L.attention_decode_fast(self.q, self.k, self.v, new, self.lens[now], self.out, self.att_ws, BEAMS,
                                MAX_PAGES, PAGE, HEADS, KV, DIM, 2)


@pytest.mark.parametrize("captured", [False, True])
def test_a_search_with_adapters(llmk, captured):
    rng = np.random.default_rng(31)
    s = Server(llmk, rng)
    graphs = []
    if captured:
        s.step(0)  # the library product's plan is made outside of a capture
        torch.cuda.synchronize()
        for now in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                s.step(now)
            graphs.append(g)
        for t, value in ((s.tables[0], -1), (s.tables[1], -1), (s.lens[0], 0), (s.lens[1], 0), (s.refs, 0)):
            t.fill_(value)
    ids = rng.integers(-1, ADAPTERS, BEAMS)
    text = [[] for _ in range(BEAMS)]  # (k, v) rows of each beam's tokens
    inv, turn = s.inv.cpu().numpy(), s.turn.cpu().numpy()
    for t in range(PAGE * MAX_PAGES - 3):
        now = t % 2
        parents = np.sort(rng.integers(0, BEAMS, BEAMS)) if t else np.full(BEAMS, -1)
        if t % 9 == 8:
            parents[rng.integers(0, BEAMS, 2)] = -1  # two leave, two begin
        ids = np.where(parents >= 0, ids[parents], rng.integers(-1, ADAPTERS, BEAMS))
        s.parents.copy_(i32(parents))
        s.ids.copy_(i32(ids))
        s.x.copy_(half(rng, BEAMS, HIDDEN))
        graphs[now].replay() if captured else s.step(now)
        torch.cuda.synchronize()
        assert s.counts[1].item() == 0
        text = [list(text[p]) if p >= 0 else [] for p in parents]
        lens = np.array([len(r) for r in text])
        assert np.array_equal(s.lens[now].cpu().numpy(), lens + 1)

        x, base, qkv = (u.cpu().numpy() for u in (s.x, s.base, s.qkv))
        want, bound = ref.lora_add(x, s.a.cpu().numpy(), s.b.cpu().numpy(), s.ranks.cpu().numpy(),
                                   s.scales.cpu().numpy(), ids, None, base, ENDS)
        assert (np.abs(qkv - want) <= bound).all()
        rows = qkv.reshape(BEAMS, -1, DIM)
        want, bound = ref.rotate(rows[:, :HEADS + KV], lens, inv, ids, turn, ROT, True)
        bound[..., ROT:] = 0.0
        q = s.q.cpu().numpy()
        assert (np.abs(q - want[:, :HEADS]) <= bound[:, :HEADS]).all()

        tables, k, v = s.tables[now].cpu().numpy(), s.k.cpu().numpy(), s.v.cpu().numpy()
        refs = np.bincount(np.concatenate([ref.held(r, s.num_pages) for r in tables]), minlength=s.num_pages)
        assert np.array_equal(refs, s.refs.cpu().numpy())
        out = s.out.cpu().numpy().astype(np.float64)
        for c in range(BEAMS):
            page, slot = tables[c, lens[c] // PAGE], lens[c] % PAGE
            assert (np.abs(k[page, slot] - want[c, HEADS:]) <= bound[c, HEADS:]).all()
            assert np.array_equal(v[page, slot], rows[c, HEADS + KV:])
            text[c].append((k[page, slot].copy(), v[page, slot].copy()))
            # the cache holds the beam's own tokens, to the bit, and attention is over them
            at = np.arange(len(text[c]))
            mine = k[tables[c, at // PAGE], at % PAGE], v[tables[c, at // PAGE], at % PAGE]
            for got, i in zip(mine, range(2)):
                assert np.array_equal(got, np.stack([r[i] for r in text[c]]))
            kk, vv = (np.repeat(m.astype(np.float64), HEADS // KV, 1) for m in mine)
            score = np.einsum("hd,jhd->hj", q[c].astype(np.float64), kk) / np.sqrt(DIM)
            w = np.exp(score - score.max(1, keepdims=True))
            e = np.einsum("hj,jhd->hd", w / w.sum(1, keepdims=True), vv)
            assert (np.abs(out[c] - e) <= 1e-3 + 4e-3 * np.abs(e)).all()  # the reference's rule


def test_two_calls_at_once(llmk):
    """Two streams with a workspace each: neither disturbs the other."""
    rng = np.random.default_rng(32)
    n, inner, out, rank, k = 70, 4096, 2048, 64, 9
    a, b = half(rng, k, 1, rank, inner, std=inner ** -0.5), half(rng, k, out, rank, std=0.1)
    x = [half(rng, n, inner) for _ in range(2)]
    y = [half(rng, n, out) for _ in range(2)]
    ids = [i32(rng.integers(-1, k, n)) for _ in range(2)]
    ws = [torch.empty(llmk.lora_add_workspace_floats(n, n, k, rank, inner, 1), device=DEV) for _ in range(2)]

    def call(i, to, stream=None):
        llmk.lora_add(x[i], inner, a, b, None, None, ids[i], None, to, out, (out,), ws[i], n, n, k, rank, inner,
                      stream=stream)
    want = [t.clone() for t in y]
    for i in range(2):
        call(i, want[i])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = [t.clone() for t in y]
        torch.cuda.synchronize()
        for i in range(2):
            call(i, got[i], streams[i].cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_cache_is_compacted_between_steps(llmk):
    """Sequences over an 8-bit cache leave, the rest are compacted, and what they attend to is the same."""
    rng = np.random.default_rng(33)
    n, max_pages = 12, 6
    tables, lens, refs, num_pages = ref.batch(rng, n, 2, 90, 16, max_pages, tails=False, spare=10)
    lens = np.maximum(lens, 1)
    pool = [torch.randn(num_pages, KV, 16, DIM, device=DEV).to(torch.float8_e4m3fn) for _ in range(2)]
    scale = [torch.exp2(torch.randint(-3, 3, (num_pages, KV), device=DEV).float()) for _ in range(2)]
    q = half(rng, n, HEADS, DIM)
    dt, dl, dr = i32(tables.reshape(-1)), i32(lens), i32(refs)
    keep = np.flatnonzero(rng.random(n) < 0.6)
    new_t, new_l = i32(np.zeros(n * max_pages)), i32(np.zeros(n))
    copies, counts = i32(np.zeros(2 * max(n, num_pages // 2))), i32([0, 0])
    m = len(keep)

    def attend(t, rows, query):
        out = torch.empty_like(query)
        llmk.kv8_attention(query, pool[0], scale[0], pool[1], scale[1], t, None, rows, out, None, m, m, 1,
                           max_pages, 16, HEADS, KV, DIM)
        return out
    ws = i32(np.zeros(llmk.kv_fork_workspace_ints(n, m, max_pages, num_pages)))
    llmk.kv_fork(dt, dl, i32(keep), None, dr, new_t, new_l, copies, counts, ws, n, m, max_pages, 16, num_pages)
    assert counts.tolist() == [0, 0] and (copies[:2 * m] == -1).all()
    query = q[torch.from_numpy(keep).to(DEV)].contiguous()
    # a sequence of no tokens holds no page: its only entry names none and is not read
    lens_now = new_l[:m].clone()
    before = attend(new_t, lens_now, query)
    ws = i32(np.zeros(llmk.kv_compact_workspace_ints(num_pages)))
    llmk.kv_compact(new_t, dr, new_t, dr, copies, counts, ws, m, max_pages, num_pages)
    llmk.kv_copy_pages(pool + scale, copies, counts, num_pages // 2, num_pages)
    live = counts[1].item()
    for t in pool + scale:  # the pools may be cut behind them
        t.view(torch.uint8)[live:] = 0x7F
    assert torch.equal(before, attend(new_t, lens_now, query)) and new_t[:m * max_pages].max().item() < live
