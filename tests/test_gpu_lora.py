"""Adapters beside a shared projection on the GPU against their definition in 64 bits."""
import numpy as np
import pytest
import torch

import _unlike as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def half(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.float16)).to(DEV)


def i32(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def f32(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(DEV)


class Case:
    """Inputs of one call. rows: of each sequence (None: one each); ids: of each sequence. Rows behind the
    last sequence, columns behind the last part, ranks behind an adapter's and adapters that nobody has hold
    NaN or numbers that would show."""

    def __init__(self, rng, ids, rows, adapters, rank, inner, ends, ranks=None, scales=True, behind=0,
                 padx=0, pady=0, whole=False):
        self.ids, self.ends, self.rank, self.inner = np.asarray(ids), tuple(ends), rank, inner
        n = self.ids.size
        self.starts = None if rows is None else np.concatenate([[0], np.cumsum(rows)])
        self.n_rows = (n if rows is None else int(self.starts[-1])) + (behind if rows is not None else 0)
        self.n_seqs, self.adapters, out = n, adapters, ends[-1]
        self.ldx, self.ldy = inner + padx, out + pady
        if whole:  # numbers whose sums are exact
            self.x = rng.integers(-8, 9, (self.n_rows, self.ldx))
            self.a = rng.integers(-4, 5, (adapters, len(ends), rank, inner))
            self.b = rng.integers(-3, 4, (adapters, out, rank))
            self.y = rng.integers(-2000, 2001, (self.n_rows, self.ldy))
        else:
            self.x = rng.standard_normal((self.n_rows, self.ldx))
            self.a = rng.standard_normal((adapters, len(ends), rank, inner)) * inner ** -0.5
            self.b = rng.standard_normal((adapters, out, rank)) * rank ** -0.5
            self.y = rng.standard_normal((self.n_rows, self.ldy))
        self.x, self.a, self.b, self.y = (t.astype(np.float16) for t in (self.x, self.a, self.b, self.y))
        self.ranks = None if ranks is None else np.asarray(ranks)
        self.scales = None
        if scales:
            self.scales = rng.choice([0.5, 1.0, 2.0], adapters) if whole else rng.uniform(-2, 2, adapters)
            self.scales = self.scales.astype(np.float32)
        self.x[:, inner:] = np.nan
        for k in range(adapters):
            r = rank if ranks is None else max(0, int(ranks[k]))
            self.a[k, :, r:] = np.nan
            self.b[k, :, r:] = np.inf
            if not (self.ids == k).any():
                self.a[k], self.b[k] = np.nan, np.nan

    def want(self):
        w, bound = ref.lora_add(self.x[:, :self.inner], self.a, self.b, self.ranks, self.scales, self.ids,
                                self.starts, self.y[:, :self.ends[-1]], self.ends)
        return w, bound

    def has(self):
        """Rows that an adapter is added to."""
        on = np.zeros(self.n_rows, bool)
        for s, k in enumerate(self.ids):
            if 0 <= k < self.adapters and (self.ranks is None or self.ranks[k] > 0):
                r0, r1 = (s, s + 1) if self.starts is None else self.starts[s:s + 2]
                on[r0:r1] = True
        return on

    def upload(self, llmk):
        floats = llmk.lora_add_workspace_floats(self.n_rows, self.n_seqs, self.adapters, self.rank,
                                                self.inner, len(self.ends))
        self.ws = torch.full((floats + 64,), float("nan"), device=DEV)
        self.t = dict(x=half(self.x), a=half(self.a), b=half(self.b), ranks=i32(self.ranks),
                      scales=f32(self.scales), ids=i32(self.ids), starts=i32(self.starts))
        self.floats = floats
        return half(self.y)

    def call(self, llmk, y, **kw):
        t = self.t
        llmk.lora_add(t["x"], self.ldx, t["a"], t["b"], t["ranks"], t["scales"], t["ids"], t["starts"], y,
                      self.ldy, self.ends, self.ws, self.n_rows, self.n_seqs, self.adapters, self.rank,
                      self.inner, **kw)

    def check(self, llmk, exact=False):
        y = self.upload(llmk)
        self.call(llmk, y, check_indices=True)
        got = y.cpu().numpy()
        out, on = self.ends[-1], self.has()
        same = got.view(np.uint16) == self.y.view(np.uint16)
        assert same[:, out:].all(), "columns behind the last part were written"
        assert same[~on].all(), "rows of no adapter were written"
        assert torch.isnan(self.ws[self.floats:]).all(), "write past the workspace"
        want, bound = self.want()
        if exact:
            with np.errstate(over="ignore"):
                assert np.array_equal(got[on, :out], want[on].astype(np.float16))
        else:
            off = np.abs(got[:, :out].astype(np.float64) - want)
            assert (off <= bound)[on].all(), (off / bound)[on].max()
        again = half(self.y)
        self.call(llmk, again)
        assert torch.equal(y.view(torch.int16), again.view(torch.int16)), "two calls differ"


def ids_of(rng, n, adapters, none=0.15):
    ids = rng.integers(0, adapters, n)
    return np.where(rng.random(n) < none, rng.choice([-1, adapters, 2 ** 31 - 1, -2 ** 31], n), ids)


@pytest.mark.parametrize("inner", [8, 16, 24, 40, 64, 136, 256, 512, 520, 1000, 2048, 4104, 8192])
@pytest.mark.parametrize("rank", [8, 16, 24, 64])
def test_widths_and_ranks(llmk, inner, rank):
    rng = np.random.default_rng([inner, rank])
    Case(rng, ids_of(rng, 7, 3), None, 3, rank, inner, (48, 72)).check(llmk)
    Case(rng, ids_of(rng, 5, 2), rng.integers(0, 30, 5), 2, rank, inner, (40,), behind=3).check(llmk)


@pytest.mark.parametrize("n,rows,adapters,rank,inner,ends", [
    (2, 64, 1, 16, 264, (4096, 5120, 6144)), (2, 150, 1, 16, 72, (4096, 5120, 6144)), (2, 100, 1, 32, 72, (11008, 22016)),
    (1, 500, 3, 8, 264, (2048,)), (2, 400, 1, 24, 72, (2560, 5120, 7680)), (12, 10, 48, 16, 72, (8192, 16384)),
    (24, 6, 96, 16, 72, (2048,)), (48, 5, 16, 16, 520, (4096, 5120, 6144)), (80, 2, 300, 8, 72, (4096, 5120, 6144)),
    (8, 1, 16, 16, 8192, (4096, 5120, 6144)), (16, 1, 32, 16, 6152, (1000,)), (1, 16, 8, 16, 8192, (2048,)),
    (700, 1, 40, 16, 136, (1024,)), (30, 3, 30, 32, 2056, (4096,))])
def test_batches_around_one_launch(llmk, n, rows, adapters, rank, inner, ends):
    """By the sizes some go in one launch and some in two, with 256, 512 or 1024 columns a block."""
    rng = np.random.default_rng([n, rows, adapters, rank])
    for same in (False, True):  # adapters as they fall, and the same for all: more tiles, and fewer, than expected
        ids = np.full(n, adapters - 1) if same else rng.permutation(max(n, adapters))[:n] % adapters
        Case(rng, ids, rng.integers(1, rows + 1, n) if rows > 1 else None, adapters, rank, inner, ends).check(llmk)


def test_columns_of_one_matrix(llmk):
    rng = np.random.default_rng(11)
    c = Case(rng, ids_of(rng, 6, 3), rng.integers(0, 9, 6), 3, 16, 136, (24, 72))
    y = c.upload(llmk)
    for first in (True, False):  # x in front of y, and behind it
        m = torch.full((c.n_rows, 136 + 72 + 24), 5.0, dtype=torch.float16, device=DEV)
        x, out = (m[:, :136], m[:, 144:216]) if first else (m[:, 88:224], m[:, 8:80])
        x.copy_(c.t["x"][:, :136])
        out.copy_(y[:, :72])
        llmk.lora_add(x, m.shape[1], c.t["a"], c.t["b"], c.t["ranks"], c.t["scales"], c.t["ids"], c.t["starts"], out,
                      m.shape[1], (24, 72), c.ws, c.n_rows, 6, 3, 16, 136)
        want = y.clone()
        c.call(llmk, want)
        assert torch.equal(out, want[:, :72]) and torch.equal(x, c.t["x"][:, :136])
        with pytest.raises(llmk.LlmkError):
            llmk.lora_add(x, m.shape[1], c.t["a"], c.t["b"], c.t["ranks"], c.t["scales"], c.t["ids"], c.t["starts"],
                          x[:, :72], m.shape[1], (24, 72), c.ws, c.n_rows, 6, 3, 16, 136)


@pytest.mark.parametrize("ends", [(8,), (16,), (24,), (64,), (72,), (264,), (1000,), (2048,), (8, 16), (16, 24, 32),
                                  (520, 584, 648), (32, 64, 96, 128, 160, 168, 176, 184), (8, 2056)])
@pytest.mark.parametrize("rank", [8, 16, 32, 136, 256])
def test_parts_and_ranks(llmk, ends, rank):
    rng = np.random.default_rng([sum(ends), rank])
    Case(rng, ids_of(rng, 9, 4), rng.integers(0, 7, 9), 4, rank, 64, ends,
         ranks=rng.integers(1, rank + 1, 4)).check(llmk)


@pytest.mark.parametrize("n,adapters,rank,ends", [
    (1, 1, 16, (16384,)), (1, 2, 32, (11008, 22016)), (3, 3, 8, (16384,)), (9, 4, 24, (8192, 16384)),
    (20, 16, 16, (6144,)), (40, 20, 16, (16384,)), (100, 3, 32, (4096, 5120, 6144)), (64, 1, 64, (16384,)),
    (30, 7, 128, (8192,)), (17, 5, 256, (2504, 5000))])
def test_wide_projections(llmk, n, adapters, rank, ends):
    """Few columns a block and many, a tile's blocks together and spread, few and many tiles a block."""
    rng = np.random.default_rng([n, ends[-1]])
    Case(rng, ids_of(rng, n, adapters), None, adapters, rank, 264, ends).check(llmk)
    rows = rng.integers(0, 60, n) if n <= 40 else rng.integers(0, 9, n)
    Case(rng, ids_of(rng, n, adapters, 0.05), rows, adapters, rank, 2048 if n < 30 else 1032, ends,
         ranks=rng.integers(1, rank + 1, adapters), behind=2).check(llmk)


@pytest.mark.parametrize("rows", [1, 2, 7, 15, 16, 17, 31, 33, 64, 65, 130, 257, 700])
def test_one_sequence(llmk, rows):
    rng = np.random.default_rng(rows)
    Case(rng, [0], [rows], 1, 16, 128, (136,), behind=2).check(llmk)
    Case(rng, [1], [rows], 2, 24, 264, (64, 128, 168), ranks=[3, 17], padx=8, pady=16).check(llmk)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 128, 200, 255, 256, 257, 300, 513, 1030])
@pytest.mark.parametrize("adapters", [1, 5, 400])
def test_one_row_each(llmk, n, adapters):
    rng = np.random.default_rng([n, adapters])
    Case(rng, ids_of(rng, n, adapters), None, adapters, 8, 72, (40,)).check(llmk)


@pytest.mark.parametrize("n,most", [(3, 200), (20, 40), (100, 9), (256, 5), (300, 4), (600, 3), (40, 100)])
def test_ragged_batches(llmk, n, most):
    """Sequences of unlike lengths, some without rows, adapters shared among them."""
    rng = np.random.default_rng([n, most])
    rows = rng.integers(0, most + 1, n)
    for adapters in (1, 4, 50):
        Case(rng, ids_of(rng, n, adapters), rows, adapters, 16, 136, (72, 104),
             ranks=rng.integers(-1, 17, adapters), behind=5, padx=16, pady=8).check(llmk)


@pytest.mark.parametrize("seed", range(12))
def test_drawn(llmk, seed):
    rng = np.random.default_rng(900 + seed)
    n, adapters = int(rng.integers(1, 40)), int(rng.integers(1, 20))
    rank = 8 * int(rng.integers(1, 17))
    ends = np.cumsum(8 * rng.integers(1, 100, int(rng.integers(1, 5))))
    Case(rng, ids_of(rng, n, adapters), None if seed % 2 else rng.integers(0, 25, n), adapters, rank,
         8 * int(rng.integers(1, 300)), [int(e) for e in ends],
         ranks=rng.integers(0, rank + 1, adapters) if seed % 3 else None, scales=seed % 4 > 0).check(llmk)


@pytest.mark.parametrize("rows,inner,rank", [(1, 2048, 16), (5, 512, 64), (40, 2048, 16), (300, 256, 8),
                                             (64, 4096, 128), (3, 8192, 256)])
def test_values_between_the_products_keep_their_bits(llmk, rows, inner, rank):
    """Whole numbers: |h| <= 32 * inner <= 2^18, which 22 bits hold, and sums below 2^24 are exact in fp32. So the
    result is the definition's, rounded once; a value held in 11 bits in between would show."""
    rng = np.random.default_rng([rows, inner, rank])
    c = Case(rng, [0, 1], [rows, rows], 2, rank, inner, (48, 112), whole=True)
    h = np.abs(np.einsum("ri,kpji->rkpj", c.x[:, :inner].astype(np.float64), c.a.astype(np.float64)))
    assert h.max() * 3 * rank < 2 ** 24  # of the whole sums
    assert h.max() > 2 ** 7
    c.check(llmk, exact=True)


def test_infinities_and_nan_stay_in_their_rows(llmk):
    rng = np.random.default_rng(11)
    for rows in (1, 3, 40):
        c = Case(rng, [0, 1, 0], [rows, rows, rows], 2, 16, 256, (64, 128))
        clean, _ = c.want()
        bad = [0, rows + rows // 2]
        c.x[bad[0], 5], c.x[bad[1], 200] = np.inf, np.nan
        y = c.upload(llmk)
        c.call(llmk, y)
        got = y.cpu().numpy().astype(np.float64)
        want, bound = c.want()
        good = np.setdiff1d(np.arange(3 * rows), bad)
        assert (np.abs(got - want) <= bound)[good].all()
        for r in bad:
            assert np.array_equal(np.isnan(got[r]), np.isnan(want[r]))
            inf = np.isinf(want[r])
            assert np.array_equal(got[r][inf], want[r][inf])


def test_magnitudes(llmk):
    """Values between the products past what fp16 holds, and subnormal ones."""
    rng = np.random.default_rng(12)
    for up, down in ((1000.0, 1e-4), (1e-4, 1.0), (60000.0, 6e-8), (6e-8, 60000.0)):
        c = Case(rng, [0, 1], [20, 1], 2, 16, 512, (128,), scales=False)
        c.x = (c.x * np.float32(up)).clip(-65000, 65000).astype(np.float16)
        c.b = (c.b * np.float32(down)).astype(np.float16)
        c.y = (c.y * np.float32(min(1.0, up * down))).astype(np.float16)
        c.check(llmk)


def test_captured_and_replayed(llmk):
    """One graph serves batches whose ids, lengths and values change; two graphs share a workspace."""
    rng = np.random.default_rng(13)
    c = Case(rng, ids_of(rng, 12, 4), rng.integers(0, 20, 12), 4, 16, 264, (64, 136), behind=20)
    d = Case(rng, ids_of(rng, 12, 4), None, 4, 16, 264, (64, 136))
    for case in (c, d):
        case.y_in = case.upload(llmk)
    if d.floats > c.floats:
        c.ws = d.ws
    d.ws = c.ws
    graphs = []
    for case in (c, d):
        case.call(llmk, case.y_in.clone())
        torch.cuda.synchronize()
        case.y_dev = case.y_in.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            case.call(llmk, case.y_dev)
        graphs.append(g)
    for replay in range(4):
        for case, g in zip((c, d), graphs):
            case.ids = ids_of(rng, 12, 4)
            case.a[:], case.b[:] = rng.standard_normal(case.a.shape), rng.standard_normal(case.b.shape)
            case.t["ids"].copy_(i32(case.ids))
            case.t["a"].copy_(half(case.a))
            case.t["b"].copy_(half(case.b))
            if case.starts is not None:
                rows = rng.integers(0, 20, 12)
                rows[3] += case.n_rows - 20 - rows.sum() if rows.sum() < case.n_rows - 20 else 0
                rows = np.minimum(rows, (case.n_rows // 12))
                case.starts = np.concatenate([[0], np.cumsum(rows)])
                case.t["starts"].copy_(i32(case.starts))
            case.y_dev.copy_(case.y_in)
            g.replay()
            torch.cuda.synchronize()
            want, bound = case.want()
            got = case.y_dev.cpu().numpy()[:, :136]
            on = case.has()
            assert (np.abs(got.astype(np.float64) - want) <= bound)[on].all()
            assert np.array_equal(got[~on].view(np.uint16), case.y[~on][:, :136].view(np.uint16))


def test_on_another_stream(llmk):
    rng = np.random.default_rng(14)
    c = Case(rng, ids_of(rng, 30, 5), None, 5, 32, 1024, (512,))
    y = c.upload(llmk)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.call(llmk, y)
    other = half(c.y)
    s.synchronize()
    c.call(llmk, other, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(y, other)
    want, bound = c.want()
    assert (np.abs(y.cpu().numpy().astype(np.float64) - want) <= bound)[c.has()].all()


def test_offsets_past_32_bits(llmk):
    """Rows of x and y and an adapter's weights whose bytes lie past 2^32."""
    rng = np.random.default_rng(16)
    n, ldx, ldy, inner = 40000, 65536, 65536, 16384
    x = torch.zeros(n, ldx, dtype=torch.float16, device=DEV)
    y = torch.zeros(n, ldy, dtype=torch.float16, device=DEV)
    a = torch.zeros(710, 1, 256, inner, dtype=torch.float16, device=DEV)  # 8 MiB each
    b = torch.zeros(710, 64, 256, dtype=torch.float16, device=DEV)
    row, rank = n - 3, 5
    x[row, :inner], y[row, :64] = half(rng.standard_normal(inner)), half(rng.standard_normal(64))
    a[709, 0, :rank] = half(rng.standard_normal((rank, inner)) * inner ** -0.5)
    b[709, :, :rank] = half(rng.standard_normal((64, rank)))
    ids = torch.full((n,), -1, dtype=torch.int32, device=DEV)
    ids[row] = 709
    ranks = torch.full((710,), rank, dtype=torch.int32, device=DEV)
    want, bound = ref.lora_add(x[row:row + 1, :inner].cpu().numpy(), a[709:].cpu().numpy(), b[709:].cpu().numpy(),
                               np.array([rank]), None, [0], None, y[row:row + 1, :64].cpu().numpy(), (64,))
    ws = torch.empty(llmk.lora_add_workspace_floats(n, n, 710, 256, inner, 1), device=DEV)
    llmk.lora_add(x, ldx, a, b, ranks, None, ids, None, y, ldy, (64,), ws, n, n, 710, 256, inner)
    got = y[row, :64].cpu().numpy().astype(np.float64)
    assert (np.abs(got - want[0]) <= bound[0]).all()
    y[row, :64] = 0
    assert not y.any()


def test_columns_of_wider_tensors(llmk):
    """x and y as views of columns: what lies beside them stays."""
    rng = np.random.default_rng(15)
    c = Case(rng, [0, 1, -1, 1], None, 2, 16, 128, (64,), padx=64, pady=32)
    c.upload(llmk)
    wide_x = torch.full((4, 320), float("nan"), dtype=torch.float16, device=DEV)
    wide_x[:, 64:192] = half(c.x[:, :128])
    wide_y = torch.full((4, 160), 7.0, dtype=torch.float16, device=DEV)
    wide_y[:, 32:96] = half(c.y[:, :64])
    t = c.t
    llmk.lora_add(wide_x[:, 64:192], 320, t["a"], t["b"], None, t["scales"], t["ids"], None,
                  wide_y[:, 32:96], 160, (64,), c.ws, 4, 4, 2, 16, 128)
    want, bound = c.want()
    got = wide_y.cpu().numpy().astype(np.float64)
    assert (got[:, :32] == 7).all() and (got[:, 96:] == 7).all()
    assert (np.abs(got[:, 32:96] - want) <= bound).all()


def test_python_refusals(llmk):
    h = torch.zeros(64, 64, dtype=torch.float16, device=DEV)
    i, f = torch.zeros(64, dtype=torch.int32, device=DEV), torch.zeros(1 << 16, device=DEV)

    def call(**kw):
        a = dict(x=h, ldx=64, a=h, b=h, ranks=None, scales=None, ids=i, starts=None, y=h, ldy=64, ends=(64,),
                 ws=f, n_rows=2, n_seqs=2, n_adapters=1, rank=8, inner=64) | kw
        llmk.lora_add(*a.values(), check_indices=True)

    call(y=torch.zeros_like(h))
    for bad in (dict(x=h[:, :32]), dict(x=h.float()), dict(x=h.t()), dict(x=h[:, ::2], ldx=64, inner=32),
                dict(x=h[:1]), dict(ldx=32, inner=32), dict(y=h[:, :56]), dict(a=h[:4]), dict(b=h[:4]),
                dict(ids=i.long()), dict(ids=i[:1]), dict(scales=f.double()), dict(ws=f[:1]), dict(ends=()),
                dict(ends=(0,)), dict(starts=i[:2]), dict(starts=i + 1), dict(ranks=i + 9),
                dict(starts=torch.tensor([0, 3, 2], dtype=torch.int32, device=DEV)),
                dict(starts=torch.tensor([0, 1, 3], dtype=torch.int32, device=DEV)), dict(n_rows=-1)):
        with pytest.raises(llmk.LlmkError):
            call(**bad)
