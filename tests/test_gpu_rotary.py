"""Rotary layouts, parts of a head and scalings on the GPU against their definition in 64 bits."""
import numpy as np
import pytest
import torch

import _unlike as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def to(a, dtype):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a, dtype)).to(DEV)


def tables(rng, n, rotary, n_tables, ids=True, scales=True):
    half = rotary // 2
    inv = (500000.0 ** (-np.arange(half) / half) / rng.uniform(1, 8, (n_tables, 1))).astype(np.float32)
    return (inv, rng.integers(-1, n_tables + 1, n) if ids else None,
            rng.uniform(0.5, 1.5, n_tables).astype(np.float32) if scales else None)


def positions(rng, n):
    p = rng.integers(0, 131072, n)
    p[:1] = 0
    if n > 4:
        p[1:5] = [2 ** 31 - 1, -2 ** 31, -1, 1000003]
    return p


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("n,heads,kv,dim,rotary", [
    (1, 32, 8, 64, 64), (5, 4, 2, 128, 32), (17, 3, 1, 80, 80), (33, 2, 2, 256, 128), (2, 1, 1, 2, 2),
    (7, 5, 0, 64, 48), (7, 0, 3, 64, 16), (9, 3, 2, 20, 6), (600, 4, 1, 64, 64), (1100, 2, 1, 32, 16),
    (3, 2, 1, 4096, 4096), (6, 2, 2, 24, 8), (4, 6, 2, 96, 24), (2100, 8, 2, 128, 128), (40, 1, 1, 513, 512)])
def test_in_place(llmk, pairs, n, heads, kv, dim, rotary):
    rng = np.random.default_rng([n, heads, dim, rotary])
    for ids, scales, pad in ((False, False, 0), (True, True, 8), (True, False, 3)):
        inv, t, s = tables(rng, n, rotary, 3 if ids else 1, ids, scales)
        pos, ld = positions(rng, n), (heads + kv) * dim + pad
        x = rng.standard_normal((n, ld)).astype(np.float16)
        d = to(x, np.float16)
        llmk.rotary_apply(d, ld, d[:, heads * dim:], ld, to(pos, np.int32), to(inv, np.float32),
                          to(t, np.int32), to(s, np.float32), n, heads, kv, dim, rotary,
                          llmk.ROTARY_PAIRS if pairs else llmk.ROTARY_HALVES)
        got = d.cpu().numpy()
        width = (heads + kv) * dim
        want, bound = ref.rotate(x[:, :width].reshape(n, -1, dim), pos, inv, t, s, rotary, pairs)
        y = got[:, :width].reshape(n, -1, dim)
        assert (np.abs(y.astype(np.float64) - want) <= bound)[..., :rotary].all()
        assert np.array_equal(got[:, width:].view(np.uint16), x[:, width:].view(np.uint16))
        assert np.array_equal(y[..., rotary:].view(np.uint16),
                              x[:, :width].reshape(n, -1, dim)[..., rotary:].view(np.uint16))


def test_separate_tensors_and_odd_addresses(llmk):
    """q and k in tensors of their own; q at an address that is no multiple of 16."""
    rng = np.random.default_rng(3)
    n, heads, kv, dim = 6, 4, 2, 64
    inv, t, s = tables(rng, n, dim, 2)
    pos = positions(rng, n)
    q, k = (rng.standard_normal((n, h, dim)).astype(np.float16) for h in (heads, kv))
    for shift in (0, 1, 4):
        flat = torch.zeros(q.size + 16, dtype=torch.float16, device=DEV)
        dq = flat[shift:shift + q.size]
        dq.copy_(to(q.reshape(-1), np.float16))
        dk = to(k, np.float16)
        llmk.rotary_apply(dq, heads * dim, dk, kv * dim, to(pos, np.int32), to(inv, np.float32),
                          to(t, np.int32), to(s, np.float32), n, heads, kv, dim, dim, check_indices=False)
        for got, x in ((dq, q), (dk, k)):
            want, bound = ref.rotate(x, pos, inv, t, s, dim, False)
            off = np.abs(got.cpu().numpy().reshape(x.shape).astype(np.float64) - want)
            assert (off <= bound).all()
        assert (flat[shift + q.size:] == 0).all() and (flat[:shift] == 0).all()


def test_as_the_plain_rotation(llmk):
    """Whole heads as halves, one table: within what llmk_rope_apply's fp16 steps are off by (two products,
    a cosine and a sine each rounded to 2^-11 of at most |x|, and the two sums' last rounding)."""
    rng = np.random.default_rng(4)
    n, heads, kv, dim = 50, 32, 8, 64
    inv = to(llmk.compute_rope_inv_freq(dim, 500000.0, 32.0, 1.0, 4.0, 8192.0), np.float32)
    pos = to(rng.integers(0, 500, n), np.int32)
    q, k = to(rng.uniform(-1, 1, (n, heads, dim)), np.float16), to(rng.uniform(-1, 1, (n, kv, dim)), np.float16)
    q2, k2 = q.clone(), k.clone()
    llmk.rope_apply(q, k, pos, inv, n, heads, kv, dim)
    llmk.rotary_apply(q2, heads * dim, k2, kv * dim, pos, inv, None, None, n, heads, kv, dim, dim)
    for a, b in ((q, q2), (k, k2)):
        assert (a.float() - b.float()).abs().max().item() <= 6 * 2.0 ** -11 + 500 * 2.0 ** -24 * 2


def scatter_case(rng, n, heads, kv, dim, rotary, page, max_pages, n_tables=2, pad=0):
    num_pages = n * max_pages + 3
    table = rng.permutation(num_pages)[:n * max_pages].reshape(n, max_pages)
    pos = rng.integers(0, page * max_pages, n)
    x = rng.standard_normal((n, (heads + 2 * kv) * dim + pad)).astype(np.float16)
    inv, t, s = tables(rng, n, rotary, n_tables)
    return num_pages, table, pos, x, inv, t, s


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("n,heads,kv,dim,rotary,page,max_pages", [
    (1, 32, 8, 64, 64, 16, 3), (7, 4, 2, 128, 32, 16, 2), (33, 3, 1, 80, 80, 16, 1), (5, 2, 2, 256, 128, 8, 4),
    (64, 1, 1, 16, 16, 1, 9), (600, 4, 2, 64, 48, 16, 2), (1500, 2, 1, 96, 96, 32, 1), (3, 2, 1, 512, 512, 16, 2)])
def test_scatter(llmk, pairs, n, heads, kv, dim, rotary, page, max_pages):
    rng = np.random.default_rng([n, heads, dim, rotary])
    num_pages, table, pos, x, inv, t, s = scatter_case(rng, n, heads, kv, dim, rotary, page, max_pages,
                                                       pad=8 * (n % 3))
    layout = llmk.ROTARY_PAIRS if pairs else llmk.ROTARY_HALVES
    poison = np.full((num_pages, page, kv, dim), 0x7F7F, np.uint16).view(np.float16)
    for nowhere in (False, True):
        p, tb = pos.copy(), table.copy()
        if nowhere and n > 2:  # rows past the table, below 0, and of a page that is none
            p[0], p[1] = page * max_pages, -1
            tb[2, p[2] // page] = -1
        kp, vp = to(poison, np.float16), to(poison, np.float16)
        q = torch.full((n, heads, dim), 9.0, dtype=torch.float16, device=DEV)
        llmk.qkv_rotary_scatter(to(x, np.float16), x.shape[1], q, kp, vp, to(tb, np.int32), to(p, np.int32),
                                to(inv, np.float32), to(t, np.int32), to(s, np.float32), n, max_pages, page,
                                heads, kv, dim, rotary, layout)
        y = x[:, :(heads + 2 * kv) * dim].reshape(n, -1, dim)
        want, bound = ref.rotate(y[:, :heads + kv], p, inv, t, s, rotary, pairs)
        exact = np.broadcast_to(np.arange(dim) >= rotary, want.shape)
        bound = np.where(exact, 0.0, bound)
        assert (np.abs(q.cpu().numpy().astype(np.float64) - want[:, :heads]) <= bound[:, :heads]).all()
        kp, vp = kp.cpu().numpy(), vp.cpu().numpy()
        left = np.ones((num_pages, page), bool)
        for r in range(n):
            if not 0 <= p[r] < page * max_pages or tb[r, p[r] // page] < 0:
                continue
            at = tb[r, p[r] // page], p[r] % page
            left[at] = False
            assert (np.abs(kp[at].astype(np.float64) - want[r, heads:]) <= bound[r, heads:]).all()
            assert np.array_equal(vp[at].view(np.uint16), y[r, heads + kv:].view(np.uint16))
        for pool in (kp, vp):
            assert (pool.view(np.uint16)[left] == 0x7F7F).all(), "another row of the pool was written"


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("n,heads,kv,dim,rotary", [
    (1601, 28, 4, 128, 64), (2600, 8, 1, 256, 256), (401, 60, 2, 256, 96), (221, 118, 1, 256, 16),
    (22300, 1, 1, 96, 96), (7001, 2, 1, 240, 16)])
def test_scatter_of_long_prompts(llmk, pairs, n, heads, kv, dim, rotary):
    test_scatter(llmk, pairs, n, heads, kv, dim, rotary, 16, 1)


def test_numbers_that_are_none(llmk):
    """Infinities and NaN reach their partner and nothing else."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, 2, 64)).astype(np.float16)
    x[1, 0, 3], x[1, 1, 40] = np.inf, np.nan
    inv, _, _ = tables(rng, 3, 64, 1)
    for pairs in (False, True):
        d = to(x, np.float16)
        llmk.rotary_apply(d, 128, None, 0, to([5, 6, 7], np.int32), to(inv, np.float32), None, None, 3, 2, 0, 64,
                          64, int(pairs))
        got = np.isfinite(d.cpu().numpy())
        want, _ = ref.rotate(np.where(np.isfinite(x), x, 0), np.array([5, 6, 7]), inv, None, None, 64, pairs)
        lost = np.zeros(x.shape, bool)
        for h, i in ((0, 3), (1, 40)):
            lost[1, h, i] = lost[1, h, (i ^ 1) if pairs else (i + 32) % 64] = True
        assert np.array_equal(got, ~lost)
        assert np.allclose(d.cpu().numpy()[~lost], want[~lost], atol=4e-3)


def test_captured_and_replayed(llmk):
    rng = np.random.default_rng(6)
    n, heads, kv, dim = 9, 4, 2, 64
    num_pages, table, pos, x, inv, t, s = scatter_case(rng, n, heads, kv, dim, 32, 16, 4)
    dev = dict(x=to(x, np.float16), pos=to(pos, np.int32), t=to(t, np.int32), table=to(table, np.int32),
               inv=to(inv, np.float32), s=to(s, np.float32))
    kp = torch.zeros((num_pages, 16, kv, dim), dtype=torch.float16, device=DEV)
    vp, q = torch.zeros_like(kp), torch.zeros((n, heads, dim), dtype=torch.float16, device=DEV)

    def step():
        llmk.qkv_rotary_scatter(dev["x"], x.shape[1], q, kp, vp, dev["table"], dev["pos"], dev["inv"],
                                dev["t"], dev["s"], n, 4, 16, heads, kv, dim, 32, 1)
        llmk.rotary_apply(q, heads * dim, None, 0, dev["pos"], dev["inv"], None, None, n, heads, 0, dim, 64 - 32)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for replay in range(3):
        dev["pos"].copy_(to(rng.integers(0, 64, n), np.int32))
        dev["x"].copy_(to(rng.standard_normal(x.shape), np.float16))
        for b in (kp, vp, q):
            b.zero_()
        g.replay()
        torch.cuda.synchronize()
        replayed = [b.clone() for b in (kp, vp, q)]
        for b in (kp, vp, q):
            b.zero_()
        step()
        for a, b in zip(replayed, (kp, vp, q)):
            assert torch.equal(a, b)


def test_python_refusals(llmk):
    h = torch.zeros(4, 256, dtype=torch.float16, device=DEV)
    pool = torch.zeros(4, 16, 1, 64, dtype=torch.float16, device=DEV)
    i, f = torch.zeros(8, dtype=torch.int32, device=DEV), torch.zeros(64, device=DEV)

    def apply(**kw):
        a = dict(q=h, ldq=256, k=h[:, 128:], ldk=256, pos=i, inv=f, t=None, s=None, n=4, heads=2, kv=1, dim=64,
                 rot=64) | kw
        llmk.rotary_apply(*a.values(), check_indices=True)

    def scatter(**kw):
        a = dict(qkv=h, ld=256, q=torch.zeros_like(h), k=pool, v=pool.clone(), tables=i, pos=i, inv=f, t=None,
                 s=None, n=4, max_pages=2, page=16, heads=2, kv=1, dim=64, rot=64) | kw
        llmk.qkv_rotary_scatter(*a.values(), check_indices=True)

    apply()
    scatter()
    for bad in (dict(k=h[:, 200:]), dict(q=h[:3]), dict(pos=i[:3]), dict(pos=i.long()), dict(inv=f[:31]),
                dict(t=i + 2), dict(t=i - 1), dict(ldq=128), dict(rot=63), dict(rot=66), dict(s=i)):
        with pytest.raises(llmk.LlmkError):
            apply(**bad)
    for bad in (dict(tables=i[:7]), dict(tables=i + 4), dict(tables=i - 1), dict(pos=i + 32), dict(pos=i - 1),
                dict(k=pool.float()), dict(q=h[:1]), dict(qkv=h[:2]), dict(dim=60), dict(t=i + 2)):
        with pytest.raises(llmk.LlmkError):
            scatter(**bad)
