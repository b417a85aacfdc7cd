"""What the entry points for adapters, rotary layouts and shared pages refuse, at the C-ABI (every call here
returns before any launch) and in Python; the host's frequency tables against their formulas; and the
restatements that the GPU tests compare with, against invariants of their own."""
import ctypes
import math

import numpy as np
import pytest
import torch

import _unlike as ref

FAKE = 0x10000  # 16-byte aligned, never dereferenced
MIS = FAKE + 4


def ints(*v):
    return (ctypes.c_int32 * len(v))(*v)


def lora(L, **kw):
    a = dict(x=FAKE, ldx=64, a=FAKE, b=FAKE, ranks=FAKE, scales=FAKE, ids=FAKE, starts=FAKE, y=FAKE,
             ldy=48, ends=ints(32, 48), parts=2, ws=FAKE, n_rows=4, n_seqs=2, n_adapters=3, rank=16,
             inner=64) | kw
    return L.llmk_lora_add(*a.values(), None)


def rotary(L, **kw):
    a = dict(q=FAKE, ldq=256, k=FAKE, ldk=128, pos=FAKE, inv=FAKE, ids=FAKE, scales=FAKE, n=0, heads=4,
             kv=2, dim=64, rot=32, tables=2, layout=0) | kw
    return L.llmk_rotary_apply(*a.values(), None)


def scatter(L, **kw):
    a = dict(qkv=FAKE, ld=512, q=FAKE, k=FAKE, v=FAKE, tables=FAKE, pos=FAKE, inv=FAKE, ids=FAKE,
             scales=FAKE, n=3, max_pages=2, page=16, heads=4, kv=2, dim=64, rot=32, n_tables=1,
             layout=1) | kw
    return L.llmk_qkv_rotary_scatter(*a.values(), None)


def copy_pages(L, **kw):
    a = dict(pools=(ctypes.c_void_p * 2)(FAKE, FAKE), sizes=(ctypes.c_size_t * 2)(64, 64), n=2,
             copies=FAKE, count=None, n_copies=0, pages=8) | kw
    return L.llmk_kv_copy_pages(*a.values(), None)


AT = [FAKE + 0x1000 * i for i in range(12)]  # arrays apart from one another


def fork(L, **kw):
    a = dict(tables=AT[0], lens=AT[1], parents=AT[2], reserve=None, refs=AT[3], new=AT[4], new_lens=AT[5],
             copies=AT[6], counts=AT[7], ws=AT[8], n_old=2, n_new=2, max_pages=4, page=16, pages=9) | kw
    return L.llmk_kv_fork(*a.values(), None)


def compact(L, **kw):
    a = dict(tables=AT[0], refs=AT[1], new=AT[2], new_refs=AT[3], copies=AT[4], counts=AT[5], ws=AT[6], n=2,
             max_pages=4, pages=9) | kw
    return L.llmk_kv_compact(*a.values(), None)


def test_lora_add_refuses_rows_that_overlap(llmk):
    """x at a megabyte; what does not overlap is refused for its workspace, which is checked in front."""
    L, E, at = llmk.lib(), llmk, 1 << 20
    wide = dict(x=at, ldx=128, ldy=128)  # rows of 64 and of 48, 128 apart
    for y in (at, at + 16, at + 2 * 48, at - 2 * 32, at + 2 * 128, at + 2 * (128 + 48), at - 2 * 128 * 3,
              at + 2 * 88):  # the last: its 48 columns end in x's next row
        assert lora(L, **wide, y=y) == E.LLMK_ERR_INVALID_VALUE, y - at
    assert lora(L, **wide | dict(ldx=64), y=at + 2 * 128) == E.LLMK_ERR_INVALID_VALUE
    assert lora(L, **wide | dict(ldy=48), y=at + 2 * 64) == E.LLMK_ERR_INVALID_VALUE  # other strides, one stretch


def test_qkv_rotary_scatter_refuses_q_over_qkv(llmk):
    at, rows, q = 1 << 20, 2 * (2 * 512 + 512), 2 * 3 * 256
    for to in (at, at + 16, at + rows - 16, at - q + 16):
        assert scatter(llmk.lib(), qkv=at, q=to) == llmk.LLMK_ERR_INVALID_VALUE, to - at


def test_lora_add_sizes_past_the_limits(llmk):
    """The call is refused, and its workspace is none."""
    L, E, most = llmk.lib(), llmk, 2 ** 31 - 8
    for bad in (dict(rank=264), dict(rank=most), dict(n_rows=(1 << 20) + 1), dict(n_seqs=2 ** 31 - 1),
                dict(inner=(1 << 24) + 8, ldx=(1 << 24) + 8), dict(inner=most, ldx=most)):
        assert lora(L, **bad) == E.LLMK_ERR_UNSUPPORTED, bad
        a = dict(n_rows=4, n_seqs=2, n_adapters=3, rank=16, inner=64) | {k: v for k, v in bad.items() if k != "ldx"}
        assert llmk.lora_add_workspace_floats(*a.values(), 2) == 0
    assert llmk.lora_add_workspace_floats(4, 2, 3, 16, 64, 9) == 0


def test_lora_add(llmk):
    L, E = llmk.lib(), llmk
    for nothing in (dict(n_rows=0), dict(n_seqs=0), dict(n_adapters=0),
                    dict(n_rows=0, n_seqs=0, x=None, y=None)):
        assert lora(L, **nothing) == 0
    for bad in (dict(n_rows=-1), dict(n_seqs=-1), dict(n_adapters=-1), dict(rank=0), dict(inner=0),
                dict(parts=0), dict(parts=9), dict(ends=None), dict(starts=None), dict(x=None),
                dict(a=None), dict(b=None), dict(ids=None), dict(y=None), dict(ws=None),
                dict(ends=ints(32, 32)), dict(ends=ints(0, 32)), dict(ends=ints(48, 32))):
        assert lora(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    for bad in (dict(rank=12), dict(inner=60), dict(ldx=56), dict(ldx=68), dict(ldy=40), dict(ldy=52),
                dict(ends=ints(30, 48))):
        assert lora(L, **bad) == E.LLMK_ERR_SHAPE, bad
    for bad in (dict(x=MIS), dict(a=MIS), dict(b=MIS), dict(y=MIS), dict(ws=MIS)):
        assert lora(L, **bad) == E.LLMK_ERR_ALIGNMENT, bad
    for bad in (dict(rank=264), dict(n_rows=(1 << 20) + 1), dict(n_seqs=(1 << 20) + 1)):
        assert lora(L, **bad) == E.LLMK_ERR_UNSUPPORTED, bad
    for nothing in ((0, 1, 1, 16, 64, 1), (1, 0, 1, 16, 64, 1), (1, 1, 0, 16, 64, 1),
                    (1, 1, 1, 0, 64, 1), (1, 1, 1, 16, 0, 1), (1, 1, 1, 16, 64, 0), (-1,) * 6):
        assert llmk.lora_add_workspace_floats(*nothing) == 0
    assert llmk.lora_add_workspace_floats(1, 1, 1, 8, 8, 1) > 0


def test_rotary(llmk):
    L, E = llmk.lib(), llmk
    assert rotary(L) == 0 and rotary(L, heads=0, kv=0, n=3) == 0
    for bad in (dict(n=-1), dict(heads=-1), dict(kv=-1), dict(dim=0), dict(rot=0)):
        assert rotary(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    for bad in (dict(rot=66), dict(ldq=255), dict(ldk=127)):
        assert rotary(L, **bad) == E.LLMK_ERR_SHAPE, bad
    for bad in (dict(q=None), dict(k=None), dict(pos=None), dict(inv=None), dict(tables=0),
                dict(layout=2), dict(layout=-1)):
        assert rotary(L, n=3, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    assert rotary(L, n=3, rot=33) == E.LLMK_ERR_SHAPE
    assert rotary(L, n=3, dim=8192, ldq=4 * 8192, ldk=2 * 8192) == E.LLMK_ERR_UNSUPPORTED

    assert scatter(L, n=0) == 0
    for bad in (dict(n=-1), dict(max_pages=0), dict(page=0), dict(heads=0), dict(kv=0), dict(dim=0),
                dict(rot=0), dict(qkv=None), dict(q=None), dict(k=None), dict(v=None), dict(tables=None),
                dict(pos=None), dict(inv=None), dict(n_tables=0), dict(layout=2)):
        assert scatter(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    for bad in (dict(dim=72), dict(rot=24), dict(rot=80), dict(ld=504), dict(ld=516)):
        assert scatter(L, **bad) == E.LLMK_ERR_SHAPE, bad
    for bad in (dict(qkv=MIS), dict(q=MIS), dict(k=MIS), dict(v=MIS)):
        assert scatter(L, **bad) == E.LLMK_ERR_ALIGNMENT, bad
    assert scatter(L, dim=528, ld=8 * 528) == E.LLMK_ERR_UNSUPPORTED


def test_pages(llmk):
    L, E = llmk.lib(), llmk
    assert copy_pages(L) == 0 and copy_pages(L, n=0, n_copies=3, pools=None) == 0
    for bad in (dict(n=-1), dict(n_copies=-1), dict(pages=0)):
        assert copy_pages(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    for bad in (dict(pools=None), dict(sizes=None), dict(copies=None),
                dict(pools=(ctypes.c_void_p * 2)(FAKE, None)), dict(sizes=(ctypes.c_size_t * 2)(64, 0))):
        assert copy_pages(L, n_copies=3, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    assert copy_pages(L, n_copies=3, sizes=(ctypes.c_size_t * 2)(64, 6)) == E.LLMK_ERR_SHAPE
    assert copy_pages(L, n_copies=3, pools=(ctypes.c_void_p * 2)(FAKE + 2, FAKE)) == E.LLMK_ERR_ALIGNMENT
    assert copy_pages(L, n_copies=3, sizes=(ctypes.c_size_t * 2)(64, (1 << 32) + 4)) == \
        E.LLMK_ERR_UNSUPPORTED

    for bad in (dict(n_old=-1), dict(n_new=-1), dict(max_pages=0), dict(page=0), dict(pages=0),
                dict(refs=None), dict(counts=None), dict(ws=None), dict(tables=None), dict(lens=None),
                dict(parents=None), dict(new=None), dict(new_lens=None), dict(copies=None)):
        assert fork(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    for bad in (dict(new=AT[0]), dict(new=AT[0] + 28), dict(new_lens=AT[1] + 4), dict(refs=AT[0]), dict(ws=AT[4]),
                dict(copies=AT[2]), dict(counts=AT[3] + 32), dict(reserve=AT[5])):
        assert fork(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    apart = dict(new=1 << 36, ws=1 << 40, new_lens=1 << 44, copies=1 << 43, tables=1 << 45)
    for bad in (dict(n_old=65536), dict(n_new=65536), dict(max_pages=(1 << 24) + 1)):
        assert fork(L, **(apart | bad)) == E.LLMK_ERR_UNSUPPORTED, bad
    assert fork(L, ws=AT[8] + 4) == E.LLMK_ERR_ALIGNMENT
    assert llmk.kv_fork_workspace_ints(-1, 1, 1, 1) == llmk.kv_fork_workspace_ints(1, 1, 0, 1) == 0

    for bad in (dict(n=-1), dict(max_pages=0), dict(pages=0), dict(refs=None), dict(new_refs=None),
                dict(copies=None), dict(counts=None), dict(ws=None), dict(tables=None), dict(new=None)):
        assert compact(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    for bad in (dict(new=AT[0] + 4), dict(new=AT[0] - 4), dict(new_refs=AT[1] + 32), dict(copies=AT[0]),
                dict(counts=AT[1]), dict(ws=AT[4]), dict(new=AT[1]), dict(new_refs=AT[0])):
        assert compact(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    apart = dict(refs=1 << 36, new_refs=1 << 37, copies=1 << 38, ws=1 << 40)
    assert compact(L, pages=(1 << 24) + 1, **apart) == E.LLMK_ERR_UNSUPPORTED
    assert llmk.kv_compact_workspace_ints(0) == 0


def test_python_refuses_host_tensors(llmk):
    h, i = torch.zeros(64, dtype=torch.float16), torch.zeros(64, dtype=torch.int32)
    f = torch.zeros(64)
    for call in (lambda: llmk.lora_add(h, 8, h, h, None, None, i, None, h, 8, (8,), f, 1, 1, 1, 8, 8),
                 lambda: llmk.rotary_apply(h, 8, h, 8, i, f, None, None, 1, 1, 1, 8, 8),
                 lambda: llmk.qkv_rotary_scatter(h, 48, h, h, h, i, i, f, None, None, 1, 1, 16, 1, 1, 16, 16),
                 lambda: llmk.kv_copy_pages([h], i, None, 1, 8),
                 lambda: llmk.kv_fork(i, i, i, None, i, i, i, i, i, i, 1, 1, 1, 16, 8),
                 lambda: llmk.kv_compact(i, i, i, i, i, i, i, 1, 1, 8)):
        with pytest.raises(llmk.LlmkError):
            call()


@pytest.mark.parametrize("rotary,theta,factor,orig", [(64, 500000.0, 8.0, 8192.0), (128, 10000.0, 4.0, 4096.0),
                                                      (2, 10000.0, 2.0, 2048.0), (6, 100.0, 1.0, 16.0),
                                                      (32, 1e6, 40.0, 1000.0), (64, 1e4, 4.0, 2.0)])
def test_frequency_tables(llmk, rotary, theta, factor, orig):
    i = np.arange(rotary // 2)
    f = theta ** (-2.0 * i / rotary)

    def near(got, want):
        np.testing.assert_allclose(got, want, rtol=2.0 ** -23)  # half a step of fp32 and 64-bit errors

    got, scale = llmk.compute_rotary_inv_freq(llmk.ROTARY_PLAIN, rotary, theta)
    near(got, f)
    assert scale == 1.0
    got, scale = llmk.compute_rotary_inv_freq(llmk.ROTARY_LINEAR, rotary, theta, factor)
    near(got, f / factor)
    assert scale == 1.0
    got, scale = llmk.compute_rotary_inv_freq(llmk.ROTARY_NTK, rotary, theta, factor)
    if rotary > 2:  # the fastest pair as trained, the slowest factor times slower
        near(got, (theta * factor ** (rotary / (rotary - 2))) ** (-2.0 * i / rotary))
        np.testing.assert_allclose([got[0], got[-1]], [1.0, f[-1] / factor], rtol=1e-6)
    else:
        near(got, f)
    got, scale = llmk.compute_rotary_inv_freq(llmk.ROTARY_YARN, rotary, theta, factor, orig)

    def pair(b):
        return rotary * math.log(orig / (2 * math.pi * b)) / (2 * math.log(theta))
    low = max(math.floor(pair(32.0)), 0)
    high = max(min(math.ceil(pair(1.0)), rotary - 1), low + 0.001)
    m = np.clip((i - low) / (high - low), 0, 1)
    near(got, f * (1 - m) + f / factor * m)
    np.testing.assert_allclose(scale, 0.1 * math.log(factor) + 1 if factor > 1 else 1.0, rtol=2.0 ** -23)
    assert np.all(np.asarray(got) <= np.float32(1.0)) and np.all(np.asarray(got) > 0)


def test_frequency_tables_refuse(llmk):
    for args in ((4, 64, 1e4), (-1, 64, 1e4), (0, 63, 1e4), (0, 0, 1e4), (0, 64, 0.0), (0, 64, math.nan),
                 (1, 64, 1e4, 0.0), (2, 64, 1e4, math.inf), (3, 64, 1e4, 4.0, 0.0),
                 (3, 64, 1.0, 4.0, 4096.0), (3, 64, 1e4, 4.0, 4096.0, 1.0, 32.0),
                 (3, 64, 1e4, 4.0, 4096.0, 32.0, 0.0)):
        with pytest.raises(llmk.LlmkError):
            llmk.compute_rotary_inv_freq(*args)


def test_restated_fork_keeps_the_books():
    """Holders are counted right whatever is forked; nobody writes to a page that others hold."""
    rng = np.random.default_rng(7)
    for trial in range(60):
        page, max_pages = int(rng.choice([1, 4, 16])), int(rng.integers(1, 9))
        n = int(rng.integers(1, 9))
        tables, lens, refs, num_pages = ref.batch(rng, n, 3, page * max_pages, page, max_pages,
                                                  spare=int(rng.integers(0, 20)))
        parents = rng.integers(-1, n + 1, int(rng.integers(1, 12)))
        reserve = rng.integers(-2, 2 * page + 1, parents.size)
        new, new_lens, after, copies, counts = ref.fork(tables, lens, parents, reserve, refs, parents.size,
                                                        max_pages, page, num_pages)
        rows = [ref.held(r, num_pages) for r in new]
        holders = np.bincount([p for r in rows for p in r], minlength=num_pages)
        assert np.array_equal(holders, after) and after.min() >= 0
        for c, row in enumerate(rows):
            for j, p in enumerate(row):
                if j >= new_lens[c] // page:
                    assert after[p] == 1
        to = copies[copies[:, 1] >= 0, 1]
        assert len(set(to)) == len(to) and not set(to) & set(copies[copies[:, 0] >= 0, 0])
        if counts[1] == 0:
            for c, row in enumerate(rows):
                room = max(int(reserve[c]), 0)
                assert len(row) == min(max_pages, -(-(int(new_lens[c]) + room) // page))


def test_restated_compaction_keeps_the_books():
    rng = np.random.default_rng(8)
    for trial in range(40):
        tables, _, refs, num_pages = ref.batch(rng, int(rng.integers(1, 9)), 3, 60, 16, 5,
                                               spare=int(rng.integers(0, 30)))
        new, after, pairs, counts = ref.compact(tables, refs)
        assert np.array_equal(after > 0, np.arange(num_pages) < counts[1])
        held = new[new >= 0]
        assert np.array_equal(np.bincount(held, minlength=num_pages), after)
        assert len(pairs) == counts[0] <= num_pages // 2
