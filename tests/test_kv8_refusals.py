"""What the entry points for the 8-bit KV cache and for drafted tokens refuse, at the C-ABI: every call
here returns before any launch. And the restatement that the GPU tests compare with, against torch's
own e4m3 conversion."""
import numpy as np
import pytest
import torch

import _kv8 as ref

FAKE = 0x10000  # 16-byte aligned, never dereferenced
MIS = FAKE + 4


def test_restated_e4m3_is_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    assert np.array_equal(codes.view(torch.float8_e4m3fn).double().numpy(), ref.VALUES,
                          equal_nan=True)
    rng = np.random.default_rng(1)
    x = np.concatenate([ref.MIDDLES, -ref.MIDDLES, ref.POSITIVE, rng.uniform(-448, 448, 4000),
                        rng.standard_normal(4000) * 0.02, [0.0, -0.0, np.nan]]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ref.encode(x), want)
    assert list(ref.encode(np.array([1e9, -1e9, np.inf]))) == [0x7E, 0xFE, 0x7F]


def append(L, **kw):
    a = dict(qkv=FAKE, ld=3 * 64, q=FAKE, k=FAKE, ks=FAKE, v=FAKE, vs=FAKE, tables=FAKE, starts=FAKE,
             lens=FAKE, inv=FAKE, n_rows=4, n_seqs=2, max_pages=3, page=16, heads=1, kv=1,
             dim=64) | kw
    return L.llmk_kv8_append(*a.values(), None)


def gather(L, **kw):
    a = dict(k=FAKE, ks=FAKE, v=FAKE, vs=FAKE, tables=FAKE, starts=FAKE, lens=FAKE, k_out=FAKE,
             v_out=FAKE, n_rows=4, n_seqs=2, max_pages=3, page=16, kv=1, dim=64) | kw
    return L.llmk_kv8_gather(*a.values(), None)


def attention(L, **kw):
    a = dict(q=FAKE, k=FAKE, ks=FAKE, v=FAKE, vs=FAKE, tables=FAKE, starts=FAKE, lens=FAKE, out=FAKE,
             ws=FAKE, n_rows=4, n_seqs=2, max_rows=2, max_pages=3, page=16, heads=4, kv=1,
             dim=64) | kw
    return L.llmk_kv8_attention(*a.values(), None)


def verify(L, **kw):
    a = dict(logits=FAKE, draft=FAKE, drafts=FAKE, starts=FAKE, t=FAKE, u=FAKE, u2=FAKE, n_acc=FAKE,
             tokens=FAKE, ws=FAKE, n_rows=4, n_seqs=2, vocab=100) | kw
    return L.llmk_verify_drafts(*a.values(), None)


@pytest.mark.parametrize("call", [append, gather, attention])
def test_cache_calls(llmk, call):
    L, E = llmk.lib(), llmk
    assert call(L, n_rows=0) == 0
    assert call(L, n_rows=0, n_seqs=0, k=None, lens=None) == 0
    assert call(L, n_seqs=0) == 0  # rows that belong to none
    for bad in (dict(n_rows=-1), dict(n_seqs=-1), dict(max_pages=0), dict(kv=0), dict(dim=0),
                dict(starts=None), dict(k=None), dict(ks=None), dict(v=None), dict(vs=None),
                dict(tables=None), dict(lens=None)):
        assert call(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    for bad in (dict(page=32), dict(dim=96), dict(dim=256)):
        assert call(L, **bad) == E.LLMK_ERR_SHAPE, bad
    for bad in (dict(k=MIS), dict(v=MIS)):
        assert call(L, **bad) == E.LLMK_ERR_ALIGNMENT, bad


def test_append(llmk):
    L, E = llmk.lib(), llmk
    for bad in (dict(qkv=None), dict(q=None), dict(inv=None), dict(heads=0)):
        assert append(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    for bad in (dict(ld=3 * 64 - 8), dict(ld=3 * 64 + 4), dict(heads=2 ** 26)):
        assert append(L, **bad) == E.LLMK_ERR_SHAPE, bad
    for bad in (dict(qkv=MIS), dict(q=MIS)):
        assert append(L, **bad) == E.LLMK_ERR_ALIGNMENT, bad


def test_gather(llmk):
    L, E = llmk.lib(), llmk
    for bad in (dict(k_out=None), dict(v_out=None)):
        assert gather(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    for bad in (dict(k_out=MIS), dict(v_out=MIS)):
        assert gather(L, **bad) == E.LLMK_ERR_ALIGNMENT, bad
    assert gather(L, kv=65537) == E.LLMK_ERR_UNSUPPORTED


def test_attention(llmk):
    L, E = llmk.lib(), llmk
    for bad in (dict(q=None), dict(out=None), dict(max_rows=0), dict(max_rows=-1), dict(heads=0)):
        assert attention(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    assert attention(L, heads=5, kv=2) == E.LLMK_ERR_SHAPE
    for bad in (dict(q=MIS), dict(out=MIS), dict(ws=MIS)):
        assert attention(L, **bad) == E.LLMK_ERR_ALIGNMENT, bad
    assert attention(L, heads=65536) == E.LLMK_ERR_UNSUPPORTED
    assert attention(L, heads=513, kv=513) == E.LLMK_ERR_UNSUPPORTED
    assert attention(L, max_pages=2 ** 27) == E.LLMK_ERR_UNSUPPORTED
    assert E.kv8_attention_workspace_floats(96) == 0
    assert 0 < E.kv8_attention_workspace_floats(64) < E.kv8_attention_workspace_floats(128) or (
        E.kv8_attention_workspace_floats(64) > 0)


def test_verify(llmk):
    L, E = llmk.lib(), llmk
    assert verify(L, n_seqs=0) == 0
    assert verify(L, n_rows=0, n_seqs=0, logits=None, ws=None) == 0
    for bad in (dict(n_rows=-1), dict(n_seqs=-1), dict(vocab=0), dict(starts=None),
                dict(logits=None), dict(drafts=None), dict(u=None), dict(u2=None),
                dict(n_acc=None), dict(tokens=None), dict(ws=None)):
        assert verify(L, **bad) == E.LLMK_ERR_INVALID_VALUE, bad
    assert verify(L, ws=MIS) == E.LLMK_ERR_ALIGNMENT
    assert verify(L, n_rows=2 ** 30, vocab=128256) == E.LLMK_ERR_UNSUPPORTED
    assert verify(L, vocab=2 ** 31 - 1) == E.LLMK_ERR_UNSUPPORTED
    assert E.verify_drafts_workspace_floats(0, 1, 8) == 0
    # 63 chunks of 2048 logits and 32 pieces of 4096: where a sequence ends, chunks of both models' rows
    # (16 bytes), sums of pieces (24 bytes)
    assert E.verify_drafts_workspace_floats(5, 1, 128256) == 12 + 63 * 2 * 5 * 4 + 32 * 6


def test_python_face_refuses_host_tensors(llmk):
    x = torch.zeros(64, dtype=torch.float16)
    with pytest.raises(llmk.LlmkError, match="CUDA tensor"):
        llmk.verify_drafts(x, None, None, None, None, None, x.float(), x.int(), x.int(), x.float(),
                           1, 1, 64)
    with pytest.raises(llmk.LlmkError, match="CUDA tensor"):
        llmk.kv8_gather(x, x, x, x, x, None, x, x, x, 1, 1, 1, 16, 1, 64)
    with pytest.raises(llmk.LlmkError, match="sizes"):
        llmk.kv8_gather(x, x, x, x, x, None, x, x, x, 1, 1, 0, 16, 1, 64)
