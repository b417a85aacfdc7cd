"""Calls of more threads than a launch takes (2^32 in a dimension) are refused as such, before any launch:
at the C-ABI, on the CPU."""
import pytest

from test_kv8_refusals import append, gather, verify

MOST = 2 ** 28 - 16  # rows of append and read-back: 256 threads for 16


@pytest.mark.parametrize("call", [append, gather])
@pytest.mark.parametrize("n_rows", [MOST + 1, 2 ** 28, 2 ** 31 - 1])
def test_rows(llmk, call, n_rows):
    assert call(llmk.lib(), n_rows=n_rows) == llmk.LLMK_ERR_UNSUPPORTED
    assert call(llmk.lib(), n_rows=n_rows, n_seqs=n_rows, starts=None) == llmk.LLMK_ERR_UNSUPPORTED
    assert call(llmk.lib(), n_rows=n_rows, n_seqs=0) == 0  # nothing to launch


@pytest.mark.parametrize("what", [
    dict(n_rows=2 ** 25, vocab=100),               # 64 threads for a chunk, of both models' rows
    dict(n_rows=2 ** 26, draft=None, vocab=100),
    dict(n_rows=2 ** 20, vocab=128256),
    dict(n_seqs=2 ** 23, vocab=100),               # 512 threads for a sequence
    dict(n_seqs=2 ** 20, vocab=128256),            # 256 for a piece of its drawn row
    dict(n_rows=2 ** 26, n_seqs=2 ** 26, starts=None, drafts=None, u=None, vocab=1)])
def test_verify(llmk, what):
    assert verify(llmk.lib(), **what) == llmk.LLMK_ERR_UNSUPPORTED
