"""Sizes past what the entry points for adapters, rotary layouts and shared pages take are refused as such, before any
launch: at the C-ABI, on the CPU."""
import pytest

from test_unlike_refusals import fork

APART = dict(refs=1 << 42, new=1 << 36, ws=1 << 40, new_lens=1 << 44, copies=1 << 43, tables=1 << 45)


@pytest.mark.parametrize("pages", [2 ** 30 + 1, 2 ** 31 - 4097, 2 ** 31 - 1])
def test_kv_fork_pages(llmk, pages):
    """Page numbers are looked at some thousands past the last one: they have to stay below 2^31."""
    for n in (2, 300):
        assert fork(llmk.lib(), **APART, pages=pages, n_new=n) == llmk.LLMK_ERR_UNSUPPORTED
