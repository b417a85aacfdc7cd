"""Sizes past what the entry points for adapters, rotary layouts and shared pages take are refused as such, before any
launch: at the C-ABI, on the CPU."""
import ctypes

import pytest

from test_unlike_refusals import FAKE, MIS, copy_pages, fork, ints, lora, scatter

APART = dict(refs=1 << 42, new=1 << 36, ws=1 << 40, new_lens=1 << 44, copies=1 << 43, tables=1 << 45)


@pytest.mark.parametrize("pages", [2 ** 30 + 1, 2 ** 31 - 4097, 2 ** 31 - 1])
def test_kv_fork_pages(llmk, pages):
    """Page numbers are looked at some thousands past the last one: they have to stay below 2^31."""
    for n in (2, 300):
        assert fork(llmk.lib(), **APART, pages=pages, n_new=n) == llmk.LLMK_ERR_UNSUPPORTED


@pytest.mark.parametrize("first,last", [(64, 1 << 32), (20, 1 << 32), (20, (1 << 32) - 4), (64, 1 << 31)])
def test_kv_copy_pages_of_more_blocks_than_a_launch_takes(llmk, first, last):
    """64 pools of small pages go in a launch of their own, those that are no whole vectors too: the call is refused
    before the first one, and not behind it."""
    pools = (ctypes.c_void_p * 65)(*[FAKE] * 65)
    sizes = (ctypes.c_size_t * 65)(*[first] * 64, last)
    for n in (256, 2 ** 31 - 1):
        assert copy_pages(llmk.lib(), pools=pools, sizes=sizes, n=65, n_copies=n) == llmk.LLMK_ERR_UNSUPPORTED


@pytest.mark.parametrize("rank,most", [(16, 65535 * 512), (128, 65535 * 512), (136, 65535 * 256), (256, 65535 * 256)])
def test_lora_add_columns(llmk, rank, most):
    """Refused by the columns alone: a misaligned x of a call that is not shows that these are not refused for it."""
    for n in (4, 1 << 20):
        sizes = dict(rank=rank, n_rows=n, n_seqs=n, parts=1, x=MIS)
        for columns, status in ((most, llmk.LLMK_ERR_ALIGNMENT), (most + 8, llmk.LLMK_ERR_UNSUPPORTED)):
            assert lora(llmk.lib(), **sizes, ends=ints(columns), ldy=columns) == status


def test_qkv_rotary_scatter_parts_of_a_head(llmk):
    """Multiples of 16, and even whole fractions of the head; a misaligned q shows that they are not refused as shapes."""
    for dim, rot, status in ((80, 20, 0), (80, 40, 0), (80, 16, 0), (64, 2, 0), (64, 24, 1), (80, 60, 1), (80, 5, 1), (16, 1, 1),
                             (80, 160, 1), (64, 6, 1)):
        want = llmk.LLMK_ERR_SHAPE if status else llmk.LLMK_ERR_ALIGNMENT
        assert scatter(llmk.lib(), dim=dim, rot=rot, ld=8 * dim, q=MIS) == want, (dim, rot)
        assert scatter(llmk.lib(), dim=dim, rot=rot, ld=8 * dim, n=0) == (llmk.LLMK_ERR_SHAPE if status else 0), (dim, rot)
