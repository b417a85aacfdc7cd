"""What the checks of the 8-bit cache's Python calls look at, with the pointers and the launch left out: the
values of a batch, on the CPU."""
import pytest
import torch

PAGE, DIM = 16, 64


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.fixture
def calls(llmk, monkeypatch):
    """The three calls on host tensors; what would be launched is noted instead."""
    launched = []

    class Lib:
        def __getattr__(self, name):
            if name.endswith("_floats"):
                return lambda *args: 0
            return lambda *args: launched.append(name) or 0

    monkeypatch.setattr(llmk, "_dev", lambda fn, t, *a: 0)
    monkeypatch.setattr(llmk, "_here", lambda fn, **tensors: None)
    monkeypatch.setattr(llmk, "_stream", lambda stream: 0)
    monkeypatch.setattr(llmk, "_lib", Lib())

    def cache(k_pages, v_pages):
        out = []
        for pages in (k_pages, v_pages):
            out += [torch.zeros((pages, 1, PAGE, DIM), dtype=torch.uint8).view(torch.float8_e4m3fn),
                    torch.ones((pages, 1))]
        return out

    def call(name, k_pages, v_pages, tables, starts, lens, n_rows):
        x = torch.zeros(n_rows * 6 * DIM, dtype=torch.float16)
        pools, n = cache(k_pages, v_pages), lens.numel()
        batch = (tables, starts, lens)
        shape = (n_rows, n, tables.numel() // n)
        if name == "kv8_append":
            llmk.kv8_append(x, 6 * DIM, x, *pools, *batch, x, *shape, PAGE, 4, 1, DIM,
                            check_indices=True)
        elif name == "kv8_gather":
            llmk.kv8_gather(*pools, *batch, x, x, *shape, PAGE, 1, DIM, check_indices=True)
        else:
            llmk.kv8_attention(x, *pools, *batch, x, None, n_rows, n, n_rows, shape[2], PAGE, 4, 1,
                               DIM, check_indices=True)
        return launched.pop() == "llmk_" + name and not launched
    return call


NAMES = ["kv8_append", "kv8_gather", "kv8_attention"]


@pytest.mark.parametrize("name", NAMES)
def test_a_page_is_one_of_both_pools(llmk, calls, name):
    """A table's pages are pages of K and of V: the smaller pool is the limit, whichever it is."""
    tables, lens = ints(0, 3, 4, 1), ints(20, 30)
    assert calls(name, 5, 5, tables, None, lens, 2)
    assert calls(name, 9, 5, tables, None, lens, 2) and calls(name, 5, 9, tables, None, lens, 2)
    for k_pages, v_pages in ((4, 9), (9, 4), (9, 1)):
        with pytest.raises(llmk.LlmkError, match="block_tables"):
            calls(name, k_pages, v_pages, ints(4, 4, 1, 3), ints(0, 20, 21), ints(20, 30), 21)


@pytest.mark.parametrize("name", NAMES)
def test_a_sequence_without_rows_names_no_page(llmk, calls, name):
    """Its table is not read: it may hold anything. With a row its pages are looked at."""
    tables, lens = ints(0, 1, 99, -7, 2, 3), ints(20, 30, 32)
    assert calls(name, 4, 4, tables, ints(0, 2, 2, 5), lens, 5)
    with pytest.raises(llmk.LlmkError, match="block_tables"):
        calls(name, 4, 4, tables, ints(0, 2, 3, 5), lens, 5)
