"""Forks whose children want more than 2^31 pages together."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("max_pages,free", [(2 ** 21 + 8, 5000), (2 ** 22 + 1024, 3), (2 ** 22 + 1024, 70000)])
def test_wanted_pages_past_32_bits(llmk, max_pages, free):
    """1024 empty children want whole rows of a wide table: over 2^31 pages, and over 2^32. The free pages go to the
    first child, in order; the pages lacking end at 2^31 - 1."""
    n, held = 1024, 7
    num_pages = free + held
    ints = 2 * n * max_pages + n * max_pages  # the workspace and the new tables
    if torch.cuda.mem_get_info()[0] < 4 * ints + (8 << 30):
        pytest.skip("not enough memory")
    i32 = dict(dtype=torch.int32, device=DEV)
    refs = torch.zeros(num_pages, **i32)
    refs[:held] = 1  # somebody else's
    new = torch.full((n, max_pages), 5, **i32)
    new_lens, copies, counts = torch.full((n,), 9, **i32), torch.full((n, 2), 9, **i32), torch.full((2,), 9, **i32)
    ws = torch.empty(llmk.kv_fork_workspace_ints(1, n, max_pages, num_pages), **i32)
    llmk.kv_fork(torch.full((1, max_pages), -1, **i32), torch.zeros(1, **i32), torch.zeros(n, **i32),
                 torch.full((n,), max_pages, **i32), refs, new, new_lens, copies, counts, ws, 1, n, max_pages, 1,
                 num_pages)
    assert counts.tolist() == [free, min(n * max_pages - free, 2 ** 31 - 1)]
    assert torch.equal(new[0, :free], torch.arange(held, num_pages, **i32))
    assert int(new[0, free:].max()) == int(new[1:].max()) == int(new.min()) == -1
    assert (refs == 1).all() and (new_lens == 0).all() and (copies == -1).all()
