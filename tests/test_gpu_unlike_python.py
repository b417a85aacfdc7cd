"""What the Python face says to arguments that are nothing the calls take: its own error, whatever they are."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("check", [False, True])
@pytest.mark.parametrize("bad", [None, "x", 3, [1.0]])
def test_pools_that_are_no_tensors(llmk, bad, check):
    pool, pairs = torch.zeros(4, 8, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for pools in ([bad], [pool, bad], (bad, pool)):
        with pytest.raises(llmk.LlmkError):
            llmk.kv_copy_pages(pools, pairs, None, 1, 4, check_indices=check)
