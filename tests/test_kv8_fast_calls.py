"""The native calls for the 8-bit KV cache and drafted tokens: no answer, and no exception set, for
anything but plainly right arguments; then the Python checks decide (tests/test_fast_calls.py has the
others)."""
import pytest
import torch


def half(n):
    return torch.zeros(n, dtype=torch.float16)


def ints(n):
    return torch.zeros(n, dtype=torch.int32)


def e4m3(n):
    return torch.zeros(n, dtype=torch.uint8).view(torch.float8_e4m3fn)


CACHE = (e4m3(1024), torch.zeros(1), e4m3(1024), torch.zeros(1))
BATCH = (ints(1), ints(2), ints(1))
CALLS = {
    "kv8_append": (half(192), 192, half(64), *CACHE, *BATCH, torch.zeros(32), 1, 1, 1, 16, 1, 1, 64,
                   0),
    "kv8_gather": (*CACHE, *BATCH, half(64), half(64), 1, 1, 1, 16, 1, 64, 0),
    "kv8_attention": (half(64), *CACHE, *BATCH, half(64), None, 1, 1, 1, 1, 16, 1, 1, 64, 0),
    "verify_drafts": (half(8), None, ints(1), ints(2), None, torch.zeros(1), torch.zeros(1), ints(1),
                      ints(1), torch.zeros(64), 1, 1, 8, 0),
}


@pytest.mark.parametrize("name", CALLS)
def test_no_answer_for_anything_but_cuda_tensors(llmk, name):
    f, args = getattr(llmk._fast, name), CALLS[name]
    assert f(*args) is None  # CPU tensors
    assert f(*args[:-1]) is None and f(*args, 0) is None  # too few and too many arguments
    for i in range(len(args)):
        for bad in (None, "x", -1, 0, 1 << 70, 1.5, object()):
            assert f(*args[:i], bad, *args[i + 1:]) is None


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_an_answer_for_what_is_right_and_none_for_each_thing_that_is_not(llmk, name):
    f = getattr(llmk._fast, name)
    args = [a.cuda() if isinstance(a, torch.Tensor) else a for a in CALLS[name]]
    if name == "kv8_attention":
        args[-1] = None
    assert f(*args) == 0
    torch.cuda.synchronize()
    for i, a in enumerate(args):
        if not isinstance(a, torch.Tensor):
            continue
        wrong = [a.cpu(), a.view(torch.uint8).view(torch.int64)[:0] if a.numel() >= 8 else "x",
                 a.double() if a.dtype == torch.float32 else "x"]
        if a.numel() > 1:
            wrong += [a[:-1], torch.stack([a, a], 1)[:, 0] if a.element_size() > 1 else "x"]
        for bad in wrong:
            if name == "verify_drafts" and i == 9 and isinstance(bad, torch.Tensor) and (
                    bad.is_cuda and bad.dtype == a.dtype and bad.is_contiguous()):
                continue  # a workspace that is larger than it need be
            assert f(*args[:i], bad, *args[i + 1:]) is None, (i, bad)
