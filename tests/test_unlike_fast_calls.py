"""The native calls for adapters, rotary layouts and shared pages: no answer, and no exception set, for
anything but plainly right arguments; then the Python checks decide."""
import pytest
import torch


def half(*n):
    return torch.zeros(n, dtype=torch.float16)


def ints(*n):
    return torch.zeros(n, dtype=torch.int32)


def floats(*n):
    return torch.zeros(n)


CALLS = {
    "lora_add": (half(2, 16), 16, half(2 * 8 * 16), half(24 * 8), ints(1), floats(1), ints(2), ints(3), half(2, 24),
                 24, (8, 24), floats(4096), 2, 2, 1, 8, 16, 0),
    "rotary_apply": (half(2, 32), 32, half(2, 16), 16, ints(2), floats(2, 8), ints(2), floats(2), 2, 2, 1, 16, 16,
                     1, 0),
    "qkv_rotary_scatter": (half(2, 64), 64, half(64), half(256), half(256), ints(2), ints(2), floats(2, 8),
                           ints(2), floats(2), 2, 1, 16, 2, 1, 16, 16, 0, 0),
    "kv_copy_pages": ([half(4, 8), ints(4, 4)], ints(2), ints(2), 1, 4, 0),
    "kv_fork": (ints(4) - 1, ints(2), ints(2), ints(2), ints(4), ints(4), ints(2), ints(4), ints(2), ints(64), 2, 2,
                2, 16, 4, 0),
    "kv_compact": (ints(4), ints(8), ints(4), ints(8), ints(8), ints(2), ints(512), 2, 2, 8, 0),
}
FREQUENCIES = {("rotary_apply", 5), ("qkv_rotary_scatter", 7)}  # fewer of them are fewer tables
# also workspaces larger than they need be, pools whose pages are not counted here, one count of two
ANY_SIZE = FREQUENCIES | {("lora_add", 11), ("kv_fork", 9), ("kv_compact", 6), ("qkv_rotary_scatter", 3),
                          ("qkv_rotary_scatter", 4), ("kv_copy_pages", 2), ("rotary_apply", 7),
                          ("qkv_rotary_scatter", 9)}
OPTIONAL = {"lora_add": (4, 5, 7), "rotary_apply": (6, 7), "qkv_rotary_scatter": (8, 9), "kv_copy_pages": (2,),
            "kv_fork": (3,), "kv_compact": ()}


@pytest.mark.parametrize("name", CALLS)
def test_no_answer_for_anything_but_cuda_tensors(llmk, name):
    f, args = getattr(llmk._fast, name), CALLS[name]
    assert f(*args) is None  # CPU tensors
    assert f(*args[:-1]) is None and f(*args, 0) is None  # too few and too many arguments
    for i in range(len(args)):
        for bad in (None, "x", -1, 0, 1 << 70, 1.5, object(), (), [], (1,) * 9, (0,), ("x",)):
            if name == "kv_copy_pages" and i == 0 and bad == []:
                continue
            assert f(*args[:i], bad, *args[i + 1:]) is None


def here(a):
    if isinstance(a, list):
        return [t.cuda() for t in a]
    return a.cuda() if isinstance(a, torch.Tensor) else a


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_an_answer_for_what_is_right_and_none_for_each_thing_that_is_not(llmk, name):
    f = getattr(llmk._fast, name)
    args = [here(a) for a in CALLS[name]]
    args[-1] = None
    assert f(*args) == 0
    for i in OPTIONAL[name]:
        assert f(*args[:i], None, *args[i + 1:]) == 0
    torch.cuda.synchronize()
    for i, a in enumerate(args):
        if not isinstance(a, torch.Tensor):
            continue
        wrong = [a.cpu(), a.double(), "x"]
        if a.numel() > 1:
            wrong.append(torch.stack([a, a], -1)[..., 0])
        if a.numel() > 1 and (name, i) not in ANY_SIZE:
            wrong.append(a.reshape(-1)[:-1])
        if (name, i) in FREQUENCIES:  # less than one table's
            wrong.append(a.reshape(-1)[:7])
        for bad in wrong:
            assert f(*args[:i], bad, *args[i + 1:]) is None, (i, bad)
    if name == "kv_copy_pages":
        for bad in ([half(4, 8)], [args[0][0].reshape(-1)[:9]], [args[0][0].t()], ["x"], [None], args[0] * 200, tuple(args[0])):
            assert f(bad, *args[1:]) is None
    if name == "lora_add":
        wide = torch.zeros(2, 64, dtype=torch.float16, device="cuda")
        assert f(wide[:, 8:24], 64, *args[2:]) == 0 and f(wide[:, 8:24], 32, *args[2:]) is None
        assert f(wide[:, :32:2], 64, *args[2:]) is None and f(wide[:1], 64, *args[2:]) is None
        for ends in ((8,) * 9, (), [8, 24], (8, 2 ** 31), (8.0, 24)):
            assert (f(*args[:10], ends, *args[11:]) == 0) == (ends == [8, 24])
    torch.cuda.synchronize()
