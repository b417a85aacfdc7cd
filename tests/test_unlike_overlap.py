"""Arrays that overlap where one of them is written: what the entry points for adapters and rotary layouts refuse. At
the C-ABI, on the CPU: no call gets as far as a launch."""
import pytest

from test_unlike_refusals import ints, lora, rotary

AT = 1 << 24


def spread(names):
    return {name: AT * (i + 1) for i, name in enumerate(names)}


APART = spread(("x", "a", "b", "ranks", "scales", "ids", "starts", "y", "ws"))
# bytes of 4 rows, 2 sequences and 3 adapters of rank 16, 64 -> 32|48 columns
SIZES = dict(x=2 * (3 * 64 + 64), a=2 * 3 * 2 * 16 * 64, b=2 * 3 * 48 * 16, ranks=12, scales=12, ids=8, starts=12,
             y=2 * (3 * 48 + 48))


@pytest.mark.parametrize("other", ["a", "b", "ranks", "scales", "ids", "starts", "ws"])
def test_lora_add_y_over_another(llmk, other):
    L, E = llmk.lib(), llmk
    size = SIZES.get(other) or 4 * llmk.lora_add_workspace_floats(4, 2, 3, 16, 64, 2)
    last = APART[other] + (size - 1) // 16 * 16  # the last 16-byte address within it
    first = APART[other] - (SIZES["y"] - 16)
    for y in (APART[other], last, first):
        assert lora(L, **APART | dict(y=y)) == E.LLMK_ERR_INVALID_VALUE, y - APART[other]


@pytest.mark.parametrize("other", ["x", "a", "b", "ranks", "scales", "ids", "starts"])
def test_lora_add_workspace_over_another(llmk, other):
    L, E = llmk.lib(), llmk
    size = 4 * llmk.lora_add_workspace_floats(4, 2, 3, 16, 64, 2)
    for ws in (APART[other], APART[other] + (SIZES[other] - 1) // 16 * 16, APART[other] - (size - 16)):
        assert lora(L, **APART | dict(ws=ws)) == E.LLMK_ERR_INVALID_VALUE, ws - APART[other]


@pytest.mark.parametrize("behind", [0, 4096 - 64 + 8])
def test_lora_add_over_a_row_of_y(llmk, behind):
    """B of 64 numbers at a row's last columns, and reaching into the next row."""
    wide = dict(ldy=4096, n_adapters=1, rank=8, ends=ints(8), parts=1)
    assert lora(llmk.lib(), **APART | wide | dict(b=APART["y"] + 2 * behind)) == llmk.LLMK_ERR_INVALID_VALUE


@pytest.mark.parametrize("behind,sizes", [
    (0, {}), (2 * 31, {}), (2 * 4 * 256 - 2 * 128, {}), (-2 * 64, {}), (-2 * 95, {}),  # heads of 64, of which 32 turn
    (2 * (3 * 256 + 3 * 64 + 31), dict(n=5)), (2 * 200, dict(ldk=136)), (2 * 3 * 256, dict(heads=1, kv=1, ldk=64)),
    (2 * (512 - 64), dict(ldq=512, ldk=512)), (2 * 40, dict(rot=64)), (-2 * 3 * 256, dict(ldk=256))])
def test_rotary_apply_q_over_k(llmk, behind, sizes):
    """What one head's turned part shares with another's, in the same row, in the next, or across strides."""
    a = dict(n=4, ldq=256, ldk=256, q=AT, k=AT + behind) | sizes
    assert rotary(llmk.lib(), **a) == llmk.LLMK_ERR_INVALID_VALUE
