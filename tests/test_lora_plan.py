"""The launches of lora_add by its sizes, over the whole range that it takes. On the CPU."""
import math
import random

import pytest

from _lora_plan import plans
from _lora_variants import SIZES, Sizes

MOST = 1 << 20


def drawn(seed, n):
    rng = random.Random(seed)

    def size(lo, hi):
        return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))
    calls = []
    for _ in range(n):
        rows = size(1, MOST)
        seqs = rng.choice([rows, size(1, MOST), size(1, 300)])
        ends, at = [], 0
        for _ in range(rng.randint(1, 8)):
            at += 8 * size(1, 65535 * 64 // 8)
            ends.append(at)
        calls.append((rows, seqs, size(1, 2 ** 31 - 1), 8 * rng.randint(1, 32), 8 * size(1, 1 << 21), tuple(ends)))
    return calls


LARGEST = [(MOST, MOST, 1 << 19, 16, 64, (8192,)), (MOST, MOST, 1 << 19, 16, 64, (8,)),
           (MOST, MOST, (1 << 31) - 1, 8, 8, (131072,)), (MOST, MOST, 1 << 20, 256, 1 << 24, (8, 16)),
           (1, MOST, 1 << 30, 32, 64, (4096, 8192)), (MOST, 1, 1, 8, 8, (8,)), (1, 1, 1, 8, 8, (8,)),
           (MOST, MOST, 256, 8, 64, (1024,)), (300000, 300000, 12000000, 16, 512, (2048,)),
           (1, 1, 49, 16, 64, (1 << 20,)), (1, 1, 2 ** 31 - 1, 16, 64, (1 << 20,)),
           (MOST, MOST, 256, 16, 64, (1 << 17,)), (MOST, MOST, 256, 256, 64, (1 << 16,)),
           (MOST, MOST, 256, 128, 64, (65535 * 512,)), (MOST, MOST, 256, 136, 64, (65535 * 256,))]


@pytest.mark.parametrize("calls", [LARGEST, drawn(1, 4000)], ids=["largest", "drawn"])
def test_estimates_and_grids(tmp_path, calls):
    """The estimates are those of the formulas, whatever the sizes; one launch is for few blocks, and every launch
    has blocks for all slots."""
    for call, p in zip(calls, plans(tmp_path, calls), strict=True):
        rows, seqs, adapters, rank, inner, ends = call
        n = min(seqs, 256)
        some = -(-seqs // 256) * (adapters * -math.expm1(n * math.log1p(-1 / adapters)) if adapters > 1 else 1)
        likely = max(some, rows / 16 + 0.5 * (some - 1))
        assert likely - 1 - 1e-6 * likely <= p["likely"] <= likely * (1 + 1e-6) and p["likely"] >= 1, (call, p)
        assert p["likely"] <= p["many"] + 1 and p["many"] >= p["windows"] * p["groups"]
        widths = [b - a for a, b in zip((0,) + ends, ends)]
        if p["one"]:
            assert rank <= 32 and p["likely"] * p["blocks"] <= 256 + 7 * p["blocks"]
            assert p["blocks"] == sum(-(-w // (128 * p["tiles"])) for w in widths)
            assert p["slots"] * p["blocks"] <= p["grid"] <= 4096, (call, p)
        else:
            assert p["grid"] == p["slots"] * p["splits"] * p["turns"] < 2 ** 32 // 256
            chunks = sum(-(-w // (512 if rank <= 128 else 256)) for w in widths)
            assert p["grid2"] == chunks * -(-p["slots"] // p["per_block"]) < 2 ** 32 // 256


def test_the_gpu_tests_take_every_way(tmp_path):
    """The cases of _lora_variants.py between them run every kernel of lora_add in every manner that the sizes choose."""
    calls = [Sizes(i).call() for i in range(len(SIZES))]
    one, two = set(), set()
    for (rows, seqs, adapters, rank, inner, ends), p in zip(calls, plans(tmp_path, calls), strict=True):
        if p["one"]:
            one |= {(p["tiles"], (rank + 15) // 16), ("together", p["together"]), ("wave", seqs <= 64)}
            one |= {("together", p["tiles"], p["together"])}
        else:
            some, run = p["splits"], p["per_block"] > 1
            two |= {("at once", p["at_once"]), ("turns", p["turns"] > 1), ("wave", seqs <= 64), ("windows", p["windows"] > 1)}
            if p["steps"] <= 2:
                two.add((p["steps"], some > 2, run))
                two.add((p["steps"], some > 1))
            else:
                two.add((p["steps"], some > 4 if p["steps"] == 4 else some > 1, run))
    both = (False, True)
    assert one >= {(t, ng) for t in (2, 4, 8) for ng in (1, 2)} | {("wave", w) for w in both}
    assert one >= {("together", t, w) for t in (2, 4, 8) for w in (0, 1)}
    assert two >= {("at once", n) for n in (1, 2, 3)} | {(w, b) for w in ("turns", "wave", "windows") for b in both}
    assert two >= {(steps, some, run) for steps in (1, 2, 4, 8) for some in both for run in both}
    assert two >= {(steps, some) for steps in (1, 2) for some in both}
