"""Rows into the paged cache whose heads turn by a whole fraction that is no multiple of 16."""
import numpy as np
import pytest
import torch

from test_gpu_rotary import scatter_case, test_scatter, to

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("n,heads,kv,dim,rotary,page,max_pages", [
    (1, 16, 16, 80, 20, 16, 3), (7, 16, 16, 80, 40, 16, 2), (300, 5, 2, 80, 20, 16, 2), (2001, 16, 16, 80, 40, 16, 1),
    (5, 2, 1, 64, 8, 8, 4), (9, 3, 1, 16, 2, 1, 9), (33, 1, 1, 16, 4, 16, 2), (6, 40, 8, 144, 72, 16, 2),
    (4, 2, 2, 512, 8, 16, 2), (3, 150, 3, 240, 60, 32, 2), (70, 1, 1, 400, 200, 16, 1), (601, 4, 2, 48, 6, 16, 1)])
def test_fractions(llmk, pairs, n, heads, kv, dim, rotary, page, max_pages):
    test_scatter(llmk, pairs, n, heads, kv, dim, rotary, page, max_pages)


@pytest.mark.parametrize("pairs", [False, True])
def test_as_in_place(llmk, pairs):
    """Bit for bit what rotary_apply gives, with one table and with several, and behind a graph."""
    rng = np.random.default_rng(8)
    n, heads, kv, dim, rotary = 19, 6, 3, 80, 20
    num_pages, table, pos, x, inv, t, s = scatter_case(rng, n, heads, kv, dim, rotary, 16, 2, 3)
    layout, dev = int(pairs), to(x, np.float16)
    d = {k: to(v, np.int32) for k, v in (("pos", pos), ("table", table), ("t", t))}
    inv, s = to(inv, np.float32), to(s, np.float32)
    q = torch.zeros((n, heads, dim), dtype=torch.float16, device="cuda")
    kp = torch.zeros((num_pages, 16, kv, dim), dtype=torch.float16, device="cuda")
    vp = torch.zeros_like(kp)

    def step(ids, scales, table_of):
        llmk.qkv_rotary_scatter(dev, x.shape[1], q, kp, vp, d["table"], d["pos"], table_of, ids, scales, n, 2, 16, heads,
                                kv, dim, rotary, layout)
    page = torch.from_numpy(table[np.arange(n), pos // 16].astype(np.int64)).cuda()
    for args in ((None, None, inv[0]), (d["t"], s, inv)):
        step(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(*args)
        for turn in range(3):
            d["pos"].copy_(to((pos + turn) % 16 + pos // 16 * 16, np.int32))
            want = dev.clone()
            llmk.rotary_apply(want, x.shape[1], want[:, heads * dim:], x.shape[1], d["pos"], args[2], args[0], args[1], n,
                              heads, kv, dim, rotary, layout)
            q.zero_(), kp.zero_()
            graph.replay()
            torch.cuda.synchronize()
            want = want[:, :(heads + kv) * dim].view(n, -1, dim)
            assert torch.equal(q, want[:, :heads])
            assert torch.equal(kp[page, (d["pos"] % 16).long()], want[:, heads:])
    with pytest.raises(llmk.LlmkError):
        llmk.qkv_rotary_scatter(dev, x.shape[1], q, kp, vp, d["table"], d["pos"], inv, None, None, n, 2, 16, heads, kv, dim,
                                24, layout)
