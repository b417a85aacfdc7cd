"""The operators of serving requests that are not alike, as cases that a program can time and check:
low-rank adapters beside a shared projection, rotary positions of several layouts and scalings, and
forking and compacting the pages of a cache.

`listed()` names the cases, `draw(rng)` gives more of the same ranges, `prepare` makes what a program
holds before the call, `run` is one pass (the operators in elementary torch where `own` is false,
through the framework's entry points where it is true), `work` what a pass cannot do without and
`exact` its result from the definition.

Adapters: sequence s owns rows row_starts[s] up to row_starts[s + 1] (None: one row each) and has
adapter ids[s] (-1: none). A projection may be a fused one of several parts (q, k and v; gate and
up): an adapter has an A [rank, in] for each part and one B [out, rank] for all of them.
Cache pages: holders are counted in `refs`; a sequence holds the pages that its table row names up to
the first negative entry. Tokens fill pages of 16 in order.

Shapes are those of the repository's model (hidden 2048, 32 query and 8 kv heads of 64, 8192 inner, 16
layers) and generic ones around it.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
PAGE = 16
THETA = 500000.0


def listed():
    return [
        # One sequence's decode step, the attention's output projection: launches and little else.
        dict(name="lora_1", kind="lora", seqs=1, rows=1, ragged=False, adapters=4, rank=16,
             mixed=False, inner=2048, parts="2048"),
        # Drafted rows of a batch on a q|k|v projection, a few adapters.
        dict(name="lora_drafts", kind="lora", seqs=48, rows=5, ragged=True, adapters=16, rank=16,
             mixed=False, inner=4096, parts="4096,1024,1024"),
        # A full batch on the down projection, nearly as many adapters as sequences.
        dict(name="lora_256", kind="lora", seqs=256, rows=1, ragged=False, adapters=100, rank=64,
             mixed=True, inner=8192, parts="2048"),
        # Prompts that arrive together, on the gate|up projection.
        dict(name="lora_prompts", kind="lora", seqs=4, rows=1001, ragged=True, adapters=8, rank=32,
             mixed=True, inner=2048, parts="8192,8192"),
        # Queries and keys of one new token, rotated where they lie: pairs, a quarter of the head.
        dict(name="rotary_1", kind="rotary", rows=1, heads=32, kv=8, dim=128, rotary=32, pairs=True,
             tables=1, max_pos=700),
        # A prompt's chunk, whole heads as halves, two scalings side by side.
        dict(name="rotary_4001", kind="rotary", rows=4001, heads=32, kv=8, dim=64, rotary=64,
             pairs=False, tables=2, max_pos=131072),
        # A full batch's decode step into the paged cache.
        dict(name="scatter_256", kind="scatter", rows=256, heads=32, kv=8, dim=64, rotary=64,
             pairs=False, tables=3, max_pos=8192, prompt=False),
        # A prompt into the paged cache, wide heads, half of each rotated as pairs.
        dict(name="scatter_prompt", kind="scatter", rows=2001, heads=28, kv=4, dim=128, rotary=64,
             pairs=True, tables=1, max_pos=4096, prompt=True),
        # Two requests of four beams each: one step of their search, all layers' pages.
        dict(name="fork_8", kind="fork", groups=2, beams=4, max_len=301, layers=16, kv=8, dim=64,
             small=False, spare=64),
        # A full batch of beams over an 8-bit cache.
        dict(name="fork_256", kind="fork", groups=64, beams=4, max_len=2048, layers=16, kv=8, dim=64,
             small=True, spare=2000),
        # A young server's cache, a few sequences gone.
        dict(name="compact_5", kind="compact", seqs=5, max_len=501, free=0.3, layers=2, kv=8, dim=64,
             small=False),
        # A long-running server's cache, half of it free, before its pools are cut.
        dict(name="compact_64", kind="compact", seqs=64, max_len=511, free=0.5, layers=8, kv=8,
             dim=64, small=False),
    ]


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], uniform over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return min(hi, max(lo, int(v)))


def draw(rng):
    kind = rng.choice(["lora", "lora", "rotary", "scatter", "fork", "compact"])
    heads, kv, dim = rng.choice([(32, 8, 64), (32, 8, 128), (20, 20, 64), (28, 4, 128), (12, 2, 64),
                                 (8, 1, 256), (16, 16, 80)])
    if kind == "lora":
        while True:
            what = rng.choice(["decode", "decode", "drafts", "prompt"])
            seqs = _log_int(rng, 1, 5 if what == "prompt" else 256)
            rows = dict(decode=1, drafts=rng.randint(2, 9),
                        prompt=_log_int(rng, 10, 2000 // seqs))[what]
            case = dict(kind=kind, seqs=seqs, rows=rows, ragged=rows > 1 and rng.random() < 0.5,
                        adapters=_log_int(rng, 1, 120), rank=rng.choice([8, 16, 16, 24, 32, 64, 128]),
                        mixed=rng.random() < 0.5, inner=rng.choice([1024, 2048, 4096, 4104, 8192]),
                        parts=rng.choice(["2048", "1000", "8192,8192", "4096,1024,1024",
                                          "2560,2560,2560", "512,512", "11008,11008"]))
            w = work(case)
            if w["bytes"] <= 190e6 and case["adapters"] * case["rank"] <= 6400:
                return case
    if kind in ("rotary", "scatter"):
        wide = max(1.0, (heads + 2 * kv) * dim / 3000)
        case = dict(kind=kind, rows=_log_int(rng, 1, int(4000 / wide)), heads=heads, kv=kv, dim=dim,
                    rotary=rng.choice([dim, dim, dim // 2, dim // 4]), pairs=rng.random() < 0.5,
                    tables=rng.choice([1, 1, 2, 7]), max_pos=rng.choice([300, 8192, 131072, 1000000]))
        if kind == "scatter":
            case["prompt"] = rng.random() < 0.5
            case["max_pos"] = max(min(case["max_pos"], 32768), case["rows"] + 16)
        return case
    small = rng.random() < 0.4
    layers = rng.choice([1, 2, 4, 8])
    page = PAGE * kv * dim * (1 if small else 2) * 2 * layers  # bytes of a page in all pools
    pages = min(2200, 500_000_000 // page)  # of the whole cache
    if kind == "fork":
        groups, beams = _log_int(rng, 1, 48), rng.choice([1, 2, 3, 4, 5, 8])
        most = max(1, (pages - 30 - 2 * groups * beams) // groups)
        if most < 2:
            groups, most = 2, max(2, (pages - 30 - 4 * beams) // 2)
        return dict(kind=kind, groups=groups, beams=beams,
                    max_len=_log_int(rng, 1, PAGE * min(most, 200)), layers=layers, kv=kv, dim=dim,
                    small=small, spare=rng.randint(30, 200))
    seqs, free = _log_int(rng, 1, 100), rng.uniform(0.05, 0.8)
    most = max(1, int(pages * (1 - free)) // seqs - 1)
    return dict(kind=kind, seqs=seqs, max_len=_log_int(rng, 1, PAGE * min(most, 200)), free=free,
                layers=layers, kv=kv, dim=dim, small=small)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _parts(case):
    return [int(p) for p in case["parts"].split(",")]


def _lora_sizes(case):
    """(rows of each sequence, adapter of each sequence, rank of each adapter): fixed by the case, so
    that its work is. Popular adapters are asked for more often; one sequence in ten has none."""
    r = np.random.default_rng([case["seqs"], case["rows"], case["adapters"], case["rank"]])
    n, k = case["seqs"], case["adapters"]
    rows = r.integers(1, case["rows"] + 1, n) if case["ragged"] else np.full(n, case["rows"])
    rows[r.integers(0, n)] = case["rows"]
    ids = np.minimum((k * r.random(n) ** 1.5).astype(np.int64), k - 1)
    ids[(r.random(n) < 0.1) & (np.arange(n) > 0)] = -1
    ranks = np.full(k, case["rank"])
    if case["mixed"]:  # of full rank, of half or of a quarter
        ranks = np.maximum(ranks >> r.integers(0, 3, k), 1)
    return rows, ids, ranks


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(shape, g, std=1.0):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).mul_(std)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def prepare(case, seed):
    return _PREPARE[case["kind"]](case, np.random.default_rng(seed), _gen(seed))


def _prepare_lora(case, rng, g):
    rows, ids, ranks = _lora_sizes(case)
    n, k, rank, inner, parts = (case["seqs"], case["adapters"], case["rank"], case["inner"],
                                _parts(case))
    n_rows, out = int(rows.sum()), sum(parts)
    # which sequence asks for which adapter differs from seed to seed, how often does not
    order = rng.permutation(k)
    ranks = ranks[np.argsort(order)]
    ids = np.where(ids >= 0, order[ids], -1)
    s = dict(kind="lora", n_rows=n_rows, n_seqs=n, n_adapters=k, max_rank=rank, inner=inner, out=out,
             parts=parts, part_ends=[int(e) for e in np.cumsum(parts)],
             row_starts=None if case["rows"] == 1 else _ints(np.concatenate([[0], np.cumsum(rows)])),
             ids=_ints(ids), ranks=_ints(ranks))
    s["x"] = _normal((n_rows, inner), g).half()
    s["y"] = _normal((n_rows, out), g).half()  # the shared projection's output
    s["a"] = _normal((k, len(parts), rank, inner), g, inner ** -0.5).half()
    s["b"] = _normal((k, out, rank), g, 0.3 * rank ** -0.5).half()
    s["scales"] = 0.5 + 1.5 * torch.rand(k, generator=g, device=DEV)
    return s


def _inv_freq(case, rng):
    """Frequency tables as models scaled for longer contexts have them: the first as trained, others
    interpolated by a factor, low frequencies more than high ones."""
    half = case["rotary"] // 2
    base = THETA ** (-np.arange(half) / half)
    ramp = np.linspace(0.0, 1.0, half)
    factors = np.concatenate([[1.0], rng.uniform(1.5, 40.0, case["tables"] - 1)])
    table = base * (1 - ramp + ramp / factors[:, None])
    return (torch.from_numpy(table.astype(np.float32)).to(DEV),
            torch.from_numpy((0.1 * np.log(factors) + 1.0).astype(np.float32)).to(DEV))


def _prepare_rotary(case, rng, g):
    n, heads, kv, dim = case["rows"], case["heads"], case["kv"], case["dim"]
    s = dict(kind=case["kind"], n_rows=n, heads=heads, kv=kv, dim=dim, rotary=case["rotary"],
             pairs=case["pairs"])
    s["inv_freq"], s["scales"] = _inv_freq(case, rng)
    s["table_ids"] = None if case["tables"] == 1 else _ints(rng.integers(0, case["tables"], n))
    s["qkv"] = _normal((n, (heads + 2 * kv) * dim), g).half()
    first = int(rng.integers(0, max(1, case["max_pos"] - n)))
    prompt = case.get("prompt", n > 256)
    pos = first + np.arange(n) if prompt else rng.integers(0, case["max_pos"], n)
    if case["kind"] == "rotary":
        s["positions"] = _ints(pos)
        return s
    # the pages written are the pool's first ones, shuffled; pages read elsewhere are not here
    if prompt:
        used = np.unique(pos // PAGE)
        table = np.zeros(int(used[-1]) + 1, np.int64)
        table[used] = rng.permutation(used.size)
        tables, num_pages = np.tile(table, (n, 1)), used.size
        # one sequence's rows of one prompt share a table row, repeated as the batch has it
    else:
        widest = int(pos.max()) // PAGE + 1
        tables, num_pages = np.zeros((n, widest), np.int64), n
        tables[np.arange(n), pos // PAGE] = rng.permutation(n)
    s.update(positions=_ints(pos), tables=_ints(tables), max_pages=tables.shape[1])
    s["k_pool"] = _normal((num_pages, PAGE, kv, dim), g).half()
    s["v_pool"] = _normal((num_pages, PAGE, kv, dim), g).half()
    s["q_out"] = torch.empty((n, heads, dim), dtype=torch.float16, device=DEV)
    return s


def _pools(case, num_pages, g, s):
    """Every layer's K and V pool behind one another: 16-bit values, or 8-bit ones with scales."""
    pools, width = 2 * case["layers"], PAGE * case["kv"] * case["dim"]
    bits = torch.int8 if case["small"] else torch.int16
    top = 128 if case["small"] else 32768
    s["pools"] = torch.randint(-top, top, (pools, num_pages, width), generator=g, device=DEV,
                               dtype=bits)
    s["pool_scales"] = None
    if case["small"]:
        s["pool_scales"] = torch.randint(0, 1 << 30, (pools, num_pages, case["kv"]), generator=g,
                                         device=DEV, dtype=torch.int32)
    s["num_pages"] = num_pages


def _fork_sizes(case):
    """(length of each group, parent of each child): fixed by the case."""
    r = np.random.default_rng([case["groups"], case["beams"], case["max_len"]])
    n, b = case["groups"], case["beams"]
    lens = r.integers(1, case["max_len"] + 1, n)
    lens[r.integers(0, n)] = case["max_len"]
    parents = (np.arange(n)[:, None] * b + r.integers(0, b, (n, b))).reshape(-1)
    return lens, parents


def _prepare_fork(case, rng, g):
    lens, parents = _fork_sizes(case)
    n, b = case["groups"], case["beams"]
    full, part = lens // PAGE, (lens % PAGE > 0).astype(np.int64)
    live = int((full + b * part).sum())
    num_pages, widest = live + case["spare"], case["max_len"] // PAGE + 1
    order, at = rng.permutation(num_pages), 0
    tables, refs = np.full((n * b, widest), -1), np.zeros(num_pages, np.int64)
    for i in range(n):  # beams share the full pages and have a last one each
        shared = order[at:at + full[i]]
        at += full[i]
        tables[i * b:(i + 1) * b, :full[i]] = shared
        refs[shared] = b
        if part[i]:
            tables[i * b:(i + 1) * b, full[i]] = order[at:at + b]
            refs[order[at:at + b]] = 1
            at += b
    s = dict(kind="fork", n=n * b, max_pages=widest, tables=_ints(tables), refs=_ints(refs),
             lens=_ints(np.repeat(lens, b)), parents=_ints(parents),
             reserve=_ints(np.ones(n * b)))  # room for the next token
    s["new_tables"], s["new_lens"] = torch.empty_like(s["tables"]), torch.empty_like(s["lens"])
    s["copies"] = torch.empty((n * b, 2), dtype=torch.int32, device=DEV)
    s["counts"] = torch.empty(2, dtype=torch.int32, device=DEV)
    _pools(case, num_pages, g, s)
    return s


def _compact_sizes(case):
    """(pages of each sequence, pages of the pool, live pages at or past the count of live ones in
    expectation): fixed by the case. Odd sequences continue the even one in front, whose first half
    they share."""
    r = np.random.default_rng([case["seqs"], case["max_len"]])
    lens = r.integers(1, case["max_len"] + 1, case["seqs"])
    lens[r.integers(0, case["seqs"])] = case["max_len"]
    pages = (lens + PAGE - 1) // PAGE
    shared = np.zeros_like(pages)
    shared[1::2] = np.minimum(pages[0::2][:pages[1::2].size], pages[1::2]) // 2
    live = int((pages - shared).sum())
    return pages, shared, live, live + int(live * case["free"] / (1 - case["free"])) + 1


def _prepare_compact(case, rng, g):
    pages, shared, live, num_pages = _compact_sizes(case)
    order, at = rng.permutation(num_pages), 0
    tables = np.full((case["seqs"], int(pages.max())), -1)
    refs = np.zeros(num_pages, np.int64)
    for i, (k, m) in enumerate(zip(pages, shared)):
        if m:
            tables[i, :m] = tables[i - 1, :m]
        tables[i, m:k] = order[at:at + k - m]
        at += k - m
        refs[tables[i, :k]] += 1
    s = dict(kind="compact", n=case["seqs"], max_pages=tables.shape[1], tables=_ints(tables),
             refs=_ints(refs))
    s["new_tables"], s["new_refs"] = torch.empty_like(s["tables"]), torch.empty_like(s["refs"])
    s["copies"] = torch.empty((num_pages // 2, 2), dtype=torch.int32, device=DEV)
    s["counts"] = torch.empty(2, dtype=torch.int32, device=DEV)
    _pools(case, num_pages, g, s)
    return s


_PREPARE = dict(lora=_prepare_lora, rotary=_prepare_rotary, scatter=_prepare_rotary,
                fork=_prepare_fork, compact=_prepare_compact)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(s):
    return (_OWN if own else _PLAIN)[s["kind"]](s)


def _llmk():
    from __graft_entry__ import load_llmk
    return load_llmk()


def _own_lora(s):
    llmk = _llmk()
    if "workspace" not in s:  # a program keeps one
        s["workspace"] = torch.empty(llmk.lora_add_workspace_floats(
            s["n_rows"], s["n_seqs"], s["n_adapters"], s["max_rank"], s["inner"], len(s["parts"])),
            device=DEV)
    llmk.lora_add(s["x"], s["inner"], s["a"], s["b"], s["ranks"], s["scales"], s["ids"],
                  s["row_starts"], s["y"], s["out"], s["part_ends"], s["workspace"], s["n_rows"],
                  s["n_seqs"], s["n_adapters"], s["max_rank"], s["inner"])
    return s["y"]


def _own_rotary(s):
    llmk, qkv = _llmk(), s["qkv"]
    llmk.rotary_apply(qkv, qkv.shape[1], qkv[:, s["heads"] * s["dim"]:], qkv.shape[1],
                      s["positions"], s["inv_freq"], s["table_ids"], s["scales"], s["n_rows"],
                      s["heads"], s["kv"], s["dim"], s["rotary"],
                      llmk.ROTARY_PAIRS if s["pairs"] else llmk.ROTARY_HALVES)
    return qkv


def _own_scatter(s):
    llmk = _llmk()
    llmk.qkv_rotary_scatter(s["qkv"], s["qkv"].shape[1], s["q_out"], s["k_pool"], s["v_pool"],
                            s["tables"], s["positions"], s["inv_freq"], s["table_ids"], s["scales"],
                            s["n_rows"], s["max_pages"], PAGE, s["heads"], s["kv"], s["dim"],
                            s["rotary"], llmk.ROTARY_PAIRS if s["pairs"] else llmk.ROTARY_HALVES)
    return s["q_out"], s["k_pool"], s["v_pool"]


def _pool_list(s):
    if "pool_list" not in s:  # a program holds its layers' pools one by one
        s["pool_list"] = list(s["pools"].unbind(0))
        if s["pool_scales"] is not None:
            s["pool_list"] += list(s["pool_scales"].unbind(0))
    return s["pool_list"]


def _next_batch(s):
    """What a search does behind a fork: the children are the next step's parents."""
    s["tables"], s["new_tables"] = s["new_tables"], s["tables"]
    s["lens"], s["new_lens"] = s["new_lens"], s["lens"]
    return s["tables"], s["lens"], s["refs"], s["counts"], s["pools"], s["pool_scales"]


def _own_fork(s):
    llmk = _llmk()
    if "workspace" not in s:
        s["workspace"] = torch.empty(llmk.kv_fork_workspace_ints(
            s["n"], s["n"], s["max_pages"], s["num_pages"]), dtype=torch.int32, device=DEV)
    llmk.kv_fork(s["tables"], s["lens"], s["parents"], s["reserve"], s["refs"], s["new_tables"],
                 s["new_lens"], s["copies"], s["counts"], s["workspace"], s["n"], s["n"],
                 s["max_pages"], PAGE, s["num_pages"])
    llmk.kv_copy_pages(_pool_list(s), s["copies"], None, s["n"], s["num_pages"])
    return _next_batch(s)


def _own_compact(s):
    llmk = _llmk()
    if "workspace" not in s:
        s["workspace"] = torch.empty(llmk.kv_compact_workspace_ints(s["num_pages"]),
                                     dtype=torch.int32, device=DEV)
    llmk.kv_compact(s["tables"], s["refs"], s["new_tables"], s["new_refs"], s["copies"], s["counts"],
                    s["workspace"], s["n"], s["max_pages"], s["num_pages"])
    llmk.kv_copy_pages(_pool_list(s), s["copies"], s["counts"], s["num_pages"] // 2,
                       s["num_pages"])
    return s["new_tables"], s["new_refs"], s["counts"], s["pools"], s["pool_scales"]


_OWN = dict(lora=_own_lora, rotary=_own_rotary, scatter=_own_scatter, fork=_own_fork,
            compact=_own_compact)


def _plain_lora(s):
    k, rank, parts, n_rows = s["n_adapters"], s["max_rank"], s["parts"], s["n_rows"]
    if s["row_starts"] is None:
        mine = s["ids"].long()
    else:
        r = torch.arange(n_rows, device=DEV)
        mine = s["ids"].long()[torch.searchsorted(s["row_starts"].long()[1:].contiguous(), r,
                                                  right=True)]
    # every row through every adapter, of which it keeps its own
    h = (s["x"].float() @ s["a"].float().view(-1, s["inner"]).T).view(n_rows, k, len(parts), rank)
    keep = (mine[:, None] == torch.arange(k, device=DEV))[:, :, None] \
        & (torch.arange(rank, device=DEV) < s["ranks"][:, None])
    h = torch.where(keep[:, :, None], h * s["scales"][:, None, None], 0.0)
    b = s["b"].float()
    add = torch.cat([h[:, :, p].reshape(n_rows, -1)
                     @ b[:, end - parts[p]:end].transpose(1, 2).reshape(k * rank, parts[p])
                     for p, end in enumerate(s["part_ends"])], 1)
    s["y"].copy_(s["y"].float() + add)
    return s["y"]


def _turned(s):
    """The queries and keys of qkv [rows, heads, dim], rotated, in 32 bits; angles in 64."""
    n, half, heads = s["n_rows"], s["rotary"] // 2, s["heads"] + s["kv"]
    table = 0 if s["table_ids"] is None else s["table_ids"].long()
    angle = s["positions"].double()[:, None] * s["inv_freq"][table].double()
    scale = s["scales"][table].view(-1, 1, 1)
    c, sn = torch.cos(angle).float()[:, None] * scale, torch.sin(angle).float()[:, None] * scale
    x = s["qkv"].view(n, -1, s["dim"])[:, :heads].float()
    turn, rest = x[..., :2 * half], x[..., 2 * half:]
    if s["pairs"]:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    else:
        a, b = turn[..., :half], turn[..., half:]
        turn = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    return torch.cat([turn, rest], -1)


def _plain_rotary(s):
    heads = s["heads"] + s["kv"]
    s["qkv"].view(s["n_rows"], -1, s["dim"])[:, :heads] = _turned(s).half()
    return s["qkv"]


def _plain_scatter(s):
    x = _turned(s)
    s["q_out"].copy_(x[:, :s["heads"]])
    pos = s["positions"].long()
    page = s["tables"].long()[torch.arange(s["n_rows"], device=DEV), pos // PAGE]
    s["k_pool"][page, pos % PAGE] = x[:, s["heads"]:].half()
    s["v_pool"][page, pos % PAGE] = s["qkv"].view(s["n_rows"], -1, s["dim"])[:,
                                                                            s["heads"] + s["kv"]:]
    return s["q_out"], s["k_pool"], s["v_pool"]


def _copy(s, src, dst):
    s["pools"][:, dst] = s["pools"][:, src]
    if s["pool_scales"] is not None:
        s["pool_scales"][:, dst] = s["pool_scales"][:, src]


def _plain_fork(s):
    n, width, refs = s["n"], s["max_pages"], s["refs"]
    old, parents, at = s["tables"].long(), s["parents"].long(), torch.arange(s["max_pages"], device=DEV)
    held = (old >= 0).cumprod(1).bool()
    lens = s["lens"].long().clamp(min=0).minimum(PAGE * held.sum(1))[parents]
    full, need = (lens // PAGE)[:, None], ((lens + s["reserve"] + PAGE - 1) // PAGE)[:, None]
    child = torch.arange(n, device=DEV)
    first = torch.full((n,), n, device=DEV).scatter_reduce_(0, parents, child, "amin")[parents] == child
    theirs, has = old[parents], held[parents]
    alone = refs[theirs.clamp(min=0)] == 1
    shares = at < full
    keeps = (shares | (first[:, None] & alone & (at < need))) & has
    fresh = (at < need) & ~keeps
    # holders: the old rows let go, the new rows take
    change = torch.zeros(s["num_pages"], dtype=torch.int64, device=DEV)
    change.index_add_(0, old.clamp(min=0).flatten(), -held.flatten().long())
    change.index_add_(0, theirs.clamp(min=0).flatten(), keeps.flatten().long())
    refs += change.to(torch.int32)
    free = (refs == 0).nonzero()[:, 0]
    place = fresh.flatten().cumsum(0).view(n, width) - 1
    wanted = fresh.sum()
    given = fresh & (place < free.numel())
    new = torch.where(given, free[place.clamp(0, free.numel() - 1)], -1)
    refs[new[given]] = 1
    s["new_tables"].copy_(torch.where(keeps, theirs, new))
    s["new_lens"].copy_(lens)
    split = given & (at == full) & (lens % PAGE > 0)[:, None] & has
    _copy(s, theirs[split], new[split])
    got = given.sum()
    s["counts"].copy_(torch.stack([got, wanted - got]))
    return _next_batch(s)


def _plain_compact(s):
    old, refs = s["tables"].long(), s["refs"]
    live = refs > 0
    page, count = torch.arange(s["num_pages"], device=DEV), live.sum()
    src, dst = (live & (page >= count)).nonzero()[:, 0], (~live & (page < count)).nonzero()[:, 0]
    to = page.clone()
    to[src] = dst
    s["new_tables"].copy_(torch.where(old >= 0, to[old.clamp(min=0)], old))
    s["new_refs"].copy_(torch.where(live & (page < count), refs, 0))
    s["new_refs"][dst] = refs[src]
    _copy(s, src, dst)
    s["counts"].copy_(torch.stack([torch.full_like(count, src.numel()), count]))
    return s["new_tables"], s["new_refs"], s["counts"], s["pools"], s["pool_scales"]


_PLAIN = dict(lora=_plain_lora, rotary=_plain_rotary, scatter=_plain_scatter, fork=_plain_fork,
              compact=_plain_compact)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "lora":
        rows, ids, ranks = _lora_sizes(case)
        parts, inner, out = len(_parts(case)), case["inner"], sum(_parts(case))
        has = ids >= 0
        n_rows, asked = int(rows[has].sum()), int(ranks[np.unique(ids[has])].sum())
        turns = int((rows[has] * ranks[ids[has]]).sum())  # rank over all rows
        per_rank = parts * inner + out
        return dict(bytes=2 * n_rows * (inner + 2 * out) + 2 * asked * per_rank + 8 * case["seqs"]
                    + 8 * case["adapters"], flops=2 * turns * per_rank)
    if kind in ("rotary", "scatter"):
        n, heads, kv, dim, rot = (case[k] for k in ("rows", "heads", "kv", "dim", "rotary"))
        small = 8 * n + 2 * rot * case["tables"]
        flops = 3 * n * (heads + kv) * rot
        if kind == "rotary":  # what is not rotated stays where it is
            return dict(bytes=4 * n * (heads + kv) * rot + small, flops=flops)
        return dict(bytes=4 * n * (heads + 2 * kv) * dim + 4 * n + small, flops=flops)
    width = PAGE * case["kv"] * case["dim"] * (1 if case["small"] else 2)
    page = 2 * case["layers"] * (width + (4 * case["kv"] if case["small"] else 0))
    if kind == "fork":
        lens, parents = _fork_sizes(case)
        n = parents.size
        partly = np.repeat(lens % PAGE > 0, case["beams"])
        copies = int(partly.sum()) - int(partly[np.unique(parents)].sum())
        entries = int(np.repeat(lens // PAGE + 1, case["beams"]).sum())
        return dict(bytes=2 * page * copies + 8 * entries + 8 * entries + 24 * n, flops=4 * entries)
    pages, _, live, num_pages = _compact_sizes(case)
    moved = int(live * (num_pages - live) / num_pages)  # of shuffled pages, on average
    entries = int(pages.sum())
    return dict(bytes=2 * page * moved + 8 * entries + 8 * num_pages, flops=2 * num_pages + entries)


# ---------------------------------------------------------------------------------------------
# the definition
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed), case)


def _exact_lora(s, case):
    y, x = s["y"].double(), s["x"].double()
    starts = (np.arange(s["n_seqs"] + 1) if s["row_starts"] is None
              else s["row_starts"].cpu().numpy())
    ranks, ids = s["ranks"].tolist(), s["ids"].tolist()
    for a in sorted(set(ids) - {-1}):
        rows = torch.from_numpy(np.concatenate(
            [np.arange(starts[i], starts[i + 1]) for i in range(s["n_seqs"]) if ids[i] == a])).to(DEV)
        r, begin = ranks[a], 0
        for p, end in enumerate(s["part_ends"]):
            h = x[rows] @ s["a"][a, p, :r].double().T.contiguous()
            y[rows, begin:end] += float(s["scales"][a]) * (
                h @ s["b"][a, begin:end, :r].double().T.contiguous())
            begin = end
    return y


def _exact_turned(s):
    n, rot = s["n_rows"], s["rotary"]
    table = torch.zeros(n, dtype=torch.long, device=DEV) if s["table_ids"] is None \
        else s["table_ids"].long()
    x = s["qkv"].double().view(n, -1, s["dim"])
    out = x.clone()
    turning = x[:, :s["heads"] + s["kv"], :rot]
    turning = turning.unflatten(-1, (-1, 2) if s["pairs"] else (2, -1))
    a, b = turning.unbind(-1 if s["pairs"] else -2)
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()[table]
    z = torch.complex(a, b) * torch.polar(s["scales"].double()[table][:, None].expand_as(angle),
                                          angle)[:, None]
    out[:, :s["heads"] + s["kv"], :rot] = torch.stack(
        [z.real, z.imag], -1 if s["pairs"] else -2).flatten(-2)
    return out


def _exact_rotary(s, case):
    return _exact_turned(s).view(s["n_rows"], -1)


def _exact_scatter(s, case):
    x, heads, kv = _exact_turned(s), s["heads"], s["kv"]
    k, v = s["k_pool"].double(), s["v_pool"].double()
    pos, tables = s["positions"].cpu().numpy(), s["tables"].cpu().numpy()
    at = torch.from_numpy(tables[np.arange(pos.size), pos // PAGE].astype(np.int64) * PAGE
                          + pos % PAGE).to(DEV)
    k.view(-1, kv, s["dim"])[at] = x[:, heads:heads + kv]
    v.view(-1, kv, s["dim"])[at] = x[:, heads + kv:]
    return x[:, :heads], k, v


def _exact_copy(s, src, dst):
    src, dst = (torch.tensor(i, dtype=torch.long, device=DEV) for i in (src, dst))
    moved = [None if p is None else p.index_copy(1, dst, p.index_select(1, src))
             for p in (s["pools"], s["pool_scales"])]
    return moved


def _exact_fork(s, case):
    old, lens, refs = s["tables"].cpu().numpy(), s["lens"].tolist(), s["refs"].tolist()
    before, parents = list(refs), s["parents"].tolist()
    new, src, dst = np.full_like(old, -1), [], []
    held = [[p for p in row if p >= 0] for row in old.tolist()]
    for row in held:
        for p in row:
            refs[p] -= 1
    wanted, seen = [], set()
    for c, p in enumerate(parents):
        full, need = lens[p] // PAGE, -(-(lens[p] + 1) // PAGE)
        for j in range(need):
            page = held[p][j] if j < len(held[p]) else -1
            if page >= 0 and (j < full or (p not in seen and before[page] == 1)):
                new[c, j] = page
                refs[page] += 1
            else:
                wanted.append((c, j, page if j == full and lens[p] % PAGE else -1))
        seen.add(p)
    free = [p for p in range(s["num_pages"]) if refs[p] == 0]
    for (c, j, page), to in zip(wanted, free):
        new[c, j] = to
        refs[to] = 1
        if page >= 0:
            src.append(page)
            dst.append(to)
    got = min(len(wanted), len(free))
    return (_ints(new), _ints([lens[p] for p in parents]), _ints(refs),
            _ints([got, len(wanted) - got]), *_exact_copy(s, src, dst))


def _exact_compact(s, case):
    refs = s["refs"].tolist()
    live = [p for p in range(s["num_pages"]) if refs[p] > 0]
    to, n = {p: p for p in live}, len(live)
    holes = [p for p in range(n) if refs[p] == 0]
    src = [p for p in live if p >= n]
    new = [refs[p] if p < n else 0 for p in range(s["num_pages"])]
    for p, hole in zip(src, holes):
        to[p], new[hole] = hole, refs[p]
    tables = [[to[p] if p >= 0 else p for p in row] for row in s["tables"].tolist()]
    return _ints(tables), _ints(new), _ints([len(src), n]), *_exact_copy(s, src, holes)


_EXACT = dict(lora=_exact_lora, rotary=_exact_rotary, scatter=_exact_scatter, fork=_exact_fork,
              compact=_exact_compact)
