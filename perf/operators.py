"""The operators of serving from an 8-bit KV cache, as cases that a program can time and check.

`listed()` names them, `draw(rng)` gives more of the same ranges, `prepare` makes what a program
holds before the call, `run` is one pass (the operators in elementary torch where `own` is false,
through the framework's entry points where it is true), `work` what a pass cannot do without and
`exact` its result from the definition in 64 bits.

The cache holds keys and values as e4m3 in pages of 16 tokens, [page, kv head, token, dim], with a
power-of-two scale for each page and kv head. Every operator takes the same description of a batch:
block tables [sequences, pages], `row_starts` (sequence s owns rows row_starts[s] up to
row_starts[s + 1]; None: one row each) and `seq_lens`, the tokens a sequence holds once the call's
rows are in; the rows are its last ones.

Shapes are those of the repository's model (32 query and 8 kv heads of 64, vocabulary 128256) and
generic ones around it.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
PAGE = 16
THETA = 500000.0
MAX_E4M3 = 448.0
MIN_EXP, MAX_EXP = -15, 7  # of a block's scale: every value is then a finite fp16


def listed():
    return [
        # One sequence's decode step: where the launch is all there is.
        dict(name="append_1", kind="append", seqs=1, rows=1, ragged=False, max_len=700, heads=32,
             kv=8, dim=64),
        # A full batch's decode step.
        dict(name="append_256", kind="append", seqs=256, rows=1, ragged=False, max_len=4096,
             heads=32, kv=8, dim=64),
        # Prompts that arrive together, behind prefixes that end inside a page.
        dict(name="append_prompts", kind="append", seqs=5, rows=2001, ragged=True, max_len=4333,
             heads=32, kv=8, dim=64),
        # A short prefix read back, and the caches of a batch (moved to another pool, or checked).
        dict(name="gather_1", kind="gather", seqs=1, rows=77, ragged=False, max_len=77, heads=32,
             kv=8, dim=64),
        dict(name="gather_64", kind="gather", seqs=64, rows=3001, ragged=True, max_len=3001,
             heads=32, kv=8, dim=64),
        # Decode attention: one young sequence, ...
        dict(name="attention_1", kind="attention", seqs=1, rows=1, ragged=False, max_len=301,
             heads=32, kv=8, dim=64),
        # ... a full batch at a serving mix of lengths, ...
        dict(name="attention_256", kind="attention", seqs=256, rows=1, ragged=False, max_len=2048,
             heads=32, kv=8, dim=64),
        # ... and few sequences with long contexts and wide heads.
        dict(name="attention_3_long", kind="attention", seqs=3, rows=1, ragged=False,
             max_len=65001, heads=32, kv=8, dim=128),
        # Drafted tokens: up to five rows a sequence.
        dict(name="attention_drafts", kind="attention", seqs=48, rows=5, ragged=True, max_len=4096,
             heads=32, kv=8, dim=64),
        # A prompt's chunk behind a cached prefix.
        dict(name="attention_prompt", kind="attention", seqs=1, rows=1507, ragged=False,
             max_len=3001, heads=32, kv=8, dim=64),
        # Four drafts of one sequence, drafted without probabilities (looked up in its own text).
        dict(name="verify_1", kind="verify", seqs=1, rows=5, ragged=False, vocab=32000,
             drafted=False, greedy=False),
        # A batch with a draft model's logits beside the target's.
        dict(name="verify_64", kind="verify", seqs=64, rows=5, ragged=False, vocab=128256,
             drafted=True, greedy=False),
    ]


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], uniform over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return min(hi, max(lo, int(v)))


def draw(rng):
    kind = rng.choice(["append", "gather", "attention", "attention", "attention", "verify"])
    if kind == "verify":
        vocab = rng.choice([32000, 50003, 128256])
        rows = rng.choice([1, 2, 3, 5, 8])
        return dict(kind=kind, seqs=_log_int(rng, 1, min(96, 41000000 // (vocab * rows))),
                    rows=rows, ragged=rows > 1 and rng.random() < 0.5, vocab=vocab,
                    drafted=rows > 1 and rng.random() < 0.6, greedy=rng.random() < 0.2)
    heads, kv, dim = rng.choice([(32, 8, 64), (32, 8, 64), (32, 8, 128), (20, 20, 64),
                                 (28, 4, 128), (12, 2, 64), (8, 1, 128)])
    layout = dict(heads=heads, kv=kv, dim=dim)
    wide = max(1, heads * dim // 2048)  # how much more a row is than the model's
    if kind == "append":
        what = rng.choice(["decode", "drafts", "prompt"])
        seqs = _log_int(rng, 1, 6 if what == "prompt" else 256)
        rows = dict(decode=1, drafts=rng.randint(2, 9),
                    prompt=_log_int(rng, 17, 5000 // (seqs * wide)))[what]
        return dict(kind=kind, seqs=seqs, rows=rows, ragged=rows > 1 and rng.random() < 0.5,
                    max_len=rows + rng.randint(1, 4096), **layout)
    if kind == "gather":
        seqs = _log_int(rng, 1, 64)
        rows = _log_int(rng, 1, 80000 * 512 // (seqs * max(512, kv * dim)))
        return dict(kind=kind, seqs=seqs, rows=rows, ragged=rows > 1 and rng.random() < 0.5,
                    max_len=rows + rng.choice([0, rng.randint(0, 1000)]), **layout)
    what = rng.choice(["decode", "decode", "drafts", "chunk"])
    if what == "chunk":
        seqs = rng.choice([1, 1, 2, 5])
        rows = _log_int(rng, 10, 1200 // (seqs * wide))
        return dict(kind=kind, seqs=seqs, rows=rows, ragged=rng.random() < 0.5,
                    max_len=rows + rng.choice([0, rng.randint(0, 1000)]), **layout)
    rows = 1 if what == "decode" else rng.randint(2, 9)
    seqs = _log_int(rng, 1, 256 if rows == 1 else 64)
    longest = min(65536, 260000 * 512 // (seqs * kv * dim))
    return dict(kind=kind, seqs=seqs, rows=rows, ragged=rows > 1 and rng.random() < 0.5,
                max_len=_log_int(rng, max(16, rows), max(17, longest)), **layout)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _sizes(case):
    """(rows, length) of each sequence: fixed by the case, so that its work is. Lengths are uniform
    up to max_len with the longest present, rows all of the case's, or uniform up to them."""
    r = np.random.default_rng([case["seqs"], case["rows"], case.get("max_len", 0)])
    n = case["seqs"]
    rows = r.integers(1, case["rows"] + 1, n) if case["ragged"] else np.full(n, case["rows"])
    rows[r.integers(0, n)] = case["rows"]
    if case["kind"] == "verify":
        return rows, None
    if case["kind"] == "gather":  # whole sequences, or the ends of longer ones
        return rows, rows + (case["max_len"] - case["rows"])
    lens = r.integers(1, case["max_len"] + 1, n)
    lens[r.integers(0, n)] = case["max_len"]
    return rows, np.maximum(lens, rows)


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(shape, g, std=1.0):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).mul_(std)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def _starts(rows):
    return _ints(np.concatenate([[0], np.cumsum(rows)]))


def _cache(pages, kv, dim, g, spread):
    """A pool of cached rows as they come from a model: normal, heads and dims of unlike size."""
    x = _normal((pages, kv, PAGE, dim), g)
    x *= torch.exp(_normal((1, kv, 1, 1), g, 0.5)) * torch.exp(_normal((1, 1, 1, dim), g, spread))
    e = torch.ceil(torch.log2(x.abs().amax((2, 3)) / MAX_E4M3)).clamp_(MIN_EXP, MAX_EXP)
    scale = torch.exp2(e)
    x /= scale[:, :, None, None]
    return x.clamp_(-MAX_E4M3, MAX_E4M3).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    rng, g = np.random.default_rng(seed), _gen(seed)
    rows, lens = _sizes(case)
    n, n_rows = case["seqs"], int(rows.sum())
    s = dict(kind=case["kind"], n_seqs=n, n_rows=n_rows, max_rows=case["rows"])
    # a batch of one row a sequence needs no row_starts
    s["row_starts"] = None if case["rows"] == 1 else _starts(rows)
    if case["kind"] == "verify":
        return _prepare_verify(case, g, rows, s)

    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    need = (lens + PAGE - 1) // PAGE
    num_pages, widest = int(need.sum()) + 3, int(need.max())
    order, at = rng.permutation(num_pages), 0  # a running server's free list is shuffled
    tables = np.zeros((n, widest), np.int32)
    for b, k in enumerate(need):
        tables[b, :k] = order[at:at + k]
        at += k
    s.update(heads=heads, kv=kv, dim=dim, max_pages=widest, tables=_ints(tables),
             seq_lens=_ints(lens))
    s["k_pool"], s["k_scale"] = _cache(num_pages, kv, dim, g, 0.4)
    s["v_pool"], s["v_scale"] = _cache(num_pages, kv, dim, g, 0.1)
    if case["kind"] == "attention":
        s["q"] = _normal((n_rows, heads, dim), g, 1.2).half()
        s["out"] = torch.empty_like(s["q"])
        return s
    if case["kind"] == "append":
        s["qkv"] = _normal((n_rows, (heads + 2 * kv) * dim), g)
        s["qkv"] *= torch.exp(_normal((n_rows, heads + 2 * kv, 1), g, 0.3)).expand(
            -1, -1, dim).reshape(n_rows, -1)  # tokens and heads of unlike size
        s["qkv"] = s["qkv"].half()
        s["q_out"] = torch.empty((n_rows, heads, dim), dtype=torch.float16, device=DEV)
        s["inv_freq"] = (THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)).float().to(
            DEV)
        # what the append changes: the rows of every page that it touches, read back from the
        # page's first token
        first = (lens - rows) // PAGE * PAGE
        s["read_starts"], n_read = _starts(lens - first), int((lens - first).sum())
    else:
        s["read_starts"], n_read = s["row_starts"], n_rows
    s["n_read"] = n_read
    s["k_out"] = torch.empty((n_read, kv, dim), dtype=torch.float16, device=DEV)
    s["v_out"] = torch.empty_like(s["k_out"])
    return s


def _prepare_verify(case, g, rows, s):
    n, n_rows, vocab = case["seqs"], s["n_rows"], case["vocab"]
    logits = _normal((n_rows, vocab), g, 2.5)
    # a few likely tokens a row, as trained models have them
    likely = torch.randint(0, vocab, (n_rows, 12), generator=g, device=DEV)
    logits.scatter_add_(1, likely, 11.0 + _normal((n_rows, 12), g, 1.5))
    draft = (logits + _normal((n_rows, vocab), g, 0.6)).half()
    s["logits"] = logits.half()
    t = 0.6 + 0.6 * torch.rand(n, generator=g, device=DEV)
    s["temperature"] = torch.zeros_like(t) if case["greedy"] else t
    s["draft_logits"] = draft if case["drafted"] else None
    # drafts that the draft model sampled, or, looked up, the target's likeliest more often than not
    row_t = torch.repeat_interleave(t, torch.from_numpy(rows).to(DEV))[:, None]
    noise = -torch.log(-torch.log(torch.rand((n_rows, vocab), generator=g, device=DEV).clamp_(
        1e-12, 1 - 1e-7)))
    guess = draft.float() / row_t
    s["drafts"] = (guess + noise if not case["greedy"] else guess).argmax(1).to(torch.int32)
    s["accept_u"] = torch.rand(n_rows, generator=g, device=DEV)
    s["sample_u"] = torch.rand(n, generator=g, device=DEV)
    s["vocab"] = vocab
    s["n_accepted"] = torch.empty(n, dtype=torch.int32, device=DEV)
    s["tokens"] = torch.empty(n_rows, dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(s):
    return (_OWN if own else _PLAIN)[s["kind"]](s)


def _llmk():
    from __graft_entry__ import load_llmk
    return load_llmk()


def _own_append(s):
    llmk = _llmk()
    llmk.kv8_append(s["qkv"], s["qkv"].shape[1], s["q_out"], s["k_pool"], s["k_scale"],
                    s["v_pool"], s["v_scale"], s["tables"], s["row_starts"], s["seq_lens"],
                    s["inv_freq"], s["n_rows"], s["n_seqs"], s["max_pages"], PAGE, s["heads"],
                    s["kv"], s["dim"])
    return s["q_out"], *_own_gather(s)


def _own_gather(s):
    _llmk().kv8_gather(s["k_pool"], s["k_scale"], s["v_pool"], s["v_scale"], s["tables"],
                       s["read_starts"], s["seq_lens"], s["k_out"], s["v_out"], s["n_read"],
                       s["n_seqs"], s["max_pages"], PAGE, s["kv"], s["dim"])
    return s["k_out"], s["v_out"]


def _own_attention(s):
    llmk = _llmk()
    if "workspace" not in s:  # a program keeps one
        s["workspace"] = torch.empty(llmk.kv8_attention_workspace_floats(s["dim"]), device=DEV)
    llmk.kv8_attention(s["q"], s["k_pool"], s["k_scale"], s["v_pool"], s["v_scale"], s["tables"],
                       s["row_starts"], s["seq_lens"], s["out"], s["workspace"], s["n_rows"],
                       s["n_seqs"], s["max_rows"], s["max_pages"], PAGE, s["heads"], s["kv"],
                       s["dim"])
    return s["out"]


def _own_verify(s):
    llmk = _llmk()
    if "workspace" not in s:
        s["workspace"] = torch.empty(
            llmk.verify_drafts_workspace_floats(s["n_rows"], s["n_seqs"], s["vocab"]), device=DEV)
    llmk.verify_drafts(s["logits"], s["draft_logits"], s["drafts"], s["row_starts"],
                       s["temperature"], s["accept_u"], s["sample_u"], s["n_accepted"],
                       s["tokens"], s["workspace"], s["n_rows"], s["n_seqs"], s["vocab"])
    return s["n_accepted"], s["tokens"]


_OWN = dict(append=_own_append, gather=_own_gather, attention=_own_attention, verify=_own_verify)


def _rows(starts, n_rows, s):
    """(sequence, place among its rows, that sequence's rows) of every row."""
    if starts is None:
        starts = torch.arange(s["n_seqs"] + 1, device=DEV)
    starts = starts.long()
    r = torch.arange(n_rows, device=DEV)
    seq = torch.searchsorted(starts[1:].contiguous(), r, right=True)
    return seq, r - starts[seq], (starts[1:] - starts[:-1])[seq]


def _slots(starts, n_rows, s):
    """(page, token of the page) of every row."""
    seq, i, count = _rows(starts, n_rows, s)
    pos = s["seq_lens"].long()[seq] - count + i
    return s["tables"].long()[seq, pos // PAGE], pos % PAGE, pos


def _plain_append(s):
    heads, kv, dim, half = s["heads"], s["kv"], s["dim"], s["dim"] // 2
    page, slot, pos = _slots(s["row_starts"], s["n_rows"], s)
    angle = pos.double()[:, None] * s["inv_freq"].double()
    c, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = s["qkv"].float().view(s["n_rows"], heads + 2 * kv, dim)
    a, b = x[:, :heads + kv, :half], x[:, :heads + kv, half:]
    rotated = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    q = rotated[:, :heads].half()
    first = torch.full((s["k_pool"].shape[0],), PAGE, device=DEV).scatter_reduce_(
        0, page, slot, "amin")
    touched = (first < PAGE).nonzero()[:, 0]
    kept = torch.arange(PAGE, device=DEV) < first[touched][:, None]  # slots held before the call
    for pool, scales, new in ((s["k_pool"], s["k_scale"], rotated[:, heads:]),
                              (s["v_pool"], s["v_scale"], x[:, heads + kv:])):
        most = torch.zeros_like(scales).scatter_reduce_(
            0, page[:, None].expand(-1, kv), new.abs().amax(-1), "amax")[touched]
        m, e = torch.frexp(most / MAX_E4M3)  # m in [1/2, 1): the exponent rounded up
        e = torch.where(most > 0, e - (m == 0.5).int(), MIN_EXP).clamp(MIN_EXP, MAX_EXP)
        before = scales[touched]
        scale = torch.ldexp(torch.ones_like(most), e)
        scale = torch.where(first[touched][:, None] > 0, torch.maximum(scale, before), scale)
        held = pool[touched].float() * (before / scale)[..., None, None]
        pool.view(torch.uint8)[touched] = torch.where(
            kept[:, None, :, None], held.to(torch.float8_e4m3fn).view(torch.uint8),
            pool.view(torch.uint8)[touched])
        scales[touched] = scale
        put = (new / scales[page][..., None]).clamp(-MAX_E4M3, MAX_E4M3)
        pool.view(torch.uint8)[page, :, slot] = put.to(torch.float8_e4m3fn).view(torch.uint8)
    return q, *_plain_gather(s)


def _plain_gather(s):
    page, slot, _ = _slots(s["read_starts"], s["n_read"], s)
    return tuple((pool.view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn).float()
                  * scale[page][..., None]).half()
                 for pool, scale in ((s["k_pool"], s["k_scale"]), (s["v_pool"], s["v_scale"])))


def _plain_attention(s):
    n, heads, kv, dim, R = s["n_seqs"], s["heads"], s["kv"], s["dim"], s["max_rows"]
    group = heads // kv
    seq, i, count = _rows(s["row_starts"], s["n_rows"], s)
    tables = s["tables"].long()

    def cached(pool, scale):  # [sequence, kv head, position, dim]
        x = pool.view(torch.uint8)[tables].view(torch.float8_e4m3fn).float()
        x = x * scale[tables][..., None, None]
        return x.transpose(1, 2).reshape(n, kv, -1, dim)

    q = torch.zeros((n, R, heads, dim), device=DEV)
    q[seq, i] = s["q"].float()
    q = q.view(n, R, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, group * R, dim)
    k = cached(s["k_pool"], s["k_scale"]).transpose(2, 3).contiguous()
    score = (q @ k).view(n, kv, group, R, -1) / math.sqrt(dim)
    last = torch.full((n, R), -1, device=DEV)  # the last position that a row sees
    last[seq, i] = s["seq_lens"].long()[seq] - count + i
    unseen = torch.arange(score.shape[-1], device=DEV) > last[..., None]
    score = score.masked_fill_(unseen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = p.view(n, kv, group * R, -1) @ cached(s["v_pool"], s["v_scale"])
    out = out.view(n, kv, group, R, dim) / torch.where(total > 0, total, 1.0)
    return out.permute(0, 3, 1, 2, 4).reshape(n, R, heads, dim)[seq, i].half()


def _plain_verify(s):
    # in 64 bits: which token a random number falls on is settled at the borders of long sums
    n, n_rows, vocab = s["n_seqs"], s["n_rows"], s["vocab"]
    seq, i, count = _rows(s["row_starts"], n_rows, s)
    last = i == count - 1
    t = s["temperature"].double()[seq][:, None]
    greedy = ~(t > 0)

    def probabilities(logits):
        x = logits.double()
        top = x.amax(1, keepdim=True)
        w = torch.exp((x - top) / torch.where(greedy, 1.0, t))
        return w / w.sum(1, keepdim=True)

    p, d = probabilities(s["logits"]), s["drafts"].long()[:, None]
    if s["draft_logits"] is None:
        q = torch.zeros_like(p).scatter_(1, d, 1.0)
    else:
        q = probabilities(s["draft_logits"])
    best = s["logits"].float().argmax(1)
    taken = s["accept_u"].double() * q.gather(1, d)[:, 0] < p.gather(1, d)[:, 0]
    taken = torch.where(greedy[:, 0], d[:, 0] == best, taken) & ~last
    # the first row of each sequence that stands: refused, or behind all drafts
    r = torch.arange(n_rows, device=DEV)
    end = torch.full((n,), n_rows, device=DEV).scatter_reduce_(
        0, seq, torch.where(taken, n_rows, r), "amin")
    w = torch.where(last[end][:, None], p[end], (p[end] - q[end]).clamp(min=0))
    w = torch.where(w.sum(1, keepdim=True) > 0, w, p[end])
    c = w.cumsum(1)
    token = (c > s["sample_u"].double()[:, None] * c[:, -1:]).to(torch.uint8).argmax(1)
    token = torch.where(greedy[end][:, 0], best[end], token)
    tokens = torch.where(r < end[seq], d[:, 0], -1)
    tokens[end] = token
    return i[end].to(torch.int32), tokens.to(torch.int32)


_PLAIN = dict(append=_plain_append, gather=_plain_gather, attention=_plain_attention,
              verify=_plain_verify)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    rows, lens = _sizes(case)
    n_rows = int(rows.sum())
    if case["kind"] == "verify":
        read = n_rows + (n_rows - case["seqs"] if case["drafted"] else 0)
        return dict(bytes=2 * read * case["vocab"] + 12 * n_rows + 12 * case["seqs"],
                    flops=5 * read * case["vocab"])
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    width, batch = kv * dim, 8 * case["seqs"]
    if case["kind"] == "attention":
        pages = int(((lens + PAGE - 1) // PAGE).sum())
        seen = int((rows * lens - rows * (rows - 1) // 2).sum())  # positions over all rows
        return dict(bytes=2 * width * int(lens.sum()) + (8 * kv + 4) * pages
                    + 4 * n_rows * heads * dim + batch, flops=4 * dim * heads * seen)
    first = (lens - rows) // PAGE * PAGE
    n_read = int((lens - first).sum()) if case["kind"] == "append" else n_rows
    pages = n_read // PAGE + case["seqs"]
    read_back = 2 * n_read * width * (1 + 2) + (8 * kv + 4) * pages + batch
    if case["kind"] == "gather":
        return dict(bytes=read_back, flops=2 * n_read * width)
    moved = n_rows * (2 * (heads + 2 * kv) * dim + 2 * heads * dim + 2 * width)
    return dict(bytes=moved + 8 * kv * pages + read_back,
                flops=n_rows * (3 * (heads + kv) * dim + 4 * width) + 2 * n_read * width)


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    rows, lens = _sizes(case)
    starts = np.concatenate([[0], np.cumsum(rows)])
    return _EXACT[case["kind"]](s, rows, lens, starts)


def _e4m3(x):
    """The nearest e4m3 value of 64-bit numbers within its range, ties to the even one."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _pages(s, b, first, last):
    """The pages that hold positions [first, last) of sequence b."""
    return s["tables"][b, first // PAGE:(last + PAGE - 1) // PAGE].long()


def _values(pool, scale, pages):
    """[position, kv head, dim] of whole pages, in 64 bits."""
    x = pool.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
    x = x * scale[pages].double()[:, :, None, None]
    return x.permute(0, 2, 1, 3).reshape(-1, pool.shape[1], pool.shape[3])


def _exact_append(s, rows, lens, starts):
    heads, kv, dim = s["heads"], s["kv"], s["dim"]
    out_q, out_k, out_v = [], [], []
    for b in range(s["n_seqs"]):
        n, first = int(rows[b]), int(lens[b] - rows[b])
        x = s["qkv"][starts[b]:starts[b] + n].double().view(n, -1, dim)
        angle = torch.outer(torch.arange(first, first + n, device=DEV).double(),
                            s["inv_freq"].double())
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        z = torch.complex(x[..., :dim // 2], x[..., dim // 2:])[:, :heads + kv] * turn
        z = torch.cat([z.real, z.imag], -1)
        out_q.append(z[:, :heads])
        base = first // PAGE * PAGE
        pages = _pages(s, b, base, int(lens[b]))
        for pool, scale, new, out in ((s["k_pool"], s["k_scale"], z[:, heads:], out_k),
                                      (s["v_pool"], s["v_scale"], x[:, heads + kv:], out_v)):
            held = _values(pool, scale, pages)[:first - base]
            every = torch.cat([held, new])
            padded = torch.zeros((pages.numel() * PAGE, kv, dim), dtype=torch.float64, device=DEV)
            padded[first - base:every.shape[0]] = new
            most = padded.view(-1, PAGE, kv, dim).abs().amax((1, 3))
            e = torch.ceil(torch.log2(most.clamp(min=2.0 ** -40) / MAX_E4M3)).clamp(MIN_EXP,
                                                                                    MAX_EXP)
            if first > base:
                e[0] = torch.maximum(e[0], torch.log2(scale[pages[0]].double()))
            by = torch.exp2(e).repeat_interleave(PAGE, 0)[:every.shape[0], :, None]
            out.append(_e4m3((every / by).clamp(-MAX_E4M3, MAX_E4M3)) * by)
    return torch.cat(out_q), torch.cat(out_k), torch.cat(out_v)


def _exact_gather(s, rows, lens, starts):
    out = ([], [])
    for b in range(s["n_seqs"]):
        first = int(lens[b] - rows[b])
        pages, base = _pages(s, b, first, int(lens[b])), first // PAGE * PAGE
        for to, pool, scale in ((out[0], s["k_pool"], s["k_scale"]),
                                (out[1], s["v_pool"], s["v_scale"])):
            to.append(_values(pool, scale, pages)[first - base:int(lens[b]) - base])
    return torch.cat(out[0]), torch.cat(out[1])


def _exact_attention(s, rows, lens, starts):
    heads, kv, dim = s["heads"], s["kv"], s["dim"]
    out = torch.empty((s["n_rows"], heads, dim), dtype=torch.float64, device=DEV)
    for b in range(s["n_seqs"]):
        n, last = int(rows[b]), int(lens[b])
        pages = _pages(s, b, 0, last)
        k = _values(s["k_pool"], s["k_scale"], pages)[:last]
        v = _values(s["v_pool"], s["v_scale"], pages)[:last]
        seen = torch.arange(last, device=DEV) <= torch.arange(last - n, last, device=DEV)[:, None]
        q = s["q"][starts[b]:starts[b] + n].double()
        for h in range(kv):
            mine = q[:, h * (heads // kv):(h + 1) * (heads // kv)].reshape(-1, dim)
            a = (mine @ k[:, h].T.contiguous()) * dim ** -0.5
            a = a.masked_fill(~seen.repeat_interleave(heads // kv, 0), -math.inf)
            out[starts[b]:starts[b] + n, h * (heads // kv):(h + 1) * (heads // kv)] = (
                torch.softmax(a, 1) @ v[:, h].contiguous()).view(n, -1, dim)
    return out


def _exact_verify(s, rows, lens, starts):
    tokens, accepted = torch.full((s["n_rows"],), -1, dtype=torch.int32), []
    drafts, u = s["drafts"].tolist(), s["accept_u"].tolist()
    for b in range(s["n_seqs"]):
        t = float(s["temperature"][b])
        for i in range(int(rows[b])):
            r = int(starts[b]) + i
            row = s["logits"][r].double()
            p = torch.softmax(row / t, 0) if t > 0 else None
            left = p
            if i + 1 < rows[b]:
                if t > 0:
                    if s["draft_logits"] is None:
                        q = torch.zeros_like(p)
                        q[drafts[r]] = 1.0
                    else:
                        q = torch.softmax(s["draft_logits"][r].double() / t, 0)
                    good = u[r] * float(q[drafts[r]]) < float(p[drafts[r]])
                    left = (p - q).clamp(min=0)
                else:
                    good = drafts[r] == int(torch.nonzero(row == row.max())[0])
                if good:
                    tokens[r] = drafts[r]
                    continue
            if t > 0:
                c = np.cumsum((left if float(left.sum()) > 0 else p).cpu().numpy())
                tokens[r] = int(np.searchsorted(c, float(s["sample_u"][b]) * c[-1], side="right"))
            else:
                tokens[r] = int(torch.nonzero(row == row.max())[0])
            accepted.append(i)
            break
    return torch.tensor(accepted, dtype=torch.int32), tokens


_EXACT = dict(append=_exact_append, gather=_exact_gather, attention=_exact_attention,
              verify=_exact_verify)
