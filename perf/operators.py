"""Serving operators on shared state, as a program that keeps many pages in flight calls them.

* ``step``   one new token for every sequence over a paged key-value cache: the
             token's key and value rows are written, then its query attends over
             what the sequence may see; optionally every key's attention weight
             is added to what it has gathered so far
* ``evict``  a cache cut to a budget by those gathered weights: the first and the
             last slots and the heaviest of the rest move, in order, to pages of
             the sequence's own
* ``beam``   one step of beam search: the best continuations over beams and
             vocabulary with the no-repeat-ngram ban, then the histories, the
             page tables and the pages in progress follow their parents

With ``own`` false a pass is computed in plain torch operations, with ``own``
true by the engine. Both work on the same tensors. The engine has a stream of
its own, which torch's does not wait for: ``prepare`` and ``exact`` wait for both
before they take memory and ``prepare`` again before it hands its tensors over;
passes follow each other on the engine's stream, and who reads their outputs
waits for the device first, as a program does that takes what a run of calls
left (an event each way between the two streams costs 40 us a pass).
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

EOS = 1
VOCAB = 129280  # the decoder's LM head
NGRAM, NGRAM_WINDOW = 35, 128  # the sampler's defaults
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one page at the start of its text, the decoder's own heads: latency
        {"name": "step_1", "kind": "step", "dtype": "f32", "seqs": 1, "heads": 10, "kv_heads": 10, "dim": 128,
         "page": 16, "longest": 277, "prefix": 0, "window": 0, "weights": False},
        # eight pages in flight, prompts of up to a thousand tokens, f32 as in the ring caches
        {"name": "step_8_f32", "kind": "step", "dtype": "f32", "seqs": 8, "heads": 10, "kv_heads": 10, "dim": 128,
         "page": 32, "longest": 1152, "prefix": 0, "window": 0, "weights": False},
        # the decoder's own visibility: the prompt and the last 128 tokens of a long text
        {"name": "step_24_window", "kind": "step", "dtype": "bf16", "seqs": 24, "heads": 10, "kv_heads": 10,
         "dim": 128, "page": 64, "longest": 8192, "prefix": 1021, "window": 128, "weights": False},
        # long documents whose caches are to be cut: the weights are gathered
        {"name": "step_16_weights", "kind": "step", "dtype": "bf16", "seqs": 16, "heads": 10, "kv_heads": 10,
         "dim": 128, "page": 16, "longest": 4096, "prefix": 0, "window": 0, "weights": True},
        # few rows over very long caches, grouped heads
        {"name": "step_2_long", "kind": "step", "dtype": "f16", "seqs": 2, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 128, "longest": 131071, "prefix": 0, "window": 0, "weights": False},
        # a full server: many ragged sequences, eight heads to a key head
        {"name": "step_128_grouped", "kind": "step", "dtype": "bf16", "seqs": 128, "heads": 16, "kv_heads": 2,
         "dim": 64, "page": 16, "longest": 16384, "prefix": 0, "window": 0, "weights": False},
        # one page's cache cut back to the prompt's length
        {"name": "evict_1", "kind": "evict", "dtype": "f32", "seqs": 1, "kv_heads": 10, "dim": 128, "page": 16,
         "longest": 1152, "budget": 1024, "sinks": 4, "recent": 128},
        # eight long documents cut to a quarter
        {"name": "evict_8", "kind": "evict", "dtype": "bf16", "seqs": 8, "kv_heads": 10, "dim": 128, "page": 32,
         "longest": 8192, "budget": 2048, "sinks": 4, "recent": 256},
        # two very long caches of grouped heads
        {"name": "evict_2_long", "kind": "evict", "dtype": "f16", "seqs": 2, "kv_heads": 8, "dim": 128, "page": 128,
         "longest": 131071, "budget": 16001, "sinks": 0, "recent": 1000},
        # one page read with four beams
        {"name": "beam_1x4", "kind": "beam", "dtype": "f32", "groups": 1, "beams": 4, "vocab": VOCAB, "length": 301,
         "generated": 140, "layers": 12, "kv_heads": 10, "dim": 128, "page": 16, "ngram": NGRAM},
        # eight pages with eight beams each
        {"name": "beam_8x8", "kind": "beam", "dtype": "f32", "groups": 8, "beams": 8, "vocab": VOCAB, "length": 1151,
         "generated": 300, "layers": 12, "kv_heads": 10, "dim": 128, "page": 32, "ngram": NGRAM},
        # many narrow groups over a smaller vocabulary of odd size, no ban
        {"name": "beam_48x5", "kind": "beam", "dtype": "bf16", "groups": 48, "beams": 5, "vocab": 50021,
         "length": 700, "generated": 65, "layers": 6, "kv_heads": 4, "dim": 64, "page": 64, "ngram": 0},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["step", "step", "evict", "beam"])
    dtype = rng.choice(sorted(TYPES))
    page = rng.choice([8, 16, 32, 64, 128])
    dim = rng.choice([64, 128, 128])
    if kind == "step":
        group, kv_heads = rng.choice([(1, 10), (1, 10), (2, 8), (4, 8), (8, 2), (7, 1)])
        longest = _between(rng, 1, 65536)
        seqs = _between(rng, 1, max(1, min(128, 800_000 // (longest * kv_heads))))
        windowed = rng.random() < 0.3
        return {"kind": kind, "dtype": dtype, "seqs": seqs, "heads": group * kv_heads, "kv_heads": kv_heads, "dim": dim,
                "page": page, "longest": longest, "prefix": _between(rng, 1, 1024) if windowed else 0,
                "window": _between(rng, 1, 512) if windowed else 0, "weights": rng.random() < 0.3}
    if kind == "evict":
        kv_heads = rng.choice([1, 2, 4, 8, 10])
        longest = _between(rng, 64, min(65536, 400_000 // kv_heads))
        seqs = _between(rng, 1, max(1, min(32, 400_000 // (longest * kv_heads))))
        budget = max(16, round(longest * rng.uniform(0.05, 0.95)))
        return {"kind": kind, "dtype": dtype, "seqs": seqs, "kv_heads": kv_heads, "dim": dim, "page": page,
                "longest": longest, "budget": budget, "sinks": rng.choice([0, 1, 4]),
                "recent": rng.randrange(0, budget // 2)}
    beams = rng.randrange(2, 17)
    generated = _between(rng, 1, 400)
    return {"kind": kind, "dtype": dtype, "groups": _between(rng, 1, max(1, 96 // beams)), "beams": beams,
            "vocab": rng.choice([VOCAB, _between(rng, 1000, 129000)]), "length": generated + _between(rng, 1, 800),
            "generated": generated, "layers": rng.randrange(1, 13), "kv_heads": rng.choice([2, 4, 10]), "dim": dim,
            "page": page, "ngram": rng.choice([0, 2, NGRAM])}


# ---- what a case stands for, from its numbers alone ----------------------------------


def _lengths(case):
    """Keys that each sequence has: the first has the longest cache, the others some part of it."""
    return [max(1, round(case["longest"] * (1.0 if s == 0 else 0.05 + 0.95 * ((s * 0.6180339887) % 1.0))))
            for s in range(case["seqs"])]


def _visible(case, n):
    """How many of n keys a token sees."""
    p = min(case["prefix"], n)
    return n if case["window"] == 0 else p + min(case["window"], n - p)


def _esize(case):
    return 4 if case["dtype"] == "f32" else 2


def work(case):
    row = case["kv_heads"] * case["dim"] * _esize(case) * 2  # one slot's K and V
    if case["kind"] == "step":
        seen = sum(_visible(case, n + 1) for n in _lengths(case))
        values = case["heads"] * case["dim"]
        moved = seen * row + case["seqs"] * (8 * values + 8 * case["kv_heads"] * case["dim"] + row)
        if case["weights"]:
            moved += 8 * seen * case["kv_heads"]
        return {"bytes": moved, "flops": 4 * seen * values}
    if case["kind"] == "evict":
        lengths = _lengths(case)
        kept = sum(min(n, case["budget"]) for n in lengths)
        return {"bytes": 4 * sum(lengths) * case["kv_heads"] + kept * (2 * row + 8 * case["kv_heads"]), "flops": 0}
    rows = case["groups"] * case["beams"]
    # of the pages in progress and the histories, about half change hands
    states = (case["length"] % case["page"]) * row * case["layers"] + 4 * case["generated"] + 4 * case["length"] // case["page"]
    return {"bytes": rows * (4 * case["vocab"] + states), "flops": 4 * rows * case["vocab"]}


# ---- the states ----------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, sigma=1.0):
    return torch.randn(shape, generator=g, device="cuda") * sigma


def _pool(g, shape, dtype):
    """A pool of pages: [pages][kv_heads][page][dim], every slot holding something."""
    t = torch.empty(shape, dtype=TYPES[dtype], device="cuda")
    return t.normal_(generator=g)


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pages(n, page):
    return -(-n // page)


def _tables(g, counts, wide, spare=3):
    """Page tables [rows][wide] with counts[s] pages of its own for row s, scattered over a pool, and the pool's size."""
    total = sum(counts) + spare
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    t = torch.zeros((len(counts), wide), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        t[s, :n] = order[at: at + n]
        at += n
    return t, total


def _step_state(case, g):
    lengths = _lengths(case)
    wide = _pages(max(lengths) + 1, case["page"])
    tables, pages = _tables(g, [_pages(n + 1, case["page"]) for n in lengths], wide)
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    n, d, kd = case["seqs"], case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    s = {"tables": tables, "lens": _int32(lengths), "k_pool": _pool(g, shape, case["dtype"]),
         "v_pool": _pool(g, shape, case["dtype"]), "q": _normal(g, (n, d), 2.0), "k": _normal(g, (n, kd)),
         "v": _normal(g, (n, kd)), "out": torch.zeros((n, d), device="cuda"), "max_len": max(lengths) + 1}
    if case["prefix"]:
        # prompts of about that length, none alike
        s["prefix"] = _int32([max(1, case["prefix"] - (r * 61) % max(1, case["prefix"] // 2)) for r in range(n)])
    if case["weights"]:
        w = torch.rand((n, case["kv_heads"], wide * case["page"]), generator=g, device="cuda")
        s["gathered"] = w * w * w
    return s


def _evict_state(case, g):
    lengths = _lengths(case)
    page, h = case["page"], case["kv_heads"]
    wide, dst_wide = _pages(max(lengths), page), _pages(case["budget"], page)
    n = case["seqs"]
    both, pages = _tables(g, [_pages(x, page) for x in lengths] + [dst_wide] * n, max(wide, dst_wide))
    tables, dst_tables = both[:n, :wide].contiguous(), both[n:, :dst_wide].contiguous()
    shape = (pages, h, page, case["dim"])
    # what attention gathers is spread over many orders of magnitude, and some keys were never looked at
    w = torch.exp(_normal(g, (n, h, wide * page), 2.0))
    w = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.1, torch.zeros_like(w), w)
    return {"tables": tables, "lens": _int32(lengths), "weights": w, "dst_tables": dst_tables,
            "k_pool": _pool(g, shape, case["dtype"]), "v_pool": _pool(g, shape, case["dtype"]),
            "dst_lens": torch.zeros(n, dtype=torch.int32, device="cuda"),
            "dst_weights": torch.zeros((n, h, dst_wide * page), device="cuda"),
            "kept": torch.zeros((n, h, case["budget"]), dtype=torch.int32, device="cuda")}


def _beam_state(case, g):
    groups, beams, vocab, page = case["groups"], case["beams"], case["vocab"], case["page"]
    rows, length, generated = groups * beams, case["length"], case["generated"]
    # the prompt's full pages are one group's, the pages after them each beam's
    wide = _pages(length + 1, page)
    shared = (length - generated) // page
    mine, pages = _tables(g, [wide] * rows, wide)
    tables = torch.where(torch.arange(wide, device="cuda")[None, :] < shared,
                         mine.view(groups, beams, wide)[:, :1].expand(groups, beams, wide).reshape(rows, wide), mine)
    shape = (pages, case["kv_heads"], page, case["dim"])
    # text that comes round again, so that the ban has work to do
    cap = generated + 100
    period = max(1, min(generated, 40))
    text = torch.randint(2, vocab, (rows, period), generator=g, device="cuda", dtype=torch.int32)
    history = torch.zeros((rows, cap), dtype=torch.int32, device="cuda")
    history[:, :generated] = text.repeat(1, _pages(generated, period))[:, :generated]
    logits = _normal(g, (rows, vocab), 2.5)
    done = torch.rand(rows, generator=g, device="cuda") < 0.1
    ints = lambda: torch.zeros(rows, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"logits": logits, "scores": -5.0 - 3.0 * torch.rand(rows, generator=g, device="cuda"),
            "done": done.to(torch.uint8), "tables": tables.contiguous(), "lens": ints() + length, "history": history,
            "history_len": ints() + generated, "parents": ints(), "tokens": ints(),
            "new_scores": torch.zeros(rows, device="cuda"), "new_done": torch.zeros(rows, dtype=torch.uint8, device="cuda"),
            "k_pools": _pool(g, (case["layers"], *shape), case["dtype"]),
            "v_pools": _pool(g, (case["layers"], *shape), case["dtype"])}


_STATES = {"step": _step_state, "evict": _evict_state, "beam": _beam_state}


def _settle():
    """What either stream was given is done: memory that torch hands out next is in no pass's use, and no pass finds
    tensors that are still being filled."""
    if own:
        torch.cuda.synchronize()


def prepare(case, seed):
    _settle()
    s = _STATES[case["kind"]](case, _generator(seed))
    s["case"] = case
    if own:  # the engine's handles of the same tensors, which a program keeps
        s["own"] = _handles(case, s)
    _settle()
    return s


# ---- the engine's calls ----------------------------------------------------------------


def _handles(case, s):
    from franken_ocr_amd import engine
    from franken_ocr_amd.device import DeviceArray, default_context

    ctx = default_context()
    types = {torch.float32: np.float32, torch.int32: np.uint32, torch.uint8: np.uint8, torch.float16: np.uint16,
             torch.bfloat16: np.uint16}

    def array(t):
        return DeviceArray.borrow(ctx, t.data_ptr(), tuple(t.shape), types[t.dtype], owner=t)

    def cache(k, v):
        return engine.PagedCache(k.shape[0], case["page"], case["kv_heads"], case["dim"], case["dtype"], k=array(k),
                                 v=array(v), ctx=ctx)

    h = {name: array(t) for name, t in s.items() if isinstance(t, torch.Tensor) and "_pool" not in name}
    if case["kind"] == "beam":
        h["caches"] = [cache(k, v) for k, v in zip(s["k_pools"], s["v_pools"])]
    else:
        h["cache"] = cache(s["k_pool"], s["v_pool"])
    h["engine"] = engine
    return h


def _own_step(s):
    case, h = s["case"], s["own"]
    h["cache"].step(h["q"], h["k"], h["v"], h["tables"], h["lens"], h["out"], max_len=s["max_len"],
                    prefix=h.get("prefix"), window=case["window"], weights=h.get("gathered"))
    return _step_out(s)


def _own_evict(s):
    case, h = s["case"], s["own"]
    h["cache"].evict(h["tables"], h["lens"], h["weights"], case["budget"], h["dst_tables"], h["dst_lens"],
                     h["dst_weights"], sinks=case["sinks"], recent=case["recent"], kept=h["kept"])
    return _evict_out(s)


def _own_beam(s):
    case, h = s["case"], s["own"]
    h["engine"].beam_select(h["logits"], h["scores"], case["beams"], h["parents"], h["tokens"], h["new_scores"],
                            done=h["done"], new_done=h["new_done"], history=h["history"],
                            history_len=h["history_len"], ngram_size=case["ngram"], window=NGRAM_WINDOW, eos=EOS)
    h["engine"].beam_reorder(h["parents"], case["beams"], tokens=h["tokens"], history=h["history"],
                             history_len=h["history_len"], caches=h["caches"], tables=h["tables"], lens=h["lens"])
    return _beam_out(s)


def _step_out(s):
    return {name: s[name] for name in ("out", "k_pool", "v_pool", "gathered") if name in s}


def _evict_out(s):
    return {name: s[name] for name in ("dst_lens", "kept", "dst_weights", "k_pool", "v_pool")}


def _beam_out(s):
    return {name: s[name] for name in ("parents", "tokens", "new_scores", "new_done", "history", "tables", "k_pools",
                                       "v_pools")}


# ---- the plain forms -------------------------------------------------------------------


def _rows(pool, tables):
    """The pool's pages by table: [rows][kv_heads][slots][dim] in 32 bits."""
    n, wide = tables.shape
    _, h, page, d = pool.shape
    return pool[tables.long()].transpose(1, 2).reshape(n, h, wide * page, d).float()


def _seen(s, slots):
    """Which slots a token sees: [seqs][slots]."""
    case, n = s["case"], s["lens"][:, None].long() + 1
    at = torch.arange(slots, device="cuda")[None, :]
    seen = at < n
    if case["window"]:
        first = s["prefix"][:, None].long() if "prefix" in s else torch.zeros_like(n)
        seen = seen & ((at < first) | (at >= n - case["window"]))
    return seen


def _plain_step(s):
    case = s["case"]
    n, h, d, page = case["seqs"], case["kv_heads"], case["dim"], case["page"]
    row, at = torch.arange(n, device="cuda"), s["lens"].long()
    where = s["tables"].long()[row, at // page]
    s["k_pool"][where, :, at % page] = s["k"].view(n, h, d).to(s["k_pool"].dtype)
    s["v_pool"][where, :, at % page] = s["v"].view(n, h, d).to(s["v_pool"].dtype)
    k, v = _rows(s["k_pool"], s["tables"]), _rows(s["v_pool"], s["tables"])
    q = s["q"].view(n, h, case["heads"] // h, d) / math.sqrt(d)
    score = (k @ q.transpose(2, 3).contiguous()).transpose(2, 3)  # [seqs][kv_heads][group][slots]
    score = score.masked_fill(~_seen(s, k.shape[2])[:, None, None, :], -math.inf)
    p = torch.exp(score - score.amax(dim=3, keepdim=True))
    p = p / p.sum(dim=3, keepdim=True)
    s["out"].copy_((p @ v).reshape(n, -1))
    if case["weights"]:
        s["gathered"] += p.sum(dim=2)
    return _step_out(s)


def _plain_evict(s):
    case = s["case"]
    page, budget, h = case["page"], case["budget"], case["kv_heads"]
    lens, slots = s["lens"].long()[:, None, None], s["weights"].shape[2]
    at = torch.arange(slots, device="cuda")
    # the heaviest first, equal ones by their slot: the weights (none negative) as whole numbers, the slot below them
    key = (s["weights"].view(torch.int32).long() << 32) | (0x7FFFFFFF - at)
    top = torch.iinfo(torch.int64).max
    protected = (at < case["sinks"]) | (at >= lens - case["recent"])
    key = torch.where(protected, top - at, key)
    key = torch.where(at < lens, key, -1 - at)
    wanted = min(budget, slots)
    chosen = key.topk(wanted, dim=2).indices
    count = torch.minimum(lens, torch.full_like(lens, budget))
    chosen = torch.where(torch.arange(wanted, device="cuda") < count, chosen, slots).sort(dim=2).values
    real = chosen < slots
    i = torch.arange(wanted, device="cuda")
    src, head = chosen.clamp(max=slots - 1), torch.arange(h, device="cuda")[None, :, None]
    row = torch.arange(case["seqs"], device="cuda")[:, None, None]
    src_page, dst_page = s["tables"].long()[row, src // page], s["dst_tables"].long()[row, i // page]
    src_page, dst_page = src_page[real], dst_page.expand(src.shape)[real]
    head, src_at, dst_at = head.expand(src.shape)[real], (src % page)[real], (i % page).expand(src.shape)[real]
    s["k_pool"][dst_page, head, dst_at] = s["k_pool"][src_page, head, src_at]
    s["v_pool"][dst_page, head, dst_at] = s["v_pool"][src_page, head, src_at]
    s["kept"][:, :, :wanted] = torch.where(real, chosen, s["kept"][:, :, :wanted]).to(torch.int32)
    s["dst_weights"][:, :, :wanted] = torch.where(real, s["weights"].gather(2, src), s["dst_weights"][:, :, :wanted])
    s["dst_lens"].copy_(count.view(-1))
    return _evict_out(s)


def _banned(s):
    """Which tokens would end an n-gram of the last window a second time: [rows][vocab]."""
    case, n, size = s["case"], s["case"]["ngram"], s["case"]["generated"]
    out = torch.zeros(s["logits"].shape, dtype=torch.bool, device="cuda")
    if n and size >= n:
        grams = s["history"][:, max(0, size - NGRAM_WINDOW): size].unfold(1, n, 1)  # [rows][grams][n]
        last = s["history"][:, None, size - (n - 1): size]
        again = (grams[:, :, : n - 1] == last).all(dim=2)
        row = torch.arange(out.shape[0], device="cuda")[:, None].expand(again.shape)
        out[row[again], grams[:, :, n - 1][again].long()] = True
    return out


def _plain_beam(s):
    case = s["case"]
    groups, beams, page = case["groups"], case["beams"], case["page"]
    x = s["logits"]
    m = x.amax(dim=1, keepdim=True)
    total = m.double() + torch.log(torch.exp((x - m).double()).sum(dim=1, keepdim=True))
    # a row's tokens in order: the logits as whole numbers of the same order, the token below them
    bits = torch.where(x == 0, torch.zeros_like(x), x).view(torch.int32).long()
    order = torch.where(bits < 0, -2147483648 - bits, bits)
    key = order * 4294967296 + (4294967295 - torch.arange(x.shape[1], device="cuda"))
    none = torch.iinfo(torch.int64).min
    best = key.masked_fill(_banned(s), none).topk(beams, dim=1)
    token = best.indices
    score = s["scores"][:, None].double() + (x.gather(1, token).double() - total)
    done, first = s["done"].bool()[:, None], torch.arange(beams, device="cuda")[None, :] == 0
    token = torch.where(done, torch.full_like(token, EOS), token)
    score = torch.where(done, s["scores"][:, None].double(), score)
    out = (best.values == none) & ~done | done & ~first
    score = score.masked_fill(out, -math.inf).view(groups, beams * beams)
    score, at = score.sort(dim=1, descending=True, stable=True)
    score, at = score[:, :beams], at[:, :beams]
    parent = at // beams
    rows = (parent + beams * torch.arange(groups, device="cuda")[:, None]).view(-1)
    s["parents"].copy_(parent.reshape(-1))
    s["tokens"].copy_(token.view(groups, -1).gather(1, at).view(-1))
    s["new_scores"].copy_(score.reshape(-1))
    s["new_done"].copy_(s["done"][rows] | (s["tokens"] == EOS))
    s["history"].copy_(s["history"][rows])
    s["history"][:, case["generated"]] = s["tokens"]
    full, rest = case["length"] // page, case["length"] % page
    s["tables"][:, :full] = s["tables"][rows, :full]
    if rest:
        mine = s["tables"][:, full].long()
        s["k_pools"][:, mine, :, :rest] = s["k_pools"][:, mine[rows], :, :rest]
        s["v_pools"][:, mine, :, :rest] = s["v_pools"][:, mine[rows], :, :rest]
    return _beam_out(s)


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"step": _own_step, "evict": _own_evict, "beam": _own_beam}[kind](s)
    return {"step": _plain_step, "evict": _plain_evict, "beam": _plain_beam}[kind](s)


# ---- the results in 64 bits, from the definitions ------------------------------------------


def _exact_step(case, s):
    page, h, d = case["page"], case["kv_heads"], case["dim"]
    group = case["heads"] // h
    outs = []
    gathered = s["gathered"].double() if case["weights"] else None
    for r, n in enumerate(_lengths(case)):
        pages = s["tables"][r, : n // page + 1].tolist()
        for name in "kv":
            s[name + "_pool"][pages[-1], :, n % page] = s[name][r].view(h, d).to(TYPES[case["dtype"]])
        keys, values = (s[name + "_pool"][pages].permute(1, 0, 2, 3).reshape(h, -1, d)[:, : n + 1] for name in "kv")
        at = list(range(n + 1))
        if case["window"]:
            p = min(int(s["prefix"][r]) if case["prefix"] else 0, n + 1)
            at = at[:p] + at[max(p, n + 1 - case["window"]):]
        at = torch.tensor(at, device="cuda")
        keys, values = keys[:, at].double(), values[:, at].double()
        q = s["q"][r].double().view(h, group, d)
        heads = []
        for j in range(group):
            p = torch.softmax((keys * q[:, j, None]).sum(dim=2) / math.sqrt(d), dim=1)  # [kv_heads][keys]
            heads.append((p[:, :, None] * values).sum(dim=1))
            if gathered is not None:
                gathered[r][:, at] += p
        outs.append(torch.stack(heads, dim=1).reshape(-1))
    out = {"out": torch.stack(outs), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    return out if gathered is None else {**out, "gathered": gathered}


def _exact_evict(case, s):
    page, h = case["page"], case["kv_heads"]
    weights = s["weights"].cpu().numpy()
    k, v, kept = s["k_pool"].clone(), s["v_pool"].clone(), s["kept"]
    dst_weights = s["dst_weights"].double()
    for r, n in enumerate(_lengths(case)):
        count = min(n, case["budget"])
        s["dst_lens"][r] = count
        to = np.arange(count)
        to_page, to_at = s["dst_tables"][r].long()[torch.from_numpy(to // page).cuda()], torch.from_numpy(to % page).cuda()
        for j in range(h):
            stay = np.arange(n)
            if n > count:
                lo, hi = case["sinks"], n - case["recent"]
                middle = np.argsort(-weights[r, j, lo:hi].astype(np.float64), kind="stable")[: count - lo - (n - hi)] + lo
                stay = np.sort(np.concatenate([np.arange(lo), middle, np.arange(hi, n)]))
            at = torch.from_numpy(stay).cuda()
            kept[r, j, :count] = at.to(torch.int32)
            dst_weights[r, j, :count] = s["weights"][r, j, at].double()
            from_page = s["tables"][r].long()[at // page]
            k[to_page, j, to_at] = s["k_pool"][from_page, j, at % page]
            v[to_page, j, to_at] = s["v_pool"][from_page, j, at % page]
    return {"dst_lens": s["dst_lens"], "kept": kept, "dst_weights": dst_weights, "k_pool": k, "v_pool": v}


def _exact_beam(case, s):
    groups, beams, page, n = case["groups"], case["beams"], case["page"], case["ngram"]
    logits, scores = s["logits"].double(), s["scores"].tolist()
    norm = torch.logsumexp(logits, dim=1).tolist()
    done, history = s["done"].tolist(), s["history"].cpu().numpy()
    size, length = case["generated"], case["length"]
    new = {name: [] for name in ("parents", "tokens", "new_scores", "new_done")}
    rows = []
    for g in range(groups):
        found = []
        for b in range(beams):
            r = g * beams + b
            if done[r]:
                found.append((-scores[r], b, 0.0, EOS))
                continue
            x = s["logits"][r].cpu().numpy().copy()
            if n and size >= n:
                text, last = history[r, :size].tolist(), history[r, size - (n - 1): size].tolist()
                for i in range(max(0, size - NGRAM_WINDOW), size - n + 1):
                    if text[i: i + n - 1] == last:
                        x[text[i + n - 1]] = -math.inf
            for t in np.argsort(-x, kind="stable")[:beams].tolist():
                found.append((-(scores[r] + (float(x[t]) - norm[r])), b, -float(x[t]), t))
        for c, b, _, t in sorted(found)[:beams]:
            rows.append(g * beams + b)
            new["parents"].append(b)
            new["tokens"].append(t)
            new["new_scores"].append(-c)
            new["new_done"].append(int(done[g * beams + b] or t == EOS))
    rows = torch.tensor(rows, device="cuda")
    out = {"parents": _int32(new["parents"]), "tokens": _int32(new["tokens"]),
           "new_scores": torch.tensor(new["new_scores"], dtype=torch.float64, device="cuda"),
           "new_done": torch.tensor(new["new_done"], dtype=torch.uint8, device="cuda")}
    out["history"] = s["history"][rows]
    out["history"][:, size] = out["tokens"]
    full, rest = length // page, length % page
    out["tables"] = s["tables"].clone()
    out["tables"][:, :full] = s["tables"][rows, :full]
    mine = s["tables"][:, full].long()
    for name in ("k_pools", "v_pools"):
        out[name] = s[name].clone()
        if rest:
            out[name][:, mine, :, :rest] = s[name][:, mine[rows], :, :rest]
    return out


def exact(case, seed):
    _settle()
    s = _STATES[case["kind"]](case, _generator(seed))
    return {"step": _exact_step, "evict": _exact_evict, "beam": _exact_beam}[case["kind"]](case, s)
