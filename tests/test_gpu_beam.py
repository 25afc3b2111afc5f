"""Beam search on the device: the selection against the definition in 64 bits,
the reordered states exactly, and a search over paged and ring caches against
the same search with every beam's states kept apart on the host.

The order of candidates is tested exactly: scores that differ by less than
1e-9 do not come up in the seeded draws (asserted), and equal ones are made
equal by construction. new_scores is the f64 score rounded to f32: within
2^-24 of it, and 1e-9 for the sum's and the exponentials' own roundings."""

from __future__ import annotations

import numpy as np
import pytest

from franken_ocr_amd import _abi, synth
from test_gpu_decoder import _device as _decoder
from test_gpu_decoder import model  # noqa: F401 (a fixture)
from test_gpu_paged import Host, _capture

pytestmark = pytest.mark.gpu

EOS = 1
NONE = 0xFFFFFFFF


def _say(msg):
    print(f"[gpu-beam] {msg}", flush=True)


def _bans(history, n, window):
    """Tokens that would end an n-gram of the last `window` tokens again."""
    size = len(history)
    if n == 0 or size < n:
        return set()
    last, start = list(history[size - (n - 1):]) if n > 1 else [], max(0, size - window) if window else 0
    return {history[i + n - 1] for i in range(start, size - n + 1) if list(history[i: i + n - 1]) == last}


def _select(logits, scores, beams, done, banned):
    """(parents, tokens, scores in f64) by the definition."""
    rows, vocab = logits.shape
    parents, tokens, new = [], [], []
    for g in range(rows // beams):
        found = []
        for b in range(beams):
            r = g * beams + b
            s = float(scores[r])
            if done[r]:
                found.append((s if s == s else -np.inf, b, 0.0, EOS))
                continue
            x = logits[r].astype(np.float64)
            ok = ~np.isnan(x)
            with np.errstate(all="ignore"):
                m = x[ok].max() if ok.any() else -np.inf
                if np.isinf(m):
                    total = m
                else:
                    total = m + np.log(np.exp(x[ok] - m).sum())
                keep = ok.copy()
                keep[[t for t in banned[r] if t < vocab]] = False
                at = np.nonzero(keep)[0]
                at = at[np.argsort(-x[at], kind="stable")[:beams]]
                for t in at.tolist():
                    c = s + (x[t] - total)
                    found.append((c if c == c else -np.inf, b, x[t], t))
        found.sort(key=lambda f: (-f[0], f[1], -f[2], f[3]))
        near = [f[0] for f in found if np.isfinite(f[0])]
        assert all(a == b or a - b > 1e-9 for a, b in zip(near, near[1:]))
        for i in range(beams):
            c, b, _, t = found[i] if i < len(found) else (-np.inf, i, 0.0, EOS)
            parents.append(b)
            tokens.append(t)
            new.append(c)
    return parents, tokens, np.array(new)


def _run(ctx, logits, scores, beams, done=None, history=None, lens=None, check=True, **kw):
    from franken_ocr_amd.engine import beam_select

    rows = len(scores)
    p, t = (ctx.to_device(np.full(rows, 77, np.uint32)) for _ in "pt")
    ns, nd = ctx.empty((rows,), np.float32), ctx.empty((rows,), np.uint8)
    dh = ctx.to_device(history) if history is not None else None
    dl = ctx.to_device(np.array(lens, np.uint32)) if lens is not None else None
    beam_select(ctx.to_device(logits), ctx.to_device(np.asarray(scores, np.float32)), beams, p, t, ns,
                done=ctx.to_device(done) if done is not None else None, new_done=nd, history=dh, history_len=dl, eos=EOS,
                check=check, **kw)
    return p.numpy().tolist(), t.numpy().tolist(), ns.numpy(), nd.numpy().tolist()


def _same(got, want, done, beams):
    p, t, s, d = got
    wp, wt, ws = want
    assert p == wp and t == wt
    fine = np.isfinite(ws)
    assert np.array_equal(s[~fine], ws[~fine].astype(np.float32))
    assert np.all(np.abs(s[fine] - ws[fine]) <= np.abs(ws[fine]) * 2.0 ** -24 + 1e-9)
    assert d == [int(bool(done[i // beams * beams + q]) or x == EOS) for i, (q, x) in enumerate(zip(wp, wt))]


@pytest.mark.parametrize("groups,beams,vocab", [(1, 1, 1), (1, 4, 129280), (3, 2, 4096), (2, 5, 4097), (2, 8, 50021),
                                                (1, 32, 12289), (4, 3, 2), (2, 16, 7), (65, 1, 300), (1, 32, 8192),
                                                (1, 32, 129280), (1, 3, 524288), (1, 32, 524287)])
def test_selection_against_64_bits(ctx, groups, beams, vocab):
    _say(f"select {groups} x {beams} over {vocab}")
    rng = np.random.default_rng(groups * 1000 + beams + vocab)
    rows = groups * beams
    logits = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
    scores = (-3 * rng.random(rows)).astype(np.float32)
    done = (rng.random(rows) < 0.2).astype(np.uint8)
    got = _run(ctx, logits, scores, beams, done)
    _same(got, _select(logits, scores, beams, done, [set()] * rows), done, beams)
    assert _run(ctx, logits, scores, beams, done)[2].tobytes() == got[2].tobytes()


def test_selection_of_odd_rows(ctx):
    """Ties, NaN, infinities, rows with nothing, beams that are not there."""
    _say("odd rows")
    rng = np.random.default_rng(5)
    beams, vocab = 4, 9000
    x = (2 * rng.standard_normal((40, vocab))).astype(np.float32)
    scores = (-2 * rng.random(40)).astype(np.float32)
    done = np.zeros(40, np.uint8)
    x[0:4] = x[0]                                       # group 0: the start, four times one row
    scores[0:4] = [0.0, -np.inf, -np.inf, -np.inf]
    x[4:8], scores[4:8] = x[4], scores[4]               # group 1: equal candidates in every beam
    x[8, ::3] = np.nan                                  # group 2: NaN among the logits
    x[9] = np.nan                                       # and nothing else
    x[10] = -np.inf                                     # no probability anywhere
    x[11, 100] = np.inf                                 # too much at one token
    x[12:16] = 0.0                                      # group 3: every logit equal
    x[12:16, 5::2] = -0.0
    done[16:20] = 1                                     # group 4: all finished, equal scores among them
    scores[17] = scores[18]
    scores[20:24] = -np.inf                             # group 5: no beam is there
    x[24:28] = np.nan                                   # group 6: nothing at all
    done[24] = 1
    x[28:32] = np.where(np.arange(vocab) < 3, x[28:32], np.nan)  # group 7: three tokens
    x[29:32] = np.nan
    x[32:36, 4095:4098] = 50.0                          # group 8: equal ones on both sides of a chunk's end
    scores[36] = np.nan                                 # group 9: a score that is none
    done[37], scores[37] = 1, np.nan
    x[38, 17] = -1e30
    got = _run(ctx, x, scores, beams, done)
    _same(got, _select(x, scores, beams, done, [set()] * 40), done, beams)


@pytest.mark.parametrize("check", [True, False])  # the ban found by a launch of its own, or by the scan where it is short
@pytest.mark.parametrize("n,window,white", [(2, 0, []), (3, 64, [5, 9]), (1, 20, []), (35, 128, []), (1, 0, [3]), (200, 0, [])])
def test_selection_with_the_ngram_ban(ctx, n, window, white, check):
    _say(f"ban n={n} window={window} check={check}")
    rng = np.random.default_rng(n)
    groups, beams, vocab, cap = 3, 4, 5000, 200
    rows = groups * beams
    lens = [int(v) for v in rng.integers(0, cap + 1, rows)]
    lens[0], lens[1] = 0, cap
    history = rng.integers(0, 12, (rows, cap)).astype(np.uint32)
    if n == 35:
        history[:] = np.tile(rng.integers(0, vocab, (rows, 40)), 5).astype(np.uint32)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    x[:, :12] += 8  # the banned ones would win
    banned = [_bans(history[r, :lens[r]].tolist(), n, window) - set(white) for r in range(rows)]
    for r in range(rows):
        for t in banned[r]:
            x[r, t] += 3
    scores = (-rng.random(rows)).astype(np.float32)
    done = np.zeros(rows, np.uint8)
    kw = dict(ngram_size=n, window=window, whitelist=ctx.to_device(np.array(white, np.uint32)) if white else None)
    got = _run(ctx, x, scores, beams, done, history, lens, check=check, **kw)
    assert n == 200 or sum(map(len, banned)) > 0
    _same(got, _select(x, scores, beams, done, banned), done, beams)
    with pytest.raises(_abi.ContractViolation, match="history_len"):
        _run(ctx, x, scores, beams, done, history, [cap + 1] * rows, **kw)


@pytest.mark.parametrize("cap,window", [(256, 0), (257, 0), (700, 256), (700, 257), (700, 0)])
def test_ban_of_short_and_long_spans(ctx, cap, window):
    """Both ways of finding the ban, on either side of what the scan's blocks take, over several chunks of a row."""
    _say(f"ban cap={cap} window={window}")
    rng = np.random.default_rng(cap + window)
    rows, beams, vocab = 6, 3, 9000
    lens = [cap, cap - 1, 2, 300 if cap > 300 else 200, 1, 0]
    history = rng.integers(0, 30, (rows, cap)).astype(np.uint32) * 300  # tokens of every chunk
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    x[:, ::300] += 8
    banned = [_bans(history[r, :lens[r]].tolist(), 2, window) for r in range(rows)]
    assert sum(map(len, banned)) > 10
    scores, done = (-rng.random(rows)).astype(np.float32), np.zeros(rows, np.uint8)
    got = _run(ctx, x, scores, beams, done, history, lens, check=False, ngram_size=2, window=window)
    _same(got, _select(x, scores, beams, done, banned), done, beams)


def test_selection_in_place(ctx):
    _say("in place")
    from franken_ocr_amd.engine import beam_select

    rng = np.random.default_rng(8)
    x = rng.standard_normal((6, 700)).astype(np.float32)
    s, done = (-rng.random(6)).astype(np.float32), np.array([0, 1, 0, 0, 0, 1], np.uint8)
    want = _select(x, s, 3, done, [set()] * 6)
    ds, dd = ctx.to_device(s), ctx.to_device(done)
    p, t = ctx.empty((6,), np.uint32), ctx.empty((6,), np.uint32)
    beam_select(ctx.to_device(x), ds, 3, p, t, ds, done=dd, new_done=dd, eos=EOS)
    _same((p.numpy().tolist(), t.numpy().tolist(), ds.numpy(), dd.numpy().tolist()), want, done, 3)


def test_refusals(ctx):
    _say("refusals")
    from franken_ocr_amd.engine import PagedCache, RingCache, beam_reorder, beam_select

    E, S = _abi.FocrHipError, _abi.ContractViolation
    twice = PagedCache(4, 16, 1, 64, ctx=ctx)
    f, u = lambda *s: ctx.empty(s, np.float32), lambda *s: ctx.to_device(np.zeros(s, np.uint32))  # noqa: E731
    for call, text in (
            (lambda: beam_select(f(33, 10), f(33), 33, u(33), u(33), f(33)), "beams 33"),
            (lambda: beam_select(f(4, 0), f(4), 2, u(4), u(4), f(4)), "empty logits row"),
            (lambda: beam_select(f(4, 9), f(4), 2, u(4), u(4), f(4), ngram_size=2), "no-repeat-ngram"),
            (lambda: beam_select(f(4, 9), f(4), 2, u(4), None, f(4)), "null"),
            (lambda: beam_reorder(u(66), 33), "beams 33"),
            (lambda: beam_reorder(u(4), 2, history=u(4, 8)), "history_len"),
            (lambda: beam_reorder(u(4), 2, caches=[PagedCache(4, 16, 1, 64, ctx=ctx)]), "null"),
            (lambda: beam_reorder(u(4), 2, caches=[PagedCache(4, 16, 1, 64, ctx=ctx), PagedCache(4, 8, 1, 64, ctx=ctx)],
                                  tables=u(4, 2), lens=u(4)), "page sizes"),
            (lambda: beam_reorder(u(4), 2, caches=[twice, twice], tables=u(4, 2), lens=u(4)), "are the same"),
            (lambda: beam_select(f(2, 524289), f(2), 2, u(2), u(2), f(2)), "tier limit"),
            (lambda: beam_reorder(u(4), 2, rings=[RingCache(3, 8, ctx=ctx)]), "3 streams"),
            (lambda: beam_reorder(u(4), 2, rings=[RingCache(4, 8, ctx=ctx)]), "record_prefill")):
        with pytest.raises(E, match=text):
            call()
    ring = RingCache(2, 8, ctx=ctx)
    row = f(10 * 128 * 3)
    ring.record_prefill(0, row, row, 3)
    ring.record_prefill(1, row, row, 2)
    with pytest.raises(_abi.StateError, match="not where its group is"):
        beam_reorder(u(2), 2, rings=[ring])
    beam_select(f(0, 10), f(0), 2, u(0), u(0), f(0))  # no groups: nothing to do
    beam_reorder(u(0), 2)
    with pytest.raises(S, match="parent"):
        beam_reorder(ctx.to_device(np.array([0, 2], np.uint32)), 2, check=True)
    with pytest.raises(_abi.StateError, match="history is full"):
        beam_reorder(u(2), 2, tokens=u(2), history=u(2, 4), history_len=ctx.to_device(np.array([4, 3], np.uint32)), check=True)
    cache = PagedCache(4, 16, 1, 64, ctx=ctx)
    t = ctx.to_device(np.array([[0, 1], [2, 1]], np.uint32))
    for lens, error, text in (([17, 18], _abi.StateError, "group"), ([17, 17], _abi.StateError, "another beam"),
                              ([33, 33], _abi.StateError, "length")):
        with pytest.raises(error, match=text):
            beam_reorder(u(2), 2, caches=[cache], tables=t, lens=ctx.to_device(np.array(lens, np.uint32)), check=True)
    with pytest.raises(S, match="page"):
        beam_reorder(u(2), 2, caches=[cache], tables=ctx.to_device(np.array([[0, 1], [2, 9]], np.uint32)),
                     lens=ctx.to_device(np.array([17, 17], np.uint32)), check=True)


@pytest.mark.parametrize("beams,groups,layers,page,dtype", [(2, 1, 1, 16, "f32"), (5, 3, 2, 32, "bf16"), (8, 2, 3, 8, "f16"),
                                                            (13, 1, 35, 16, "f32"), (32, 2, 1, 64, "bf16"), (1, 4, 1, 16, "f16")])
def test_reorder_moves_the_states(ctx, beams, groups, layers, page, dtype):
    """Histories, tables, pages in progress (also more caches than one launch takes) and rings, exactly."""
    _say(f"reorder {groups} x {beams}, {layers} layers")
    from franken_ocr_amd.engine import RingCache, beam_reorder

    rng = np.random.default_rng(beams * 100 + layers)
    rows, cap = groups * beams, 90
    lens = [NONE if g == 3 else int(v) for g, v in enumerate(rng.integers(0, 5 * page, groups))]
    if groups > 1:
        lens[1] = 2 * page  # a page just filled
    lens = [lens[r // beams] for r in range(rows)]
    kv, dim = 2, 64
    hosts = [Host(rng, ctx, lens, page, kv, dim, dtype, wide=7) for _ in range(layers)]
    tables = hosts[0].tables.copy()
    for h in hosts:
        h.tables = tables
        for name in "kv":  # what the pages hold
            vals = rng.standard_normal(h.k.shape).astype(np.float32)
            vals = vals.astype(np.float16).astype(np.float32) if dtype == "f16" else vals
            if dtype == "bf16":
                vals = ((vals.view(np.uint32) >> 16) << 16).view(np.float32)
            setattr(h, name, vals)
        from test_gpu_paged import _bits

        h.dk.copy_from(_bits(h.k, dtype))
        h.dv.copy_from(_bits(h.v, dtype))
    parents = rng.integers(0, beams, rows).astype(np.uint32)
    tokens = rng.integers(0, 1000, rows).astype(np.uint32)
    history = rng.integers(0, 1000, (rows, cap)).astype(np.uint32)
    sizes = np.repeat(rng.integers(0, cap, groups), beams).astype(np.uint32)
    rings = [RingCache(rows, 16, ctx=ctx) for _ in range(2)] if rows <= 16 else []
    held = []
    for ring in rings:
        parts = {}
        for s in range(rows):
            pk = ctx.to_device(rng.standard_normal((10, 9, 128)).astype(np.float32))
            ring.record_prefill(s, pk, pk, 9)
            at = ring.regions(s)
            for name in ("ring_k", "ring_v"):
                x = rng.standard_normal((10, 128, 128)).astype(np.float32)
                _abi.call("focr_hip_h2d", ctx.handle, at[name], x.ctypes.data, x.nbytes)
                parts[s, name] = x
            ring.set_state(s, 128 if s // beams % 2 else 50, 3 if s // beams % 2 else 50)
        held.append(parts)
    dt, dl = ctx.to_device(tables), ctx.to_device(np.array(lens, np.uint32))
    dh, dn = ctx.to_device(history), ctx.to_device(sizes)
    beam_reorder(ctx.to_device(parents), beams, tokens=ctx.to_device(tokens), history=dh, history_len=dn, advance=True,
                 caches=[h.cache for h in hosts], tables=dt, lens=dl, rings=rings, check=True)
    src = np.arange(rows) // beams * beams + parents
    want = history.copy()
    for r in range(rows):
        want[r, :sizes[r]] = history[src[r], :sizes[r]]
        if sizes[r] < cap:
            want[r, sizes[r]] = tokens[r]
    assert np.array_equal(dh.numpy(), want) and np.array_equal(dn.numpy(), sizes + 1)
    wt = tables.copy()
    for r in range(rows):
        if lens[r] != NONE:
            full = lens[r] // page
            wt[r, :full] = tables[src[r], :full]
    assert np.array_equal(dt.numpy(), wt)
    for h in hosts:
        k0, v0 = h.k.copy(), h.v.copy()
        for r in range(rows):
            if lens[r] != NONE and lens[r] % page:
                full, rest = lens[r] // page, lens[r] % page
                h.k[tables[r, full], :, :rest] = k0[tables[src[r], full], :, :rest]
                h.v[tables[r, full], :, :rest] = v0[tables[src[r], full], :, :rest]
        h.same_pools()
    for ring, parts in zip(rings, held):
        for s in range(rows):
            at = ring.regions(s)
            count = 128 if s // beams % 2 else 50
            for name in ("ring_k", "ring_v"):
                x = np.empty((10, 128, 128), np.float32)
                _abi.call("focr_hip_d2h", ctx.handle, x.ctypes.data, at[name], x.nbytes)
                assert np.array_equal(x[:, :count], parts[src[s], name][:, :count])


def test_reorder_without_check_leaves_what_is_no_group(ctx):
    """Parents out of range are the slot itself; a group of different lengths keeps its tables and pages."""
    _say("reorder, unchecked")
    from franken_ocr_amd.engine import beam_reorder

    rng = np.random.default_rng(3)
    host = Host(rng, ctx, [20, 21, 40, 40, 40], 16, 2, 64, "f32", wide=4)
    # a group of [20, 21] cannot be made with the third beam's length: two groups of one table each
    parents = np.array([1, 0], np.uint32)
    t, n = ctx.to_device(host.tables[:2]), ctx.to_device(np.array([20, 21], np.uint32))
    beam_reorder(ctx.to_device(parents), 2, caches=[host.cache], tables=t, lens=n)
    assert np.array_equal(t.numpy(), host.tables[:2])
    host.same_pools()
    t, n = ctx.to_device(host.tables[2:]), ctx.to_device(np.array([40, 40, 40], np.uint32))
    bad = host.tables[2:].copy()
    beam_reorder(ctx.to_device(np.array([1, 3, 0xFFFFFFFF], np.uint32)), 3, caches=[host.cache], tables=t, lens=n)
    want = bad.copy()
    want[0, :2] = bad[1, :2]
    assert np.array_equal(t.numpy(), want)
    k0, v0 = host.k.copy(), host.v.copy()
    host.k[bad[0, 2], :, :8], host.v[bad[0, 2], :, :8] = k0[bad[1, 2], :, :8], v0[bad[1, 2], :, :8]
    host.same_pools()
    # a page in progress that the cache does not have: the group's pages stay
    bad = host.tables[2:].copy()
    bad[1, 2] = host.pages + 5
    beam_reorder(ctx.to_device(np.array([1, 0, 0], np.uint32)), 3, caches=[host.cache], tables=ctx.to_device(bad), lens=n)
    host.same_pools()


@pytest.mark.parametrize("beams,groups,kv,ldw,length,layers", [(2, 3, 3, 77, 40, 2), (5, 2, 1, 1000, 999, 35), (8, 1, 10, 64, 1, 1),
                                                               (13, 2, 2, 4099, 4098, 2), (32, 1, 1, 300, 257, 1)])
def test_reorder_moves_gathered_weights(ctx, beams, groups, kv, ldw, length, layers):
    """Every cache's gathered weights up to the length follow the parents, exactly; what lies behind it, a group that
    is none, a cache without weights: as they were."""
    _say(f"reorder weights {groups} x {beams}, {layers} layers")
    from franken_ocr_amd.engine import PagedCache, beam_reorder

    rng = np.random.default_rng(beams)
    rows, page, wide = groups * beams, 32, -(-(length + 40) // 32)
    lens = np.repeat([length if g != 1 else length + 7 for g in range(groups)], beams).astype(np.uint32)  # one past ldw
    if groups == 3:
        lens[-1] += 1  # no group: its lengths differ
    caches = [PagedCache(rows * wide, page, kv + i % 2, 64, "bf16", ctx=ctx) for i in range(layers)]
    tables = np.arange(rows * wide, dtype=np.uint32).reshape(rows, wide)
    w = [None if i == 1 else rng.random((rows, kv + i % 2, ldw)).astype(np.float32) for i in range(layers)]
    dw = [x if x is None else ctx.to_device(x) for x in w]
    parents = rng.integers(0, beams, rows).astype(np.uint32)
    dt = ctx.to_device(tables)
    beam_reorder(ctx.to_device(parents), beams, caches=caches, tables=dt, lens=ctx.to_device(lens), weights=dw)
    same = [len(set(lens[g * beams:(g + 1) * beams].tolist())) == 1 for g in range(groups)]
    src = np.array([r // beams * beams + parents[r] if same[r // beams] else r for r in range(rows)])
    for x, d in zip(w, dw):
        if x is not None:
            want = x.copy()
            for r in range(rows):
                want[r, :, :lens[r]] = x[src[r], :, :lens[r]]
            assert np.array_equal(d.numpy(), want)
    assert np.array_equal(dt.numpy()[:, :1], tables[src, :1] if length >= page else tables[:, :1])


def test_search_gathers_and_evicts_by_its_own_beams(ctx):
    """Steps that gather weights, reordered by drawn parents, then the eviction: each slot's weights are those of its
    ancestors' probabilities, kept apart on the host in 64 bits, and what it keeps are its own keys."""
    _say("weights of beams")
    from franken_ocr_amd.engine import PagedCache, beam_reorder
    from test_gpu_paged import _attend, _stay

    rng = np.random.default_rng(47)
    groups, beams, kv, heads, dim, page, steps, wide = 2, 3, 2, 6, 64, 8, 25, 8
    rows, prompts = groups * beams, [19, 8]
    cache = PagedCache(rows * (wide + 2), page, kv, dim, "f32", ctx=ctx)
    order = rng.permutation(rows * (wide + 2)).astype(np.uint32)
    tables, dst = order[: rows * wide].reshape(rows, wide).copy(), order[rows * wide:].reshape(rows, 2)

    class Beam:
        def __init__(self, k, v):
            self.kv, self.k, self.v = kv, k, v
            self.w, self.tol = np.zeros((kv, wide * page)), np.zeros((kv, wide * page))

        def rows(self, s, keys):
            return self.k[keys].astype(np.float64), self.v[keys].astype(np.float64)

        def after(self, k, v):
            b = Beam(np.concatenate([self.k, k[None]]), np.concatenate([self.v, v[None]]))
            b.w, b.tol = self.w.copy(), self.tol.copy()
            return b

    host = []
    for g in range(groups):
        k, v = (rng.standard_normal((prompts[g], kv, dim)).astype(np.float32) for _ in "kv")
        for b in range(beams):
            host.append(Beam(k, v))
    dt = ctx.to_device(tables)
    for r in range(rows):
        n = prompts[r // beams]
        flat = [ctx.to_device(x.reshape(n, -1)) for x in (host[r].k, host[r].v)]
        cache.write(*flat, ctx.to_device(np.arange(n, dtype=np.uint32)), dt, seq=ctx.to_device(np.full(n, r, np.uint32)), check=True)
    lens = ctx.to_device(np.repeat(prompts, beams).astype(np.uint32))
    dw, out = ctx.to_device(np.zeros((rows, kv, wide * page), np.float32)), ctx.empty((rows, heads * dim), np.float32)
    scale = 1.0 / np.sqrt(np.float32(dim))
    for i in range(steps):
        q = rng.standard_normal((rows, heads, dim)).astype(np.float32) * 2
        k, v = (rng.standard_normal((rows, kv, dim)).astype(np.float32) for _ in "kv")
        cache.step(ctx.to_device(q.reshape(rows, -1)), ctx.to_device(k.reshape(rows, -1)), ctx.to_device(v.reshape(rows, -1)),
                   dt, lens, out, weights=dw, advance=True, check=True)
        for r in range(rows):
            host[r] = host[r].after(k[r], v[r])
            _, _, keys, w, wt = _attend(host[r], 0, q[r], len(host[r].k), 0, 0, scale)
            host[r].w[:, keys] += w
            host[r].tol[:, keys] += wt + 2.0 ** -24 * (1 + host[r].w[:, keys])
        parents = rng.integers(0, beams, rows).astype(np.uint32)
        beam_reorder(ctx.to_device(parents), beams, caches=[cache], tables=dt, lens=lens, weights=[dw], check=True)
        host = [host[r // beams * beams + parents[r]] for r in range(rows)]
        got = dw.numpy()
        for r in range(rows):
            assert np.all(np.abs(got[r] - host[r].w) <= host[r].tol), (i, r)
    budget, dst_w = 2 * page, ctx.empty((rows, kv, 2 * page), np.float32)
    kept = ctx.empty((rows, kv, budget), np.uint32)
    cache.evict(dt, lens, dw, budget, ctx.to_device(dst), lens, dst_w, sinks=1, recent=3, kept=kept, check=True)
    pools = []
    for at in cache.regions().values():
        x = np.empty((rows * (wide + 2), kv, page, dim), np.float32)
        _abi.call("focr_hip_d2h", ctx.handle, x.ctypes.data, at, x.nbytes)
        pools.append(x)
    slots = np.arange(budget)
    for r in range(rows):
        for h in range(kv):
            stay = _stay(got[r, h], len(host[r].k), budget, 1, 3)
            assert np.array_equal(kept.numpy()[r, h], stay)
            for x, rows_of in zip(pools, (host[r].k, host[r].v)):
                assert np.array_equal(x[dst[r, slots // page], h, slots % page], rows_of[stay, h])


def test_reorder_refuses_tables_without_their_caches(ctx):
    _say("tables without caches")
    from franken_ocr_amd.engine import beam_reorder

    u = lambda *s: ctx.to_device(np.zeros(s, np.uint32))  # noqa: E731
    with pytest.raises(_abi.FocrHipError, match="none is given"):
        beam_reorder(u(2), 2, tables=u(2, 2), lens=u(2))


def test_reorder_refuses_weights_that_do_not_fit(ctx):
    _say("refusals of weights")
    from franken_ocr_amd.engine import PagedCache, beam_reorder

    caches = [PagedCache(4, 16, 1, 64, ctx=ctx) for _ in "ab"]
    u, w = (lambda *s: ctx.to_device(np.zeros(s, np.uint32))), (lambda *s: ctx.to_device(np.zeros(s, np.float32)))
    one = w(2, 1, 32)
    for weights, text in (([one], "1 weights for 2 caches"), ([one, w(2, 2, 32)], "weights of shape"),
                          ([w(2, 1, 16), one], "widths"), ([one, one], "are the same"), ([one, w(1, 1, 32)], "weights of shape"),
                          ([w(2, 1, 0), w(2, 1, 0)], "ldw 0")):
        with pytest.raises(_abi.FocrHipError, match=text):
            beam_reorder(u(2), 2, caches=caches, tables=u(2, 2), lens=u(2), weights=weights)


def test_beam_search_over_pages_and_rings(ctx):
    """Eight steps of search with a little model (one attention over what was read): the paged cache whose beams
    share the prompt's pages, and the ring caches, against every beam's keys kept apart on the host in 64 bits."""
    _say("search")
    from franken_ocr_amd.engine import HEAD_DIM, NUM_HEADS, PagedCache, RingCache, beam_reorder, beam_select

    rng = np.random.default_rng(31)
    groups, beams, vocab, page, steps = 2, 3, 500, 16, 30
    rows, D = groups * beams, NUM_HEADS * HEAD_DIM
    prompts = [37, 20]
    emb = {n: rng.standard_normal((vocab, D)).astype(np.float32) for n in "qkv"}
    w_out = (rng.standard_normal((D, vocab)) * (6 / np.sqrt(D))).astype(np.float32)
    wide = -(-(max(prompts) + steps + 1) // page)
    cache = PagedCache(rows * wide, page, NUM_HEADS, HEAD_DIM, "f32", ctx=ctx)
    tables = rng.permutation(rows * wide).astype(np.uint32).reshape(rows, wide)
    ring = RingCache(rows, 64, ctx=ctx)
    host = [[] for _ in range(rows)]  # each beam's (k, v) rows
    for g in range(groups):
        k, v = (rng.standard_normal((prompts[g], NUM_HEADS, HEAD_DIM)).astype(np.float32) for _ in "kv")
        full = prompts[g] // page
        for b in range(beams):
            r = g * beams + b
            tables[r, :full] = tables[g * beams, :full]  # the prompt's full pages are shared
            hm = [ctx.to_device(np.ascontiguousarray(a.transpose(1, 0, 2))) for a in (k, v)]
            ring.record_prefill(r, hm[0], hm[1], prompts[g])
            host[r] = [(k[i], v[i]) for i in range(prompts[g])]
        dt = ctx.to_device(tables)
        for b in range(beams):
            pos = np.arange(prompts[g], dtype=np.uint32)
            if b:
                pos[: full * page] = NONE
            cache.write(ctx.to_device(k.reshape(-1, D)), ctx.to_device(v.reshape(-1, D)), ctx.to_device(pos), dt,
                        seq=ctx.to_device(np.full(prompts[g], g * beams + b, np.uint32)), check=True)
    lens = ctx.to_device(np.repeat(prompts, beams).astype(np.uint32))
    scores = np.full(rows, -np.inf, np.float32)
    scores[::beams] = 0.0
    ds, dd = ctx.to_device(scores), ctx.to_device(np.zeros(rows, np.uint8))
    history, hl = ctx.to_device(np.zeros((rows, steps), np.uint32)), ctx.to_device(np.zeros(rows, np.uint32))
    p, t = ctx.empty((rows,), np.uint32), ctx.empty((rows,), np.uint32)
    out, out_ring = ctx.empty((rows, D), np.float32), ctx.empty((rows, D), np.float32)
    tokens, texts, done, mixed = np.full(rows, 2), [[] for _ in range(rows)], np.zeros(rows, np.uint8), 0
    for i in range(steps):
        q, k, v = (emb[n][tokens] for n in "qkv")
        dq, dk, dv = (ctx.to_device(a) for a in (q, k, v))
        cache.step(dq, dk, dv, dt, lens, out, advance=True)
        ring.step(dq, dk, dv, out_ring)
        got = out.numpy()
        assert np.allclose(got, out_ring.numpy(), rtol=0, atol=1e-4)
        for r in range(rows):
            host[r] = host[r] + [(k[r].reshape(NUM_HEADS, HEAD_DIM), v[r].reshape(NUM_HEADS, HEAD_DIM))]
            hk, hv = (np.stack([e[j] for e in host[r]]).astype(np.float64) for j in (0, 1))
            sc = np.einsum("nhd,hd->hn", hk, q[r].reshape(NUM_HEADS, HEAD_DIM).astype(np.float64)) / np.sqrt(HEAD_DIM)
            pr = np.exp(sc - sc.max(axis=1, keepdims=True))
            pr /= pr.sum(axis=1, keepdims=True)
            # scores under 60, values under 5: 2 (136 u 60 + 2^-22 + 131 u) 5 < 1e-2 at the very worst; 1e-4 of it taken
            assert np.allclose(got[r].reshape(NUM_HEADS, HEAD_DIM), np.einsum("hn,nhd->hd", pr, hv), rtol=0, atol=1e-4)
        logits = got @ w_out
        now = ds.numpy()
        banned = [_bans(texts[r], 2, 0) for r in range(rows)]
        want = _select(logits, now, beams, done, banned)
        beam_select(ctx.to_device(logits), ds, beams, p, t, ds, done=dd, new_done=dd, history=history, history_len=hl,
                    ngram_size=2, window=0, eos=EOS, check=True)
        assert p.numpy().tolist() == want[0] and t.numpy().tolist() == want[1]
        beam_reorder(p, beams, tokens=t, history=history, history_len=hl, advance=True, caches=[cache], tables=dt, lens=lens,
                     rings=[ring], check=True)
        src = np.arange(rows) // beams * beams + np.array(want[0])
        mixed += int(np.any(src != np.arange(rows)))
        host, texts = [host[s] for s in src], [texts[s] + [x] for s, x in zip(src, want[1])]
        tokens, done = np.array(want[1]), dd.numpy()
        assert history.numpy()[:, : i + 1].tolist() == texts
    assert mixed > steps // 3
    assert lens.numpy().tolist() == np.repeat([x + steps for x in prompts], beams).tolist()


def test_beam_search_over_the_decoder(ctx, model):  # noqa: F811
    """Decoder.step, beam_select and beam_reorder of its rings: each beam's text, fed to fresh caches token by token,
    has the score that the search gave it. A row of the decoder is the same whatever the other rows are, so the logits
    are the same bits; a score is rounded to f32 once a step, at most half a unit of its place each time."""
    _say("search over the decoder")
    from franken_ocr_amd.engine import RingCache, beam_reorder, beam_select

    H, V, G, beams, steps = 1280, 4096, 24, 3, 7
    layers, _, dec = _decoder(ctx, model)
    kv = [[ctx.to_device(synth.f32_normal(synth.seed_of(24000 + 2 * n + i), 10 * G * 128)) for i in (0, 1)] for n in range(3)]
    emb = synth.f32_normal(synth.seed_of(24100), V * H).reshape(V, H)

    def fresh():
        caches = []
        for k, v in kv:
            c = RingCache(beams, G, ctx=ctx)
            for s in range(beams):
                c.record_prefill(s, k, v, G)
            caches.append(c)
        return caches

    caches = fresh()
    logits, greedy = ctx.empty((beams, V), np.float32), ctx.empty((beams,), np.uint32)
    scores = ctx.to_device(np.array([0.0, -np.inf, -np.inf], np.float32))
    p, t = ctx.empty((beams,), np.uint32), ctx.empty((beams,), np.uint32)
    history, size = ctx.to_device(np.zeros((beams, steps), np.uint32)), ctx.to_device(np.zeros(beams, np.uint32))
    tokens, moved = np.full(beams, 5), 0
    for i in range(steps):
        dec.step(caches, np.full(beams, G + i, np.uint32), ctx.to_device(emb[tokens]), greedy, logits)
        if i == 0:  # a beam of one is the greedy step
            one = [ctx.empty((1,), np.uint32) for _ in "pt"]
            beam_select(logits.view_rows(0, 1), ctx.to_device(np.zeros(1, np.float32)), 1, *one, ctx.empty((1,), np.float32))
            assert one[1].numpy()[0] == greedy.numpy()[0]
        beam_select(logits, scores, beams, p, t, scores, history=history, history_len=size, ngram_size=2, window=0, eos=V)
        beam_reorder(p, beams, tokens=t, history=history, history_len=size, advance=True, rings=caches, check=True)
        tokens = t.numpy()
        moved += int(np.any(p.numpy() != np.arange(beams)))
    texts, got = history.numpy(), scores.numpy()
    assert moved > 0 and len({tuple(x) for x in texts.tolist()}) == beams
    assert np.all(np.diff(got) <= 0)
    again, feed, want = fresh(), np.full(beams, 5), np.zeros(beams)
    for i in range(steps):
        dec.step(again, np.full(beams, G + i, np.uint32), ctx.to_device(emb[feed]), greedy, logits)
        x = logits.numpy().astype(np.float64)
        m = x.max(axis=1)
        total = m + np.log(np.exp(x - m[:, None]).sum(axis=1))
        feed = texts[:, i]
        want += x[np.arange(beams), feed] - total
    assert np.all(np.abs(got - want) <= steps * (2.0 ** -24 * np.abs(want) + 1e-9)), (got, want)


@pytest.mark.parametrize("before", [0, 3])
def test_captured_reorder_of_rings_that_grow(ctx, before):
    """Rings reordered by a graph that was captured when they held `before` rows, replayed after eager steps: every
    row that they hold by then follows its parent, as by an eager call."""
    _say(f"captured, rings of {before} rows")
    from franken_ocr_amd.device import Context
    from franken_ocr_amd.engine import RingCache, beam_reorder

    c = Context(0)
    rng = np.random.default_rng(43)
    groups, beams, D = 2, 3, 1280
    rows = groups * beams
    rings = [RingCache(rows, 8, ctx=c) for _ in "ab"]  # by the graph, by eager calls
    for s in range(rows):
        k = c.to_device(rng.standard_normal((10, 4, 128)).astype(np.float32))
        for ring in rings:
            ring.record_prefill(s, k, k, 4)
    p, out = c.empty((rows,), np.uint32), c.empty((rows, D), np.float32)

    def steps(n):
        for _ in range(n):
            q, k, v = (c.to_device(rng.standard_normal((rows, D)).astype(np.float32)) for _ in "qkv")
            for ring in rings:
                ring.step(q, k, v, out)
            c.synchronize()  # before the rows go

    def held(ring):
        got = []
        for s in range(rows):
            at = ring.regions(s)
            for name in ("ring_k", "ring_v"):
                x = np.empty((10, 128, 128), np.float32)
                _abi.call("focr_hip_d2h", c.handle, x.ctypes.data, at[name], x.nbytes)
                got.append(x)
        return np.stack(got)

    steps(before)
    replay = _capture(c, lambda: beam_reorder(p, beams, rings=[rings[0]]))
    count = before
    for more in (2, 5, 60, 100):  # the last past the rings' end
        steps(more)
        count = min(128, count + more)
        parents = rng.integers(0, beams, rows).astype(np.uint32)
        p.copy_from(parents)
        assert replay() == 0
        c.synchronize()
        beam_reorder(p, beams, rings=[rings[1]])
        a, b = held(rings[0])[:, :, :count], held(rings[1])[:, :, :count]
        assert np.array_equal(a, b), more


def test_selection_leaves_a_captured_samplers_scratch(ctx):
    """A captured sampler call, then wider selections with a long ban: the graph's bitmaps and flags stay its own."""
    _say("captured sampler beside selections")
    from franken_ocr_amd.device import Context
    from franken_ocr_amd.engine import beam_select, sample_rows

    c = Context(0)
    rng = np.random.default_rng(44)
    vocab, cap = 3000, 300
    text = np.resize(np.arange(2, 42), cap).astype(np.uint32)  # after 40 tokens every one of them ends a 2-gram again
    logits = rng.standard_normal((2, vocab)).astype(np.float32)
    logits[0, 12] = logits[1, 22] = 40.0  # what came after the last token 40 tokens ago, and what has not come yet
    x, h, n = c.to_device(logits), c.to_device(np.stack([text, text])), c.to_device(np.array([90, 20], np.uint32))
    tok = c.empty((2,), np.uint32)

    def sample():
        sample_rows(x, tok, h, n, 2, 0)

    sample()
    want = tok.numpy()
    assert want[0] != 12 and want[1] == 22
    replay = _capture(c, sample)
    for rows, wide in ((8, 129280), (2000, 500)):
        p, t, s = c.empty((rows,), np.uint32), c.empty((rows,), np.uint32), c.to_device(np.zeros(rows, np.float32))
        beam_select(c.to_device(rng.standard_normal((rows, wide)).astype(np.float32)), s, 4, p, t, s,
                    history=c.to_device(np.zeros((rows, cap), np.uint32)), history_len=c.to_device(np.full(rows, cap, np.uint32)),
                    ngram_size=2, window=0)
        held = [c.empty((1 << 16,), np.uint8) for _ in range(8)]  # takes what was freed, if anything was
        for a in held:
            a.copy_from(np.full(1 << 16, 255, np.uint8))
        tok.copy_from(np.zeros(2, np.uint32))
        assert replay() == 0
        c.synchronize()
        assert np.array_equal(tok.numpy(), want)
        assert all(np.all(a.numpy() == 255) for a in held)


def test_captured_beam_step_replays(ctx):
    """Selection and reordering in one graph, replayed on changing logits, against the same calls made eagerly."""
    _say("captured")
    from franken_ocr_amd.device import Context
    from franken_ocr_amd.engine import PagedCache, beam_reorder, beam_select

    c = Context(0)
    rng = np.random.default_rng(41)
    groups, beams, vocab = 2, 4, 6000
    rows = groups * beams
    pool = rng.standard_normal((rows * 3, 2, 16, 64)).astype(np.float32)
    tables = np.arange(rows * 3, dtype=np.uint32).reshape(rows, 3)
    sides = []
    for _ in range(2):
        s = {"cache": PagedCache(rows * 3, 16, 2, 64, "f32", k=c.to_device(pool), v=c.to_device(pool), ctx=c),
             "t": c.to_device(tables), "n": c.to_device(np.full(rows, 25, np.uint32)),
             "h": c.to_device(rng.integers(0, 9, (rows, 64)).astype(np.uint32) * 0 + 3), "hl": c.to_device(np.full(rows, 10, np.uint32)),
             "x": c.empty((rows, vocab), np.float32), "s": c.to_device(np.zeros(rows, np.float32)),
             "p": c.empty((rows,), np.uint32), "tok": c.empty((rows,), np.uint32)}
        sides.append(s)

    def step(s):
        beam_select(s["x"], s["s"], beams, s["p"], s["tok"], s["s"], history=s["h"], history_len=s["hl"], ngram_size=2, window=0)
        beam_reorder(s["p"], beams, tokens=s["tok"], history=s["h"], history_len=s["hl"], advance=True, caches=[s["cache"]],
                     tables=s["t"], lens=s["n"])

    with pytest.raises(_abi.StateError, match="scratch"):
        _capture(c, lambda: step(sides[0]))
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    for s in sides:
        s["x"].copy_from(x)
        step(s)
    replay = _capture(c, lambda: step(sides[0]))
    for i in range(5):
        x = rng.standard_normal((rows, vocab)).astype(np.float32)
        for s in sides:
            s["x"].copy_from(x)
        assert replay() == 0
        c.synchronize()
        step(sides[1])
        for name in ("p", "tok", "s", "h", "hl", "t"):
            assert np.array_equal(sides[0][name].numpy(), sides[1][name].numpy()), (i, name)
        assert np.array_equal(sides[0]["cache"]._keep[0].numpy(), sides[1]["cache"]._keep[0].numpy())
