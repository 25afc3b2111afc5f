"""The paged key-value cache against the formulas in 64 bits.

What a call may not look at (slots past a length, outside a window, pages of
nobody) holds NaN in every test here. Tolerance of an output, per element: with
u = 2^-24, S the largest sum |scale q_i k_i| of a key and n the keys seen, a
score is off by at most (D + 4) u S (the dot's fused additions, the scale
folded into q), an exponential by 2^-22 of itself besides (hardware exp2, one
ulp, and the rounding of its argument, at most 2 S + 1 apart), and a chain of
sums by its length, at most n + 64, times u. Numerator and denominator both
have these, so
  |out - exact| <= sum_j P_j |v_j| * 2 ((D + 4 + 4) u S + 2^-22 + (n + 64) u)
and a gathered weight is off by P_j times that and the roundings of its sum."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from franken_ocr_amd import _abi

pytestmark = pytest.mark.gpu

NONE = 0xFFFFFFFF
U = 2.0 ** -24


def _say(msg):
    print(f"[gpu-paged] {msg}", flush=True)


# ---- the cache's types on the host -------------------------------------------------


def _round(x, dtype):
    """f32 values as the cache's type holds them (to nearest, ties to even), in f32."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x
    if dtype == "f16":
        return x.astype(np.float16).astype(np.float32)
    b = x.view(np.uint32).astype(np.uint64)
    b = (b + 0x7FFF + ((b >> 16) & 1)) >> 16 << 16
    return b.astype(np.uint32).view(np.float32)


def _bits(x, dtype):
    """The rounded values' storage."""
    if dtype == "f32":
        return np.ascontiguousarray(x, np.float32)
    if dtype == "f16":
        return x.astype(np.float16)
    return (np.ascontiguousarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def _np_type(dtype):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[dtype]


def _values(raw, dtype):
    return (raw.astype(np.uint32) << 16).view(np.float32) if dtype == "bf16" else raw.astype(np.float32)


class Host:
    """A cache and its tables as numpy holds them: every slot NaN until it is written."""

    def __init__(self, rng, ctx, lens, page, kv, dim, dtype, wide=None, spare=2):
        from franken_ocr_amd.engine import PagedCache

        self.rng, self.ctx, self.page, self.kv, self.dim, self.dtype = rng, ctx, page, kv, dim, dtype
        self.lens = list(lens)
        need = [0 if n == NONE else -(-(n + 1) // page) for n in lens]
        self.wide = wide or max(need + [1])
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages).astype(np.uint32)
        self.tables = np.full((len(lens), self.wide), NONE, np.uint32)  # entries of nobody name no page
        at = 0
        for s, n in enumerate(need):
            self.tables[s, :n] = order[at: at + n]
            at += n
        self.k = np.full((self.pages, kv, page, dim), np.nan, np.float32)
        self.v = self.k.copy()
        for s, n in enumerate(lens):
            if n != NONE:
                for j in range(n):
                    self.put(s, j, rng.standard_normal((kv, dim)), rng.standard_normal((kv, dim)))
        raw = [_bits(x, dtype) for x in (self.k, self.v)]
        self.dk, self.dv = (ctx.to_device(x) for x in raw)
        self.cache = PagedCache(self.pages, page, kv, dim, dtype, k=self.dk, v=self.dv, ctx=ctx)
        self.dt, self.dl = ctx.to_device(self.tables), ctx.to_device(np.array(lens, np.uint32))

    def put(self, s, j, k, v):
        at = self.tables[s, j // self.page], slice(None), j % self.page
        self.k[at], self.v[at] = _round(k, self.dtype), _round(v, self.dtype)

    def rows(self, s, keys):
        pages = self.tables[s, keys // self.page]
        return self.k[pages, :, keys % self.page].astype(np.float64), self.v[pages, :, keys % self.page].astype(np.float64)

    def pools(self):
        return self.dk.numpy(), self.dv.numpy()

    def same_pools(self):
        for got, want in zip(self.pools(), (self.k, self.v)):
            assert np.array_equal(_values(got, self.dtype), want, equal_nan=True)


def _seen(n, prefix, window):
    keys = np.arange(n)
    return keys if not window else keys[(keys < prefix) | (keys >= n - window)]


def _attend(host, s, q, n, prefix, window, scale):
    """Output, its tolerance, and the keys with their gathered probabilities and tolerance."""
    heads, d = q.shape
    keys = _seen(n, prefix, window)
    if len(keys) == 0:
        return np.zeros((heads, d)), np.zeros((heads, d)), keys, np.zeros((host.kv, 0)), np.zeros((host.kv, 0))
    k, v = host.rows(s, keys)
    group = heads // host.kv
    out, tol = np.zeros((heads, d)), np.zeros((heads, d))
    w, wt = np.zeros((host.kv, len(keys))), np.zeros((host.kv, len(keys)))
    for h in range(heads):
        kk, vv = k[:, h // group], v[:, h // group]
        sc = kk @ (q[h].astype(np.float64) * scale)
        big = (np.abs(kk) @ np.abs(q[h].astype(np.float64) * scale)).max()
        p = np.exp(sc - sc.max())
        p /= p.sum()
        rel = 2 * ((d + 8) * U * big + 2.0 ** -22 + (len(keys) + 64) * U)
        out[h], tol[h] = p @ vv, (p @ np.abs(vv)) * rel
        w[h // group] += p
        wt[h // group] += p * rel + (group + 1) * U
    return out, tol, keys, w, wt


CASES = [  # dtype, heads, kv heads, dim, page, lengths, prefix, window
    ("f32", 10, 10, 128, 16, [0, 1, 63, 64, 65, NONE, 300], 0, 0),
    ("bf16", 10, 10, 128, 32, [1, 2, 127, 513], 0, 0),
    ("f16", 4, 4, 64, 8, [5, 31, 32, 33, 700], 0, 0),
    ("f32", 6, 2, 64, 1, [0, 17, 100], 0, 0),             # three heads to a key head, one slot to a page
    ("bf16", 16, 2, 128, 16, [257, 4, 0, 64], 0, 0),      # eight
    ("f16", 24, 2, 64, 64, [1000, 1], 0, 0),              # twelve: two head tiles, the second half empty
    ("f32", 64, 1, 128, 128, [200, 3], 0, 0),             # sixty-four to one
    ("bf16", 5, 1, 256, 16, [129, 77], 0, 0),
    ("f32", 2, 1, 256, 1024, [1500, 64], 0, 0),
    ("f16", 14, 2, 256, 16, [2050, 9], 0, 0),
    ("bf16", 10, 10, 128, 16, [1, 9, 200, 1300, NONE, 40], 37, 128),
    ("f32", 4, 2, 64, 32, [600, 5, 130, 0], 0, 100),      # a window alone
    ("f16", 8, 8, 128, 16, [5000, 4999], 1000, 1),
]


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_and_step_against_64_bits(ctx, case, step):
    dtype, heads, kv, dim, page, lens, prefix, window = CASES[case]
    _say(f"case {case} {CASES[case]} step={step}")
    rng = np.random.default_rng(100 + case)
    host = Host(rng, ctx, lens, page, kv, dim, dtype)
    n, scale = len(lens), 1.0 / np.sqrt(np.float32(dim))
    ldq, ldkv, ldo = heads * dim + 3, kv * dim + 5, heads * dim + 1  # rows that start anywhere
    q = (1.5 * rng.standard_normal((n, ldq))).astype(np.float32)
    ks, vs = (rng.standard_normal((n, ldkv)).astype(np.float32) for _ in "kv")
    prefixes = np.array([max(0, prefix - 3 * s) for s in range(n)], np.uint32)
    slots = host.wide * page
    w0 = rng.random((n, kv, slots)).astype(np.float32)
    dout, dw = ctx.to_device(np.full((n, ldo), 7.0, np.float32)), ctx.to_device(w0)
    args = dict(prefix=ctx.to_device(prefixes) if prefix else None, window=window, weights=dw, n_heads=heads, ldq=ldq,
                ldo=ldo, check=True)
    if step:
        host.cache.step(ctx.to_device(q), ctx.to_device(ks), ctx.to_device(vs), host.dt, host.dl, dout, ldkv=ldkv,
                        advance=True, **args)
        for s in range(n):
            if lens[s] != NONE:
                host.put(s, lens[s], ks[s, :kv * dim].reshape(kv, dim), vs[s, :kv * dim].reshape(kv, dim))
    else:
        host.cache.attention(ctx.to_device(q), host.dt, host.dl, dout, **args)
    got, gw = dout.numpy(), dw.numpy()
    want_lens = [x if x == NONE else x + step for x in lens]
    assert host.dl.numpy().tolist() == want_lens
    host.same_pools()
    assert np.array_equal(got[:, heads * dim:], np.full((n, ldo - heads * dim), 7.0))  # between the rows: left
    for s, x in enumerate(want_lens):
        if x == NONE:
            assert np.all(got[s] == 7.0) and np.array_equal(gw[s], w0[s])
            continue
        out, tol, keys, w, wt = _attend(host, s, q[s, :heads * dim].reshape(heads, dim), x, int(prefixes[s]), window, scale)
        err = np.abs(got[s, :heads * dim].reshape(heads, dim) - out)
        assert np.all(err <= tol), (s, float((err - tol).max()))
        want = w0[s].astype(np.float64)
        want[:, keys] += w
        bound = np.zeros_like(want)
        bound[:, keys] = wt + U * (1 + np.abs(want[:, keys]))
        assert np.all(np.abs(gw[s] - want) <= bound), s
    # the same call gives the same bits
    again = ctx.to_device(np.full((n, ldo), 7.0, np.float32))
    args["weights"] = None
    host.cache.attention(ctx.to_device(q), host.dt, host.dl, again, **args)
    assert np.array_equal(again.numpy(), got)


MANY_SPLITS = [  # more than 64 splits of a row, whose joins have 1024 threads
    ("bf16", 4, 4, 64, 16, [5000, 100, 0], 0, 0),
    ("f32", 3, 1, 64, 64, [4800, NONE, 4799], 0, 0),
    ("f16", 2, 1, 256, 32, [5000, 64], 0, 0),
    ("bf16", 2, 2, 256, 128, [6001], 5000, 100),
]
EVERY_KERNEL = [(dtype, 2 * group, 2, dim, 8, [70, 0, NONE, 17], 0, 0)
                for dtype in ("f32", "f16", "bf16") for dim in (64, 128, 256) for group in (1, 2, 3)]


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("case", range(len(MANY_SPLITS)))
def test_joins_of_many_splits_against_64_bits(ctx, monkeypatch, case, step):
    monkeypatch.setitem(globals(), "CASES", MANY_SPLITS)
    test_attention_and_step_against_64_bits(ctx, case, step)


@pytest.mark.parametrize("case", range(len(EVERY_KERNEL)))
def test_steps_of_every_type_width_and_group_against_64_bits(ctx, monkeypatch, case):
    monkeypatch.setitem(globals(), "CASES", EVERY_KERNEL)
    test_attention_and_step_against_64_bits(ctx, case, True)


def test_write_rows_of_several_sequences(ctx):
    _say("write")
    rng = np.random.default_rng(7)
    for dtype in ("f32", "f16", "bf16"):
        host = Host(rng, ctx, [40, 17, 90], 16, 3, 64, dtype)
        seq = np.array([2, 0, 1, 0, 2, 1, 0], np.uint32)
        pos = np.array([3, 40, NONE, 0, 90, 17, 15], np.uint32)
        rows = rng.standard_normal((2, 7, 200)).astype(np.float32) * np.array([1e-6, 1, 1e6, 1, 3e4, 1, 1])[None, :, None].astype(np.float32)
        rows[0, 1, :5] = [0.0, -0.0, 2.0 ** -140, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8]  # ties and tiny values
        host.cache.write(ctx.to_device(rows[0]), ctx.to_device(rows[1]), ctx.to_device(pos), host.dt, seq=ctx.to_device(seq),
                         ldkv=200, check=True)
        with np.errstate(over="ignore"):
            for i in range(7):
                if pos[i] != NONE:
                    host.put(seq[i], int(pos[i]), rows[0, i, :192].reshape(3, 64), rows[1, i, :192].reshape(3, 64))
        host.same_pools()


def test_bad_pages_are_neither_read_nor_written(ctx):
    """Without check: a table that names pages the cache does not have, lengths past the tables."""
    _say("bad pages, unchecked")
    rng = np.random.default_rng(8)
    host = Host(rng, ctx, [50, 20, 40], 16, 2, 64, "f32")
    q = rng.standard_normal((3, 128)).astype(np.float32)
    bad = host.tables.copy()
    bad[0, 1] = host.pages          # keys 16 .. 31 of sequence 0
    bad[1, 1] = 0xFFFFFFF0          # where sequence 1's step would write
    lens = np.array([50, 20, 9999], np.uint32)  # sequence 2: cut to what the tables hold, on pages that are none
    dl, dout = ctx.to_device(lens), ctx.empty((3, 128), np.float32)
    host.cache.step(ctx.to_device(q), ctx.to_device(q), ctx.to_device(q), ctx.to_device(bad), dl, dout, advance=True)
    got = dout.numpy()
    assert dl.numpy().tolist() == [51, 21, 9999]
    host.put(0, 50, q[0].reshape(2, 64), q[0].reshape(2, 64))
    host.same_pools()
    keys = np.array([j for j in range(51) if not 16 <= j < 32])
    k, v = host.rows(0, keys)
    for h in range(2):
        sc = k[:, h] @ q[0].reshape(2, 64)[h].astype(np.float64) / 8
        p = np.exp(sc - sc.max())
        assert np.allclose(got[0].reshape(2, 64)[h], (p / p.sum()) @ v[:, h], rtol=0, atol=1e-4)


@pytest.mark.parametrize("heads", [2, 8])
def test_a_sequence_on_pages_that_are_none(ctx, heads):
    """Without check: 0 / 0 where no slot that is seen has a page, the other sequences as they are."""
    _say(f"pages of nobody, {heads} heads")
    rng = np.random.default_rng(19)
    host = Host(rng, ctx, [30, 20, 40], 16, 2, 64, "bf16")
    bad = host.tables.copy()
    bad[1] = NONE
    q = rng.standard_normal((3, heads, 64)).astype(np.float32)
    dout, dw = ctx.empty((3, heads * 64), np.float32), ctx.to_device(np.zeros((3, 2, 48), np.float32))
    host.cache.attention(ctx.to_device(q.reshape(3, -1)), ctx.to_device(bad), host.dl, dout, weights=dw)
    got, gw = dout.numpy().reshape(3, heads, 64), dw.numpy()
    assert np.all(np.isnan(got[1])) and np.all(np.isnan(gw[1, :, :20])) and np.all(gw[1, :, 20:] == 0)
    for s in (0, 2):
        out, tol, keys, w, wt = _attend(host, s, q[s], host.lens[s], 0, 0, 1.0 / np.sqrt(np.float32(64)))
        assert np.all(np.abs(got[s] - out) <= tol)
        assert np.all(np.abs(gw[s][:, keys] - w) <= wt + U * (1 + w))


@pytest.mark.parametrize("what", ["len", "page", "full", "dst page", "dst shared", "dst read", "seq", "pos"])
def test_check_reports_before_anything_is_written(ctx, what):
    _say(f"check: {what}")
    rng = np.random.default_rng(9)
    host = Host(rng, ctx, [50, 20, 33], 16, 2, 64, "f32", wide=4, spare=8)
    q = ctx.to_device(rng.standard_normal((3, 128)).astype(np.float32))
    out = ctx.to_device(np.full((3, 128), 7.0, np.float32))
    tables, lens, max_len = host.tables.copy(), np.array(host.lens, np.uint32), None
    free = sorted(set(range(host.pages)) - set(tables[tables != NONE].tolist()))
    dst = np.array(free[:6], np.uint32).reshape(3, 2)
    error, seq, pos = _abi.ContractViolation, np.array([0, 1, 2], np.uint32), np.array([1, 2, 3], np.uint32)
    if what == "len":
        lens[1], error = 65, _abi.StateError
    elif what == "full":
        max_len, error = 50, _abi.StateError
    elif what == "page":
        tables[2, 1] = host.pages
    elif what == "dst page":
        dst[1, 0] = host.pages
    elif what == "dst shared":
        dst[2, 1] = dst[0, 0]
    elif what == "dst read":
        dst[2, 1] = tables[0, 3]
    elif what == "seq":
        seq[1] = 3
    else:
        pos[2], error = 64, _abi.StateError
    dt, dl = ctx.to_device(tables), ctx.to_device(lens)
    with pytest.raises(error):
        if what in ("len", "page", "full"):
            host.cache.step(q, q, q, dt, dl, out, max_len=max_len, advance=True, check=True)
        elif what in ("seq", "pos"):
            host.cache.write(q, q, ctx.to_device(pos), dt, seq=ctx.to_device(seq), check=True)
        else:
            w = ctx.to_device(rng.random((3, 2, 64)).astype(np.float32))
            host.cache.evict(dt, dl, w, 30, ctx.to_device(dst), dl, ctx.to_device(np.zeros((3, 2, 32), np.float32)),
                             check=True)
    assert np.all(out.numpy() == 7.0) and np.array_equal(dl.numpy(), lens)
    host.same_pools()


def test_refusals(ctx):
    _say("refusals")
    from franken_ocr_amd.engine import PagedCache

    E, S = _abi.FocrHipError, _abi.ContractViolation
    for kw, text in (((8, 12, 2, 64, "f32"), "page_size"), ((8, 2048, 2, 64, "f32"), "page_size"),
                     ((8, 16, 2, 80, "f32"), "head_dim"), ((0, 16, 2, 64, "f32"), "n_pages"),
                     ((8, 16, 0, 64, "f32"), "n_kv_heads"), ((1 << 28, 16, 2, 64, "bf16"), "2\\^32")):
        with pytest.raises(S, match=text):
            PagedCache(*kw, ctx=ctx)
    pool = ctx.empty((8, 2, 16, 64), np.float32)
    with pytest.raises(E, match="one pool"):
        PagedCache(8, 16, 2, 64, "f32", k=pool, ctx=ctx)
    with pytest.raises(S, match="a pool of"):
        PagedCache(9, 16, 2, 64, "f32", k=pool, v=pool, ctx=ctx)
    c = PagedCache(8, 16, 2, 64, "f32", ctx=ctx)
    q, out = ctx.empty((2, 256), np.float32), ctx.empty((2, 256), np.float32)
    kv = ctx.empty((2, 128), np.float32)
    t, n = ctx.to_device(np.zeros((2, 2), np.uint32)), ctx.to_device(np.zeros(2, np.uint32))
    w = ctx.empty((2, 2, 32), np.float32)
    for call, text in (
            (lambda: c.attention(q, t, n, out, n_heads=3), "n_heads"),
            (lambda: c.attention(q, t, n, out, max_len=33), "max_len"),
            (lambda: c.attention(q, t, n, out, scale=float("nan")), "scale"),
            (lambda: c.attention(q, t, n, out, scale=-1.0), "scale"),
            (lambda: c.attention(q, t, n, out, n_heads=2, ldq=100), "stride"),
            (lambda: c.attention(q, t, n, out, weights=ctx.empty((2, 2, 31), np.float32)), "ldw"),
            (lambda: c.step(q, kv, None, t, n, out), "null"),
            (lambda: c.step(q, kv, kv, t, n, out, max_len=0), "max_len"),
            (lambda: c.evict(t, n, w, 0, t, n, w), "other pages"),
            (lambda: c.evict(t, n, w, 0, ctx.empty((2, 2), np.uint32), n, ctx.empty((2, 2, 32), np.float32)), "budget"),
            (lambda: c.evict(t, n, w, 8, ctx.empty((2, 2), np.uint32), n, ctx.empty((2, 2, 32), np.float32), sinks=5,
                             recent=4), "exceed the budget"),
            (lambda: c.evict(t, n, w, 20, ctx.empty((2, 1), np.uint32), n, ctx.empty((2, 2, 32), np.float32)), "do not hold"),
            (lambda: c.evict(t, n, w, 20, ctx.empty((2, 2), np.uint32), n, ctx.empty((2, 2, 19), np.float32)), "weights"),
            (lambda: c.write(kv, kv, ctx.empty((3,), np.uint32), t), "k of shape")):
        with pytest.raises(E, match=text):
            call()
    c.attention(ctx.empty((0, 256), np.float32), ctx.empty((0, 2), np.uint32), ctx.empty((0,), np.uint32),
                ctx.empty((0, 256), np.float32), n_heads=4)  # no sequences: nothing to do


def test_overlapping_pools_are_refused(ctx):
    """Keys and values in one memory, and caches of one call that share some: every row would be written twice."""
    _say("overlapping pools")
    from franken_ocr_amd.device import DeviceArray
    from franken_ocr_amd.engine import PagedCache, beam_reorder

    page = 2 * 16 * 64 * 4
    pool = ctx.empty((20 * page,), np.uint8)
    at = lambda p: DeviceArray.borrow(ctx, pool.ptr + p * page, (4 * page,), np.uint8)  # noqa: E731
    for k, v in ((0, 0), (0, 3), (7, 4)):
        with pytest.raises(_abi.FocrHipError, match="pools overlap"):
            PagedCache(4, 16, 2, 64, "f32", k=at(k), v=at(v), ctx=ctx)
    pair = lambda k, v: PagedCache(4, 16, 2, 64, "f32", k=at(k), v=at(v), ctx=ctx)  # noqa: E731
    a, n, p = pair(0, 4), ctx.to_device(np.zeros(2, np.uint32)), ctx.to_device(np.array([1, 0], np.uint32))
    t = ctx.to_device(np.array([[0, 1], [2, 3]], np.uint32))
    for k, v in ((8, 1), (4, 8), (3, 12), (8, 7)):
        with pytest.raises(_abi.FocrHipError, match="overlap"):
            beam_reorder(p, 2, caches=[a, pair(k, v)], tables=t, lens=n)
    beam_reorder(p, 2, caches=[a, pair(8, 12)], tables=t, lens=n)  # end to end


def test_scores_without_an_end(ctx):
    """Keys of -inf scores count for nothing; where there are no others, 0 / 0; a NaN key spreads."""
    _say("infinite scores")
    rng = np.random.default_rng(11)
    host = Host(rng, ctx, [100, 100, 100, 100], 16, 1, 64, "f32")
    q = np.abs(rng.standard_normal((4, 64))).astype(np.float32) + 0.1
    for s, keys in ((0, range(0, 100, 2)), (1, range(100)), (3, range(64))):
        for j in keys:
            host.k[host.tables[s, j // 16], 0, j % 16, 5] = -np.inf
    host.k[host.tables[2, 3], 0, 1, 0] = np.nan
    host.dk.copy_from(host.k)
    dout = ctx.empty((4, 64), np.float32)
    host.cache.attention(ctx.to_device(q), host.dt, host.dl, dout)
    got = dout.numpy()
    assert np.all(np.isnan(got[1])) and np.all(np.isnan(got[2]))
    for s, keys in ((0, np.arange(1, 100, 2)), (3, np.arange(64, 100))):
        k, v = host.rows(s, keys)
        sc = k[:, 0] @ q[s].astype(np.float64) / 8
        big = (np.abs(k[:, 0]) @ q[s].astype(np.float64)).max() / 8
        p = np.exp(sc - sc.max())
        p /= p.sum()
        tol = (p @ np.abs(v[:, 0])) * 2 * (72 * U * big + 2.0 ** -22 + 164 * U)
        assert np.all(np.abs(got[s] - p @ v[:, 0]) <= tol)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_infinities_with_grouped_heads(ctx, dtype):
    """Where q and the probabilities are split into terms: infinite keys (-inf scores), infinite values, NaN."""
    _say(f"infinities, grouped, {dtype}")
    rng = np.random.default_rng(14)
    heads, dim = 5, 64
    host = Host(rng, ctx, [100, 700, 100, 90, 40], 16, 1, dim, dtype)
    q = np.abs(rng.standard_normal((5, heads * dim))).astype(np.float32) + 0.1
    for s, keys in ((0, range(0, 100, 2)), (1, range(200, 700, 3)), (4, range(40))):
        for j in keys:
            host.k[host.tables[s, j // 16], 0, j % 16, 5] = -np.inf
    host.v[host.tables[2, 1], 0, 3, 7] = np.inf    # sequence 2, key 19
    host.v[host.tables[2, 2], 0, 1, 8] = -np.inf
    host.k[host.tables[3, 5], 0, 9, 0] = np.nan    # sequence 3, key 89
    host.dk.copy_from(_bits(host.k, dtype))
    host.dv.copy_from(_bits(host.v, dtype))
    dout = ctx.empty((5, heads * dim), np.float32)
    host.cache.attention(ctx.to_device(q), host.dt, host.dl, dout)
    got = dout.numpy().reshape(5, heads, dim)
    assert np.all(np.isnan(got[3])) and np.all(np.isnan(got[4]))
    for s in (0, 1, 2):
        out, tol, _, _, _ = _attend_finite(host, s, q[s].reshape(heads, dim), host.lens[s])
        if s == 2:
            assert np.all(got[2, :, 7] == np.inf) and np.all(got[2, :, 8] == -np.inf)
            out[:, 7:9], got[2, :, 7:9] = 0.0, 0.0
            tol[:, 7:9] = 0.0
        assert np.all(np.abs(got[s] - out) <= tol), s


def _attend_finite(host, s, q, n):
    """_attend over the keys without an infinite coordinate (the others' scores are -inf)."""
    keys = np.arange(n)
    k, v = host.rows(s, keys)
    keys = keys[np.isfinite(k[:, 0]).all(axis=1)]
    rows = host.rows

    class Part:
        kv = host.kv

        def rows(self, s_, keys_):
            kk, vv = rows(s_, keys[keys_])
            return kk, np.where(np.isinf(vv), 0.0, vv)

    return _attend(Part(), s, q, len(keys), 0, 0, 1.0 / np.sqrt(np.float32(q.shape[1])))


@pytest.mark.parametrize("dtype,unit", [("f16", 2.0 ** -20), ("bf16", 2.0 ** -126), ("f32", 2.0 ** -126), ("bf16", 2.0 ** 100),
                                        ("f16", 2.0 ** 12)])
@pytest.mark.parametrize("heads", [1, 2, 8])
def test_small_and_large_values(ctx, dtype, unit, heads):
    """Caches whose values are subnormal, or large, in their type: products and sums in f32 as they are."""
    _say(f"values of {unit} in {dtype}, {heads} heads")
    rng = np.random.default_rng(15)
    dim = 64
    host = Host(rng, ctx, [150, 33], 16, 1, dim, dtype)
    for s, n in enumerate(host.lens):
        for j in range(n):
            host.put(s, j, unit * rng.standard_normal((1, dim)), unit * rng.standard_normal((1, dim)))
    host.dk.copy_from(_bits(host.k, dtype))
    host.dv.copy_from(_bits(host.v, dtype))
    q = (rng.standard_normal((2, heads * dim)) / unit).astype(np.float32)
    if unit == 2.0 ** -126:
        q = (rng.standard_normal((2, heads * dim)) * 2.0 ** 120).astype(np.float32)
    dout = ctx.empty((2, heads * dim), np.float32)
    host.cache.attention(ctx.to_device(q), host.dt, host.dl, dout)
    got = dout.numpy().reshape(2, heads, dim)
    for s, n in enumerate(host.lens):
        out, tol, _, _, _ = _attend(host, s, q[s].reshape(heads, dim), n, 0, 0, 1.0 / np.sqrt(np.float32(dim)))
        # besides: what a sum of subnormal f32 products rounds away, half of the least one a product or sum
        assert np.all(np.abs(got[s] - out) <= tol + n * 2.0 ** -149), (s, float(np.abs(got[s] - out).max()))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads,dim", [(1, 64), (5, 64), (3, 128), (17, 256)])
def test_probabilities_far_below_the_greatest(ctx, dtype, heads, dim):
    """One heavy key with small, subnormal or zero values beside keys that are up to 70 octaves lighter and have large
    values: every probability keeps the bits that f32 gives it, whatever the others are.
    A score is one product here, off by at most 5 u of itself (the scale folded into q, the product, the exponential's
    argument), so a probability and the sum of them are off by 5 u S + 2^-22 and n + 64 roundings each."""
    _say(f"light keys with large values, {dtype}, {heads} heads, {dim} wide")
    rng = np.random.default_rng(16)
    octaves = [4, 14, 15, 18, 24, 27, 28, 29, 30, 34, 38, 41, 48, 70]
    n = 150
    host = Host(rng, ctx, [n] * len(octaves), 16, 1, dim, dtype)
    q = np.zeros((len(octaves), heads, dim), np.float32)
    q[:, :, 0] = 1 + 0.01 * np.arange(heads)
    for s, deep in enumerate(octaves):
        heavy = int(rng.integers(n))
        for j in range(n):
            k, v = np.zeros((1, dim)), rng.standard_normal((1, dim)) * 2.0 ** 13
            k[0, 0] = -deep * np.log(2) * rng.uniform(0.95, 1.0)
            if j == heavy:
                k[0, 0], v = 0.0, np.resize([2.0 ** -10, 0.0, 2.0 ** -24, 1.0], (1, dim))
            host.put(s, j, k, v)
    host.dk.copy_from(_bits(host.k, dtype))
    host.dv.copy_from(_bits(host.v, dtype))
    dout = ctx.empty((len(octaves), heads * dim), np.float32)
    host.cache.attention(ctx.to_device(q.reshape(len(octaves), -1)), host.dt, host.dl, dout, scale=1.0)
    got = dout.numpy().reshape(q.shape)
    for s, deep in enumerate(octaves):
        k, v = host.rows(s, np.arange(n))
        for h in range(heads):
            sc = k[:, 0, 0] * float(q[s, h, 0])
            p = np.exp(sc - sc.max())
            p /= p.sum()
            tol = (p @ np.abs(v[:, 0])) * 2 * (5 * U * np.abs(sc).max() + 2.0 ** -22 + (n + 64) * U)
            assert np.all(np.abs(got[s, h] - p @ v[:, 0]) <= tol), (deep, h, float((np.abs(got[s, h] - p @ v[:, 0]) / tol).max()))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads,dim", [(2, 128), (4, 64), (16, 128), (20, 256)])
def test_query_rows_of_mixed_magnitude(ctx, dtype, heads, dim):
    """A query row with one coordinate far above the others, where the keys are zero: the others keep their bits."""
    _say(f"mixed query rows, {dtype}, {heads} heads, {dim} wide")
    rng = np.random.default_rng(17)
    far = [0, 12, 16, 20, 24, 27, 28, 29, 32, 36]  # octaves between the large coordinate and the others
    n = 100
    host = Host(rng, ctx, [n] * len(far), 32, 1, dim, dtype)
    for s in range(len(far)):
        for j in range(n):
            k = rng.standard_normal((1, dim)) * 2.0 ** 12
            k[0, 7] = 0.0
            host.put(s, j, k, rng.standard_normal((1, dim)))
    host.dk.copy_from(_bits(host.k, dtype))
    host.dv.copy_from(_bits(host.v, dtype))
    q = (rng.standard_normal((len(far), heads, dim)) * 2.0 ** -11).astype(np.float32)
    for s, octaves in enumerate(far):
        q[s, :, 7] = 2.0 ** (octaves - 11)
    dout = ctx.empty((len(far), heads * dim), np.float32)
    host.cache.attention(ctx.to_device(q.reshape(len(far), -1)), host.dt, host.dl, dout)
    got = dout.numpy().reshape(q.shape)
    for s, octaves in enumerate(far):
        out, tol, _, _, _ = _attend(host, s, q[s], n, 0, 0, 1.0 / np.sqrt(np.float32(dim)))
        assert np.all(np.abs(got[s] - out) <= tol), (octaves, float((np.abs(got[s] - out) / tol).max()))


def test_scores_of_a_window_take_the_windows_room(ctx):
    """Weights under a window alone: scratch for the keys that it shows, whatever the tables hold, and the same results."""
    _say("scores of a window")
    from franken_ocr_amd.device import Context

    c = Context(0)
    rng = np.random.default_rng(18)
    window, heads, dim = 100, 16, 64
    host = Host(rng, c, [300, 100, 99, 0, NONE, 101, 1], 16, 2, dim, "bf16", wide=4096)  # 65536 slots
    n = len(host.lens)
    q = rng.standard_normal((n, heads, dim)).astype(np.float32)
    dout, dw = c.empty((n, heads * dim), np.float32), c.to_device(np.zeros((n, 2, 65536), np.float32))
    host.cache.attention(c.to_device(q.reshape(n, -1)), host.dt, host.dl, dout, window=window, weights=dw, check=True)
    assert c.scratch_bytes() < 2 << 20  # 112 rows of scores over all slots take 29 MB, of two splits of 64 keys 0.1
    got, gw = dout.numpy().reshape(n, heads, dim), dw.numpy()
    for s, x in enumerate(host.lens):
        if x == NONE:
            continue
        out, tol, keys, w, wt = _attend(host, s, q[s], x, 0, window, 1.0 / np.sqrt(np.float32(dim)))
        assert np.all(np.abs(got[s] - out) <= tol), s
        want, bound = np.zeros((2, 65536)), np.zeros((2, 65536))
        want[:, keys], bound[:, keys] = w, wt + U * (1 + w)
        assert np.all(np.abs(gw[s] - want) <= bound), s


def test_far_offsets(ctx):
    """Pages past 2^32 bytes and 2^31 values of a pool."""
    _say("far offsets")
    from franken_ocr_amd.engine import PagedCache

    rng = np.random.default_rng(12)
    pages, page, kv, dim = 9000, 64, 16, 256  # 2^20 bytes a page: 9.4 GB a pool
    cache = PagedCache(pages, page, kv, dim, "f32", ctx=ctx)
    at = cache.regions()
    table = np.array([[8999, 8197, 0]], np.uint32)
    k, v = (rng.standard_normal((3, kv, page, dim)).astype(np.float32) for _ in "kv")
    for base, x in ((at["k"], k), (at["v"], v)):
        for i, p in enumerate(table[0].tolist()):
            _abi.call("focr_hip_h2d", ctx.handle, C.c_void_p(base + p * x[i].nbytes), x[i].ctypes.data_as(C.c_void_p), x[i].nbytes)
    q = rng.standard_normal((1, kv * dim)).astype(np.float32)
    row = rng.standard_normal((1, kv * dim)).astype(np.float32)
    dl, dout = ctx.to_device(np.array([70], np.uint32)), ctx.empty((1, kv * dim), np.float32)
    cache.step(ctx.to_device(q), ctx.to_device(row), ctx.to_device(row), ctx.to_device(table), dl, dout, check=True)
    back = np.empty((kv, page, dim), np.float32)
    _abi.call("focr_hip_d2h", ctx.handle, back.ctypes.data_as(C.c_void_p), C.c_void_p(at["k"] + 8197 * back.nbytes), back.nbytes)
    k[1, :, 6] = v[1, :, 6] = row.reshape(kv, dim)
    assert np.array_equal(back, k[1])
    kk = k.transpose(1, 0, 2, 3).reshape(kv, -1, dim)[:, :71].astype(np.float64)
    vv = v.transpose(1, 0, 2, 3).reshape(kv, -1, dim)[:, :71].astype(np.float64)
    qq = q.reshape(kv, dim).astype(np.float64) / 16
    for h in range(kv):
        sc = kk[h] @ qq[h]
        p = np.exp(sc - sc.max())
        p /= p.sum()
        tol = (p @ np.abs(vv[h])) * 2 * (264 * U * (np.abs(kk[h]) @ np.abs(qq[h])).max() + 2.0 ** -22 + 135 * U)
        assert np.all(np.abs(dout.numpy().reshape(kv, dim)[h] - p @ vv[h]) <= tol)
    cache.free()


def test_paged_steps_see_what_the_ring_sees(ctx):
    """The prompt as prefix and a window of 128: the R-SWA step's own outputs, past the ring's first turn."""
    _say("ring against pages")
    from franken_ocr_amd.engine import HEAD_DIM, NUM_HEADS, PagedCache, RingCache

    rng = np.random.default_rng(13)
    G, steps, page, wide = 90, 150, 32, 8
    ring = RingCache(2, 128, ctx=ctx)
    cache = PagedCache(2 * wide, page, NUM_HEADS, HEAD_DIM, "f32", ctx=ctx)
    tables = rng.permutation(2 * wide).astype(np.uint32).reshape(2, wide)
    dt, dl = ctx.to_device(tables), ctx.to_device(np.full(2, G, np.uint32))
    for s in range(2):
        k, v = (rng.standard_normal((G, NUM_HEADS, HEAD_DIM)).astype(np.float32) for _ in "kv")
        hm = [ctx.to_device(np.ascontiguousarray(x.transpose(1, 0, 2))) for x in (k, v)]
        ring.record_prefill(s, hm[0], hm[1], G)
        cache.write(ctx.to_device(k.reshape(G, -1)), ctx.to_device(v.reshape(G, -1)), ctx.to_device(np.arange(G, dtype=np.uint32)),
                    dt, seq=ctx.to_device(np.full(G, s, np.uint32)), check=True)
    prefix = ctx.to_device(np.full(2, G, np.uint32))
    a, b = (ctx.empty((2, NUM_HEADS * HEAD_DIM), np.float32) for _ in "ab")
    for i in range(steps):
        q, k, v = (ctx.to_device(rng.standard_normal((2, NUM_HEADS * HEAD_DIM)).astype(np.float32)) for _ in "qkv")
        ring.step(q, k, v, a)
        cache.step(q, k, v, dt, dl, b, prefix=prefix, window=128, advance=True)
        if i in (0, 1, 100, 126, 127, 128, 129, 149):
            # each is off the exact value by at most 2 (136 u S + 2^-22 + 282 u) max |v|, S under 80, |v| under 5:
            # 3e-3 at worst; the sums' roundings mostly cancel
            assert np.allclose(a.numpy(), b.numpy(), rtol=0, atol=1e-4), i
    assert dl.numpy().tolist() == [G + steps] * 2


# ---- eviction -------------------------------------------------------------------------


def _stay(w, n, budget, sinks, recent):
    if n <= budget:
        return np.arange(n)
    lo, hi = sinks, n - recent
    key = np.where(np.isnan(w[lo:hi]), -np.inf, w[lo:hi].astype(np.float64))
    nan = np.isnan(w[lo:hi])
    order = np.lexsort((np.arange(hi - lo), nan, -key))  # weight, then NaN behind -inf, then the slot
    return np.sort(np.concatenate([np.arange(lo), order[: budget - lo - recent] + lo, np.arange(hi, n)]))


@pytest.mark.parametrize("dtype,kv,dim,page,lens,budget,sinks,recent", [
    ("f32", 3, 128, 16, [200, 40, 41, 0, NONE, 1], 40, 4, 10),
    ("bf16", 2, 64, 8, [1000, 999, 100], 100, 0, 0),
    ("f16", 1, 256, 64, [3000, 2049], 1025, 1, 1024),   # sinks and recent leave nothing to choose
    ("f32", 2, 64, 32, [5000, 4097], 2047, 0, 7),
    ("bf16", 4, 128, 1, [70, 33], 1, 0, 0),
    ("f32", 1, 64, 16, [100, 20], 500, 3, 3),           # a budget that nothing reaches
    ("f16", 2, 128, 128, [40000], 20000, 2, 77),
])
def test_evict_keeps_the_heaviest(ctx, dtype, kv, dim, page, lens, budget, sinks, recent):
    _say(f"evict {dtype} {lens} to {budget}")
    rng = np.random.default_rng(sum(x for x in lens if x != NONE) + budget)
    n = len(lens)
    longest = max(x for x in lens if x != NONE)
    most = min(budget, longest)
    dst_wide = -(-most // page)
    need = n * dst_wide
    host = Host.__new__(Host)
    host.rng, host.ctx, host.page, host.kv, host.dim, host.dtype = rng, ctx, page, kv, dim, dtype
    from franken_ocr_amd.engine import PagedCache

    pages_of = [0 if x == NONE else -(-x // page) for x in lens]
    host.wide, host.pages = max(pages_of), sum(pages_of) + need + 1
    order = rng.permutation(host.pages).astype(np.uint32)
    host.tables = np.full((n, host.wide), NONE, np.uint32)
    at = need
    for s, c in enumerate(pages_of):
        host.tables[s, :c] = order[at: at + c]
        at += c
    dst = order[:need].reshape(n, dst_wide).copy()
    host.k, host.v = (_round(rng.standard_normal((host.pages, kv, page, dim)), dtype) for _ in "kv")
    host.dk, host.dv = ctx.to_device(_bits(host.k, dtype)), ctx.to_device(_bits(host.v, dtype))
    cache = PagedCache(host.pages, page, kv, dim, dtype, k=host.dk, v=host.dv, ctx=ctx)
    ldw = host.wide * page + 3
    w = np.exp(3 * rng.standard_normal((n, kv, ldw))).astype(np.float32)
    w[rng.random(w.shape) < 0.3] = 0.0       # equal ones
    w[rng.random(w.shape) < 0.05] = -0.0     # equal to those
    w[rng.random(w.shape) < 0.02] = np.nan
    w[rng.random(w.shape) < 0.01] = np.inf
    w[rng.random(w.shape) < 0.02] = -1.0
    dw, dst_w = ctx.to_device(w), ctx.to_device(np.full((n, kv, most + 2), 7.0, np.float32))
    kept = ctx.to_device(np.full((n, kv, budget), 9, np.uint32))
    dl = ctx.to_device(np.array(lens, np.uint32))
    cache.evict(ctx.to_device(host.tables), dl, dw, budget, ctx.to_device(dst), dl, dst_w, sinks=sinks, recent=recent,
                max_len=longest, kept=kept, check=True)
    got_w, got_kept = dst_w.numpy(), kept.numpy()
    assert dl.numpy().tolist() == [x if x == NONE else min(x, budget) for x in lens]
    k0, v0 = host.k.copy(), host.v.copy()
    for s, x in enumerate(lens):
        for h in range(kv):
            stay = np.arange(0) if x == NONE else _stay(w[s, h], x, budget, sinks, recent)
            c = len(stay)
            assert np.array_equal(got_kept[s, h, :c], stay), (s, h)
            assert np.all(got_kept[s, h, c:] == 9) and np.all(got_w[s, h, c:] == 7.0)
            assert np.array_equal(got_w[s, h, :c], w[s, h, stay], equal_nan=True)
            to, src = np.arange(c), host.tables[s, stay // page]
            host.k[dst[s, to // page], h, to % page] = k0[src, h, stay % page]
            host.v[dst[s, to // page], h, to % page] = v0[src, h, stay % page]
    host.same_pools()
    # without the list of slots, the same rows
    host.dk.copy_from(_bits(k0, dtype))
    host.dv.copy_from(_bits(v0, dtype))
    dl.copy_from(np.array(lens, np.uint32))
    cache.evict(ctx.to_device(host.tables), dl, dw, budget, ctx.to_device(dst), dl, dst_w, sinks=sinks, recent=recent,
                max_len=longest)
    host.same_pools()


@pytest.mark.parametrize("dtype,kv,dim,page,lens,budget,sinks,recent", [
    ("bf16", 2, 64, 128, [12000, 9000, 8193, 5, NONE], 4000, 4, 128),                   # a row in one tile of 16384 slots
    ("f16", 1, 64, 64, [16384, 16383], 12300, 0, 1),                                    # ties at the threshold: zeros
    ("bf16", 2, 64, 128, [33000, 17000, 16385, 16384] + [40 + s for s in range(61)], 25000, 1, 300),  # 130 rows: tile by tile
    ("f16", 3, 64, 128, [100] * 50 + [40001], 29000, 7, 0),                             # the same, ties across its tiles
    ("bf16", 2, 64, 128, [40001, 300, 0, NONE, 16385], 29000, 7, 0),                    # few rows: a block to a tile
    ("f32", 2, 256, 16, [500, 90], 100, 3, 20),                                         # rows of 1 KB
])
def test_evict_of_every_selection(ctx, dtype, kv, dim, page, lens, budget, sinks, recent):
    test_evict_keeps_the_heaviest(ctx, dtype, kv, dim, page, lens, budget, sinks, recent)


# ---- graphs, streams, contexts --------------------------------------------------------


def _hip():
    path = next(ln.split()[-1] for ln in open("/proc/self/maps") if "libamdhip64" in ln)
    return C.CDLL(path)


def _capture(ctx, call):
    hip, stream = _hip(), C.c_void_p(ctx.stream())
    graph, ex = C.c_void_p(), C.c_void_p()
    ctx.synchronize()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    try:
        call()
    finally:
        rc = hip.hipStreamEndCapture(stream, C.byref(graph))
    assert rc == 0
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
    hip.hipGraphDestroy(graph)
    return lambda: hip.hipGraphLaunch(ex, stream)


def test_captured_step_replays_while_lengths_grow(ctx):
    """One captured step, replayed: lengths, pages and weights as by calls; then larger calls that outgrow
    the scratch the graph uses, and the graph again."""
    _say("captured step")
    from franken_ocr_amd.device import Context

    c = Context(0)
    rng = np.random.default_rng(21)
    pages = rng.permutation(24).astype(np.uint32).reshape(3, 8)
    from franken_ocr_amd.engine import PagedCache

    pool = _round(rng.standard_normal((24, 2, 16, 64)), "bf16")
    caches, lens, outs, ws, q, k = [], [], [], [], [], []
    dt = c.to_device(pages)
    for _ in "ab":
        caches.append(PagedCache(24, 16, 2, 64, "bf16", k=c.to_device(_bits(pool, "bf16")), v=c.to_device(_bits(pool, "bf16")), ctx=c))
        lens.append(c.to_device(np.array([30, 61, 5], np.uint32)))
        outs.append(c.empty((3, 256), np.float32))
        ws.append(c.to_device(np.zeros((3, 2, 128), np.float32)))
        q.append(c.empty((3, 256), np.float32))
        k.append(c.empty((3, 128), np.float32))

    def step(i):
        caches[i].step(q[i], k[i], k[i], dt, lens[i], outs[i], weights=ws[i], advance=True)

    with pytest.raises(_abi.StateError, match="scratch"):
        _capture(c, lambda: step(0))  # nothing is there yet
    step(0)
    c.synchronize()
    lens[0].copy_from(np.array([30, 61, 5], np.uint32))
    ws[0].copy_from(np.zeros((3, 2, 128), np.float32))
    caches[0]._keep[0].copy_from(_bits(pool, "bf16"))
    caches[0]._keep[1].copy_from(_bits(pool, "bf16"))
    replay = _capture(c, lambda: step(0))
    for i in range(6):
        x, y = rng.standard_normal((3, 256)).astype(np.float32), rng.standard_normal((3, 128)).astype(np.float32)
        for j in range(2):
            q[j].copy_from(x)
            k[j].copy_from(y)
        assert replay() == 0
        c.synchronize()
        step(1)
        assert np.array_equal(outs[0].numpy(), outs[1].numpy()), i
        assert np.array_equal(ws[0].numpy(), ws[1].numpy()) and np.array_equal(lens[0].numpy(), lens[1].numpy())
        assert np.array_equal(caches[0]._keep[0].numpy(), caches[1]._keep[0].numpy())
        if i == 2:  # a larger call: other scratch, the graph's stays
            big = Host(rng, c, [900, 800, 700, 600], 16, 2, 64, "f32")
            big.cache.attention(c.to_device(rng.standard_normal((4, 256)).astype(np.float32)), big.dt, big.dl, c.empty((4, 256), np.float32),
                                weights=c.to_device(np.zeros((4, 2, big.wide * 16), np.float32)))
    assert lens[0].numpy().tolist() == [36, 67, 11]
    with pytest.raises(_abi.StateError, match="check"):
        _capture(c, lambda: caches[0].step(q[0], k[0], k[0], dt, lens[0], outs[0], check=True))


def test_a_cache_outlives_its_context(ctx):
    """A cache made with a context that is gone by now: used with another, and freed."""
    _say("cache of a closed context")
    from franken_ocr_amd.device import Context
    from franken_ocr_amd.engine import PagedCache

    rng = np.random.default_rng(23)
    c = Context(0)
    cache = PagedCache(6, 16, 1, 64, "f32", ctx=c)
    c.close()
    cache.ctx = ctx
    k, v = (rng.standard_normal((40, 64)).astype(np.float32) for _ in "kv")
    q = rng.standard_normal((1, 64)).astype(np.float32)
    t, n, out = ctx.to_device(np.array([[4, 1, 5]], np.uint32)), ctx.to_device(np.array([40], np.uint32)), ctx.empty((1, 64), np.float32)
    cache.write(ctx.to_device(k), ctx.to_device(v), ctx.to_device(np.arange(40, dtype=np.uint32)), t,
                seq=ctx.to_device(np.zeros(40, np.uint32)), check=True)
    cache.attention(ctx.to_device(q), t, n, out, check=True)
    sc = k.astype(np.float64) @ q[0] / 8
    p = np.exp(sc - sc.max())
    p /= p.sum()
    tol = (p @ np.abs(v)) * 2 * (72 * U * (np.abs(k) @ np.abs(q[0])).max() / 8 + 2.0 ** -22 + 104 * U)
    assert np.all(np.abs(out.numpy()[0] - p @ v) <= tol)
    cache.free()


def test_two_contexts_at_once(ctx):
    """Calls of two contexts on caches of their own, issued in turn without waiting."""
    _say("two contexts")
    from franken_ocr_amd.device import Context

    rng = np.random.default_rng(22)
    cs = [Context(0), Context(0)]
    hosts = [Host(rng, c, [700, 300], 16, 2, 128, "f32") for c in cs]
    qs = [c.to_device(rng.standard_normal((2, 256)).astype(np.float32)) for c in cs]
    alone = []
    for c, h, q in zip(cs, hosts, qs):
        o = c.empty((2, 256), np.float32)
        h.cache.attention(q, h.dt, h.dl, o)
        alone.append(o.numpy())
    outs = [[c.empty((2, 256), np.float32) for _ in range(8)] for c in cs]
    for i in range(8):
        for c, h, q, o in zip(cs, hosts, qs, outs):
            h.cache.attention(q, h.dt, h.dl, o[i])
    for o, want in zip(outs, alone):
        for x in o:
            assert np.array_equal(x.numpy(), want)
