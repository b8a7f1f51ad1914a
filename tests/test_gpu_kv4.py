"""The paged 4-bit K/V cache on the device against 64 bits (tests/kv4_reference.py).

Stored codes and scale bytes are compared bit for bit (the kernel computes the value in 64
bits, so the nearest code is the reference's); queries to half a step of their type; the
attention to the allowance that kv4_reference derives from its roundings, and, over all
outputs, to a relative 2-norm of 1e-5 in f32 and 2^-8 in bf16 (every output's own rounding
is at most 2^-8 of it)."""
import ctypes as C

import numpy as np
import pytest

import kv4_reference as R
import oracle_lib as O
import ttlab_amd as T

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = T.Device(0)
    yield d
    d.close()


class Held:
    """Device buffers of a test, given back at its end."""

    def __init__(self, dev):
        self.dev, self.bufs = dev, []

    def up(self, a):
        self.bufs.append(self.dev.upload(a))
        return self.bufs[-1]

    def new(self, nbytes, fill=None):
        b = self.dev.alloc(max(int(nbytes), 256))
        if fill is not None:
            self.dev.fill(b, fill)
        self.bufs.append(b)
        return b


@pytest.fixture
def held(dev):
    h = Held(dev)
    yield h
    dev.sync()
    for b in h.bufs:
        b.free()


def cumulative(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


def rope_table(n, hd, rng):
    angle = np.arange(n)[:, None] * 150000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    return (np.stack([np.cos(angle), np.sin(angle)], -1) * 1.3466).astype(np.float32)


def to_dtype(x, dtype):
    """(f64 values as held, the array to upload)."""
    if dtype == T.TTL_DTYPE_BF16:
        v, bits = R.bf16_round(x)
        return v.astype(np.float64), bits
    f = np.ascontiguousarray(x, np.float32)
    return f.astype(np.float64), f


def read(buf, shape, dtype):
    n = int(np.prod(shape))
    if dtype == T.TTL_DTYPE_BF16:
        return R.from_bf16(buf.download(np.uint16, n)).reshape(shape).astype(np.float64)
    return buf.download(np.float32, n).reshape(shape).astype(np.float64)


F32, BF16 = T.TTL_DTYPE_F32, T.TTL_DTYPE_BF16


# ---- the store and the read-back ---------------------------------------------------------------


def run_store(dev, held, pool, table, lengths, news, heads, x, xd, qd, bias, rope, tiled=False, pad=0, starts=True,
              max_length=None, rope_positions=None):
    """Returns q, the pool's bytes after the call, and the pool buffer."""
    tokens = int(sum(news)) + pad
    pb = held.up(pool.bytes)
    cache = T.kv4_cache(pb, pool.pages, pool.kv_heads, pool.hd, pool.page)
    batch = T.kv4_batch(len(lengths), tokens, held.up(table), table.shape[1], held.up(np.asarray(lengths, np.int32)),
                        held.up(cumulative(news)) if starts else None, max_length, pool.page)
    q = held.new(tokens * heads * pool.hd * 4, 0x5a)
    dev.qkv_rope_store_kv4(cache, batch, heads, held.up(x), xd, held.up(bias) if bias is not None else None,
                           held.up(rope), rope_positions or len(rope), q, qd, tiled)
    after = pb.download(np.uint8).reshape(pool.bytes.shape)
    return read(q, (tokens, heads, pool.hd), qd), after, pb, cache, batch


@pytest.mark.parametrize("heads,kv_heads,hd,page,xd,qd,tiled", [
    (64, 8, 64, 64, F32, F32, True), (64, 8, 64, 16, F32, BF16, False), (64, 8, 64, 128, BF16, BF16, True),
    (20, 4, 128, 32, F32, F32, False), (3, 3, 64, 256, BF16, F32, False), (8, 1, 128, 16, F32, BF16, False),
    (33, 11, 64, 16, F32, F32, False)])
@pytest.mark.parametrize("with_bias", [True, False])
def test_store(dev, held, heads, kv_heads, hd, page, xd, qd, tiled, with_bias):
    rng = np.random.default_rng(heads * 1000 + hd + page)
    lengths, news, pad = [70, 1, 0, 33, 300], [5, 1, 0, 33, 40], 3
    pool = R.Pool(40, kv_heads, hd, page, seed=1)
    table = R.tables(rng, lengths, page, 40)
    width = (heads + 2 * kv_heads) * hd
    tokens = sum(news) + pad
    x64, x = to_dtype(rng.standard_normal((tokens, width)), xd)
    bias = rng.standard_normal(width).astype(np.float32) if with_bias else None
    rope = rope_table(300, hd, rng)
    logical = x64
    if tiled:   # columns of x are ttl_qkv_row_source's
        src = np.empty(5120, np.int32)
        T._check(dev.lib.ttl_qkv_row_source(src.ctypes.data), "ttl_qkv_row_source")
        logical = np.empty_like(x64)
        logical[:, src] = x64
    q, after, pb, cache, batch = run_store(dev, held, pool, table, lengths, news, heads, x, xd, qd, bias, rope, tiled,
                                           pad)
    at = np.concatenate([np.arange(n - m, n) for n, m in zip(lengths, news)])
    seq = np.repeat(np.arange(5), news)
    qr, kr, vr = R.rotate(logical[:len(at)], bias, rope, at, heads, kv_heads, hd)
    for i in range(len(at)):
        pool.put(table[seq[i]], at[i], kr[i], vr[i])
    assert np.array_equal(after, pool.bytes)            # what was stored, and nothing else touched
    # one rounding: half a step of the type, and 2^-50 of the two products' magnitudes
    half = 2.0 ** -8 if qd == BF16 else 2.0 ** -24
    assert (np.abs(q[:len(at)] - qr) <= half * np.abs(qr) + 2.0 ** -45).all()
    fill = R.from_bf16(np.uint16([0x5a5a])) if qd == BF16 else np.uint32([0x5a5a5a5a]).view(np.float32)
    assert (q[len(at):] == float(fill[0])).all()        # padding rows left as they were
    # the values back, bit for bit
    k, v = held.new(tokens * kv_heads * hd * 4, 0x5a), held.new(tokens * kv_heads * hd * 4, 0x5a)
    dev.kv4_dequantize(cache, batch, k, v)
    kg, vg = (read(b, (tokens, kv_heads, hd), F32) for b in (k, v))
    for i in range(len(at)):
        kk, vv = pool.get(table[seq[i]], np.array([at[i]]))
        assert np.array_equal(kg[i], kk[0]) and np.array_equal(vg[i], vv[0])
    pat = float(np.uint32([0x5a5a5a5a]).view(np.float32)[0])
    assert (kg[len(at):] == pat).all() and (vg[len(at):] == pat).all()


def test_store_block_edges(dev, held):
    """Zeros, ties, the border between two exponents, the smallest and largest values, and
    values that are not finite, in keys (at position 0 with cos 1, sin 0) and values."""
    hd, kv = 64, 2
    rows = []
    base = np.zeros(64)
    for unit in (0, -60, 100, -124):
        b = base.copy()
        b[:12] = np.array([6, 5, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -0.25, 5.0000005, 0.7499999, -6.5]) * 2.0 ** unit
        b[32:40] = np.array([6.9999995, -7 / 2, 3.5, 1, 0.5, 0.25, -0.125, 0]) * 2.0 ** unit
        rows.append(b)
        rows.append(np.concatenate([np.full(32, 7.0 * 2.0 ** unit), -np.full(32, 5.0 * 2.0 ** unit)]))
    rows += [base, -base, np.full(64, 1e-45), np.full(64, 3e-39), np.full(64, 3.4028e38), np.full(64, -1.7e38),
             np.linspace(-3e38, 3e38, 64)]
    for bad in (np.inf, -np.inf, np.nan):
        b = np.linspace(-1, 1, 64)
        b[40] = bad
        rows.append(b)
    rows = np.array(rows).astype(np.float32)
    n = len(rows)
    x = np.zeros((n, 3 * hd * kv), np.float32).reshape(n, 3 * kv, hd)
    x[:, kv:2 * kv] = rows[:, None]
    x[:, 2 * kv:] = rows[::-1][:, None]
    rope = np.zeros((1, hd // 2, 2), np.float32)
    rope[..., 0] = 1.0
    pool = R.Pool(n, kv, hd, 16, seed=2)
    table = np.arange(n, dtype=np.int32)[:, None]      # a sequence a row, all at position 0
    q, after, *_ = run_store(dev, held, pool, table, [1] * n, [1] * n, kv, x.reshape(n, -1), F32, F32, None, rope,
                             starts=False)
    for i in range(n):
        with np.errstate(invalid="ignore"):
            lo, hi = rows[i, :32].astype(np.float64), rows[i, 32:].astype(np.float64)
            k = np.concatenate([lo - hi * 0.0, lo * 0.0 + hi])
        pool.put(table[i], 0, np.tile(k, (kv, 1)), np.tile(rows[n - 1 - i].astype(np.float64), (kv, 1)))
    assert np.array_equal(after, pool.bytes)


def test_store_overflow_of_the_rotation_is_a_nan_block(dev, held):
    """Finite inputs whose rotated value is no finite f32."""
    x = np.full((1, 3 * 64), 3e38, np.float32)
    rope = np.full((1, 32, 2), 1.3, np.float32)
    pool = R.Pool(1, 1, 64, 16, seed=3)
    q, after, *_ = run_store(dev, held, pool, np.zeros((1, 1), np.int32), [1], [1], 1, x, F32, F32, None, rope,
                             starts=False)
    _, k, v = R.rotate(x.astype(np.float64), None, rope, np.array([0]), 1, 1, 64)
    pool.put(np.zeros(1, np.int32), 0, k[0], v[0])
    assert np.array_equal(after, pool.bytes)
    assert pool.ks[0, 0, 0].tolist() == [127, 255]       # lo: 3e38 x 1.3 - 3e38 x 1.3 = 0
    assert np.isinf(q[0, 0, 32:]).all() and (q[0, 0, :32] == 0).all()


def test_store_rows_without_a_place(dev, held):
    """A page outside the pool, a sequence longer than max_length, a position past the
    rotation table, an idle slot, more rows than positions: nothing else is touched."""
    rng = np.random.default_rng(5)
    pool = R.Pool(6, 2, 64, 16, seed=4)
    lengths = [20, 20, 40, 33, 0, 3, 5]
    news = [2, 2, 2, 2, 1, 5, 1]
    table = np.full((7, 3), -1, np.int32)
    table[0, 1] = 6                     # one past the last page
    table[1, 1] = -1
    table[2] = [0, 1, 2]                # longer than max_length = 38
    table[3] = [0, 1, 2]                # positions 31 and 32: 32 is past the table of 32
    table[5, 0], table[6, 0] = 3, 4
    x = rng.standard_normal((sum(news), 6 * 64)).astype(np.float32)
    rope = rope_table(32, 64, rng)
    q, after, pb, cache, batch = run_store(dev, held, pool, table, lengths, news, 2, x, F32, F32, None, rope,
                                           max_length=38)
    at = cumulative(news)
    put = [(3, 31, at[3]), (5, 0, at[5] + 2), (5, 1, at[5] + 3), (5, 2, at[5] + 4), (6, 4, at[6])]
    fine = np.zeros(sum(news), bool)
    for s, p, i in put:
        qr, kr, vr = R.rotate(x[i:i + 1], None, rope, np.array([p]), 2, 2, 64)
        pool.put(table[s], p, kr[0], vr[0])
        assert (np.abs(q[i] - qr[0]) <= 2.0 ** -24 * np.abs(qr[0]) + 2.0 ** -45).all()
        fine[i] = True
    idle = np.zeros(sum(news), bool)
    idle[[at[4], at[5], at[5] + 1]] = True
    assert np.array_equal(after, pool.bytes)
    assert (q[idle] == 0).all() and np.isnan(q[~fine & ~idle]).all()
    k = held.new(sum(news) * 2 * 64 * 4)
    dev.kv4_dequantize(cache, batch, k, None)
    kg = read(k, (sum(news), 2, 64), F32)
    held_rows = fine.copy()
    held_rows[at[3] + 1] = True        # position 32 has a place in the cache; only its rotation was missing
    assert np.isfinite(kg[held_rows & fine]).all() and (kg[idle] == 0).all() and np.isnan(kg[~held_rows & ~idle]).all()


# ---- attention --------------------------------------------------------------------------------------


def run_attention(dev, held, pb, pool, table, lengths, news, q, heads, dtype, window, scale, sinks, pad=0,
                  max_length=None, starts=None):
    """news None: decode."""
    tokens = len(q)
    cache = T.kv4_cache(pb, pool.pages, pool.kv_heads, pool.hd, pool.page)
    st = cumulative(news) if news is not None else None
    batch = T.kv4_batch(len(lengths), tokens, held.up(table), table.shape[1], held.up(np.asarray(lengths, np.int32)),
                        held.up(st) if news is not None else None, max_length, pool.page)
    att = T.kv4_attention(heads, dtype, window, scale, held.up(sinks) if sinks is not None else None)
    need = dev.attention_kv4_workspace_bytes(cache, batch, att)
    ws = held.new(need, 0xff) if need else None
    out = held.new(tokens * heads * pool.hd * 4, 0x5a)
    f = dev.attention_decode_kv4 if news is None else dev.attention_prefill_kv4
    f(cache, batch, att, held.up(q), out, ws, need)
    return read(out, (tokens, heads, pool.hd), dtype)


def check_attention(got, q, pool, table, lengths, news, heads, dtype, window, scale, sinks):
    row, err2, ref2 = 0, 0.0, 0.0
    for s, (n, m) in enumerate(zip(lengths, news)):
        if m == 0:
            continue
        if n <= 0:
            assert (got[row:row + m] == 0).all(), s
            row += m
            continue
        first = max(0, n - m + 1 - window) if window else 0
        pos = np.arange(first, n)
        k, v = pool.get(table[s], pos)
        at = np.arange(n - m, n)
        ref, mag, smax, vsum = R.attention(q[row:row + m], k, v, at, first, window, scale, sinks)
        tol = R.allowance(ref, mag, smax, vsum, len(pos), pool.hd, dtype == BF16)
        off = np.abs(got[row:row + m] - ref)
        assert np.isfinite(got[row:row + m]).all(), (s, n, m)
        assert (off <= tol).all(), (s, n, m, float((off / np.maximum(tol, 1e-300)).max()))
        err2 += (off ** 2).sum()
        ref2 += (ref ** 2).sum()
        row += m
    if ref2:
        assert np.sqrt(err2 / ref2) <= (2.0 ** -8 if dtype == BF16 else 1e-5)


SHAPES = [(64, 8, 64, 64), (64, 8, 64, 16), (20, 4, 128, 32), (6, 2, 64, 256), (5, 5, 128, 16), (32, 1, 64, 128),
          (40, 2, 64, 64)]


@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [0, 1, 100, 128])
def test_decode(dev, held, heads, kv_heads, hd, page, dtype, window):
    rng = np.random.default_rng(heads + hd + window)
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 0, 127, 129, 200, 257, 700]
    pages = sum(-(-n // page) for n in lengths) + 2
    pool = R.Pool(pages, kv_heads, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, pages)
    q, qb = to_dtype(rng.standard_normal((len(lengths), heads, hd)) * 1.5, dtype)
    sinks = None if window == 100 else rng.standard_normal(heads).astype(np.float32)
    scale = float(np.float32(hd ** -0.5))
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, None, qb, heads, dtype, window, scale,
                        sinks)
    check_attention(got, q, pool, table, lengths, [1] * len(lengths), heads, dtype, window, scale, sinks)


@pytest.mark.parametrize("length,dtype,window", [(5000, F32, 0), (5000, BF16, 0), (20011, BF16, 0), (20011, F32, 0),
                                                 (20011, F32, 3000)])
def test_decode_long(dev, held, length, dtype, window):
    rng = np.random.default_rng(length)
    heads, kv = 16, 2
    lengths = [length, 1, length // 3]
    pages = sum(-(-n // 64) for n in lengths)
    pool = R.Pool(pages, kv, 64, 64).randomise(rng)
    table = R.tables(rng, lengths, 64, pages)
    q, qb = to_dtype(rng.standard_normal((3, heads, 64)) * 2, dtype)
    sinks = rng.standard_normal(heads).astype(np.float32)
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, None, qb, heads, dtype, window, 0.125,
                        sinks)
    check_attention(got, q, pool, table, lengths, [1] * 3, heads, dtype, window, 0.125, sinks)


@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [0, 33, 128])
def test_prefill(dev, held, heads, kv_heads, hd, page, dtype, window):
    rng = np.random.default_rng(heads + hd + window + 7)
    lengths = [1, 40, 0, 64, 200, 3, 131, 17, 300]
    news = [1, 40, 2, 17, 3, 0, 130, 16, 1]
    pages = sum(-(-n // page) for n in lengths) + 2
    pool = R.Pool(pages, kv_heads, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, pages)
    pad = 5
    q, qb = to_dtype(rng.standard_normal((sum(news) + pad, heads, hd)) * 1.5, dtype)
    sinks = None if window == 33 else rng.standard_normal(heads).astype(np.float32)
    scale = float(np.float32(hd ** -0.5))
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, window, scale,
                        sinks)
    check_attention(got, q, pool, table, lengths, news, heads, dtype, window, scale, sinks)
    fill = R.from_bf16(np.uint16([0x5a5a])) if dtype == BF16 else np.uint32([0x5a5a5a5a]).view(np.float32)
    assert (got[sum(news):] == float(fill[0])).all()


@pytest.mark.parametrize("new,length,dtype", [(5, 6000, BF16), (2, 6000, F32), (700, 1500, BF16), (300, 900, F32)])
def test_prefill_long(dev, held, new, length, dtype):
    rng = np.random.default_rng(new)
    heads, kv = 16, 2
    lengths, news = [length, 50, length // 2], [new, 50, max(1, new // 3)]
    pages = sum(-(-n // 64) for n in lengths)
    pool = R.Pool(pages, kv, 64, 64).randomise(rng)
    table = R.tables(rng, lengths, 64, pages)
    q, qb = to_dtype(rng.standard_normal((sum(news), heads, 64)) * 2, dtype)
    sinks = rng.standard_normal(heads).astype(np.float32)
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, 0, 0.125, sinks)
    check_attention(got, q, pool, table, lengths, news, heads, dtype, 0, 0.125, sinks)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("prefill", [False, True])
def test_masked_positions_have_no_influence(dev, held, dtype, prefill):
    """Positions behind the length and before the window hold NaN blocks or the largest
    values, and pages before the window are given back: the same bits as with zeros there."""
    rng = np.random.default_rng(11)
    heads, kv, hd, page, window = 16, 2, 64, 16, 50
    lengths = [150, 67, 30, 129]
    news = [9, 3, 30, 2] if prefill else None
    pages = sum(-(-n // page) for n in lengths)
    clean = R.Pool(pages, kv, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, pages)
    rows = []
    for fill in ("zero", "nan", "huge"):
        pool = R.Pool(pages, kv, hd, page)
        pool.bytes[...] = clean.bytes
        for s, n in enumerate(lengths):
            m = news[s] if prefill else 1
            lo = max(0, n - m + 1 - window)
            for p in list(range(lo)) + list(range(n, -(-n // page) * page)):
                g, i = table[s, p // page], p % page
                for c, b in ((pool.kc, pool.ks), (pool.vc, pool.vs)):
                    c[g, :, i] = 0 if fill == "zero" else 0x77
                    b[g, :, i] = {"zero": 0, "nan": 255, "huge": 252}[fill]
        t = table.copy()
        for s, n in enumerate(lengths):
            m = news[s] if prefill else 1
            t[s, :max(0, n - m + 1 - window) // page] = -1     # pages given back before the window
        q, qb = to_dtype(np.random.default_rng(3).standard_normal((sum(news) if prefill else 4, heads, hd)), dtype)
        sinks = np.zeros(heads, np.float32)
        rows.append(run_attention(dev, held, held.up(pool.bytes), pool, t, lengths, news, qb, heads, dtype, window,
                                  0.125, sinks))
    check_attention(rows[0], q, clean, table, lengths, news or [1] * 4, heads, dtype, window, 0.125, sinks)
    assert np.array_equal(rows[0], rows[1]) and np.array_equal(rows[0], rows[2])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("what", ["k", "v", "v_block1"])
def test_nan_blocks_reach_those_who_see_them(dev, held, dtype, what):
    """A NaN block of one position of one head: with it in K the rows that see it are NaN,
    in V those rows' dims of the block; every other output keeps its value."""
    rng = np.random.default_rng(12)
    heads, kv, hd, page, window = 8, 2, 64, 16, 40
    lengths, news = [100, 60], [60, 60]
    pool = R.Pool(12, kv, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, 12)
    at = 55                                         # of both sequences; kv head 1
    blocks = {"k": [0], "v": [0, 1], "v_block1": [1]}[what]
    q, qb = to_dtype(rng.standard_normal((120, heads, hd)), dtype)
    before = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, window, 0.125,
                           None)
    check_attention(before, q, pool, table, lengths, news, heads, dtype, window, 0.125, None)
    for s in range(2):
        (pool.ks if what == "k" else pool.vs)[table[s, at // page], 1, at % page, blocks] = 255
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, window, 0.125,
                        None)
    expect = np.zeros(got.shape, bool)
    for s in range(2):
        pos = np.arange(lengths[s] - news[s], lengths[s])
        see = np.nonzero((pos >= at) & (pos < at + window))[0] + 60 * s
        for blk in (range(2) if what == "k" else blocks):
            expect[see[:, None], np.arange(heads // 2, heads)[None], 32 * blk:32 * blk + 32] = True
    assert np.array_equal(np.isnan(got), expect)
    check = np.where(expect, 0.0, got - before)
    mag = np.abs(before) + 1.0
    assert (np.abs(check) <= (2.0 ** -8 if dtype == BF16 else 1e-5) * mag).all()
    # one token a sequence
    dec = run_attention(dev, held, held.up(pool.bytes), pool, table, [at + 1, at + 2], None,
                        qb[:2], heads, dtype, window, 0.125, None)
    assert np.isnan(dec[:, heads // 2:, 32:] if what != "k" else dec[:, heads // 2:]).all()
    assert np.isfinite(dec[:, :heads // 2]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("prefill", [False, True])
def test_values_of_any_magnitude(dev, held, dtype, prefill):
    """Values from 2^-100 to 2^100, by position, by dim, and next to each other; a later
    token's huge value does not touch an earlier one's output."""
    rng = np.random.default_rng(13)
    heads, kv, hd, page = 8, 2, 64, 32
    lengths = [90, 90, 90, 90]
    news = [64] * 4 if prefill else None
    pool = R.Pool(16, kv, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, 16)
    scale_of = [lambda p: 2.0 ** -100, lambda p: 2.0 ** 100, lambda p: 2.0 ** (100 if p == 70 else 0),
                lambda p: 2.0 ** rng.integers(-60, 20)]
    for s in range(4):
        for p in range(90):
            k, v = pool.get(table[s], np.array([p]))
            pool.put(table[s], p, k[0], v[0] * scale_of[s](p))
    n = 256 if prefill else 4
    q, qb = to_dtype(rng.standard_normal((n, heads, hd)), dtype)
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, 0, 0.125, None)
    check_attention(got, q, pool, table, lengths, news or [1] * 4, heads, dtype, 0, 0.125, None)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scores_and_sinks_of_any_size(dev, held, dtype):
    """Scores of hundreds, a negative scale, zero queries, sinks far above and below the
    scores, infinite sinks."""
    rng = np.random.default_rng(14)
    heads, kv, hd = 16, 2, 64
    lengths, news = [130, 40], [3, 40]
    pool = R.Pool(6, kv, hd, 64).randomise(rng)
    table = R.tables(rng, lengths, 64, 6)
    q, qb = to_dtype(rng.standard_normal((43, heads, hd)) * np.array([30.0, 0.0, 1e-20, 1.0] * 4)[None, :, None], dtype)
    for sinks in (np.linspace(-300, 300, heads).astype(np.float32), np.full(heads, -1e30, np.float32),
                  np.full(heads, -np.inf, np.float32)):
        for scale in (0.125, -0.125, 0.0):
            got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, 0, scale,
                                sinks)
            check_attention(got, q, pool, table, lengths, news, heads, dtype, 0, scale, sinks)
    high = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, 0, 0.125,
                         np.full(heads, 1e30, np.float32))
    assert (high == 0).all()                        # the sink takes everything


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_queries_that_are_not_finite(dev, held, dtype, bad):
    rng = np.random.default_rng(15)
    heads, kv, hd = 8, 2, 64
    lengths, news = [130, 40], [3, 40]
    pool = R.Pool(6, kv, hd, 64).randomise(rng)
    table = R.tables(rng, lengths, 64, 6)
    q = rng.standard_normal((43, heads, hd))
    q[1, 2, 5] = q[20, 7, 63] = bad
    for m, l in ((news, lengths), (None, [130] * 1 + [40] * 42)):
        t = table if m else table[[0] + [1] * 42]
        qv, qb = to_dtype(q, dtype)
        got = run_attention(dev, held, held.up(pool.bytes), pool, t, l, m, qb, heads, dtype, 0, 0.125, None)
        nan = np.zeros((43, heads), bool)
        nan[1, 2] = nan[20, 7] = True
        assert np.array_equal(np.isnan(got).all(-1), nan) and np.array_equal(np.isnan(got).any(-1), nan)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_rows_without_a_place(dev, held, dtype):
    """Too long a sequence, pages outside the pool (where the row sees them), idle slots."""
    rng = np.random.default_rng(16)
    heads, kv, hd, page = 8, 2, 64, 16
    pool = R.Pool(9, kv, hd, page).randomise(rng)
    pb = held.up(pool.bytes)
    lengths = [20, 41, 20, 20, 0, -3]
    table = np.tile(np.arange(3, dtype=np.int32), (6, 1))
    table[2, 0], table[3, 1] = 9, -5
    q, qb = to_dtype(rng.standard_normal((6, heads, hd)), dtype)
    got = run_attention(dev, held, pb, pool, table, lengths, None, qb, heads, dtype, 0, 0.125, None, max_length=40)
    check_attention(got[:1], q[:1], pool, table[:1], lengths[:1], [1], heads, dtype, 0, 0.125, None)
    assert np.isnan(got[1:4]).all() and (got[4:] == 0).all()
    # within a window of 4 sequence 2's bad first page is not seen
    got = run_attention(dev, held, pb, pool, table, lengths, None, qb, heads, dtype, 4, 0.125, None, max_length=40)
    assert np.isfinite(got[2]).all() and np.isnan(got[[1, 3]]).all()
    # the same by runs of tokens: rows before position 0 are idle, a row of the long sequence NaN
    lengths, news = [20, 41, 20, 2], [4, 3, 20, 5]
    q, qb = to_dtype(rng.standard_normal((32, heads, hd)), dtype)
    table = np.tile(np.arange(3, dtype=np.int32), (4, 1))
    table[2, 1] = 1 << 30
    got = run_attention(dev, held, pb, pool, table, lengths, news, qb, heads, dtype, 0, 0.125, None, max_length=40)
    assert np.isfinite(got[:4]).all() and np.isnan(got[4:7]).all()
    assert np.isfinite(got[7:23]).all() and np.isnan(got[23:27]).all()   # positions 16.. need the bad page
    assert (got[27:30] == 0).all() and np.isfinite(got[30:]).all() and (got[30:] != 0).any()


def test_pages_past_four_gigabytes(dev, held):
    """A pool of 5 GB: the pages used lie at its start and at its end."""
    heads, kv, hd, page = 8, 8, 64, 256
    record = kv * page * 68
    pages = 5 * (1 << 30) // record
    small = R.Pool(4, kv, hd, page)
    rng = np.random.default_rng(17)
    pb = held.new(pages * record)
    where = np.array([pages - 1, 0, pages - 2, pages // 2], np.int32)
    rope = rope_table(600, hd, rng)
    lengths, news = [600, 10], [600, 10]
    table = np.array([[where[0], where[1], where[2]], [where[3], -1, -1]], np.int32)
    here = np.array([[0, 1, 2], [3, -1, -1]], np.int32)
    x = rng.standard_normal((610, (heads + 2 * kv) * hd)).astype(np.float32)
    cache = T.kv4_cache(pb, pages, kv, hd, page)
    batch = T.kv4_batch(2, 610, held.up(table), 3, held.up(np.int32(lengths)), held.up(cumulative(news)), 768, page)
    q = held.new(610 * heads * hd * 4)
    dev.qkv_rope_store_kv4(cache, batch, heads, held.up(x), F32, None, held.up(rope), 600, q, F32)
    at = np.concatenate([np.arange(600), np.arange(10)])
    qr, kr, vr = R.rotate(x, None, rope, at, heads, kv, hd)
    for i in range(610):
        small.put(here[0 if i < 600 else 1], at[i], kr[i], vr[i])
    k, v = held.new(610 * kv * hd * 4), held.new(610 * kv * hd * 4)
    dev.kv4_dequantize(cache, batch, k, v)
    for b, pick in ((k, 0), (v, 1)):
        want = np.concatenate([small.get(here[s], np.arange(n))[pick] for s, n in enumerate(lengths)])
        assert np.array_equal(read(b, (610, kv, hd), F32), want)
    qv = read(q, (610, heads, hd), F32)
    att = T.kv4_attention(heads, F32, 0, 0.125, None)
    need = dev.attention_kv4_workspace_bytes(cache, batch, att)
    out = held.new(610 * heads * hd * 4)
    dev.attention_prefill_kv4(cache, batch, att, q, out, held.new(need) if need else None, need)
    check_attention(read(out, (610, heads, hd), F32), qv, small, here, lengths, news, heads, F32, 0, 0.125, None)
    last = T.kv4_batch(2, 2, batch.page_table, 3, batch.lengths, None, 768, page)
    q2 = held.up(qv[[599, 609]].astype(np.float32))
    need = dev.attention_kv4_workspace_bytes(cache, last, att)
    out = held.new(2 * heads * hd * 4)
    dev.attention_decode_kv4(cache, last, att, q2, out, held.new(need) if need else None, need)
    check_attention(read(out, (2, heads, hd), F32), qv[[599, 609]], small, here, lengths, [1, 1], heads, F32, 0, 0.125,
                    None)


# ---- together, as they are used -----------------------------------------------------------------------


def test_serving_run(dev, held):
    """Two ragged prompts, then decode steps, from the framework's own Q/K/V product on: the
    paged cache's outputs against the dense f32 path of the same values (the cache read back
    into a dense cache, ttl_attention_prefill / ttl_attention_decode), sliding and full."""
    rng = np.random.default_rng(20)
    news, steps, page = [77, 130], 3, 32
    capacity = 192
    blocks = O.synth_q8_0(0x77000003, 5, 5120 * 90)
    src = np.empty(5120, np.int32)
    T._check(dev.lib.ttl_qkv_row_source(src.ctypes.data), "ttl_qkv_row_source")
    w = dev.q8_upload(blocks, 5120, 2880, src, 5120)
    bias = held.up(rng.standard_normal(5120).astype(np.float32))
    rope = held.up(rope_table(capacity, 64, rng))
    sinks_h = rng.standard_normal(64).astype(np.float32)
    sinks = held.up(sinks_h)
    pool = R.Pool(14, 8, 64, page, fill=0xff)
    pb = held.up(pool.bytes)
    cache = T.kv4_cache(pb, 14, 8, 64, page)
    table = R.tables(rng, [n + steps for n in news], page, 14)
    tb = held.up(table)
    lengths = np.array(news, np.int32)
    lb = held.up(lengths)

    def project(tokens):
        x = held.up(rng.standard_normal((tokens, 2880)).astype(np.float32))
        qkv = held.new(tokens * 5120 * 4)
        dev.matmul_q8_0(w, None, x, tokens, None, qkv)
        return qkv

    def dense(s, n):
        """Sequence s's first n positions as a dense f32 cache."""
        one = T.kv4_batch(1, n, held.up(table[s:s + 1]), table.shape[1], held.up(np.int32([n])),
                          held.up(np.int32([0, n])), None, page)
        k, v = held.new(capacity * 512 * 4, 0), held.new(capacity * 512 * 4, 0)
        dev.kv4_dequantize(cache, one, k, v)
        return k, v

    # the prompts
    total = sum(news)
    starts = cumulative(news)
    batch = T.kv4_batch(2, total, tb, table.shape[1], lb, held.up(starts), None, page)
    q = held.new(total * 4096 * 4)
    dev.qkv_rope_store_kv4(cache, batch, 64, project(total), F32, bias, rope, capacity, q, F32, tiled=True)
    for layer, window in ((0, 128), (1, 0)):
        att = T.kv4_attention(64, F32, window, 0.125, sinks)
        need = dev.attention_kv4_workspace_bytes(cache, batch, att)
        out = held.new(total * 4096 * 4)
        dev.attention_prefill_kv4(cache, batch, att, q, out, held.new(need) if need else None, need)
        got = out.download(np.float32, total * 4096).reshape(total, 4096)
        for s in range(2):
            k, v = dense(s, news[s])
            o = held.new(news[s] * 4096 * 4)
            qs = held.up(q.download(np.float32, total * 4096).reshape(total, 4096)[starts[s]:starts[s + 1]])
            dev.attention_prefill(qs, k, v, sinks, 0, news[s], capacity, layer, o)
            ref = o.download(np.float32, news[s] * 4096).reshape(news[s], 4096)
            assert O.rel_l2(got[starts[s]:starts[s + 1]], ref) <= 1e-5
    # decode steps
    for step in range(steps):
        lengths += 1
        lb.upload(lengths)
        batch = T.kv4_batch(2, 2, tb, table.shape[1], lb, None, None, page)
        q = held.new(2 * 4096 * 4)
        dev.qkv_rope_store_kv4(cache, batch, 64, project(2), F32, bias, rope, capacity, q, F32, tiled=True)
        for layer, window in ((0, 128), (1, 0)):
            att = T.kv4_attention(64, F32, window, 0.125, sinks)
            need = dev.attention_kv4_workspace_bytes(cache, batch, att)
            out = held.new(2 * 4096 * 4)
            dev.attention_decode_kv4(cache, batch, att, q, out, held.new(need) if need else None, need)
            got = out.download(np.float32, 2 * 4096).reshape(2, 4096)
            for s in range(2):
                k, v = dense(s, int(lengths[s]))
                ws = held.new(dev.lib.ttl_attention_workspace_bytes(capacity))
                o = held.new(4096 * 4)
                qs = held.up(q.download(np.float32, 2 * 4096)[4096 * s:4096 * (s + 1)])
                dev.attention_decode(qs, k, v, sinks, held.up(np.int32([lengths[s] - 1])), capacity, layer, ws, o)
                assert O.rel_l2(got[s], o.download(np.float32, 4096)) <= 1e-5
    w.free()


def test_captured_steps(dev, held):
    """A store and an attention captured once and replayed as the lengths grow, with eager
    work between the replays: every replay equals the eager calls."""
    rng = np.random.default_rng(21)
    heads, kv, hd, page, seqs = 64, 8, 64, 64, 3
    start = np.array([700, 63, 0], np.int32)
    stride = 20
    table = rng.permutation(64)[:seqs * stride].reshape(seqs, stride).astype(np.int32)
    pool = R.Pool(64, kv, hd, page).randomise(rng)
    pools = [held.up(pool.bytes), held.up(pool.bytes)]
    lb, tb = held.up(start), held.up(table)
    rope = held.up(rope_table(1280, hd, rng))
    xb = held.new(seqs * 5120 * 4)
    sinks = held.up(rng.standard_normal(heads).astype(np.float32))
    outs, calls = [], []
    for p in pools:
        cache = T.kv4_cache(p, 64, kv, hd, page)
        batch = T.kv4_batch(seqs, seqs, tb, stride, lb, None, None, page)
        q, out = held.new(seqs * 4096 * 4), held.new(seqs * 4096 * 4)
        atts = [T.kv4_attention(heads, F32, w, 0.125, sinks) for w in (0, 128)]
        need = max(dev.attention_kv4_workspace_bytes(cache, batch, a) for a in atts)
        ws = held.new(need, 0xff)
        outs.append((out, held.new(seqs * 4096 * 4)))

        def call(cache=cache, batch=batch, q=q, o=outs[-1], atts=atts, ws=ws, need=need):
            dev.qkv_rope_store_kv4(cache, batch, heads, xb, F32, None, rope, 1280, q, F32)
            for a, dst in zip(atts, o):
                dev.attention_decode_kv4(cache, batch, a, q, dst, ws, need)

        calls.append(call)
    graph = dev.capture(calls[1])
    for step in range(6):
        lb.upload(start + (1 + step) * np.array([1, 1, 0 if step < 3 else 1], np.int32))
        xb.upload(rng.standard_normal((seqs, 5120)).astype(np.float32))
        calls[0]()
        dev.sync()
        graph.launch()
        for a, b in zip(*outs):
            assert np.array_equal(a.download(np.float32, seqs * 4096).view(np.uint32),
                                  b.download(np.float32, seqs * 4096).view(np.uint32)), step
        assert np.array_equal(pools[0].download(np.uint8), pools[1].download(np.uint8))
    graph.free()


def test_two_contexts_at_once(dev, held):
    """Calls of two contexts (two streams) that overlap, each with its own workspace."""
    rng = np.random.default_rng(22)
    heads, kv, hd, page = 16, 2, 64, 64
    lengths = [9000, 3000]
    pages = sum(-(-n // page) for n in lengths)
    pool = R.Pool(pages, kv, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, pages)
    pb = held.up(pool.bytes)
    other = T.Device(0)
    try:
        work = []
        for d in (dev, other):
            q = rng.standard_normal((2, heads, hd)).astype(np.float32)
            cache = T.kv4_cache(pb, pages, kv, hd, page)
            batch = T.kv4_batch(2, 2, held.up(table), table.shape[1], held.up(np.int32(lengths)), None, 9000, page)
            att = T.kv4_attention(heads, F32, 0, 0.125, None)
            need = d.attention_kv4_workspace_bytes(cache, batch, att)
            work.append((d, cache, batch, att, q, held.up(q), held.new(2 * heads * hd * 4), held.new(need), need))
        dev.sync()
        for _ in range(20):
            for d, cache, batch, att, _, q, out, ws, need in work:
                d.attention_decode_kv4(cache, batch, att, q, out, ws, need)
        for d, cache, batch, att, qh, q, out, ws, need in work:
            d.sync()
            check_attention(read(out, (2, heads, hd), F32), qh.astype(np.float64), pool, table, lengths, [1, 1], heads,
                            F32, 0, 0.125, None)
    finally:
        other.close()


@pytest.mark.parametrize("prefill", [False, True])
def test_results_repeat(dev, held, prefill):
    """The same call twice gives the same bits, whatever the workspace held."""
    rng = np.random.default_rng(23)
    lengths = [5000, 100]
    pool = R.Pool(90, 8, 64, 64).randomise(rng)
    table = R.tables(rng, lengths, 64, 90)
    pb = held.up(pool.bytes)
    news = [6, 6] if prefill else None
    q = rng.standard_normal((12 if prefill else 2, 64, 64)).astype(np.float32)
    a, b = (run_attention(dev, held, pb, pool, table, lengths, news, q, 64, F32, 0, 0.125, None) for _ in range(2))
    assert np.array_equal(a, b)


# ---- the ways a call is cut -------------------------------------------------------------------------
#
# By the queries that a sequence has on average for a key/value head: 8 and fewer, 16, 32, more;
# blocks divided among workgroups or taken whole; outputs joined by 4 waves, one, or part of one.


@pytest.mark.parametrize("heads,kv_heads,hd,page,news", [
    (16, 2, 64, 16, [1, 1, 1, 0, 1]), (16, 2, 64, 64, [1, 3, 2, 0, 1]), (16, 2, 64, 16, [3, 1, 6, 2, 4]),
    (16, 2, 64, 64, [7, 1, 9, 0, 8]), (20, 4, 128, 32, [1, 1, 2, 0, 1]), (20, 4, 128, 128, [2, 1, 4, 1, 3]),
    (20, 4, 128, 16, [6, 1, 9, 2, 5]), (20, 4, 128, 64, [21, 1, 30, 0, 14])])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [0, 100])
def test_prefill_few_tokens(dev, held, heads, kv_heads, hd, page, news, dtype, window):
    rng = np.random.default_rng(sum(news) + window)
    lengths = [6000, 1, 130, 0, 2501]
    pages = sum(-(-n // page) for n in lengths) + 1
    pool = R.Pool(pages, kv_heads, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, pages)
    q, qb = to_dtype(rng.standard_normal((sum(news) + 3, heads, hd)) * 1.5, dtype)
    sinks = rng.standard_normal(heads).astype(np.float32)
    scale = float(np.float32(hd ** -0.5))
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, window, scale,
                        sinks)
    check_attention(got, q, pool, table, lengths, news, heads, dtype, window, scale, sinks)
    fill = R.from_bf16(np.uint16([0x5a5a])) if dtype == BF16 else np.uint32([0x5a5a5a5a]).view(np.float32)
    assert (got[sum(news):] == float(fill[0])).all()


@pytest.mark.parametrize("group,kv_heads,news_to", [(8, 1, 0), (20, 1, 0), (4, 2, 2), (8, 1, 5), (8, 2, 24)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_sequences(dev, held, group, kv_heads, news_to, dtype):
    """More blocks than a workgroup has threads, of very different lengths, some without rows."""
    rng = np.random.default_rng(31 + group + news_to)
    count, heads, page = 700, group * kv_heads, 16
    lengths = rng.integers(0, 60, count)
    lengths[rng.integers(0, count, 6)] = [3000, 900, 1, 257, 64, 2000]
    lengths[0], lengths[-1] = 0, 500
    news = rng.integers(0, news_to + 1, count) if news_to else None
    pages = int(sum(-(-n // page) for n in lengths)) + 1
    pool = R.Pool(pages, kv_heads, 64, page).randomise(rng)
    table = R.tables(rng, lengths, page, pages)
    if news_to:
        # (no more new tokens than a sequence holds, or none at all of it: idle rows)
        news = np.where(lengths > 0, np.minimum(news, lengths), news)
    each = news if news_to else np.ones(count, np.int64)
    q, qb = to_dtype(rng.standard_normal((int(each.sum()), heads, 64)), dtype)
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, 0, 0.125, None)
    check_attention(got, q, pool, table, lengths, each, heads, dtype, 0, 0.125, None)


@pytest.mark.parametrize("heads,kv_heads,hd,news,lengths,window", [
    (64, 8, 64, [1030], [1030], 0),             # blocks enough to be taken whole
    (64, 8, 64, [700, 1, 0, 350], [5000, 1, 9, 901], 100),
    (64, 8, 64, [300, 290], [900, 290], 0),     # short ones, half as many
    (64, 8, 64, [300], [3001], 0),              # divided
    (20, 4, 128, [900, 130], [901, 600], 0),
    (20, 4, 128, [150, 3], [2000, 700], 0),
])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_prompts(dev, held, heads, kv_heads, hd, news, lengths, window, dtype):
    rng = np.random.default_rng(sum(news))
    page = 64
    pages = sum(-(-n // page) for n in lengths)
    pool = R.Pool(pages, kv_heads, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, pages)
    q, qb = to_dtype(rng.standard_normal((sum(news), heads, hd)) * 1.5, dtype)
    sinks = rng.standard_normal(heads).astype(np.float32)
    scale = float(np.float32(hd ** -0.5))
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, window, scale,
                        sinks)
    check_attention(got, q, pool, table, lengths, news, heads, dtype, window, scale, sinks)


@pytest.mark.parametrize("heads,kv_heads,hd,news", [(20, 4, 128, None), (20, 4, 128, [2, 3]), (20, 4, 128, [90, 40]),
                                                    (40, 4, 64, None), (16, 2, 64, [2, 5]), (16, 2, 64, [90, 40])])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_outside_the_half_range(dev, held, heads, kv_heads, hd, news, dtype):
    """Single blocks of V with scale bytes below 104 or above 140, from the middle of a sequence on."""
    rng = np.random.default_rng(41)
    page, lengths = 32, [1500, 300]
    pool = R.Pool(64, kv_heads, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, 64)
    for s, p, d, f in [(0, 800, 3, 2.0 ** 30), (0, 801, hd - 1, 2.0 ** -60), (0, 1300, 40, 2.0 ** 20), (1, 10, 0, 2.0 ** 100),
                       (1, 299, 33, 2.0 ** 19)]:
        k, v = pool.get(table[s], np.array([p]))
        v[0, :, d // 32 * 32:d // 32 * 32 + 32] *= f
        pool.put(table[s], p, k[0], v[0])
    n = sum(news) if news else 2
    q, qb = to_dtype(rng.standard_normal((n, heads, hd)), dtype)
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, 0, 0.125, None)
    check_attention(got, q, pool, table, lengths, news or [1, 1], heads, dtype, 0, 0.125, None)


@pytest.mark.parametrize("news", [[3, 2], [40, 1], [200, 60]])
def test_captured_prompts(dev, held, news):
    """A prompt pass captured once, replayed for other lengths and another division of its rows,
    with eager work between the replays."""
    rng = np.random.default_rng(sum(news))
    heads, kv, page, seqs, tokens = 64, 8, 64, 2, sum(news)
    stride = 40
    table = rng.permutation(128)[:seqs * stride].reshape(seqs, stride).astype(np.int32)
    pool = R.Pool(128, kv, 64, page).randomise(rng)
    pb, tb, lb, sb = held.up(pool.bytes), held.up(table), held.up(np.int32([1, 1])), held.up(cumulative(news))
    cache = T.kv4_cache(pb, 128, kv, 64, page)
    batch = T.kv4_batch(seqs, tokens, tb, stride, lb, sb, None, page)
    att = T.kv4_attention(heads, BF16, 0, 0.125, None)
    need = dev.attention_kv4_workspace_bytes(cache, batch, att)
    q = held.new(tokens * heads * 64 * 2)
    outs = [held.new(tokens * heads * 64 * 2, 0x5a) for _ in range(2)]
    spaces = [held.new(max(need, 16), 0xff) for _ in range(2)]
    graph = dev.capture(lambda: dev.attention_prefill_kv4(cache, batch, att, q, outs[1], spaces[1], need))
    for step, (lengths, split) in enumerate([([2000, 100], news), ([2400, 900], news[::-1]), ([tokens, 0], [tokens, 0]),
                                             ([3, 2500], [1, tokens - 1]), ([2000, 100], news)]):
        lb.upload(np.int32(lengths))
        sb.upload(cumulative(split))
        q.upload(to_dtype(rng.standard_normal((tokens, heads, 64)), BF16)[1])
        dev.attention_prefill_kv4(cache, batch, att, q, outs[0], spaces[0], need)
        dev.sync()
        graph.launch()
        dev.sync()
        a, b = (o.download(np.uint16, tokens * heads * 64) for o in outs)
        assert np.array_equal(a, b) and (a != 0x5a5a).any(), step
    graph.free()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("window", [0, 200])
def test_widest_group(dev, held, dtype, prefill, window):
    """64 query heads a key/value head, the most there are."""
    rng = np.random.default_rng(51)
    heads, lengths, news = 128, [900, 1, 0, 2100], [3, 1, 1, 2]
    pool = R.Pool(60, 2, 64, 64).randomise(rng)
    table = R.tables(rng, lengths, 64, 60)
    each = news if prefill else [1] * 4
    q, qb = to_dtype(rng.standard_normal((sum(each), heads, 64)), dtype)
    sinks = rng.standard_normal(heads).astype(np.float32)
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news if prefill else None, qb, heads,
                        dtype, window, 0.125, sinks)
    check_attention(got, q, pool, table, lengths, each, heads, dtype, window, 0.125, sinks)


@pytest.mark.parametrize("heads,kv_heads,hd,page", [(64, 8, 64, 64), (64, 8, 64, 32), (20, 4, 128, 64), (20, 4, 128, 16)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new,length", [(200, 300), (120, 2500)])
@pytest.mark.parametrize("missing", [-1, 1 << 30])
def test_a_missing_page_in_a_prompt(dev, held, heads, kv_heads, hd, page, dtype, new, length, missing):
    """NaN for the rows that see it, through a window; the others as without it."""
    rng = np.random.default_rng(53)
    window = 40
    lengths, news = [length, 64], [new, 64]
    pages = sum(-(-n // page) for n in lengths)
    pool = R.Pool(pages, kv_heads, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, pages)
    gone = (length - 150) // page                       # the page of a position inside the prompt
    q, qb = to_dtype(rng.standard_normal((new + 64, heads, hd)), dtype)
    broken = table.copy()
    broken[0, gone] = missing
    pb = held.up(pool.bytes)
    whole, got = (run_attention(dev, held, pb, pool, t, lengths, news, qb, heads, dtype, window, 0.125, None)
                  for t in (table, broken))
    at = np.arange(length - new, length)
    sees = (at >= gone * page) & (at - window + 1 < (gone + 1) * page)
    assert sees.any() and not sees.all()
    assert np.isnan(got[:new][sees]).all()
    assert np.array_equal(got[:new][~sees], whole[:new][~sees]) and np.array_equal(got[new:], whole[new:])
    check_attention(whole, q, pool, table, lengths, news, heads, dtype, window, 0.125, None)


@pytest.mark.parametrize("heads,kv_heads,hd,page", [(64, 8, 64, 64), (8, 2, 64, 16), (5, 5, 128, 32), (20, 4, 128, 64),
                                                    (3, 3, 64, 128)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("with_sinks", [False, True])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("capacity", [256, 1500])       # blocks taken whole, and divided
def test_prompts_with_more_rows_than_positions(dev, held, heads, kv_heads, hd, page, dtype, with_sinks, window,
                                               capacity):
    """Rows before position 0 next to rows that see positions, in prompts long enough for a wave to
    have queries of its own: zeros for the ones, the others as they are without them."""
    rng = np.random.default_rng(61 + heads + window)
    news = [130, 131, 97, 170]
    lengths = [n - more for n, more in zip(news, (3, 7, 20, 30))]
    pages = sum(-(-n // page) for n in lengths)
    pool = R.Pool(pages, kv_heads, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, pages, capacity // page + 1)
    q, qb = to_dtype(rng.standard_normal((sum(news), heads, hd)) * 1.5, dtype)
    sinks = rng.standard_normal(heads).astype(np.float32) if with_sinks else None
    scale = float(np.float32(hd ** -0.5))
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, window, scale,
                        sinks, max_length=capacity)
    check_attention(got, q, pool, table, lengths, news, heads, dtype, window, scale, sinks)


# ---- the weights' bits -------------------------------------------------------------------------------
#
# (heads, kv heads, head width, new tokens; None: decode) that take each of the kernels' ways of working
WAYS = [(8, 1, 64, None), (8, 1, 64, [2]), (8, 1, 64, [4]), (8, 1, 64, [70]), (8, 1, 64, [300]), (8, 1, 128, None),
        (8, 1, 128, [2]), (8, 1, 128, [4]), (8, 1, 128, [70])]


def put_all(pool, table_row, k, v):
    """k, v f64 [positions][kv_heads][hd] from position 0 on."""
    at = np.arange(len(k))
    page, slot = np.asarray(table_row)[at // pool.page], at % pool.page
    for x, c, b in ((k, pool.kc, pool.ks), (v, pool.vc, pool.vs)):
        code, byte = R.quantise(x)
        c[page, :, slot], b[page, :, slot] = R.pack(code), byte


def check_close(got, q, pool, table, lengths, news, heads, dtype, window, scale, sinks):
    row = 0
    for s, (n, m) in enumerate(zip(lengths, news)):
        first = max(0, n - m + 1 - window) if window else 0
        k, v = pool.get(table[s], np.arange(first, n))
        ref, mag, smax, vsum = R.attention(q[row:row + m], k, v, np.arange(n - m, n), first, window, scale, sinks)
        tol = R.close_allowance(ref, mag, smax, vsum, n - first, pool.hd, dtype == BF16)
        off = np.abs(got[row:row + m] - ref)
        assert (off <= tol).all(), (s, n, m, float((off / np.maximum(tol, 1e-300)).max()))
        row += m


@pytest.mark.parametrize("heads,kv_heads,hd,news", WAYS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("top", [0, 1900, 3600])
def test_small_weights_count(dev, held, heads, kv_heads, hd, news, dtype, top):
    """One key up to 60 nats above thousands of equal ones, with a v of zero in half the dims: what
    is left there is the small weights' sum."""
    n, page = 4001, 64
    pool = R.Pool(63, kv_heads, hd, page)
    table = np.arange(63, dtype=np.int32)[None]
    for codes, scales, x in ((pool.kc, pool.ks, 0.0), (pool.vc, pool.vs, 1.0)):
        code, byte = R.quantise(np.full(hd, x))
        codes[...], scales[...] = R.pack(code), byte
    k, v = np.zeros((kv_heads, hd)), np.ones((kv_heads, hd))
    k[:, 0], v[:, :hd // 2] = 1.0, 0.0
    pool.put(table[0], top, k, v)
    rows = news[0] if news else 1
    x = np.zeros((rows, heads, hd))
    x[:, :, 0] = 8.0 * np.array([0, 10, 18, 21, 23, 30, 45, 60])   # (bf16 holds these)
    q, qb = to_dtype(x, dtype)
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, [n], news, qb, heads, dtype, 0, 0.125, None)
    check_close(got, q, pool, table, [n], news or [1], heads, dtype, 0, 0.125, None)


@pytest.mark.parametrize("heads,kv_heads,hd,news", WAYS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_weights_keep_their_bits(dev, held, heads, kv_heads, hd, news, dtype):
    """Values of alternating sign under nearly equal weights: what is left of a sum is the weights'
    differences, far below their own rounding to 11 bits."""
    rows, page = news[0] if news else 1, 64
    n = max(rows, 2)
    pool = R.Pool(5, kv_heads, hd, page)
    table = np.arange(5, dtype=np.int32)[None]
    k, v = np.zeros((n, kv_heads, hd)), np.ones((n, kv_heads, hd))
    k[::2, :, 0], v[1::2] = 1.0, -1.0
    put_all(pool, table[0], k, v)
    x = np.zeros((rows, heads, hd))
    x[:, :, 0] = 8.0 * np.linspace(0.001, 0.011, rows * heads).reshape(rows, heads)
    q, qb = to_dtype(x, dtype)
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, [n], news, qb, heads, dtype, 0, 0.125, None)
    check_close(got, q, pool, table, [n], news or [1], heads, dtype, 0, 0.125, None)


@pytest.mark.parametrize("heads,kv_heads,hd,news", WAYS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("length", [1, 2, 5, 90, 700])
def test_the_largest_values(dev, held, heads, kv_heads, hd, news, dtype, length):
    """V up to the largest that a block holds, or as large as positions times V stay below 2^128;
    scores grow along the sequence, so weights do."""
    rng = np.random.default_rng(81 + length)
    rows, page = news[0] if news else 1, 64
    n = max(length, rows)
    e = min(125, int(np.floor(128 - np.log2(6 * n))))
    pool = R.Pool(16, kv_heads, hd, page)
    table = rng.permutation(16).astype(np.int32)[None]
    k = rng.standard_normal((n, kv_heads, hd)) * 0.2
    k[:, :, 0] = np.arange(n)[:, None] / n
    v = np.full((n, kv_heads, hd), 6.0 * 2.0 ** e)
    v[:, :, 1::3] *= -1.0 / 3.0
    v[:, :, 2] = 0.0
    put_all(pool, table[0], k, v)
    x = rng.standard_normal((rows, heads, hd)) * 0.5
    x[:, :, 0] = np.linspace(-40, 160, heads)
    q, qb = to_dtype(x, dtype)
    sinks = rng.standard_normal(heads).astype(np.float32)
    for s in (None, sinks):
        got = run_attention(dev, held, held.up(pool.bytes), pool, table, [n], news, qb, heads, dtype, 0, 0.125, s)
        assert np.isfinite(got).all()
        check_close(got, q, pool, table, [n], news or [1], heads, dtype, 0, 0.125, s)


@pytest.mark.parametrize("news,tokens", [([3, 5], 6), ([3, 5], 2), ([90, 300], 301), ([400, 90], 120), ([700], 650)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_starts_past_the_rows(dev, held, news, tokens, dtype):
    """Arrays that hold fewer rows than starts names: the rows that are there as in the whole call,
    in the store, the read-back and the attention."""
    rng = np.random.default_rng(91 + tokens)
    heads, kv, hd, page = 8, 1, 64, 64
    lengths = [n + 400 * s for s, n in enumerate(news)]
    pages = sum(-(-n // page) for n in lengths)
    pool = R.Pool(pages, kv, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, pages)
    total = sum(news)
    x = rng.standard_normal((total, (heads + 2 * kv) * hd)).astype(np.float32)
    rope, tb, lb = held.up(rope_table(max(lengths), hd, rng)), held.up(table), held.up(np.int32(lengths))
    sb, xb = held.up(cumulative(news)), held.up(x)
    att = T.kv4_attention(heads, dtype, 0, 0.125, None)
    size = 2 if dtype == BF16 else 4
    seen = []
    for rows in (total, tokens):
        pb = held.up(pool.bytes)
        cache = T.kv4_cache(pb, pages, kv, hd, page)
        batch = T.kv4_batch(len(news), rows, tb, table.shape[1], lb, sb, None, page)
        q, out = (held.new(total * heads * hd * size, 0x5a) for _ in range(2))
        dev.qkv_rope_store_kv4(cache, batch, heads, xb, F32, None, rope, max(lengths), q, dtype)
        k = held.new(total * kv * hd * 4, 0x5a)
        dev.kv4_dequantize(cache, batch, k, None)
        stored = pb.download(np.uint8)
        # (over the whole call's cache: the rows left out are keys of those behind them)
        if rows == total:
            full = cache
        need = dev.attention_kv4_workspace_bytes(full, batch, att)
        dev.attention_prefill_kv4(full, batch, att, q, out, held.new(need) if need else None, need)
        seen.append((read(q, (total, heads, hd), dtype), read(k, (total, kv, hd), F32),
                     read(out, (total, heads, hd), dtype), stored))
    (q0, k0, o0, _), (q1, k1, o1, stored) = seen
    assert np.array_equal(q0[:tokens], q1[:tokens]) and np.array_equal(k0[:tokens], k1[:tokens])
    whole, row = R.Pool(pages, kv, hd, page), 0
    whole.bytes[...] = seen[0][3].reshape(whole.bytes.shape)
    for s, (n, m) in enumerate(zip(lengths, news)):
        here = min(m, max(tokens - row, 0))
        kf, vf = whole.get(table[s], np.arange(n))
        ref, mag, smax, vsum = R.attention(q1[row:row + here], kf, vf, np.arange(n - m, n - m + here), 0, 0, 0.125, None)
        tol = R.close_allowance(ref, mag, smax, vsum, n, hd, dtype == BF16)
        for o in (o0, o1):
            assert (np.abs(o[row:row + here] - ref) <= tol).all(), s
        row += m
    for a in (q1, k1, o1):
        assert (a[tokens:] == a[-1, -1, -1]).all()
    # what the rows that are there stored, and nothing else
    after = R.Pool(pages, kv, hd, page)
    after.bytes[...] = pool.bytes
    at = np.concatenate([np.arange(n - m, n) for n, m in zip(lengths, news)])
    seq = np.repeat(np.arange(len(news)), news)
    _, kr, vr = R.rotate(x, None, rope.download(np.float32).reshape(max(lengths), hd // 2, 2), at, heads, kv, hd)
    for i in range(tokens):
        after.put(table[seq[i]], at[i], kr[i], vr[i])
    assert np.array_equal(stored.reshape(after.bytes.shape), after.bytes)


@pytest.mark.parametrize("news", [None, [3, 1, 90, 5], [80, 70, 90, 75]])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_short_sequences_need_no_workspace(dev, held, news, dtype):
    rng = np.random.default_rng(95)
    heads, kv, lengths = 16, 2, [90, 200, 95, 130]
    pool = R.Pool(12, kv, 64, 64).randomise(rng)
    table = R.tables(rng, lengths, 64, 12)
    each = news or [1] * 4
    q, qb = to_dtype(rng.standard_normal((sum(each), heads, 64)), dtype)
    cache = T.kv4_cache(held.up(pool.bytes), 12, kv, 64, 64)
    batch = T.kv4_batch(4, sum(each), held.up(table), table.shape[1], held.up(np.int32(lengths)),
                        held.up(cumulative(news)) if news else None, 200)
    att = T.kv4_attention(heads, dtype, 0, 0.125, None)
    assert dev.attention_kv4_workspace_bytes(cache, batch, att) == 0
    out = held.new(sum(each) * heads * 64 * 4)
    (dev.attention_prefill_kv4 if news else dev.attention_decode_kv4)(cache, batch, att, held.up(qb), out)
    check_close(read(out, q.shape, dtype), q, pool, table, lengths, each, heads, dtype, 0, 0.125, None)


@pytest.mark.parametrize("heads,kv_heads,hd,page", [(256, 256, 64, 16), (512, 256, 128, 32)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("news", [None, [2, 3], [70, 66]])
def test_most_kv_heads(dev, held, heads, kv_heads, hd, page, dtype, news):
    rng = np.random.default_rng(96)
    lengths = [300, 70]
    pages = sum(-(-n // page) for n in lengths)
    pool = R.Pool(pages, kv_heads, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, pages)
    each = news or [1, 1]
    q, qb = to_dtype(rng.standard_normal((sum(each), heads, hd)), dtype)
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, news, qb, heads, dtype, 0, 0.125, None)
    check_close(got, q, pool, table, lengths, each, heads, dtype, 0, 0.125, None)


@pytest.mark.parametrize("heads,kv_heads,hd,news", WAYS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 12, 2.0 ** 24, 2.0 ** 27])
def test_huge_scores(dev, held, heads, kv_heads, hd, news, dtype, size):
    """Exact scores of up to 2^29 in magnitude, the largest of them shared by three positions."""
    n, page = 900, 64
    pool = R.Pool(15, kv_heads, hd, page)
    table = np.arange(15, dtype=np.int32)[None]
    rng = np.random.default_rng(97)
    rows = news[0] if news else 1
    k0 = rng.choice([-3.0, -2.0, -1.0, -0.5, 0.0, 0.5, 1.0, 2.0, 3.0], n)
    k0[[5, 300, n - rows]] = 4.0
    k = np.zeros((n, kv_heads, hd))
    k[:, :, 0] = k0[:, None]
    put_all(pool, table[0], k, rng.standard_normal((n, kv_heads, hd)))
    x = np.zeros((rows, heads, hd))
    x[:, :, 0] = 8.0 * size * np.linspace(0.5, 1.0, heads)[None] * (1.0 + 0.25 * (np.arange(rows) % 2))[:, None] * 0.75
    q, qb = to_dtype(x, dtype)
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, [n], news, qb, heads, dtype, 0, 0.125, None)
    ref, mag, smax, vsum = R.attention(q, *pool.get(table[0], np.arange(n)), np.arange(n - rows, n), 0, 0, 0.125, None)
    # (the scores are exact; their differences in units of log 2 take two roundings, 2^-23 of them, and
    # a difference of more than 200 is a weight of zero)
    tol = R.close_allowance(ref, mag, np.full_like(smax, min(100.0, 8.0 * size)), vsum, n, hd, dtype == BF16)
    assert (np.abs(got - ref) <= tol).all()


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_very_many_sequences(dev, held, prefill, dtype):
    """More blocks than a call divides (2^16), over shared pages: rows of one length are alike."""
    rng = np.random.default_rng(98)
    count, heads, page = 70001, 8, 16
    pool = R.Pool(80, 1, 64, page).randomise(rng)
    one = rng.permutation(80)[:70].astype(np.int32)
    known = np.array([1, 2, 15, 16, 17, 64, 65, 300, 1100, 0])
    lengths = known[rng.integers(0, len(known), count)]
    table = np.tile(one[None], (count, 1))
    q1, qb1 = to_dtype(rng.standard_normal((1, heads, 64)), dtype)
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, lengths, np.ones(count, np.int64) if prefill else None,
                        np.ascontiguousarray(np.broadcast_to(qb1, (count, heads, 64))), heads, dtype, 0, 0.125, None)
    for n in known:
        rows = got[lengths == n]
        assert len(rows) and (rows == rows[0]).all(), n
        check_attention(rows[:1], q1, pool, table[:1], [n], [1], heads, dtype, 0, 0.125, None)


@pytest.mark.parametrize("heads,kv_heads,hd,page,news", [(16, 2, 64, 16, None), (16, 2, 64, 64, [3, 2]),
                                                         (16, 2, 64, 16, [90, 70]),
                                                         (10, 2, 128, 16, None), (10, 2, 128, 64, [3, 2]),
                                                         (10, 2, 128, 16, [90, 70])])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_least_alignment(dev, held, heads, kv_heads, hd, page, news, dtype):
    """Every array at the least alignment that the header names (16 bytes; 4 for index arrays and
    sinks), and what lies next to q and out left as it was."""
    rng = np.random.default_rng(99)
    lengths = [130, 300]
    pages = sum(-(-n // page) for n in lengths)
    pool = R.Pool(pages, kv_heads, hd, page).randomise(rng)
    table = R.tables(rng, lengths, page, pages)
    each = news or [1, 1]
    rows, size = sum(each), 2 if dtype == BF16 else 4

    def at(a, offset):
        a = np.ascontiguousarray(a)
        b = held.new(a.nbytes + 64, 0x5a)
        raw = np.full(a.nbytes + 64, 0x5a, np.uint8)
        raw[offset:offset + a.nbytes] = a.view(np.uint8).reshape(-1)
        b.upload(raw)
        return b, b.ptr + offset

    width = (heads + 2 * kv_heads) * hd
    x, bias = rng.standard_normal((rows, width)).astype(np.float32), rng.standard_normal(width).astype(np.float32)
    rope = rope_table(300, hd, rng)
    sinks = rng.standard_normal(heads).astype(np.float32)
    pb, pp = at(pool.bytes, 16)
    qb, qp = at(np.full(rows * heads * hd * size, 0x5a, np.uint8), 16)
    ob, op = at(np.full(rows * heads * hd * size, 0x5a, np.uint8), 16)
    cache = T.kv4_cache(pp, pages, kv_heads, hd, page)
    batch = T.kv4_batch(2, rows, at(table, 4)[1], table.shape[1], at(np.int32(lengths), 4)[1],
                        at(cumulative(news), 4)[1] if news else None)
    dev.qkv_rope_store_kv4(cache, batch, heads, at(x, 16)[1], F32, at(bias, 16)[1], at(rope, 16)[1], 300, qp, dtype)
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lengths, each)])
    qr, kr, vr = R.rotate(x, bias, rope, pos, heads, kv_heads, hd)
    for i, s in enumerate(np.repeat([0, 1], each)):
        pool.put(table[s], pos[i], kr[i], vr[i])
    raw = pb.download(np.uint8)
    assert np.array_equal(raw[16:16 + pool.bytes.nbytes], pool.bytes.reshape(-1)) and (raw[:16] == 0x5a).all()
    assert (raw[16 + pool.bytes.nbytes:] == 0x5a).all()
    att = T.kv4_attention(heads, dtype, 0, 0.125, at(sinks, 4)[1])
    need = dev.attention_kv4_workspace_bytes(cache, batch, att)
    ws = held.new(need) if need else None
    (dev.attention_prefill_kv4 if news else dev.attention_decode_kv4)(cache, batch, att, qp, op, ws, need)
    got = []
    for b in (qb, ob):
        raw = b.download(np.uint8)
        assert (raw[:16] == 0x5a).all() and (raw[16 + rows * heads * hd * size:] == 0x5a).all()
        data = raw[16:16 + rows * heads * hd * size]
        got.append((R.from_bf16(data.view(np.uint16)) if dtype == BF16 else data.view(np.float32))
                   .reshape(rows, heads, hd).astype(np.float64))
    assert (np.abs(got[0] - qr) <= (2.0 ** -8 if dtype == BF16 else 2.0 ** -24) * np.abs(qr) + 2.0 ** -45).all()
    check_close(got[1], got[0], pool, table, lengths, each, heads, dtype, 0, 0.125, sinks)


@pytest.mark.parametrize("heads,kv_heads,hd,news", WAYS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("e", [-104, -112, -120, -126])
def test_the_smallest_values(dev, held, heads, kv_heads, hd, news, dtype, e):
    """V in blocks of the smallest scales: what f32 holds of the output, down to its subnormals."""
    rng = np.random.default_rng(101)
    rows, page, n = news[0] if news else 1, 64, 333
    pool = R.Pool(16, kv_heads, hd, page)
    table = rng.permutation(16).astype(np.int32)[None]
    put_all(pool, table[0], rng.standard_normal((n, kv_heads, hd)),
            rng.choice([-6.0, -3.0, -1.0, 0.5, 1.5, 2.0, 4.0], (n, kv_heads, hd)) * 2.0 ** e)
    q, qb = to_dtype(rng.standard_normal((rows, heads, hd)), dtype)
    got = run_attention(dev, held, held.up(pool.bytes), pool, table, [n], news, qb, heads, dtype, 0, 0.125, None)
    check_close(got, q, pool, table, [n], news or [1], heads, dtype, 0, 0.125, None)
