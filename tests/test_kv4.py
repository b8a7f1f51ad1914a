"""The paged 4-bit K/V cache without a device: the pool's size, the refusals (every check
comes before the first use of the device), and the 64-bit reference's own blocks."""
import ctypes as C

import numpy as np
import pytest

import kv4_reference as R
import ttlab_amd as T

LIB = T.load_library()
CTX = C.create_string_buffer(4096)   # stands for a context: the refusals do not look at it
P = 1 << 20                          # a 16-byte aligned address that is never read


def cache(**kw):
    d = dict(kv_heads=8, head_dim=64, page_positions=64, pages=10, pool=P)
    d.update(kw)
    return T.Kv4CacheDesc(**d)


def batch(**kw):
    d = dict(sequences=3, tokens=3, table_stride=4, max_length=200, page_table=P, lengths=P, starts=None)
    d.update(kw)
    return T.Kv4BatchDesc(**d)


def attention(**kw):
    d = dict(heads=64, window=0, scale=0.125, dtype=0, sinks=P)
    d.update(kw)
    return T.Kv4AttentionDesc(**d)


def store(c, b, heads=64, qkv=P, xd=0, order=0, bias=P, rope=P, n=200, q=P, qd=0, ctx=CTX):
    return LIB.ttl_qkv_rope_store_kv4(ctx, C.byref(c) if c else None, C.byref(b) if b else None, heads, qkv, xd, order,
                                      bias, rope, n, q, qd)


def attend(c, b, a, q=P, out=P, ws=P, size=1 << 30, ctx=CTX, prefill=False):
    f = LIB.ttl_attention_prefill_kv4 if prefill else LIB.ttl_attention_decode_kv4
    return f(ctx, C.byref(c) if c else None, C.byref(b) if b else None, C.byref(a) if a else None, q, out, ws, size)


INVALID, SHAPE = -1, -2
BAD_CACHE = [(dict(head_dim=96), SHAPE), (dict(head_dim=0), SHAPE), (dict(kv_heads=0), SHAPE),
             (dict(kv_heads=257), SHAPE), (dict(page_positions=8), SHAPE), (dict(page_positions=48), SHAPE),
             (dict(page_positions=512), SHAPE), (dict(page_positions=0), SHAPE), (dict(pages=0), SHAPE),
             (dict(pages=1 << 31), SHAPE), (dict(pool=None), INVALID), (dict(pool=P + 8), INVALID)]
BAD_BATCH = [(dict(page_table=None), INVALID), (dict(lengths=None), INVALID), (dict(tokens=4), SHAPE),
             (dict(max_length=0), SHAPE), (dict(max_length=257), SHAPE), (dict(table_stride=0), SHAPE),
             (dict(max_length=(1 << 30) + 1, table_stride=1 << 30), SHAPE), (dict(sequences=(1 << 20) + 1), SHAPE),
             (dict(tokens=(1 << 24) + 1, starts=P), SHAPE)]


@pytest.mark.parametrize("bad,code", BAD_CACHE)
def test_bad_caches_are_refused(bad, code):
    c = cache(**bad)
    assert store(c, batch()) == code
    assert LIB.ttl_kv4_dequantize(CTX, C.byref(c), C.byref(batch()), P, P) == code
    assert attend(c, batch(), attention()) == code
    assert attend(c, batch(starts=P), attention(), prefill=True) == code
    if "pool" not in bad:
        assert LIB.ttl_kv4_pool_bytes(C.byref(c)) == 0


@pytest.mark.parametrize("bad,code", BAD_BATCH)
def test_bad_batches_are_refused(bad, code):
    b = batch(**bad)
    assert store(cache(), b) == code
    assert LIB.ttl_kv4_dequantize(CTX, C.byref(cache()), C.byref(b), P, P) == code
    assert attend(cache(), b, attention(), prefill=b.starts is not None) == code
    assert b"ttl_attention" in LIB.ttl_last_error()


def test_bad_store_arguments_are_refused():
    c, b = cache(), batch()
    assert store(c, b, ctx=None) == INVALID
    assert store(None, b) == INVALID and store(c, None) == INVALID
    for bad in (dict(qkv=None), dict(rope=None), dict(q=None), dict(n=0), dict(qkv=P + 4), dict(bias=P + 8),
                dict(rope=P + 4), dict(q=P + 2), dict(xd=2), dict(qd=3), dict(xd=-1), dict(order=2)):
        assert store(c, b, **bad) == INVALID, bad
    for bad in (dict(heads=0), dict(heads=60), dict(heads=8 * 65), dict(heads=8, order=1)):
        assert store(c, b, **bad) == SHAPE, bad
    assert store(cache(head_dim=128), b, order=1) == SHAPE
    big = batch(sequences=1, tokens=1 << 24, starts=P)
    assert store(cache(kv_heads=256, head_dim=128), big, heads=256 * 64) == SHAPE
    assert LIB.ttl_kv4_dequantize(None, C.byref(c), C.byref(b), P, P) == INVALID
    assert LIB.ttl_kv4_dequantize(CTX, C.byref(c), C.byref(b), P + 4, P) == INVALID


def test_bad_attention_arguments_are_refused():
    c, b, a = cache(), batch(), attention()
    assert attend(c, b, a, ctx=None) == INVALID
    assert attend(None, b, a) == INVALID and attend(c, None, a) == INVALID and attend(c, b, None) == INVALID
    for bad in (dict(q=None), dict(out=None), dict(q=P + 8), dict(out=P + 4)):
        assert attend(c, b, a, **bad) == INVALID, bad
    for bad, code in ((dict(heads=0), SHAPE), (dict(heads=12), SHAPE), (dict(heads=8 * 65), SHAPE),
                      (dict(dtype=2), INVALID), (dict(dtype=-1), INVALID), (dict(scale=float("nan")), INVALID),
                      (dict(scale=float("inf")), INVALID)):
        assert attend(c, b, attention(**bad)) == code, bad
    assert attend(c, batch(starts=P), a) == INVALID                 # decode takes no starts
    assert attend(c, b, a, prefill=True) == INVALID                 # prefill needs them


def test_workspace_is_checked():
    # one long sequence: its positions are split, so a workspace is needed
    c, a = cache(pages=4096), attention()
    for b, prefill in ((batch(sequences=1, tokens=1, table_stride=2048, max_length=131072), False),
                       (batch(sequences=1, tokens=4, table_stride=2048, max_length=131072, starts=P), True)):
        need = LIB.ttl_attention_kv4_workspace_bytes(C.byref(c), C.byref(b), C.byref(a))
        if need:
            assert attend(c, b, a, size=need - 1, prefill=prefill) == INVALID
            assert attend(c, b, a, ws=None, prefill=prefill) == INVALID
            assert attend(c, b, a, ws=P + 128, prefill=prefill) == INVALID
    # shapes that are refused need none
    assert LIB.ttl_attention_kv4_workspace_bytes(None, C.byref(b), C.byref(a)) == 0
    assert LIB.ttl_attention_kv4_workspace_bytes(C.byref(c), None, C.byref(a)) == 0
    assert LIB.ttl_attention_kv4_workspace_bytes(C.byref(c), C.byref(b), None) == 0
    assert LIB.ttl_attention_kv4_workspace_bytes(C.byref(c), C.byref(batch(max_length=0)), C.byref(a)) == 0
    assert LIB.ttl_attention_kv4_workspace_bytes(C.byref(c), C.byref(b), C.byref(attention(heads=3))) == 0


def test_empty_batches_do_nothing():
    for b in (batch(sequences=0, tokens=0, page_table=None, lengths=None, table_stride=0, max_length=0),
              batch(sequences=2, tokens=0, starts=P)):
        assert store(cache(), b, qkv=None, rope=None, q=None) == 0
        assert LIB.ttl_kv4_dequantize(CTX, C.byref(cache()), C.byref(b), None, None) == 0
        assert attend(cache(), b, attention(), q=None, out=None, ws=None, size=0, prefill=b.starts is not None) == 0
        assert LIB.ttl_attention_kv4_workspace_bytes(C.byref(cache()), C.byref(b), C.byref(attention())) == 0


def test_pool_bytes():
    # kv_heads (head_dim + head_dim / 16) bytes a position
    for kv_heads, hd, page, pages in ((8, 64, 64, 10), (1, 128, 16, 3), (5, 64, 256, 1), (8, 64, 16, 2000000)):
        assert T.kv4_pool_bytes(pages, kv_heads, hd, page) == pages * page * kv_heads * (hd + hd // 16)
        assert R.Pool(min(pages, 3), kv_heads, hd, page).bytes.nbytes == min(pages, 3) * page * kv_heads * (hd + hd // 16)
    with pytest.raises(T.TtlError):
        T.kv4_pool_bytes(1, head_dim=80)


def test_reference_blocks():
    """Known answers of the block rule."""
    x = np.zeros((6, 32))
    x[0, :9] = [6, 5, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -0.25]      # ties go to the even code
    x[1, 0] = 6.999                                                 # below 7: stays at 2^0, rounds to 6
    x[2, 0] = 7.0                                                   # 7: the next exponent, 3.5 -> 4
    x[3, 0] = 2.0 ** 127 * 1.9                                      # the largest exponent saturates
    x[4, 3] = np.inf
    x[5, 0] = 2.0 ** -128                                           # 0.25 of the smallest unit: a tie, to zero
    code, byte = R.quantise(x)
    assert byte[:, 0].tolist() == [127, 127, 128, 252, 255, 127]
    assert code[0, :9].tolist() == [7, 6, 0, 2, 2, 4, 4, 6, 8]
    v = R.values(code, byte)
    assert v[1, 0] == 6.0 and v[2, 0] == 8.0 and v[3, 0] == 6 * 2.0 ** 125 and np.isnan(v[4]).all() and not v[5].any()
    # never off by more than the half step of the grid around a value below 7 units
    r = np.random.RandomState(0).standard_normal((2000, 32)) * np.exp(np.random.RandomState(1).randn(2000, 1) * 20)
    code, byte = R.quantise(r)
    unit = np.ldexp(1.0, byte.astype(int) - 127)
    a, err = np.abs(r) / unit, np.abs(R.values(code, byte) - r) / unit
    assert a.max() < 7.0 and a.max(1).min() >= 3.5
    assert (err <= np.where(a < 2, 0.25, np.where(a < 4, 0.5, 1.0))).all()


def test_calls_past_a_launch_are_refused():
    """2^24 rows: more threads than one launch counts."""
    c, b = cache(), batch(sequences=1, tokens=1 << 24, starts=P)
    assert store(c, b) == SHAPE and b"too many" in LIB.ttl_last_error()
    assert LIB.ttl_kv4_dequantize(CTX, C.byref(c), C.byref(b), P, P) == SHAPE
    assert attend(c, b, attention(heads=64 * 8), prefill=True) == SHAPE


class Calls:
    """Stands for the library: keeps what the binding hands on."""

    def __getattr__(self, name):
        def call(*args):
            self.last = (name, [a._obj for a in args if hasattr(a, "_obj")])
            return 0
        return call


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_the_default_bound_is_the_page_table(page):
    """Without a max_length the calls take what the table holds in the cache's own pages, whatever
    kv4_batch was told of them; one that is given is kept."""
    dev = object.__new__(T.Device)
    dev.lib, dev.ctx = Calls(), None
    c, a = T.kv4_cache(P, 40, 8, 64, page), T.kv4_attention(64)
    made = [T.kv4_batch(3, 3, P, 7, P), T.kv4_batch(3, 3, P, 7, P, None, 100), T.kv4_batch(3, 3, P, 1 << 28, P),
            T.kv4_batch(3, 3, P, 7, P)]
    made[3].max_length = 90
    for b, bound in zip(made, (7 * page, 100, 1 << 30, 90)):
        for call in (lambda: dev.qkv_rope_store_kv4(c, b, 64, P, 0, P, P, 9, P, 0), lambda: dev.kv4_dequantize(c, b, P, P),
                     lambda: dev.attention_kv4_workspace_bytes(c, b, a), lambda: dev.attention_decode_kv4(c, b, a, P, P),
                     lambda: dev.attention_prefill_kv4(c, b, a, P, P)):
            call()
            _, args = dev.lib.last
            held = args[1]
            assert args[0] is c and held.max_length == bound
            assert (held.sequences, held.tokens, held.table_stride, held.page_table, held.lengths, held.starts) == (
                3, 3, b.table_stride, P, P, None)


def test_a_missing_workspace_is_refused():
    """Calls that are certain to need one (a long sequence, divided) and ones that need none."""
    c, a = cache(pages=4096), attention()
    for b, prefill in ((batch(sequences=1, tokens=1, table_stride=2048, max_length=131072), False),
                       (batch(sequences=1, tokens=4, table_stride=2048, max_length=131072, starts=P), True),
                       (batch(sequences=1, tokens=300, table_stride=2048, max_length=131072, starts=P), True)):
        need = LIB.ttl_attention_kv4_workspace_bytes(C.byref(c), C.byref(b), C.byref(a))
        assert need > 0
        assert attend(c, b, a, size=need - 1, prefill=prefill) == INVALID
        assert str(need).encode() in LIB.ttl_last_error()
        assert attend(c, b, a, size=0, prefill=prefill) == INVALID
        assert attend(c, b, a, ws=None, size=need, prefill=prefill) == INVALID
        assert attend(c, b, a, ws=P + 128, size=need, prefill=prefill) == INVALID
    for b in (batch(max_length=200), batch(tokens=600, starts=P, max_length=200)):
        assert LIB.ttl_attention_kv4_workspace_bytes(C.byref(c), C.byref(b), C.byref(a)) == 0
