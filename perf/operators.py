"""The paged 4-bit K/V cache's operators as cases that can be timed and checked.

Three operators of a program that serves several sequences over one pool of pages: storing
the keys and values of new tokens (bias, position rotation, quantisation to MXFP4 blocks),
attention of one token per sequence over the cached positions, and attention of runs of
prompt tokens over them.  Head counts are gpt-oss's (64 query and 8 key/value heads of 64)
unless a case says otherwise; contexts are those of the decode benchmarks and up to the
model's longest.

Where `own` is false, run() computes the operators in plain torch; where it is true, it
calls the library.  exact() evaluates the definitions in 64 bits, sequence by sequence.

The pool is uint8 [pages][kv_heads][record], a record being K codes [page][hd / 2], V codes
[page][hd / 2], K scales [page][hd / 32], V scales [page][hd / 32].
"""
import ctypes as C
import math
import os
import sys

import torch

own = False

WINDOW = 128                  # sliding window of the even layers


def _case(name, kind, **kw):
    c = {"name": name, "kind": kind, "heads": 64, "kv_heads": 8, "hd": 64, "page": 64, "window": 0, "sinks": True,
         "dtype": "f32", "sequences": 1, "length": 2048, "spread": 0.0, "idle": False}
    c.update(kw)
    return c


def listed():
    return [
        # The store of one decode step for 32 sequences, straight from the batched Q/K/V
        # product of this framework (its row order).
        _case("store_decode_32", "store", sequences=32, new=1, length=2048, spread=0.9, tiled=True),
        # The store of a prefill pass over three ragged prompts, queries handed on in bf16.
        _case("store_prompt_ragged", "store", sequences=3, new=1024, length=1500, spread=0.6, page=16, dtype="bf16",
              tiled=False),
        # A decode step of one sequence at the decode benchmark's context, full layer: the
        # smallest call, where latency counts.
        _case("decode_1_2048", "decode"),
        # The same step's sliding layer for a batch, one slot of it idle.
        _case("decode_32_window", "decode", sequences=32, length=4096, spread=0.9, window=WINDOW, idle=True),
        # A serving batch with ragged contexts, bf16 queries.
        _case("decode_64_ragged", "decode", sequences=64, length=8192, spread=0.95, dtype="bf16", page=128),
        # One sequence at the model's longest context.
        _case("decode_1_131072", "decode", length=131072, dtype="bf16"),
        # A large even batch at the 120b benchmark's context, f32 queries.
        _case("decode_128_4096", "decode", sequences=128, length=4096),
        # Another head layout: 128-wide heads, 5 query heads a key/value head, odd context.
        _case("decode_16_hd128", "decode", heads=20, kv_heads=4, hd=128, sequences=16, length=3001, spread=0.5,
              dtype="bf16", page=16, sinks=False),
        # A 512-token pass of the framework's own prefill at its end of a 2048-token prompt.
        _case("prompt_512_at_1536", "prompt", new=512, length=2048),
        # Several ragged prompt passes in one call, sliding layer.
        _case("prompt_ragged_window", "prompt", sequences=6, new=700, length=2500, spread=0.8, window=WINDOW,
              dtype="bf16", page=16),
        # Few new tokens over long contexts (drafted tokens checked in one pass).
        _case("prompt_4_tokens_16k", "prompt", sequences=8, new=4, length=16384, spread=0.3, dtype="bf16"),
        # A whole 4096-token prompt in one call.
        _case("prompt_4096", "prompt", new=4096, length=4096, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["store", "decode", "decode", "prompt", "prompt"])
    heads, kv_heads, hd = rng.choice([(64, 8, 64), (64, 8, 64), (64, 8, 64), (32, 8, 128), (20, 4, 128), (16, 16, 64)])
    c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "hd": hd, "page": rng.choice([16, 32, 64, 128, 256]),
         "window": rng.choice([0, 0, WINDOW, rng.randint(1, 1000)]), "sinks": rng.random() < 0.7,
         "dtype": rng.choice(["f32", "bf16"]), "spread": rng.choice([0.0, round(rng.random(), 3)]), "idle": False}
    c["sequences"] = _log(rng, 1, 128)
    if kind == "store":
        c["new"] = rng.choice([1, _log(rng, 1, 2048 // c["sequences"] + 1)])
        c["length"] = max(c["new"], _log(rng, 1, 4096))
        c["tiled"] = (heads, kv_heads, hd) == (64, 8, 64) and rng.random() < 0.5
    elif kind == "decode":
        c["length"] = _log(rng, 1, 4 * 131072 // c["sequences"] if c["sequences"] > 4 else 131072)
        c["idle"] = c["sequences"] > 1 and rng.random() < 0.3
    else:
        c["sequences"] = _log(rng, 1, 16)
        c["new"] = _log(rng, 2, 4096 // c["sequences"])
        c["length"] = max(c["new"], _log(rng, 2, min(32768, 4096 * 4096 // (c["sequences"] * c["new"]))))
    return c


# ---- the batch's shape, from the case alone --------------------------------------------------


def _fractions(n, step):
    return [(i * step) % 1.0 for i in range(n)]


def _lengths(c):
    """Cached positions of each sequence, the call's own tokens included; the first is the
    longest, an idle slot (the last) has none."""
    n = [1 + int((c["length"] - 1) * (1.0 - c["spread"] * f)) for f in _fractions(c["sequences"], 0.6180339887)]
    if c["idle"]:
        n[-1] = 0
    return n


def _news(c):
    """New tokens of each sequence."""
    if c["kind"] == "decode" or c["new"] == 1:
        return [1] * c["sequences"]
    n = [1 + int((c["new"] - 1) * (1.0 - c["spread"] * f)) for f in _fractions(c["sequences"], 0.4142135624)]
    return [min(a, b) for a, b in zip(n, _lengths(c))]


# ---- MXFP4 blocks and the pool ---------------------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantise(x):
    """x [..., hd] (in 32 or 64 bits) as codes uint8 [..., hd / 2] and E8M0 bytes [..., hd / 32]:
    per 32 values the smallest exponent e with every magnitude below 7 x 2^e, nearest E2M1 of
    x / 2^e, ties to the even code."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    m = b.abs().amax(-1, keepdim=True)
    f, e = torch.frexp(m)  # m = f 2^e, f in [0.5, 1): m < 7 2^(e - 3) for f < 0.875
    e = torch.where(f < 0.875, e - 3, e - 2).clamp(-126, 125)
    a = torch.ldexp(b.abs(), -e)
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    scale = torch.where((code > 0).any(-1, keepdim=True), (e + 127).to(torch.uint8), torch.zeros_like(e, dtype=torch.uint8))
    code = (code | (torch.signbit(b).to(torch.uint8) << 3)).reshape(*x.shape[:-1], -1, 2)
    return code[..., 0] | (code[..., 1] << 4), scale[..., 0]


def _values(codes, scales):
    """The blocks' values, f32 [..., hd]."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
    v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1)
    v = v.reshape(*codes.shape[:-1], -1, 32)
    return torch.ldexp(v, (scales.to(torch.int32) - 127)[..., None]).reshape(*codes.shape[:-1], -1)


def _views(pool, c):
    """K codes, V codes, K scales, V scales of a pool, each [pages][kv_heads][page][...]."""
    p, hd = c["page"], c["hd"]
    widths = [hd // 2, hd // 2, hd // 32, hd // 32]
    return [x.unflatten(-1, (p, -1)) for x in pool.split([p * w for w in widths], -1)]


# ---- inputs from a seed --------------------------------------------------------------------------


def _inputs(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 29)

    def normal(*shape, sigma=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * sigma

    heads, kv, hd, page = c["heads"], c["kv_heads"], c["hd"], c["page"]
    lengths, news = _lengths(c), _news(c)
    used = [-(-n // page) for n in lengths]
    pages = sum(used) + 3                       # a pool has pages that no sequence holds
    stride = max(used) + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((c["sequences"], stride), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    pool = torch.empty(pages, kv, page * (hd + hd // 16), dtype=torch.uint8, device="cuda")
    views = _views(pool, c)
    gain = torch.exp(normal(kv, 1, hd, sigma=0.5))  # keys have strong and weak channels
    views[0][:], views[2][:] = _quantise(normal(pages, kv, page, hd) * gain)
    views[1][:], views[3][:] = _quantise(normal(pages, kv, page, hd))
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    starts = [sum(news[:i]) for i in range(len(news) + 1)]
    t = {"pool": pool, "table": table, "tokens": starts[-1], "dtype": dt,
         "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
         "starts": torch.tensor(starts, dtype=torch.int32, device="cuda")}
    if c["kind"] == "store":
        t["qkv"] = normal(t["tokens"], (heads + 2 * kv) * hd)
        t["bias"] = normal((heads + 2 * kv) * hd, sigma=0.1)
        angle = (torch.arange(max(lengths), device="cuda", dtype=torch.float64)[:, None] *
                 150000.0 ** (-2.0 * torch.arange(hd // 2, device="cuda", dtype=torch.float64) / hd)[None])
        t["rope"] = (torch.stack([torch.cos(angle), torch.sin(angle)], -1) * (1.0 + 0.1 * math.log(32.0))).float()
    else:
        t["q"] = normal(t["tokens"], heads, hd, sigma=1.5).to(dt)
        t["sinks"] = normal(heads) if c["sinks"] else None
    return t


class _State:
    pass


def prepare(case, seed):
    st = _State()
    st.case, st.t = case, _inputs(case, seed)
    heads, kv, hd, n = case["heads"], case["kv_heads"], case["hd"], st.t["tokens"]
    st.out = [torch.empty(n, heads, hd, dtype=st.t["dtype"], device="cuda")]
    if case["kind"] == "store":
        st.out += [torch.empty(n, kv, hd, device="cuda") for _ in range(2)]
    st.plan = None  # the library's descriptors and workspace, made on the first pass
    return st


# ---- one pass ----------------------------------------------------------------------------------


def run(st):
    if own:
        return _run_own(st)
    return _plain_store(st) if st.case["kind"] == "store" else _plain_attention(st)


def _token_rows(t, n):
    """Each row's sequence and position."""
    row = torch.arange(t["tokens"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(t["starts"], row, right=True) - 1
    return seq, (t["lengths"][seq] - t["starts"][seq + 1] + row).long()


def _tiled_order(heads, kv, hd):
    """For each column of the framework's Q/K/V product, its place in q | k | v: 16-column
    tiles, of query and key heads 8 dims and the 8 that they rotate with."""
    col = torch.arange((heads + 2 * kv) * hd, device="cuda")
    tile, r = col // 16, col % 16
    j = tile % 4
    dim = torch.where(tile >= (heads + kv) * 4, 16 * j + r, torch.where(r < 8, 8 * j + r, 24 + 8 * j + r))
    return (tile // 4) * hd + dim


def _plain_store(st):
    c, t = st.case, st.t
    heads, kv, hd = c["heads"], c["kv_heads"], c["hd"]
    seq, pos = _token_rows(t, c["sequences"])
    x = t["qkv"].double()
    if c["tiled"]:
        x = torch.empty_like(x).index_copy_(1, _tiled_order(heads, kv, hd), x)
    x = (x + t["bias"].double()).reshape(-1, heads + 2 * kv, hd)
    cs = t["rope"][pos].double()[:, None]
    lo, hi = x[:, :heads + kv, :hd // 2], x[:, :heads + kv, hd // 2:]
    qk = torch.cat([lo * cs[..., 0] - hi * cs[..., 1], lo * cs[..., 1] + hi * cs[..., 0]], -1)
    page, slot = t["table"][seq, pos // c["page"]].long(), pos % c["page"]
    kc, vc, ks, vs = _views(t["pool"], c)
    kc[page, :, slot], ks[page, :, slot] = _quantise(qk[:, heads:])
    vc[page, :, slot], vs[page, :, slot] = _quantise(x[:, heads + kv:])
    return [qk[:, :heads].to(t["dtype"]), _values(kc[page, :, slot], ks[page, :, slot]),
            _values(vc[page, :, slot], vs[page, :, slot])]


def _plain_attention(st):
    """Every sequence padded to the longest, scores and weights whole in memory."""
    c, t = st.case, st.t
    heads, kv, hd, b = c["heads"], c["kv_heads"], c["hd"], c["sequences"]
    rows = max(_news(c))
    held = t["pool"][t["table"].clamp(min=0).long()]                   # [b][stride][kv][record]
    kc, vc, ks, vs = (x.transpose(1, 2).flatten(2, 3) for x in _views(held, c))
    k, v = _values(kc, ks), _values(vc, vs)                            # [b][kv][positions][hd]
    n = t["starts"].diff()
    local = torch.arange(rows, device="cuda")[None, :]
    row = (t["starts"][:-1, None] + torch.minimum(local, n[:, None] - 1)).long()
    q = t["q"].float()[row]                                            # [b][rows][heads][hd]
    q = q.reshape(b, rows, kv, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, hd)
    at = (t["lengths"] - n)[:, None] + local                           # [b][rows]
    pos = torch.arange(k.shape[2], device="cuda")[None, None]
    seen = (pos <= at[..., None]) & (pos < t["lengths"][:, None, None])
    if c["window"]:
        seen &= pos > at[..., None] - c["window"]
    seen = seen[:, None, :, None]                                      # [b][1][rows][1][positions]
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(hd))
    s = s.reshape(b, kv, rows, heads // kv, -1).masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    if t["sinks"] is not None:
        m = torch.maximum(m, t["sinks"].reshape(1, kv, 1, heads // kv, 1))
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = s.sub_(m).exp_()
    den = p.sum(-1, keepdim=True)
    if t["sinks"] is not None:
        den = den + torch.exp(t["sinks"].reshape(1, kv, 1, heads // kv, 1) - m)
    o = torch.matmul(p.reshape(b, kv, -1, p.shape[-1]), v).reshape(b, kv, rows, heads // kv, hd)
    o = torch.where(den > 0, o / den, torch.zeros_like(o)).permute(0, 2, 1, 3, 4).reshape(b, rows, heads, hd)
    return [o[local < n[:, None]].to(t["dtype"])]


# ---- the library's calls ---------------------------------------------------------------------------

_DEV = []


def _device():
    if not _DEV:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tt-lab_amd"))
        import ttlab_amd
        _DEV.extend([ttlab_amd, ttlab_amd.Device(0)])
    return _DEV


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _run_own(st):
    lib, dev = _device()
    c, t = st.case, st.t
    if st.plan is None:
        dtype = lib.TTL_DTYPE_BF16 if c["dtype"] == "bf16" else lib.TTL_DTYPE_F32
        cache = lib.kv4_cache(t["pool"].data_ptr(), t["pool"].shape[0], c["kv_heads"], c["hd"], c["page"])
        batch = lib.kv4_batch(c["sequences"], t["tokens"], t["table"].data_ptr(), t["table"].shape[1],
                              t["lengths"].data_ptr(), None if c["kind"] == "decode" else t["starts"].data_ptr(),
                              max(_lengths(c)))
        st.plan = [dtype, cache, batch]
        if c["kind"] != "store":
            st.heads = lib.kv4_attention(c["heads"], dtype, window=c["window"], scale=1.0 / math.sqrt(c["hd"]),
                                         sinks=None if t["sinks"] is None else t["sinks"].data_ptr())
            need = dev.attention_kv4_workspace_bytes(cache, batch, st.heads)
            st.ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()  # the library works on a stream of its own: the inputs have to be there
    dtype, cache, batch = st.plan
    if c["kind"] == "store":
        dev.qkv_rope_store_kv4(cache, batch, c["heads"], _ptr(t["qkv"]), lib.TTL_DTYPE_F32, _ptr(t["bias"]),
                               _ptr(t["rope"]), t["rope"].shape[0], _ptr(st.out[0]), dtype, tiled=c["tiled"])
        dev.kv4_dequantize(cache, batch, _ptr(st.out[1]), _ptr(st.out[2]))
    else:
        call = dev.attention_decode_kv4 if c["kind"] == "decode" else dev.attention_prefill_kv4
        call(cache, batch, st.heads, _ptr(t["q"]), _ptr(st.out[0]), _ptr(st.ws), st.ws.numel())
    return st.out


# ---- the least a pass needs --------------------------------------------------------------------------


def work(case):
    c = case
    heads, kv, hd = c["heads"], c["kv_heads"], c["hd"]
    size = 2 if c["dtype"] == "bf16" else 4
    row = kv * (hd + hd // 16)                  # bytes of one cached position
    lengths, news = _lengths(c), _news(c)
    n = sum(news)
    if c["kind"] == "store":
        # q, k and v in, the rotation's rows (each once), q out, the blocks written and read
        # back as f32
        return {"bytes": n * (4 * (heads + 2 * kv) * hd + size * heads * hd + 2 * row + 8 * kv * hd) +
                4 * (heads + 2 * kv) * hd + max(lengths) * hd * 4 * (1 if n > max(lengths) else n / max(lengths)),
                "flops": n * (heads + kv) * hd * 3.0}
    b, f = 2 * size * n * heads * hd, 0.0
    for length, new in zip(lengths, news):
        first = length - new                    # of the new tokens
        w = c["window"] or length + 1
        lo = max(0, first + 1 - w)
        b += max(0, length - lo) * row
        # visible pairs: position p sees min(p + 1, w)
        whole = max(0, min(length, w) - max(first, 0))
        pairs = sum(range(max(first, 0) + 1, max(first, 0) + 1 + whole)) + (new - whole) * w if length else 0
        f += 4.0 * pairs * heads * hd
    return {"bytes": b, "flops": f}


# ---- 64-bit values -------------------------------------------------------------------------------------


def _exact_values(codes, scales):
    """E2M1 from its bits: sign, two exponent bits, one fraction bit; E8M0 2^(byte - 127)."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    ex, fr = (n >> 1) & 3, (n & 1).double()
    mag = torch.where(ex == 0, 0.5 * fr, (1.0 + 0.5 * fr) * torch.exp2(ex.double() - 1.0))
    v = torch.where(n >= 8, -mag, mag)
    return v * torch.exp2(scales.double() - 127.0).repeat_interleave(32, -1)


def _nearest_block(x):
    """Values that blocks of 32 hold for x (64 bits): the smallest exponent at which the
    largest magnitude stays under 7, the nearest of the eight magnitudes, of two equally
    near the one with the even code."""
    b = x.unflatten(-1, (-1, 32))
    e = torch.floor(torch.log2(b.abs().amax(-1, keepdim=True) / 7.0)) + 1.0
    unit = torch.exp2(e)
    even_first = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], dtype=torch.float64, device=x.device)
    pick = ((b.abs() / unit)[..., None] - even_first).abs().min(-1).indices
    return (even_first[pick] * torch.sign(b) * unit).flatten(-2)


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    heads, kv, hd, page, group = c["heads"], c["kv_heads"], c["hd"], c["page"], c["heads"] // c["kv_heads"]
    lengths, news = _lengths(c), _news(c)
    outs, row = [], 0
    if c["kind"] == "store":
        x = t["qkv"].double()
        if c["tiled"]:
            place = _tiled_order(heads, kv, hd)
            x = x[:, torch.argsort(place)]
        x = x + t["bias"].double()
        at = torch.cat([torch.arange(a - n, a, device="cuda") for a, n in zip(lengths, news)])
        x = x.reshape(-1, heads + 2 * kv, 2, hd // 2)
        turn = torch.view_as_complex(t["rope"][at].double())[:, None]
        z = torch.complex(x[:, :heads + kv, 0], x[:, :heads + kv, 1]) * turn
        qk = torch.cat([z.real, z.imag], -1)
        return [qk[:, :heads], _nearest_block(qk[:, heads:]), _nearest_block(x[:, heads + kv:].flatten(-2))]
    kc, vc, ks, vs = _views(t["pool"], c)
    for s, (length, new) in enumerate(zip(lengths, news)):
        if length == 0:
            outs.append(torch.zeros(new, heads, hd, dtype=torch.float64, device="cuda"))
            row += new
            continue
        first = length - new
        lo = max(0, first + 1 - c["window"]) if c["window"] else 0
        pos = torch.arange(lo, length, device="cuda")
        at = t["table"][s, pos // page].long()
        k = _exact_values(kc[at, :, pos % page], ks[at, :, pos % page])     # [positions][kv][hd]
        v = _exact_values(vc[at, :, pos % page], vs[at, :, pos % page])
        q = t["q"][row:row + new].double()
        mine = torch.arange(first, length, device="cuda")[:, None]
        hide = pos[None] > mine
        if c["window"]:
            hide |= pos[None] <= mine - c["window"]
        o = torch.empty(new, heads, hd, dtype=torch.float64, device="cuda")
        for h in range(heads):
            w = (q[:, h] @ k[:, h // group].T.contiguous()) / math.sqrt(hd)
            w.masked_fill_(hide, -math.inf)
            if t["sinks"] is not None:
                w = torch.cat([w, t["sinks"][h].double().expand(new, 1)], 1)
            w = torch.softmax(w, 1)
            o[:, h] = w[:, :pos.numel()] @ v[:, h // group].contiguous()
        outs.append(o)
        row += new
    return [torch.cat(outs)]
