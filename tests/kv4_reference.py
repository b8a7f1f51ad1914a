"""The paged 4-bit K/V cache in 64 bits (numpy): blocks, pool layout, store and attention,
written from the definitions in include/ttlab_hip.h, and what tests build batches with."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
F32_MAX = np.float64(np.finfo(np.float32).max)


def quantise(x):
    """x f64 [..., hd] -> codes uint8 [..., hd] (one per value) and bytes uint8 [..., hd / 32]."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(over="ignore", invalid="ignore"):
        finite = np.isfinite(b.astype(np.float32)).all(-1)
    m = np.where(finite, np.abs(np.where(np.isfinite(b), b, 0.0)).max(-1), 0.0)
    e = np.full(m.shape, -126)
    for cand in range(125, -127, -1):       # the smallest e with m < 7 x 2^e
        e = np.where(m < np.ldexp(7.0, cand), cand, e)
    e = np.where(m >= np.ldexp(7.0, 125), 125, e)
    a = np.where(finite[..., None], np.ldexp(np.abs(np.where(finite[..., None], b, 0.0)), -e[..., None]), 0.0)
    d = np.abs(a[..., None] - E2M1)
    near = d == d.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1)).astype(np.uint8)
    byte = np.where((code > 0).any(-1), e + 127, 127)
    byte = np.where(finite, byte, 255).astype(np.uint8)
    code = np.where(finite[..., None], code | (np.signbit(b).astype(np.uint8) << 3), 0).astype(np.uint8)
    return code.reshape(x.shape), byte


def values(code, byte):
    """The values of codes [..., hd] and bytes [..., hd / 32], f64; NaN for byte 255."""
    v = E2M1[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(np.int64) - 127))
    return v * np.repeat(s, 32, axis=-1)


def pack(code):
    return (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)


def unpack(b):
    return np.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)


class Pool:
    """A pool on the host, as views of its bytes: [pages][kv_heads][page][...]."""

    def __init__(self, pages, kv_heads=8, hd=64, page=64, fill=None, seed=0):
        self.pages, self.kv_heads, self.hd, self.page = pages, kv_heads, hd, page
        self.record = page * (hd + hd // 16)
        shape = (pages, kv_heads, self.record)
        self.bytes = (np.random.RandomState(seed).randint(0, 256, shape).astype(np.uint8) if fill is None
                      else np.full(shape, fill, np.uint8))
        at = [0]
        for w in (hd // 2, hd // 2, hd // 32, hd // 32):
            at.append(at[-1] + page * w)
        self.kc, self.vc, self.ks, self.vs = (
            self.bytes[:, :, at[i]:at[i + 1]].reshape(pages, kv_heads, page, -1) for i in range(4))

    def put(self, table_row, position, k, v):
        """k, v f64 [kv_heads][hd] at a position."""
        p, s = table_row[position // self.page], position % self.page
        for x, c, b in ((k, self.kc, self.ks), (v, self.vc, self.vs)):
            code, byte = quantise(x)
            c[p, :, s] = pack(code)
            b[p, :, s] = byte

    def get(self, table_row, positions):
        """k, v f64 [positions][kv_heads][hd]."""
        p, s = np.asarray(table_row)[positions // self.page], positions % self.page
        return (values(unpack(self.kc[p, :, s]), self.ks[p, :, s]), values(unpack(self.vc[p, :, s]), self.vs[p, :, s]))

    def randomise(self, rng, sigma=1.0):
        """Normal keys (with strong and weak channels) and values everywhere."""
        gain = np.exp(0.5 * rng.standard_normal((self.kv_heads, 1, self.hd)))
        shape = (self.pages, self.kv_heads, self.page, self.hd)
        for g, c, b in ((gain * sigma, self.kc, self.ks), (sigma, self.vc, self.vs)):
            code, byte = quantise(rng.standard_normal(shape) * g)
            c[...] = pack(code)
            b[...] = byte
        return self


def tables(rng, lengths, page, pages, stride=None):
    """A page table int32 [sequences][stride] of distinct random pages; -1 where none is used."""
    used = [-(-int(n) // page) if n > 0 else 0 for n in lengths]
    stride = stride or max(max(used), 1) + 1
    order = rng.permutation(pages)
    assert sum(used) <= pages
    t = np.full((len(lengths), stride), -1, np.int32)
    at = 0
    for s, n in enumerate(used):
        t[s, :n] = order[at:at + n]
        at += n
    return t


def rotate(x, bias, rope, positions, heads, kv_heads, hd):
    """q, k, v f64 [tokens][...][hd] of q | k | v columns x [tokens][(heads + 2 kv_heads) hd]."""
    x = x.astype(np.float64) + (0.0 if bias is None else bias.astype(np.float64))
    x = x.reshape(len(x), heads + 2 * kv_heads, hd)
    cs = rope.astype(np.float64)[positions][:, None]
    lo, hi = x[:, :heads + kv_heads, :hd // 2], x[:, :heads + kv_heads, hd // 2:]
    with np.errstate(invalid="ignore", over="ignore"):
        qk = np.concatenate([lo * cs[..., 0] - hi * cs[..., 1], lo * cs[..., 1] + hi * cs[..., 0]], -1)
    return qk[:, :heads], qk[:, heads:], x[:, heads + kv_heads:]


def attention(q, k, v, positions, first, window, scale, sinks):
    """q f64 [rows][heads][hd] at `positions` over k, v f64 [n][kv_heads][hd] of positions
    first ..; returns the outputs and, per output, sum p |v| / den (what rounding errors of
    the weights scale with), per row and head the largest sum |q| |k| scale, and per output
    the sum of the |v| that it sees."""
    rows, heads, hd = q.shape
    group = heads // k.shape[1]
    at = first + np.arange(len(k))[None]
    seen = at <= positions[:, None]
    if window:
        seen &= at > positions[:, None] - window
    out = np.zeros(q.shape)
    mag = np.zeros(q.shape)
    smax = np.zeros((rows, heads))
    vsum = np.zeros(q.shape)
    for h in range(heads):
        g = h // group
        with np.errstate(invalid="ignore"):
            s = np.where(seen, q[:, h] @ k[:, g].T * scale, -np.inf)
            smax[:, h] = np.where(seen, np.abs(q[:, h]) @ np.abs(k[:, g]).T * abs(scale), 0.0).max(1)
            m = s.max(1, keepdims=True)
            if sinks is not None:
                m = np.maximum(m, float(sinks[h]))
            m = np.where(np.isneginf(m), 0.0, m)
            p = np.where(seen, np.exp(s - m), 0.0)
            den = p.sum(1, keepdims=True) + (np.exp(float(sinks[h]) - m) if sinks is not None else 0.0)
            vis = seen.any(1)
            if np.isfinite(v[:, g]).all():  # (an unseen value times a weight of 0 is 0)
                n = np.where(vis[:, None], den, 1.0)
                out[:, h], mag[:, h] = p @ v[:, g] / n, p @ np.abs(v[:, g]) / n
                vsum[:, h] = seen @ np.abs(v[:, g])
                continue
            for r in np.nonzero(vis)[0]:
                w, vv = p[r][seen[r]], v[:, g][seen[r]]
                out[r, h] = w @ vv / den[r]
                mag[r, h] = w @ np.abs(vv) / den[r]
                vsum[r, h] = np.abs(vv).sum(0)
    return out, mag, smax, vsum


def bf16_round(x):
    """f32 values of x rounded to bf16 (nearest even), and their bits."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    bits = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return from_bf16(bits), bits


def from_bf16(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def allowance(ref, mag, smax, vsum, n, hd, bf16):
    """How far an output may be from 64 bits.  Scores: hd products summed in f32 in any
    order are off by at most hd 2^-24 of their sum of magnitudes, and the units of log 2 and
    the exponential's own error add 8 roundings of a value of that size; a weight moves by
    twice that (its own and the maximum's).  Weights' and outputs' sums of n terms: n 2^-24
    each, relative to the sum of magnitudes; 32 more roundings for the rest (rescaling, joins,
    the sink, the division).  A bf16 output: the weights in f16 (2^-11) and the output's own
    rounding (2^-8).
    Small weights: a score seen before (once the largest) has its weight held as 2^7, in f16,
    whose smallest step is 2^-24.  What the last f16 plane rounds off is at most half of it,
    2^-25 / 2^7 = 2^-32 of that weight, which is at most 1 of the final sum: 2^-32 |v| for each
    position seen.  (It shows where the large weights meet a v of exactly zero, as one
    in eight E2M1 codes is.)  Below f32's smallest normal value bits of an output may be lost."""
    u = 2.0 ** -24
    floor = 2.0 ** -32 * vsum + 2.0 ** -133
    rel = 2.0 * (hd + 8) * u * smax[..., None] + (2 * n + 32) * u
    if bf16:
        return mag * (rel + 2.0 ** -11) * 1.01 + 2.0 ** -8 * np.abs(ref) * 1.01 + floor
    return mag * (rel + 2.0 ** -22) * 1.01 + floor


def close_allowance(ref, mag, smax, vsum, n, hd, bf16):
    """allowance() for weights that keep f32's range: bf16 planes, each the nearest bf16 of what the
    ones before leave.  A plane leaves at most half a step, 2^-8 of what it takes, so three leave
    2^-24 of a weight (an f32 output) and two 2^-16 (a bf16 one).  Scores, sums and an output's
    own rounding as there.  The largest weight so far is held as 2^-8 at least, and what is held
    below f32's smallest normal value, 2^-126, may be lost: 2^-118 |v| for each position seen."""
    u = 2.0 ** -24
    rel = 2.0 * (hd + 8) * u * smax[..., None] + (2 * n + 32) * u + (2.0 ** -16 if bf16 else 2.0 ** -24)
    return mag * rel * 1.01 + (2.0 ** -8 * np.abs(ref) * 1.01 if bf16 else 0.0) + 2.0 ** -118 * vsum + 2.0 ** -133
