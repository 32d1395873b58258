"""Plain numpy forms in 64 bits of the paged cache in 8 bits, of head norms in the append and of windows with sinks, and
device copies of their inputs, for the tests."""
import numpy as np

import gie
from paged_plain import GUARD, TINY, UNIT, Cache

BLOCK, LEAST = 16, 2.0 ** -64


def e4m3_values():
    """What the 256 codes stand for; the two that stand for a NaN count as 480."""
    code = np.arange(256)
    power, fraction = (code >> 3) & 15, code & 7
    value = np.where(power == 0, fraction * 2.0 ** -9, (8 + fraction) * 2.0 ** (power - 10.0))
    return np.where(code >= 128, -value, value)


E4M3 = e4m3_values()


def decode(codes, cache):
    return codes.view(np.int8).astype(np.float64) if cache == "int8" else E4M3[codes]


def encode_e4m3(y):
    """Nearest code, ties to even, of values within 448 (numpy's rint rounds ties to even steps, and an even step is an
    even last bit)."""
    a = np.abs(y)
    power = np.floor(np.log2(np.maximum(a, 2.0 ** -6)))
    power = np.where(np.exp2(power) > np.maximum(a, 2.0 ** -6), power - 1, power)
    step = np.exp2(power - 3)
    value = np.rint(a / step) * step
    code = np.searchsorted(E4M3[:127], value).astype(np.uint8)
    assert np.array_equal(E4M3[code], value)
    return np.where(np.signbit(y), code | 128, code).astype(np.uint8)


def scale_for(most, cache):
    """In FP32, as the library defines it."""
    most = np.maximum(np.asarray(most, np.float32), np.float32(LEAST))
    if cache == "int8":
        return (most / np.float32(127)).astype(np.float32)
    mantissa, power = np.frexp(most.astype(np.float64))  # 448 = 0.875 2^9
    return np.ldexp(1.0, power - 9 + (mantissa > 0.875)).astype(np.float32)


def encode(x, scale, cache):
    """Codes of FP32 values under FP32 scales, with the library's steps: one quotient in FP32, one rounding."""
    y = x.astype(np.float32) / scale.astype(np.float32)
    if cache == "int8":
        return np.rint(np.clip(y, -127, 127)).astype(np.int8).view(np.uint8)
    return encode_e4m3(np.clip(y.astype(np.float64), -448, 448))


class Cache8(Cache):
    """A batch over 8-bit pages: blocks of sizes that differ by orders of magnitude, older values in every slot."""

    def __init__(self, *args, cache="int8", spread=1.0, **kw):
        super().__init__(*args, **kw)
        self.cache = cache
        self.problem = dict(self.problem, cache=cache)
        shape = (self.pages, self.kv, self.page // BLOCK, BLOCK, self.dim)
        for n in ("k", "v"):
            size = np.exp(spread * self.rng.normal(size=shape[:3]))[..., None, None]
            x = (self.rng.normal(size=shape) * size).astype(np.float32)
            scale = scale_for(np.abs(x).max((3, 4)), cache)
            setattr(self, n + "_scales", scale)
            setattr(self, n + "_pages", encode(x, scale[..., None, None], cache).reshape(self.pages, self.kv, self.page, self.dim))

    def values_of(self, name):
        scale = np.repeat(getattr(self, name + "_scales").astype(np.float64), BLOCK, axis=2)
        return decode(getattr(self, name + "_pages"), self.cache) * scale[..., None]

    def device(self):
        d = {"q": self.rows(self.q), "k": self.rows(self.k), "v": self.rows(self.v)}
        for n in ("k_pages", "v_pages", "k_scales", "v_scales"):
            d[n] = gie.to_device(np.ascontiguousarray(getattr(self, n)), extra=GUARD)
        d["starts"] = gie.to_device(self.starts)
        d["lens"] = gie.to_device(np.array(self.lens, np.int32))
        d["table"] = gie.to_device(self.table)
        return d

    def attend(self, d=None, stream=None, **more):
        d = d or self.device()
        p = self.p(**more)
        size = gie.kv8_attention_workspace_size(p)
        ws, out = gie.DeviceBuffer(size + GUARD), self.blank_rows(self.heads)
        ws.fill(0xFF)  # NaN in every type
        gie.synchronize()
        print("attend8", p, self.new[:8], self.lens[:8], flush=True)
        at = 2 * self.offset
        gie.kv8_attention(p, d["q"].addr + at, d["k_pages"].addr, d["v_pages"].addr, d["k_scales"].addr,
                          d["v_scales"].addr, d["starts"].addr, d["lens"].addr, d["table"].addr, out.addr + at,
                          workspace=ws.addr, ws_bytes=size, stream=stream)
        gie.synchronize()
        assert (ws.download(np.uint8, GUARD, offset=size) == 0xFF).all(), "written past the workspace"
        return self.read_rows(out, self.heads)


def position_of(c):
    """Sequence, position and whether it is valid, of every row."""
    seq = np.repeat(np.arange(len(c.new)), c.new)
    position = np.concatenate([length - n + np.arange(n) for n, length in zip(c.new, c.lens)] or [np.zeros(0)]).astype(np.int64)
    return seq, position, (position >= 0) & (position < c.max_pages * c.page)


def attention(c, scale=None, softcap=0.0, window=0, sinks=0):
    """The attention in 64 bits and a bound for each output value.

    Scores: exact products summed in FP32, off by (D + 4) 2^-24 sum |q k|. In 8 bits the code is exact, the row of q goes to
    FP16 under a power of 2 that puts its largest value into 2^14 .. 2^15, so a value is off by at most 2^-39 of that one
    (D 2^-39 max|q| max|k| for the sum), and three more factors in FP32 come on top: (D + 8) 2^-24. A cap doubles that
    and adds 2^-20 of itself. Weights: exp of it, relative 4 e + 2^-16 (the exponent's own rounding at magnitudes up to
    256, and in 8 bits log2 of a block's scale, at most 80, off by 2^-23 of it), rounded once: to the tokens' type, or in
    8 bits to FP16 together with the block's scale: 2^-11, and half of FP16's smallest step, 2^-25, where the largest
    weight times scale lies at 2^7 or above. The sums over n keys 2^-23 n. The output rounds once more."""
    in_8 = isinstance(c, Cache8)
    scale = c.dim ** -0.5 if scale is None else scale
    k_all, v_all = (c.values_of("k"), c.values_of("v")) if in_8 else (c.k_pages.astype(np.float64), c.v_pages.astype(np.float64))
    out = np.zeros((c.tokens, c.heads, c.dim))
    bound = np.full_like(out, TINY[c.precision])
    u = UNIT[c.precision]
    group = c.heads // c.kv
    seq, position, valid = position_of(c)
    for t in np.flatnonzero(valid):
        pos = position[t]
        keys = np.arange(pos + 1)
        if window:
            keys = keys[(keys > pos - window) | (keys < sinks)]
        page, slot = c.table[seq[t], keys // c.page], keys % c.page
        ok = (page >= 0) & (page < c.pages)
        page = np.where(ok, page, 0)
        k = (k_all[page, :, slot] * ok[:, None, None]).transpose(1, 2, 0)  # [kv][dim][keys]
        v = (v_all[page, :, slot] * ok[:, None, None]).transpose(1, 0, 2)  # [kv][keys][dim]
        q = c.q[t].astype(np.float64).reshape(c.kv, group, c.dim)
        s = (q @ k) * scale
        e = ((c.dim + 8) * 2.0 ** -24 * (np.abs(q) @ np.abs(k)).max(2) +
             (c.dim * 2.0 ** -39 * np.abs(q).max(2) * np.abs(k).max((1, 2))[:, None] if in_8 else 0)) * abs(scale)
        if softcap:
            s = softcap * np.tanh(s / softcap)
            e = 2 * e + 2.0 ** -20 * softcap
        w = np.exp(s - s.max(2, keepdims=True))
        w /= w.sum(2, keepdims=True)
        o, size = w @ v, w @ np.abs(v)
        rel = (2.0 ** -11 if in_8 else u) + 4 * e[..., None] + 2.0 ** -16 + len(keys) * 2.0 ** -23
        if in_8:
            vs = c.v_scales[page, :, slot // BLOCK].astype(np.float64).T * ok  # [kv][keys]
            codes = np.abs(v) / np.maximum(vs, 1e-300)[..., None]
            small = 2.0 ** -32 * (w * vs[:, None]).max(2)[..., None] * codes.sum(1)[:, None]
        else:
            small = TINY[c.precision] * 2 ** 8 * np.abs(v).sum(1)[:, None]
        inner = rel * size + small
        out[t] = o.reshape(c.heads, c.dim)
        bound[t] += (inner + u * (np.abs(o) + inner)).reshape(c.heads, c.dim)
    return out, bound


def turned(c, x, weight, eps, rotary, interleaved, cos, sin):
    """Rows of x normed (weight not None) and rotated in 64 bits, and how far FP32 may be off before its last rounding: the
    norm's sum of D squares, root, quotient and two products (D / 2 + 8) 2^-24, the rotation 4 2^-24 of |u| + |v|."""
    x = x.astype(np.float64)
    slack = np.zeros_like(x)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
        slack = (c.dim / 2 + 8) * 2.0 ** -24 * np.abs(x)
    _, position, valid = position_of(c)
    y, off = x.copy(), slack.copy()
    half = rotary // 2
    if half:
        a, b = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, half), slice(half, rotary))
        at = np.where(valid, position, 0)
        cs, sn = cos[at][:, None].astype(np.float64), sin[at][:, None].astype(np.float64)
        u, w = x[..., a], x[..., b]
        y[..., a], y[..., b] = u * cs - w * sn, u * sn + w * cs
        turn = 4 * 2.0 ** -24
        off[..., a] = slack[..., a] * np.abs(cs) + slack[..., b] * np.abs(sn) + turn * (np.abs(u * cs) + np.abs(w * sn))
        off[..., b] = slack[..., a] * np.abs(sn) + slack[..., b] * np.abs(cs) + turn * (np.abs(u * sn) + np.abs(w * cs))
    y[~valid], off[~valid] = 0, 0
    return y, off
