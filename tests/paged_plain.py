"""Plain numpy forms of the paged cache's operators in 64 bits, and device copies of their inputs, for the tests."""
import numpy as np

import gie
import oracle as O

UNIT = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"fp16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half a smallest step
GUARD = 256


class Cache:
    """A batch: `new` and `lens` (new ones counted) of each sequence, scattered pages, every slot holding older values
    (or `stale`), rows of q, k, v that stand `gap` elements further apart than they are long."""

    def __init__(self, new, lens, heads=4, kv_heads=2, dim=64, page=16, precision="fp16", seed=0, gap=0, offset=0,
                 max_pages=None, stale=None, extra_pages=3, **problem):
        self.new, self.lens, self.heads, self.kv, self.dim, self.page = list(new), list(lens), heads, kv_heads, dim, page
        self.precision, self.gap, self.offset = precision, gap, offset
        rng = self.rng = np.random.default_rng(seed)
        need = [-(-max(n, 0) // page) for n in self.lens]
        self.max_pages = max_pages or max(1, max(need))
        need = [min(n, self.max_pages) for n in need]
        self.pages = sum(need) + extra_pages
        order, at = rng.permutation(self.pages), 0
        self.table = rng.integers(0, self.pages, (len(need), self.max_pages)).astype(np.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.tokens = sum(self.new)
        self.starts = np.cumsum([0] + self.new).astype(np.int32)
        self.q = self.values((self.tokens, heads, dim))
        self.k = self.values((self.tokens, kv_heads, dim))
        self.v = self.values((self.tokens, kv_heads, dim))
        shape = (self.pages, kv_heads, page, dim)
        self.k_pages, self.v_pages = self.values(shape), self.values(shape)
        if stale is not None:
            used = np.zeros((self.pages, page), bool)
            for b, n in enumerate(self.lens):
                for j in range(min(n, self.max_pages * page)):
                    used[self.table[b, j // page], j % page] = True
            for pages in (self.k_pages, self.v_pages):
                pages.transpose(0, 2, 1, 3)[~used] = stale
        self.problem = problem

    def values(self, shape):
        return O.quantize(self.precision, self.rng.normal(size=shape).astype(np.float32)).reshape(shape)

    def p(self, **more):
        q, kv = self.heads * self.dim + self.gap, self.kv * self.dim + self.gap
        return gie.PagedKv(**{**dict(batch=len(self.new), total_tokens=self.tokens, q_heads=self.heads, kv_heads=self.kv,
                                     head_dim=self.dim, page_size=self.page, num_pages=self.pages,
                                     max_pages=self.max_pages, precision=self.precision, q_stride=q, k_stride=kv,
                                     v_stride=kv, o_stride=q), **self.problem, **more})

    def rows(self, a):
        """Device copy of [tokens][heads][dim] with the gap behind every row and the offset before the first."""
        a = gie.host_to_storage(a, self.precision).reshape(a.shape[0], -1)
        flat = np.full(self.offset + a.shape[0] * (a.shape[1] + self.gap) + GUARD, 0xA5A5, np.uint16)
        flat[self.offset:self.offset + a.shape[0] * (a.shape[1] + self.gap)].reshape(a.shape[0], -1)[:, :a.shape[1]] = a
        return gie.to_device(flat)

    def blank_rows(self, heads):
        n = self.offset + self.tokens * (heads * self.dim + self.gap) + GUARD
        d = gie.DeviceBuffer(2 * n)
        d.fill(0xA5)
        return d

    def read_rows(self, d, heads):
        """The rows of a device buffer as floats; whatever surrounds them must still be poison."""
        raw = d.download(np.uint16, d.nbytes // 2)
        row = heads * self.dim + self.gap
        body = raw[self.offset:self.offset + self.tokens * row].reshape(self.tokens, row)
        assert (raw[:self.offset] == 0xA5A5).all() and (raw[self.offset + self.tokens * row:] == 0xA5A5).all()
        assert (body[:, heads * self.dim:] == 0xA5A5).all(), "written between the rows"
        return gie.storage_to_float(np.ascontiguousarray(body[:, :heads * self.dim]).reshape(-1), self.precision).reshape(
            self.tokens, heads, self.dim)

    def device(self):
        d = {"q": self.rows(self.q), "k": self.rows(self.k), "v": self.rows(self.v)}
        for n in ("k_pages", "v_pages"):
            d[n] = gie.to_device(gie.host_to_storage(getattr(self, n), self.precision))
        d["starts"] = gie.to_device(self.starts)
        d["lens"] = gie.to_device(np.array(self.lens, np.int32))
        d["table"] = gie.to_device(self.table)
        return d

    def attend(self, d=None, stream=None, **more):
        d = d or self.device()
        p = self.p(**more)
        size = gie.paged_attention_workspace_size(p)
        ws, out = gie.DeviceBuffer(size + GUARD), self.blank_rows(self.heads)
        ws.fill(0xFF)  # NaN in every type
        gie.synchronize()
        print("attend", p, self.new[:8], self.lens[:8], flush=True)
        at = 2 * self.offset
        gie.paged_attention(p, d["q"].addr + at, d["k_pages"].addr, d["v_pages"].addr, d["starts"].addr, d["lens"].addr,
                            d["table"].addr, out.addr + at, workspace=ws.addr, ws_bytes=size, stream=stream)
        gie.synchronize()
        assert (ws.download(np.uint8, GUARD, offset=size) == 0xFF).all(), "written past the workspace"
        return self.read_rows(out, self.heads)

    def plain(self, scale=None, softcap=0.0, window=0):
        """The attention in 64 bits and a bound for each output value.

        A score is a sum of exact products in FP32: off by at most (D + 4) 2^-24 sum|scale q k| =: e, capped scores by
        twice that and 2^-20 of the cap more. A weight is exp(score - m) with m within the scores: relative error 2 e (its own
        and m's, which cancels in the quotient only where it is the same) plus 2^-20 for exp2 and its argument, which
        reaches 128 in magnitude where it matters; it is rounded once to the storage type (u, and half its smallest
        step at a magnitude not under 2^-8 of the largest). Both sums run in FP32 over n terms (n 2^-24 each). The
        output rounds once more."""
        scale = self.dim ** -0.5 if scale is None else scale
        out = np.zeros((self.tokens, self.heads, self.dim))
        bound = np.full_like(out, TINY[self.precision])
        u, group, capacity = UNIT[self.precision], self.heads // self.kv, self.max_pages * self.page
        for b, (n, length) in enumerate(zip(self.new, self.lens)):
            for i in range(n):
                pos = length - n + i
                if pos < 0 or pos >= capacity:
                    continue
                keys = np.arange(max(0, pos - window + 1) if window else 0, pos + 1)
                page, slot = self.table[b, keys // self.page], keys % self.page
                ok = (page >= 0) & (page < self.pages)
                page = np.where(ok, page, 0)
                k = self.k_pages[page, :, slot].astype(np.float64) * ok[:, None, None]
                v = self.v_pages[page, :, slot].astype(np.float64) * ok[:, None, None]
                t = self.starts[b] + i
                for h in range(self.heads):
                    q = self.q[t, h].astype(np.float64)
                    s = (k[:, h // group] @ q) * scale
                    e = (self.dim + 4) * 2.0 ** -24 * (np.abs(k[:, h // group]) @ np.abs(q)).max() * abs(scale)
                    if softcap:
                        s = softcap * np.tanh(s / softcap)
                        e = 2 * e + 2.0 ** -20 * softcap
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    o = w @ v[:, h // group]
                    size = w @ np.abs(v[:, h // group])
                    out[t, h] = o
                    rel = u + 4 * e + 2.0 ** -18 + len(keys) * 2.0 ** -23
                    small = TINY[self.precision] * 2 ** 8 * np.abs(v[:, h // group]).sum(0)
                    inner = rel * size + small
                    bound[t, h] += inner + u * (np.abs(o) + inner)
        return out, bound

    def rotate(self, x, rotary, interleaved, cos, sin):
        """Rows of x turned by their positions in 64 bits, zero without a valid position; and the positions."""
        half = rotary // 2
        y = x.astype(np.float64).copy()
        position = np.empty(self.tokens, np.int64)
        for b, (n, length) in enumerate(zip(self.new, self.lens)):
            position[self.starts[b]:self.starts[b] + n] = length - n + np.arange(n)
        placed = (position >= 0) & (position < self.max_pages * self.page)
        if half:
            a, c = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, half), slice(half, rotary))
            at = np.where(placed, position, 0)
            cs, sn = cos[at][:, None].astype(np.float64), sin[at][:, None].astype(np.float64)
            u, w = x[..., a].astype(np.float64), x[..., c].astype(np.float64)
            y[..., a], y[..., c] = u * cs - w * sn, u * sn + w * cs
        y[~placed] = 0
        return y, position, placed
