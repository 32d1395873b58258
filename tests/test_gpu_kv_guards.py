"""The appends write the slots of their tokens (and the older codes and the scale of a block whose scale grows) and nothing
else: every other bit of the cache, and the bytes behind each of its buffers, stay as they were, also where q_starts and
seq_lens hold nonsense."""
import numpy as np
import pytest

import gie
from kv8_plain import BLOCK, Cache8
from paged_plain import GUARD, Cache

pytestmark = pytest.mark.gpu
PATTERN = 0x5A
BUFFERS = {"same": ("k_pages", "v_pages"), "int8": ("k_pages", "v_pages", "k_scales", "v_scales")}
BUFFERS["fp8"] = BUFFERS["int8"]


def batch(cache, *args, **kw):
    return Cache(*args, **kw) if cache == "same" else Cache8(*args, cache=cache, **kw)


def image(c, cache, name):
    a = np.ascontiguousarray(getattr(c, name))
    return gie.host_to_storage(a, c.precision).reshape(a.shape) if cache == "same" else a


def guarded(c, cache):
    """The batch on the device, a pattern behind every buffer of the cache."""
    d = c.device()
    for n in BUFFERS[cache]:
        a = image(c, cache, n)
        d[n] = gie.DeviceBuffer(a.nbytes + GUARD)
        d[n].fill(PATTERN)
        d[n].upload(a)
    return d


def places(c, starts, lens):
    """Where each token goes: rows bounded to [0, tokens), positions to the table; (sequence, position) or None."""
    out = []
    for t in range(c.tokens):
        b = max([i for i in range(len(lens)) if starts[i] <= t], default=0)
        first = min(max(starts[b], 0), c.tokens)
        count = min(max(starts[b + 1], first), c.tokens) - first
        position = lens[b] - count + t - first
        there = first <= t < first + count and 0 <= position < c.max_pages * c.page
        out.append((b, position) if there else None)
    return out


def check_writes(c, cache, starts=None, lens=None, norm=True, with_q=True, rotary=0):
    d = guarded(c, cache)
    starts, lens = c.starts.tolist() if starts is None else starts, list(c.lens) if lens is None else lens
    d["starts"].upload(np.array(starts, np.int32))
    d["lens"].upload(np.array(lens, np.int32))
    weight = gie.to_device(np.linspace(0.5, 1.5, c.dim).astype(np.float32))
    tables = [gie.to_device(t) for t in gie.rotary_tables(c.max_pages * c.page, rotary)] if rotary else None
    q_out = c.blank_rows(c.heads)
    gie.synchronize()
    p = c.p(norm_eps=1e-5, rotary_dim=rotary, max_positions=c.max_pages * c.page)
    print("guards", cache, p, starts, lens, flush=True)
    (gie.kv_append_normed if cache == "same" else gie.kv8_append)(
        p, d["k"].addr, d["v"].addr, d["starts"].addr, d["lens"].addr, d["table"].addr, *[d[n].addr for n in BUFFERS[cache]],
        q_norm=weight.addr if norm and with_q else None, k_norm=weight.addr if norm else None,
        cos=tables[0].addr if rotary else None, sin=tables[1].addr if rotary else None,
        q=d["q"].addr if with_q else None, q_out=q_out.addr if with_q else None)
    gie.synchronize()
    c.read_rows(q_out, c.heads)
    written = np.zeros((c.pages, c.page), bool)  # slots that may change
    blocks = np.zeros((c.pages, c.page // BLOCK), bool)
    for place in places(c, starts, lens):
        if place is None:
            continue
        page, slot = c.table[place[0], place[1] // c.page], place[1] % c.page
        if 0 <= page < c.pages:
            blocks[page, slot // BLOCK] = True
            written[page, slot if cache == "same" else slice(slot // BLOCK * BLOCK, slot + 1)] = True
    for n in BUFFERS[cache]:
        before = image(c, cache, n)
        raw = d[n].download(np.uint8, d[n].nbytes)
        assert (raw[before.nbytes:] == PATTERN).all(), "behind " + n
        now = raw[:before.nbytes].view(before.dtype).reshape(before.shape)
        axes, may = ((0, 2, 1), blocks) if n.endswith("scales") else ((0, 2, 1, 3), written)
        same = now.transpose(axes).view(np.uint8 if now.dtype == np.uint8 else f"u{now.itemsize}")
        assert np.array_equal(same[~may], before.transpose(axes).view(same.dtype)[~may]), n


@pytest.mark.parametrize("cache", sorted(BUFFERS))
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_nothing_else_is_written(dim, cache):
    for new, lens in (([1], [1]), ([1] * 7, [1, 16, 17, 31, 32, 33, 100]), ([5, 0, 33, 70], [5, 9, 50, 133])):
        for rotary in (0, dim // 32 * 16, 6):
            check_writes(batch(cache, new, lens, dim=dim, seed=dim), cache, rotary=rotary)
        check_writes(batch(cache, new, lens, dim=dim, page=48, seed=dim), cache, norm=False, with_q=False)


@pytest.mark.parametrize("cache", sorted(BUFFERS))
@pytest.mark.parametrize("starts,lens", [([0, 100, 8], [20, 20]), ([-5, 4, 50], [20, 20]), ([0, 4, 2], [20, 2 ** 31 - 1]),
                                         ([3, 5, 6], [-2 ** 31, 7]), ([8, 8, 8], [20, 20]), ([0, 8, 8], [64, 64]),
                                         ([0, 3, 8], [1, 2])])
def test_nonsense_stays_in_bounds(starts, lens, cache):
    for dim, page in ((64, 16), (128, 32)):
        check_writes(batch(cache, [4, 4], [20, 20], dim=dim, page=page, seed=13), cache, starts, lens, rotary=32)


@pytest.mark.parametrize("cache", sorted(BUFFERS))
def test_pages_that_are_not_there_and_positions_past_the_table(cache):
    c = batch(cache, [3, 40], [100, 60], dim=128, seed=12)
    c.table[0, 6] = -1
    c.table[1, 1] = c.pages
    c.table[1, 3] = 2 ** 31 - 1
    check_writes(c, cache, rotary=128)
    check_writes(batch(cache, [20, 3, 1], [7, 3, 0], dim=64, seed=1), cache)
    check_writes(batch(cache, [20, 40], [70, 30], dim=64, max_pages=4, seed=2), cache)


@pytest.mark.parametrize("cache", ["int8", "fp8"])
def test_reading_calls_leave_the_cache(cache):
    c = Cache8([3, 40], [90, 300], dim=128, cache=cache, seed=3)
    d = guarded(c, cache)
    c.attend(d=d, window=50, sinks=7)
    k, v = c.blank_rows(c.kv), c.blank_rows(c.kv)
    gie.kv8_read(c.p(), *[d[n].addr for n in BUFFERS[cache]], d["starts"].addr, d["lens"].addr, d["table"].addr, k.addr, v.addr)
    gie.synchronize()
    for n in BUFFERS[cache]:
        a = image(c, cache, n)
        raw = d[n].download(np.uint8, d[n].nbytes)
        assert np.array_equal(raw[:a.nbytes], a.reshape(-1).view(np.uint8)) and (raw[a.nbytes:] == PATTERN).all()
