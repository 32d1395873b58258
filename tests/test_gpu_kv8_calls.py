"""PagedKv8::attention where maxima move late, rows have no position, batches are large and calls overlap; bounds as in
tests/kv8_plain.py."""
import numpy as np
import pytest

import gie
from kv8_plain import Cache8, attention, encode, scale_for

pytestmark = pytest.mark.gpu
CACHES = ["int8", "fp8"]


def check(c, **kw):
    got = c.attend(**kw).astype(np.float64)
    want, bound = attention(c, **{k: v for k, v in kw.items() if k in ("scale", "softcap", "window", "sinks")})
    assert np.isfinite(got).all()
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), (float(off.max()), np.argwhere(off > 0)[:4].tolist(), int((off > 0).sum()))
    return got


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("new", [1, 12, 150])
def test_maxima_that_keep_moving(new, dim, cache):
    """Blocks whose keys grow: every block's scores pass all before it by more than FP16 holds, for half of the rows; the
    other half have them fall."""
    c = Cache8([new], [400], heads=4, kv_heads=2, dim=dim, cache=cache, seed=dim + new, spread=0)
    ones = np.ones((1,), np.float32)
    s = np.float32(1 / 64) if cache == "fp8" else np.float32(1 / 100)
    c.k_pages[:] = encode(ones, s, cache)[0]
    for j in range(25):
        c.k_scales[c.table[0, j]] = s * (j + 1) * 16
    c.q[:] = np.abs(c.q) / dim ** 0.5
    c.q[:, ::2] *= -1
    check(c)
    check(c, window=100, sinks=40)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_rows_without_a_position_beside_rows_with_one(dim, cache):
    got = check(Cache8([200, 40], [150, 40], heads=2, kv_heads=1, dim=dim, cache=cache, seed=1))
    assert (got[:50] == 0).all() and (got[50:] != 0).any()
    got = check(Cache8([90], [100], heads=4, kv_heads=1, dim=dim, max_pages=4, cache=cache, seed=2))  # positions 64.. are none
    assert (got[54:] == 0).all()


@pytest.mark.parametrize("batch,dim", [(65, 64), (130, 128), (300, 256)])
def test_many_sequences(batch, dim):
    rng = np.random.default_rng(batch)
    for most in (1, 30):
        new = rng.integers(0, most + 1, batch).tolist()
        lens = [n + int(rng.integers(0, 60)) for n in new]
        check(Cache8(new, lens, heads=4, kv_heads=2, dim=dim, cache=CACHES[most % 2], seed=batch))


@pytest.mark.parametrize("dim", [128, 256])
def test_values_of_very_different_size(dim):
    """Blocks of values 2^20 apart in both directions: what the large ones weigh little and the small ones much."""
    for new in (1, 70):
        c = Cache8([new], [300], heads=4, kv_heads=2, dim=dim, precision="bf16", cache="int8", seed=3)
        for j in range(19):
            c.v_scales[c.table[0, j]] *= np.float32(2.0 ** (20 * (j % 3 - 1)))
        check(c)


def test_calls_on_two_streams_at_once():
    """Calls that share a cache but neither workspace nor output, enqueued together, give what each gives alone."""
    a = Cache8([1] * 3, [3000, 40, 700], dim=128, heads=8, kv_heads=2, page=64, cache="int8", seed=5)
    d = a.device()
    hints = dict(max_new=1, max_len=3000)
    want = a.attend(d=d, **hints)
    p = a.p(**hints)
    size = gie.kv8_attention_workspace_size(p)
    streams = [gie.Stream() for _ in range(2)]
    ws = [gie.DeviceBuffer(size + 16) for _ in streams]
    outs = [a.blank_rows(a.heads) for _ in streams]
    gie.synchronize()
    for _ in range(8):
        for s, w, o in zip(streams, ws, outs):
            gie.kv8_attention(p, d["q"].addr, d["k_pages"].addr, d["v_pages"].addr, d["k_scales"].addr, d["v_scales"].addr,
                              d["starts"].addr, d["lens"].addr, d["table"].addr, o.addr, workspace=w.addr, ws_bytes=size, stream=s)
    gie.synchronize()
    assert all(np.array_equal(a.read_rows(o, a.heads), want) for o in outs)


def test_one_prompt_of_several_rounds():
    """More workgroups than the device holds at once, tiles past the 64 that a wave looks up at once, and sequences that
    share their first pages."""
    c = Cache8([40, 40, 1], [4500, 4500, 4400], heads=4, kv_heads=1, dim=64, page=32, cache="fp8", seed=6)
    c.table[1, :100] = c.table[0, :100]
    check(c)
    check(c, max_new=40, max_len=4500, window=4200, sinks=10)
    c = Cache8([1, 1], [9000, 8000], heads=2, kv_heads=1, dim=64, page=16, cache="int8", seed=7)
    check(c, max_new=1, max_len=64)  # nothing is split: one wave takes more tiles than it looks up at once


def test_scales_for_nothing_and_for_the_largest():
    for cache in CACHES:
        for most in (0.0, 3.3e38):
            c = Cache8([5], [21], heads=2, kv_heads=1, dim=64, precision="bf16", cache=cache, seed=8)
            c.k[:] = most / 4 if most else 0
            c.v[:] = most / 4 if most else 0
            d = c.device()
            gie.kv8_append(c.p(), d["k"].addr, d["v"].addr, d["starts"].addr, d["lens"].addr, d["table"].addr,
                           d["k_pages"].addr, d["v_pages"].addr, d["k_scales"].addr, d["v_scales"].addr)
            k, v = c.blank_rows(1), c.blank_rows(1)
            gie.kv8_read(c.p(), d["k_pages"].addr, d["v_pages"].addr, d["k_scales"].addr, d["v_scales"].addr,
                         d["starts"].addr, d["lens"].addr, d["table"].addr, k.addr, v.addr)
            gie.synchronize()
            scales = d["v_scales"].download(np.float32, c.v_scales.size)
            assert np.isfinite(scales).all() and (scales > 0).all()
            for got, x in ((c.read_rows(k, 1), c.k), (c.read_rows(v, 1), c.v)):
                assert np.isfinite(got).all()
                # half of a step of e4m3 and BF16's rounding (int8's step is smaller)
                assert (np.abs(got - x)[-4:] <= 2.0 ** -4 * np.abs(x)[-4:] * 1.1).all()
    assert scale_for(0, "int8") > 0
