"""PagedKv8::attention under caps past 64, which have kernels of their own, at every head size; blocks of scale NaN beside
sinks; what an append built in steps leaves. Bounds as in tests/kv8_plain.py."""
import numpy as np
import pytest

import gie
from kv8_plain import BLOCK, Cache8, attention

pytestmark = pytest.mark.gpu
CACHES = ["int8", "fp8"]
DIMS = [64, 96, 128, 256]
STEP = ([1] * 9, [1, 2, 15, 16, 17, 63, 64, 65, 300])
CHUNKS = ([5, 0, 33, 130, 1, 64], [5, 9, 140, 133, 301, 64])


def check(c, **kw):
    got = c.attend(**kw).astype(np.float64)
    want, bound = attention(c, **{k: v for k, v in kw.items() if k in ("scale", "softcap", "window", "sinks")})
    assert np.isfinite(got).all()
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), (float(off.max()), np.argwhere(off > 0)[:4].tolist(), int((off > 0).sum()))
    return got


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("new,lens", [STEP, CHUNKS], ids=["step", "chunks"])
def test_large_caps(new, lens, dim, cache):
    """Scores well inside the cap (the polynomial), and of its size and past it (the exponential), of either sign."""
    for i, (softcap, size) in enumerate(((65.0, 1), (100.0, 16), (1000.0, 1))):
        c = Cache8(new, lens, dim=dim, precision=("fp16", "bf16")[i % 2], cache=cache, seed=dim + i)
        c.q *= np.float32(size)
        check(c, softcap=softcap)
        check(c, softcap=softcap, window=70, sinks=5)
        check(c, softcap=softcap, scale=-0.3 * dim ** -0.5)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("new", [1, 130])
def test_large_caps_of_parts_that_are_joined(new, dim, cache):
    c = Cache8([new, 3], [3000, 50], dim=dim, heads=2, kv_heads=1, page=48, precision="bf16", seed=new, cache=cache)
    c.q *= 8
    for hints in (dict(max_new=new, max_len=3000), dict()):
        check(c, softcap=100.0, **hints)
    check(c, softcap=100.0, window=1500, sinks=64, max_new=new, max_len=3000)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", DIMS)
def test_negative_scales_at_every_size(dim, cache):
    for new, lens in (STEP, CHUNKS):
        c = Cache8(new, lens, dim=dim, cache=cache, seed=dim)
        check(c, scale=-0.7 * dim ** -0.5)
        check(c, scale=-0.7 * dim ** -0.5, softcap=9.0)


# ------------------------------------------------------------------------------------------------- scales that are NaN
def sees(position, j, window, sinks):
    return j <= position and (not window or j > position - window or j < sinks)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(30, 5), (100, 40), (64, 16), (17, 1)])
@pytest.mark.parametrize("new,lens", [([1, 1], [300, 171]), ([9, 1], [300, 240]), ([70, 33], [400, 300])])
def test_blocks_between_sinks_and_window_never_show(new, lens, window, sinks, dim, cache):
    """Every block that no row sees has scale NaN and codes of all ones: the rest of the last sinks' tile, what lies
    between, and the granule before the window."""
    c = Cache8(new, lens, dim=dim, page=32, cache=cache, seed=window)
    want, bound = attention(c, window=window, sinks=sinks)
    visible = np.zeros((c.pages, c.page // BLOCK), bool)
    for b, (n, length) in enumerate(zip(new, lens)):
        for j in range(length):
            if any(sees(p, j, window, sinks) for p in range(length - n, length)):
                visible[c.table[b, j // c.page], j % c.page // BLOCK] = True
    assert (~visible[c.table[0, :lens[0] // c.page]]).sum() >= 8  # a real gap
    for n in "kv":
        getattr(c, n + "_scales").transpose(0, 2, 1)[~visible] = np.nan
        pages = getattr(c, n + "_pages").reshape(c.pages, c.kv, -1, BLOCK, c.dim).transpose(0, 2, 1, 3, 4)
        pages[~visible] = 0x7f
    for hints in (dict(), dict(max_new=max(new), max_len=max(lens))):
        got = c.attend(window=window, sinks=sinks, **hints)
        assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(30, 5), (100, 40)])
@pytest.mark.parametrize("new,length", [(1, 300), (9, 300), (150, 400)])
def test_nan_scales_beside_sinks_reach_only_rows_that_see_their_block(new, length, window, sinks, dim, cache):
    first = length - new
    for where in "kv":
        for at in (0, sinks // BLOCK * BLOCK + BLOCK, max(0, first - window - 16), max(0, first - window + 1), first):
            c = Cache8([new], [length], heads=4, kv_heads=2, dim=dim, cache=cache, seed=at)
            want, bound = attention(c, window=window, sinks=sinks)
            getattr(c, where + "_scales")[c.table[0, at // c.page], 1, at % c.page // BLOCK] = np.nan
            got = c.attend(window=window, sinks=sinks)
            block = range(at // BLOCK * BLOCK, at // BLOCK * BLOCK + BLOCK)
            hit = np.array([any(sees(p, j, window, sinks) for j in block) for p in range(first, length)])
            ok = np.abs(got - want) <= bound
            assert ok[~hit].all() and ok[:, :2].all()  # the other key head too
            assert np.isnan(got[hit][:, 2:]).all()


# ------------------------------------------------------------------------------------------------- appends in steps
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("chunks", [[64, 33], [1, 30, 1, 1, 17, 2, 64, 1, 5], [1] * 40])
def test_every_value_is_off_by_its_own_roundings(chunks, cache):
    """A value is rounded when it is written, and again for each later chunk that writes into its block of 16, if the
    scale grows then. int8: half of the last scale each. e4m3: the first rounding 2^-4 of the value or half of the
    smallest step, and a growth moves it exactly unless it falls among the subnormals, where it is half of the smallest
    step. Then the read's rounding, and 2^-12 of all that for FP32."""
    kw = dict(heads=2, kv_heads=2, dim=64, page=32, precision="bf16", cache=cache, max_pages=4)
    c = Cache8([1], [1], seed=6, **kw)
    c.table[0] = [2, 0, 3, 1]
    d, kept, length = c.device(), {"k": [], "v": []}, 0
    roundings = np.zeros(sum(chunks), int)
    rng = np.random.default_rng(7)
    for n in chunks:
        e = Cache8([n], [length + n], seed=int(rng.integers(1 << 30)), **kw)
        size = np.float32(2.0 ** rng.integers(-2, 4))
        for name in "kv":
            setattr(e, name, getattr(e, name) * size)  # exact in BF16
            kept[name].append(getattr(e, name))
            d[name] = e.rows(getattr(e, name))
        d["starts"].upload(e.starts)
        d["lens"].upload(np.array([length + n], np.int32))
        gie.kv8_append(e.p(num_pages=c.pages), d["k"].addr, d["v"].addr, d["starts"].addr, d["lens"].addr, d["table"].addr,
                       *[d[x].addr for x in ("k_pages", "v_pages", "k_scales", "v_scales")])
        gie.synchronize()
        roundings[length // BLOCK * BLOCK:length + n] += 1
        length += n
    whole = Cache8([length], [length], seed=6, **kw)
    d["starts"].upload(whole.starts)
    rows = [whole.blank_rows(2) for _ in range(2)]
    gie.kv8_read(whole.p(num_pages=c.pages), *[d[x].addr for x in ("k_pages", "v_pages", "k_scales", "v_scales")],
                 d["starts"].addr, d["lens"].addr, d["table"].addr, *[r.addr for r in rows])
    gie.synchronize()
    at, count = np.arange(length), roundings[:, None, None]
    for name, r in zip("kv", rows):
        x = np.concatenate(kept[name]).astype(np.float64)
        s = d[name + "_scales"].download(np.float32, c.k_scales.size).reshape(c.k_scales.shape)
        s = s[c.table[0, at // 32], :, at % 32 // BLOCK].astype(np.float64)[..., None]
        off = 0.5 * s * count if cache == "int8" else np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s) + 2.0 ** -10 * s * (count - 1)
        got = whole.read_rows(r, 2)
        assert (np.abs(got - x) <= (off + 2.0 ** -8 * (np.abs(x) + off)) * (1 + 2.0 ** -12)).all()
