"""PagedKv8 on the GPU against plain numpy in 64 bits (tests/kv8_plain.py, which also derives the bounds): append into and
read out of a paged cache in 8 bits with a scale for each block of 16 positions and head, and attention over it."""
import numpy as np
import pytest

import gie
from kv8_plain import BLOCK, E4M3, Cache8, attention, decode, encode, encode_e4m3, position_of, scale_for, turned
from paged_plain import TINY, UNIT

pytestmark = pytest.mark.gpu
CACHES = ["int8", "fp8"]

APPENDS = {"one": ([1], [1]), "step": ([1] * 7, [1, 16, 17, 31, 32, 33, 100]), "chunks": ([5, 0, 33, 70], [5, 9, 50, 133])}


def append(c, d, rotary=0, interleaved=False, cos=None, sin=None, q_norm=None, k_norm=None, eps=1e-5, with_q=True,
           in_place=False, stream=None, **more):
    """The call; returns the device buffer of the turned q."""
    dev = {n: gie.to_device(a) for n, a in (("cos", cos), ("sin", sin), ("q_norm", q_norm), ("k_norm", k_norm)) if a is not None}
    p = c.p(rotary_dim=rotary, interleaved=interleaved, max_positions=c.max_pages * c.page, norm_eps=eps, **more)
    q_out = d["q"] if in_place else c.blank_rows(c.heads)
    gie.synchronize()
    print("append8", p, c.new[:8], c.lens[:8], flush=True)
    at = 2 * c.offset
    gie.kv8_append(p, d["k"].addr + at, d["v"].addr + at, d["starts"].addr, d["lens"].addr, d["table"].addr,
                   d["k_pages"].addr, d["v_pages"].addr, d["k_scales"].addr, d["v_scales"].addr,
                   q=d["q"].addr + at if with_q else None, q_out=q_out.addr + at if with_q else None,
                   **{n: b.addr for n, b in dev.items()}, stream=stream)
    gie.synchronize()
    return q_out


def cache_of(c, d):
    """Codes and scales on the device, and that nothing behind them was written."""
    got = {}
    for n in ("k", "v"):
        got[n + "_pages"] = d[n + "_pages"].download(np.uint8, c.k_pages.size).reshape(c.k_pages.shape)
        got[n + "_scales"] = d[n + "_scales"].download(np.float32, c.k_scales.size).reshape(c.k_scales.shape)
    return got


def check_append(c, rotary, interleaved, norm=True, **kw):
    """Stored values lie within half a step of the formula's (int8: half a scale; e4m3: 2^-4 of the value or half of the
    smallest step), the scale follows the largest one, older codes of a block move only if its scale does and then by at
    most half a step, everything else keeps its bits."""
    d = c.device()
    rng = np.random.default_rng(rotary + 1)
    cos, sin = (rng.uniform(-1, 1, (c.max_pages * c.page, rotary // 2)).astype(np.float32) for _ in range(2))
    weights = [rng.uniform(0.5, 1.5, c.dim).astype(np.float32) if norm else None for _ in range(2)]
    with_q = kw.get("with_q", True)
    turn = dict(eps=1e-5, rotary=rotary, interleaved=interleaved, cos=cos, sin=sin)
    q_out = append(c, d, q_norm=weights[0] if with_q else None, k_norm=weights[1], **turn, **kw)
    if with_q:
        want, off = turned(c, c.q, weights[0], **turn)
        off = off + UNIT[c.precision] * (np.abs(want) + off) + 2.0 ** -25
        assert (np.abs(c.read_rows(q_out, c.heads) - want) <= off).all()
    now = cache_of(c, d)
    seq, position, valid = position_of(c)
    page = np.where(valid, c.table[seq, np.clip(position // c.page, 0, c.max_pages - 1)], -1) if c.tokens else np.zeros(0, int)
    stored = (page >= 0) & (page < c.pages)
    touched = np.zeros((c.pages, c.page), bool)
    touched[page[stored], position[stored] % c.page] = True
    blocks = touched.reshape(c.pages, -1, BLOCK).any(2)
    for n, x, w in (("k", c.k, weights[1]), ("v", c.v, None)):
        want, off = turned(c, x, w, **turn) if n == "k" else (x.astype(np.float64), np.zeros(x.shape))
        before, before_scale = getattr(c, n + "_pages"), getattr(c, n + "_scales")
        codes, scales = now[n + "_pages"], now[n + "_scales"]
        # untouched blocks, and slots behind the new ones
        grid = np.repeat(blocks, BLOCK, axis=1)
        last = np.zeros((c.pages, c.page), bool)
        for pg, bl in np.argwhere(blocks):
            new = np.flatnonzero(touched[pg, bl * BLOCK:(bl + 1) * BLOCK])
            last[pg, bl * BLOCK + new.max() + 1:(bl + 1) * BLOCK] = True
        keep = ~grid | last
        assert np.array_equal(codes.transpose(0, 2, 1, 3)[keep], before.transpose(0, 2, 1, 3)[keep]), "other slots"
        assert np.array_equal(scales.transpose(0, 2, 1)[~blocks], before_scale.transpose(0, 2, 1)[~blocks]), "other scales"
        for pg, bl in np.argwhere(blocks):
            slots = np.arange(bl * BLOCK, (bl + 1) * BLOCK)
            rows = np.flatnonzero(stored & (page == pg) & (position % c.page // BLOCK == bl))
            first = (position[rows] % BLOCK).min()
            for h in range(c.kv):
                y, tol = want[rows, h], off[rows, h]
                most, slack = np.abs(y).max(), tol.max()
                old = before_scale[pg, h, bl] if first else np.float32(0)
                s = float(scales[pg, h, bl])
                low, high = (max(float(scale_for(m, c.cache)), float(old)) for m in (max(most - slack, 0), most + slack))
                assert low * (1 - 2.0 ** -22) <= s <= high * (1 + 2.0 ** -22), (s, low, high)
                got = decode(codes[pg, h, slots], c.cache) * s
                half = 0.5 * s * (1 + 2.0 ** -14) if c.cache == "int8" else \
                    np.maximum(2.0 ** -4 * (np.abs(y) + tol), 2.0 ** -10 * s) * (1 + 2.0 ** -14)
                assert (np.abs(got[position[rows] % BLOCK] - y) <= half + tol).all()
                was = decode(before[pg, h, slots[:first]], c.cache) * float(before_scale[pg, h, bl])
                if first and s == old:
                    assert np.array_equal(codes[pg, h, slots[:first]], before[pg, h, slots[:first]])
                elif first:
                    half = 0.5 * s * (1 + 2.0 ** -14) if c.cache == "int8" else np.maximum(2.0 ** -4 * np.abs(was), 2.0 ** -10 * s)
                    assert (np.abs(got[:first] - was) <= half).all()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 0), (96, 64), (128, 128), (128, 32), (256, 256), (128, 6), (96, 96), (64, 2)])
def test_append(dim, rotary, interleaved, cache):
    for i, batch in enumerate(sorted(APPENDS)):
        for norm in (False, True):
            check_append(Cache8(*APPENDS[batch], dim=dim, precision=("fp16", "bf16")[(i + norm) % 2], cache=cache,
                                seed=rotary), rotary, interleaved, norm)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads,kv_heads,page", [(1, 1, 16), (3, 3, 48), (32, 8, 64), (5, 1, 32), (40, 8, 16)])
def test_append_heads_and_pages(heads, kv_heads, page, cache):
    check_append(Cache8([3, 40], [9, 100], heads=heads, kv_heads=kv_heads, dim=128, page=page, cache=cache, seed=heads), 128, False)
    check_append(Cache8([3, 40], [9, 100], heads=heads, kv_heads=kv_heads, dim=128, page=page, cache=cache, seed=heads),
                 128, True, with_q=False)


@pytest.mark.parametrize("gap,offset", [(8, 0), (3, 0), (0, 1), (5, 7), (64, 8)])
@pytest.mark.parametrize("in_place", [False, True])
def test_append_strides_and_alignment(gap, offset, in_place):
    for interleaved, cache in ((False, "int8"), (True, "fp8")):
        for dim, rotary in ((96, 64), (64, 6)):
            check_append(Cache8(*APPENDS["chunks"], dim=dim, gap=gap, offset=offset, cache=cache, seed=gap), rotary,
                         interleaved, in_place=in_place)


@pytest.mark.parametrize("cache", CACHES)
def test_append_without_room(cache):
    check_append(Cache8([20, 3, 1], [7, 3, 0], dim=64, seed=1, cache=cache), 64, False)
    check_append(Cache8([20, 40], [70, 30], dim=64, max_pages=4, seed=2, cache=cache), 32, True)
    c = Cache8([3, 40], [100, 60], dim=128, seed=12, cache=cache)
    c.table[0, 6] = -1
    c.table[1, 1] = c.pages
    c.table[1, 3] = 2 ** 31 - 1
    check_append(c, 128, False, stream=gie.Stream())


@pytest.mark.parametrize("batch", [65, 130, 4100])
def test_append_many_sequences(batch):
    rng = np.random.default_rng(batch)
    new = rng.integers(0, 3, batch).tolist()
    lens = [n + int(rng.integers(0, 20)) for n in new]
    check_append(Cache8(new, lens, heads=2, kv_heads=1, dim=64, seed=batch, cache=CACHES[batch % 2]), 64, False)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("precision", ["fp16", "bf16"])
def test_append_codes_bit_for_bit(cache, precision):
    """Without a norm and a rotation every step is one FP32 operation that numpy has too: equal scales and codes. Token by
    token, so that a block's scale grows several times."""
    page, lens = 32, 45
    c = Cache8([1], [1], heads=2, kv_heads=2, dim=64, page=page, precision=precision, cache=cache, max_pages=2, seed=3)
    d = c.device()
    codes = {n: getattr(c, n + "_pages").copy() for n in ("k_pages", "v_pages") for n in (n[0],)}
    scales = {n: getattr(c, n + "_scales").copy() for n in "kv"}
    for position in range(lens):
        rows = {n: gie.storage_to_float(gie.host_to_storage(
            (c.rng.normal(size=(1, 2, 64)) * np.exp(c.rng.normal())).astype(np.float32), precision), precision).reshape(1, 2, 64)
            for n in "kv"}
        if position == 20:
            rows["k"][:] = 0
        if position == 33:
            rows["v"][0, 1, 5] = 448.0 * 2  # a value that is the border of a power of 2
        for n in "kv":
            setattr(c, n, rows[n])
            d[n] = c.rows(rows[n])
        d["lens"].upload(np.array([position + 1], np.int32))
        c.lens = [position + 1]
        append(c, d)
        pg, slot = c.table[0, position // page], position % page
        block, first = slot // BLOCK, slot % BLOCK
        for n in "kv":
            for h in range(2):
                new = scale_for(np.abs(rows[n][0, h]).max(), cache)
                old = scales[n][pg, h, block]
                s = max(new, old) if first else new
                at = slice(block * BLOCK, block * BLOCK + first)
                if first and s > old:
                    was = codes[n][pg, h, at]
                    # what the code stood for, divided by the new scale, each one FP32 operation
                    moved = decode(was, cache).astype(np.float32) * old / s
                    codes[n][pg, h, at] = np.rint(moved).astype(np.int8).view(np.uint8) if cache == "int8" else \
                        encode_e4m3(moved.astype(np.float64))
                codes[n][pg, h, slot] = encode(rows[n][0, h], np.float32(s), cache)
                scales[n][pg, h, block] = s
        now = cache_of(c, d)
        for n in "kv":
            assert np.array_equal(now[n + "_scales"], scales[n]), (position, n)
            assert np.array_equal(decode(now[n + "_pages"], cache), decode(codes[n], cache)), (position, n)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_not_finite(cache, bad):
    """The block's scale becomes a NaN and stays one until its first position is written again; other blocks and heads
    keep their values."""
    c = Cache8([20], [26], heads=4, kv_heads=2, dim=64, cache=cache, max_pages=3, seed=4)
    c.v[3, 1, 7] = bad     # position 9, block 0
    c.k[12, 0, 63] = bad   # position 18, block 1
    d = c.device()
    append(c, d)
    now = cache_of(c, d)
    for n, block, head in (("v", 0, 1), ("k", 1, 0)):
        for h in range(2):
            for b in range(2):
                assert np.isnan(now[n + "_scales"][c.table[0, b], h, 0]) == (b == block and h == head)
    other = cache_of(c, d)["k_pages"][c.table[0, 0], 1, 6:16]
    assert np.array_equal(other, encode(c.k[:10, 1], now["k_scales"][c.table[0, 0], 1, 0], cache))
    # a later token of block 1 keeps the NaN, a first token of it takes it away
    for new, length, nan in ((1, 27, True), (11, 27, False)):
        e = Cache8([new], [length], heads=4, kv_heads=2, dim=64, cache=cache, max_pages=3, seed=4)
        for n in ("k", "v", "q"):
            d[n] = e.rows(getattr(e, n))
        d["starts"].upload(e.starts)
        d["lens"].upload(np.array(e.lens, np.int32))
        e.table = c.table
        append(e, d)
        assert np.isnan(cache_of(c, d)["k_scales"][c.table[0, 1], 0, 0]) == nan


def test_append_out_of_range_stays_in_bounds():
    c = Cache8([4, 4], [20, 20], dim=64, seed=13)
    for starts, lens in (([0, 100, 8], [20, 20]), ([-5, 4, 50], [20, 20]), ([0, 4, 2], [20, 2 ** 31 - 1]),
                         ([3, 5, 6], [-2 ** 31, 7])):
        d = c.device()
        d["starts"].upload(np.array(starts, np.int32))
        d["lens"].upload(np.array(lens, np.int32))
        q = append(c, d)
        c.read_rows(q, c.heads)
        cache_of(c, d)


# ------------------------------------------------------------------------------------------------- read
def read(c, d, with_k=True, with_v=True, stream=None):
    k, v = c.blank_rows(c.kv), c.blank_rows(c.kv)
    gie.synchronize()
    print("read8", c.p(), c.new[:8], c.lens[:8], flush=True)
    at = 2 * c.offset
    gie.kv8_read(c.p(), d["k_pages"].addr, d["v_pages"].addr, d["k_scales"].addr, d["v_scales"].addr, d["starts"].addr,
                 d["lens"].addr, d["table"].addr, k.addr + at if with_k else None, v.addr + at if with_v else None, stream=stream)
    gie.synchronize()
    return c.read_rows(k, c.kv), c.read_rows(v, c.kv)


def check_read(c, **kw):
    """One product in FP32 and one rounding: off by half a step of the type (u of the value, half of FP16's smallest step
    under its normal range) and what the product's own rounding adds, 2^-24 of the value. Numpy's bits of the two roundings
    are no measure: the device may round the exact product once, which differs where FP32's rounding lands on a tie."""
    got = read(c, c.device(), **kw)
    seq, position, valid = position_of(c)
    page = np.where(valid, c.table[seq, np.clip(position // c.page, 0, c.max_pages - 1)], -1)
    stored = (page >= 0) & (page < c.pages)
    for n, rows in zip("kv", got):
        if not kw.get("with_" + n, True):
            poison = gie.storage_to_float(np.array([0xA5A5], np.uint16), c.precision)[0]
            assert (rows == poison).all()
            continue
        pg, slot = np.where(stored, page, 0), position % c.page
        x = decode(getattr(c, n + "_pages")[pg, :, slot], c.cache) * \
            getattr(c, n + "_scales")[pg, :, slot // BLOCK].astype(np.float64)[..., None]
        x[~stored] = 0
        nan = np.isnan(x)
        assert np.array_equal(np.isnan(rows), nan) and (rows[~stored] == 0).all()
        off = (UNIT[c.precision] * (1 + 2.0 ** -24) + 2.0 ** -24) * np.abs(x) + TINY[c.precision]
        assert (np.abs(rows - x) <= off)[~nan].all()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("precision", ["fp16", "bf16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (96, 48), (128, 64), (256, 32)])
def test_read(dim, page, precision, cache):
    for new, lens in (([1], [1]), ([40, 0, 3, 130], [40, 7, 50, 130]), ([1] * 6, [1, 16, 17, 33, 100, 64])):
        check_read(Cache8(new, lens, dim=dim, page=page, precision=precision, cache=cache, seed=dim))


@pytest.mark.parametrize("gap,offset", [(8, 0), (3, 0), (0, 1), (5, 7)])
def test_read_strides_and_one_of_two(gap, offset):
    for kw in (dict(), dict(with_k=False), dict(with_v=False), dict(stream=gie.Stream())):
        check_read(Cache8([40, 9], [70, 9], dim=96, heads=6, kv_heads=3, gap=gap, offset=offset, cache="fp8", seed=gap), **kw)


@pytest.mark.parametrize("cache", CACHES)
def test_read_without_place_and_with_nan_scales(cache):
    check_read(Cache8([20, 3, 1], [7, 3, 0], dim=64, seed=1, cache=cache))
    check_read(Cache8([20, 40], [70, 30], dim=64, max_pages=4, seed=2, cache=cache))
    c = Cache8([100, 60], [100, 60], dim=128, seed=12, cache=cache)
    c.table[0, 2] = -1
    c.table[1, 1] = c.pages
    c.table[1, 3] = 2 ** 31 - 1
    c.k_scales[c.table[0, 0], 1] = np.nan
    check_read(c)


def test_read_every_code():
    """All 256 codes of e4m3, the NaN ones as 480, and of int8 (-128 too, which append never writes)."""
    for cache in CACHES:
        c = Cache8([16], [16], heads=1, kv_heads=1, dim=64, cache=cache, seed=0)
        c.k_pages[c.table[0, 0], 0] = np.arange(16 * 64, dtype=np.int64).astype(np.uint8).reshape(16, 64)
        check_read(c)
        rows, _ = read(c, c.device())
        assert np.isfinite(rows).all()


@pytest.mark.parametrize("cache", CACHES)
def test_append_then_read(cache):
    """A sequence built from chunks of many sizes comes back: every value within half a step for each time that its block's
    scale may have grown after it."""
    rng = np.random.default_rng(5)
    chunks = [1, 30, 1, 1, 17, 2, 64, 1, 5]
    c = Cache8([1], [1], heads=2, kv_heads=2, dim=64, page=32, precision="bf16", cache=cache, max_pages=4, seed=6)
    d, kept = c.device(), {"k": [], "v": []}
    grown, length = [], 0
    for n in chunks:
        length += n
        e = Cache8([n], [length], heads=2, kv_heads=2, dim=64, page=32, precision="bf16", cache=cache, max_pages=4,
                   seed=int(rng.integers(1 << 30)))
        e.table = c.table
        e.pages = c.pages
        for name in "kv":
            setattr(e, name, gie.storage_to_float(gie.host_to_storage(getattr(e, name) * np.float32(length), "bf16").reshape(-1), "bf16").reshape(
                n, 2, 64))
            kept[name].append(getattr(e, name))
            d[name] = e.rows(getattr(e, name))
        d["q"] = e.rows(e.q)
        d["starts"].upload(e.starts)
        d["lens"].upload(np.array(e.lens, np.int32))
        append(e, d)
        grown += [len(chunks)] * n
    whole = Cache8([length], [length], heads=2, kv_heads=2, dim=64, page=32, precision="bf16", cache=cache, max_pages=4, seed=6)
    whole.table, whole.pages = c.table, c.pages
    d["starts"].upload(whole.starts)
    d["lens"].upload(np.array([length], np.int32))
    got, now = dict(zip("kv", read(whole, d))), cache_of(c, d)
    pos = np.arange(length)
    for name in "kv":
        x = np.concatenate(kept[name]).astype(np.float64)
        s = now[name + "_scales"][c.table[0, pos // 32], :, pos % 32 // BLOCK].astype(np.float64)[..., None]
        # at most as many roundings as chunks reach the block after the value: each of the nine ones here
        if cache == "int8":
            step = 0.5 * s * len(chunks)
        else:  # a power of 2 moves normal values exactly: one rounding, and among the subnormals one for each growth
            step = np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s * len(chunks))
        assert (np.abs(got[name] - x) <= (step + 2.0 ** -8 * (np.abs(x) + step)) * (1 + 2.0 ** -12)).all()


# ------------------------------------------------------------------------------------------------- attention
def check(c, **kw):
    got = c.attend(**kw).astype(np.float64)
    want, bound = attention(c, **{k: v for k, v in kw.items() if k in ("scale", "softcap", "window", "sinks")})
    assert np.isfinite(got).all()
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), (float(off.max()), np.argwhere(off > 0)[:4].tolist(), int((off > 0).sum()))
    return got


BATCHES = {
    "one": ([1], [1]),
    "step": ([1] * 9, [1, 2, 15, 16, 17, 63, 64, 65, 300]),
    "few": ([3, 1, 0, 5, 2], [3, 40, 77, 5, 130]),
    "chunks": ([5, 0, 33, 130, 1, 64], [5, 9, 140, 133, 301, 64]),
    "prompt": ([200], [200]),
    "late": ([70], [400]),
}


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("precision", ["fp16", "bf16"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("batch", sorted(BATCHES))
def test_attend_batches(batch, dim, precision, cache):
    new, lens = BATCHES[batch]
    check(Cache8(new, lens, dim=dim, precision=precision, cache=cache, seed=dim))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (3, 1), (10, 2), (7, 1), (16, 2), (40, 1), (66, 1), (12, 4)])
def test_attend_groups(heads, kv_heads):
    for i, (new, lens) in enumerate((BATCHES["few"], ([1, 1], [33, 90]), ([40], [100]))):
        check(Cache8(new, lens, heads=heads, kv_heads=kv_heads, dim=128, precision="bf16", cache=CACHES[i % 2], seed=heads))


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128, 256])
def test_attend_page_sizes(page):
    for i, (new, lens) in enumerate((BATCHES["step"], BATCHES["chunks"])):
        check(Cache8(new, lens, page=page, dim=128, cache=CACHES[(i + page // 16) % 2], seed=page))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (16, 16), (31, 4), (64, 70), (100, 33), (1000, 5)])
@pytest.mark.parametrize("softcap", [0.0, 2.0, 100.0])
def test_attend_windows_sinks_and_caps(window, sinks, softcap, cache):
    for new, lens in (BATCHES["step"], BATCHES["chunks"], BATCHES["late"]):
        check(Cache8(new, lens, dim=64, page=32, precision="bf16", cache=cache, seed=window), window=window, sinks=sinks,
              softcap=softcap)


def test_attend_scales():
    for scale in (1.0, -0.3, 1e-3, 4.0):
        check(Cache8([3, 20], [50, 90], dim=64, cache="int8", seed=5), scale=scale)
        check(Cache8([3, 20], [50, 90], dim=64, cache="fp8", precision="bf16", seed=5), scale=scale, softcap=9.0)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("size", [2.0 ** -60, 1e-6, 1e4])
def test_attend_sizes_of_values(cache, size):
    """Values and queries far from 1 in BF16: scales, codes and the row's own factor take them, scores stay ordinary."""
    for new, lens in (([1, 1], [90, 300]), ([70], [200])):
        c = Cache8(new, lens, dim=128, precision="bf16", cache=cache, seed=7)
        c.v_scales *= np.float32(size)
        check(c)
        c = Cache8(new, lens, dim=128, precision="bf16", cache=cache, seed=8)
        c.k_scales *= np.float32(size)
        c.q = gie.storage_to_float(gie.host_to_storage((c.q / size).astype(np.float32), "bf16").reshape(-1), "bf16").reshape(c.q.shape)
        check(c)


@pytest.mark.parametrize("gap,offset", [(8, 0), (3, 0), (0, 1), (5, 7), (64, 8)])
def test_attend_strides_and_alignment(gap, offset):
    for batch in ("few", "chunks"):
        check(Cache8(*BATCHES[batch], dim=96, seed=gap, gap=gap, offset=offset, cache="fp8"))


@pytest.mark.parametrize("length", [700, 2049, 5000])
@pytest.mark.parametrize("new", [1, 7, 150])
@pytest.mark.parametrize("hints", [dict(), dict(max_new=1, max_len=100), dict(max_new=4096, max_len=1 << 20)])
def test_attend_long_contexts_and_hints(length, new, hints):
    c = Cache8([new, 1], [length, 40], dim=64, heads=2, kv_heads=1, page=64, seed=length, cache=CACHES[length % 2])
    check(c, **hints)
    check(c, window=600, sinks=20, **hints)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", [96, 128, 256])
@pytest.mark.parametrize("new", [1, 40, 130])
def test_attend_long_contexts_are_joined(dim, new, cache):
    for heads, kv_heads in ((2, 1), (12, 2)):
        c = Cache8([new, 3], [3000, 50], dim=dim, heads=heads, kv_heads=kv_heads, page=48, precision="bf16", seed=new, cache=cache)
        check(c, max_new=new, max_len=3000)
    check(c, window=1500, softcap=5.0, sinks=64)


@pytest.mark.parametrize("cache", CACHES)
def test_attend_rows_that_see_nothing(cache):
    got = check(Cache8([20, 3, 1], [7, 3, 0], dim=64, seed=1, cache=cache))
    assert (got[:13] == 0).all() and (got[-1] == 0).all()
    got = check(Cache8([20, 40], [70, 30], dim=64, max_pages=4, seed=2, cache=cache), window=9, sinks=3)
    assert (got[14:20] == 0).all() and (got[20:30] == 0).all()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_attend_blocks_that_nobody_sees_never_show(cache, dim):
    """Blocks behind the last position, and blocks that every window has passed, with scale NaN and every code."""
    for new, lens, window in (([1, 1], [40, 300], 0), ([33, 130], [140, 133], 0), ([1, 70], [300, 400], 30)):
        c = Cache8(new, lens, dim=dim, page=32, cache=cache, seed=3)
        want, bound = attention(c, window=window)
        visible = np.zeros((c.pages, c.page // BLOCK), bool)
        for b, (n, length) in enumerate(zip(new, lens)):
            for j in range(max(0, length - n - window + 1) if window else 0, length):
                visible[c.table[b, j // c.page], j % c.page // BLOCK] = True
        for n in "kv":
            getattr(c, n + "_scales").transpose(0, 2, 1)[~visible] = np.nan
            pages = getattr(c, n + "_pages").reshape(c.pages, c.kv, -1, BLOCK, c.dim).transpose(0, 2, 1, 3, 4)
            pages[~visible] = 0x7f
        got = c.attend(window=window)
        assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("new,lens,window", [([40], [40], 0), ([150, 9], [200, 9], 0), ([150], [300], 20), ([1], [300], 40)])
def test_attend_nan_scales_reach_only_rows_that_see_their_block(cache, new, lens, window):
    for dim in (64, 128, 256):
        for where in "kv":
            for at in (lens[0] - 1, lens[0] - max(1, new[0] // 2), max(0, lens[0] - new[0] - 3), 0):
                c = Cache8(new, lens, heads=4, kv_heads=2, dim=dim, cache=cache, seed=at)
                want, bound = attention(c, window=window)
                getattr(c, where + "_scales")[c.table[0, at // c.page], 1, at % c.page // BLOCK] = np.nan
                got = c.attend(window=window)
                position = np.arange(lens[0] - new[0], lens[0])
                start = at // BLOCK * BLOCK
                sees = position >= start
                if window:
                    sees &= position - window < start + BLOCK - 1
                sees = np.concatenate([sees, np.zeros(sum(new[1:]), bool)])
                assert (np.abs(got - want) <= bound)[~sees].all()
                assert (np.abs(got - want) <= bound)[:, :2].all()  # the other key head
                assert np.isnan(got[sees][:, 2:]).all()


def test_attend_not_finite_queries_stay_in_their_row():
    for precision in ("fp16", "bf16"):
        for bad in (np.nan, np.inf):
            c = Cache8([50], [80], dim=128, precision=precision, seed=9)
            want, bound = attention(c)
            c.q[7, 2, 3] = bad
            got = c.attend()
            assert np.isnan(got[7, 2]).all()
            ok = np.abs(got - want) <= bound
            ok[7, 2] = True
            assert ok.all()


@pytest.mark.parametrize("cache", CACHES)
def test_attend_large_scores(cache):
    """Scores of hundreds either way, and keys that each pass all before them."""
    c = Cache8([1, 40], [500, 300], dim=64, precision="bf16", cache=cache, seed=10)
    c.k_scales *= np.float32(32)
    c.q *= 4
    check(c)
    c = Cache8([30], [200], dim=64, cache=cache, seed=11, spread=0)
    c.k_pages[:] = encode(np.ones((1,), np.float32), np.float32(0.0625), cache)[0]
    for j in range(13):
        c.k_scales[c.table[0, j], :, 0] = (j + 1) / 16
    c.q[:] = np.abs(c.q)
    check(c)


@pytest.mark.parametrize("cache", CACHES)
def test_attend_blocks_of_zeros_keep_their_weight(cache):
    """Values of zero have the smallest scale there is, and their weights count in full: beside ordinary values, beside
    large ones, and alone."""
    for new, lens in (([1], [200]), ([80], [200])):
        for size in (1.0, 2.0 ** 20):
            c = Cache8(new, lens, dim=128, precision="bf16", cache=cache, seed=12)
            c.v_scales *= np.float32(size)
            for j in range(0, 13, 2):
                c.v_pages[c.table[0, j]] = 0
                c.v_scales[c.table[0, j]] = scale_for(0, cache)
            check(c)
        c.v_pages[:] = 0
        c.v_scales[:] = scale_for(0, cache)
        assert (c.attend() == 0).all()


def test_attend_scales_of_zero_count_as_the_smallest():
    c = Cache8([1, 40], [100, 90], dim=64, cache="int8", seed=13)
    want, bound = attention(c)
    for b in range(2):
        c.v_scales[c.table[b, 1]] = 0
        c.k_scales[c.table[b, 2]] = 0
    c.v_pages[c.table[:2, 1]] = 0
    check(c)


def test_attend_pages_that_are_not_there_read_as_zeros():
    for cache in CACHES:
        c = Cache8([3, 40], [100, 60], dim=128, seed=12, cache=cache)
        c.table[0, 2] = -1
        c.table[1, 1] = c.pages
        c.table[1, 3] = 2 ** 31 - 1
        check(c)
        check(c, window=50, sinks=7)


def test_attend_lengths_and_starts_out_of_range_stay_in_bounds():
    c = Cache8([4, 4], [20, 20], dim=64, seed=13)
    d = c.device()
    for starts, lens in (([0, 100, 8], [20, 20]), ([-5, 4, 50], [20, 20]), ([0, 4, 2], [20, 2 ** 31 - 1]),
                         ([3, 5, 6], [-2 ** 31, 7])):
        d["starts"].upload(np.array(starts, np.int32))
        d["lens"].upload(np.array(lens, np.int32))
        c.attend(d=d)


def test_rows_of_no_sequence_are_left_alone():
    c = Cache8([4, 4], [20, 20], dim=64, seed=13)
    d = c.device()
    d["starts"].upload(np.array([2, 4, 6], np.int32))
    poison = gie.storage_to_float(np.array([0xA5A5], np.uint16), "fp16")[0]
    for got in (c.attend(d=d), *read(c, d), c.read_rows(append(c, d), c.heads)):
        assert (got[[0, 1, 6, 7]] == poison).all() and (got[2:6] != poison).all()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("lens", [[1], [5000], [100, 2000]])
def test_attend_same_bits_every_time_and_on_a_stream(lens, cache):
    c = Cache8([1] * len(lens), lens, dim=128, heads=8, kv_heads=1, page=64, seed=14, cache=cache)
    d, s = c.device(), gie.Stream()
    hints = dict(max_new=1, max_len=max(lens))
    first = c.attend(d=d, **hints)
    assert np.array_equal(first, c.attend(d=d, **hints)) and np.array_equal(first, c.attend(d=d, stream=s, **hints))


def test_cache_past_32_bit_offsets():
    """Over 8 GiB of codes each: pages whose offsets pass 2^32, in all three calls."""
    import torch
    page, kv, dim, heads = 256, 8, 256, 16
    pages = 2 ** 33 // (page * kv * dim) + 40
    k, v = (torch.zeros((pages, kv, page, dim), dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones((pages, kv, page // BLOCK), dtype=torch.float32, device="cuda") for _ in range(2))
    c = Cache8([1, 37], [700, 300], heads=heads, kv_heads=kv, dim=dim, page=page, precision="bf16", seed=15)
    far = np.array([[pages - 1, pages - 17, pages // 2 + 1], [pages - 2, pages // 2 + 33, 0]], np.int32)
    for b in range(2):
        for i, n in enumerate(far[b]):
            for big, small in ((k, c.k_pages), (v, c.v_pages), (ks, c.k_scales), (vs, c.v_scales)):
                big[int(n)] = torch.from_numpy(small[c.table[b, i]].copy()).cuda()
    torch.cuda.synchronize()
    p, d, out = c.p(num_pages=pages), c.device(), c.blank_rows(heads)
    table = gie.to_device(far)
    where = (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), d["starts"].addr, d["lens"].addr, table.addr)
    ws = gie.DeviceBuffer(max(16, gie.kv8_attention_workspace_size(p)))
    gie.kv8_attention(p, d["q"].addr, *where, out.addr, workspace=ws.addr, ws_bytes=ws.nbytes)
    gie.synchronize()
    want, bound = attention(c)
    assert (np.abs(c.read_rows(out, heads) - want) <= bound).all()
    gie.kv8_append(p, d["k"].addr, d["v"].addr, *where[4:], *where[:4])
    rows = [c.blank_rows(kv) for _ in range(2)]
    gie.kv8_read(p, *where, rows[0].addr, rows[1].addr)
    gie.synchronize()
    for got, x, s in ((rows[0], c.k, ks), (rows[1], c.v, vs)):
        got = c.read_rows(got, kv)
        # half a step of the block's scale, which the largest of the block's values bounds, and BF16's rounding
        most = max(float(s[int(far[0, 2])].max()), float(s[int(far[1, 1])].max()))
        assert (np.abs(got - x) <= 0.5 * most + 2.0 ** -8 * (np.abs(x) + most)).all()


@pytest.mark.parametrize("cache", CACHES)
def test_captured_graph_replays(cache):
    """Append with norms, attention and read as one captured graph, replayed with other work in between."""
    import torch
    c = Cache8([1, 5, 1], [300, 40, 1500], dim=128, heads=8, kv_heads=2, page=64, seed=16, max_pages=40, cache=cache)
    d = c.device()
    cos, sin = (gie.to_device(t) for t in gie.rotary_tables(40 * 64, 128))
    norm = gie.to_device(np.linspace(0.5, 1.5, 128).astype(np.float32))
    p = c.p(rotary_dim=128, max_positions=40 * 64, max_len=1500, max_new=5, norm_eps=1e-6, window=200, sinks=5)
    ws = gie.DeviceBuffer(max(16, gie.kv8_attention_workspace_size(p)))
    qr, out, k, v = c.blank_rows(c.heads), c.blank_rows(c.heads), c.blank_rows(c.kv), c.blank_rows(c.kv)
    pages = [d[n].addr for n in ("k_pages", "v_pages", "k_scales", "v_scales")]
    where = [d[n].addr for n in ("starts", "lens", "table")]

    def step(stream):
        gie.kv8_append(p, d["k"].addr, d["v"].addr, *where, *pages, q_norm=norm.addr, k_norm=norm.addr, cos=cos.addr,
                       sin=sin.addr, q=d["q"].addr, q_out=qr.addr, stream=stream)
        gie.kv8_attention(p, qr.addr, *pages, *where, out.addr, workspace=ws.addr, ws_bytes=ws.nbytes, stream=stream)
        gie.kv8_read(p, *pages, *where, k.addr, v.addr, stream=stream)

    def reset(lens):
        for n in ("k_pages", "v_pages", "k_scales", "v_scales"):
            d[n].upload(np.ascontiguousarray(getattr(c, n)))
        d["lens"].upload(np.array(lens, np.int32))

    def results():
        return [c.read_rows(out, c.heads), c.read_rows(k, c.kv), c.read_rows(v, c.kv)]

    lengths, want = [[300, 40, 1500], [301, 41, 1501]], []
    for lens in lengths:
        reset(lens)
        step(None)
        gie.synchronize()
        want.append(results())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for i in (1, 0, 1, 0):
        reset(lengths[i])
        for b in (out, k, v):
            b.fill(0xA5)
        ws.fill(0xFF)
        torch.ones(1 << 20, device="cuda").mul_(2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(np.array_equal(a, b) for a, b in zip(results(), want[i]))


def test_block_step_together():
    """Prompts, then steps, through append with norms and attention, against the same from the stored values in 64 bits."""
    for cache, precision in (("int8", "bf16"), ("fp8", "fp16")):
        c = Cache8([37, 1, 90], [37, 1, 90], heads=8, kv_heads=2, dim=64, page=32, precision=precision, cache=cache, max_pages=5, seed=17)
        d, lens = c.device(), [37, 1, 90]
        cos, sin = gie.rotary_tables(5 * 32, 64)
        rng = np.random.default_rng(1)
        weights = [rng.uniform(0.5, 1.5, 64).astype(np.float32) for _ in range(2)]
        for new in ([37, 1, 90], [1, 1, 1], [1, 0, 1], [1, 20, 1]):
            if new != c.new:
                lens = [a + n for a, n in zip(lens, new)]
                e = Cache8(new, lens, heads=8, kv_heads=2, dim=64, page=32, precision=precision, cache=cache, max_pages=5,
                           seed=sum(lens))
                e.table, e.pages = c.table, c.pages
                for n in "qkv":
                    d[n] = e.rows(getattr(e, n))
                d["starts"].upload(e.starts)
                d["lens"].upload(np.array(lens, np.int32))
            else:
                e = c
            d["q"] = append(e, d, rotary=64, cos=cos, sin=sin, q_norm=weights[0], k_norm=weights[1], with_q=True)
            got = e.attend(d=d, max_new=max(new), max_len=max(lens))
            now = cache_of(c, d)
            for n, a in now.items():
                setattr(e, n, a)
            e.q = e.read_rows(d["q"], 8)
            want, bound = attention(e)
            assert (np.abs(got - want) <= bound).all()


def test_no_tokens_is_no_work():
    c = Cache8([0, 0], [5, 9], dim=64)
    assert gie.kv8_attention_workspace_size(c.p()) >= 0
    p = gie.PagedKv(0, 0, 2, 1, 64, 16, 1, 1, cache="int8")
    gie.kv8_attention(p, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    gie.kv8_append(p, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    gie.kv8_read(p, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    gie.synchronize()
