"""PagedKv::append_normed, and windows with sinks in PagedKv::attention, on the GPU against plain numpy in 64 bits."""
import numpy as np
import pytest

import gie
from kv8_plain import attention, position_of, turned
from paged_plain import UNIT, Cache

pytestmark = pytest.mark.gpu

APPENDS = {"one": ([1], [1]), "step": ([1] * 7, [1, 16, 17, 31, 32, 33, 100]), "chunks": ([5, 0, 33, 70], [5, 9, 50, 133])}


def check_append(c, rotary, interleaved, norms=(True, True), with_q=True, in_place=False, stream=None, eps=1e-5):
    d = c.device()
    rng = np.random.default_rng(rotary + 1)
    cos, sin = (rng.uniform(-1, 1, (c.max_pages * c.page, rotary // 2)).astype(np.float32) for _ in range(2))
    wq, wk = (rng.uniform(-1.5, 1.5, c.dim).astype(np.float32) if n else None for n in norms)
    dev = {n: gie.to_device(a) for n, a in (("cos", cos), ("sin", sin), ("q_norm", wq if with_q else None), ("k_norm", wk))
           if a is not None and a.size}
    p = c.p(rotary_dim=rotary, interleaved=interleaved, max_positions=c.max_pages * c.page, norm_eps=eps)
    q_out = d["q"] if in_place else c.blank_rows(c.heads)
    gie.synchronize()
    print("append_normed", p, c.new[:8], c.lens[:8], flush=True)
    at = 2 * c.offset
    gie.kv_append_normed(p, d["k"].addr + at, d["v"].addr + at, d["starts"].addr, d["lens"].addr, d["table"].addr,
                         d["k_pages"].addr, d["v_pages"].addr, q=d["q"].addr + at if with_q else None,
                         q_out=q_out.addr + at if with_q else None, **{n: b.addr for n, b in dev.items()}, stream=stream)
    gie.synchronize()
    turn = dict(eps=eps, rotary=rotary, interleaved=interleaved, cos=cos, sin=sin)
    u = UNIT[c.precision]

    def near(got, x, w, rows=slice(None)):
        want, off = turned(c, x, w, **turn)
        want, off = want[rows], off[rows]
        assert (np.abs(got - want) <= off + u * (np.abs(want) + off) + 2.0 ** -25).all()

    if with_q:
        near(c.read_rows(q_out, c.heads), c.q, wq)
    seq, position, valid = position_of(c)
    page = np.where(valid, c.table[seq, np.clip(position // c.page, 0, c.max_pages - 1)], -1)
    rows = np.flatnonzero((page >= 0) & (page < c.pages))
    touched = np.zeros((c.pages, c.page), bool)
    touched[page[rows], position[rows] % c.page] = True
    k, v = (gie.storage_to_float(d[n].download(np.uint16, c.k_pages.size), c.precision).reshape(c.k_pages.shape)
            for n in ("k_pages", "v_pages"))
    near(k[page[rows], :, position[rows] % c.page], c.k, wk, rows)
    assert np.array_equal(v[page[rows], :, position[rows] % c.page], c.v[rows])
    for now, before in ((k, c.k_pages), (v, c.v_pages)):
        assert np.array_equal(now.transpose(0, 2, 1, 3)[~touched], before.transpose(0, 2, 1, 3)[~touched]), "other slots"


@pytest.mark.parametrize("precision", ["fp16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 0), (96, 64), (128, 128), (128, 32), (256, 256), (128, 6), (96, 96), (64, 2)])
def test_append_normed(dim, rotary, interleaved, precision):
    for batch in sorted(APPENDS):
        check_append(Cache(*APPENDS[batch], dim=dim, precision=precision, seed=rotary), rotary, interleaved)


@pytest.mark.parametrize("norms", [(True, False), (False, True), (False, False)])
def test_one_norm_or_none(norms):
    for dim, rotary in ((96, 64), (128, 6)):
        check_append(Cache(*APPENDS["chunks"], dim=dim, seed=1), rotary, False, norms=norms)


@pytest.mark.parametrize("heads,kv_heads,page", [(1, 1, 16), (3, 3, 48), (32, 8, 64), (5, 1, 32), (40, 8, 16), (66, 1, 16)])
def test_heads_and_pages(heads, kv_heads, page):
    for kw in (dict(interleaved=False), dict(interleaved=True, with_q=False)):
        check_append(Cache([3, 40], [9, 100], heads=heads, kv_heads=kv_heads, dim=128, page=page, seed=heads), 128, **kw)


@pytest.mark.parametrize("gap,offset", [(8, 0), (3, 0), (0, 1), (5, 7), (64, 8)])
@pytest.mark.parametrize("in_place", [False, True])
def test_strides_and_alignment(gap, offset, in_place):
    for interleaved in (False, True):
        for dim, rotary in ((96, 64), (64, 6)):
            check_append(Cache(*APPENDS["chunks"], dim=dim, gap=gap, offset=offset, seed=gap), rotary, interleaved, in_place=in_place)


def test_without_room():
    check_append(Cache([20, 3, 1], [7, 3, 0], dim=64, seed=1), 64, False)
    check_append(Cache([20, 40], [70, 30], dim=64, max_pages=4, seed=2), 32, True)
    c = Cache([3, 40], [100, 60], dim=128, seed=12)
    c.table[0, 6] = -1
    c.table[1, 1] = c.pages
    c.table[1, 3] = 2 ** 31 - 1
    check_append(c, 128, False, stream=gie.Stream())


def test_heads_of_zeros_and_eps():
    """A head of zeros stays zeros; eps counts where values are small."""
    c = Cache([6], [9], dim=64, precision="bf16", seed=3)
    c.q[2], c.k[4] = 0, 0
    c.k[1] *= np.float32(2.0 ** -9)
    check_append(c, 64, False, eps=1e-6)
    check_append(c, 64, False, eps=0.25)


def test_many_tokens_and_sequences():
    """Several tokens to a workgroup, and batches past one round of the search for a row's sequence."""
    for batch, dim in ((65, 64), (700, 128), (4100, 96)):
        rng = np.random.default_rng(batch)
        new = rng.integers(0, 3, batch).tolist()
        lens = [n + int(rng.integers(0, 20)) for n in new]
        check_append(Cache(new, lens, heads=2, kv_heads=1, dim=dim, seed=batch), 64, False)
    check_append(Cache([1500], [1600], heads=4, kv_heads=2, dim=128, page=64, precision="bf16", seed=1), 128, False)


def test_not_finite_heads_stay_alone():
    c = Cache([5], [5], dim=64, seed=4)
    c.q[2, 1, 7] = np.nan
    c.k[3, 0, 9] = np.inf
    d = c.device()
    w = gie.to_device(np.ones(64, np.float32))
    out = c.blank_rows(c.heads)
    gie.kv_append_normed(c.p(norm_eps=1e-5), d["k"].addr, d["v"].addr, d["starts"].addr, d["lens"].addr, d["table"].addr,
                         d["k_pages"].addr, d["v_pages"].addr, q_norm=w.addr, k_norm=w.addr, q=d["q"].addr, q_out=out.addr)
    gie.synchronize()
    q = c.read_rows(out, c.heads)
    assert np.isnan(q[2, 1]).all()
    q[2, 1] = 0
    assert np.isfinite(q).all()
    k = gie.storage_to_float(d["k_pages"].download(np.uint16, c.k_pages.size), c.precision).reshape(c.k_pages.shape)
    assert np.isnan(k[c.table[0, 0], 0, 3, 9]) and np.isfinite(k[c.table[0, 0], 1]).all()


def test_same_as_append_without_norms():
    """With neither norm the call is append's, bit for bit."""
    for rotary, interleaved in ((128, False), (64, True), (6, False)):
        c = Cache(*APPENDS["chunks"], dim=128, precision="bf16", seed=5)
        cos, sin = (gie.to_device(t) for t in gie.rotary_tables(c.max_pages * c.page, rotary))
        p = c.p(rotary_dim=rotary, interleaved=interleaved, max_positions=c.max_pages * c.page)
        got = []
        for call in (gie.kv_append, gie.kv_append_normed):
            d, out = c.device(), c.blank_rows(c.heads)
            call(p, d["k"].addr, d["v"].addr, d["starts"].addr, d["lens"].addr, d["table"].addr, d["k_pages"].addr,
                 d["v_pages"].addr, cos=cos.addr, sin=sin.addr, q=d["q"].addr, q_out=out.addr)
            gie.synchronize()
            got.append([b.download(np.uint16, b.nbytes // 2) for b in (out, d["k_pages"], d["v_pages"])])
        assert all(np.array_equal(a, b) for a, b in zip(*got))


# ------------------------------------------------------------------------------------------------- windows with sinks
BATCHES = {
    "step": ([1] * 9, [1, 2, 15, 16, 17, 63, 64, 65, 300]),
    "chunks": ([5, 0, 33, 130, 1, 64], [5, 9, 140, 133, 301, 64]),
    "late": ([70], [400]),
}


def check(c, **kw):
    got = c.attend(**kw).astype(np.float64)
    want, bound = attention(c, **{k: v for k, v in kw.items() if k in ("scale", "softcap", "window", "sinks")})
    assert np.isfinite(got).all()
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), (float(off.max()), np.argwhere(off > 0)[:4].tolist(), int((off > 0).sum()))
    return got


@pytest.mark.parametrize("precision", ["fp16", "bf16"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("window,sinks", [(1, 1), (2, 16), (16, 17), (31, 4), (64, 70), (100, 33), (1000, 5), (0, 9)])
def test_sinks(window, sinks, dim, precision):
    for batch in sorted(BATCHES):
        check(Cache(*BATCHES[batch], dim=dim, page=32, precision=precision, seed=window), window=window, sinks=sinks,
              softcap=2.0 if sinks == 33 else 0.0)


@pytest.mark.parametrize("new", [1, 40, 130])
@pytest.mark.parametrize("sinks", [1, 64, 200, 1 << 30])
def test_sinks_of_long_contexts(new, sinks):
    """Parts of the keys that lie in the sinks, in the window and in both; more sinks than there are positions."""
    for heads, kv_heads, dim in ((2, 1, 64), (12, 2, 128)):
        c = Cache([new, 3], [3000, 50], dim=dim, heads=heads, kv_heads=kv_heads, page=48, precision="bf16", seed=new)
        for hints in (dict(), dict(max_new=new, max_len=3000), dict(max_new=1, max_len=64)):
            check(c, window=700, sinks=sinks, **hints)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("new,length", [(1, 300), (9, 300), (150, 300)])
def test_values_that_are_not_finite_in_and_behind_sinks(bad, new, length):
    """In a sink: every row carries it on. Between the sinks and the window: only rows whose window holds it."""
    window, sinks = 40, 5
    for dim in (64, 128):
        for at in (3, 5, 15, length - new // 2 - 42):
            c = Cache([new], [length], heads=4, kv_heads=2, dim=dim, seed=at)
            want, bound = attention(c, window=window, sinks=sinks)
            c.v_pages[c.table[0, at // c.page], 1, at % c.page, 5] = bad
            got = c.attend(window=window, sinks=sinks)
            position = np.arange(length - new, length)
            sees = (position >= at) & ((position < at + window) | (at < sinks))
            ok = np.abs(got - want) <= bound
            assert ok[~sees].all() and ok[:, :2].all()
            hit = got[sees][:, 2:, 5]
            assert (np.isnan(hit) if np.isnan(bad) else hit == bad).all()
            assert ok[sees][:, 2:][..., np.delete(np.arange(dim), 5)].all()


def test_sinks_without_a_window_change_nothing():
    c = Cache(*BATCHES["chunks"], dim=128, seed=6)
    assert np.array_equal(c.attend(), c.attend(sinks=50))


def test_sinks_rows_that_see_nothing():
    got = check(Cache([20, 40], [70, 30], dim=64, max_pages=4, seed=2), window=9, sinks=20)
    assert (got[14:20] == 0).all() and (got[20:30] == 0).all()
