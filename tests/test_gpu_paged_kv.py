"""PagedKv::append and PagedKv::attention on the GPU against plain numpy in 64 bits (tests/paged_plain.py, which also
derives the bounds): one token and chunks, ragged batches with empty sequences, page ends inside tiles, windows, capped
scores, grouped heads, odd strides, rows that see nothing, values that are not finite in places nobody sees."""
import numpy as np
import pytest

import gie
from paged_plain import UNIT, Cache

pytestmark = pytest.mark.gpu


def check(c, **kw):
    got = c.attend(**{k: v for k, v in kw.items()}).astype(np.float64)
    want, bound = c.plain(**{k: v for k, v in kw.items() if k in ("scale", "softcap", "window")})
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


@pytest.mark.parametrize("precision", ["fp16", "bf16"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("batch", sorted(BATCHES))
def test_batches(batch, dim, precision):
    new, lens = BATCHES[batch]
    check(Cache(new, lens, dim=dim, precision=precision, seed=dim))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (3, 1), (10, 2), (7, 1), (16, 2), (40, 1), (66, 1), (12, 4)])
def test_groups(heads, kv_heads):
    for new, lens in (BATCHES["few"], ([1, 1], [33, 90]), ([40], [100])):
        check(Cache(new, lens, heads=heads, kv_heads=kv_heads, dim=128, precision="bf16", seed=heads))


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128, 256])
def test_page_sizes(page):
    for new, lens in (BATCHES["step"], BATCHES["chunks"]):
        check(Cache(new, lens, page=page, dim=128, seed=page))


@pytest.mark.parametrize("window", [1, 2, 16, 31, 64, 100, 1000])
@pytest.mark.parametrize("softcap", [0.0, 2.0])
def test_windows_and_caps(window, softcap):
    for new, lens in (BATCHES["step"], BATCHES["chunks"], BATCHES["late"]):
        check(Cache(new, lens, dim=64, page=32, precision="bf16", seed=window), window=window, softcap=softcap)


def test_scales():
    for scale in (1.0, -0.3, 1e-3, 4.0):
        check(Cache([3, 20], [50, 90], dim=64, seed=5), scale=scale)
    check(Cache([3, 20], [50, 90], dim=256, precision="bf16", seed=6), softcap=30.0)


@pytest.mark.parametrize("gap,offset", [(8, 0), (3, 0), (0, 1), (5, 7), (64, 8)])
def test_strides_and_alignment(gap, offset):
    for batch in ("few", "chunks"):
        check(Cache(*BATCHES[batch], dim=96, seed=gap, gap=gap, offset=offset))


@pytest.mark.parametrize("length", [700, 2049, 5000])
@pytest.mark.parametrize("new", [1, 7, 150])
@pytest.mark.parametrize("hints", [dict(), dict(max_new=1, max_len=100), dict(max_new=4096, max_len=1 << 20)])
def test_long_contexts_and_hints(length, new, hints):
    """The hints choose the launch, never the result; a context longer than the hint says is read whole."""
    c = Cache([new, 1], [length, 40], dim=64, heads=2, kv_heads=1, page=64, seed=length)
    check(c, **hints)
    check(c, window=600, **hints)


@pytest.mark.parametrize("dim", [96, 128, 256])
@pytest.mark.parametrize("new", [1, 40, 130])
def test_long_contexts_are_joined(dim, new):
    """Few workgroups over a long context: its keys are split, one part and many for the rows of one call."""
    for heads, kv_heads in ((2, 1), (12, 2)):
        c = Cache([new, 3], [3000, 50], dim=dim, heads=heads, kv_heads=kv_heads, page=48, precision="bf16", seed=new)
        check(c, max_new=new, max_len=3000)
    check(c, window=1500, softcap=5.0)


def test_rows_that_see_nothing():
    """More new tokens than the sequence holds, and sequences longer than their row of the page table."""
    got = check(Cache([20, 3, 1], [7, 3, 0], dim=64, seed=1))
    assert (got[:13] == 0).all() and (got[-1] == 0).all()
    got = check(Cache([20, 40], [70, 30], dim=64, max_pages=4, seed=2))  # capacity 64: positions 64.. are not valid
    assert (got[14:20] == 0).all() and (got[20:30] == 0).all()


@pytest.mark.parametrize("stale", [np.nan, np.inf, 6e4])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_stale_slots_never_show(stale, dim):
    for batch in ("step", "few", "chunks"):
        check(Cache(*BATCHES[batch], dim=dim, stale=stale, seed=3))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("new,lens,window", [([40], [40], 0), ([150, 9], [200, 9], 0), ([150], [300], 20), ([1], [300], 40)])
def test_not_finite_values_reach_only_rows_that_see_them(bad, new, lens, window):
    """A value that is not finite at one position: rows before it (and rows whose window has passed it) keep their
    exact bound; rows that see it carry it on."""
    for dim in (64, 128):
        for where in ("v", "k"):
            for at in (lens[0] - 1, lens[0] - max(1, new[0] // 2), max(0, lens[0] - new[0] - 3), 0):
                c = Cache(new, lens, heads=4, kv_heads=2, dim=dim, seed=at)
                want, bound = c.plain(window=window)
                pages = c.v_pages if where == "v" else c.k_pages
                pages[c.table[0, at // c.page], 1, at % c.page, 5] = bad
                got = c.attend(window=window)
                position = np.arange(lens[0] - new[0], lens[0])
                sees = (position >= at) & ((position < at + window) if window else True)
                sees = np.concatenate([sees, np.zeros(sum(new[1:]), bool)])
                assert (np.abs(got - want) <= bound)[~sees].all()
                assert (np.abs(got - want) <= bound)[:, :2].all()  # the other key head
                if where == "v":
                    hit = got[sees][:, 2:, 5]
                    assert (np.isnan(hit) if np.isnan(bad) else hit == bad).all()
                    rest = np.delete(np.arange(dim), 5)
                    assert (np.abs(got - want) <= bound)[sees][:, 2:, rest].all()
                elif np.isnan(bad):
                    assert np.isnan(got[sees][:, 2:]).all()


@pytest.mark.parametrize("dim", [96, 256])
@pytest.mark.parametrize("precision", ["fp16", "bf16"])
@pytest.mark.parametrize("new,window", [(150, 0), (9, 0), (150, 20)])
def test_not_finite_values_in_wide_heads(dim, precision, new, window):
    """As above at the other head sizes, an infinity and a NaN in different values of different positions."""
    c = Cache([new], [200], heads=4, kv_heads=2, dim=dim, precision=precision, seed=dim + new)
    want, bound = c.plain(window=window)
    spots = [(195, 0, np.inf), (190, dim - 1, -np.inf), (150, dim // 2 + 3, np.nan)]
    for at, d, bad in spots:
        c.v_pages[c.table[0, at // c.page], 1, at % c.page, d] = bad
    got = c.attend(window=window)
    position = np.arange(200 - new, 200)
    touched = np.zeros((new, 4, dim), bool)
    for at, d, bad in spots:
        sees = (position >= at) & ((position < at + window) if window else True)
        touched[sees, 2:, d] = True
        hit = got[sees][:, 2:, d]
        assert (np.isnan(hit) if np.isnan(bad) else hit == bad).all()
    assert (np.abs(got - want) <= bound)[~touched].all()


def test_not_finite_queries_stay_in_their_row():
    c = Cache([50], [80], dim=128, seed=9)
    want, bound = c.plain()
    c.q[7, 2, 3] = np.nan
    got = c.attend()
    assert np.isnan(got[7, 2]).all()
    ok = np.abs(got - want) <= bound
    ok[7, 2] = True
    assert ok.all()


def test_large_scores():
    """Scores of hundreds either way: the running maximum has to move, nothing overflows."""
    c = Cache([1, 40], [500, 300], dim=64, precision="bf16", seed=10)
    c.k_pages *= 32
    c.q *= 4
    check(c)
    c = Cache([30], [200], dim=64, seed=11)
    ramp = np.arange(200, dtype=np.float32)
    for j in range(200):  # every key larger than all before it
        c.k_pages[c.table[0, j // 16], :, j % 16] = ramp[j] / 16
    c.q[:] = np.abs(c.q)
    check(c)


def test_pages_that_are_not_there_read_as_zeros():
    c = Cache([3, 40], [100, 60], dim=128, seed=12)
    c.table[0, 2] = -1
    c.table[1, 1] = c.pages
    c.table[1, 3] = 2 ** 31 - 1
    check(c)
    check(c, window=50)


def test_lengths_and_starts_out_of_range_stay_in_bounds():
    """Nothing is promised about such rows but that memory outside the outputs is left alone."""
    c = Cache([4, 4], [20, 20], dim=64, seed=13)
    d = c.device()
    for starts, lens in (([0, 100, 8], [20, 20]), ([-5, 4, 50], [20, 20]), ([0, 4, 2], [20, 2 ** 31 - 1]),
                         ([3, 5, 6], [-2 ** 31, 7])):
        d["starts"].upload(np.array(starts, np.int32))
        d["lens"].upload(np.array(lens, np.int32))
        c.attend(d=d)


def test_rows_of_no_sequence_are_left_alone():
    c = Cache([4, 4], [20, 20], dim=64, seed=13)
    d = c.device()
    d["starts"].upload(np.array([2, 4, 6], np.int32))
    d["lens"].upload(np.array([20, 20], np.int32))
    got = c.attend(d=d)
    poison = gie.storage_to_float(np.array([0xA5A5], np.uint16), "fp16")[0]
    assert (got[[0, 1, 6, 7]] == poison).all() and (got[2:6] != poison).all()


@pytest.mark.parametrize("lens", [[1], [5000], [100, 2000]])
def test_same_bits_every_time_and_on_a_stream(lens):
    c = Cache([1] * len(lens), lens, dim=128, heads=8, kv_heads=1, page=64, seed=14)
    d, s = c.device(), gie.Stream()
    hints = dict(max_new=1, max_len=max(lens))
    first = c.attend(d=d, **hints)
    assert np.array_equal(first, c.attend(d=d, **hints)) and np.array_equal(first, c.attend(d=d, stream=s, **hints))


def test_cache_past_32_bit_offsets():
    """A cache of over 8 GiB for keys and values each: pages whose byte and element offsets pass 2^32."""
    import torch
    page, kv, dim, heads = 256, 8, 256, 16
    pages = 2 ** 33 // (page * kv * dim * 2) + 40
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.zeros((pages, kv, page, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    c = Cache([1, 37], [700, 300], heads=heads, kv_heads=kv, dim=dim, page=page, precision="bf16", seed=15)
    far = np.array([[pages - 1, pages - 17, pages // 2 + 1], [pages - 2, pages // 2 + 33, 0]], np.int32)
    for b in range(2):
        for i, n in enumerate(far[b]):
            for big, small in ((k, c.k_pages), (v, c.v_pages)):
                big[int(n)] = torch.from_numpy(small[c.table[b, i]].copy()).cuda().to(torch.bfloat16)
    torch.cuda.synchronize()
    p, d, out = c.p(num_pages=pages), c.device(), c.blank_rows(heads)
    table = gie.to_device(far)
    ws = gie.DeviceBuffer(max(16, gie.paged_attention_workspace_size(p)))
    gie.paged_attention(p, d["q"].addr, k.data_ptr(), v.data_ptr(), d["starts"].addr, d["lens"].addr, table.addr, out.addr,
                        workspace=ws.addr, ws_bytes=ws.nbytes)
    gie.synchronize()
    want, bound = c.plain()
    assert (np.abs(c.read_rows(out, heads) - want) <= bound).all()
    # and the append: the new tokens' slots of the far pages
    gie.kv_append(p, d["k"].addr, d["v"].addr, d["starts"].addr, d["lens"].addr, table.addr, k.data_ptr(), v.data_ptr())
    gie.synchronize()
    new = k[int(far[0, 2]), :, 699 % page].float().cpu().numpy()
    assert np.array_equal(new, c.k[0])
    for i in range(37):
        at = 300 - 37 + i
        assert np.array_equal(v[int(far[1, at // page]), :, at % page].float().cpu().numpy(), c.v[1 + i])


def test_captured_graph_replays():
    """Append and attention as one captured graph, replayed with other work in between, against the eager calls."""
    import torch
    c = Cache([1, 5, 1], [300, 40, 1500], dim=128, heads=8, kv_heads=2, page=64, seed=16, max_pages=40)
    d = c.device()
    cos, sin = (gie.to_device(t) for t in gie.rotary_tables(40 * 64, 128))
    p = c.p(rotary_dim=128, max_positions=40 * 64, max_len=1500, max_new=5)
    ws = gie.DeviceBuffer(max(16, gie.paged_attention_workspace_size(p)))
    qr, out = c.blank_rows(c.heads), c.blank_rows(c.heads)

    def step(stream):
        gie.kv_append(p, d["k"].addr, d["v"].addr, d["starts"].addr, d["lens"].addr, d["table"].addr, d["k_pages"].addr,
                      d["v_pages"].addr, cos=cos.addr, sin=sin.addr, q=d["q"].addr, q_out=qr.addr, stream=stream)
        gie.paged_attention(p, qr.addr, d["k_pages"].addr, d["v_pages"].addr, d["starts"].addr, d["lens"].addr,
                            d["table"].addr, out.addr, workspace=ws.addr, ws_bytes=ws.nbytes, stream=stream)

    step(None)
    gie.synchronize()
    want = [c.read_rows(out, c.heads)]
    more = [301, 41, 1501]
    d["lens"].upload(np.array(more, np.int32))
    step(None)
    gie.synchronize()
    want.append(c.read_rows(out, c.heads))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for i in (1, 0, 1, 0):
        d["lens"].upload(np.array(more if i else [300, 40, 1500], np.int32))
        out.fill(0xA5)
        ws.fill(0xFF)
        torch.ones(1 << 20, device="cuda").mul_(2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(c.read_rows(out, c.heads), want[i])


# ------------------------------------------------------------------------------------------------- append
def check_append(c, rotary, interleaved, with_q=True, in_place=False, stream=None):
    """Turned values: two products and a sum in FP32 (3 roundings of 2^-24 of |u cos| + |v sin|) and one rounding to the
    storage type; everything else is copied bit for bit."""
    d = c.device()
    rng = np.random.default_rng(rotary)
    rows, half = c.max_pages * c.page, rotary // 2
    cos, sin = (rng.uniform(-1, 1, (rows, half)).astype(np.float32) for _ in range(2))
    dc, ds = (gie.to_device(t) if half else None for t in (cos, sin))
    p = c.p(rotary_dim=rotary, interleaved=interleaved, max_positions=rows)
    q_out = d["q"] if in_place else c.blank_rows(c.heads)
    gie.synchronize()
    print("append", p, c.new, c.lens, flush=True)
    at = 2 * c.offset
    gie.kv_append(p, d["k"].addr + at, d["v"].addr + at, d["starts"].addr, d["lens"].addr, d["table"].addr,
                  d["k_pages"].addr, d["v_pages"].addr, cos=dc.addr if half else None, sin=ds.addr if half else None,
                  q=d["q"].addr + at if with_q else None, q_out=q_out.addr + at if with_q else None, stream=stream)
    gie.synchronize()
    u = UNIT[c.precision]

    def near(got, x):
        want, position, placed = c.rotate(x, rotary, interleaved, cos, sin)
        size = c.rotate(np.abs(x), rotary, interleaved, np.abs(cos), -np.abs(sin))[0]
        other = c.rotate(np.abs(x), rotary, interleaved, np.abs(cos), np.abs(sin))[0]
        size = np.maximum(np.abs(size), np.abs(other))
        slack = 4 * 2.0 ** -24 * size
        assert (np.abs(got - want) <= slack + u * (np.abs(want) + slack) + 2.0 ** -25).all()
        same = np.s_[..., rotary:]
        assert np.array_equal(got[same], want[same].astype(np.float32))
        return want, position, placed

    want_q = c.rotate(c.q, rotary, interleaved, cos, sin)
    if with_q:
        near(c.read_rows(q_out, c.heads), c.q)
    _, position, placed = want_q
    shape = c.k_pages.shape
    k, v = (gie.storage_to_float(d[n].download(np.uint16, c.k_pages.size), c.precision).reshape(shape)
            for n in ("k_pages", "v_pages"))
    seq = np.repeat(np.arange(len(c.new)), c.new)
    touched = np.zeros((c.pages, c.page), bool)
    new_k, new_v = np.zeros_like(c.k), np.zeros_like(c.v)
    for t in range(c.tokens):
        page = c.table[seq[t], position[t] // c.page] if placed[t] else -1
        if 0 <= page < c.pages:
            touched[page, position[t] % c.page] = True
            new_k[t], new_v[t] = k[page, :, position[t] % c.page], v[page, :, position[t] % c.page]
        else:  # not stored: nothing to compare
            new_k[t] = gie.storage_to_float(gie.host_to_storage(c.rotate(c.k, rotary, interleaved, cos, sin)[0][t].astype(np.float32), c.precision), c.precision)
            new_v[t] = c.v[t] if placed[t] else 0
    near(new_k, c.k)
    assert np.array_equal(new_v[placed], c.v[placed])
    for now, before in ((k, c.k_pages), (v, c.v_pages)):
        assert np.array_equal(now.transpose(0, 2, 1, 3)[~touched], before.transpose(0, 2, 1, 3)[~touched]), "other slots"


APPENDS = {"one": ([1], [1]), "step": ([1] * 7, [1, 16, 17, 31, 32, 33, 100]), "chunks": ([5, 0, 33, 70], [5, 9, 50, 133])}


@pytest.mark.parametrize("precision", ["fp16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 0), (96, 64), (128, 128), (128, 32), (256, 256), (128, 6), (96, 96), (64, 2)])
def test_append(dim, rotary, interleaved, precision):
    for batch in sorted(APPENDS):
        check_append(Cache(*APPENDS[batch], dim=dim, precision=precision, seed=rotary), rotary, interleaved)


@pytest.mark.parametrize("heads,kv_heads,page", [(1, 1, 16), (3, 3, 48), (32, 8, 64), (5, 1, 32), (40, 8, 16)])
def test_append_heads_and_pages(heads, kv_heads, page):
    check_append(Cache([3, 40], [9, 100], heads=heads, kv_heads=kv_heads, dim=128, page=page, seed=heads), 128, False)
    check_append(Cache([3, 40], [9, 100], heads=heads, kv_heads=kv_heads, dim=128, page=page, seed=heads), 128, True,
                 with_q=False)


@pytest.mark.parametrize("gap,offset", [(8, 0), (3, 0), (0, 1), (5, 7), (64, 8)])
@pytest.mark.parametrize("in_place", [False, True])
def test_append_strides_and_alignment(gap, offset, in_place):
    for interleaved in (False, True):
        check_append(Cache(*APPENDS["chunks"], dim=96, gap=gap, offset=offset, seed=gap), 64, interleaved, in_place=in_place)


def test_append_without_room():
    check_append(Cache([20, 3, 1], [7, 3, 0], dim=64, seed=1), 64, False)
    check_append(Cache([20, 40], [70, 30], dim=64, max_pages=4, seed=2), 32, True)
    c = Cache([3, 40], [100, 60], dim=128, seed=12)
    c.table[0, 6] = -1
    c.table[1, 1] = c.pages
    c.table[1, 3] = 2 ** 31 - 1
    check_append(c, 128, False, stream=gie.Stream())


def test_many_sequences():
    """Batches past 64 and 4096 sequences: the search for a row's sequence takes another round."""
    for batch in (65, 130, 4100):
        rng = np.random.default_rng(batch)
        new = rng.integers(0, 3, batch).tolist()
        lens = [n + int(rng.integers(0, 20)) for n in new]
        check_append(Cache(new, lens, heads=2, kv_heads=1, dim=64, seed=batch), 64, False)
        if batch < 4000:
            check(Cache(new, lens, heads=2, kv_heads=1, dim=64, seed=batch))


def test_no_tokens_is_no_work():
    c = Cache([0, 0], [5, 9], dim=64)
    assert gie.paged_attention_workspace_size(c.p()) >= 0
    p = gie.PagedKv(0, 0, 2, 1, 64, 16, 1, 1)
    gie.paged_attention(p, 0, 0, 0, 0, 0, 0, 0)
    gie.kv_append(p, 0, 0, 0, 0, 0, 0, 0)
    gie.synchronize()
