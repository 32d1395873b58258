"""PagedKv::attention where its scores and weights are hardest to hold: caps far above every score and far below them,
a key that outweighs a long rest of the cache by more than the storage type's steps reach, scores of millions."""
import numpy as np
import pytest

import gie
from paged_plain import TINY, UNIT, Cache

pytestmark = pytest.mark.gpu


def capped(c, cap):
    """The attention with capped scores in 64 bits, and a bound that a cap does not widen: scores as an uncapped call
    has them (paged_plain.Cache.plain: (D + 4) 2^-24 sum|scale q k| =: e), the cap 2^-19 of the capped score more
    (products, 2^x and a reciprocal in FP32, each within 2^-22 of itself where the quotient is not under 0.2); the
    cap's slope is at most 1, so it does not magnify e."""
    out = np.zeros((c.tokens, c.heads, c.dim))
    bound = np.zeros_like(out)
    u, tiny, group = UNIT[c.precision], TINY[c.precision], c.heads // c.kv
    for b, (n, length) in enumerate(zip(c.new, c.lens)):
        for i in range(n):
            keys = np.arange(length - n + i + 1)
            page, slot = c.table[b, keys // c.page], keys % c.page
            k, v = c.k_pages[page, :, slot].astype(np.float64), c.v_pages[page, :, slot].astype(np.float64)
            t = c.starts[b] + i
            for h in range(c.heads):
                q = c.q[t, h].astype(np.float64)
                s = k[:, h // group] @ q * c.dim ** -0.5
                size = np.abs(k[:, h // group]) @ np.abs(q)
                e = (c.dim + 4) * 2.0 ** -24 * size[np.isfinite(size)].max() * c.dim ** -0.5
                s = cap * np.tanh(s / cap)
                e += 2.0 ** -19 * np.abs(s).max()
                w = np.exp(s - s.max())
                w /= w.sum()
                o, size = w @ v[:, h // group], w @ np.abs(v[:, h // group])
                inner = (u + 4 * e + 2.0 ** -18 + len(keys) * 2.0 ** -23) * size
                inner += tiny * 2 ** 8 * np.abs(v[:, h // group]).sum(0)
                out[t, h] = o
                bound[t, h] = inner + u * (np.abs(o) + inner) + tiny
    return out, bound


def check(c, cap):
    got = c.attend(softcap=cap).astype(np.float64)
    want, bound = capped(c, cap)
    off = np.abs(got - want) - bound
    assert np.isfinite(got).all() and (off <= 0).all(), (cap, float(off.max()), int((off > 0).sum()))


CAPS = [1e-30, 0.5, 3.0, 50.0, 1e3, 1e4, 1e5, 1e6, 1e9, 1e30, 3e38]


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("dim,precision", [(64, "fp16"), (96, "bf16"), (128, "fp16"), (256, "bf16"), (256, "fp16")])
def test_caps_of_any_size(cap, dim, precision):
    """Scores around 1, and around 8: against the smaller caps some lie on either side of the form's change."""
    for batch in (([3, 1, 2], [300, 77, 16]), ([70], [150])):
        c = Cache(*batch, dim=dim, precision=precision, seed=dim)
        check(c, cap)
        c.q *= 8
        check(c, cap)


def test_a_cap_in_reach_of_no_score_changes_nothing():
    """Far above the scores the cap is the identity to the last bit of a score."""
    for new, lens in (([40], [200]), ([1], [200])):
        c = Cache(new, lens, dim=128, seed=1)
        plain = c.attend()
        for cap in (1e12, 1e30, 3e38):
            off = np.abs(c.attend(softcap=cap) - plain)
            assert (off <= 2 * UNIT["fp16"] * (np.abs(plain) + 0.01)).all(), (cap, float(off.max()))


@pytest.mark.parametrize("cap", [64.0, 65.0, 200.0, 1000.0])
@pytest.mark.parametrize("dim,precision", [(64, "bf16"), (128, "fp16"), (256, "bf16")])
def test_scores_on_either_side_of_a_large_cap(cap, dim, precision):
    """Scores of tens and hundreds beside scores around 1: some keys past the cap, some far below it."""
    for batch in (([3, 1], [300, 77]), ([70], [150])):
        c = Cache(*batch, dim=dim, precision=precision, seed=dim + 1)
        c.q *= 8
        c.k_pages[::2] *= 16
        check(c, cap)


@pytest.mark.parametrize("cap", [30.0, 100.0])
def test_a_key_that_is_infinite_scores_the_cap(cap):
    c = Cache([1, 40], [50, 60], dim=64, seed=4)
    c.q = np.abs(c.q)
    c.k_pages[c.table[0, 2], :, 5, 3] = np.inf  # position 37 of the first sequence
    c.k_pages[c.table[1, 0], :, 7, 9] = -np.inf  # position 7 of the second
    check(c, cap)


@pytest.mark.parametrize("gap", [20.0, 23.4, 25.2, 27.0])
@pytest.mark.parametrize("new", [1, 33])
@pytest.mark.parametrize("precision", ["fp16", "bf16"])
def test_small_weights_of_a_long_cache_are_not_lost(gap, new, precision):
    """One key at the front and a rest of 2^17 - 1 whose weights are 2^-gap of its own, in one part or in few (the batch fills
    the device). All values are 1, so the result is too, if what the sum of the weights counts also enters the product.

    Bound: a weight is rounded once (u), or to within 2^-32 of the first key's in FP16's last steps (its weights are
    at least 2^7 at the maximum); n / 16 and n / 32 additions in FP32 follow one another in the product and in the
    sum; the argument of 2^x is off by the score's rounding in FP32 (2^-24 of up to 32), and its result by 2^-22."""
    import torch
    dim, kv, page, batch, n = 64, 64, 256, 4, 1 << 17
    pages = n // page
    dtype = torch.float16 if precision == "fp16" else torch.bfloat16
    k, v = (torch.zeros((pages, kv, page, dim), dtype=dtype, device="cuda") for _ in range(2))
    v += 1
    # scores in powers of 2: q k log2(e) scale, all of it exact in the storage type but the scale
    k[:, :, :, 0] = -1
    k[0, :, 0, 0] = 0
    q = torch.zeros((batch * new, kv, dim), dtype=dtype, device="cuda")
    q[:, :, 0] = 1
    scale = float(np.float32(gap * np.log(2.0)))
    out = torch.full_like(q, 7)
    starts = torch.arange(0, batch * new + 1, new, dtype=torch.int32).cuda()
    lens = torch.full((batch,), n, dtype=torch.int32).cuda()
    table = torch.arange(pages, dtype=torch.int32).repeat(batch, 1).contiguous().cuda()
    p = gie.PagedKv(batch, batch * new, kv, kv, dim, page, pages, pages, precision=precision, scale=scale, max_new=new,
                    max_len=n)
    size = gie.paged_attention_workspace_size(p)
    ws = gie.DeviceBuffer(max(16, size))
    torch.cuda.synchronize()
    print("attend", p, flush=True)
    gie.paged_attention(p, q.data_ptr(), k.data_ptr(), v.data_ptr(), starts.data_ptr(), lens.data_ptr(), table.data_ptr(),
                        out.data_ptr(), workspace=ws.addr, ws_bytes=size)
    torch.cuda.synchronize()
    u, rest = UNIT[precision], n * 2.0 ** -gap
    share = rest / (1 + rest)
    small = 2.0 ** -32 * n / (1 + rest) if precision == "fp16" else 0
    bound = u * share + small + (n / 16 + n / 32 + 40) * 2.0 ** -24 * share + 2.0 ** -17 * share
    bound += u * (1 + bound)
    worst = float((out.float() - 1).abs().max())
    assert worst <= bound, (worst, bound)


@pytest.mark.parametrize("k0,step", [(512, 1), (10240, 2), (24576, 4)])  # scores of 1e6, 2.1e7 and 5e7
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("precision", ["fp16", "bf16"])
def test_scores_of_millions(k0, step, new, precision):
    """Every 32 keys a score that is larger by one step of FP32 (or 1): all of them exact, so that the weights are
    exp(step * i) whatever the scores' size is. Bound: weights and result rounded once, 2^x within 2^-20 of itself."""
    c = Cache([new], [320], dim=64, heads=2, kv_heads=1, precision=precision, seed=3)
    block = np.arange(320) // 32
    c.q[:] = 0
    c.q[..., 0], c.q[..., 1] = 2048, 1
    c.k_pages[:] = 0
    for j in range(320):
        c.k_pages[c.table[0, j // c.page], :, j % c.page, :2] = k0, step * block[j]
    got = c.attend(scale=1.0).astype(np.float64)
    v = c.v_pages[c.table[0, np.arange(320) // c.page], 0, np.arange(320) % c.page].astype(np.float64)
    u = UNIT[precision]
    for i in range(new):
        seen = 320 - new + i + 1
        w = np.exp(step * (block[:seen] - block[seen - 1]).astype(np.float64))
        w /= w.sum()
        want, size = w @ v[:seen], w @ np.abs(v[:seen])
        bound = (u + 2.0 ** -20 + seen * 2.0 ** -24 + 2.0 ** -16) * size
        bound += u * (np.abs(want) + bound) + TINY[precision]
        assert (np.abs(got[i] - want) <= bound).all(), (k0, i, float((np.abs(got[i] - want) - bound).max()))
