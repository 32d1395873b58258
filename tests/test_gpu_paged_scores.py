"""PagedKv::attention where its scores are hardest to hold: caps far above every score and far below them."""
import numpy as np
import pytest

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
