"""PagedKv8::attention at the ends of BF16's range: what an append may write has to count as it reads. Bounds as in
tests/kv8_plain.py."""
import numpy as np
import pytest

import gie
from kv8_plain import Cache8, attention, scale_for

pytestmark = pytest.mark.gpu
CACHES = ["int8", "fp8"]
DIMS = [64, 96, 128, 256]
LARGEST = float(np.float32(np.finfo(np.float32).max) * np.float32(0.99))
BATCHES = [([1, 1], [90, 300]), ([70], [200])]


def check(c, **kw):
    got = c.attend(**kw).astype(np.float64)
    want, bound = attention(c, **{k: v for k, v in kw.items() if k in ("scale", "softcap")})
    assert np.isfinite(got).all()
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), (float(off.max()), np.argwhere(off > 0)[:4].tolist(), int((off > 0).sum()))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", DIMS)
def test_blocks_of_the_largest_values(dim, cache):
    """Scales of V as an append writes them for values of 3.4e38 (int8: 2^121)."""
    for new, lens in BATCHES:
        c = Cache8(new, lens, dim=dim, precision="bf16", cache=cache, seed=1)
        c.v_scales[:] = scale_for(LARGEST, cache)
        if cache == "fp8":  # codes within 224, so that no value passes FP32's range
            c.v_pages = np.where((c.v_pages & 0x7f) > 0x76, 0x76, c.v_pages).astype(np.uint8)
        check(c)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("dim", DIMS)
def test_keys_of_the_largest_values(dim, softcap, cache):
    """Scales of K likewise, with queries and a scale of the scores that make ordinary ones of them."""
    for new, lens in BATCHES:
        c = Cache8(new, lens, dim=dim, precision="bf16", cache=cache, seed=2)
        c.k_scales[:] = scale_for(LARGEST, cache)
        if cache == "fp8":
            c.k_pages = np.where((c.k_pages & 0x7f) > 0x76, 0x76, c.k_pages).astype(np.uint8)
        c.q = c.q * np.float32(2.0 ** -95)  # exact in BF16
        check(c, scale=2.0 ** -33, softcap=softcap)


@pytest.mark.parametrize("cache", CACHES)
def test_append_and_attention_agree_on_the_largest(cache):
    """A sequence of one value: attention gives it back, whatever the weights."""
    c = Cache8([20], [20], dim=64, precision="bf16", cache=cache, seed=3)
    x = float(gie.storage_to_float(gie.host_to_storage(np.array([3.0e38 if cache == "int8" else 2.0 ** 127], np.float32), "bf16"), "bf16")[0])
    c.v[:] = x
    c.q[:] = 0
    d = c.device()
    gie.kv8_append(c.p(), d["k"].addr, d["v"].addr, d["starts"].addr, d["lens"].addr, d["table"].addr, d["k_pages"].addr,
                   d["v_pages"].addr, d["k_scales"].addr, d["v_scales"].addr)
    gie.synchronize()
    got = c.attend(d=d)
    # one code, half a step of it (int8 127 is exact up to the scale's rounding), and BF16's rounding
    assert (np.abs(got - x) <= (2.0 ** -8 + 2.0 ** -12) * x).all()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", DIMS)
def test_blocks_of_values_2_to_the_100_apart(dim, cache):
    """Weights of the smaller blocks count in the sum in full, whichever block comes first, in one part and in joined ones."""
    for new, lens, hints in (([1, 1], [90, 300], {}), ([70], [200], {}), ([1], [3000], dict(max_new=1, max_len=3000))):
        for first in (0, 1):
            c = Cache8(new, lens, dim=dim, heads=2, kv_heads=1, page=16, precision="bf16", cache=cache, seed=4)
            for j in range(c.max_pages):
                c.v_scales[c.table[0, j]] *= np.float32(2.0 ** (50 if j % 2 == first else -50))
            got = c.attend(**hints).astype(np.float64)
            want, bound = attention(c)
            assert (np.abs(got - want) <= bound).all()
