"""What PagedKv::append_normed and PagedKv8 refuse, with which status. Needs no GPU: every refusal comes from the host's
checks before anything is enqueued. And the plain forms' own arithmetic (tests/kv8_plain.py)."""
import ctypes
import math

import numpy as np
import pytest

import gie
from kv8_plain import E4M3, decode, encode, encode_e4m3, scale_for

A, B, C, W, S, T, KS, VS = (0x10000 * i for i in range(1, 9))  # addresses that are never read
EINVAL, EUNSUPPORTED = -1, -2


def status(f, *a, **k):
    with pytest.raises(gie.GieError) as e:
        f(*a, **k)
    return e.value.status


def paged(**k):
    return gie.PagedKv(**{**dict(batch=2, total_tokens=3, q_heads=8, kv_heads=2, head_dim=64, page_size=16, num_pages=8,
                                 max_pages=4, cache="int8"), **k})


def append8(p, **k):
    gie.kv8_append(p, **{**dict(k=A, v=B, q_starts=S, seq_lens=S, page_table=T, k_pages=C, v_pages=W, k_scales=KS,
                                v_scales=VS), **k})


def normed(p, **k):
    gie.kv_append_normed(p, **{**dict(k=A, v=B, q_starts=S, seq_lens=S, page_table=T, k_pages=C, v_pages=W), **k})


def read8(p, **k):
    gie.kv8_read(p, **{**dict(k_pages=C, v_pages=W, k_scales=KS, v_scales=VS, q_starts=S, seq_lens=S, page_table=T, k=A,
                              v=B), **k})


def attend8(p, **k):
    gie.kv8_attention(p, **{**dict(q=A, k_pages=C, v_pages=W, k_scales=KS, v_scales=VS, q_starts=S, seq_lens=S,
                                   page_table=T, out=B, workspace=W, ws_bytes=1 << 40), **k})


@pytest.mark.parametrize("bad", [
    dict(batch=-1), dict(total_tokens=-1), dict(batch=0), dict(q_heads=7), dict(head_dim=0), dict(page_size=0),
    dict(q_stride=511), dict(k_stride=127), dict(v_stride=127), dict(o_stride=511), dict(rotary_dim=31),
    dict(rotary_dim=66), dict(window=-1), dict(sinks=-1), dict(norm_eps=-1e-6), dict(norm_eps=math.nan),
    dict(norm_eps=math.inf), dict(softcap=-1.0), dict(scale=math.nan)])
def test_bad_problems(bad):
    for call in (gie.kv8_attention_workspace_size, append8, read8, attend8):
        assert status(call, paged(**bad)) == "InvalidArgument"
    for call in (gie.paged_attention_workspace_size, normed):
        assert status(call, paged(**bad, cache="")) == "InvalidArgument"


@pytest.mark.parametrize("bad", [dict(precision="fp32"), dict(head_dim=80), dict(page_size=8), dict(max_pages=1 << 27),
                                 dict(batch=1 << 30)])
def test_unsupported(bad):
    for call in (gie.kv8_attention_workspace_size, append8, read8, attend8):
        assert status(call, paged(**bad)) == "Unsupported"
    assert status(normed, paged(**bad, cache="")) == "Unsupported"


def test_calls_go_with_what_the_pages_hold():
    for call in (gie.kv8_attention_workspace_size, append8, read8, attend8):
        assert status(call, paged(cache="")) == "InvalidArgument"
    assert status(normed, paged()) == "InvalidArgument"
    assert status(gie.paged_attention_workspace_size, paged()) == "InvalidArgument"
    assert status(gie.paged_attention, paged(), A, C, W, S, S, T, B) == "InvalidArgument"
    assert status(gie.kv_append, paged(), A, B, S, S, T, C, W) == "InvalidArgument"
    p = paged()
    p._c.code = 3
    assert status(append8, p) == "InvalidArgument"


POINTERS = [dict(k_pages=0), dict(v_pages=0), dict(q_starts=0), dict(seq_lens=0), dict(page_table=0), dict(k_pages=C + 8),
            dict(v_pages=C), dict(q_starts=S + 2)]
SCALES = [dict(k_scales=0), dict(v_scales=0), dict(k_scales=VS), dict(k_scales=KS + 2)]
ROWS = [dict(k=0), dict(v=0), dict(k=A + 1), dict(q=A), dict(q_out=A), dict(q_norm=T), dict(k_norm=T + 2),
        dict(q=A, q_out=B, q_norm=T + 1)]


@pytest.mark.parametrize("bad", POINTERS + SCALES + ROWS)
def test_append8_refuses_bad_pointers(bad):
    assert status(append8, paged(), **bad) == "InvalidArgument"


@pytest.mark.parametrize("bad", POINTERS + ROWS)
def test_append_normed_refuses_bad_pointers(bad):
    assert status(normed, paged(cache=""), **bad) == "InvalidArgument"


@pytest.mark.parametrize("bad", POINTERS + SCALES + [dict(k=A + 1), dict(v=B + 1), dict(k=B)])
def test_read_refuses_bad_pointers(bad):
    assert status(read8, paged(), **bad) == "InvalidArgument"


@pytest.mark.parametrize("bad", POINTERS + SCALES + [dict(q=0), dict(out=0), dict(out=A), dict(q=A + 1)])
def test_attention_refuses_bad_pointers(bad):
    assert status(attend8, paged(), **bad) == "InvalidArgument"


def test_appends_refuse_tables_that_do_not_fit():
    for call, cache in ((append8, "fp8"), (normed, "")):
        assert status(call, paged(cache=cache, rotary_dim=64, max_positions=64)) == "InvalidArgument"                # no tables
        assert status(call, paged(cache=cache, rotary_dim=64, max_positions=63), cos=A, sin=A) == "InvalidArgument"  # too short
        assert status(call, paged(cache=cache, q_stride=600), q=A, q_out=A) == "InvalidArgument"                     # in place


def test_attention_workspace_is_checked():
    p = paged(batch=1, total_tokens=1, max_pages=4096, max_new=1, max_len=65536)
    n = gie.kv8_attention_workspace_size(p)
    if n:
        assert status(attend8, p, ws_bytes=n - 1) == "WorkspaceTooSmall"
        assert status(attend8, p, workspace=None, ws_bytes=0) == "WorkspaceTooSmall"
        assert status(attend8, p, workspace=W + 4) == "InvalidArgument"
    assert gie.kv8_attention_workspace_size(paged(total_tokens=0, max_pages=4096, max_len=65536)) == 0


def geom(**k):
    d = dict(batch=2, total_tokens=3, q_heads=8, kv_heads=2, head_dim=64, page_size=16, num_pages=8, max_pages=4, q_stride=512,
             k_stride=128, v_stride=128, o_stride=512, scale=0.125)
    return gie.GiePagedGeom(**{**d, **k})


def kernels(code=1, dtype=None, **k):
    """The kernels' own entry points: their statuses."""
    g, dt = ctypes.byref(geom(**k)), gie.FP16 if dtype is None else dtype
    h = gie.hip()
    return [h.gie_hip_kv8_append(dt, code, g, A, A, B, T, T, None, None, S, S, T, B, C, W, KS, VS, None),
            h.gie_hip_kv8_read(dt, code, g, C, W, KS, VS, S, S, T, A, B, None),
            h.gie_hip_kv8_attention(dt, code, g, A, C, W, KS, VS, S, S, T, B, A, 1 << 60, None)]


def test_kernel_entries_refuse():
    for bad in (dict(code=0), dict(code=3), dict(batch=-1), dict(page_size=24), dict(head_dim=40), dict(sinks=-1), dict(q_stride=5)):
        assert kernels(**bad) == [EINVAL] * 3, bad
    assert kernels(dtype=gie.FP32) == [EUNSUPPORTED] * 3
    assert kernels(head_dim=32, q_stride=512) == [EUNSUPPORTED] * 3
    h = gie.hip()
    for eps in (-1.0, math.nan, math.inf):
        g = ctypes.byref(geom(norm_eps=eps))
        assert h.gie_hip_kv8_append(gie.FP16, 1, g, A, A, B, T, T, None, None, S, S, T, B, C, W, KS, VS, None) == EINVAL
        assert h.gie_hip_kv_append_normed(gie.FP16, g, A, A, B, T, T, None, None, S, S, T, B, C, W, None) == EINVAL
    for bad in (dict(scale=0.0), dict(scale=math.inf), dict(softcap=math.inf)):
        g = ctypes.byref(geom(**bad))
        assert h.gie_hip_kv8_attention(gie.FP16, 1, g, A, C, W, KS, VS, S, S, T, B, A, 1 << 60, None) == EINVAL


def test_launches_past_their_limits_are_refused():
    """More threads than a launch takes; refused before anything is enqueued."""
    h, many = gie.hip(), 1 << 29
    g = ctypes.byref(geom(total_tokens=many, q_heads=2, q_stride=128, o_stride=128, batch=1))
    assert h.gie_hip_kv8_append(gie.FP16, 1, g, A, A, B, None, None, None, None, S, S, T, B, C, W, KS, VS, None) == EUNSUPPORTED
    assert h.gie_hip_kv8_read(gie.FP16, 1, g, C, W, KS, VS, S, S, T, A, B, None) == EUNSUPPORTED
    assert h.gie_hip_kv_append_normed(gie.FP16, g, A, A, B, T, T, None, None, S, S, T, B, C, W, None) == EUNSUPPORTED
    g = ctypes.byref(geom(total_tokens=1, batch=many))
    assert h.gie_hip_kv8_append(gie.FP16, 1, g, A, A, B, None, None, None, None, S, S, T, B, C, W, KS, VS, None) == EUNSUPPORTED


# ---- the plain forms themselves
def test_e4m3_codes():
    assert E4M3[0x01] == 2.0 ** -9 and E4M3[0x08] == 2.0 ** -6 and E4M3[0x38] == 1.0 and E4M3[0x7e] == 448.0 and E4M3[0xfe] == -448.0
    codes = np.array([c for c in range(256) if c & 0x7f != 0x7f], np.uint8)
    assert np.array_equal(encode_e4m3(E4M3[codes])[codes != 0x80], codes[codes != 0x80])
    mid = (E4M3[:126] + E4M3[1:127]) / 2  # ties go to the even code
    assert (encode_e4m3(mid) % 2 == 0).all()


def test_scales_and_codes_stay_in_range():
    rng = np.random.default_rng(0)
    for cache, largest in (("int8", 127), ("fp8", 448)):
        most = np.concatenate([[0.0, 2.0 ** -70, 448.0, 896.0, 447.9, 448.1, 3e38], np.exp(rng.uniform(-60, 60, 1000))]).astype(np.float32)
        scale = scale_for(most, cache)
        assert (scale > 0).all() and np.isfinite(scale).all()
        top = decode(encode(most, scale, cache), cache)
        assert (np.abs(top) <= largest).all()
        real = most >= 2.0 ** -64
        assert (top[real] >= (127 if cache == "int8" else 224)).all()
