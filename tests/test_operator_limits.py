"""Refusals of the kernels' own C-ABI (gie_hip_*) and limits on sizes. Needs no GPU: each call returns from the host's
checks before anything is enqueued."""
import ctypes
import math

import pytest

import gie

A, B, C, W, S, T = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 0x60000  # addresses that are never read
EINVAL, EUNSUPPORTED = -1, -2


def geom(**k):
    d = dict(batch=2, total_tokens=3, q_heads=8, kv_heads=2, head_dim=64, page_size=16, num_pages=8, max_pages=4,
             q_stride=512, k_stride=128, v_stride=128, o_stride=512, scale=0.125)
    return gie.GiePagedGeom(**{**d, **k})


def attend(**k):
    return gie.hip().gie_hip_paged_attention(gie.FP16, ctypes.byref(geom(**k)), A, C, W, S, S, T, B, W, 1 << 40, None)


@pytest.mark.parametrize("bad", [dict(scale=0.0), dict(scale=-0.0), dict(scale=math.inf), dict(scale=-math.inf),
                                 dict(scale=math.nan), dict(softcap=math.inf), dict(softcap=math.nan)])
def test_attention_refuses_scales_without_an_answer(bad):
    # a scale of 0 times a masked score is a NaN; 0 stands for the default in PagedKvProblem only
    assert attend(**bad) == EINVAL


def paged(**k):
    d = dict(batch=1, total_tokens=1, q_heads=8, kv_heads=2, head_dim=256, page_size=16, num_pages=8, max_pages=4)
    return gie.PagedKv(**{**d, **k})


@pytest.mark.parametrize("heads", [dict(q_heads=1 << 25, kv_heads=1), dict(q_heads=1 << 23, kv_heads=1 << 23),
                                   dict(q_heads=1 << 22, kv_heads=1 << 21)])
def test_heads_past_their_offsets_are_refused(heads):
    """The kernels place a head within its token by a 32-bit offset, and count a token's pieces in 32 bits."""
    p = paged(**heads)
    for call in (lambda: gie.paged_attention_workspace_size(p),
                 lambda: gie.kv_append(p, A, B, S, S, T, C, W),
                 lambda: gie.paged_attention(p, A, C, W, S, S, T, B, workspace=W, ws_bytes=1 << 40)):
        with pytest.raises(gie.GieError) as e:
            call()
        assert e.value.status == "Unsupported"
    wide = dict(batch=1, total_tokens=1, head_dim=256, q_stride=1 << 34, o_stride=1 << 34, k_stride=1 << 33,
                v_stride=1 << 33, **heads)
    assert attend(**wide) == EINVAL
    g = geom(**wide)
    assert gie.hip().gie_hip_kv_append(gie.FP16, ctypes.byref(g), None, A, B, None, None, S, S, T, None, C, W, None) == EINVAL


@pytest.mark.parametrize("dtype", [gie.FP32, gie.FP16, gie.BF16])
def test_quantize_rows_refuses_rows_past_its_counters(dtype):
    """A row's last step would wrap the 32-bit counter of its values."""
    for features in ((1 << 30) + 1, (1 << 31) - 1):
        n = 1 << 31
        assert gie.hip().gie_hip_quantize_rows(dtype, A, n, 1, features, B, n, S, None) == EUNSUPPORTED


def test_linear_refuses_too_many_tiles_before_it_quantizes():
    g = gie.GieLinearGeom(1 << 20, 64, 1 << 20, 64, 64, 1 << 20, 0)
    assert gie.hip().gie_hip_linear_i8(gie.FP16, ctypes.byref(g), A, None, B, S, None, C, W, 1 << 60, None) == EUNSUPPORTED


@pytest.mark.parametrize("tokens,out", [((1 << 31) - 1, 1), (17, (1 << 31) - 1), ((1 << 31) - 60, 200)])
def test_linear_counts_tiles_in_64_bits(tokens, out):
    g = gie.GieLinearGeom(tokens, 16, out, 16, 16, out, 0)
    assert gie.hip().gie_hip_linear_i8(gie.FP16, ctypes.byref(g), A, S, B, S, None, C, W, 1 << 60, None) == EUNSUPPORTED


def test_linear_workspace_that_is_needed_is_checked():
    p = gie.LinearI8(64, 512, 128)  # tokens quantized into it
    n = gie.linear_i8_workspace_size(p)
    assert n >= 64 * 512 + 64 * 4
    for workspace, ws_bytes, want in ((W, n - 1, "WorkspaceTooSmall"), (None, 0, "WorkspaceTooSmall"),
                                      (None, n, "WorkspaceTooSmall"), (W + 8, n, "InvalidArgument")):
        with pytest.raises(gie.GieError) as e:
            gie.linear_i8(p, A, B, S, C, workspace=workspace, ws_bytes=ws_bytes)
        assert e.value.status == want


def test_attention_workspace_that_is_needed_is_checked():
    p = gie.PagedKv(1, 1, 8, 2, 64, 16, 8, 4096, max_new=1, max_len=65536)
    n = gie.paged_attention_workspace_size(p)
    assert n > 0
    for workspace, ws_bytes, want in ((W, n - 1, "WorkspaceTooSmall"), (None, 0, "WorkspaceTooSmall"),
                                      (W + 4, n, "InvalidArgument")):
        with pytest.raises(gie.GieError) as e:
            gie.paged_attention(p, A, C, B, S, S, T, W, workspace=workspace, ws_bytes=ws_bytes)
        assert e.value.status == want


def test_no_tokens_need_no_workspace():
    assert gie.paged_attention_workspace_size(gie.PagedKv(2, 0, 8, 2, 64, 16, 8, 4096, max_len=65536)) == 0
