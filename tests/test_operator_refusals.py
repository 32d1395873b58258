"""What LinearI8 and PagedKv refuse, with which status, and the host tables of the rotation. Needs no GPU: every refusal
comes from the host's checks before anything is enqueued."""
import math

import numpy as np
import pytest

import gie

A, B, C, W, S, T = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 0x60000  # addresses that are never read


def status(f, *a, **k):
    with pytest.raises(gie.GieError) as e:
        f(*a, **k)
    return e.value.status


def linear(**k):
    d = dict(tokens=4, in_features=64, out_features=32)
    d.update(k)
    return gie.LinearI8(**d)


@pytest.mark.parametrize("bad", [dict(tokens=-1), dict(in_features=0), dict(out_features=0), dict(out_features=-3),
                                 dict(ld_x=63), dict(ld_w=10), dict(ld_y=31), dict(ld_x=-64)])
def test_linear_refuses_bad_extents(bad):
    assert status(gie.linear_i8_workspace_size, linear(**bad)) == "InvalidArgument"
    assert status(gie.linear_i8, linear(**bad), A, B, S, C, workspace=W, ws_bytes=1 << 20) == "InvalidArgument"
    assert status(gie.quantize_rows, linear(**bad), A, B, S) == "InvalidArgument"


@pytest.mark.parametrize("bad", [dict(precision="tf32"), dict(in_features=131072)])
def test_linear_unsupported(bad):
    assert status(gie.linear_i8_workspace_size, linear(**bad)) == "Unsupported"


@pytest.mark.parametrize("call", [
    dict(x=0), dict(w=0), dict(w_scale=0), dict(y=0), dict(x_scale=S), dict(bias=T), dict(x=A + 1), dict(y=C + 1),
    dict(w_scale=S + 2), dict(y=A), dict(workspace=W + 8)])
def test_linear_refuses_bad_pointers(call):
    d = dict(x=A, w=B, w_scale=S, y=C, workspace=W, ws_bytes=1 << 20)
    d.update(call)
    x, w, w_scale, y = (d.pop(n) for n in ("x", "w", "w_scale", "y"))
    assert status(gie.linear_i8, linear(), x, w, w_scale, y, **d) == "InvalidArgument"


def test_linear_scales_and_bias_go_with_the_problem():
    assert status(gie.linear_i8, linear(quantized=True), A, B, S, C, workspace=W, ws_bytes=1 << 20) == "InvalidArgument"
    assert status(gie.linear_i8, linear(has_bias=True), A, B, S, C, workspace=W, ws_bytes=1 << 20) == "InvalidArgument"


def test_linear_workspace_is_checked():
    p = linear()
    n = gie.linear_i8_workspace_size(p)
    if n:
        assert status(gie.linear_i8, p, A, B, S, C, workspace=W, ws_bytes=n - 1) == "WorkspaceTooSmall"
        assert status(gie.linear_i8, p, A, B, S, C) == "WorkspaceTooSmall"


def paged(**k):
    d = dict(batch=2, total_tokens=3, q_heads=8, kv_heads=2, head_dim=64, page_size=16, num_pages=8, max_pages=4)
    d.update(k)
    return gie.PagedKv(**d)


def append(p, **k):
    d = dict(k=A, v=B, q_starts=S, seq_lens=S, page_table=T, k_pages=C, v_pages=W)
    d.update(k)
    gie.kv_append(p, **d)


def attend(p, **k):
    d = dict(q=A, k_pages=C, v_pages=W, q_starts=S, seq_lens=S, page_table=T, out=B, workspace=W, ws_bytes=1 << 40)
    d.update(k)
    gie.paged_attention(p, **d)


@pytest.mark.parametrize("bad", [
    dict(batch=-1), dict(total_tokens=-1), dict(batch=0), dict(q_heads=0), dict(kv_heads=0), dict(q_heads=7),
    dict(head_dim=0), dict(page_size=0), dict(num_pages=0), dict(max_pages=0), dict(q_stride=511), dict(k_stride=127),
    dict(v_stride=127), dict(o_stride=511), dict(rotary_dim=31), dict(rotary_dim=66), dict(rotary_dim=-2),
    dict(window=-1), dict(max_new=-1), dict(max_len=-1), dict(softcap=-1.0), dict(softcap=math.inf),
    dict(scale=math.nan)])
def test_paged_refuses_bad_problems(bad):
    assert status(gie.paged_attention_workspace_size, paged(**bad)) == "InvalidArgument"
    assert status(append, paged(**bad)) == "InvalidArgument"
    assert status(attend, paged(**bad)) == "InvalidArgument"


@pytest.mark.parametrize("bad", [dict(precision="fp32"), dict(precision="tf32"), dict(head_dim=80),
                                 dict(head_dim=512), dict(page_size=8), dict(page_size=17),
                                 dict(max_pages=1 << 27)])
def test_paged_unsupported(bad):
    assert status(gie.paged_attention_workspace_size, paged(**bad)) == "Unsupported"
    assert status(append, paged(**bad)) == "Unsupported"
    assert status(attend, paged(**bad)) == "Unsupported"


@pytest.mark.parametrize("bad", [
    dict(k=0), dict(v=0), dict(k_pages=0), dict(v_pages=0), dict(q_starts=0), dict(seq_lens=0), dict(page_table=0),
    dict(k_pages=C + 8), dict(v_pages=C), dict(k=A + 1), dict(q=A), dict(q_out=A), dict(q_starts=S + 2)])
def test_append_refuses_bad_pointers(bad):
    assert status(append, paged(), **bad) == "InvalidArgument"


def test_append_refuses_tables_that_do_not_fit():
    assert status(append, paged(rotary_dim=64, max_positions=64)) == "InvalidArgument"                  # no tables
    assert status(append, paged(rotary_dim=64, max_positions=63), cos=A, sin=A) == "InvalidArgument"    # too short
    assert status(append, paged(q_stride=600), q=A, q_out=A) == "InvalidArgument"                       # in place


@pytest.mark.parametrize("bad", [dict(q=0), dict(out=0), dict(out=A), dict(q=A + 1), dict(k_pages=0),
                                 dict(v_pages=W + 2), dict(v_pages=C), dict(page_table=T + 1)])
def test_attention_refuses_bad_pointers(bad):
    assert status(attend, paged(), **bad) == "InvalidArgument"


def test_paged_refuses_a_batch_past_its_indexes():
    # the host's tile counts and the device's search add tokens and sequences in 32 bits
    for batch in (1 << 30, (1 << 31) - 1):
        bad = paged(batch=batch)
        assert status(gie.paged_attention_workspace_size, bad) == "Unsupported"
        assert status(append, bad) == "Unsupported"
        assert status(attend, bad) == "Unsupported"


def test_attention_workspace_is_checked():
    p = paged(total_tokens=1, batch=1, max_pages=4096, max_new=1, max_len=65536)
    n = gie.paged_attention_workspace_size(p)
    if n:
        assert status(attend, p, ws_bytes=n - 1) == "WorkspaceTooSmall"
        assert status(attend, p, workspace=None, ws_bytes=0) == "WorkspaceTooSmall"
        assert status(attend, p, workspace=W + 4) == "InvalidArgument"


def test_rotary_tables():
    cos, sin = gie.rotary_tables(100, 8, base=500.0)
    f = 500.0 ** (-2.0 * np.arange(4) / 8)
    angle = np.arange(100)[:, None] * f
    assert np.abs(cos - np.cos(angle)).max() <= 2.0 ** -24 and np.abs(sin - np.sin(angle)).max() <= 2.0 ** -24
    cos, sin = gie.rotary_tables(100, 8, base=500.0, factor=4.0, magnitude=2.0)
    assert np.abs(cos - 2 * np.cos(angle / 4)).max() <= 2.0 ** -23
    # by wavelength: the first frequency (6.3 positions) stays, the last (over 500) is divided, those between blended
    cos, _ = gie.rotary_tables(100, 8, base=500.0, factor=4.0, original_positions=100)
    turns = 100 * f / (2 * np.pi)
    keep = np.clip((turns - 1) / 3, 0, 1)
    assert keep[0] == 1 and keep[-1] == 0
    scaled = keep * f + (1 - keep) * f / 4
    assert np.abs(cos - np.cos(np.arange(100)[:, None] * scaled)).max() <= 2.0 ** -23
    for bad in (dict(max_positions=0, rotary_dim=8), dict(max_positions=4, rotary_dim=7), dict(max_positions=4, rotary_dim=8, factor=0.5),
                dict(max_positions=4, rotary_dim=8, base=-1.0)):
        assert status(gie.rotary_tables, **bad) == "InvalidArgument"
