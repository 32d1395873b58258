"""Callers that fill the structures of gie_kv_append and gie_paged_attention as they were before the cache in 8 bits, head
norms and sinks: what lies behind the structures' last fields is not theirs to set, and no call may read it."""
import ctypes

import numpy as np
import pytest

import gie

INTS, STRIDES = ctypes.c_int, ctypes.c_int64


class Problem(ctypes.Structure):
    """gie_paged_kv_problem, and room behind it that belongs to something else."""
    _fields_ = [(n, INTS) for n in ("batch", "total_tokens", "q_heads", "kv_heads", "head_dim", "page_size", "num_pages",
                                    "max_pages", "precision")] + \
               [(n, STRIDES) for n in ("q_stride", "k_stride", "v_stride", "o_stride")] + \
               [(n, INTS) for n in ("rotary_dim", "interleaved", "max_positions")] + \
               [(n, ctypes.c_float) for n in ("scale", "softcap")] + [(n, INTS) for n in ("window", "max_new", "max_len")] + \
               [("behind", ctypes.c_ubyte * 64)]


class Geom(ctypes.Structure):
    """gie_paged_geom, likewise."""
    _fields_ = [(n, INTS) for n in ("batch", "total_tokens", "q_heads", "kv_heads", "head_dim", "page_size", "num_pages",
                                    "max_pages")] + Problem._fields_[9:]


BEHIND = {"ones": b"\xff" * 64, "small": b"\x02\x00\x00\x00" * 16, "nan": np.float32(np.nan).tobytes() * 16, "large": b"\x7f" * 64}
FIELDS = dict(batch=2, total_tokens=3, q_heads=8, kv_heads=2, head_dim=64, page_size=16, num_pages=8, max_pages=4096,
              q_stride=512, k_stride=128, v_stride=128, o_stride=512, scale=0.125, window=4096, max_new=2, max_len=65536)


def filled(kind, what, **more):
    s = kind(**{**FIELDS, **more})
    ctypes.memmove(ctypes.addressof(s) + kind.behind.offset, what, 64)
    return s


def symbol(lib, name, *types, result=INTS):
    """The entry with argument types of its own: gie.py's go with the structures that it fills."""
    return ctypes.CFUNCTYPE(result, *types)((name, lib))


def workspace(problem):
    n = ctypes.c_size_t()
    f = symbol(gie.capi(), "gie_paged_attention_workspace_size", ctypes.c_void_p, ctypes.c_void_p)
    assert f(ctypes.addressof(problem), ctypes.addressof(n)) == 0
    return n.value


def test_the_structures_end_where_they_did():
    assert Problem.behind.offset == 104 and Geom.behind.offset == 96


@pytest.mark.parametrize("what", sorted(BEHIND))
def test_workspace_sizes(what):
    assert workspace(filled(Problem, BEHIND[what], precision=1)) == workspace(filled(Problem, bytes(64), precision=1)) > 0
    f = symbol(gie.hip(), "gie_hip_paged_attention_workspace", ctypes.c_void_p, result=ctypes.c_size_t)
    geoms = [filled(Geom, b) for b in (BEHIND[what], bytes(64))]
    sizes = [f(ctypes.addressof(g)) for g in geoms]
    assert sizes[0] == sizes[1] > 0


@pytest.mark.parametrize("what", sorted(BEHIND))
def test_calls_without_tokens(what):
    """Nothing to do, so no GPU: what is behind the structure is no reason to refuse it."""
    vp = ctypes.c_void_p
    p, g = filled(Problem, BEHIND[what], precision=1, total_tokens=0), filled(Geom, BEHIND[what], total_tokens=0)
    assert symbol(gie.capi(), "gie_kv_append", *[vp] * 13)(ctypes.addressof(p), *[None] * 12) == 0
    assert symbol(gie.capi(), "gie_paged_attention", *[vp] * 9, ctypes.c_size_t, vp)(
        ctypes.addressof(p), *[None] * 8, 0, None) == 0
    assert symbol(gie.hip(), "gie_hip_kv_append", INTS, *[vp] * 13)(gie.FP16, ctypes.addressof(g), *[None] * 12) == 0
    assert symbol(gie.hip(), "gie_hip_paged_attention", INTS, *[vp] * 9, ctypes.c_size_t, vp)(
        gie.FP16, ctypes.addressof(g), *[None] * 8, 0, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("what", sorted(BEHIND))
def test_append_and_attention(what):
    """The same bits as with zeros behind the structures: no sinks, whatever lies where a longer structure has them."""
    from paged_plain import Cache
    vp, results = ctypes.c_void_p, []
    for behind in (bytes(64), BEHIND[what]):
        c = Cache([3, 40], [90, 300], heads=8, kv_heads=2, dim=64, page=16, seed=5)
        d = c.device()
        more = dict(total_tokens=c.tokens, num_pages=c.pages, max_pages=c.max_pages, window=30, max_new=40, max_len=300)
        p, g = filled(Problem, behind, precision=1, **more), filled(Geom, behind, **more)
        size = workspace(p)
        ws, out = gie.DeviceBuffer(max(16, size)), [c.blank_rows(8) for _ in range(3)]
        rows, where = [d[n].addr for n in "qkv"], [d[n].addr for n in ("starts", "lens", "table")]
        pages = [d[n].addr for n in ("k_pages", "v_pages")]
        gie.synchronize()
        assert symbol(gie.capi(), "gie_kv_append", *[vp] * 13)(
            ctypes.addressof(p), *rows, None, None, *where, out[0].addr, *pages, None) == 0
        assert symbol(gie.capi(), "gie_paged_attention", *[vp] * 9, ctypes.c_size_t, vp)(
            ctypes.addressof(p), out[0].addr, *pages, *where, out[1].addr, ws.addr, ws.nbytes, None) == 0
        assert symbol(gie.hip(), "gie_hip_paged_attention", INTS, *[vp] * 9, ctypes.c_size_t, vp)(
            gie.FP16, ctypes.addressof(g), out[0].addr, *pages, *where, out[2].addr, ws.addr, ws.nbytes, None) == 0
        gie.synchronize()
        results.append([c.read_rows(o, 8) for o in out])
    assert all(np.array_equal(a, b) for a, b in zip(*results))
    assert np.array_equal(results[0][1], results[0][2])


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [0, 64, 6])
def test_the_older_entries_do_what_the_newer_ones_do(rotary):
    """gie_kv_append beside gie_kv_append_normed without norms, gie_paged_attention beside gie_kv_attention without sinks."""
    from paged_plain import Cache
    vp, results = ctypes.c_void_p, []
    for older in (True, False):
        c = Cache([3, 40], [90, 300], heads=8, kv_heads=2, dim=64, page=16, seed=6)
        d = c.device()
        tables = [gie.to_device(t) for t in gie.rotary_tables(c.max_pages * 16, rotary)] if rotary else []
        turn = [t.addr for t in tables] or [None, None]
        more = dict(rotary_dim=rotary, max_positions=c.max_pages * 16, window=50, max_new=40, max_len=300)
        p = c.p(**more)
        ws, out = gie.DeviceBuffer(max(16, gie.paged_attention_workspace_size(p))), [c.blank_rows(8) for _ in range(2)]
        rows, where = [d[n].addr for n in "qkv"], [d[n].addr for n in ("starts", "lens", "table")]
        pages = [d[n].addr for n in ("k_pages", "v_pages")]
        gie.synchronize()
        at = ctypes.addressof(p._c)
        if older:
            assert symbol(gie.capi(), "gie_kv_append", *[vp] * 13)(at, *rows, *turn, *where, out[0].addr, *pages, None) == 0
            assert symbol(gie.capi(), "gie_paged_attention", *[vp] * 9, ctypes.c_size_t, vp)(
                at, out[0].addr, *pages, *where, out[1].addr, ws.addr, ws.nbytes, None) == 0
        else:
            assert symbol(gie.capi(), "gie_kv_append_normed", *[vp] * 15)(
                at, *rows, None, None, *turn, *where, out[0].addr, *pages, None) == 0
            assert symbol(gie.capi(), "gie_kv_attention", *[vp] * 9, ctypes.c_size_t, vp)(
                at, out[0].addr, *pages, *where, out[1].addr, ws.addr, ws.nbytes, None) == 0
        gie.synchronize()
        results.append([c.read_rows(o, 8) for o in out] + [d[n].download(np.uint16, c.k_pages.size) for n in ("k_pages", "v_pages")])
    assert all(np.array_equal(a, b) for a, b in zip(*results))


def test_no_structure_is_refused():
    """A null structure, by the older entries and by the newer ones."""
    vp, size, n = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t()
    for name, pointers in (("gie_kv_append", 13), ("gie_kv_append_normed", 15), ("gie_kv8_append", 17), ("gie_kv8_read", 11)):
        assert symbol(gie.capi(), name, *[vp] * pointers)(*[None] * pointers) == 1
    for name in ("gie_paged_attention", "gie_kv_attention"):
        assert symbol(gie.capi(), name, *[vp] * 9, size, vp)(*[None] * 9, 0, None) == 1
        assert symbol(gie.capi(), name + "_workspace_size", vp, vp)(None, ctypes.addressof(n)) == 1
        assert symbol(gie.hip(), name.replace("gie_", "gie_hip_"), INTS, *[vp] * 9, size, vp)(gie.FP16, *[None] * 9, 0, None) == -1
        assert symbol(gie.hip(), name.replace("gie_", "gie_hip_") + "_workspace", vp, result=size)(None) == 0
    assert symbol(gie.hip(), "gie_hip_kv_append", INTS, *[vp] * 13)(gie.FP16, *[None] * 13) == -1
    assert symbol(gie.hip(), "gie_hip_kv_append_normed", INTS, *[vp] * 15)(gie.FP16, *[None] * 15) == -1
