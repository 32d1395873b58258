"""LinearI8 and quantize_rows on the GPU against plain numpy: the 8-bit values and scales bit for bit, the product
against its definition in 64 bits.

Bound of an output value: float(acc) rounds once, the two scales and the bias add three FP32 roundings, so before the
last rounding the value is within 4 * 2^-24 * (|acc * s * w| + |bias|) of the exact one; the store adds half a step of
its type (unit roundoff 2^-24, 2^-11, 2^-8; in FP16 at least half its smallest step, 2^-25)."""
import numpy as np
import pytest

import gie
import oracle as O

pytestmark = pytest.mark.gpu

UNIT = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
GUARD = 64  # poisoned bytes behind every output


def quantize_plain(x):
    """The definition of q and scale, in FP32 operations."""
    x = x.astype(np.float32)
    with np.errstate(all="ignore"):
        a = np.abs(x).max(axis=1)
        bad = ~np.isfinite(x).all(axis=1)
        a = np.where(bad, np.float32(1), np.maximum(a, np.float32(2.0 ** -100))).astype(np.float32)
        q = np.rint(np.where(bad[:, None], np.float32(0), x) * (np.float32(127) / a)[:, None])
    scale = np.where(bad, np.float32(np.nan), a / np.float32(127)).astype(np.float32)
    return q.astype(np.int8), scale


def strided(a, ld, offset_bytes=0):
    """Device copy of the rows of `a`, ld elements apart, the gaps and what surrounds them poisoned."""
    flat = np.full(a.shape[0] * ld * a.itemsize + offset_bytes + GUARD, 0xA5, np.uint8)
    view = flat[offset_bytes:offset_bytes + a.shape[0] * ld * a.itemsize].reshape(a.shape[0], ld * a.itemsize)
    view[:, :a.shape[1] * a.itemsize] = np.ascontiguousarray(a).view(np.uint8).reshape(a.shape[0], -1)
    return gie.to_device(flat)


def run_linear(m, k, n, precision="fp16", bias=False, relu=False, quantized=False, ld_x=0, ld_w=0, ld_y=0, x_off=0,
               w_off=0, seed=0, x=None, stream=None, dist="normal"):
    rng = np.random.default_rng(seed * 7919 + m * 31 + k * 17 + n)
    if quantized:
        xq = rng.integers(-128, 128, (m, k)).astype(np.int8)
        x_scale = rng.uniform(0.5, 2, m).astype(np.float32) / 100
    else:
        if x is None:
            x = rng.normal(size=(m, k)).astype(np.float32) * (1 + 9 * (rng.random(k) < 0.05))
        x = O.quantize(precision, x.astype(np.float32))
        xq, x_scale = quantize_plain(x)
    w = rng.integers(-128, 128, (n, k)).astype(np.int8)
    w_scale = rng.uniform(0.5, 2, n).astype(np.float32) / (64 * k ** 0.5)
    b = O.quantize(precision, rng.uniform(-1, 1, n).astype(np.float32)) if bias else None
    p = gie.LinearI8(m, k, n, precision=precision, has_bias=bias, relu=relu, quantized=quantized, ld_x=ld_x, ld_w=ld_w,
                     ld_y=ld_y)
    esz = 4 if precision == "fp32" else 2
    storage = np.uint32 if esz == 4 else np.uint16
    xs = xq if quantized else gie.host_to_storage(x, precision).view(storage)
    dx, dw = strided(xs.reshape(m, k), ld_x or k, x_off), strided(w, ld_w or k, w_off)
    dxs, dws = gie.to_device(x_scale), gie.to_device(w_scale)
    db = gie.to_device(gie.host_to_storage(b, precision)) if bias else None
    ldy = ld_y or n
    dy = gie.DeviceBuffer(m * ldy * esz + GUARD)
    dy.fill(0xA5)
    size = gie.linear_i8_workspace_size(p)
    ws = gie.DeviceBuffer(size + GUARD)
    ws.fill(0xA5)
    gie.synchronize()
    print(f"linear {m}x{k}x{n} {precision} q={quantized} ld={ld_x},{ld_w},{ld_y} off={x_off},{w_off}", flush=True)
    gie.linear_i8(p, dx.addr + x_off, dw.addr + w_off, dws.addr, dy.addr, x_scale=dxs.addr if quantized else None,
                  bias=db.addr if bias else None, workspace=ws.addr, ws_bytes=size, stream=stream)
    gie.synchronize()
    raw = dy.download(np.uint8, dy.nbytes)
    assert (raw[m * ldy * esz:] == 0xA5).all(), "written past y"
    assert (ws.download(np.uint8, ws.nbytes)[size:] == 0xA5).all(), "written past the workspace"
    rows = raw[:m * ldy * esz].reshape(m, ldy * esz)
    assert (rows[:, n * esz:] == 0xA5).all(), "written between the rows of y"
    got = gie.storage_to_float(np.ascontiguousarray(rows[:, :n * esz]).view(storage).reshape(-1), precision)
    got = got.reshape(m, n).astype(np.float64)
    main = (xq.astype(np.float64) @ w.astype(np.float64).T) * (x_scale.astype(np.float64)[:, None] * w_scale)
    want = main + (b.astype(np.float64) if bias else 0)
    bound = 4 * 2.0 ** -24 * (np.abs(main) + (np.abs(b) if bias else 0))
    if relu:
        want = np.where(want < 0, 0, want)
    bound = bound + UNIT[precision] * (np.abs(want) + bound) + (2.0 ** -25 if precision == "fp16" else 0)
    return got, want, bound


def check(*args, **kw):
    got, want, bound = run_linear(*args, **kw)
    assert np.isfinite(want).all()
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), (float(off.max()), np.argwhere(~(off <= 0))[:4].tolist())


@pytest.mark.parametrize("precision", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 64, 16), (3, 100, 33), (1, 4096, 256), (16, 512, 128),
                                   (17, 130, 70), (64, 256, 192), (65, 1000, 515), (130, 96, 258), (300, 640, 320)])
def test_shapes(precision, shape):
    check(*shape, precision=precision, bias=True, relu=False)


@pytest.mark.parametrize("shape", [(1, 64, 16), (5, 33, 7), (40, 2048, 96), (128, 128, 256), (257, 320, 513),
                                   (512, 1024, 512)])
@pytest.mark.parametrize("precision", ["fp16", "fp32"])
def test_given_scales(shape, precision):
    check(*shape, precision=precision, quantized=True, relu=True, bias=True)


@pytest.mark.parametrize("m", [1, 2, 4, 7, 8, 15, 16, 31, 32, 33, 48, 63, 64, 96, 127, 128, 129, 200, 256])
def test_every_token_count(m):
    check(m, 384, 272, precision="bf16")


@pytest.mark.parametrize("k", [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 1023, 1025])
@pytest.mark.parametrize("m", [2, 150])
def test_every_ragged_depth(m, k):
    check(m, k, 130, precision="fp32", quantized=True)
    check(m, k, 130, precision="fp16")


@pytest.mark.parametrize("layout", [dict(ld_x=272, ld_w=288, ld_y=200), dict(ld_x=261, ld_w=259, ld_y=131),
                                    dict(x_off=2, w_off=1), dict(x_off=6, w_off=4, ld_w=260), dict(w_off=8, ld_x=264)])
@pytest.mark.parametrize("m", [1, 20, 140])
def test_strides_and_alignment(layout, m):
    check(m, 257, 130, precision="fp16", bias=True, **layout)
    check(m, 256, 128, precision="bf16", quantized=True, **layout)


@pytest.mark.parametrize("m", [1, 100, 300])
def test_long_sums_are_exact(m):
    """Both operands at -128 over the deepest product: the 32-bit sum must not saturate or wrap."""
    k, n = 131071, 32
    p = gie.LinearI8(m, k, n, precision="fp32", quantized=True)
    dx, dw = gie.DeviceBuffer(m * k), gie.DeviceBuffer(n * k)
    dx.fill(0x80)
    dw.fill(0x80)
    one_m, one_n = gie.to_device(np.ones(m, np.float32)), gie.to_device(np.ones(n, np.float32))
    dy, ws = gie.DeviceBuffer(4 * m * n), gie.DeviceBuffer(max(16, gie.linear_i8_workspace_size(p)))
    gie.linear_i8(p, dx.addr, dw.addr, one_n.addr, dy.addr, x_scale=one_m.addr, workspace=ws.addr, ws_bytes=ws.nbytes)
    gie.synchronize()
    assert (dy.download(np.float32, m * n) == np.float32(16384.0 * k)).all()


def test_rows_of_zeros_tiny_and_not_finite_values():
    m, k, n = 9, 200, 64
    rng = np.random.default_rng(3)
    x = rng.normal(size=(m, k)).astype(np.float32)
    x[1] = 0
    x[2, 5] = np.inf
    x[3, 199] = np.nan
    x[4, 0] = -np.inf
    x[5] *= 1e-38
    x[6] *= 1e37
    x[7] = -0.0
    with np.errstate(over="ignore"):
        got, want, bound = run_linear(m, k, n, precision="bf16", x=x, relu=True)
    for r in (2, 3, 4):
        assert np.isnan(got[r]).all(), r
    rest = [r for r in range(m) if r not in (2, 3, 4)]
    assert (got[[1, 7]] == 0).all()
    assert (np.abs(got[rest] - want[rest]) <= bound[rest] + 2.0 ** -133).all()  # bf16's smallest step


@pytest.mark.parametrize("precision", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 64), (5, 4096), (7, 1001), (300, 520), (2, 20011)])
def test_quantize_rows_bit_exact(precision, shape):
    m, k = shape
    rng = np.random.default_rng(m * 100 + k)
    x = O.quantize(precision, (rng.normal(size=shape) * 10 ** rng.uniform(-3, 3, (m, 1))).astype(np.float32))
    if m > 2:
        x[1] = 0
        x[2, k // 2] = np.nan
    for ld, off in ((0, 0), (k + 3, 0), (k + 8, 4)):
        p = gie.LinearI8(m, k, 1, precision=precision, ld_x=ld)
        storage = gie.host_to_storage(x, precision)
        dx = strided(storage.reshape(m, k), ld or k, off)
        dq, ds = gie.DeviceBuffer(m * k + GUARD), gie.DeviceBuffer(4 * m + GUARD)
        dq.fill(0xA5)
        ds.fill(0xA5)
        gie.synchronize()
        print(f"quantize {shape} {precision} ld={ld} off={off}", flush=True)
        gie.quantize_rows(p, dx.addr + off, dq.addr, ds.addr)
        gie.synchronize()
        q, scale = quantize_plain(x)
        assert np.array_equal(dq.download(np.int8, m * k).reshape(m, k), q)
        assert np.array_equal(ds.download(np.float32, m), scale, equal_nan=True)
        assert (dq.download(np.uint8, GUARD, offset=m * k) == 0xA5).all()
        assert (ds.download(np.uint8, GUARD, offset=4 * m) == 0xA5).all()


def test_same_bits_every_time_and_on_a_stream():
    s = gie.Stream()
    first = run_linear(33, 2048, 96, precision="fp32", bias=True)[0]
    assert np.array_equal(first, run_linear(33, 2048, 96, precision="fp32", bias=True)[0])
    assert np.array_equal(first, run_linear(33, 2048, 96, precision="fp32", bias=True, stream=s)[0])


def test_no_tokens_is_no_work():
    p = gie.LinearI8(0, 64, 64)
    assert gie.linear_i8_workspace_size(p) == 0
    gie.linear_i8(p, 0, 0, 0, 0)
    gie.quantize_rows(p, 0, 0, 0)
    gie.synchronize()


@pytest.mark.parametrize("shape", [(4090, 200, 4085), (4096, 128, 4096), (2040, 200, 2030), (1000, 333, 1000)])
@pytest.mark.parametrize("layout", [dict(), dict(ld_x=352, ld_w=336, ld_y=4104), dict(ld_x=353, ld_w=341, ld_y=4099)])
def test_large_tiles(shape, layout):
    """Enough tokens and channels for tiles of 256, 128 and 64, whole and with ragged edges, rows that 16-byte pieces fit
    and rows that they do not."""
    check(*shape, precision="bf16", bias=True, **layout)
    check(*shape, precision="fp32", quantized=True, relu=True, **layout)
