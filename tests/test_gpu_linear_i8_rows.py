"""LinearI8 where few long tokens are quantized inside the product's launch: rows that its threads keep in registers
whole, by a value less and a value more, and rows that are read a second time; the largest value in any part of them."""
import numpy as np
import pytest

from test_gpu_linear_i8 import run_linear

import gie

pytestmark = pytest.mark.gpu

# a workgroup keeps 4 pieces of 16 bytes for each of its 512 threads: 16384 values of 16 bits, 8192 of 32
SHAPES = {"fp16": [(1, 16383), (1, 16384), (1, 16385), (1, 28672), (1, 32767), (1, 32768), (2, 16384), (4, 8192)],
          "bf16": [(1, 16391), (1, 24576), (2, 16381)],
          "fp32": [(1, 8191), (1, 8192), (1, 8193), (1, 14336), (1, 32768), (2, 16384), (3, 10001)]}


@pytest.mark.parametrize("precision,m,k", [(p, *s) for p in SHAPES for s in SHAPES[p]])
@pytest.mark.parametrize("largest", ["first", "kept", "rest", "last"])
def test_long_rows_quantized_in_the_product(precision, m, k, largest):
    kept = min(k, 8192 if precision == "fp32" else 16384)
    at = {"first": 0, "kept": kept - 1, "rest": min(kept, k - 1), "last": k - 1}[largest]
    x = np.random.default_rng(k + m).normal(size=(m, k)).astype(np.float32)
    x[:, at] = -40 * np.arange(1, m + 1)
    assert gie.linear_i8_workspace_size(gie.LinearI8(m, k, 48, precision=precision)) == 0, "inside the product"
    got, want, bound = run_linear(m, k, 48, precision=precision, bias=True, x=x)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("precision", ["fp16", "fp32"])
@pytest.mark.parametrize("at", [0, -1])
def test_long_rows_that_are_not_finite(precision, at):
    x = np.random.default_rng(3).normal(size=(1, 30011)).astype(np.float32)
    x[0, at] = np.nan
    got, _, _ = run_linear(1, 30011, 33, precision=precision, x=x)
    assert np.isnan(got).all()
