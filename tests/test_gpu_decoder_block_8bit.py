"""The decoder's attention block with head norms, the cache in 8 bits (appended, attended with a window and sinks, read back)
and the 8-bit projections, checked by the example itself against 64 bits."""
import os
import subprocess

import pytest

import gie

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_decoder_block_with_a_cache_in_8_bits(cache):
    r = subprocess.run([os.path.join(gie.LIB_DIR, "decoder_block"), cache], capture_output=True, text=True, timeout=60)
    print(r.stdout, r.stderr)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.count("PASS") == 4 and "FAIL" not in r.stdout
