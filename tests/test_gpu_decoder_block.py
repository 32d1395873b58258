"""The example that runs the 8-bit projections, the cache append and the attention together as a decoder's attention
block, checked by itself against the same block in 64 bits on the host."""
import os
import subprocess

import pytest

import gie

pytestmark = pytest.mark.gpu


def test_decoder_block_example():
    r = subprocess.run([os.path.join(gie.LIB_DIR, "decoder_block")], capture_output=True, text=True, timeout=60)
    print(r.stdout, r.stderr)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.count("PASS") == 2 and "FAIL" not in r.stdout
