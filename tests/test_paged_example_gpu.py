"""The paged decoding example end to end: chunked prefill, decoding, verify blocks and rollback over
two layers, against the same attention on unquantised keys and values."""

from __future__ import annotations

import os
import sys

import pytest

from conftest import PKG

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences,prompt,steps,drafts", [(6, 300, 4, 4), (3, 1100, 2, 6), (1, 1, 3, 1)])
def test_paged_decode_example(gpu, sequences, prompt, steps, drafts):
    """A group of 32 normal values spans 4.07 sigma, its step is 4.07 / 15 sigma and its rounding error that
    over sqrt(12): 7.8 % of the values. Keys bring as much again through the scores of unit queries
    (sqrt(64) 0.078 / 8), 11 % together; 15 % leaves room for steps of few rows."""
    sys.path.insert(0, os.path.join(PKG, "examples"))
    import paged_decode

    worst, nbytes, tokens = paged_decode.run(sequences, prompt, steps, drafts)
    assert set(worst) >= {"first chunk", "decode", "verify", "decode after rollback"}
    assert all(0 < off < 0.15 for off in worst.values()), worst
    assert nbytes == tokens * 4 * 80      # 5 bits for each of 2 x 64 dims of four kv heads
