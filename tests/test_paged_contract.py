"""What the paged 8-bit cache promises at its borders, on the CPU: rows that lost tokens, sizes at the end of 32 bits, refusals with a message."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import paged_oracle as P


def test_a_row_that_lost_tokens_gets_no_block():
    """past_lens beyond the held blocks: no block and no slot, what is lacking counts; set back, or with nothing held and nothing new, the row is served."""
    def call(past, new, held):
        table, ring, counters = np.full((2, 6), -1, np.int32), np.arange(8, dtype=np.int32), np.array([2, 6, 0, 0], np.int32)
        table[0, :held] = [0, 1][:held]
        held = np.array([held, 0], np.int32)
        _, slots, _ = P.slots(np.array([past, 0]), np.array([new, 3]), held, table, ring, counters, 16, 96, 8, 8)
        return held.tolist(), slots.tolist(), int(counters[2])

    assert call(33, 2, 2) == ([2, 1], [-1, -1, 32, 33, 34, -1, -1, -1], 1)
    assert call(33, 0, 2) == ([2, 1], [32, 33, 34, -1, -1, -1, -1, -1], 1)
    assert call(1, 1, 0) == ([0, 1], [-1, 32, 33, 34, -1, -1, -1, -1], 1)
    assert call(32, 2, 2) == ([3, 1], [32, 33, 48, 49, 50, -1, -1, -1], 0)
    assert call(33, 0, 0) == ([3, 1], [80, 81, 82, -1, -1, -1, -1, -1], 0)
