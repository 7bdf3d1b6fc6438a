"""Sizes that the operators of a serving step refuse because their index arithmetic ends there (no GPU: what is refused is refused on the host)."""
import ctypes as C

import pytest

from qwen_inference_engine_b200 import _lib
from test_cpu_serving_step import batch, refused


@pytest.mark.parametrize("n", [2 ** 30 + 1, 2 ** 31 - 5, 2 ** 31 - 1])
def test_layout_of_more_rows_than_a_thread_counts(n):
    """a thread's next row, up to 2^18 behind its last one, is a number of 32 bits"""
    refused(_lib.lib().qie_batch_layout(batch(max_tokens=n), None), "batch_layout", "2^30")
