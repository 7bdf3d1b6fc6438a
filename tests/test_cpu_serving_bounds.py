"""Sizes that the operators of a serving step refuse because their index arithmetic ends there (no GPU: what is refused is refused on the host)."""
import ctypes as C

import pytest

from qwen_inference_engine_b200 import _lib
from qwen_inference_engine_b200._lib import LogitRulesView
from test_cpu_serving_step import P, batch, refused


@pytest.mark.parametrize("n", [2 ** 30 + 1, 2 ** 31 - 5, 2 ** 31 - 1])
def test_layout_of_more_rows_than_a_thread_counts(n):
    """a thread's next row, up to 2^18 behind its last one, is a number of 32 bits"""
    refused(_lib.lib().qie_batch_layout(batch(max_tokens=n), None), "batch_layout", "2^30")


def rules(**over):
    d = dict(tok_start=P, tokens=P, n_tokens=0)
    d.update(over)
    return C.byref(LogitRulesView(**d))


@pytest.mark.parametrize("n", [2 ** 29, 2 ** 30, 2 ** 31 - 1])
def test_logits_of_a_longer_list_than_a_token_is_counted(n):
    """how often a token is there is a number of 29 bits; more of one token would carry into what stands above it, and lead outside the list of biases"""
    refused(_lib.lib().qie_logits_process(P, 100, 2 * P, 100, 0, 2, 100, rules(n_tokens=n), None), "logits_process", "2^29")


def test_logits_of_the_longest_lists():
    assert _lib.lib().qie_logits_process(P, 100, P, 100, 0, 0, 100, rules(n_tokens=2 ** 29 - 1, bias_start=P, bias_ids=P, bias=P, n_bias=2 ** 30), None) == 0
