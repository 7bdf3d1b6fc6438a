"""Sizes that the operators of a serving step refuse because their index arithmetic ends there (no GPU: what is refused is refused on the host)."""
import ctypes as C

import pytest

from qwen_inference_engine_b200 import _lib
from qwen_inference_engine_b200._lib import LogitRulesView, RopePlan
from test_cpu_serving_step import P, batch, kv, refused, rope_rows


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


@pytest.mark.parametrize("heads,hd", [(2 ** 14 + 1, 1024), (2 ** 21, 1024), (2 ** 22, 1024), (2 ** 31 - 1, 1024), (2 ** 31 - 1, 2)])
def test_rotary_rows_of_more_places_than_a_grid_has(heads, hd):
    """a row's places are numbers of 32 bits and its share of the grid one of 16: wider rows were counted modulo 2^32, and a part of them turned"""
    refused(rope_rows(heads=heads, hd=hd, plan=C.byref(RopePlan(P, 2, 0, 1.0)), xs=heads * hd, outs=heads * hd), "rope_rows", "2^24")
    view, plan, wide = kv(head_dim=hd, n_kv_heads=2), C.byref(RopePlan(P, 2, 0, 1.0)), heads * hd
    refused(_lib.lib().qie_rope_store(view, 0, P, wide, 2 * P, wide, P, 2 * hd, P, 2 * hd, plan, P, P, 2, heads, None), "rope_store", "2^24")
    view = kv(head_dim=hd, n_kv_heads=heads // 2 + 1)
    refused(_lib.lib().qie_rope_store(view, 0, P, hd, 2 * P, hd, P, 2 * wide, P, 2 * wide, plan, P, P, 2, 1, None), "rope_store", "2^24")
