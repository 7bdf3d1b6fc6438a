"""What the operators over a cache in 8 bits refuse on the host: no GPU."""
import ctypes as C
import math
import re

import pytest

from qwen_inference_engine_b200 import _lib
from qwen_inference_engine_b200._lib import Kv8View, RopePlan
from test_cpu_serving_step import P, batch, refused


def kv8(**over):
    d = dict(codes=P, scale=P, n_pages=40, page_size=16, n_layers=2, n_kv_heads=2, head_dim=64, code=0)
    d.update(over)
    return C.byref(Kv8View(**d))


POOLS = [dict(codes=0), dict(scale=0), dict(codes=P + 8), dict(n_pages=0), dict(page_size=0), dict(n_kv_heads=0), dict(n_layers=0), dict(head_dim=96), dict(head_dim=256), dict(code=2), dict(code=-1),
         dict(n_pages=1 << 27), dict(n_layers=1 << 25), dict(n_pages=2 ** 31 - 1, page_size=2 ** 31 - 1, n_layers=2 ** 31 - 1, n_kv_heads=2 ** 31 - 1)]


@pytest.mark.parametrize("view,over", [(v, {}) for v in POOLS] +
                         [({}, o) for o in (dict(layer=2), dict(layer=-1), dict(q=0), dict(out=0), dict(k=0), dict(v=0), dict(pos=0), dict(row=0), dict(ks=127), dict(vs=127), dict(qs=255), dict(n=-1),
                                            dict(n=2 ** 30 + 1), dict(q=2 * P, qs=384), dict(heads=-1), dict(rope=None), dict(heads=2 ** 18, qs=2 ** 24, outs=2 ** 24),
                                            *(dict(rope=C.byref(RopePlan(f, r, 0, 1.0))) for f, r in ((0, 64), (P, 0), (P, 63), (P, 66), (P, -2))))])
def test_rope_store8(view, over):
    a = dict(layer=0, q=P, qs=256, out=2 * P, outs=256, k=P, ks=128, v=P, vs=128, pos=P, row=P, n=2, heads=4, rope=C.byref(RopePlan(P, 64, 1, 1.0)))
    a.update(over)
    refused(_lib.lib().qie_rope_store8(kv8(**view), a["layer"], a["q"], a["qs"], a["out"], a["outs"], a["k"], a["ks"], a["v"], a["vs"], a["rope"], a["pos"], a["row"], a["n"], a["heads"], None),
            "rope_store8")


@pytest.mark.parametrize("view,over", [(v, {}) for v in POOLS] + [({}, o) for o in (dict(layer=2), dict(layer=-1), dict(row=0), dict(n=-1), dict(n=2 ** 30 + 1), dict(ks=127), dict(vs=127))] +
                         [(dict(n_kv_heads=2 ** 18 + 1, n_pages=1), dict(ks=2 ** 25, vs=2 ** 25))])
def test_kv8_read(view, over):
    a = dict(layer=0, row=P, n=2, k=P, ks=128, v=P, vs=128)
    a.update(over)
    refused(_lib.lib().qie_kv8_read(kv8(**view), a["layer"], a["row"], a["n"], a["k"], a["ks"], a["v"], a["vs"], None), "kv8_read")


@pytest.mark.parametrize("view,over", [(v, {}) for v in POOLS] + [
    (dict(n_kv_heads=3), {}), (dict(n_kv_heads=1), dict(heads=129, qs=129 * 64, outs=129 * 64)), (dict(page_size=8), {}), (dict(n_pages=41), {}), ({}, dict(layer=2)), ({}, dict(window=-1)),
    ({}, dict(scale=-1.0)), ({}, dict(scale=math.nan)), ({}, dict(scale=math.inf)), ({}, dict(qs=255)), ({}, dict(qs=260)), ({}, dict(outs=260)), ({}, dict(qs=1 << 38)), ({}, dict(q=P + 8)),
    ({}, dict(out=P + 2)), ({}, dict(q=0)), ({}, dict(out=0)), ({}, dict(b=dict(q_start=0))), ({}, dict(b=dict(kv_len=0))), ({}, dict(b=dict(block_table=0))), ({}, dict(b=dict(work=P + 4))),
    ({}, dict(b=dict(max_tokens=1 << 24))), ({}, dict(b=dict(slots=0, max_seqs=2))), ({}, dict(b=dict(n_req=9000)))])
def test_attention8(view, over):
    a = dict(layer=0, q=P, qs=256, out=P, outs=256, heads=4, window=0, scale=0.0, b={})
    a.update(over)
    refused(_lib.lib().qie_attention_batch8(kv8(**view), a["layer"], batch(**a["b"]), a["q"], a["qs"], a["out"], a["outs"], a["heads"], a["window"], a["scale"], None), "attention_batch8")


def test_without_a_pool_or_batch():
    L = _lib.lib()
    refused(L.qie_rope_store8(None, 0, P, 256, P, 256, P, 128, P, 128, None, P, P, 2, 0, None), "rope_store8")
    refused(L.qie_kv8_read(None, 0, P, 2, P, 128, P, 128, None), "kv8_read")
    refused(L.qie_attention_batch8(None, 0, batch(), P, 256, P, 256, 4, 0, 0.0, None), "attention_batch8")
    refused(L.qie_attention_batch8(kv8(), 0, None, P, 256, P, 256, 4, 0, 0.0, None), "attention_batch8")
    assert L.qie_attention_batch8_work(kv8(head_dim=96), 4) == 0 and L.qie_attention_batch8_work(kv8(), 5) == 0 and L.qie_attention_batch8_work(None, 4) == 0


def test_nothing_to_do_needs_no_device():
    L = _lib.lib()
    assert L.qie_rope_store8(kv8(), 0, P, 256, P, 256, P, 128, P, 128, C.byref(RopePlan(P, 64, 0, 1.0)), P, P, 0, 4, None) == 0
    assert L.qie_rope_store8(kv8(), 0, None, 0, None, 0, P, 128, P, 128, None, None, P, 0, 0, None) == 0
    assert L.qie_kv8_read(kv8(), 0, P, 0, P, 128, P, 128, None) == 0 and L.qie_kv8_read(kv8(), 0, P, 5, None, 0, None, 0, None) == 0
    for over in (dict(n_req=0), dict(max_tokens=0)):
        assert L.qie_attention_batch8(kv8(), 0, batch(**over), P, 256, P, 256, 4, 0, 0.0, None) == 0


def test_fields_in_the_headers_order():
    src = re.sub(r"/\*.*?\*/", "", open(_lib.HEADER_PATH).read(), flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\} qie_kv8_view;", src).group(1)
    fields = [re.search(r"(\w+)\s*$", f).group(1) for line in body.split(";") if line.strip() for f in line.split(",")]
    assert fields == [f for f, _ in Kv8View._fields_]
