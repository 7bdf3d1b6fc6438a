"""What the operators of a serving step refuse on the host, and the rotary frequencies (host code): no GPU."""
import ctypes as C
import math

import numpy as np
import pytest

from qwen_inference_engine_b200 import _lib
from qwen_inference_engine_b200._lib import BatchView, KvView, LogitRulesView, QieError, RopePlan

P = 1 << 20  # stands for a device pointer; nothing reads it on the host
ARRAYS = ("cached", "n_new", "slots", "block_table", "free_ring", "ring_in", "ring_out", "q_start", "kv_len", "pos", "slot", "row", "status", "work")


def batch(**over):
    d = dict(n_req=4, max_tokens=8, max_seqs=4, max_pages=10, n_pages=40, page_size=16, work_bytes=1 << 30, **{a: P * (i + 1) for i, a in enumerate(ARRAYS)})
    d.update(over)
    return C.byref(BatchView(**d))


def kv(**over):
    d = dict(pool=P, n_pages=40, page_size=16, n_layers=2, n_kv_heads=2, head_dim=64)
    d.update(over)
    return C.byref(KvView(**d))


def refused(rc, *words):
    msg = _lib.lib().qie_last_error().decode()
    assert rc == -1, (rc, msg)
    assert all(w in msg for w in words), msg


@pytest.mark.parametrize("over", [dict(n_req=-1), dict(n_req=8193), dict(max_tokens=-1), dict(max_pages=0), dict(page_size=0), dict(n_pages=0), dict(max_seqs=0),
                                  dict(max_seqs=-1), dict(max_pages=1 << 27), dict(n_pages=1 << 27), dict(slots=0, max_seqs=3), dict(kv_len=2 * P, cached=2 * P), dict(kv_len=2 * P),
                                  *({a: 0} for a in ARRAYS if a not in ("slots", "work"))])
def test_layout(over):
    refused(_lib.lib().qie_batch_layout(batch(**over), None), "batch_layout")


def test_layout_without_a_batch():
    refused(_lib.lib().qie_batch_layout(None, None), "batch_layout")


def rope_rows(x=P, xs=256, out=P, outs=256, plan=None, pos=P, n=3, heads=2, hd=128):
    plan = C.byref(RopePlan(P, 128, 0, 1.0)) if plan is None else plan
    return _lib.lib().qie_rope_rows(x, xs, out, outs, plan, pos, n, heads, hd, None)


@pytest.mark.parametrize("over", [dict(x=0), dict(out=0), dict(pos=0), dict(n=-1), dict(n=2 ** 30 + 1), dict(heads=-1), dict(xs=255), dict(outs=255), dict(hd=1026, xs=4096, outs=4096), dict(hd=126),
                                  dict(outs=300), *(dict(plan=C.byref(RopePlan(f, r, 0, 1.0))) for f, r in ((0, 64), (P, 0), (P, 63), (P, 130), (P, -2)))])
def test_rope_rows(over):
    refused(rope_rows(**over), "rope_rows")


def test_nothing_to_do_needs_no_device():
    L = _lib.lib()
    assert rope_rows(n=0) == 0 and rope_rows(heads=0, xs=0, outs=0) == 0
    assert L.qie_logits_process(P, 9, P, 9, 0, 0, 9, C.byref(LogitRulesView()), None) == 0
    for over in (dict(n_req=0), dict(max_tokens=0)):
        assert L.qie_attention_batch(kv(), 0, batch(**over), P, 256, P, 256, 4, 0, 0.0, None) == 0


@pytest.mark.parametrize("view,over", [(dict(pool=0), {}), (dict(n_pages=0), {}), (dict(page_size=0), {}), (dict(n_kv_heads=0), {}), (dict(n_pages=1 << 27), {}),
                                       (dict(head_dim=62), {}), ({}, dict(layer=2)), ({}, dict(layer=-1)), ({}, dict(q=0)), ({}, dict(k=0)), ({}, dict(v=0)), ({}, dict(pos=0)),
                                       ({}, dict(row=0)), ({}, dict(ks=127)), ({}, dict(vs=127)), ({}, dict(qs=255)), ({}, dict(n=-1)), ({}, dict(n=2 ** 30 + 1)), ({}, dict(q=2 * P, qs=384))])
def test_rope_store(view, over):
    a = dict(layer=0, q=P, qs=256, k=P, ks=128, v=P, vs=128, pos=P, row=P, n=2, heads=4)
    a.update(over)
    refused(_lib.lib().qie_rope_store(kv(**view), a["layer"], a["q"], a["qs"], 2 * P, 256, a["k"], a["ks"], a["v"], a["vs"], C.byref(RopePlan(P, 64, 1, 1.0)), a["pos"],
                                      a["row"], a["n"], a["heads"], None), "rope_store")


@pytest.mark.parametrize("view,over", [(dict(pool=0), {}), (dict(head_dim=96), {}), (dict(n_kv_heads=3), {}), (dict(n_kv_heads=1), dict(heads=129, qs=129 * 64, outs=129 * 64)),
                                       (dict(page_size=8), {}), (dict(n_pages=41), {}), (dict(n_layers=1 << 25), {}), ({}, dict(layer=2)), ({}, dict(window=-1)), ({}, dict(scale=-1.0)),
                                       ({}, dict(scale=math.nan)), ({}, dict(scale=math.inf)), ({}, dict(qs=255)), ({}, dict(qs=260)), ({}, dict(outs=260)), ({}, dict(q=P + 8)),
                                       ({}, dict(out=P + 2)), ({}, dict(q=0)), ({}, dict(out=0)), ({}, dict(b=dict(q_start=0))), ({}, dict(b=dict(kv_len=0))),
                                       ({}, dict(b=dict(block_table=0))), ({}, dict(b=dict(work=P + 4))), ({}, dict(b=dict(max_tokens=1 << 24))), ({}, dict(b=dict(slots=0, max_seqs=2))), ({}, dict(b=dict(n_req=9000)))])
def test_attention(view, over):
    a = dict(layer=0, q=P, qs=256, out=P, outs=256, heads=4, window=0, scale=0.0, b={})
    a.update(over)
    refused(_lib.lib().qie_attention_batch(kv(**view), a["layer"], batch(**a["b"]), a["q"], a["qs"], a["out"], a["outs"], a["heads"], a["window"], a["scale"], None),
            "attention_batch")


def test_attention_work_of_refused_shapes():
    assert _lib.lib().qie_attention_batch_work(kv(head_dim=96), 4) == 0 and _lib.lib().qie_attention_batch_work(kv(), 5) == 0


@pytest.mark.parametrize("rules,over", [({}, dict(logits=0)), ({}, dict(out=0)), ({}, dict(dtype=2)), ({}, dict(rows=-1)), ({}, dict(rows=65536)), ({}, dict(vocab=0)),
                                        ({}, dict(stride=99)), ({}, dict(out_stride=99)), ({}, dict(logits=P + 1)), ({}, dict(dtype=1, logits=P + 2)), ({}, dict(out=P, stride=128)),
                                        (dict(repetition=P), {}), (dict(presence=P), {}), (dict(frequency=P), {}), (dict(gen_start=P), {}),
                                        (dict(tok_start=P, n_tokens=5), {}), (dict(tok_start=P, tokens=P, n_tokens=-1), {}), (dict(bias_start=P, bias=P, n_bias=3), {}),
                                        (dict(bias_start=P, bias_ids=P, n_bias=3), {}), (dict(bias_ids=P, bias=P, n_bias=3), {}), (dict(mask=P, n_masks=2, mask_words=3), {}),
                                        (dict(mask=P, n_masks=-1, mask_words=4), {})])
def test_logits(rules, over):
    a = dict(logits=P, stride=100, out=2 * P, out_stride=100, dtype=0, rows=2, vocab=100)
    a.update(over)
    refused(_lib.lib().qie_logits_process(a["logits"], a["stride"], a["out"], a["out_stride"], a["dtype"], a["rows"], a["vocab"], C.byref(LogitRulesView(**rules)), None),
            "logits_process")


# ---------------------------------------------------------------- frequencies
def frequencies(*a, **k):
    from qwen_inference_engine_b200 import layers as L
    return L.Rope.frequencies(*a, **k)


@pytest.mark.parametrize("rotated,base", [(2, 10000.0), (64, 1e6), (128, 10000.0), (50, 5e5)])
def test_frequencies(rotated, base):
    w = base ** (-2 * np.arange(rotated // 2) / rotated)
    near = dict(rtol=1e-14, atol=0)
    got, f = frequencies(rotated, base)
    assert f == 1.0 and np.allclose(got, w, **near)
    assert np.allclose(frequencies(rotated, base, "linear", 8.0)[0], w / 8, **near)
    if rotated > 2:
        got, f = frequencies(rotated, base, "ntk", 4.0)
        assert f == 1.0 and np.allclose(got, (base * 4 ** (rotated / (rotated - 2))) ** (-2 * np.arange(rotated // 2) / rotated), rtol=1e-13, atol=0)
        assert np.isclose(got[-1], w[-1] / 4, rtol=1e-12) and got[0] == 1  # the slowest pair turns a quarter as fast, the fastest one as it did
    turns = 8192 * w / (2 * math.pi)
    got, f = frequencies(rotated, base, "parts", 8.0, 8192)
    assert f == 1.0
    for t, a, b in zip(turns, got, w):
        want = b if t >= 4 else b / 8 if t <= 1 else b * (t - 1) / 3 + b / 8 * (1 - (t - 1) / 3)
        assert math.isclose(a, want, rel_tol=1e-13)
    got, f = frequencies(rotated, base, "yarn", 4.0, 32768)
    assert math.isclose(f, 0.1 * math.log(4) + 1, rel_tol=1e-7)
    lo, hi = (rotated * math.log(32768 / (r * 2 * math.pi)) / (2 * math.log(base)) for r in (32, 1))
    lo, hi = max(0, math.floor(lo)), min(rotated - 1, math.ceil(hi))
    for i, (a, b) in enumerate(zip(got, w)):
        ramp = min(1, max(0, (i - lo) / max(hi - lo, 1e-3)))
        assert math.isclose(a, b * (1 - ramp) + b / 4 * ramp, rel_tol=1e-13)


def test_scale_one_changes_nothing():
    for kind in ("linear", "ntk", "yarn", "parts"):
        got, f = frequencies(64, 1e6, kind, 1.0, 4096)
        assert f == 1.0 and np.allclose(got, frequencies(64, 1e6)[0], rtol=1e-15, atol=0), kind


@pytest.mark.parametrize("a", [(0,), (3,), (64, 1.0), (64, math.nan), (64, 1e4, "linear", 0.5), (64, 1e4, "linear", math.nan), (2, 1e4, "ntk", 2.0), (64, 1e4, "yarn", 2.0, 0),
                               (64, 1e4, "yarn", 2.0, 4096, 1.0, 32.0), (64, 1e4, "parts", 2.0, 4096, 4.0, 1.0), (64, 1e4, "parts", 2.0, 4096, -1.0, 4.0)])
def test_frequencies_refused(a):
    with pytest.raises(QieError) as e:
        frequencies(*a)
    assert e.value.code == -1 and "rope_frequencies" in str(e.value)


def test_fields_in_the_headers_order():
    """the Python structures name the fields of the header's, in its order"""
    import re
    src = re.sub(r"/\*.*?\*/", "", open(_lib.HEADER_PATH).read(), flags=re.S)
    for name, view in (("qie_batch", BatchView), ("qie_rope_plan", RopePlan), ("qie_logit_rules", LogitRulesView)):
        body = re.search(r"typedef struct \{([^}]*)\} %s;" % name, src).group(1)
        fields = [re.search(r"(\w+)\s*$", f).group(1) for line in body.split(";") if line.strip() for f in line.split(",")]
        assert fields == [f for f, _ in view._fields_], name
