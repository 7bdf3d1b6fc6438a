"""The Python forms of a serving step's operators with tensors that only say what they are: what each form hands on, and what it turns away (no GPU)."""
import types

import pytest

torch = pytest.importorskip("torch")

bf16, i32, f32, f64 = torch.bfloat16, torch.int32, torch.float32, torch.float64


class Told:
    """a contiguous tensor of a device, as far as the forms ask"""
    is_cuda = True

    def __init__(self, *shape, dtype=bf16, device=0):
        self.shape, self.dtype, self.index, self.device = torch.Size(shape), dtype, device, f"cuda:{device}"

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 1 << 20

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def stride(self):
        return tuple(self.shape[i + 1:].numel() for i in range(len(self.shape)))


@pytest.fixture
def L(monkeypatch):
    from qwen_inference_engine_b200 import layers
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append(name) or 0

    monkeypatch.setattr(torch, "_C", types.SimpleNamespace(_cuda_getDevice=lambda: 0, _cuda_getCurrentRawStream=lambda dev: 40 + dev))
    monkeypatch.setattr(layers._lib, "lib", Lib)
    monkeypatch.setattr(layers, "calls", calls, raising=False)
    return layers


def made_there(what, first, *a, **k):
    """an object over tensors of another device, made while that is the current one"""
    torch._C._cuda_getDevice = first.get_device
    made = what(first, *a, **k)
    torch._C._cuda_getDevice = lambda: 0
    return made


def rope_rows(L, **dev):
    d = dict(x=0, out=0, pos=0, freq=0)
    d.update(dev)
    rope = made_there(L.Rope, Told(32, dtype=f64, device=d["freq"]))
    L.launch_rope_rows(Told(4, 128, device=d["x"]), Told(4, 128, device=d["out"]), Told(4, dtype=i32, device=d["pos"]), rope, 2, 64)


def rope_store(L, **dev):
    d = dict(q=0, k=0, v=0, q_out=0, pool=0, pos=0, row=0, freq=0)
    d.update(dev)
    rope = made_there(L.Rope, Told(32, dtype=f64, device=d["freq"]))
    pool = L.KvPool.over(Told(3, 1, 2, 1, 16, 64, device=d["pool"]))
    L.launch_rope_store(Told(4, 128, device=d["q"]), Told(4, 64, device=d["k"]), Told(4, 64, device=d["v"]), Told(4, 128, device=d["q_out"]), pool, 0,
                        Told(4, dtype=i32, device=d["pos"]), Told(4, dtype=i32, device=d["row"]), rope, 2)


def logits(L, **dev):
    d = dict(logits=0, out=0, rules=0)
    d.update(dev)
    rules = made_there(L.LogitRules, Told(4, dtype=i32, device=d["rules"]), Told(9, dtype=i32, device=d["rules"]), repetition=Told(3, dtype=f32, device=d["rules"]))
    L.launch_logits(Told(3, 100, device=d["logits"]), Told(3, 100, device=d["out"]), rules)


FORMS = {rope_rows: ("x", "out", "pos", "freq"), rope_store: ("q", "k", "v", "q_out", "pool", "pos", "row", "freq"), logits: ("logits", "out", "rules")}


@pytest.mark.parametrize("form,name", [(form, name) for form, names in FORMS.items() for name in names])
def test_every_tensor_is_of_the_current_device(L, form, name):
    form(L)
    assert len(L.calls) == 1
    with pytest.raises(AssertionError):
        form(L, **{name: 1})
    assert len(L.calls) == 1, "a call reached the library"


def test_rules_of_nothing_have_no_device(L):
    L.launch_logits(Told(3, 100), Told(3, 100), L.LogitRules())
    assert L.calls == ["qie_logits_process"]


def batch_of(L, pages=3):
    return L.Batch(Told(1, pages, dtype=i32), 16, pages, 1, 4, **{n: Told(5, dtype=i32) for n in ("ring_out", "q_start", "kv_len", "pos", "slot", "row", "status")})


@pytest.fixture
def areas(L, monkeypatch):
    """work areas in bytes: heads of 64 take 1000, of 128 2000; a call of attention with less than its heads take is refused as by the library"""
    import weakref
    made = []

    def empty(n, dtype, device):
        t = Told(n, dtype=dtype)
        made.append(weakref.ref(t))
        return t

    need = {64: 1000, 128: 2000}

    class Lib:
        def qie_attention_batch_work(self, view, n_q):
            return need.get(view._obj.head_dim, 0)

        def qie_attention_batch(self, view, layer, batch, *rest):
            L.calls.append((view._obj.head_dim, batch._obj.work_bytes))
            return 0

    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(L._lib, "lib", Lib)
    return made


def attend(L, batch, hd):
    L.launch_attn_batch(Told(4, 2 * hd), Told(4, 2 * hd), L.KvPool.over(Told(3, 1, 2, 1, 16, hd)), 0, batch, 2)


def test_work_area_grows_with_the_heads(L, areas):
    """one batch over pools of both head sizes; an area that a captured graph may have is kept"""
    batch = batch_of(L)
    for hd in (64, 64, 128, 64, 128):
        attend(L, batch, hd)
    assert L.calls == [(64, 1000), (64, 1000), (128, 2000), (64, 2000), (128, 2000)]
    assert len(areas) == 2 and all(a() is not None for a in areas)


def test_reserved_work_area_is_taken(L, areas):
    batch = batch_of(L)
    for hd in (128, 64):
        batch.reserve(L.KvPool.over(Told(3, 1, 2, 1, 16, hd)), 2)
    attend(L, batch, 128)
    batch.view.work_bytes -= 1  # the caller's word stands, and the library refuses it
    attend(L, batch, 128)
    assert L.calls == [(128, 2000), (128, 1999)] and len(areas) == 1


def test_heads_without_a_work_area(L, areas):
    """heads that the operator does not take get none, and the library says so; the batch serves others all the same"""
    batch = batch_of(L)
    attend(L, batch, 96)
    attend(L, batch, 64)
    assert L.calls == [(96, 0), (64, 1000)]
