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
