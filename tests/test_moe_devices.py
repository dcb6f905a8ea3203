"""What the Python side of the mixture-of-experts operators asks of its tensors
(places, types, shapes, strides), on the CPU: tensors that only claim a GPU, and
a library that only notes its calls."""
import pytest

import ggml_hip as G
from ggml_hip import moe as M

torch = pytest.importorskip("torch")


class On:
    """A CPU tensor that says it lives on a GPU (-1: the CPU)."""

    def __init__(self, t, device=0):
        self._t, self._on = t, device

    def __getattr__(self, name):
        return getattr(self._t, name)

    def __getitem__(self, at):
        return On(self._t[at], self._on)

    def view(self, *shape):
        return On(self._t.view(*shape), self._on)

    def new_empty(self, *a, **kw):
        return On(self._t.new_empty(*a, **kw), self._on)

    is_cuda = property(lambda self: self._on >= 0)

    def get_device(self):
        return self._on


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            if name.endswith("workspace_size"):
                return 4096
            self.calls.append(name)
            return 0
        return entry


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(M, "_lib", lambda: lib)
    monkeypatch.setattr(M, "_raw_stream", lambda *_: 0)
    return lib


def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def _rows(*shape):
    """int8 rows on 16-byte boundaries."""
    flat = torch.zeros(4096 + 16, dtype=torch.int8)
    at = -flat.data_ptr() % 16
    n = 1
    for s in shape:
        n *= s
    return flat[at:at + n].view(shape)


I8, I32 = torch.int8, torch.int32
ARGS = {  # entry: tensors by name, and the call
    "moe_route": (dict(logits=_t(3, 8), bias=_t(8), ids=_t(3, 2, dtype=I32), weights=_t(3, 2)),
                  lambda t: G.route(t["logits"], 2, bias=t["bias"], ids=t["ids"], weights=t["weights"])),
    "quantize_i8": (dict(x=_t(3, 32), out=_rows(3, 32), scale=_t(3)), lambda t: G.quantize_i8(t["x"], t["out"], t["scale"])),
    "mul_mat_i8": (dict(w=_rows(5, 32), w_scale=_t(5), x=_rows(3, 32), x_scale=_t(3), out=_t(3, 5), workspace=_t(1024)),
                   lambda t: G.mul_mat_i8(t["w"], t["w_scale"], t["x"], t["x_scale"], t["out"], t["workspace"])),
    "mul_mat_id_i8": (dict(w=_rows(4, 5, 32), w_scale=_t(4, 5), x=_rows(3, 1, 32), ids=_t(3, 2, dtype=I32), x_scale=_t(3, 1),
                           out=_t(3, 2, 5), workspace=_t(1024)),
                      lambda t: G.mul_mat_id_i8(t["w"], t["w_scale"], t["x"], t["ids"], t["x_scale"], t["out"], t["workspace"])),
    "moe_combine": (dict(y=_t(3, 2, 8), weights=_t(3, 2), ids=_t(3, 2, dtype=I32), add=_t(3, 8), out=_t(3, 8)),
                    lambda t: G.combine(t["y"], t["weights"], t["ids"], t["add"], t["out"])),
}


@pytest.mark.parametrize("entry", ARGS)
def test_tensors_on_one_gpu(entry, library):
    tensors, call = ARGS[entry]
    call({k: On(t) for k, t in tensors.items()})
    call({k: On(t, 1) for k, t in tensors.items()})
    assert library.calls == [f"hip_qmm_{entry}"] * 2
    for name in tensors:
        for elsewhere in (-1, 1):
            with pytest.raises(G.HipQmmError):
                call({k: On(t, elsewhere if k == name else 0) for k, t in tensors.items()})
    assert len(library.calls) == 2


@pytest.mark.parametrize("entry", ARGS)
def test_types_and_shapes(entry, library):
    tensors, call = ARGS[entry]
    for name, t in tensors.items():
        if name == "workspace":
            continue
        wrong = [t.to(torch.float64 if t.dtype != I8 else torch.uint8), t[:-1], t.new_zeros(*t.shape, 1)]
        if name in ("bias", "scale", "w_scale", "x_scale"):
            wrong.pop()  # of these the number of values counts
        for bad in wrong:
            with pytest.raises(G.HipQmmError):
                call({k: On(bad if k == name else u) for k, u in tensors.items()})
    for name, t in tensors.items():
        if name == "workspace" or t.dim() < 2:
            continue
        if name in ("scale", "w_scale", "x_scale"):
            continue
        twice = t.new_zeros(*t.shape[:-1], 2 * t.shape[-1])[..., ::2]  # elements apart
        with pytest.raises(G.HipQmmError):
            call({k: On(twice if k == name else u) for k, u in tensors.items()})
    assert not library.calls


@pytest.mark.parametrize("entry", ["mul_mat_i8", "mul_mat_id_i8"])
def test_rows_of_bytes(entry, library):
    tensors, call = ARGS[entry]
    for name in ("w", "x"):
        t = tensors[name]
        flat = torch.zeros(8192, dtype=torch.int8)
        at = -flat.data_ptr() % 16
        shift = flat[at + 8:at + 8 + t.numel()].view(t.shape)
        odd = flat[at:at + t.numel() // 32 * 40].view(*t.shape[:-1], 40)[..., :32]
        same = t[..., :1, :].expand(t.shape) if t.shape[-2] > 1 else None
        for bad in (shift, odd, same):
            if bad is not None:
                with pytest.raises(G.HipQmmError):
                    call({k: On(bad if k == name else u) for k, u in tensors.items()})
    assert not library.calls


def test_the_last_rows_chunk(library):
    """Rows whose length is no multiple of 16 are read to the next one: never behind the tensor's memory."""
    def call(w, x):
        G.mul_mat_i8(On(w), On(_t(w.shape[0])), On(x), On(_t(x.shape[0])))
    def rows(n, K, total):
        s = torch.zeros(total + 16, dtype=torch.int8)
        at = -s.data_ptr() % 16
        s = s[at:at + total].clone() if at == 0 else s[at:at + total]
        return s
    good = _rows(3, 32)[:, :20]
    call(good, good)
    tail = torch.zeros(2 * 32 + 20, dtype=torch.int8)
    if tail.data_ptr() % 16 == 0:
        short = tail.as_strided((3, 20), (32, 1))
        for a, b in ((short, good), (good, short)):
            with pytest.raises(G.HipQmmError):
                call(a, b)
    assert len(library.calls) == 1


@pytest.mark.parametrize("entry", ["mul_mat_i8", "mul_mat_id_i8"])
def test_workspaces(entry, library):
    tensors, call = ARGS[entry]

    def run(ws):
        call({k: On(ws if k == "workspace" else t) for k, t in tensors.items()})
    run(torch.zeros(1024))  # 4096 bytes
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(4096), torch.zeros(8192, dtype=torch.uint8)[::2],
               torch.zeros(4095, dtype=torch.uint8), torch.zeros(1023)):
        with pytest.raises(G.HipQmmError):
            run(ws)
    assert len(library.calls) == 1


def test_calls_without_tokens(library):
    t = lambda *shape, dtype=torch.float32: On(torch.zeros(shape, dtype=dtype))  # noqa: E731
    w = On(_rows(5, 32))
    assert G.mul_mat_i8(w, t(5), t(0, 32)).shape == (0, 5)
    assert G.mul_mat_id_i8(On(_rows(2, 5, 32)), t(2, 5), t(0, 1, 32), t(0, 3, dtype=I32)).shape == (0, 3, 5)
    assert G.mul_mat_i8(On(_rows(5, 32)[:, :20]), t(5), t(0, 20, dtype=I8), t(0)).shape == (0, 5)
    assert G.combine(t(0, 2, 8), t(0, 2)).shape == (0, 8)
    assert G.quantize_i8(t(0, 32))[0].shape == (0, 32)
    assert not library.calls


def test_unknown_gating(library):
    with pytest.raises(G.HipQmmError):
        G.route(On(_t(2, 8)), 2, gating="relu")
    with pytest.raises(G.HipQmmError):
        G.route(On(_t(2, 8)), 0)
    assert not library.calls


def test_one_row_an_expert(library):
    """Rows of quantize_i8 as weights of experts with one row each, by indexing: 16-byte aligned and as far apart."""
    ids, x = On(_t(3, 2, dtype=I32)), On(_t(3, 1, 20))
    for w in (_rows(4, 32)[:, :20][:, None], _rows(4, 1, 32)[..., :20], _rows(4, 5, 32)[:, 2:3, :20]):
        assert G.mul_mat_id_i8(On(w), On(_t(4, 1)), x, ids).shape == (3, 2, 1)
    assert len(library.calls) == 3
    for w in (_rows(4, 20)[:, None], _rows(4, 40)[:, :20][:, None]):
        with pytest.raises(G.HipQmmError):
            G.mul_mat_id_i8(On(w), On(_t(4, 1)), x, ids)
    assert len(library.calls) == 3


@pytest.mark.parametrize("shape", [(3, 0), (2, 3, 0), (1, 1, 0)])
def test_rows_without_values(shape, monkeypatch):
    """The library's refusal (a row has 1 to 131071 values), whatever the dimensions."""
    real = M._lib()
    monkeypatch.setattr(M, "_lib", lambda: real)
    monkeypatch.setattr(M, "_raw_stream", lambda *_: 0)
    with pytest.raises(G.HipQmmError):
        G.quantize_i8(On(torch.zeros(shape)))
