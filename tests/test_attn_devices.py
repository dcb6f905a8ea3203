"""What the Python side of the attention operators asks of its tensors' places,
on the CPU: tensors that only claim a GPU, and a library that only notes its
calls."""
import pytest

import ggml_hip as G
from ggml_hip import attn as A

torch = pytest.importorskip("torch")


class On:
    """A CPU tensor that says it lives on a GPU (-1: the CPU)."""

    def __init__(self, t, device=0):
        self._t, self._on = t, device

    def __getattr__(self, name):
        return getattr(self._t, name)

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
    monkeypatch.setattr(A, "_lib", lambda: lib)
    monkeypatch.setattr(A, "_raw_stream", lambda *_: 0)
    return lib


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _kv(device=0):
    c = torch.zeros((4, 2, 16, 64), dtype=torch.float16)
    return G.PagedKV(On(c, device), On(c, device))


ARGS = {  # entry: tensors by name, and the call
    "attn_paged": (dict(q=torch.zeros(3, 4, 64), table=_i32(3, 2), lens=_i32(3), starts=_i32(4), out=torch.zeros(3, 4, 64),
                        workspace=torch.zeros(4096, dtype=torch.uint8)),
                   lambda kv, t: G.attn_paged(t["q"], kv, t["table"], t["lens"], q_starts=t["starts"], out=t["out"],
                                              workspace=t["workspace"])),
    "kv_compact": (dict(table=_i32(3, 2), lens=_i32(3), out=_i32(3, 2), workspace=torch.zeros(4096, dtype=torch.uint8)),
                   lambda kv, t: G.compact_pages(kv, t["table"], t["lens"], out=t["out"], workspace=t["workspace"])),
    "kv_copy_pages": (dict(src=_i32(3), dst=_i32(3), n=_i32(3)), lambda kv, t: G.copy_pages(kv, t["src"], t["dst"], t["n"])),
    "rope_kv_store": (dict(q=torch.zeros(3, 4, 64), k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), pos=_i32(3),
                           steps=torch.zeros(32, dtype=torch.int64), slots=_i32(3), out=torch.zeros(3, 4, 64)),
                      lambda kv, t: G.rope_kv_store(t["q"], t["k"], t["v"], t["pos"], t["steps"], kv, t["slots"], out=t["out"])),
    "rope_f32": (dict(x=torch.zeros(3, 4, 64), pos=_i32(3), steps=torch.zeros(32, dtype=torch.int64), out=torch.zeros(3, 4, 64)),
                 lambda kv, t: G.rope(t["x"], t["pos"], t["steps"], out=t["out"])),
}


@pytest.mark.parametrize("entry", ARGS)
def test_tensors_on_one_gpu(entry, library):
    tensors, call = ARGS[entry]
    call(_kv(), {k: On(t) for k, t in tensors.items()})
    call(_kv(1), {k: On(t, 1) for k, t in tensors.items()})
    assert library.calls == [f"hip_qmm_{entry}"] * 2
    for name in tensors:
        for elsewhere in (-1, 1):
            with pytest.raises(G.HipQmmError):
                call(_kv(), {k: On(t, elsewhere if k == name else 0) for k, t in tensors.items()})
    assert len(library.calls) == 2


@pytest.mark.parametrize("entry", ["attn_paged", "kv_compact"])
def test_workspaces(entry, library):
    tensors, call = ARGS[entry]
    def run(ws):
        call(_kv(), {k: On(ws if k == "workspace" else t) for k, t in tensors.items()})
    run(torch.zeros(1024))  # 4096 bytes
    assert len(library.calls) == 1
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(4096), torch.zeros(8192, dtype=torch.uint8)[::2],
               torch.zeros(4095, dtype=torch.uint8), torch.zeros(1023)):
        with pytest.raises(G.HipQmmError):
            run(ws)
    assert len(library.calls) == 1


def test_the_current_gpu(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 70 + device)
    assert A._raw_stream(1) == 71
    with pytest.raises(G.HipQmmError):
        A._raw_stream(0)


def test_calls_without_tokens(monkeypatch):
    """Empty tensors have no address: nothing to do, as for the C entries with no tokens."""
    monkeypatch.setattr(A, "_raw_stream", lambda *_: 0)
    t = lambda *shape, dtype=torch.float32: On(torch.zeros(shape, dtype=dtype))  # noqa: E731
    pos, steps, kv = t(0, dtype=torch.int32), t(32, dtype=torch.int64), _kv()
    assert G.rope(t(0, 4, 64), pos, steps).shape == (0, 4, 64)
    assert G.rope(t(3, 0, 64), t(3, dtype=torch.int32), steps).shape == (3, 0, 64)
    out = t(0, 4, 64)
    assert G.rope(t(0, 4, 64), pos, steps, out=out) is out
    none = t(0, 2, 64)
    assert G.rope_kv_store(t(0, 4, 64), none, none, pos, steps, kv, pos).shape == (0, 4, 64)
    assert G.rope_kv_store(None, none, none, pos, steps, kv, pos) is None
    G.copy_pages(kv, pos, pos)
    assert G.attn_paged(t(0, 4, 64), kv, t(0, 2, dtype=torch.int32), pos).shape == (0, 4, 64)
    with pytest.raises(G.HipQmmError):
        G.rope(t(0, 4, 64), t(1, dtype=torch.int32), steps)
    with pytest.raises(G.HipQmmError):
        G.rope_kv_store(t(0, 4, 64), none, none, pos, steps, kv, pos, layout="other")
