"""On whose stream empty_cache_e2m1 makes and clears a cache, with stand-ins for CUDA's streams."""

import contextlib
import types

import pytest

from tests.conftest import load_package

ob = load_package()
torch = pytest.importorskip("torch")
SIZES = (2, 2, 16, 64)


@pytest.fixture
def made(monkeypatch):
    """[(device, stream entered)] of the caches that are made."""
    native, entered, made = ob.native, [], []
    if not (native.PKG / "libomni_b200.so").is_file():
        pytest.skip("library not built")

    @contextlib.contextmanager
    def enter(stream):
        assert hasattr(stream, "device_index")  # as torch.cuda.stream wants it
        entered.append(stream)
        yield
        entered.pop()

    def external(pointer, device):
        return types.SimpleNamespace(cuda_stream=pointer, device_index=device)

    native._t.codes  # looks torch's names up
    monkeypatch.setattr(native._t, "cuda", types.SimpleNamespace(stream=enter, ExternalStream=external))
    monkeypatch.setattr(native._t, "current_device", lambda: 1)
    monkeypatch.setattr(native._t, "raw_stream", lambda device: 0)
    monkeypatch.setattr(native._t, "zeros", lambda shape, dtype, device: made.append(
        (str(device), (entered[-1].cuda_stream, entered[-1].device_index) if entered else None)))
    return made


def _stream(device):
    return types.SimpleNamespace(cuda_stream=0x77, device_index=device)


def test_of_the_stream_s_device(made):
    for device in ("cuda", "cuda:3", torch.device("cuda:3")):
        ob.empty_cache_e2m1(*SIZES, device=device, stream=_stream(3))
    assert [s for _, s in made] == [(0x77, 3)] * 3
    del made[:]
    ob.empty_cache_e2m1(*SIZES, device="cuda:1")
    ob.empty_cache_e2m1(*SIZES, device="cpu", stream=_stream(3))
    assert made == [("cuda:1", None), ("cpu", None)]


def test_of_another_library_s_stream(made):
    ob.empty_cache_e2m1(*SIZES, stream=types.SimpleNamespace(cuda_stream=0x88))
    ob.empty_cache_e2m1(*SIZES, device="cuda:2", stream=types.SimpleNamespace(cuda_stream=0x88))
    assert [s for _, s in made] == [(0x88, 1), (0x88, 2)]


def test_another_device_s_stream_is_refused(made):
    with pytest.raises(ob.NativeError):
        ob.empty_cache_e2m1(*SIZES, device="cuda:1", stream=_stream(3))
    assert not made
