"""Where the operators' outputs lie when a call is given a stream of its own: in that
stream's memory, not in a block that the current stream has just freed and a kernel
there may still use, nor in one that goes back to the current stream while the call
is under way."""

import contextlib
import types

import pytest

from tests.conftest import load_package

torch = pytest.importorskip("torch")
ob = load_package()
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def _calls(device, rows, cols, heads):
    """Each helper with its inputs made: name -> call(stream) -> the tensors that it made."""
    g = torch.Generator().manual_seed(3)
    x, r, w = (torch.randn(*n, generator=g).to(BF16).to(device) for n in ((rows, cols), (rows, cols), (cols,)))
    a = torch.randn(rows, cols, generator=g).to(E4M3).to(device)
    b = torch.randn(256, cols, generator=g).to(E4M3).to(device)
    sa, sb = torch.ones(rows, cols // 128, device=device), torch.ones(2, cols // 128, device=device)
    q = torch.randn(2, heads, 40, 64, generator=g).to(BF16).to(device)
    return {
        "rms_norm": lambda s: ob.rms_norm(x, w, residual=r, stream=s),
        "rms_norm_e4m3": lambda s: ob.rms_norm_e4m3(x, w, residual=r, stream=s),
        "rms_norm_e4m3 of pitched rows": lambda s: ob.rms_norm_e4m3(x[:, :125], w[:125], residual=r[:, :125], stream=s),
        "quantize_e4m3": lambda s: ob.quantize_e4m3(x, stream=s),
        "quantize_e4m3 in blocks": lambda s: ob.quantize_e4m3(x, block_rows=128, stream=s),
        "linear_e4m3": lambda s: (ob.linear_e4m3(a, sa, b, sb, stream=s),),
        "attention_window": lambda s: (ob.attention_window(q, q, q, window=9, stream=s),),
    }


NAMES = ["rms_norm", "rms_norm_e4m3", "rms_norm_e4m3 of pitched rows", "quantize_e4m3", "quantize_e4m3 in blocks",
         "linear_e4m3", "attention_window"]


@pytest.mark.parametrize("name", NAMES)
def test_allocations_and_launch_are_the_streams(monkeypatch, name):
    """On the host, with what stands between the helpers and a device replaced: every
    allocation and the launch happen while the stream is the current one."""
    native, entered, made, launched = ob.native, [], [], []
    stream = types.SimpleNamespace(cuda_stream=0x77, device_index=0)

    @contextlib.contextmanager
    def enter(s):
        entered.append(s)
        yield
        entered.pop()

    def watched(make):
        def call(*args, **kwargs):
            made.append(bool(entered) and entered[-1] is stream)
            return make(*args, **kwargs)

        return call

    call = _calls("cpu", 4, 256, 2)[name]
    native._t.codes  # looks torch's names up
    monkeypatch.setattr(native._t, "cuda", types.SimpleNamespace(stream=enter))
    monkeypatch.setattr(native._t, "empty_like", watched(torch.empty_like))
    monkeypatch.setattr(torch.Tensor, "new_empty", watched(torch.Tensor.new_empty))
    monkeypatch.setattr(native, "_device_of", lambda *_: 0)
    monkeypatch.setattr(native, "_call", lambda *_: launched.append(bool(entered) and entered[-1] is stream))
    call(stream)
    assert made and all(made) and launched == [True] and not entered
    made.clear(), launched.clear()
    call(None)
    assert made and not any(made) and launched == [False]


def test_calls_that_make_no_tensor_stay_on_the_current_stream(monkeypatch):
    """They are launched on the stream that was given, and it is not entered."""
    native, launched = ob.native, []
    stream = types.SimpleNamespace(cuda_stream=0x77, device_index=0)
    x = torch.zeros(4, 256, dtype=BF16)
    a, b, s = x.to(E4M3), torch.zeros(256, 256).to(E4M3), torch.ones(4, 2)
    q = torch.zeros(2, 2, 40, 64, dtype=BF16)
    native._t.codes
    monkeypatch.setattr(native._t, "cuda", None)
    monkeypatch.setattr(native._t, "empty_like", None)
    monkeypatch.setattr(torch.Tensor, "new_empty", None)
    monkeypatch.setattr(native, "_device_of", lambda *_: 0)
    monkeypatch.setattr(native, "_call", lambda name, device, on, *_: launched.append(on))
    ob.rms_norm(x, x[0], out=x, stream=stream)
    ob.rms_norm(x, x[0], residual=x, out=x.clone(), residual_out=x, stream=stream)
    ob.linear_e4m3(a, s, b, s[:2], out=x, stream=stream)
    ob.attention_window(q, q, q, out=q.clone(), stream=stream)
    assert launched == [stream] * 4


def test_a_stream_of_another_device_is_refused():
    stream = types.SimpleNamespace(cuda_stream=0x77, device_index=1)
    tensor = types.SimpleNamespace(get_device=lambda: 0)
    with pytest.raises(ob.NativeError, match="stream must be on the tensors' device"):
        ob.native._on("rms_norm", stream, tensor)


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _blocks(tensors):
    """The storages' address ranges."""
    found = []
    for t in tensors:
        if t is not None:
            s = t.untyped_storage()
            found.append((s.data_ptr(), s.data_ptr() + s.nbytes()))
    return found


def _apart(left, right):
    return all(a1 <= b0 or b1 <= a0 for a0, a1 in left for b0, b1 in right)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_outputs_are_no_memory_of_the_current_stream(gpu, name):
    """Neither blocks that the current stream has freed, nor, once dropped, blocks that
    it is given next; and the results are those of a plain call."""
    call = _calls("cuda", 300, 1024, 4)[name]
    want = [t for t in call(None) if t is not None]
    kept = [t.clone() for t in want]
    shapes = [(t.shape, t.dtype) for t in want]
    freed = _blocks(want)
    del want
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    # The freed blocks are still being written on the current stream when the call comes.
    busy = [torch.empty(s, dtype=d, device="cuda") for s, d in shapes]
    torch.cuda._sleep(20_000_000)
    for b in busy:
        b.view(torch.uint8).fill_(0x55)
    freed += _blocks(busy)
    del busy, b
    got = [t for t in call(stream) if t is not None]
    assert _apart(_blocks(got), freed)
    torch.cuda.synchronize()
    for g, k in zip(got, kept):
        assert torch.equal(g.view(torch.uint8), k.view(torch.uint8))
    dropped = _blocks(got)
    del got, g
    assert _apart(_blocks([torch.empty(s, dtype=d, device="cuda") for s, d in shapes]), dropped)
    ob.library().sync_check()


def _older_calls(device):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, 4, 70, 64, generator=g).to(BF16).to(device)
    rows = torch.randn(2 * 70, 4 * 72, generator=g).to(device)
    held = torch.full((2,), 70, dtype=torch.int32, device=device)
    return {
        "attention_bhld": lambda s: ob.attention_bhld(x, x, x, stream=s),
        "attention_rows": lambda s: ob.attention_rows(rows, rows, rows, 4, stream=s),
        "attention_rows of a batch": lambda s: ob.attention_rows(rows, rows, rows, 4, batch=2, lengths=held, stream=s),
    }


OLDER = ["attention_bhld", "attention_rows", "attention_rows of a batch"]


@pytest.mark.parametrize("named", [True, False])
@pytest.mark.parametrize("name", OLDER)
def test_attention_outputs_and_workspaces_are_the_streams(monkeypatch, name, named):
    """The bidirectional attention's helpers, with a torch stream and with an object that
    only has its cuda_stream."""
    native, entered, made, launched = ob.native, [], [], []
    stream = types.SimpleNamespace(cuda_stream=0x77, **({"device_index": 0} if named else {}))
    torch_stream = stream if named else types.SimpleNamespace(cuda_stream=0x77, device_index=-1)

    @contextlib.contextmanager
    def enter(s):
        entered.append(s)
        yield
        entered.pop()

    real_empty = torch.empty

    def empty(*args, **kwargs):
        made.append(bool(entered) and entered[-1] is torch_stream)
        return real_empty(*args, **kwargs)

    class Entry:
        def __getattr__(self, name):
            return lambda *args: (1 << 10 if name.endswith("workspace") else
                                  launched.append(entered[-1].cuda_stream if entered else 0))

    call = _older_calls("cpu")[name]
    native._t.codes
    monkeypatch.setattr(native._t, "cuda", types.SimpleNamespace(
        stream=enter, ExternalStream=lambda ptr, device: torch_stream if ptr == 0x77 else None))
    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: entered[-1] if entered else stream)
    monkeypatch.setattr(native, "library", lambda: types.SimpleNamespace(lib=Entry(), check=lambda status: None))
    call(stream)
    assert made and all(made) and launched == [0x77] and not entered


@pytest.mark.gpu
@pytest.mark.parametrize("name", OLDER)
def test_attention_outputs_are_no_memory_of_the_current_stream(gpu, name):
    call = _older_calls("cuda")[name]
    want = call(None)
    kept, freed = want.clone(), _blocks([want])
    del want
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    busy = torch.empty_like(kept)
    torch.cuda._sleep(20_000_000)
    busy.fill_(3)
    freed += _blocks([busy])
    del busy
    got = call(stream)
    assert _apart(_blocks([got]), freed)
    torch.cuda.synchronize()
    assert torch.equal(got, kept)
    dropped = _blocks([got])
    del got
    assert _apart(_blocks([torch.empty_like(kept)]), dropped)
    ob.library().sync_check()
