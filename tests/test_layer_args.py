"""Refusals of the 8-bit layer entry points, which answer before they touch a
device: bad arguments are refused on a machine without one."""

import ctypes as C

import pytest

from tests.conftest import load_package

ob = load_package()
E4M3, BF16, F32, F16 = 3, 1, 0, 2
# Addresses that nothing reads: a refused call launches nothing.
X, R, W, H, O, S = (0x10000 * i for i in range(1, 7))


@pytest.fixture(scope="module")
def lib():
    path = ob.native.PKG / "libomni_b200.so"
    if not path.is_file():
        pytest.skip("library not built")
    return ob.library().lib


def _norm(lib, **k):
    a = dict(x=X, residual=R, weight=W, residual_out=H, out=O, scales=None, rows=4, cols=256, xs=256, rs=256, hs=256,
             os=256, eps=1e-6, dtype=BF16, out_dtype=BF16)
    a.update(k)
    return lib.omni_b200_rms_norm(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(weight=None), dict(out=None), dict(residual=None), dict(residual_out=None), dict(dtype=E4M3),
    dict(dtype=-1), dict(out_dtype=F32), dict(out_dtype=E4M3), dict(scales=S), dict(cols=0), dict(cols=(1 << 24) + 1),
    dict(xs=255), dict(rs=255), dict(hs=0), dict(os=100), dict(xs=(1 << 40) + 8), dict(eps=-1.0),
    dict(eps=float("nan")), dict(eps=float("inf")), dict(x=X + 1), dict(out=O + 1), dict(weight=W + 1),
    dict(out_dtype=E4M3, scales=S + 2), dict(rows=(1 << 40) + 1),
    dict(out=H), dict(out=X, residual_out=X), dict(residual_out=X, hs=264), dict(residual_out=R, hs=264),
    dict(out=X, os=264), dict(out=R, os=264), dict(out=X, out_dtype=E4M3, scales=S),
])
def test_rms_norm_refuses(lib, bad):
    assert _norm(lib, **bad) == 1
    assert b"rms_norm" in lib.omni_b200_last_error()


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(q=None), dict(scales=None), dict(dtype=E4M3), dict(cols=0), dict(block=64), dict(block=0),
    dict(xs=100), dict(qs=255), dict(x=X + 1), dict(scales=S + 1), dict(rows=8388481, block=128),
])
def test_quantize_refuses(lib, bad):
    a = dict(x=X, q=O, scales=S, rows=4, cols=256, xs=256, qs=256, block=1, dtype=BF16)
    a.update(bad)
    assert lib.omni_b200_quantize_e4m3(*a.values(), None) == 1
    assert b"quantize_e4m3" in lib.omni_b200_last_error()


@pytest.mark.parametrize("status,bad", [
    (1, dict(a=None)), (1, dict(sa=None)), (1, dict(w=None)), (1, dict(sw=None)), (1, dict(out=None)),
    (1, dict(n=0)), (1, dict(k=0)), (1, dict(lda=255)), (1, dict(lda=264)), (1, dict(ldw=240)), (1, dict(ldw=257)),
    (1, dict(ldo=127)), (1, dict(a=X + 8)), (1, dict(w=W + 4)), (1, dict(out=O + 1)), (1, dict(bias=R + 1)),
    (1, dict(sa=S + 2)), (1, dict(dtype=E4M3)), (1, dict(n=(1 << 22) + 1, ldo=1 << 23)),
    (1, dict(m=(1 << 30) + 1)), (4, dict(m=1 << 30, n=1 << 22, ldo=1 << 22)),
])
def test_linear_refuses(lib, status, bad):
    a = dict(a=X, sa=S, w=W, sw=H, bias=None, out=O, m=4, n=128, k=256, lda=256, ldw=256, ldo=128, dtype=BF16)
    a.update(bad)
    assert lib.omni_b200_linear_e4m3(*a.values(), None) == status
    assert b"linear_e4m3" in lib.omni_b200_last_error()


def test_no_rows_is_no_work(lib):
    """Without rows nothing is launched and no pointer is looked at."""
    assert _norm(lib, rows=0, x=None, out=None, weight=None, residual=None, residual_out=None) == 0
    assert lib.omni_b200_quantize_e4m3(None, None, None, 0, 128, 128, 128, 1, BF16, None) == 0
    assert lib.omni_b200_linear_e4m3(None, None, None, None, None, None, 0, 8, 16, 16, 16, 8, BF16, None) == 0


def test_helpers_refuse():
    torch = pytest.importorskip("torch")
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(256, dtype=torch.bfloat16)
    refused = pytest.raises(ob.NativeError)
    for call in (lambda: ob.rms_norm(x, w), lambda: ob.rms_norm_e4m3(x, w), lambda: ob.quantize_e4m3(x)):
        with refused as e:  # tensors of the host
            call()
        assert e.value.status == 1
    q, s = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.zeros(4, 2)
    for call in (
        lambda: ob.rms_norm(x, w.float()),
        lambda: ob.rms_norm(x, w[:128]),
        lambda: ob.rms_norm(x, w, residual=x[:2]),
        lambda: ob.rms_norm(x, w, residual=x.float()),
        lambda: ob.rms_norm(x, w, residual_out=x),
        lambda: ob.rms_norm(x, w, out=x.float()),
        lambda: ob.rms_norm(x.int(), w.int()),
        lambda: ob.quantize_e4m3(x, block_rows=32),
        lambda: ob.quantize_e4m3(x.double()),
        lambda: ob.linear_e4m3(x, s, q, s[:1]),
        lambda: ob.linear_e4m3(q, s, q[:, :128], s[:1]),
        lambda: ob.linear_e4m3(q, s[:3], q, s[:1]),
        lambda: ob.linear_e4m3(q, s.double(), q, s[:1]),
        lambda: ob.linear_e4m3(q, s, q, s[:1], bias=w),
        lambda: ob.linear_e4m3(q, s, q, s[:1], out=x),
        lambda: ob.linear_e4m3(q, s, q, s[:1], out_dtype=torch.float64),
        lambda: ob.linear_e4m3(q, s, q, s[:1]),
    ):
        with refused as e:
            call()
        assert e.value.status == 1


def test_linear_helper_refuses_strided_columns():
    """Of a single row too, whose row stride does not matter."""
    torch = pytest.importorskip("torch")
    q, s = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.zeros(4, 2)
    row = torch.zeros(256, 4).to(torch.float8_e4m3fn)[:, :1].t()  # [1, 256], every fourth element
    for call in (lambda: ob.linear_e4m3(row, s[:1], q, s[:1]), lambda: ob.linear_e4m3(q, s, row, s[:1])):
        with pytest.raises(ob.NativeError, match="columns must be contiguous"):
            call()


def _window(lib, strides=None, **k):
    a = dict(q=X, k=R, v=W, out=O, batch=2, heads=4, kv_heads=2, q_len=3, kv_len=40, hd=64, strides=None, lengths=None,
             q_lengths=None, window=8, right=0, sinks=1, scale=0.0, dtype=BF16, out_dtype=BF16)
    a.update(k)
    if strides is not None:
        a["strides"] = (C.c_int64 * 12)(*strides)
    return lib.omni_b200_attention_window(*a.values(), None)


_PLAIN = [768, 192, 64, 5120, 2560, 64, 5120, 2560, 64, 768, 192, 64]


def _with(i, value):
    return dict(strides=_PLAIN[:i] + [value] + _PLAIN[i + 1:])


@pytest.mark.parametrize("status,bad", [
    (1, dict(q=None)), (1, dict(k=None)), (1, dict(v=None)), (1, dict(out=None)), (1, dict(batch=-1)),
    (1, dict(heads=0)), (1, dict(kv_heads=0)), (1, dict(kv_heads=3)), (1, dict(q_len=-1)), (1, dict(kv_len=0)),
    (1, dict(kv_len=(1 << 30) + 1)), (4, dict(hd=0)), (4, dict(hd=60)), (4, dict(hd=136)), (1, dict(window=2**31 - 1)),
    (1, dict(right=-1)), (1, dict(right=2**31 - 1)), (1, dict(sinks=-1)), (1, dict(sinks=2**31 - 1)),
    (1, dict(scale=float("nan"))), (1, dict(scale=float("inf"))), (1, dict(dtype=F32)), (1, dict(dtype=E4M3)),
    (1, dict(out_dtype=F16)), (1, dict(q=X + 2)), (1, dict(k=R + 8)), (1, dict(v=W + 8)), (1, dict(out=O + 1)),
    (1, dict(lengths=S + 1)), (1, dict(q_lengths=S + 2)), (4, dict(batch=1 << 20, heads=1 << 12)),
    (1, _with(0, 0)), (1, _with(1, 63)), (1, _with(2, 68)), (1, _with(4, -64)), (1, _with(8, 0)), (1, _with(11, 32)),
    (1, _with(5, (1 << 38) + 8)),
])
def test_window_refuses(lib, status, bad):
    assert _window(lib, **bad) == status
    assert b"attention_window" in lib.omni_b200_last_error()


def test_window_without_queries_is_no_work(lib):
    assert _window(lib, batch=0, q=None, k=None, v=None, out=None) == 0
    assert _window(lib, q_len=0, q=None, k=None, v=None, out=None) == 0


def test_window_helper_refuses():
    torch = pytest.importorskip("torch")
    q, k = torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 40, 64, dtype=torch.bfloat16)
    n = torch.zeros(2, dtype=torch.int32)
    for call in (
        lambda: ob.attention_window(q, k, k),  # tensors of the host
        lambda: ob.attention_window(q[0], k, k),
        lambda: ob.attention_window(q, k, k[:, :1]),
        lambda: ob.attention_window(q[:1], k, k),
        lambda: ob.attention_window(q[..., :32], k, k),
        lambda: ob.attention_window(q.half(), k, k),
        lambda: ob.attention_window(q.float(), k.float(), k.float()),
        lambda: ob.attention_window(q, k, k, lengths=n.long()),
        lambda: ob.attention_window(q, k, k, q_lengths=n[:1]),
        lambda: ob.attention_window(q, k, k, out=q[:, :2]),
        lambda: ob.attention_window(q, k, k, out=q, out_dtype=torch.float32),
        lambda: ob.attention_window(q, k, k, out_dtype=torch.float16),
    ):
        with pytest.raises(ob.NativeError) as e:
            call()
        assert e.value.status == 1


@pytest.mark.parametrize("name", ["window", "right", "sinks"])
@pytest.mark.parametrize("value", [1 << 31, (1 << 32) + 5, -(1 << 32) - 1])
def test_window_helper_refuses_what_32_bits_do_not_hold(name, value):
    """They would arrive as other numbers."""
    torch = pytest.importorskip("torch")
    q, k = torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 40, 64, dtype=torch.bfloat16)
    with pytest.raises(ob.NativeError, match="below 2\\^31"):
        ob.attention_window(q, k, k, **{name: value})


@pytest.mark.parametrize("lda,ldw", [(997, 1008), (1008, 997), (0, 0)])
def test_linear_without_rows_looks_at_no_stride(lib, lda, ldw):
    """An empty tensor's pitch is whatever its maker says: torch calls a [0, 997] slice
    of padded rows contiguous, with 997 columns between its rows."""
    assert lib.omni_b200_linear_e4m3(X, S, W, H, None, O, 0, 300, 997, lda, ldw, 300, BF16, None) == 0


def test_linear_helper_of_an_empty_batch_with_odd_columns(lib, monkeypatch):
    torch = pytest.importorskip("torch")
    native = ob.native
    native._t.codes
    monkeypatch.setattr(native, "_device_of", lambda *_: 0)
    monkeypatch.setattr(native, "_call", lambda name, device, stream, *args: ob.library().check(getattr(lib, name)(*args, None)))
    for cols in (997, 1000):
        x = torch.zeros(5, cols, dtype=torch.bfloat16)[:0]
        w = torch.zeros(300, (cols + 15) // 16 * 16).to(torch.float8_e4m3fn)[:, :cols]
        scales = torch.ones(3, 8)
        for q, s in (ob.quantize_e4m3(x), ob.rms_norm_e4m3(x, torch.zeros(cols, dtype=torch.bfloat16))[:2]):
            assert ob.linear_e4m3(q, s, w, scales).shape == (0, 300)
