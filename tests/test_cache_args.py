"""Refusals of rotary, of the 4-bit cache's entry points and of the attention over it, which
answer before they touch a device."""

import contextlib
import ctypes as C
import types

import pytest

from tests.conftest import load_package

ob = load_package()
F32, BF16, F16, E4M3 = 0, 1, 2, 3
# Addresses that nothing reads: a refused call launches nothing.
Q, QO, K, KO, P, F, L, T, W = (0x10000 * i for i in range(1, 10))
I6, I12 = C.c_int64 * 6, C.c_int64 * 12


@pytest.fixture(scope="module")
def lib():
    path = ob.native.PKG / "libomni_b200.so"
    if not path.is_file():
        pytest.skip("library not built")
    return ob.library().lib


def _rotary(lib, **k):
    a = dict(q=Q, qo=QO, k=K, ko=KO, positions=P, frequencies=F, axes=bytes(32), batch=2, heads=4, kv_heads=2, tokens=8,
             head_dim=64, pairs=32, n_axes=2, strides=None, p_strides=None, adjacent=0, inverse=0, position_type=0,
             f64=0, dtype=BF16)
    a.update(k)
    return lib.omni_b200_rotary(*a.values(), None)


PLAIN = [2048, 512, 64]


@pytest.mark.parametrize("status,bad", [
    (1, dict(q=None)), (1, dict(qo=None)), (1, dict(k=None)), (1, dict(ko=None)), (1, dict(positions=None)),
    (1, dict(frequencies=None)), (1, dict(dtype=E4M3)), (1, dict(dtype=-1)), (1, dict(position_type=3)),
    (1, dict(position_type=-1)), (1, dict(batch=-1)), (1, dict(tokens=-1)), (1, dict(heads=0)),
    (1, dict(heads=65536)), (1, dict(kv_heads=0)), (1, dict(kv_heads=-1)), (1, dict(head_dim=0)),
    (1, dict(head_dim=63)), (1, dict(head_dim=65537)), (1, dict(pairs=0)), (1, dict(pairs=33, axes=None)),
    (1, dict(pairs=257, axes=None, head_dim=1024)), (1, dict(n_axes=0)), (1, dict(n_axes=257)),
    (1, dict(axes=bytes([0] * 31 + [2]))), (1, dict(q=Q + 1)), (1, dict(qo=QO + 1)), (1, dict(k=K + 1)),
    (1, dict(ko=KO + 1)), (1, dict(positions=P + 2)), (1, dict(positions=P + 4, position_type=1)),
    (1, dict(frequencies=F + 2)), (1, dict(frequencies=F + 4, f64=1)), (1, dict(ko=QO)), (1, dict(qo=K)),
    (1, dict(ko=Q)), (1, dict(strides=I12(63, 512, 64, *PLAIN, *PLAIN, *PLAIN))),
    (1, dict(strides=I12(*PLAIN, *PLAIN, *PLAIN, 2048, 512, 0))),
    (1, dict(strides=I12(*PLAIN, (1 << 38) + 1, 512, 64, *PLAIN, *PLAIN))),
    (1, dict(qo=Q, strides=I12(*PLAIN, 2048, 512, 128, *PLAIN, *PLAIN))),
    (1, dict(ko=K, strides=I12(*PLAIN, *PLAIN, *PLAIN, 4096, 512, 64))),
    (1, dict(p_strides=(C.c_int64 * 3)(8, -1, 1))), (4, dict(batch=1 << 20, tokens=1 << 20)),
])
def test_rotary_refuses(lib, status, bad):
    assert _rotary(lib, **bad) == status
    assert b"rotary" in lib.omni_b200_last_error()


def _described(**k):
    a = dict(data=Q, table=T, pages=8, page_tokens=32, table_width=3, page_stride=2 * 2304, head_stride=2304)
    a.update(k)
    return ob.native._CacheE2m1(*a.values())


BAD_CACHES = [
    dict(data=None), dict(data=Q + 8), dict(table=T + 2), dict(pages=0), dict(pages=-1), dict(page_tokens=0),
    dict(page_tokens=24), dict(page_tokens=-16), dict(table_width=0), dict(table_width=1 << 26), dict(table=None, pages=1),
    dict(page_stride=2 * 2304 - 8), dict(page_stride=2288), dict(head_stride=2288), dict(head_stride=2312),
    dict(page_stride=0), dict(head_stride=0), dict(page_stride=(1 << 38) + 16),
]


def _rows(lib, read, cache=None, **k):
    a = dict(k=K, v=KO, lengths=L, counts=W, batch=2, heads=2, rows=4, head_dim=64, strides=None, dtype=BF16)
    a.update(k)
    described = C.byref(_described(**(cache or {}))) if cache != "none" else None
    k, v, rest = a["k"], a["v"], list(a.values())[2:]
    if read:
        return lib.omni_b200_cache_read_e2m1(described, k, v, *rest, None)
    return lib.omni_b200_cache_write_e2m1(k, v, described, *rest, None)


BAD_ROWS = [
    (1, dict(k=None)), (1, dict(v=None)), (1, dict(lengths=None)), (1, dict(lengths=L + 2)), (1, dict(counts=W + 1)),
    (1, dict(batch=-1)), (1, dict(heads=0)), (1, dict(rows=-1)), (1, dict(rows=(1 << 30) + 1)), (1, dict(head_dim=0)),
    (1, dict(head_dim=60)), (1, dict(head_dim=136)), (1, dict(dtype=E4M3)), (1, dict(k=K + 8)), (1, dict(v=KO + 2)),
    (1, dict(strides=I6(512, 256, 60, 512, 256, 64))), (1, dict(strides=I6(512, 256, 64, 512, 260, 64))),
    (1, dict(strides=I6(512, 256, 64, 512, 0, 64))), (1, dict(strides=I6((1 << 38) + 8, 256, 64, 512, 256, 64))),
    (4, dict(batch=8, rows=1 << 30, heads=10)),
]


@pytest.mark.parametrize("read", [False, True])
def test_cache_rows_refuse(lib, read):
    name = b"cache_read_e2m1" if read else b"cache_write_e2m1"
    for status, bad in BAD_ROWS + [(1, dict(cache=c)) for c in BAD_CACHES] + [(1, dict(cache="none"))]:
        assert _rows(lib, read, **bad) == status, bad
        assert name in lib.omni_b200_last_error()
    assert _rows(lib, read, rows=0, k=None, v=None, lengths=None, cache=dict(data=None)) == 0
    assert _rows(lib, read, batch=0, k=None, v=None) == 0
    assert _rows(lib, False, dtype=F32) == 1


def _window(lib, cache=None, **k):
    a = dict(q=K, out=KO, lengths=L, counts=W, batch=2, heads=4, kv_heads=2, rows=1, kv_len=96, head_dim=64,
             strides=None, window=0, right=0, sinks=0, scale=0.0, dtype=BF16, out_dtype=BF16, workspace=None, bytes=0)
    a.update(k)
    q, rest = a.pop("q"), a
    described = C.byref(_described(**(cache or {}))) if cache != "none" else None
    return lib.omni_b200_attention_window_e2m1(q, described, *rest.values(), None)


@pytest.mark.parametrize("status,bad", [
    (1, dict(q=None)), (1, dict(out=None)), (1, dict(lengths=None)), (1, dict(lengths=L + 1)), (1, dict(counts=W + 2)),
    (1, dict(batch=-1)), (1, dict(heads=3)), (1, dict(heads=0)), (1, dict(kv_heads=0)), (1, dict(rows=-1)),
    (1, dict(kv_len=0)), (1, dict(kv_len=97)), (1, dict(kv_len=-1)), (1, dict(head_dim=4)), (1, dict(head_dim=256)),
    (1, dict(window=(1 << 30) + 1)), (1, dict(right=-1)), (1, dict(right=(1 << 30) + 1)), (1, dict(sinks=-1)),
    (1, dict(scale=float("nan"))), (1, dict(scale=float("inf"))), (1, dict(dtype=F32)), (1, dict(out_dtype=F16)),
    (1, dict(q=K + 8)), (1, dict(out=KO + 1)), (1, dict(rows=2, strides=I6(512, 128, 60, 512, 128, 64))),
    (1, dict(strides=I6(256, 68, 64, 256, 64, 64))), (1, dict(strides=I6(256, 64, 64, 256, 0, 64))),
    (1, dict(rows=600)), (1, dict(rows=600, workspace=Q, bytes=2 * 2 * 96 * 64 * 4 - 1)),
    (1, dict(rows=600, workspace=Q + 8, bytes=1 << 20)), (1, dict(rows=1 << 30, batch=1 << 10)),
    (1, dict(cache="none")),
] + [(1, dict(cache=c)) for c in BAD_CACHES])
def test_window_refuses(lib, status, bad):
    assert _window(lib, **bad) == status
    assert b"attention_window_e2m1" in lib.omni_b200_last_error()


def test_queries_of_sizes(lib):
    assert lib.omni_b200_cache_e2m1_bytes(16, 128) == 2304 and lib.omni_b200_cache_e2m1_bytes(64, 72) == 4 * 18 * 96
    for tokens, dim in ((0, 64), (8, 64), (16, 0), (16, 60), (16, 136), (16, -8), (1 << 31, 64)):
        assert lib.omni_b200_cache_e2m1_bytes(tokens, dim) == 0
    size = lib.omni_b200_attention_window_e2m1_workspace
    assert size(2, 4, 2, 1, 4096, 64, 0, 0, 0) == 0
    assert size(2, 4, 2, 4096, 4096, 64, 0, 0, 0) == 2 * 2 * 4096 * 64 * 4
    assert size(2, 4, 3, 4096, 4096, 64, 0, 0, 0) == 0 and size(-1, 4, 2, 4096, 4096, 64, 0, 0, 0) == 0
    # No queries, no work: no pointer is looked at.
    assert _window(lib, rows=0, q=None, out=None, lengths=None) == 0
    assert _window(lib, batch=0, q=None, out=None, lengths=None) == 0
    assert _rotary(lib, tokens=0, q=None, qo=None, k=None, ko=None, positions=None, frequencies=None) == 0


def test_helpers_refuse():
    torch = pytest.importorskip("torch")
    bf16 = torch.bfloat16
    q, k = torch.zeros(2, 4, 3, 64, dtype=bf16), torch.zeros(2, 2, 3, 64, dtype=bf16)
    where, frequencies = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(32)
    held, cache = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 1152, dtype=torch.uint8)
    refused = pytest.raises(ob.NativeError)
    for bad in (
        dict(q=q[0]), dict(q=q.double()), dict(k=k.half()), dict(k=k[:1]), dict(k=k[..., :32]), dict(k=k[0]),
        dict(positions=where.double()), dict(positions=where[:1]), dict(positions=where[None, None]),
        dict(frequencies=frequencies.half()), dict(frequencies=frequencies[None]), dict(frequencies=frequencies[::2]),
        dict(axes=bytes(31)), dict(q_out=q[:1]), dict(q_out=q.half()), dict(k_out=k.half()), dict(k=None, k_out=k),
        dict(q=q.transpose(2, 3).contiguous().transpose(2, 3)), dict(),
    ):
        a = dict(q=q, k=k, positions=where, frequencies=frequencies)
        a.update(bad)
        with refused:
            ob.rotary(**a)
    for bad in (
        dict(k=k.float(), v=k.float()), dict(v=k.half()), dict(v=k[:, :1]), dict(k=q, v=q), dict(cache=cache[0]),
        dict(cache=cache.view(torch.int8)), dict(cache=cache[..., :1000]), dict(cache=cache[..., ::2]),
        dict(cache=cache[..., :0]), dict(lengths=held[:1]), dict(lengths=held.long()), dict(q_lengths=held.float()),
        dict(table=held), dict(table=held.view(1, 2)), dict(table=held.view(2, 1).long()),
        dict(k=k[..., :60], v=k[..., :60]), dict(),
    ):
        a = dict(k=k, v=k, cache=cache, lengths=held)
        a.update(bad)
        with refused:
            ob.cache_write_e2m1(**a)
    for bad in (
        dict(head_dim=0), dict(head_dim=128, rows=3, cache=cache[..., :1152]), dict(lengths=held[None]),
        dict(dtype=torch.float64), dict(out=(k, k.half())), dict(out=(k, k), rows=4), dict(out=(k, k), dtype=torch.float32),
        dict(out=(k[..., :32], k[..., :32])), dict(out=(q, q)), dict(rows=2), dict(),
    ):
        a = dict(cache=cache, head_dim=64, lengths=held)
        a.update(bad)
        with refused:
            ob.cache_read_e2m1(**a)
    for bad in (
        dict(q=q.float()), dict(q=q[0]), dict(window=1 << 31), dict(sinks=-(1 << 31)), dict(right=1 << 40),
        dict(kv_len=1 << 31), dict(kv_len=-1), dict(out=q.float()[:1]), dict(out=q.half()), dict(out_dtype=torch.float16),
        dict(q=q[..., :24]), dict(lengths=held[:1]), dict(),
    ):
        a = dict(q=q, cache=cache, lengths=held)
        a.update(bad)
        with refused:
            ob.attention_window_e2m1(**a)
    for bad in ((0, 2, 16, 64), (2, 0, 16, 64), (2, 2, 8, 64), (2, 2, 16, 60), (2, 2, -16, 64), (2, 2, 1 << 31, 64)):
        with refused:
            ob.empty_cache_e2m1(*bad, device="cpu")
    assert ob.empty_cache_e2m1(3, 2, 32, 80, device="cpu").shape == (3, 2, 2 * 18 * 96)
    for bad in ([], [0, 0], [3, -1]):
        with refused:
            ob.rotary_axes(bad)


NAMES = ["rotary", "rotary of q alone", "cache_read_e2m1", "attention_window_e2m1", "attention_window_e2m1 of a prompt",
         "attention_window_e2m1 of a prompt into a tensor"]


def _calls(torch, device):
    g = torch.Generator().manual_seed(3)
    q = torch.randn(2, 4, 600, 64, generator=g).to(torch.bfloat16).to(device)
    where = torch.arange(600, dtype=torch.int32, device=device).expand(2, 600)
    frequencies = torch.rand(32, generator=g).to(device)
    cache = torch.zeros(2, 2, 608 // 16 * 1152, dtype=torch.uint8, device=device)
    held = torch.full((2,), 600, dtype=torch.int32, device=device)
    return {
        "rotary": lambda s: ob.rotary(q, q[:, :2], where, frequencies, stream=s),
        "rotary of q alone": lambda s: ob.rotary(q, None, where, frequencies, stream=s),
        "cache_read_e2m1": lambda s: ob.cache_read_e2m1(cache, 64, held, rows=600, stream=s),
        "attention_window_e2m1": lambda s: ob.attention_window_e2m1(q[:, :, :1], cache, held, stream=s),
        "attention_window_e2m1 of a prompt": lambda s: ob.attention_window_e2m1(q, cache, held, stream=s),
        "attention_window_e2m1 of a prompt into a tensor":
            lambda s: ob.attention_window_e2m1(q, cache, held, out=torch.zeros_like(q), stream=s),
    }


@pytest.mark.parametrize("name", NAMES)
def test_allocations_and_launch_are_the_streams(lib, monkeypatch, name):
    """Outputs and workspaces are made, and the kernel launched, while the stream is the current one."""
    torch = pytest.importorskip("torch")
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

    call = _calls(torch, "cpu")[name]
    native._t.codes  # looks torch's names up
    monkeypatch.setattr(native._t, "cuda", types.SimpleNamespace(stream=enter))
    monkeypatch.setattr(torch.Tensor, "new_empty", watched(torch.Tensor.new_empty))
    monkeypatch.setattr(native._t, "empty_like", watched(torch.empty_like))
    monkeypatch.setattr(native, "_device_of", lambda *_: 0)
    monkeypatch.setattr(native, "_call", lambda *_: launched.append(bool(entered) and entered[-1] is stream))
    call(stream)
    assert made and all(made) and launched == [True] and not entered
