"""The 8-bit layer operators on the GPU against the same formulas in 64 bits.

Tolerances, from arithmetic:
  * rms_norm: fp32 throughout, rounded once.  A sum of squares of at most 2^14
    columns is added in chains of at most 64 and a tree of at most 10 levels: relative
    error below 74 * 2^-24, halved by the root; rsqrt and three products add 5 *
    2^-24.  48 * 2^-24 covers it.  The output's rounding is half a step: eps / 2 of
    the value, or half of fp16's smallest step.
  * e4m3: half a step is 2^-4 of the value, at least 2^-10 of the scale (steps of
    2^-9 below 2^-6).  Relative slack of 2^-16 for the scale's and the value's own
    fp32 errors.
  * linear_e4m3: products of e4m3 values are exact.  The tensor cores keep at least
    13 bits below the largest addend (what 8-bit pipelines of the generation before
    kept), four additions a group: at most 2^-11 of the sum of magnitudes; plus the
    output's rounding.  Where every sum is a small whole number the result is exact.
"""

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ob():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from tests.conftest import load_package

    return load_package()


def _randn(*shape, seed, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def _strided(t, pad):
    """The same rows with `pad` columns between them."""
    wide = torch.full((t.shape[0], t.shape[1] + pad), 7.0, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _norm64(x, w, res, eps):
    h = x.double() + (res.double() if res is not None else 0)
    return h, h / torch.sqrt(h.square().mean(dim=1, keepdim=True) + eps) * w.double()


def _half_step(ref, dtype):
    eps = torch.finfo(dtype).eps / 2
    return ref.abs() * eps + (2.0**-25 if dtype == F16 else 0.0)


def _check_rounded(got, ref, dtype, relative):
    assert got.dtype == dtype
    err = (got.double() - ref).abs()
    tol = ref.abs() * relative + _half_step(ref, dtype) * (1 + 2.0**-8) + 1e-37
    assert bool((err <= tol).all()), f"worst {float((err - tol).max()):.3e} past the tolerance"


def _group_max(y, block_rows=1):
    rows, cols = y.shape
    pr, pc = -(-rows // block_rows) * block_rows, -(-cols // 128) * 128
    wide = torch.zeros(pr, pc, dtype=torch.float64, device=y.device)
    wide[:rows, :cols] = y.abs()
    return wide.view(pr // block_rows, block_rows, pc // 128, 128).amax(dim=(1, 3))


def _widen(scales, rows, cols, block_rows=1):
    return scales.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def _check_quantized(q, scales, y, block_rows=1):
    rows, cols = y.shape
    assert q.dtype == torch.float8_e4m3fn and q.shape == y.shape
    want = (_group_max(y, block_rows) / 448).clamp_min(2.0**-126)
    assert scales.shape == want.shape
    assert bool(((scales.double() - want).abs() <= want * 2.0**-17).all())
    s = _widen(scales, rows, cols, block_rows)
    err = (q.double() * s - y).abs()
    tol = torch.maximum(y.abs() * 2.0**-4, s * 2.0**-10) * (1 + 2.0**-12) + y.abs() * 2.0**-16
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.4f} of the tolerance"


NORM_SHAPES = [(1, 1), (3, 7), (1, 8), (5, 64), (2, 128), (9, 136), (1, 1000), (4, 1024), (301, 1152), (7, 2048),
               (2, 4096), (3, 4304), (5, 8192), (2, 8200), (2, 16384), (2, 16392), (1, 20001), (700, 250)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_rms_norm(ob, rows, cols, dtype):
    x = _randn(rows, cols, seed=cols + rows, dtype=dtype)
    res = _randn(rows, cols, seed=cols + rows + 1, dtype=dtype, scale=3.0)
    w = _randn(cols, seed=cols, dtype=dtype)
    for r in (None, res):
        h, y = _norm64(x, w, r, 1e-5)
        got, hout = ob.rms_norm(x, w, residual=r, eps=1e-5)
        _check_rounded(got, y, dtype, 48 * 2.0**-24)
        q, scales, hq = ob.rms_norm_e4m3(x, w, residual=r, eps=1e-5)
        _check_quantized(q, scales, y)
        if r is None:
            assert hout is None and hq is None
        else:
            _check_rounded(hout, h, dtype, 2.0**-24)
            assert torch.equal(hout, hq)
    ob.library().sync_check()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,cols", [(2500, 33), (2500, 511), (1300, 513), (1300, 1013), (1300, 1025), (301, 2001),
                                       (301, 3727), (301, 4097), (1300, 8191), (40, 9001)])
def test_rms_norm_of_rows_that_vectors_cannot_read(ob, rows, cols, dtype):
    """Odd columns, each kernel with more rows than run at once; and in place."""
    test_rms_norm(ob, rows, cols, dtype)
    x, res, w = (_randn(*n, seed=cols + i, dtype=dtype) for i, n in enumerate([(rows, cols), (rows, cols), (cols,)]))
    want, hwant = ob.rms_norm(x, w, residual=res)
    ob.rms_norm(x, w, residual=res, residual_out=res, out=x)
    assert torch.equal(x, want) and torch.equal(res, hwant)


@pytest.mark.parametrize("rows,cols", [(20000, 200), (9000, 512), (9000, 1152), (9000, 1280), (5000, 1536), (5000, 2048),
                                       (3000, 8192)])
def test_rms_norm_of_many_rows(ob, rows, cols):
    """More rows than run at once, whose next ones are loaded ahead; and in place."""
    test_rms_norm(ob, rows, cols, BF16)
    x, res, w = (_randn(*n, seed=cols + i, dtype=BF16) for i, n in enumerate([(rows, cols), (rows, cols), (cols,)]))
    want, hwant = ob.rms_norm(x, w, residual=res)
    ob.rms_norm(x, w, residual=res, residual_out=res, out=x)
    assert torch.equal(x, want) and torch.equal(res, hwant)


@pytest.mark.parametrize("cols", [257, 512, 1152])
def test_rms_norm_strides_and_places(ob, cols):
    """Pitched rows, a residual updated in place, and an output in x's place."""
    x, res = _randn(33, cols, seed=1, dtype=BF16), _randn(33, cols, seed=2, dtype=BF16)
    w = _randn(cols, seed=3, dtype=BF16)
    want, hwant = ob.rms_norm(x, w, residual=res)
    xs, rs, wide = _strided(x, 8), _strided(res, 24), _strided(torch.zeros_like(x), 16)
    got, h = ob.rms_norm(xs, w, residual=rs, residual_out=rs, out=wide)
    assert torch.equal(got, want) and torch.equal(rs, hwant) and h is rs
    assert bool((xs._base[:, cols:] == 7).all()) and bool((rs._base[:, cols:] == 7).all())
    x2 = x.clone()
    ob.rms_norm(x2, w, residual=res, out=x2)
    assert torch.equal(x2, want)
    x3 = x.clone()
    got3, _ = ob.rms_norm(x3, w, residual=res, residual_out=x3)
    assert torch.equal(got3, want) and torch.equal(x3, hwant)


def test_rms_norm_zero_nan_and_inf_rows(ob):
    """A row of zeros gives zeros, a NaN its own row's NaNs, other rows stay."""
    x = _randn(6, 1024, seed=5, dtype=BF16)
    x[1] = 0
    x[2, 77] = float("nan")
    x[3, 500] = float("inf")
    w = _randn(1024, seed=6, dtype=BF16)
    y, _ = ob.rms_norm(x, w)
    q, s, _ = ob.rms_norm_e4m3(x, w)
    clean = [0, 4, 5]
    assert bool(torch.isfinite(y[clean].float()).all()) and bool((y[1] == 0).all())
    assert bool(torch.isnan(y[2].float()).all())
    assert bool(torch.isnan(y[3, 500].float())) and bool((y[3, :500] == 0).all())
    assert bool((q[1].float() == 0).all()) and bool((s[1] == 2.0**-126).all())
    _check_quantized(q[clean], s[clean], _norm64(x[clean], w, None, 1e-6)[1])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 130), (127, 200), (128, 256), (129, 1152), (300, 4304),
                                       (17, 77), (40, 17000)])
def test_quantize(ob, rows, cols, block_rows, dtype):
    x = _randn(rows, cols, seed=rows * cols, dtype=dtype, scale=0.3)
    q, s = ob.quantize_e4m3(x, block_rows=block_rows)
    _check_quantized(q, s, x.double(), block_rows)
    wide = _strided(x, 16 if cols % 16 == 0 else 3)
    q2, s2 = ob.quantize_e4m3(wide, block_rows=block_rows)
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(9001, 128), (9001, 997), (30001, 64), (9001, 1152), (2001, 4097), (3001, 4304)])
def test_quantize_many_rows(ob, rows, cols, block_rows, dtype):
    """More groups than run at once, a row's last one short or single."""
    x = _randn(rows, cols, seed=rows + cols, dtype=dtype, scale=0.3)
    q, s = ob.quantize_e4m3(x, block_rows=block_rows)
    _check_quantized(q, s, x.double(), block_rows)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("cols", [120, 125, 384])
def test_quantize_to_any_address(ob, cols, block_rows):
    """q at an odd address with an odd pitch; the bytes between its rows stay."""
    x = _randn(150, cols, seed=cols, dtype=BF16)
    want, s = ob.quantize_e4m3(x, block_rows=block_rows)
    pitch = cols + 7
    room = torch.full((150 * pitch + 3,), 0x55, dtype=torch.uint8, device="cuda")
    s2 = torch.empty_like(s)
    lib = ob.library()
    lib.check(lib.lib.omni_b200_quantize_e4m3(x.data_ptr(), room.data_ptr() + 3, s2.data_ptr(), 150, cols, cols, pitch,
                                              block_rows, 1, torch.cuda.current_stream().cuda_stream))
    got = room[3:].view(150, pitch)
    assert torch.equal(got[:, :cols], want.view(torch.uint8)) and torch.equal(s2, s)
    assert bool((got[:, cols:] == 0x55).all()) and bool((room[:3] == 0x55).all())


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("cols", [384, 390])
def test_quantize_special_values(ob, block_rows, cols):
    x = _randn(200, cols, seed=9)
    x[:, :128] = 0
    x[5, 130] = float("nan")
    x[6, 300] = float("inf")
    x[7, 256:cols] = 1e-42  # subnormal: the scale stays at its floor for a row of them
    q, s = ob.quantize_e4m3(x, block_rows=block_rows)
    f = q.float()
    assert bool((f[:, :128] == 0).all()) and bool((s[:, 0] == 2.0**-126).all())
    assert bool(torch.isnan(f[5, 130])) and int(torch.isnan(f[:, 128:256]).sum()) == 1
    block = 6 if block_rows == 1 else 0
    assert bool(torch.isinf(s[block, 2])) and bool(torch.isnan(f[6, 300])) and float(f[6, 299]) == 0
    assert bool(torch.isfinite(f[8 if block_rows == 1 else 150]).all())


def test_quantize_every_value(ob):
    """e4m3 values with the scale 1 come back as they are (448 in each group)."""
    codes = torch.tensor([c for c in range(256) if c & 0x7F != 0x7F], dtype=torch.uint8)
    v = codes.view(torch.float8_e4m3fn).float()
    x = torch.full((2, 128), 448.0)
    x[0, :127], x[1, :127] = v[:127], v[127:]
    q, s = ob.quantize_e4m3(x.cuda())
    assert bool((s == 1).all()) and torch.equal(q.float().cpu(), x)


# ------------------------------------------------------------------ products
def _operands(m, n, k, seed):
    """e4m3 operands with row pitches of 16 bytes and scales over a few octaves."""
    def matrix(rows, pitch, s):
        t = torch.zeros(rows, pitch, dtype=torch.uint8).view(torch.float8_e4m3fn)
        t[:, :k] = torch.randn(rows, k, generator=torch.Generator().manual_seed(s)).mul(40).clamp(-448, 448).to(
            torch.float8_e4m3fn)
        t.view(torch.uint8)[:, k:] = 0x7F  # NaN between the rows: never read
        return t.cuda()[:, :k]

    pitch, groups = (k + 15) // 16 * 16, -(-k // 128)
    a, w = matrix(m, pitch, seed), matrix(n, pitch + 16, seed + 1)
    sa = torch.exp(_randn(m, groups, seed=seed + 2)) * 2.0**-8
    sw = torch.exp(_randn(-(-n // 128), groups, seed=seed + 3)) * 2.0**-8
    return a, sa, w, sw


def _product64(a, sa, w, sw):
    (m, k), n = a.shape, w.shape[0]
    da, dw = a.double() * _widen(sa, m, k), w.double() * _widen(sw, n, k, 128)
    return da @ dw.t(), da.abs() @ dw.abs().t()


PRODUCTS = [(1, 1, 16), (1, 128, 128), (1, 4096, 4096), (3, 200, 100), (7, 129, 1), (16, 256, 1152), (17, 300, 129),
            (32, 64, 640), (33, 1152, 1152), (61, 4304, 1152), (64, 512, 2000), (65, 384, 256), (128, 1000, 4304),
            (129, 257, 130), (300, 640, 512), (513, 128, 1024), (2500, 1101, 200), (2500, 1104, 1152),
            (20000, 64, 256), (1300, 2304, 640)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_linear(ob, m, n, k):
    a, sa, w, sw = _operands(m, n, k, seed=m + n + k)
    ref, mag = _product64(a, sa, w, sw)
    for dtype, with_bias in ((F32, False), (BF16, True), (F16, True), (F32, True)):
        bias = _randn(n, seed=k, dtype=dtype) if with_bias else None
        got = ob.linear_e4m3(a, sa, w, sw, bias=bias, out_dtype=dtype)
        want = ref + bias.double() if with_bias else ref
        err = (got.double() - want).abs()
        # fp32: the groups' sums, the scales' product and the bias, one rounding each.
        groups = -(-k // 128)
        tol = mag * 2.0**-11 + (mag + want.abs()) * (groups + 3) * 2.0**-24 + _half_step(want, dtype) * (1 + 2.0**-8)
        assert bool((err <= tol).all()), f"{dtype}: worst {float((err / tol).max()):.3f} of the tolerance"
        assert torch.equal(got, ob.linear_e4m3(a, sa, w, sw, bias=bias, out_dtype=dtype))
    ob.library().sync_check()


@pytest.mark.parametrize("m,n,k", [(1, 130, 384), (19, 256, 1152), (128, 513, 640), (200, 300, 4096), (2500, 1300, 1152),
                                   (1300, 4304, 256)])
def test_linear_exact_on_whole_numbers(ob, m, n, k):
    """Values in {-2..2} and power-of-two scales: every partial sum is a whole number
    of at most 2^11 before the scales, so nothing may be off."""
    g = torch.Generator().manual_seed(m)
    a = torch.randint(-2, 3, (m, k), generator=g).float().cuda()
    w = torch.randint(-2, 3, (n, k), generator=g).float().cuda()
    groups = -(-k // 128)
    sa = torch.exp2(torch.randint(-2, 3, (m, groups), generator=g).float()).cuda()
    sw = torch.exp2(torch.randint(-2, 3, (-(-n // 128), groups), generator=g).float()).cuda()
    a, w = a.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    ref, _ = _product64(a, sa, w, sw)
    assert torch.equal(ob.linear_e4m3(a, sa, w, sw, out_dtype=F32).double(), ref)


@pytest.mark.parametrize("m,n", [(5, 200), (150, 64), (2500, 1100)])
def test_linear_writes_its_rows_only(ob, m, n):
    """A pitched output: the columns between the rows and the rows behind stay."""
    a, sa, w, sw = _operands(m, n, 256, seed=4)
    want = ob.linear_e4m3(a, sa, w, sw)
    for pad in (8, 3):
        wide = torch.full((m + 3, n + pad), 5.0, dtype=BF16, device="cuda")
        ob.linear_e4m3(a, sa, w, sw, out=wide[:m, :n])
        assert torch.equal(wide[:m, :n], want)
        assert bool((wide[:, n:] == 5).all()) and bool((wide[m:] == 5).all())


@pytest.mark.parametrize("m", [3, 100, 2500])
def test_linear_nan_stays_in_its_row(ob, m):
    a, sa, w, sw = _operands(m, 1100, 300, seed=8)
    want = ob.linear_e4m3(a, sa, w, sw)
    a.view(torch.uint8)[1, 200] = 0x7F
    got = ob.linear_e4m3(a, sa, w, sw)
    assert bool(torch.isnan(got[1].float()).all())
    keep = [r for r in range(m) if r != 1]
    assert torch.equal(got[keep], want[keep])


def test_empty_calls(ob):
    x, w = torch.empty(0, 256, dtype=BF16, device="cuda"), _randn(256, seed=1, dtype=BF16)
    y, _ = ob.rms_norm(x, w)
    q, s, h = ob.rms_norm_e4m3(x, w, residual=x)
    assert y.shape == (0, 256) and q.shape == (0, 256) and s.shape == (0, 2) and h.shape == (0, 256)
    wq, ws = ob.quantize_e4m3(_randn(300, 256, seed=2), block_rows=128)
    assert ob.linear_e4m3(q, s, wq, ws).shape == (0, 300)
    assert ob.quantize_e4m3(x)[0].shape == (0, 256)
    ob.library().sync_check()


@pytest.mark.parametrize("rows", [2, 300, 2500])
def test_layer_captured_and_replayed(ob, rows):
    """Norm, product and quantisation in one graph on a stream of its own; a replay
    sees new inputs, and two graphs do not disturb each other."""
    w = _randn(1152, seed=1, dtype=BF16)
    wq, ws = ob.quantize_e4m3(_randn(1104, 1152, seed=2, scale=0.03), block_rows=128)

    def layer(x, r):
        q, s, h = ob.rms_norm_e4m3(x, w, residual=r)
        y = ob.linear_e4m3(q, s, wq, ws)
        q2, s2 = ob.quantize_e4m3(y)
        return h, y, q2.view(torch.uint8), s2

    stream = torch.cuda.Stream()
    captured = []
    for seed in (10, 20):
        x, r = _randn(rows, 1152, seed=seed, dtype=BF16), _randn(rows, 1152, seed=seed + 1, dtype=BF16)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = layer(x, r)
        captured.append((graph, x, r, out))
    for k in range(2):
        for graph, x, r, out in captured:
            x.copy_(_randn(rows, 1152, seed=30 + k, dtype=BF16))
            graph.replay()
        torch.cuda.synchronize()
        for graph, x, r, out in captured:
            for got, want in zip(out, layer(x, r)):
                assert torch.equal(got, want)
    ob.library().sync_check()


def test_linear_on_two_streams_at_once(ob):
    args = [_operands(m, 1100, 1152, seed=m) for m in (4, 2500)]
    want = [ob.linear_e4m3(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(10):
        for s, a in zip(streams, args):
            got.append(ob.linear_e4m3(*a, stream=s))
            with torch.cuda.stream(s):
                got[-1].record_stream(s)
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2])
    ob.library().sync_check()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,cols", [(32771, 128), (9001, 512), (4099, 1024), (2503, 2048), (1501, 4096), (1031, 8192),
                                       (3650, 1152), (977, 4304)])
def test_rms_norm_many_rows(ob, rows, cols, dtype):
    """Enough rows for the kernel that streams them, the last turn not full; pitched
    rows, the residual updated in place."""
    x = _strided(_randn(rows, cols, seed=cols, dtype=dtype), 16)
    res = _randn(rows, cols, seed=cols + 1, dtype=dtype, scale=3.0)
    w = _randn(cols, seed=cols, dtype=dtype)
    h, y = _norm64(x, w, res, 1e-5)
    q, scales, hq = ob.rms_norm_e4m3(x, w, residual=res, eps=1e-5)
    _check_quantized(q, scales, y)
    _check_rounded(hq, h, dtype, 2.0**-24)
    inplace = _strided(res, 8)
    got, hout = ob.rms_norm(x, w, residual=inplace, eps=1e-5, residual_out=inplace)
    _check_rounded(got, y, dtype, 48 * 2.0**-24)
    assert torch.equal(hout, hq) and bool((inplace._base[:, cols:] == 7).all())
    got, _ = ob.rms_norm(x, w, eps=1e-5)
    _check_rounded(got, _norm64(x, w, None, 1e-5)[1], dtype, 48 * 2.0**-24)
    q, scales = ob.quantize_e4m3(x)
    _check_quantized(q, scales, x.double())
    ob.library().sync_check()


@pytest.mark.parametrize("cols", [1, 997, 1000])
def test_empty_calls_with_odd_columns(ob, cols):
    """No rows, of a width that the producers pad: a layer with nothing to do."""
    x, w = torch.empty(0, cols, dtype=BF16, device="cuda"), _randn(cols, seed=1, dtype=BF16)
    wq, ws = ob.quantize_e4m3(_randn(300, cols, seed=2), block_rows=128)
    bias = _randn(300, seed=3, dtype=BF16)
    for q, s in (ob.quantize_e4m3(x), ob.rms_norm_e4m3(x, w)[:2], ob.rms_norm_e4m3(x, w, residual=x)[:2]):
        assert ob.linear_e4m3(q, s, wq, ws, bias=bias).shape == (0, 300)
    ob.library().sync_check()
