"""The layer operators where a kernel goes round: stages of a ring that are filled again,
rows past those that run at once.  Each test says which kernel its shapes reach, and fails
when a change of the rules that choose a kernel takes them elsewhere.  Tolerances as in
test_layer_gpu.py."""

import re

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import tests.test_layer_gpu as base  # noqa: E402
from tests.launches import launched  # noqa: E402
from tests.test_layer_gpu import BF16, F16, F32, _half_step, _product64  # noqa: E402


@pytest.fixture(scope="module")
def ob():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from tests.conftest import load_package

    return load_package()


# ----------------------------------------------------- products of few rows
def _few_rows(call, tmp_path):
    """(rows of a tile, CTAs of a cluster, stages of a CTA's ring) of a product of few rows."""
    (name, grid, _), = launched(call, tmp_path)
    found = re.search(r"linear_e4m3_fewILi(\d+)E", name)
    assert found, name
    tile = int(found.group(1))
    return tile, grid[0], 180 * 1024 // (128 * 128 + tile * 128)  # FewShape<tile>::STAGES


# m, n, k, rows of the tile, CTAs of a cluster.  With one CTA the sums go out without a
# cluster (tiles of 64 and 128 rows never run so: the other kernel is cheaper there).
FEW = [(1, 16385, 4100, 16, 1), (13, 9600, 2000, 16, 1), (7, 8192, 8192, 16, 2), (1, 1024, 14336, 16, 8),
       (32, 14336, 4096, 32, 1), (20, 16385, 2000, 32, 1), (17, 1000, 14340, 32, 8), (64, 8200, 4096, 64, 2),
       (61, 1101, 14336, 64, 8), (128, 4096, 8192, 128, 4), (100, 641, 8200, 128, 8), (120, 300, 14336, 128, 8)]


def _e4m3(values):
    """e4m3 [rows, k] with a row pitch of 16 bytes and NaN between the rows."""
    rows, k = values.shape
    wide = torch.full((rows, (k + 15) // 16 * 16 + 16), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    wide[:, :k] = values.to(torch.float8_e4m3fn)
    return wide[:, :k]


@pytest.mark.parametrize("m,n,k,tile,parts", FEW)
def test_linear_of_few_rows_refills_its_ring(ob, tmp_path, m, n, k, tile, parts):
    """More groups of k to a CTA than its ring has stages."""
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    groups = -(-k // 128)
    a, w = (_e4m3((torch.randn(rows, k, generator=g, device="cuda") * 40).clamp(-448, 448)) for rows in (m, n))
    sa, sw = (torch.exp(torch.randn(rows, groups, generator=g, device="cuda")) * 2.0**-8 for rows in (m, -(-n // 128)))
    got_tile, got_parts, stages = _few_rows(lambda: ob.linear_e4m3(a, sa, w, sw), tmp_path)
    assert (got_tile, got_parts) == (tile, parts) and groups // parts > stages
    ref, mag = _product64(a, sa, w, sw)
    for dtype, with_bias in ((F32, False), (BF16, True), (F16, False)):
        bias = torch.randn(n, generator=g, device="cuda").to(dtype) if with_bias else None
        got = ob.linear_e4m3(a, sa, w, sw, bias=bias, out_dtype=dtype)
        want = ref + bias.double() if with_bias else ref
        err = (got.double() - want).abs()
        tol = mag * 2.0**-11 + (mag + want.abs()) * (groups + 3) * 2.0**-24 + _half_step(want, dtype) * (1 + 2.0**-8)
        assert bool((err <= tol).all()), f"{dtype}: worst {float((err / tol).max()):.3f} of the tolerance"
        assert torch.equal(got, ob.linear_e4m3(a, sa, w, sw, bias=bias, out_dtype=dtype))
    ob.library().sync_check()


@pytest.mark.parametrize("m,n,k,tile,parts", FEW)
def test_linear_of_few_rows_is_exact_on_whole_numbers(ob, tmp_path, m, n, k, tile, parts):
    """Values in {-2..2}, scales in {1/2, 1, 2}: a group's sum is a whole number of at most
    2^9, a factor one of 2^-2..2^2, so the sums of up to 113 groups are multiples of 2^-2
    below 2^18: 20 bits, exact in any order.  A stage read a turn early or late shows."""
    g = torch.Generator(device="cuda").manual_seed(m)
    groups = -(-k // 128)
    a, w = (_e4m3(torch.randint(-2, 3, (rows, k), generator=g, device="cuda").float()) for rows in (m, n))
    sa, sw = (torch.exp2(torch.randint(-1, 2, (rows, groups), generator=g, device="cuda").float())
              for rows in (m, -(-n // 128)))
    got_tile, got_parts, stages = _few_rows(lambda: ob.linear_e4m3(a, sa, w, sw, out_dtype=F32), tmp_path)
    assert (got_tile, got_parts) == (tile, parts) and groups // parts > stages
    ref, _ = _product64(a, sa, w, sw)
    for _ in range(3):
        assert torch.equal(ob.linear_e4m3(a, sa, w, sw, out_dtype=F32).double(), ref)
    ob.library().sync_check()


# ------------------------------------------------------- quantised quotients
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols,pad", [(20000, 1024, 0), (20000, 1152, 0), (20000, 1000, 24), (20000, 997, 0),
                                           (20000, 1024, 3)])
def test_quantize_rounds_as_a_division(ob, rows, cols, pad, block_rows, dtype):
    """Every byte is that of x / scale in fp32, rounded to nearest even.  Quotients half way
    between two e4m3 values are what tells: of 8.4 million such inputs a product with the
    scale's reciprocal rounds 4158 otherwise in bf16, 460 in fp16 and 4 in fp32."""
    g = torch.Generator(device="cuda").manual_seed(rows + cols + pad)
    wide = torch.exp(torch.randn(cols + pad, generator=g, device="cuda"))
    x = (torch.randn(rows, cols + pad, generator=g, device="cuda") * wide).to(dtype)[:, :cols]
    q, s = ob.quantize_e4m3(x, block_rows=block_rows)
    scales = s.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    # A 53-bit quotient rounded to 24 bits is the 24-bit quotient (53 >= 2 * 24 + 2).
    want = (x.double() / scales.double()).float().to(torch.float8_e4m3fn)
    assert torch.equal(q.view(torch.uint8), want.view(torch.uint8))
    top = torch.zeros(-(-rows // block_rows) * block_rows, -(-cols // 128) * 128, device="cuda")
    top[:rows, :cols] = x.abs()
    top = top.view(-1, block_rows, s.shape[1], 128).amax(dim=(1, 3))
    assert torch.equal(s, (top.double() / 448).float())
    ob.library().sync_check()


# -------------------------------------------------------- norms of many rows
def _goes_round(call, rows, kernel, tmp_path):
    """That the call's kernel is `kernel`, with fewer CTAs than its rows would take."""
    (name, (grid,), _), = launched(call, tmp_path)
    found = re.search(r"(rows(?:_\w+)?_kernel)I(?:f|6__half|13__nv_bfloat16)((?:L[bi]\d+E)+)E", name)
    assert found, name
    numbers = [int(n) for n in re.findall(r"L[bi](\d+)E", found.group(2))][1:]
    assert (found.group(1), *numbers) == kernel
    each = {"rows_kernel": lambda tpr, vpt, r: r, "rows_odd_kernel": lambda warps, groups: 8 // warps,
            "rows_stream_kernel": lambda tpr, vpt: 256 // tpr, "rows_scalar_kernel": lambda: 1}[kernel[0]](*numbers)
    assert rows > grid * each


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,cols,kernel", [
    # Widths that 16-byte loads cannot read.
    (20000, 33, ("rows_odd_kernel", 1, 4)), (20000, 1013, ("rows_odd_kernel", 1, 8)),
    (2500, 2001, ("rows_odd_kernel", 8, 2)), (2500, 3727, ("rows_odd_kernel", 8, 4)),
    (2500, 8191, ("rows_odd_kernel", 8, 8)), (2500, 9001, ("rows_scalar_kernel",)),
    (1500, 16400, ("rows_scalar_kernel",)),  # more than registers hold
    # A warp, or a CTA, for each row.
    (20000, 200, ("rows_kernel", 32, 1, 4)), (9000, 512, ("rows_kernel", 32, 2, 4)), (9000, 1024, ("rows_kernel", 32, 4, 4)),
    (9000, 1152, ("rows_kernel", 32, 5, 4)), (9000, 1536, ("rows_kernel", 32, 6, 4)),
    (2700, 1544, ("rows_kernel", 128, 2, 1)), (2040, 2048, ("rows_kernel", 128, 2, 1)),
    (1020, 4096, ("rows_kernel", 128, 4, 1)), (500, 8192, ("rows_kernel", 256, 4, 1)),
    (1100, 8200, ("rows_kernel", 512, 4, 1)), (1100, 12000, ("rows_kernel", 512, 4, 1)),
    (1100, 16384, ("rows_kernel", 512, 4, 1)),
    # The ring.
    (2501, 2048, ("rows_stream_kernel", 64, 4)), (1501, 4096, ("rows_stream_kernel", 128, 4)),
    (1031, 8192, ("rows_stream_kernel", 256, 4)),
], ids=lambda v: "-".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_rms_norm_of_more_rows_than_run_at_once(ob, tmp_path, rows, cols, kernel, dtype):
    """With and without a residual, in both output types, and in place."""
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x, res, w = (torch.randn(*n, generator=g, device="cuda").to(dtype) for n in ((rows, cols), (rows, cols), (cols,)))
    for r in (None, res):
        _goes_round(lambda: ob.rms_norm(x, w, residual=r), rows, kernel, tmp_path)
        _goes_round(lambda: ob.rms_norm_e4m3(x, w, residual=r), rows, kernel, tmp_path)
        h, y = base._norm64(x, w, r, 1e-6)
        got, hout = ob.rms_norm(x, w, residual=r)
        base._check_rounded(got, y, dtype, 48 * 2.0**-24)
        q, scales, hq = ob.rms_norm_e4m3(x, w, residual=r)
        base._check_quantized(q, scales, y)
        if r is not None:
            base._check_rounded(hout, h, dtype, 2.0**-24)
            assert torch.equal(hout, hq)
        del h, y
    ob.rms_norm(x, w, residual=res, residual_out=res, out=x)
    assert torch.equal(x, got) and torch.equal(res, hout)
    ob.library().sync_check()


# ------------------------------------------------------------- far-off rows
def _far(t, total=2**32 + 2**20):
    """The same rows, so far apart that the last one lies past 2^32 elements."""
    rows, cols = t.shape
    stride = -(-total // (rows - 1) // 16) * 16
    wide = torch.empty((rows - 1) * stride + cols, dtype=t.dtype, device="cuda").as_strided((rows, cols), (stride, 1))
    wide.view(torch.uint8 if t.element_size() == 1 else t.dtype).copy_(t.view(torch.uint8) if t.element_size() == 1 else t)
    return wide


@pytest.mark.parametrize("rows,cols", [(9, 1024), (9, 999), (130, 4096), (3, 20001), (600, 8192)])
def test_rows_past_32_bits(ob, rows, cols):
    g = torch.Generator(device="cuda").manual_seed(cols)
    x, res, w = (torch.randn(*n, generator=g, device="cuda").to(BF16) for n in ((rows, cols), (rows, cols), (cols,)))
    want, hwant = ob.rms_norm(x, w, residual=res)
    xf, rf, out = _far(x), _far(res), _far(torch.zeros_like(x))
    got, h = ob.rms_norm(xf, w, residual=rf, residual_out=rf, out=out)
    assert torch.equal(got, want) and torch.equal(h, hwant)
    for block_rows in (1, 128):
        q, s = ob.quantize_e4m3(x, block_rows=block_rows)
        qf, sf = ob.quantize_e4m3(xf, block_rows=block_rows)
        assert torch.equal(qf.view(torch.uint8), q.view(torch.uint8)) and torch.equal(sf, s)
    ob.library().sync_check()


@pytest.mark.parametrize("m,n,k,kernel", [(5, 700, 1024, "few"), (33, 257, 1100, "few"), (300, 600, 512, "big")])
def test_product_of_rows_past_32_bits(ob, tmp_path, m, n, k, kernel):
    g = torch.Generator(device="cuda").manual_seed(m)
    a, sa = ob.quantize_e4m3(torch.randn(m, k, generator=g, device="cuda"))
    w, sw = ob.quantize_e4m3(torch.randn(n, k, generator=g, device="cuda"), block_rows=128)
    want = ob.linear_e4m3(a, sa, w, sw)
    af, wf, out = _far(a), _far(w), _far(torch.zeros_like(want))
    (name, _, _), = launched(lambda: ob.linear_e4m3(af, sa, wf, sw, out=out), tmp_path)
    assert f"linear_e4m3_{kernel}" in name
    out.zero_()
    assert torch.equal(ob.linear_e4m3(af, sa, wf, sw, out=out), want)
    ob.library().sync_check()
