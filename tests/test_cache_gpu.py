"""The 4-bit key/value cache on the GPU: writing and reading it against the quantisation's
definition in 64 bits (they are exact), attention over it against softmax attention in 64
bits over what the cache stands for, and all of them as a layer calls them.

Attention's tolerance, from arithmetic.  With A = the softmax-weighted mean of |v|, for each
output element:
  * the weights are rounded for the product with v, to f16 where few queries read the cache,
    to the operand type for prompts, and their sum may be taken before or after that:
    2 * eps / 2 * A;
  * scores are fp32 sums of exact products: at most D * 2^-24 of the sum of magnitudes,
    below 2^-12 in the exponent for these inputs, so 2^-12 * A with the exponential's own
    2^-22;
  * f16 weights below 2^-14 of the row's largest lose at most 2^-25 each, times the
    largest |v|;
  * the output's rounding, half a step.
"""

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
KEPT = 123.0
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


@pytest.fixture(scope="module")
def ob():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from tests.conftest import load_package

    return load_package()


def _i32(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")


def _tensor(shape, layout, dtype, seed, spread=0.0):
    b, h, t, d = shape
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, t, h, d, generator=g)
    if spread:
        x = x * torch.exp(spread * torch.randn(b, t, h, d, generator=g))
    x = x.to(dtype)
    if layout == "tokens":
        return x.cuda().transpose(1, 2)
    if layout == "heads":
        return x.cuda().transpose(1, 2).contiguous()
    wide = torch.full((b, t, h * d + 40), KEPT, dtype=dtype)  # rows of a wider matrix
    wide[..., 16:16 + h * d] = x.flatten(2)
    return wide.cuda()[..., 16:16 + h * d].unflatten(2, (h, d)).transpose(1, 2)


def _stored(x):
    """What the cache stands for, from the definition in 64 bits: every product and comparison
    here is exact, the inputs having at most 11 significant bits."""
    out = torch.full(x.shape, math.nan, dtype=torch.float64, device=x.device)
    x = x.double()
    for at in range(0, x.shape[-1], 32):
        part = x[..., at:at + 32]
        top = part.abs().amax(dim=-1, keepdim=True)
        finite = part.isfinite().all(dim=-1, keepdim=True)
        top = torch.where(finite, top, 1.0)
        low = torch.exp2(torch.frexp(top)[1].double() - 9)  # 6 * 32 * low <= top, or half of that
        low = torch.where(6 * 64 * low <= top, 2 * low, low)
        low = torch.where(6 * 32 * low > top, low / 2, low)  # a step of the scale: 32 to 64 of them
        steps = torch.floor(top / (6 * low))
        steps = steps - (6 * steps * low > top).double() + (6 * (steps + 1) * low <= top).double()
        twice = 2 * (top - 6 * steps * low)  # against 6 * low: below, on or above the middle
        steps = steps + ((twice > 6 * low) | ((twice == 6 * low) & (steps % 2 == 1))).double()
        scale = (steps * low).clamp(2.0**-14, 10752.0)
        value = torch.zeros_like(part)
        for code in range(1, 8):
            middle = (E2M1[code - 1] + E2M1[code]) / 2 * scale
            up = part.abs() >= middle if code % 2 == 0 else part.abs() > middle
            value = torch.where(up, E2M1[code] * scale, value)
        out[..., at:at + 32] = torch.where(finite, value * torch.sign(part), math.nan)
    return out


def _table(batch, each, spare, seed):
    g = torch.Generator().manual_seed(seed)
    pages = batch * each + spare
    return torch.randperm(pages, generator=g)[:batch * each].view(batch, each).to(torch.int32).cuda(), pages


def _made(ob, B, Hkv, D, capacity, page, seed=0):
    """(cache, table): pages in any order, or a page for each sequence (page 0)."""
    if page == 0:
        cache = ob.empty_cache_e2m1(B, Hkv, (capacity + 15) // 16 * 16, D)
        table = None
    else:
        table, pages = _table(B, -(-capacity // page), 3, seed)
        cache = ob.empty_cache_e2m1(pages, Hkv, page, D)
    cache.random_(0, 256, generator=torch.Generator("cuda").manual_seed(seed))
    return cache, table


def _same(a, b):
    a, b = a.double(), b.double()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.masked_fill(a.isnan(), 0.0), b.masked_fill(b.isnan(), 0.0))


# ------------------------------------------------------------ writing and reading
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("layout", ["tokens", "heads", "rows"])
@pytest.mark.parametrize("B,Hkv,D,page,lengths,counts", [
    (1, 1, 8, 16, [1], [1]),
    (1, 2, 128, 0, [37], [37]),
    (3, 8, 128, 64, [1, 64, 200], [1, 1, 1]),
    (2, 3, 64, 32, [100, 31], [100, 31]),
    (4, 2, 80, 16, [33, 0, 16, 50], [5, 0, 16, 17]),
    (2, 1, 96, 48, [150, 97], [60, 1]),
    (2, 5, 72, 0, [200, 3], [9, 3]),
    (1, 2, 32, 128, [1000], [999]),
    (3, 1, 24, 16, [5, 17, 30], [5, 2, 30]),
])
def test_written_and_read(ob, dtype, layout, B, Hkv, D, page, lengths, counts):
    """Rows come back as the definition says; others of the cache and of the outputs stay."""
    capacity, rows = max(max(lengths), 1), max(max(counts), 1)
    cache, table = _made(ob, B, Hkv, D, capacity, page)
    k, v = (_tensor((B, Hkv, rows, D), layout, dtype, s, 1.5) for s in (1, 2))
    held, m = _i32(lengths), _i32(counts)
    whole = torch.full((B,), capacity, dtype=torch.int32, device="cuda")
    before = ob.cache_read_e2m1(cache, D, whole, rows=capacity, table=table, dtype=F32)
    bytes_before = cache.clone()
    assert ob.cache_write_e2m1(k, v, cache, held, q_lengths=m, table=table) is cache
    after = ob.cache_read_e2m1(cache, D, whole, rows=capacity, table=table, dtype=F32)
    got = [torch.full((B, Hkv, rows, D), KEPT, dtype=F32, device="cuda") for _ in range(2)]
    assert ob.cache_read_e2m1(cache, D, held, q_lengths=m, table=table, out=got)[0] is got[0]
    for x, old, new, read in zip((k, v), before, after, got):
        want = _stored(x)
        for b in range(B):
            n, c = lengths[b], counts[b]
            assert _same(read[b, :, :c], want[b, :, :c])
            assert bool((read[b, :, c:] == KEPT).all())
            assert _same(new[b, :, n - c:n], want[b, :, :c])
            assert _same(new[b, :, :n - c], old[b, :, :n - c]) and _same(new[b, :, n:], old[b, :, n:])
    if table is not None:  # pages of no sequence
        spare = [i for i in range(cache.shape[0]) if i not in set(table.flatten().tolist())]
        assert torch.equal(cache[spare], bytes_before[spare])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_every_value_of_the_type(ob, dtype):
    """All 65536 bit patterns, in groups that hold one large value and in groups of neighbours."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    near = bits.view(1, 1, 65536 // 128, 128)
    g = torch.Generator().manual_seed(1)
    mixed = bits[torch.randperm(65536, generator=g)].view(1, 1, 65536 // 128, 128)
    tops = torch.randn(1, 1, 65536 // 128, 4, generator=g).exp().to(dtype) * 4  # scales of all fractions
    small = (mixed.float().nan_to_num(0, 0, 0).clamp(-4, 4)).to(dtype)
    small.view(1, 1, -1, 4, 32)[..., 0] = tops
    held = _i32([512])
    for x in (near, mixed, small):
        x = x.contiguous().cuda()
        cache = ob.empty_cache_e2m1(1, 1, 512, 128)
        ob.cache_write_e2m1(x, x.flip(2).contiguous(), cache, held)
        for read in (F32, BF16, F16):
            k, v = ob.cache_read_e2m1(cache, 128, held, dtype=read)
            want = _stored(x)
            assert k.dtype == read and _same(k, want) and _same(v, want.flip(2))


def test_quotients_in_the_middle(ob):
    """Elements half way between two values, for every fraction of a scale: to the even code."""
    fractions = torch.arange(32, 64).double()  # the scale's six bits
    middles = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    rows = torch.zeros(32, 32, dtype=torch.float64)
    rows[:, 0] = 6 * fractions
    for i, m in enumerate(middles):
        rows[:, 1 + 2 * i], rows[:, 2 + 2 * i] = m * fractions, -m * fractions
    for shift in (-18, -10, 0, 5):
        x = (rows * 2.0**shift).to(F16)
        exact = x.double() == rows * 2.0**shift  # an f16 holds them all (nine bits), its subnormals not
        x = x.view(1, 1, 32, 32).cuda()
        cache = ob.empty_cache_e2m1(1, 1, 32, 32)
        ob.cache_write_e2m1(x, x, cache, _i32([32]))
        k, v = ob.cache_read_e2m1(cache, 32, _i32([32]), dtype=F32)
        assert _same(k, _stored(x)) and torch.equal(k, v)
        if shift >= -10:
            assert bool(exact.all())


def test_layout(ob):
    """The bytes lie as the layout's description says."""
    D, G = 96, 3
    k, v = _tensor((1, 2, 32, D), "heads", BF16, 3), _tensor((1, 2, 32, D), "heads", BF16, 4)
    cache = ob.empty_cache_e2m1(1, 2, 32, D)
    ob.cache_write_e2m1(k, v, cache, _i32([32]))
    data, want = cache.cpu(), (_stored(k).cpu(), _stored(v).cpu())
    size = 18 * D
    assert cache.shape == (1, 2, 2 * size)

    def value(nibble):
        return E2M1[nibble & 7] * (-1 if nibble & 8 else 1)

    for h in range(2):
        for t in range(32):
            block = data[0, h, t // 16 * size:(t // 16 + 1) * size]
            scales = block[16 * D:].view(torch.float16).double()
            r = t % 16
            for d in range(D):
                byte = int(block[r * D // 2 + d // 2])
                s = float(scales[((r % 8) * G + d // 32) * 2 + r // 8])
                assert value(byte >> 4 * (d % 2)) * s == float(want[0][0, h, t, d])
                x, g, c = d // 16, d % 8, r % 8 // 2
                at = 8 * D + x // 2 * 256 + (4 * g + c) * 8 + x % 2 * 4 + r // 8 * 2 + d % 16 // 8
                s = float(scales[16 * G + d // 32 * 16 + c * 4 + r // 8 * 2 + r % 2])
                assert value(int(block[at]) >> 4 * (r % 2)) * s == float(want[1][0, h, t, d])


def test_lengths_out_of_range(ob):
    """Positions below 0 and past the pages are neither read nor written."""
    D, Hkv = 64, 2
    cache, table = _made(ob, 3, Hkv, D, 32, 16, 5)
    k, v = _tensor((3, Hkv, 24, D), "heads", BF16, 6), _tensor((3, Hkv, 24, D), "heads", BF16, 7)
    held = _i32([10, 40, -3])
    ob.cache_write_e2m1(k, v, cache, held, table=table)
    out = [torch.full((3, Hkv, 24, D), KEPT, dtype=BF16, device="cuda") for _ in range(2)]
    ob.cache_read_e2m1(cache, D, held, table=table, out=out)
    for x, got in zip((k, v), out):
        want = _stored(x)
        assert bool((got[0, :, :14] == KEPT).all()) and _same(got[0, :, 14:], want[0, :, 14:])
        assert _same(got[1, :, :16], want[1, :, :16]) and bool((got[1, :, 16:] == KEPT).all())
        assert bool((got[2] == KEPT).all())
    far = _i32([2**31 - 1, 2**30, -2**31])
    before = cache.clone()
    ob.cache_write_e2m1(k, v, cache, far, table=table)
    assert torch.equal(cache, before)


def test_pages_that_are_none(ob):
    """Entries outside the cache: nothing is written there, they read as NaN; entries behind a
    sequence's last page are not looked at."""
    D, Hkv = 64, 2
    cache = ob.empty_cache_e2m1(4, Hkv, 16, D)
    table = _i32([[0, 7, 1], [2, -1, -5]])
    k, v = _tensor((2, Hkv, 40, D), "heads", F16, 8), _tensor((2, Hkv, 40, D), "heads", F16, 9)
    held, m = _i32([40, 15]), _i32([40, 15])
    ob.cache_write_e2m1(k, v, cache, held, q_lengths=m, table=table)
    got = ob.cache_read_e2m1(cache, D, held, rows=40, q_lengths=m, table=table, dtype=F16)
    for x, y in zip((k, v), got):
        want = _stored(x)
        want[0, :, 16:32] = math.nan
        assert _same(y[0], want[0]) and _same(y[1, :, :15], want[1, :, :15])
    assert bool((cache[3] == 0).all())
    q = _tensor((2, 4, 1, D), "heads", F16, 10)
    out = ob.attention_window_e2m1(q, cache, held, table=table)
    assert bool(out[0].isnan().all()) and bool(out[1].isfinite().all())
    out = ob.attention_window_e2m1(q, cache, held, table=table, window=8)  # none of its keys is there
    assert bool(out.isfinite().all())
    q = _tensor((2, 4, 40, D), "heads", F16, 11)  # several rows: only those past the missing page
    out = ob.attention_window_e2m1(q[:, :, -12:], cache, held, table=table, window=8)
    assert bool(out[0, :, :-8].isnan().any()) and bool(out[0, :, -1:].isfinite().all())


# ------------------------------------------------------------------ attention
def _attended(q, k, v, lengths, counts, window, right, sinks, scale):
    """(out, A) in 64 bits over k, v [B, Hkv, capacity, D]; rows without keys are zeros."""
    B, H, T, D = q.shape
    group = H // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mean = torch.zeros_like(out)
    for b in range(B):
        n, m = lengths[b], counts[b]
        if n == 0 or m == 0:
            continue
        p = torch.arange(n - m, n, device=q.device)[:, None]
        s = torch.arange(n, device=q.device)[None]
        seen = s <= p + right
        if window > 0:
            seen &= (s > p - window) | (s < sinks)
        kk, vv = (x[b, :, :n].double().repeat_interleave(group, 0) for x in (k, v))
        e = q[b, :, :m].double() @ kk.transpose(1, 2) * (scale if scale > 0 else D**-0.5)
        w = torch.nan_to_num(torch.softmax(e.masked_fill(~seen, -math.inf), dim=2))
        out[b, :, :m], mean[b, :, :m] = w @ vv, w @ vv.abs()
    return out, mean


def _check(got, q, k, v, lengths, counts, window=0, right=0, sinks=0, scale=0.0, prompt=False):
    want, mean = _attended(q, k, v, lengths, counts, window, right, sinks, scale)
    eps = torch.finfo(q.dtype).eps if prompt else 2.0**-10
    keys = k.shape[2] if window <= 0 else min(k.shape[2], window + right + sinks)
    most = max([float(v[b, :, :n].abs().max()) for b, n in enumerate(lengths) if n] or [0.0])
    tol = mean * (eps + 2.0**-12) + keys * 2.0**-25 * most + 1e-30
    tol = tol + want.abs() * torch.finfo(got.dtype).eps / 2 * (1 + 2.0**-8) + (2.0**-25 if got.dtype == F16 else 0)
    for b in range(q.shape[0]):
        m = counts[b]
        err = (got[b, :, :m].double() - want[b, :, :m]).abs()
        assert bool((err <= tol[b, :, :m]).all()), (
            f"sequence {b}: worst {float((err / tol[b, :, :m]).nan_to_num(1e9).max()):.3f} of the tolerance")
        assert bool((got[b, :, m:] == KEPT).all()), f"sequence {b}: rows past its queries changed"


def _case(ob, B, H, Hkv, T, D, page, lengths, counts, dtype, layout="tokens", seed=20):
    """q, a cache whose tokens past each sequence's are any bytes, its table, and k and v as it stands for."""
    capacity = max(max(lengths), 1)
    cache, table = _made(ob, B, Hkv, D, capacity, page, seed)
    k, v = (_tensor((B, Hkv, capacity, D), "heads", dtype, seed + s, 0.3) for s in (1, 2))
    ob.cache_write_e2m1(k, v, cache, _i32(lengths), q_lengths=_i32(lengths), table=table)
    return _tensor((B, H, T, D), layout, dtype, seed + 3), cache, table, _stored(k), _stored(v)


# B, H, Hkv, T, D, page, lengths, counts, window, right, sinks
TOKENS = [
    (1, 1, 1, 1, 64, 0, [1], [1], 0, 0, 0),
    (1, 2, 1, 1, 8, 16, [17], [1], 5, 0, 2),
    (2, 4, 2, 1, 64, 32, [300, 1], [1, 1], 100, 0, 4),
    (1, 16, 2, 1, 128, 64, [2048], [1], 512, 0, 4),
    (3, 6, 2, 2, 72, 16, [129, 16, 15], [2, 2, 1], 40, 0, 1),
    (2, 8, 1, 2, 96, 48, [500, 33], [2, 2], 64, 0, 130),
    (1, 5, 5, 4, 80, 128, [700], [4], 0, 0, 3),
    (2, 3, 3, 16, 32, 16, [40, 0], [16, 0], 7, 3, 2),
    (1, 32, 1, 1, 16, 256, [1000], [1], 33, 0, 0),
    (1, 1, 1, 60, 24, 16, [61], [60], 10, 100, 5),
    (1, 4, 4, 1, 128, 0, [16000], [1], 0, 0, 0),
    (20, 32, 8, 1, 128, 32, list(range(1, 261, 13)), [1] * 20, 1, 0, 0),
    (2, 8, 2, 7, 64, 16, [7, 3], [7, 7], 0, 0, 0),
    (1, 8, 8, 1, 120, 16, [31], [1], 16, 0, 16),
    (1, 2, 1, 8, 128, 0, [4096], [8], 1000, 5, 40),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", TOKENS)
def test_few_queries(ob, case, dtype):
    B, H, Hkv, T, D, page, lengths, counts, window, right, sinks = case
    q, cache, table, k, v = _case(ob, B, H, Hkv, T, D, page, lengths, counts, dtype)
    for out_dtype in (dtype, F32):
        out = torch.full(q.shape, KEPT, dtype=out_dtype, device="cuda")
        got = ob.attention_window_e2m1(q, cache, _i32(lengths), q_lengths=_i32(counts), table=table, window=window,
                                       right=right, sinks=sinks, out=out)
        assert got is out
        _check(out, q, k, v, lengths, counts, window, right, sinks)
    ob.library().sync_check()


PROMPTS = [
    (1, 1, 1, 65, 64, 0, [65], [65], 0, 0, 0),
    (1, 2, 1, 257, 64, 16, [257], [257], 100, 0, 4),
    (2, 4, 2, 300, 128, 64, [700, 300], [300, 299], 128, 0, 1),
    (1, 3, 3, 1000, 72, 48, [1000], [1000], 129, 0, 130),
    (1, 4, 1, 200, 80, 256, [3000], [200], 500, 0, 300),
    (2, 1, 1, 130, 32, 16, [128, 0], [128, 0], 20, 0, 2),
    (1, 2, 2, 400, 16, 0, [400], [400], 0, 50, 0),
    (1, 8, 2, 128, 8, 32, [128], [128], 1, 0, 0),
    (3, 8, 4, 150, 96, 16, [150, 3, 77], [150, 3, 20], 0, 0, 0),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", PROMPTS)
def test_prompts(ob, case, dtype):
    B, H, Hkv, T, D, page, lengths, counts, window, right, sinks = case
    q, cache, table, k, v = _case(ob, B, H, Hkv, T, D, page, lengths, counts, dtype, "rows")
    for out_dtype in (dtype, F32):
        out = torch.full(q.shape, KEPT, dtype=out_dtype, device="cuda")
        ob.attention_window_e2m1(q, cache, _i32(lengths), q_lengths=_i32(counts), table=table, window=window,
                                 right=right, sinks=sinks, out=out)
        _check(out, q, k, v, lengths, counts, window, right, sinks, prompt=True)
    ob.library().sync_check()


@pytest.mark.parametrize("scale", [0.01, 1.0])
@pytest.mark.parametrize("power", [-60, -20, 0, 30])
def test_queries_of_any_size(ob, scale, power):
    """bf16 queries far outside f16's range: what matters is scale * q."""
    B, H, Hkv, T, D, page, lengths = 1, 4, 2, 1, 64, 16, [150]
    q, cache, table, k, v = _case(ob, B, H, Hkv, T, D, page, lengths, [1], BF16)
    q = (q.float() * 2.0**power).to(BF16)
    q[0, 0, 0, 5] = 2.0 ** (power + 3)  # one element above the others
    got = torch.full(q.shape, KEPT, dtype=F32, device="cuda")
    ob.attention_window_e2m1(q, cache, _i32(lengths), table=table, scale=scale * 2.0**-power, out=got)
    _check(got, q, k, v, lengths, [1], scale=scale * 2.0**-power)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_queries_of_zeros_and_masks_past_everything(ob, dtype):
    """Equal scores give means of the values; windows and first tokens beyond the sequence."""
    B, H, Hkv, T, D, page, lengths = 2, 6, 2, 2, 72, 32, [90, 33]
    q, cache, table, k, v = _case(ob, B, H, Hkv, T, D, page, lengths, [T] * B, dtype)
    q = q.contiguous()
    q[0, 1] = 0
    for window, right, sinks, scale in ((0, 0, 0, 0.0), (1 << 30, 1 << 30, 1 << 30, 0.0), (5, 0, 1 << 30, 1e-30), (91, 2, 90, 3.0)):
        out = torch.full(q.shape, KEPT, dtype=F32, device="cuda")
        ob.attention_window_e2m1(q, cache, _i32(lengths), table=table, window=window, right=right, sinks=sinks,
                                 scale=scale, out=out)
        _check(out, q, k, v, lengths, [T] * B, min(window, 1000), min(right, 1000), min(sinks, 1000), scale)


def test_queries_that_are_not_finite(ob):
    for T, case in ((1, TOKENS[2]), (2, TOKENS[4])):
        B, H, Hkv, _, D, page, lengths, counts, window, right, sinks = case
        for bad in (math.inf, -math.inf, math.nan):
            q, cache, table, k, v = _case(ob, B, H, Hkv, T, D, page, lengths, counts, BF16)
            q = q.contiguous()
            q[0, 1, 0, 3] = bad
            got = ob.attention_window_e2m1(q, cache, _i32(lengths), q_lengths=_i32([T] * B), table=table)
            assert bool(got[0, 1, 0].isnan().all())
            assert bool(got[0, 0].isfinite().all()) and bool(got[1:].isfinite().all())


def test_keys_that_are_not_finite(ob):
    """NaN in the cache reaches the queries that see it, and no other sequence or head."""
    B, H, Hkv, T, D, page, lengths = 2, 4, 2, 1, 64, 16, [100, 60]
    q, cache, table, _, _ = _case(ob, B, H, Hkv, T, D, page, lengths, [1, 1], BF16)
    k, v = (_tensor((B, Hkv, 100, D), "heads", BF16, s) for s in (31, 32))
    k[0, 1, 50, 7], v[1, 0, 10, 3] = math.nan, math.inf
    ob.cache_write_e2m1(k, v, cache, _i32(lengths), q_lengths=_i32(lengths), table=table)
    got = ob.attention_window_e2m1(q, cache, _i32(lengths), table=table)
    assert bool(got[0, 2:].isnan().all()) and bool(got[0, :2].isfinite().all())
    assert bool(got[1, :2, :, :32].isnan().all()) and bool(got[1, :2, :, 32:].isfinite().all())
    assert bool(got[1, 2:].isfinite().all())
    got = ob.attention_window_e2m1(q, cache, _i32(lengths), table=table, window=49)
    assert bool(got.isfinite().all())  # hidden from all queries


def test_offsets_past_32_bits(ob):
    """A cache of more than 4 GB: its last pages, and strides that leave gaps."""
    D, Hkv, page = 128, 8, 256
    size = ob.library().lib.omni_b200_cache_e2m1_bytes(page, D)
    pages = 2**32 // (size * Hkv) + 8
    if torch.cuda.mem_get_info()[0] < 8e9:
        pytest.skip("not enough memory")
    cache = ob.empty_cache_e2m1(pages, Hkv, page, D)
    table = _i32([[pages - 1, 3], [0, pages - 2]])
    lengths = [400, 300]
    k, v = (_tensor((2, Hkv, 400, D), "heads", BF16, s) for s in (41, 42))
    ob.cache_write_e2m1(k, v, cache, _i32(lengths), q_lengths=_i32(lengths), table=table)
    got = ob.cache_read_e2m1(cache, D, _i32(lengths), rows=400, q_lengths=_i32(lengths), table=table)
    for x, y in zip((k, v), got):
        want = _stored(x)
        for b, n in enumerate(lengths):
            assert _same(y[b, :, :n], want[b, :, :n])
    q = _tensor((2, 16, 1, D), "heads", BF16, 43)
    out = torch.full(q.shape, KEPT, dtype=F32, device="cuda")
    ob.attention_window_e2m1(q, cache, _i32(lengths), table=table, out=out)
    _check(out, q, _stored(k), _stored(v), lengths, [1, 1])
    # A layer's part of one buffer for all layers: pages and heads with gaps between them.
    wide = torch.zeros(5, 3, 2, 2 * size, dtype=torch.uint8, device="cuda")
    part = wide[:, 1, :, :size]
    table = _i32([[4, 2], [0, 1]])
    ob.cache_write_e2m1(k[:, :2], v[:, :2], part, _i32(lengths), q_lengths=_i32(lengths), table=table)
    out = torch.full((2, 4, 1, D), KEPT, dtype=F32, device="cuda")
    ob.attention_window_e2m1(q[:, :4], part, _i32(lengths), table=table, out=out)
    _check(out, q[:, :4], _stored(k[:, :2]), _stored(v[:, :2]), lengths, [1, 1])
    assert bool((wide[:, 0] == 0).all()) and bool((wide[:, 2] == 0).all()) and bool((wide[..., size:] == 0).all())


# ----------------------------------------------------------- as they are used
def _layer_step(ob, x, wq, wk, wv, cache, table, where, frequencies, axes, lengths, H, Hkv, D, kv_len):
    """One attention layer: projections, positions, the cache, attention."""
    B, T, _ = x.shape
    q = (x @ wq).view(B, T, H, D).transpose(1, 2)
    k = (x @ wk).view(B, T, Hkv, D).transpose(1, 2)
    v = (x @ wv).view(B, T, Hkv, D).transpose(1, 2)
    ob.rotary(q, k, where, frequencies, axes=axes, q_out=q, k_out=k)
    ob.cache_write_e2m1(k, v, cache, lengths, table=table)
    out = torch.empty(B, T, H, D, dtype=x.dtype, device=x.device)
    ob.attention_window_e2m1(q, cache, lengths, table=table, kv_len=kv_len, out=out.transpose(1, 2))
    return q, k, v, out


@pytest.mark.parametrize("captured", [False, True])
def test_prompt_then_tokens(ob, captured):
    """A prompt and then tokens one by one (captured: replays of one graph), against attention
    in 64 bits over what the cache should stand for."""
    torch.manual_seed(0)
    B, H, Hkv, D, page, prompt, new = 2, 8, 2, 64, 16, 130, 21
    wq, wk, wv = (torch.randn(256, h * D, device="cuda").to(BF16) / 16 for h in (H, Hkv, Hkv))
    table, pages = _table(B, -(-(prompt + new) // page), 1, 50)
    cache = ob.empty_cache_e2m1(pages, Hkv, page, D)
    frequencies = (10000.0 ** (-torch.arange(32).double() / 32)).float().cuda()
    axes = ob.rotary_axes([8, 12, 12])
    x = torch.randn(B, prompt + new, 256, device="cuda").to(BF16)
    where = torch.randint(0, 200, (3, B, prompt + new), device="cuda")
    lengths = torch.full((B,), prompt, dtype=torch.int32, device="cuda")
    args = (cache, table)
    q, k, v, out = _layer_step(ob, x[:, :prompt], wq, wk, wv, *args, where[:, :, :prompt], frequencies, axes, lengths,
                               H, Hkv, D, prompt + new)
    keys, values = _stored(k), _stored(v)
    got = out.transpose(1, 2)
    _check(got, q, keys, values, [prompt] * B, [prompt] * B, prompt=True)
    step_x, step_where = x[:, :1].clone(), where[:, :, :1].clone()
    graph = torch.cuda.CUDAGraph()
    if captured:
        lengths.fill_(1)  # what capturing would write, were it to run: it does not
        with torch.cuda.graph(graph):
            held = _layer_step(ob, step_x, wq, wk, wv, *args, step_where, frequencies, axes, lengths, H, Hkv, D,
                               prompt + new)
    for i in range(prompt, prompt + new):
        step_x.copy_(x[:, i:i + 1])
        step_where.copy_(where[:, :, i:i + 1])
        lengths.fill_(i + 1)
        if captured:
            graph.replay()
            q, k, v, out = held
        else:
            q, k, v, out = _layer_step(ob, step_x, wq, wk, wv, *args, step_where, frequencies, axes, lengths, H, Hkv,
                                       D, prompt + new)
        keys, values = torch.cat([keys, _stored(k)], 2), torch.cat([values, _stored(v)], 2)
        _check(out.transpose(1, 2), q, keys, values, [i + 1] * B, [1] * B)
    ob.library().sync_check()


def test_same_bits_each_time_and_on_another_stream(ob):
    for case in (TOKENS[3], TOKENS[11], PROMPTS[2]):
        B, H, Hkv, T, D, page, lengths, counts, window, right, sinks = case
        q, cache, table, _, _ = _case(ob, B, H, Hkv, T, D, page, lengths, counts, BF16)
        held, m = _i32(lengths), _i32(counts)

        def call(**kw):
            out = torch.full(q.shape, KEPT, dtype=BF16, device="cuda")
            return ob.attention_window_e2m1(q, cache, held, q_lengths=m, table=table, window=window, sinks=sinks, out=out, **kw)

        want = call()
        streams = [torch.cuda.Stream() for _ in range(3)]
        torch.cuda.synchronize()
        got = [call(stream=s) for s in streams for _ in range(4)]
        torch.cuda.synchronize()
        for y in got:
            assert torch.equal(y, want)


def test_nothing_to_do(ob):
    cache = ob.empty_cache_e2m1(2, 2, 16, 64)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    k = torch.empty(0, 2, 3, 64, dtype=BF16, device="cuda")
    ob.cache_write_e2m1(k, k, cache, none)
    k = torch.empty(2, 2, 0, 64, dtype=BF16, device="cuda")
    ob.cache_write_e2m1(k, k, cache, _i32([5, 5]))
    q = torch.empty(2, 4, 0, 64, dtype=BF16, device="cuda")
    assert ob.attention_window_e2m1(q, cache, _i32([5, 5])).shape == q.shape
    q = torch.randn(2, 4, 3, 64, device="cuda").to(BF16)
    out = ob.attention_window_e2m1(q, cache, _i32([0, 0]))
    assert bool((out == 0).all())
    assert bool((cache == 0).all())
