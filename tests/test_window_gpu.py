"""attention_window on the GPU against softmax attention in 64 bits.

Tolerance, from arithmetic.  With A = the softmax-weighted mean of |v|, for each
output element:
  * the weights are rounded to the operand type for the product with v and their
    sum may be taken before or after that: 2 * eps / 2 * A;
  * scores are fp32 sums of exact products: at most D * 2^-24 of the sum of
    magnitudes, below 2^-12 in the exponent for these inputs, so 2^-12 * A with
    the exponential's own 2^-22;
  * fp16 weights below 2^-14 of the row's largest lose at most 2^-25 each, times
    the largest |v|;
  * the output's rounding, half a step.
Keys and values past a sequence's length are NaN in every test, rows past its
queries must stay as they were.
"""

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
KEPT = 123.0


@pytest.fixture(scope="module")
def ob():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from tests.conftest import load_package

    return load_package()


def _tensor(shape, layout, dtype, gen):
    b, h, n, d = shape
    if layout == "heads":
        return torch.randn(b, h, n, d, generator=gen).to(dtype).cuda()
    if layout == "tokens":
        return torch.randn(b, n, h, d, generator=gen).to(dtype).cuda().transpose(1, 2)
    # rows of a wider matrix, as a joint projection leaves them
    wide = torch.full((b, n, h * d + 40), KEPT, dtype=dtype)
    wide[..., 16:16 + h * d] = torch.randn(b, n, h * d, generator=gen).to(dtype)
    return wide.cuda()[..., 16:16 + h * d].unflatten(2, (h, d)).transpose(1, 2)


def _inputs(B, H, Hkv, Lq, Lk, D, dtype, layout, seed):
    g = torch.Generator().manual_seed(seed)
    return [_tensor((B, h, n, D), layout, dtype, g) for h, n in ((H, Lq), (Hkv, Lk), (Hkv, Lk))]


def _reference(q, k, v, window, right, sinks, lengths, q_lengths, scale=0.0):
    """(out, A, most |v|, seen) in 64 bits; rows without keys are zeros."""
    B, H, Lq, D = q.shape
    Hkv, Lk = k.shape[1:3]
    group = H // Hkv
    out = torch.zeros(B, H, Lq, D, dtype=torch.float64, device=q.device)
    mean = torch.zeros_like(out)
    for b in range(B):
        n, m = (Lk if lengths is None else lengths[b]), (Lq if q_lengths is None else q_lengths[b])
        if n == 0 or m == 0:
            continue
        p = torch.arange(n - m, n, device=q.device)[:, None]
        s = torch.arange(n, device=q.device)[None]
        seen = s <= p + right
        if window > 0:
            seen &= (s > p - window) | (s < sinks)
        kk = k[b, :, :n].double().repeat_interleave(group, 0)
        vv = v[b, :, :n].double().repeat_interleave(group, 0)
        e = q[b, :, :m].double() @ kk.transpose(1, 2) * (scale if scale > 0 else D**-0.5)
        w = torch.nan_to_num(torch.softmax(e.masked_fill(~seen, -math.inf), dim=2))
        out[b, :, :m], mean[b, :, :m] = w @ vv, w @ vv.abs()
    return out, mean


def _check(got, q, k, v, window, right, sinks, lengths, q_lengths, scale=0.0):
    want, mean = _reference(q, k, v, window, right, sinks, lengths, q_lengths, scale)
    eps = torch.finfo(q.dtype).eps
    tol = mean * (eps + 2.0**-12) + want.abs() * torch.finfo(got.dtype).eps / 2 * (1 + 2.0**-8) + 1e-30
    if q.dtype == F16:
        keys = k.shape[2] if window <= 0 else min(k.shape[2], window + right + sinks)
        most = max(float(v[b, :, :n].abs().max()) if n else 0.0
                   for b, n in enumerate(lengths or [k.shape[2]] * q.shape[0]))
        tol = tol + keys * 2.0**-25 * most
        if got.dtype == F16:
            tol = tol + 2.0**-25
    for b in range(q.shape[0]):
        m = q.shape[2] if q_lengths is None else q_lengths[b]
        err = (got[b, :, :m].double() - want[b, :, :m]).abs()
        assert bool((err <= tol[b, :, :m]).all()), (
            f"sequence {b}: worst {float((err / tol[b, :, :m]).nan_to_num(1e9).max()):.3f} of the tolerance")
        if q_lengths is not None:
            assert bool((got[b, :, m:] == KEPT).all()), f"sequence {b}: rows past its queries changed"


def _run(ob, q, k, v, lengths=None, q_lengths=None, out_dtype=None, out=None, **kw):
    k, v = k.clone(), v.clone()
    if lengths is not None:
        for b, n in enumerate(lengths):
            k[b, :, n:] = float("nan")
            v[b, :, n:] = float("nan")
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if out is None:
        out = torch.full(q.shape, KEPT, dtype=out_dtype or q.dtype, device="cuda")
    got = ob.attention_window(q, k, v, lengths=i32(lengths), q_lengths=i32(q_lengths), out=out, **kw)
    ob.library().sync_check()
    assert got is out
    return got


# B, H, Hkv, Lq, Lk, D, window, right, sinks
TOKENS = [
    (1, 1, 1, 1, 1, 64, 0, 0, 0),
    (1, 2, 1, 1, 17, 8, 5, 0, 2),
    (2, 4, 2, 1, 300, 64, 100, 0, 4),
    (1, 16, 2, 1, 2048, 128, 512, 0, 4),
    (3, 6, 2, 2, 129, 72, 40, 0, 1),
    (2, 8, 1, 7, 500, 96, 64, 0, 130),
    (1, 5, 5, 4, 700, 80, 0, 0, 3),
    (2, 3, 3, 16, 40, 32, 7, 3, 2),
    (1, 64, 1, 1, 1000, 16, 33, 0, 0),
    (1, 1, 1, 60, 61, 24, 10, 100, 5),
    (1, 4, 4, 1, 16000, 128, 0, 0, 0),
    (20, 32, 8, 1, 260, 128, 1, 0, 0),
]
PROMPTS = [
    (1, 1, 1, 65, 65, 64, 0, 0, 0),
    (1, 2, 1, 257, 257, 64, 100, 0, 4),
    (2, 4, 2, 300, 700, 128, 128, 0, 1),
    (1, 3, 3, 1000, 1000, 72, 129, 0, 130),
    (1, 2, 2, 515, 515, 96, 60, 59, 5),
    (1, 4, 1, 200, 3000, 80, 500, 0, 300),
    (2, 1, 1, 130, 128, 32, 20, 0, 2),
    (1, 2, 2, 400, 400, 16, 0, 50, 0),
    (1, 8, 2, 128, 128, 8, 1, 0, 0),
    (1, 2, 2, 300, 1500, 40, 64, 2000, 7),
    (1, 2, 1, 1200, 1200, 128, 0, 0, 0),
    (3, 40, 8, 600, 600, 64, 300, 10, 64),
]
# Work enough for the kernel of 128-row blocks whatever its rule weighs.
WIDE = [
    (16, 8, 8, 128, 130, 64, 40, 0, 3),
    (8, 32, 4, 129, 129, 128, 0, 0, 0),
    (24, 8, 8, 257, 300, 72, 60, 59, 5),
    (40, 8, 8, 130, 128, 32, 20, 0, 2),
    (16, 24, 8, 200, 400, 80, 100, 0, 130),
    (12, 16, 16, 300, 700, 96, 128, 0, 1),
    (60, 20, 10, 256, 256, 8, 1, 0, 0),
    (60, 16, 2, 250, 250, 16, 0, 50, 0),
    (9, 24, 24, 390, 1500, 40, 64, 2000, 7),
    (64, 8, 8, 100, 100, 24, 7, 300, 0),
    (2, 64, 64, 1000, 1000, 128, 129, 0, 300),
    (700, 2, 2, 65, 70, 64, 16, 0, 1),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("layout", ["heads", "tokens", "rows"])
@pytest.mark.parametrize("case", TOKENS + PROMPTS + WIDE, ids=lambda c: "-".join(map(str, c)))
def test_window(ob, case, layout, dtype):
    B, H, Hkv, Lq, Lk, D, window, right, sinks = case
    q, k, v = _inputs(B, H, Hkv, Lq, Lk, D, dtype, layout, seed=sum(case))
    mask = dict(window=window, right=right, sinks=sinks)
    for out_dtype in (dtype, F32):
        got = _run(ob, q, k, v, out_dtype=out_dtype, **mask)
        _check(got, q, k, v, window, right, sinks, None, None)
    assert torch.equal(got, _run(ob, q, k, v, out_dtype=F32, **mask))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", [
    (6, 4, 2, 1, 300, 64, 100, 0, 4), (6, 6, 2, 5, 200, 72, 30, 4, 70), (6, 2, 1, 16, 90, 128, 0, 0, 0),
    (6, 2, 2, 300, 300, 64, 50, 0, 4), (6, 4, 1, 280, 900, 128, 200, 20, 150), (6, 2, 2, 520, 640, 96, 0, 0, 0),
    (6, 3, 3, 333, 400, 32, 17, 5, 3), (6, 40, 8, 640, 640, 96, 0, 0, 0), (6, 40, 20, 300, 900, 128, 200, 20, 150),
    (6, 48, 48, 520, 640, 72, 17, 5, 3), (6, 64, 64, 333, 400, 32, 0, 0, 0), (600, 4, 4, 130, 140, 64, 30, 0, 2),
], ids=lambda c: "-".join(map(str, c)))
def test_window_lengths(ob, case, dtype):
    """Sequences of several lengths: empty, one key, queries that outnumber the keys
    (rows with no key give zeros), lengths inside and at the ends of tiles."""
    B, H, Hkv, Lq, Lk, D, window, right, sinks = case
    q, k, v = _inputs(B, H, Hkv, Lq, Lk, D, dtype, "heads", seed=sum(case) + 1)
    lengths = [Lk, 0, 1, min(Lk, 129), Lk - 1, min(Lk, 128)] * (B // 6)
    mask = dict(window=window, right=right, sinks=sinks)
    for q_lengths in (None, [Lq, Lq, Lq, max(1, Lq // 2), 0, min(Lq, 128)] * (B // 6)):
        for out_dtype in (dtype, F32):
            got = _run(ob, q, k, v, lengths, q_lengths, out_dtype=out_dtype, **mask)
            _check(got, q, k, v, window, right, sinks, lengths, q_lengths)
    # Lengths beyond the tensors count as their sizes, negative ones as none.
    far = _run(ob, q, k, v, [Lk] * (B - 1) + [0], [Lq] * B, **mask)
    i32 = dict(dtype=torch.int32, device="cuda")
    clamped = ob.attention_window(q, k, v, lengths=torch.tensor([Lk + 99] * (B - 1) + [-3], **i32),
                                  q_lengths=torch.tensor([2**31 - 1] * B, **i32), **mask)
    ob.library().sync_check()
    assert torch.equal(far, clamped)


@pytest.mark.parametrize("B,H,Lq", [(1, 2, 1), (1, 2, 300), (8, 32, 300)])
def test_window_scale_and_large_scores(ob, B, H, Lq):
    """Scores of a few hundred: the maximum is subtracted before the exponential."""
    q, k, v = _inputs(B, H, H, Lq, 600, 64, BF16, "heads", seed=3)
    for scale in (0.01, 2.0):
        got = _run(ob, q, k, v, window=100, sinks=3, scale=scale, out_dtype=F32)
        want, mean = _reference(q, k, v, 100, 0, 3, None, None, scale)
        # Score errors grow with the scores: fp32 sums of 64 products of up to 16,
        # times the scale, against 2^-24: below 64 * 2^-24 * 1024 * scale.
        tol = mean * (2 * 2.0**-8 + 2.0**-8 * scale) + want.abs() * 2.0**-20
        assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("B,H,Lq", [(2, 4, 1), (2, 4, 200), (20, 16, 200)])
def test_window_writes_its_rows_only(ob, B, H, Lq):
    """An output inside a larger tensor: what lies around it stays."""
    q, k, v = _inputs(B, H, 2, Lq, 256, 64, BF16, "tokens", seed=5)
    want = _run(ob, q, k, v, window=60, sinks=2)
    wide = torch.full((B, Lq + 2, H, 80), KEPT, dtype=BF16, device="cuda")
    inner = wide[:, 1:Lq + 1, :, 8:72].transpose(1, 2)
    _run(ob, q, k, v, window=60, sinks=2, out=inner)
    assert torch.equal(inner, want)
    odd = torch.full((B, Lq, H, 65), KEPT, dtype=BF16, device="cuda")  # rows that no 16-byte store reaches
    _run(ob, q, k, v, window=60, sinks=2, out=odd[..., 1:].transpose(1, 2))
    assert torch.equal(odd[..., 1:].transpose(1, 2), want) and bool((odd[..., 0] == KEPT).all())
    inner.fill_(KEPT)
    assert bool((wide == KEPT).all())


@pytest.mark.parametrize("H,Lq", [(4, 2), (4, 300), (64, 300)])
def test_window_captured_on_two_streams(ob, H, Lq):
    """Two captured calls with inputs of their own, replayed together and again with
    other lengths, give what plain calls give."""
    graphs = []
    for seed in (1, 2):
        q, k, v = _inputs(3, H, 2, Lq, 700, 64, BF16, "heads", seed=seed)
        lengths = torch.tensor([700, 350, 301], dtype=torch.int32, device="cuda")
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            ob.attention_window(q, k, v, window=128, sinks=4, lengths=lengths, out=out)
        graphs.append((graph, stream, q, k, v, lengths, out))
    for turn in range(2):
        for graph, stream, *_, lengths, out in graphs:
            lengths.copy_(torch.tensor([699 - 90 * turn, 500, 320], dtype=torch.int32))
        torch.cuda.synchronize()
        for graph, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for graph, stream, q, k, v, lengths, out in graphs:
            assert torch.equal(out, ob.attention_window(q, k, v, window=128, sinks=4, lengths=lengths))
    ob.library().sync_check()


def test_window_of_everything_is_plain_attention(ob):
    """No window and full lookahead is what attention_bhld computes."""
    q, k, v = _inputs(2, 3, 3, 500, 500, 64, BF16, "heads", seed=9)
    plain = ob.attention_bhld(q, k, v, out_dtype=F32)
    got = ob.attention_window(q, k, v, right=500, out_dtype=F32)
    ob.library().sync_check()
    assert torch.allclose(got, plain, rtol=0, atol=2.0**-8 * float(v.abs().max()))


def test_window_empty_calls(ob):
    q, k, v = _inputs(2, 2, 1, 4, 8, 64, BF16, "heads", seed=1)
    assert ob.attention_window(q[:0], k[:0], v[:0]).shape == (0, 2, 4, 64)
    assert ob.attention_window(q[:, :, :0], k, v).shape == (2, 2, 0, 64)
    ob.library().sync_check()


def test_layer_of_all_operators(ob):
    """The operators together as a layer uses them: norm with the residual, product,
    windowed attention over the joint projection's rows, quantisation, product.  Each
    step is checked against its definition in 64 bits on the inputs it got."""
    B, n, H, Hkv, D = 3, 400, 16, 4, 64
    d, rows = H * D, 3 * 400
    g = torch.Generator().manual_seed(11)
    x, res = (torch.randn(rows, d, generator=g).to(BF16).cuda() for _ in range(2))
    norm = (1 + 0.1 * torch.randn(d, generator=g)).to(BF16).cuda()
    w_in, s_in = ob.quantize_e4m3(torch.randn((H + 2 * Hkv) * D, d, generator=g).cuda() * d**-0.5, block_rows=128)
    w_out, s_out = ob.quantize_e4m3(torch.randn(d, d, generator=g).cuda() * d**-0.5, block_rows=128)
    bias = torch.randn(d, generator=g).to(BF16).cuda()
    lengths = [400, 133, 0]
    held = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    q, scales, h = ob.rms_norm_e4m3(x, norm, residual=res)
    joint = ob.linear_e4m3(q, scales, w_in, s_in).view(B, n, H + 2 * Hkv, D).transpose(1, 2)
    parts = joint[:, :H], joint[:, H:H + Hkv], joint[:, H + Hkv:]
    mixed = torch.zeros(B, n, H, D, dtype=BF16, device="cuda")
    ob.attention_window(*parts, window=64, sinks=4, lengths=held, q_lengths=held, out=mixed.transpose(1, 2))
    a, a_scales = ob.quantize_e4m3(mixed.view(rows, d))
    y = ob.linear_e4m3(a, a_scales, w_out, s_out, bias=bias)
    ob.library().sync_check()

    def wide(t, s, block):
        return t.double() * s.double().repeat_interleave(block, 0)[:t.shape[0]].repeat_interleave(128, 1)[:, :t.shape[1]]

    h64 = x.double() + res.double()
    y64 = h64 / torch.sqrt(h64.square().mean(1, keepdim=True) + 1e-6) * norm.double()
    # e4m3: half a step of 2^-4, at least 2^-10 of the group's scale.
    s = scales.double().repeat_interleave(128, 1)
    assert bool(((wide(q, scales, 1) - y64).abs() <= torch.maximum(y64.abs() * 2.0**-4, s * 2.0**-10) * 1.001).all())
    assert bool(((h.double() - h64).abs() <= h64.abs() * 2.0**-8).all())

    def product(t, ts, w, ws):
        a64, w64 = wide(t, ts, 1), wide(w, ws, 128)
        return a64 @ w64.t(), a64.abs() @ w64.abs().t()

    want, mag = product(q, scales, w_in, s_in)
    got = joint.transpose(1, 2).reshape(rows, -1).double()
    assert bool(((got - want).abs() <= mag * 2.0**-11 + want.abs() * 2.0**-8).all())
    ref, mean = _reference(*parts, 64, 0, 4, lengths, lengths)
    err = (mixed.transpose(1, 2).double() - ref).abs()
    assert bool((err <= mean * (2.0**-7 + 2.0**-12) + ref.abs() * 2.0**-8 + 1e-30).all())
    want, mag = product(a, a_scales, w_out, s_out)
    want = want + bias.double()
    assert bool(((y.double() - want).abs() <= mag * 2.0**-11 + want.abs() * 2.0**-8 * 1.01).all())
    assert bool((y.view(B, n, d)[2] == bias).all())  # a sequence without keys mixes to zeros


def test_different_operators_at_once(ob):
    """Kernels that share SMs, shared memory and tensor memory, on four streams: each
    call's bits are those of the call alone."""
    q, k, v = _inputs(2, 8, 2, 300, 900, 128, BF16, "heads", seed=1)
    q1, k1, v1 = _inputs(4, 8, 8, 1, 2000, 64, BF16, "tokens", seed=2)
    e, _, _ = _inputs(2, 4, 4, 500, 500, 72, BF16, "heads", seed=3)
    x = torch.randn(700, 1152, generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    w, sw = ob.quantize_e4m3(x[:640], block_rows=128)
    a, sa = ob.quantize_e4m3(x)
    calls = [
        lambda s: ob.attention_window(q, k, v, window=200, sinks=4, stream=s),
        lambda s: ob.linear_e4m3(a[:5].contiguous(), sa[:5], w, sw, stream=s),
        lambda s: ob.attention_window(q1, k1, v1, window=700, stream=s),
        lambda s: ob.attention_bhld(e, e, e, stream=s),
        lambda s: ob.linear_e4m3(a, sa, w, sw, stream=s),
        lambda s: ob.rms_norm(x, x[0].contiguous(), stream=s)[0],
        lambda s: ob.quantize_e4m3(x, stream=s)[0].view(torch.uint8),
    ]
    want = [c(None) for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(4)], []
    for turn in range(12):
        for i, c in enumerate(calls):
            s = streams[(i + turn) % 4]
            with torch.cuda.stream(s):  # its own memory pool, and small copies in order
                got.append((i, c(s)))
    torch.cuda.synchronize()
    for i, g in got:
        assert torch.equal(g, want[i]), f"call {i}"
    ob.library().sync_check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", [
    (1, 4, 2, 1, 300, 64, 100, 0, 4), (3, 16, 2, 2, 2048, 128, 512, 0, 4), (2, 3, 3, 16, 10, 32, 7, 3, 2),
    (1, 1, 1, 60, 40, 24, 10, 2, 5), (2, 4, 2, 300, 700, 128, 128, 0, 1), (24, 8, 8, 257, 250, 72, 60, 59, 5),
    (16, 24, 8, 200, 150, 80, 0, 0, 0), (64, 8, 8, 100, 100, 24, 7, 300, 0),
], ids=lambda c: "-".join(map(str, c)))
def test_window_queries_that_are_not_finite(ob, case, dtype):
    """A query whose scores hold a NaN or an infinity gives what the softmax gives, NaN, not
    numbers; one that sees no key gives zeros all the same; other rows do not change."""
    B, H, Hkv, Lq, Lk, D, window, right, sinks = case
    q, k, v = _inputs(B, H, Hkv, Lq, Lk, D, dtype, "heads", seed=sum(case) + 2)
    k[..., 1] = k[..., 1].abs() + 0.5  # with a query's -inf there every score is -inf
    mask = dict(window=window, right=right, sinks=sinks)
    plain = _run(ob, q, k, v, out_dtype=F32, **mask)
    sees = torch.arange(Lq, device="cuda") + Lk - Lq + right >= 0  # any key at all
    for value, column in ((float("nan"), 5), (float("inf"), 1), (-float("inf"), 1)):
        for head, rows in ((0, slice(0, None, 3)), (H - 1, slice(1, None, 2)), (0, slice(Lq - 1, Lq))):
            bad = q.clone()
            bad[:, head, rows, column] = value
            got = _run(ob, bad, k, v, out_dtype=F32, **mask)
            spoilt = torch.zeros(B, H, Lq, dtype=torch.bool, device="cuda")
            spoilt[:, head, rows] = True
            assert bool(torch.isnan(got[spoilt & sees]).all()), f"query {value}: numbers in its row"
            assert torch.equal(got[~(spoilt & sees)], plain[~(spoilt & sees)])
            assert bool((got[..., ~sees, :] == 0).all())


def _kernels(ob, cases, tmp_path):
    """The kernels that the cases run: {name: template instances}, and "clusters": sizes."""
    import re

    from tests.launches import launched

    found = {}
    for B, H, Hkv, Lq, Lk, D, window, right, sinks in cases:
        q, k, v = _inputs(B, H, Hkv, Lq, Lk, D, BF16, "heads", seed=1)
        (name, grid, _), = launched(lambda: ob.attention_window(q, k, v, window=window, right=right, sinks=sinks), tmp_path)
        kind, instance = re.search(r"(window_[a-z]+_kernel)ILi(\d)E", name).groups()
        found.setdefault(kind, set()).add(int(instance))
        if kind == "window_tokens_kernel":
            found.setdefault("clusters", set()).add(grid[0] // (B * Hkv))
    return found


def test_window_cases_reach_both_kernels(ob, tmp_path):
    """The lists above are meant for one kernel each, in every template instance of it: a
    change of the rule that chooses would show here."""
    tokens = _kernels(ob, TOKENS, tmp_path)
    assert tokens == {"window_tokens_kernel": {1, 2, 3, 4}, "clusters": {1, 4, 16}}
    assert _kernels(ob, WIDE, tmp_path) == {"window_prompt_kernel": {1, 2}}
    assert set(_kernels(ob, PROMPTS, tmp_path)) == {"window_prompt_kernel", "window_tokens_kernel", "clusters"}


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("clusters,case", [
    (2, (2, 4, 2, 1, 300, 64, 0, 0, 4)), (2, (3, 6, 3, 5, 450, 128, 0, 3, 0)), (4, (3, 4, 2, 1, 1000, 72, 0, 0, 0)),
    (8, (3, 8, 2, 1, 1800, 32, 1200, 5, 70)), (8, (2, 4, 1, 2, 1500, 96, 0, 0, 0)), (16, (2, 4, 2, 1, 2500, 128, 0, 0, 0)),
], ids=lambda c: str(c) if isinstance(c, int) else "-".join(map(str, c)))
def test_window_of_every_cluster_size(ob, tmp_path, clusters, case, dtype):
    """Keys split over CTAs, with sequences so short that some of them get none."""
    B, H, Hkv, Lq, Lk, D, window, right, sinks = case
    assert _kernels(ob, [case], tmp_path)["clusters"] == {clusters}
    q, k, v = _inputs(B, H, Hkv, Lq, Lk, D, dtype, "tokens", seed=sum(case) + 3)
    mask = dict(window=window, right=right, sinks=sinks)
    for lengths in (None, [Lk, 17, 0][:B], [Lk - 1, Lk // 2, 65][:B]):
        for out_dtype in (dtype, F32):
            got = _run(ob, q, k, v, lengths, out_dtype=out_dtype, **mask)
            _check(got, q, k, v, window, right, sinks, lengths, None)


@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,D,kernel", [(1, 4, 2, 1, 260, 64, "tokens"), (1, 8, 1, 3, 300, 128, "tokens"),
                                                    (2, 64, 64, 140, 150, 64, "prompt"), (2, 64, 64, 129, 130, 128, "prompt")])
def test_window_offsets_past_32_bits(ob, tmp_path, B, H, Hkv, Lq, Lk, D, kernel):
    """Tokens so far apart that the last ones lie more than 2^32 elements into their tensors."""
    from tests.launches import launched

    q, k, v = _inputs(B, H, Hkv, Lq, Lk, D, BF16, "heads", seed=4)
    lengths = [Lk, Lk - 2][:B]
    mask = dict(window=100, sinks=3)
    want = _run(ob, q, k, v, lengths, **mask)

    def apart(t, heads, n):
        """[B, heads, n, D] with more than 2^32 elements between its first and last token."""
        stride = -(-(2**32 + 2**20) // (n - 1) // 8) * 8 if n > 1 else heads * B * D
        room = torch.empty((n - 1) * stride + heads * B * D, dtype=BF16, device="cuda")
        wide = room.as_strided((B, heads, n, D), (heads * D, D, stride, 1))
        wide.copy_(t)
        return wide

    out = apart(torch.full_like(q, KEPT), H, Lq)
    ins = apart(q, H, Lq), apart(k, Hkv, Lk), apart(v, Hkv, Lk)
    held = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    (name, _, _), = launched(lambda: ob.attention_window(*ins, lengths=held, out=out, **mask), tmp_path)
    assert f"window_{kernel}_kernel" in name
    out.fill_(KEPT)
    ob.attention_window(*ins, lengths=held, out=out, **mask)
    ob.library().sync_check()
    assert torch.equal(out, want)
