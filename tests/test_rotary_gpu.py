"""rotary on the GPU against its formula in 64 bits.

Tolerance, from arithmetic, for y0 = x0 cos - x1 sin (y1 alike), relative to |x0| + |x1|:
  * the turn's fraction is rounded to fp32 as a number of half turns below 1: pi * 2^-24;
  * sincospif is within 2 units in the last place: 2^-23;
  * two products and their difference: 2 * 2^-24;
  together below 2^-21.  The fp64 angle passes three roundings (and one in the reference):
  |angle| * 2^-51.  Then the output's rounding, half a step (f16: at least 2^-25).
"""

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
KEPT = 7.0


@pytest.fixture(scope="module")
def ob():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from tests.conftest import load_package

    return load_package()


def _tensor(shape, layout, dtype, seed):
    b, h, t, d = shape
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, t, h, d, generator=g).to(dtype)
    if layout == "tokens":
        return x.cuda().transpose(1, 2)
    if layout == "heads":
        return x.cuda().transpose(1, 2).contiguous()
    # columns of a wider row, as a joint projection leaves them, at an odd place
    wide = torch.full((b, t, h * d + 9), KEPT, dtype=dtype)
    wide[..., 3:3 + h * d] = x.flatten(2)
    return wide.cuda()[..., 3:3 + h * d].unflatten(2, (h, d)).transpose(1, 2)


def _reference(x, positions, frequencies, axes, adjacent, inverse):
    """(out, |x0| + |x1|, |angle|) in 64 bits."""
    out, size, far = x.double(), torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(x, dtype=torch.float64)
    n = frequencies.numel()
    for i in range(n):
        angle = (positions[axes[i]].double() * frequencies[i].double())[:, None]
        i0, i1 = (2 * i, 2 * i + 1) if adjacent else (i, i + n)
        c, s = torch.cos(angle), torch.sin(angle) * (-1 if inverse else 1)
        x0, x1 = x[..., i0].double(), x[..., i1].double()
        out[..., i0], out[..., i1] = x0 * c - x1 * s, x1 * c + x0 * s
        for j in (i0, i1):
            size[..., j], far[..., j] = x0.abs() + x1.abs(), angle.abs().expand_as(x0)
    return out, size, far


def _check(got, x, positions, frequencies, axes, adjacent, inverse):
    want, size, far = _reference(x, positions, frequencies, axes, adjacent, inverse)
    tol = size * (2.0**-21 + far * 2.0**-51) + want.abs() * torch.finfo(x.dtype).eps / 2 * (1 + 2.0**-16)
    tol = tol + (2.0**-25 if x.dtype == F16 else 1e-40)
    assert bool(((got.double() - want).abs() <= tol).all())
    tail = 2 * frequencies.numel()
    assert torch.equal(got[..., tail:], x[..., tail:])


# B, H, Hkv, T, D, pairs, axes
SIZES = [
    (1, 1, 1, 1, 2, 1, 1),
    (1, 32, 8, 1, 128, 64, 1),
    (2, 3, 1, 17, 72, 36, 2),
    (3, 4, 4, 33, 80, 20, 3),
    (1, 2, 1, 5, 7, 3, 2),
    (2, 5, 0, 300, 64, 32, 4),
    (1, 1, 1, 1000, 16, 7, 1),
    (7, 2, 2, 3, 512, 256, 2),
    (1, 40, 8, 700, 128, 64, 3),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("layout,adjacent,inverse,positions", [
    ("tokens", False, False, torch.int64), ("heads", True, True, torch.int32), ("odd", False, True, torch.float32),
    ("odd", True, False, torch.int64),
])
def test_against_the_formula(ob, dtype, size, layout, adjacent, inverse, positions):
    B, H, Hkv, T, D, pairs, A = size
    q = _tensor((B, H, T, D), layout, dtype, 1)
    k = _tensor((B, Hkv, T, D), layout, dtype, 2) if Hkv else None
    g = torch.Generator().manual_seed(3)
    where = torch.randint(0, 5000, (A, B, T), generator=g).to(positions).cuda()
    frequencies = (10000.0 ** (-torch.arange(pairs).double() / pairs)).to(F32 if inverse else torch.float64).cuda()
    axes = [(i * 7) % A for i in range(pairs)]
    q_out, k_out = ob.rotary(q, k, where if A > 1 else where[0], frequencies, axes=axes, adjacent=adjacent,
                             inverse=inverse)
    _check(q_out, q, where, frequencies, axes, adjacent, inverse)
    if Hkv:
        _check(k_out, k, where, frequencies, axes, adjacent, inverse)
    else:
        assert k_out is None


@pytest.mark.parametrize("position", [0, 1, 131071, 2**24 + 1, 2**31 - 1, -5])
def test_far_positions(ob, position):
    q = _tensor((1, 2, 1, 64), "heads", F32, 4)
    where = torch.full((1, 1), position, dtype=torch.int32, device="cuda")
    frequencies = (10000.0 ** (-torch.arange(32).double() / 32)).cuda()
    got, _ = ob.rotary(q, None, where, frequencies)
    _check(got, q, where[None], frequencies, [0] * 32, False, False)


@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("layout", ["tokens", "odd"])
def test_in_place_and_what_lies_around(ob, adjacent, layout):
    """In place, columns behind the pairs and around the heads stay as they are."""
    q, k = _tensor((2, 3, 19, 40), layout, BF16, 5), _tensor((2, 1, 19, 40), layout, BF16, 6)
    where = torch.arange(19, device="cuda").expand(2, 19)  # one row of positions for both: a stride of 0
    frequencies = torch.rand(12, device="cuda")
    want = ob.rotary(q, k, where, frequencies, adjacent=adjacent)
    before = q.clone()
    got = ob.rotary(q, k, where, frequencies, adjacent=adjacent, q_out=q, k_out=k)
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(q[..., 24:], before[..., 24:])
    if layout == "odd":
        base = q._base if q._base is not None else q
        wide = base.as_strided((2, 19, 3 * 40 + 9), (19 * 129, 129, 1), 0)
        assert bool((wide[..., :3] == KEPT).all()) and bool((wide[..., 123:] == KEPT).all())


def test_back_and_gradients(ob):
    """inverse undoes the turn, and is its gradient: by the formula and by differences."""
    q, k = _tensor((1, 2, 9, 24), "tokens", F32, 7), _tensor((1, 1, 9, 24), "tokens", F32, 8)
    where = torch.randint(0, 300, (3, 1, 9), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    frequencies = torch.logspace(0, -2, 10, device="cuda")
    axes = ob.rotary_axes([4, 3, 3], interleaved=True)
    assert list(axes) == [0, 1, 2, 0, 1, 2, 0, 1, 2, 0] and list(ob.rotary_axes([1, 2])) == [0, 1, 1]
    turned = ob.rotary(q, k, where, frequencies, axes=axes)
    back = ob.rotary(*turned, where, frequencies, axes=axes, inverse=True)
    for x, y in zip((q, k), back):  # two turns, each within 2^-21 of |x0| + |x1| and its rounding
        assert float((x - y).abs().max()) <= 3 * 2.0**-20 * float(x.abs().max())
    gq, gk = _tensor((1, 2, 9, 24), "heads", F32, 9), _tensor((1, 1, 9, 24), "heads", F32, 10)
    dq, dk = ob.rotary(gq, gk, where, frequencies, axes=axes, inverse=True)
    x = q.double().requires_grad_()
    y, n = x.clone(), 10
    angle = torch.stack([where[a].double() * frequencies[i].double() for i, a in enumerate(axes)], -1)[:, None]
    x0, x1 = x[..., :n], x[..., n:2 * n]
    y = torch.cat([x0 * angle.cos() - x1 * angle.sin(), x1 * angle.cos() + x0 * angle.sin(), x[..., 2 * n:]], -1)
    (y * gq.double()).sum().backward()
    assert float((dq.double() - x.grad).abs().max()) <= 2.0**-20 * 2 * float(gq.abs().max())
    # The operator is linear: a step along d changes <rotary(q), g> by <d, rotary^-1(g)>.
    d = _tensor((1, 1, 9, 24), "heads", F32, 11)
    moved = ob.rotary(k + d, None, where, frequencies, axes=axes)[0].double() - turned[1].double()
    left, right = float((moved * gk.double()).sum()), float((d.double() * dk.double()).sum())
    # 216 terms; k + d and both turns are rounded: 4 * 2^-21 of products of numbers below 8.
    assert abs(left - right) <= 216 * 64 * 2.0**-19


def test_new_outputs_are_laid_out_as_their_inputs(ob):
    """So that a projection's rows stay rows."""
    q, k = _tensor((2, 3, 5, 16), "tokens", BF16, 20), _tensor((2, 2, 5, 16), "heads", BF16, 21)
    q_out, k_out = ob.rotary(q, k, torch.zeros(2, 5, dtype=torch.int32, device="cuda"), torch.ones(8, device="cuda"))
    assert q_out.stride() == q.stride() and k_out.stride() == k.stride()
    assert torch.equal(q_out, q) and torch.equal(k_out, k)  # position 0 turns nothing


def test_not_finite(ob):
    q = _tensor((1, 1, 3, 8), "heads", F32, 12)
    where = torch.tensor([[0.0, float("inf"), float("nan")]], device="cuda")
    got, _ = ob.rotary(q, None, where, torch.ones(4, device="cuda"))
    assert torch.equal(got[0, 0, 0], q[0, 0, 0]) and bool(got[0, 0, 1:].isnan().all())


def test_no_tokens(ob):
    q = torch.empty(1, 2, 0, 8, dtype=BF16, device="cuda")
    got, _ = ob.rotary(q, None, torch.empty(1, 0, dtype=torch.int32, device="cuda"), torch.ones(4, device="cuda"))
    assert got.shape == q.shape


def test_captured_and_on_another_stream(ob):
    q, k = _tensor((1, 8, 64, 64), "tokens", BF16, 13), _tensor((1, 2, 64, 64), "tokens", BF16, 14)
    where = torch.arange(64, device="cuda").view(1, 64)
    frequencies = torch.logspace(0, -4, 32, device="cuda")
    want = ob.rotary(q, k, where, frequencies)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = ob.rotary(q, k, where, frequencies, stream=s)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ob.rotary(q, k, where, frequencies)
    where.add_(1000)
    graph.replay()
    after = ob.rotary(q, k, where, frequencies)
    torch.cuda.synchronize()
    assert torch.equal(held[0], after[0]) and torch.equal(held[1], after[1])
    assert not torch.equal(after[0], want[0])


def test_rows_past_32_bits(ob):
    """Elements past 2^31 of a tensor, read and written."""
    T, H, D = 140000, 128, 128
    if torch.cuda.mem_get_info()[0] < 14e9:
        pytest.skip("not enough memory")
    q = torch.zeros(1, T, H, D, dtype=BF16, device="cuda").transpose(1, 2)
    q[:, :, -2:] = _tensor((1, H, 2, D), "heads", BF16, 15)
    where = torch.arange(T, device="cuda").view(1, T)
    frequencies = (10000.0 ** (-torch.arange(64).double() / 64)).cuda()
    ob.rotary(q, None, where, frequencies, q_out=q)
    x = _tensor((1, H, 2, D), "heads", BF16, 15)
    _check(q[:, :, -2:].contiguous(), x, where[None, :, -2:], frequencies, [0] * 64, False, False)
