"""attention_window_e2m1 where the cache holds what is not finite behind some queries' masks: a
query gives NaN where it sees such a key or value, and is as if they were not there where it does
not.  One bad token at a time, at each edge of the masks, then all of them.

Tolerances are those of test_cache_gpu.py; the reference is softmax attention in 64 bits over the
keys that a query sees, with NaN wherever it sees one."""

import math

import pytest

from tests.test_cache_gpu import BF16, F16, F32, KEPT, _i32, _made, _stored, _tensor, ob  # noqa: F401
from tests.test_cache_paths_gpu import CLUSTER, LIST, PROMPT, _names

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _attended(q, k, v, n, m, window, right, sinks):
    """(out, mean of |v|, most |v|) of one sequence in 64 bits, NaN where a query sees one."""
    H, _, D = q.shape
    group = H // k.shape[0]
    p = torch.arange(n - m, n, device=q.device)[:, None]
    s = torch.arange(n, device=q.device)[None]
    seen = s <= p + right
    if window > 0:
        seen &= (s > p - window) | (s < sinks)
    kk, vv = (x[:, :n].double().repeat_interleave(group, 0) for x in (k, v))
    lost = (seen & kk.isnan().any(dim=2)[:, None]).any(dim=2, keepdim=True)
    lost = lost | (seen.double() @ vv.isnan().double() > 0)
    kk, vv = kk.nan_to_num(0.0), vv.nan_to_num(0.0)
    e = q[:, :m].double() @ kk.transpose(1, 2) * D**-0.5
    w = torch.nan_to_num(torch.softmax(e.masked_fill(~seen, -math.inf), dim=2))
    return (w @ vv).masked_fill(lost, math.nan), w @ vv.abs(), float(vv.abs().max())


def _check(got, q, k, v, lengths, counts, window, right, sinks, prompt):
    eps = torch.finfo(q.dtype).eps if prompt else 2.0**-10
    for b, (n, m) in enumerate(zip(lengths, counts)):
        assert bool((got[b, :, m:] == KEPT).all())
        if n == 0 or m == 0:
            continue
        want, mean, most = _attended(q[b], k[b], v[b], n, m, window, right, sinks)
        tol = mean * (eps + 2.0**-12) + n * 2.0**-25 * most + want.abs() * 2.0**-23 + 1e-30
        mine = got[b, :, :m].double()
        if prompt:  # all columns of a query that sees a value which is none
            want = want.masked_fill(want.isnan().any(dim=2, keepdim=True), math.nan)
        assert torch.equal(mine.isnan(), want.isnan())
        assert bool(((mine - want).abs() <= tol)[~want.isnan()].all())


def _edges(n, m, window, right, sinks):
    """Tokens that some queries see and some do not, and their neighbours."""
    at = {n - 1, n - 2, n - m, n - m + 1, n - m // 2, n - m + right, n - m + right + 1, 0, n // 3}
    if window > 0:
        at |= {n - m - window, n - m - window + 1, n - window, n - window - 1, n - m // 2 - window, sinks - 1, sinks}
    return sorted(t for t in at if 0 <= t < n)


def _go(ob, tmp_path, case, dtype, kernels):  # noqa: F811
    B, H, Hkv, T, D, page, lengths, counts, window, right, sinks = case
    capacity = max(lengths)
    cache, table = _made(ob, B, Hkv, D, capacity, page, 150)
    k, v = (_tensor((B, Hkv, capacity, D), "heads", dtype, s, 0.3) for s in (151, 152))
    q = _tensor((B, H, T, D), "tokens", dtype, 153)
    held, m = _i32(lengths), _i32(counts)
    out = torch.full(q.shape, KEPT, dtype=F32, device="cuda")

    def call():
        return ob.attention_window_e2m1(q, cache, held, q_lengths=m, table=table, window=window, right=right,
                                        sinks=sinks, out=out)

    assert _names(call, tmp_path) == kernels
    g = torch.Generator().manual_seed(154)

    def spoil(of, b, token):
        head, column = (int(torch.randint(0, x, (1,), generator=g)) for x in (Hkv, D))
        of[b, head, token, column] = (math.nan, math.inf, -math.inf)[token % 3]

    bad = [(b, t) for b in range(B) for t in _edges(lengths[b], counts[b], window, right, sinks)]
    for b, t in bad:
        if b > 2:
            break
        kk, vv = k.clone(), v.clone()
        spoil(vv, b, t)
        ob.cache_write_e2m1(kk, vv, cache, held, q_lengths=held, table=table)
        out.fill_(KEPT)
        call()
        _check(out, q, _stored(kk), _stored(vv), lengths, counts, window, right, sinks, kernels == PROMPT)
    kk, vv = k.clone(), v.clone()
    for b, t in bad:
        spoil(kk if t == lengths[b] - 1 else vv, b, t)
    ob.cache_write_e2m1(kk, vv, cache, held, q_lengths=held, table=table)
    out.fill_(KEPT)
    call()
    _check(out, q, _stored(kk), _stored(vv), lengths, counts, window, right, sinks, kernels == PROMPT)
    ob.library().sync_check()


FEW = [
    ((2, 8, 2, 5, 128, 64, [300, 77], [5, 4], 0, 0, 0), CLUSTER),
    ((2, 8, 2, 7, 64, 32, [500, 90], [7, 3], 60, 0, 9), CLUSTER),
    ((1, 4, 4, 16, 96, 16, [200], [16], 33, 5, 20), CLUSTER),
    ((1, 40, 2, 3, 72, 48, [1000], [3], 100, 0, 3), CLUSTER),
    ((1, 6, 3, 60, 32, 16, [61], [60], 10, 100, 5), CLUSTER),
    ((16, 32, 8, 5, 64, 64, list(range(64, 1025, 64)), [5] * 16, 0, 0, 0), CLUSTER),
    ((1, 8, 2, 40, 128, 48, [40000], [40], 0, 0, 0), LIST),
    ((1, 8, 2, 40, 96, 48, [40000], [40], 20000, 7, 41), LIST),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case,kernels", FEW)
def test_values_that_some_queries_do_not_see(ob, tmp_path, case, kernels, dtype):  # noqa: F811
    _go(ob, tmp_path, case, dtype, kernels)


# B, H, Hkv, T, D, page, lengths, counts, window, right, sinks
PROMPTS = [
    (1, 4, 1, 600, 64, 16, [650], [600], 0, 0, 0),
    (2, 8, 2, 300, 128, 64, [700, 300], [300, 299], 128, 0, 1),
    (1, 8, 2, 200, 96, 48, [1000], [200], 77, 30, 70),
    (3, 16, 4, 260, 32, 32, [260, 0, 500], [260, 0, 200], 40, 0, 130),
    (1, 4, 1, 400, 72, 64, [3000], [400], 1500, 0, 20),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", PROMPTS)
def test_values_that_some_queries_of_a_prompt_do_not_see(ob, tmp_path, case, dtype):  # noqa: F811
    _go(ob, tmp_path, case, dtype, PROMPT)


@pytest.mark.parametrize("case", PROMPTS)
def test_missing_pages_that_some_queries_of_a_prompt_do_not_see(ob, case):  # noqa: F811
    """A page that is none is NaN for the queries that see a key there, and for no others."""
    B, H, Hkv, T, D, page, lengths, counts, window, right, sinks = case
    cache, table = _made(ob, B, Hkv, D, max(lengths), page, 160)
    k, v = (_tensor((B, Hkv, max(lengths), D), "heads", F16, s, 0.3) for s in (161, 162))
    q = _tensor((B, H, T, D), "tokens", F16, 163)
    held, m = _i32(lengths), _i32(counts)
    ob.cache_write_e2m1(k, v, cache, held, q_lengths=held, table=table)
    b = max(range(B), key=lambda b: lengths[b])
    n = lengths[b]
    for at in sorted({(n - 1) // page, (n - counts[b]) // page, max(n - counts[b] - window, 0) // page, sinks // page}):
        some = table.clone()
        some[b, at] = -1
        kk, vv = _stored(k), _stored(v)
        kk[b, :, at * page:(at + 1) * page] = math.nan
        out = torch.full(q.shape, KEPT, dtype=F32, device="cuda")
        ob.attention_window_e2m1(q, cache, held, q_lengths=m, table=some, window=window, right=right, sinks=sinks, out=out)
        _check(out, q, kk, vv, lengths, counts, window, right, sinks, True)
