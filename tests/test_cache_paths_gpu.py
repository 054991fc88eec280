"""attention_window_e2m1 where its kernels go round: each way to split the keys, every cluster
size, CTAs with more tiles than they work out at once, one sequence among empty ones, captured
calls replayed with other lengths, calls on several streams at once.  A captured call says which
kernels it launched, so that a change of a rule cannot take a case away unseen.  Tolerances and
references are those of test_cache_gpu.py."""

import math

import pytest

from tests.launches import launched
from tests.test_cache_gpu import BF16, F16, F32, KEPT, _check, _i32, _stored, _tensor, ob  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _paged(ob, B, Hkv, D, width, page, lengths, dtype, seed):
    """(cache, table, k, v): sequences of these lengths in a table `width` pages wide, whose
    entries past a sequence's pages are none; k and v as the cache stands for, up to the longest."""
    most = max(max(lengths), 1)
    need = [-(-n // page) for n in lengths]
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(need) + 1, generator=g).to(torch.int32)
    table = torch.full((B, width), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    table = table.cuda()
    cache = ob.empty_cache_e2m1(sum(need) + 1, Hkv, page, D)
    cache.random_(0, 256, generator=torch.Generator("cuda").manual_seed(seed))
    k, v = (_tensor((B, Hkv, most, D), "heads", dtype, seed + s, 0.3) for s in (1, 2))
    ob.cache_write_e2m1(k, v, cache, _i32(lengths), q_lengths=_i32(lengths), table=table)
    return cache, table, _stored(k), _stored(v)


def _names(call, tmp_path):
    return [next(n for n in ("e2m1_cluster", "e2m1_list", "e2m1_join", "cache_read", "window_prompt") if n in name)
            for name, _, _ in launched(call, tmp_path)]


# B, H, Hkv, T, D, page, lengths, window, sinks, kernels, rows of a tile
LIST, CLUSTER, PROMPT = ["e2m1_list", "e2m1_join"], ["e2m1_cluster"], ["cache_read", "window_prompt"]
CASES = [
    (1, 8, 2, 1, 64, 128, [65000], 0, 0, LIST, 8),        # one tile for each key head, many parts
    (1, 8, 2, 1, 128, 64, [20011], 0, 0, CLUSTER, 8),
    (2, 16, 1, 1, 128, 256, [130000, 7], 0, 0, LIST, 16),
    (1, 40, 2, 1, 96, 64, [100000], 0, 0, LIST, 24),      # of which 20 are there
    (1, 8, 2, 40, 128, 48, [40000], 0, 0, LIST, 24),      # seven tiles of rows
    (1, 6, 2, 33, 80, 32, [3000], 700, 40, CLUSTER, 8),
    (1, 4, 4, 1, 32, 16, [120000], 0, 0, LIST, 8),
    (64, 20, 2, 1, 64, 64, list(range(7, 1000, 16)) + [1000], 0, 0, CLUSTER, 16),
    (16, 40, 2, 1, 64, 64, list(range(500, 2001, 100)), 1900, 5, CLUSTER, 24),
    (1, 8, 2, 300, 64, 64, [900], 0, 0, PROMPT, None),
    (8, 16, 16, 128, 128, 64, [128] * 8, 0, 0, PROMPT, None),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", CASES)
def test_each_way(ob, tmp_path, case, dtype):  # noqa: F811
    B, H, Hkv, T, D, page, lengths, window, sinks, kernels, height = case
    cache, table, k, v = _paged(ob, B, Hkv, D, -(-max(lengths) // page), page, lengths, dtype, 60)
    q = _tensor((B, H, T, D), "tokens", dtype, 63)
    counts = [min(T, n) for n in lengths]
    held, m = _i32(lengths), _i32(counts)
    out = torch.full(q.shape, KEPT, dtype=F32, device="cuda")

    def call():
        return ob.attention_window_e2m1(q, cache, held, q_lengths=m, table=table, window=window, sinks=sinks, out=out)

    assert _names(call, tmp_path) == kernels
    if height:
        assert all(f"ILi{-(-D // 32) * 32}ELi{height // 8}E" in name for name, _, _ in launched(call, tmp_path))
    call()
    _check(out, q, k, v, lengths, counts, window, 0, sinks, prompt=kernels == PROMPT)
    ob.library().sync_check()


@pytest.mark.parametrize("keys,parts", [(100, 1), (400, 2), (600, 4), (1500, 8), (4000, 16), (9000, 16)])
@pytest.mark.parametrize("rows", [4, 16])
def test_cluster_sizes(ob, tmp_path, keys, parts, rows):  # noqa: F811
    cache, table, k, v = _paged(ob, 1, 2, 128, -(-keys // 64), 64, [keys], BF16, 70)
    q = _tensor((1, 2 * rows, 1, 128), "tokens", BF16, 73)
    out = torch.full(q.shape, KEPT, dtype=F32, device="cuda")

    def call():
        return ob.attention_window_e2m1(q, cache, _held, table=table, kv_len=keys, out=out)

    _held = _i32([keys])
    (name, grid, _), = launched(call, tmp_path)
    assert "e2m1_cluster" in name and grid[0] == 2 * parts
    call()
    _check(out, q, k, v, [keys], [1])


@pytest.mark.parametrize("H,T", [(4, 1), (4, 3), (4, 5)])
def test_more_tiles_than_a_cta_works_out_at_once(ob, tmp_path, H, T):  # noqa: F811
    """Short sequences in wide tables: hundreds of tiles for a CTA, sequences without keys and
    without queries among them."""
    g = torch.Generator().manual_seed(H + T)
    B, Hkv, D, page = 5000, 2, 32, 16
    lengths = torch.randint(0, 60, (B,), generator=g)
    lengths[torch.rand(B, generator=g) < 0.3] = 0
    lengths[1000:2500] = 0  # CTAs that find nothing in their 32 tiles
    counts = torch.minimum(lengths, torch.randint(0, T + 1, (B,), generator=g))
    counts[1000:1400] = T  # queries of sequences without keys: rows of zeros
    lengths, counts = lengths.tolist(), counts.tolist()
    cache, table, k, v = _paged(ob, B, Hkv, D, 512, page, lengths, BF16, 80)
    q = _tensor((B, H, T, D), "heads", BF16, 83)
    held, m = _i32(lengths), _i32(counts)
    out = torch.full(q.shape, KEPT, dtype=F32, device="cuda")

    def call():
        return ob.attention_window_e2m1(q, cache, held, q_lengths=m, table=table, out=out)

    assert _names(call, tmp_path) == LIST
    call()
    # Queries at positions below 0 (more queries than keys) see nothing: zeros.
    want = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    mean, mine = torch.zeros_like(want), torch.zeros(B, 1, T, 1, dtype=torch.bool, device="cuda")
    n = torch.tensor(lengths, device="cuda").view(B, 1, 1)
    c = torch.tensor(counts, device="cuda").view(B, 1, 1)
    p = n - c + torch.arange(T, device="cuda").view(1, T, 1)
    s = torch.arange(k.shape[2], device="cuda").view(1, 1, -1)
    seen = ((s < n) & (s <= p))[:, None]
    kk, vv = (x.nan_to_num(0.0).repeat_interleave(H // Hkv, 1) for x in (k, v))
    e = (q.double() @ kk.transpose(2, 3) * D**-0.5).masked_fill(~seen, -math.inf)
    w = torch.nan_to_num(torch.softmax(e, dim=3))
    want, mean = w @ vv, w @ vv.abs()
    mine = (torch.arange(T, device="cuda")[None] < c.view(B, 1))[:, None, :, None].expand_as(want)
    tol = mean * (2.0**-10 + 2.0**-12) + 60 * 2.0**-25 * float(vv.abs().max()) + want.abs() * 2.0**-23 + 1e-30
    assert bool(((out.double() - want).abs() <= tol)[mine].all())
    assert bool((out[~mine] == KEPT).all())


def test_one_sequence_among_empty_ones(ob, tmp_path):  # noqa: F811
    """All CTAs of the list share the tiles of one sequence."""
    B, Hkv, D, page = 101, 2, 64, 32
    lengths = [0] * 50 + [30001] + [0] * 50
    cache, table, k, v = _paged(ob, B, Hkv, D, -(-30001 // page), page, lengths, F16, 90)
    q = _tensor((B, 8, 1, D), "heads", F16, 93)
    held, out = _i32(lengths), torch.full(q.shape, KEPT, dtype=F16, device="cuda")

    def call():
        return ob.attention_window_e2m1(q, cache, held, table=table, out=out)

    assert _names(call, tmp_path) == LIST
    call()
    alone = [slice(50, 51)]
    _check(out[alone[0]], q[50:51], k[50:51], v[50:51], [30001], [1])
    assert bool((out[:50] == 0).all()) and bool((out[51:] == 0).all())


def test_replayed_with_other_lengths(ob, tmp_path):  # noqa: F811
    """A captured call works its list out anew from the lengths and pages at each replay."""
    B, Hkv, D, page = 3, 2, 128, 64
    lengths = [40000, 20000, 100]
    cache, table, k, v = _paged(ob, B, Hkv, D, 625, page, lengths, BF16, 100)
    q = _tensor((B, 8, 1, D), "tokens", BF16, 103)
    held = _i32([64, 64, 64])
    assert _names(lambda: ob.attention_window_e2m1(q, cache, held, table=table), tmp_path) == LIST
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ob.attention_window_e2m1(q, cache, held, table=table, out_dtype=F32)
    for now in ([40000, 20000, 100], [1, 0, 100], [39999, 19, 64], [0, 20000, 99]):
        held.copy_(_i32(now))
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, k, v, now, [1, 1, 1])


def test_calls_at_once(ob):  # noqa: F811
    """Lists, joins and clusters of several streams under way together."""
    cases = []
    for seed, (B, H, Hkv, D, page, lengths) in enumerate([
        (1, 8, 2, 64, 128, [65000]), (2, 16, 1, 128, 256, [33000, 7]), (1, 8, 2, 128, 64, [20011]),
        (4, 32, 8, 128, 64, [5000, 100, 9000, 1]),
    ]):
        cache, table, _, _ = _paged(ob, B, Hkv, D, -(-max(lengths) // page), page, lengths, BF16, 110 + seed)
        q = _tensor((B, H, 1, D), "tokens", BF16, 113 + seed)
        cases.append((q, cache, _i32(lengths), table))
    want = [ob.attention_window_e2m1(q, c, n, table=t) for q, c, n, t in cases]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for turn in range(12):
        for i, s in enumerate(streams):
            j = (i + turn) % len(cases)
            q, c, n, t = cases[j]
            got.append((j, ob.attention_window_e2m1(q, c, n, table=t, stream=s)))
    torch.cuda.synchronize()
    for j, y in got:
        assert torch.equal(y, want[j])


@pytest.mark.parametrize("lengths,T", [([700, 650], 60), ([1500, 3], 100)])
def test_tiles_of_many_rows(ob, tmp_path, lengths, T):  # noqa: F811
    """Hundreds of rows of a key head, windows and first tokens, keys past the queries."""
    B, H, Hkv, D = 2, 8, 2, 64
    cache, table, k, v = _paged(ob, B, Hkv, D, 30, 64, lengths, BF16, 120)
    q = _tensor((B, H, T, D), "tokens", BF16, 123)
    counts = [min(T, n) for n in lengths]
    for window, right, sinks in ((0, 0, 0), (100, 0, 17), (33, 30, 4), (0, 1000, 0), (1, 0, 0)):
        out = torch.full(q.shape, KEPT, dtype=F32, device="cuda")

        def call():
            return ob.attention_window_e2m1(q, cache, held, q_lengths=m, table=table, window=window, right=right,
                                            sinks=sinks, kv_len=max(lengths), out=out)

        held, m = _i32(lengths), _i32(counts)
        assert _names(call, tmp_path) in (CLUSTER, LIST)
        call()
        _check(out, q, k, v, lengths, counts, window, right, sinks)


def test_missing_pages_of_long_sequences(ob):  # noqa: F811
    """An entry that is none far into a sequence, in a list and in a cluster."""
    for keys, at in ((65000, 400), (20011, 200), (20011, 311)):
        cache, table, k, v = _paged(ob, 2, 2, 64, -(-keys // 64), 64, [keys, 500], F16, 130)
        q = _tensor((2, 8, 1, 64), "heads", F16, 133)
        table[0, at] = cache.shape[0]
        out = ob.attention_window_e2m1(q, cache, _i32([keys, 500]), table=table)
        assert bool(out[0].isnan().all())
        got = torch.full((1, 8, 1, 64), KEPT, dtype=F16, device="cuda")
        got.copy_(out[1:])
        _check(got, q[1:], k[1:], v[1:], [500], [1])
        n = (keys // 64 - at) * 64 - 5  # a window that ends before the missing page
        out = ob.attention_window_e2m1(q, cache, _i32([keys, 500]), table=table, window=min(n, keys - (at + 1) * 64))
        assert bool(out.isfinite().all())
