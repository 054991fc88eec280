"""attention_window_e2m1 under windows, first tokens and keys past the queries: where a list's
CTAs share what a mask leaves of a tile, and prompts, whose rows of a key head are more than
its kernel for few rows takes.  A captured call says which kernels it launched.  Tolerances and
references are those of test_cache_gpu.py."""

import pytest

from tests.launches import launched
from tests.test_cache_gpu import BF16, F16, F32, KEPT, _case, _check, _i32, _tensor, ob  # noqa: F401
from tests.test_cache_paths_gpu import CLUSTER, LIST, PROMPT, _names, _paged

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# B, H, Hkv, T, D, page, lengths, window, right, sinks, rows of a tile
LISTS = [
    (1, 8, 2, 1, 64, 64, [65000], 40000, 0, 40, 8),
    (1, 8, 2, 1, 64, 64, [65000], 20000, 0, 20003, 8),  # shares that end among the first tokens
    (1, 4, 4, 1, 32, 16, [120000], 50000, 0, 33333, 8),
    (1, 8, 2, 1, 128, 128, [131072], 65536, 0, 0, 8),
    (2, 16, 1, 1, 128, 256, [130000, 70000], 90000, 0, 33, 16),
    (1, 16, 2, 60, 48, 64, [30000], 25000, 100, 10, 16),
    (1, 8, 2, 40, 128, 48, [40000], 20000, 7, 41, 24),
    (1, 8, 2, 40, 128, 48, [40000], 9000, 30, 15001, 24),
    (1, 40, 2, 1, 96, 64, [100000], 60000, 0, 1001, 24),
    (3, 24, 3, 9, 80, 32, [50000, 49000, 20000], 30001, 5, 77, 24),
    # Sequences far shorter than their pages: shares of tiles that have few keys, or none.
    (160, 4, 1, 3, 32, 16, [16384] + list(range(159)), 16000, 0, 35, 16),
    (150, 4, 1, 1, 32, 16, list(range(148, 0, -1)) + [0, 16384], 16000, 0, 35, 8),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", LISTS)
def test_lists_under_masks(ob, tmp_path, case, dtype):  # noqa: F811
    B, H, Hkv, T, D, page, lengths, window, right, sinks, height = case
    cache, table, k, v = _paged(ob, B, Hkv, D, -(-max(lengths) // page), page, lengths, dtype, 140)
    q = _tensor((B, H, T, D), "tokens", dtype, 143)
    counts = [min(T, n) for n in lengths]
    held, m = _i32(lengths), _i32(counts)
    out = torch.full(q.shape, KEPT, dtype=F32, device="cuda")

    def call():
        return ob.attention_window_e2m1(q, cache, held, q_lengths=m, table=table, window=window, right=right,
                                        sinks=sinks, out=out)

    assert _names(call, tmp_path) == LIST
    assert all(f"ILi{-(-D // 32) * 32}ELi{height // 8}E" in name for name, _, _ in launched(call, tmp_path))
    call()
    _check(out, q, k, v, lengths, counts, window, right, sinks)
    ob.library().sync_check()


@pytest.mark.parametrize("lengths,T", [([700, 650], 60), ([1500, 3], 100)])
def test_clusters_of_many_rows(ob, tmp_path, lengths, T):  # noqa: F811
    """Hundreds of rows of a key head go to clusters: the kernel that test_cache_paths_gpu.py's
    test of the same sizes has, whose numbers it checks."""
    B, H, Hkv, D = 2, 8, 2, 64
    cache, table, _, _ = _paged(ob, B, Hkv, D, 30, 64, lengths, BF16, 120)
    q = _tensor((B, H, T, D), "tokens", BF16, 123)
    held, m = _i32(lengths), _i32([min(T, n) for n in lengths])
    for window, right, sinks in ((0, 0, 0), (100, 0, 17), (33, 30, 4), (0, 1000, 0), (1, 0, 0)):
        assert _names(lambda: ob.attention_window_e2m1(
            q, cache, held, q_lengths=m, table=table, window=window, right=right, sinks=sinks,
            kv_len=max(lengths)), tmp_path) == CLUSTER


# B, H, Hkv, T, D, page, lengths, counts, window, right, sinks
PROMPTS = [
    (1, 4, 1, 600, 64, 16, [650], [600], 0, 0, 0),
    (1, 8, 2, 200, 32, 32, [900], [200], 100, 40, 33),
    (3, 8, 1, 150, 96, 48, [500, 0, 150], [150, 0, 149], 77, 9, 70),
    (2, 16, 1, 100, 16, 16, [700, 90], [100, 90], 0, 0, 0),
    (1, 16, 2, 300, 8, 16, [300], [300], 0, 1000, 0),
    (4, 4, 1, 257, 128, 64, [257, 1, 600, 0], [257, 1, 200, 0], 0, 3, 0),
    (1, 4, 4, 1100, 72, 32, [2000], [1100], 300, 0, 5),
    (2, 8, 1, 129, 120, 64, [129, 1000], [129, 129], 513, 65, 64),
    (1, 32, 1, 33, 64, 0, [400], [33], 0, 7, 0),
    (1, 4, 1, 400, 128, 64, [3000], [400], 1500, 0, 20),
    (3, 8, 1, 200, 64, 32, [100, 0, 500], [200, 200, 200], 0, 0, 0),  # more queries than keys
    (3, 8, 1, 200, 80, 32, [100, 1, 199], [200, 150, 200], 50, 30, 9),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", PROMPTS)
def test_prompts_by_the_prompts_kernel(ob, tmp_path, case, dtype):  # noqa: F811
    B, H, Hkv, T, D, page, lengths, counts, window, right, sinks = case
    q, cache, table, k, v = _case(ob, B, H, Hkv, T, D, page, lengths, counts, dtype, "rows")
    held, m = _i32(lengths), _i32(counts)
    for out_dtype in (dtype, F32):
        out = torch.full(q.shape, KEPT, dtype=out_dtype, device="cuda")

        def call():
            return ob.attention_window_e2m1(q, cache, held, q_lengths=m, table=table, window=window, right=right,
                                            sinks=sinks, out=out)

        assert _names(call, tmp_path) == PROMPT
        call()
        _check(out, q, k, v, lengths, counts, window, right, sinks, prompt=True)
    ob.library().sync_check()


# Prompts by their length that have few rows of a key head all the same, with the tolerance of
# the kernel that takes them.
FEW = [
    (1, 1, 1, 65, 64, 0, [65], [65], 0, 0, 0),
    (2, 1, 1, 130, 32, 16, [128, 0], [128, 0], 20, 0, 2),
    (1, 2, 2, 400, 16, 0, [400], [400], 0, 50, 0),
    (1, 8, 2, 128, 8, 32, [128], [128], 1, 0, 0),
    (3, 8, 4, 150, 96, 16, [150, 3, 77], [150, 3, 20], 0, 0, 0),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", FEW)
def test_prompts_of_few_rows(ob, tmp_path, case, dtype):  # noqa: F811
    B, H, Hkv, T, D, page, lengths, counts, window, right, sinks = case
    q, cache, table, k, v = _case(ob, B, H, Hkv, T, D, page, lengths, counts, dtype, "rows")
    held, m = _i32(lengths), _i32(counts)
    out = torch.full(q.shape, KEPT, dtype=F32, device="cuda")

    def call():
        return ob.attention_window_e2m1(q, cache, held, q_lengths=m, table=table, window=window, right=right,
                                        sinks=sinks, out=out)

    assert _names(call, tmp_path) == CLUSTER
    call()
    _check(out, q, k, v, lengths, counts, window, right, sinks)
    ob.library().sync_check()


def test_a_captured_prompt_replayed_with_other_lengths_and_pages(ob, tmp_path):  # noqa: F811
    """Lengths, pages and the workspace's old contents are the replay's own matter."""
    B, H, Hkv, T, D, page = 2, 8, 1, 150, 64, 32
    q, cache, table, k, v = _case(ob, B, H, Hkv, T, D, page, [400, 400], [T, T], F16)
    held, m = _i32([400, 400]), _i32([T, T])
    out = torch.full(q.shape, KEPT, dtype=F32, device="cuda")

    def call():
        return ob.attention_window_e2m1(q, cache, held, q_lengths=m, table=table, window=90, right=2, sinks=5, out=out)

    assert _names(call, tmp_path) == PROMPT
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lengths, counts in (([400, 37], [T, 37]), ([0, 399], [9, 100]), ([200, 1], [T, 0])):
        held.copy_(_i32(lengths))
        m.copy_(_i32(counts))
        out.fill_(KEPT)
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, k, v, lengths, counts, 90, 2, 5, prompt=True)
    table.copy_(table.flip(0))  # the sequences change places
    held.copy_(_i32([333, 400]))
    m.copy_(_i32([T, T]))
    graph.replay()
    torch.cuda.synchronize()
    _check(out, q, k.flip(0), v.flip(0), [333, 400], [T, T], 90, 2, 5, prompt=True)
