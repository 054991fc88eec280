"""attention_window_e2m1 at the ends of its ranges: keys whose weights are far below the largest,
and as many keys as the entry point takes."""

import math

import pytest

from tests.test_cache_gpu import BF16, F16, F32, KEPT, _check, _i32, _stored, _tensor, ob  # noqa: F401
from tests.test_cache_paths_gpu import LIST, PROMPT, _names

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


# A first token, and keys at 2^-below of its weight whose values alone are not 0: the result is
# what they sum to.  The weights are rounded to multiples of 2^-24 where the largest is 2^7 or
# more: each loses at most 2^-25 / 2^7 of it.  Sums run over the keys of a tile, in whatever
# order, so with A the weighted mean of |v| the tolerance is A (2^-10 + 2^-12) + keys * 2^-32 * |v|.
@pytest.mark.parametrize("below", [24.6, 25.5, 30.0])
@pytest.mark.parametrize("B,T,keys,dtype", [
    (1, 1, 131072, BF16), (600, 1, 4096, BF16), (600, 1, 4096, F16), (700, 3, 1000, F16),  # tiles of one CTA
    (1, 600, 8192, F16), (1, 600, 8192, BF16),  # prompts
])
def test_keys_far_below_the_largest(ob, tmp_path, B, T, keys, dtype, below):  # noqa: F811
    D = 32
    k = torch.zeros(1, 1, keys, D, dtype=dtype, device="cuda")
    v = torch.zeros_like(k)
    k[..., 0], k[:, :, 0, 0] = -6.0, 6.0
    v[:, :, 1:] = torch.rand(keys - 1, D, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) + 0.5
    cache = ob.empty_cache_e2m1(-(-keys // 16), 1, 16, D)
    pages = torch.arange(cache.shape[0], dtype=torch.int32, device="cuda")
    ob.cache_write_e2m1(k, v, cache, _i32([keys]), table=pages[None])
    table = pages.expand(B, -1).contiguous()  # a prefix that all sequences share
    q = torch.zeros(B, 1, T, D, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    scale = below / (12 * math.log2(math.e))
    held = _i32([keys] * B)

    def call():
        return ob.attention_window_e2m1(q, cache, held, table=table, right=T, scale=scale, out_dtype=F32)

    assert (_names(call, tmp_path) == PROMPT) == (T == 600)
    got = call().double()
    e = torch.full((keys,), 2.0**-below, dtype=torch.float64, device="cuda")
    e[0] = 1.0
    want = (e / e.sum()) @ _stored(v)[0, 0]
    eps = torch.finfo(BF16).eps if T == 600 and dtype == BF16 else 2.0**-10
    tol = want * (eps + 2.0**-12) + keys * 2.0**-32 * 2.0
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


def test_as_many_keys_as_there_may_be(ob, tmp_path):  # noqa: F811
    """2^30 keys for 512 rows of a key head: more than 2^31 blocks in all tiles.  The pages of the
    table are a few, over and over; a key of those at its ends and in its middle weighs 2^50 times
    what others do, so that the sums are theirs."""
    D, page, H = 32, 1024, 512
    width = 2**30 // page
    k, v = (_tensor((1, 1, 5 * page, D), "heads", BF16, s) for s in (171, 172))
    k[..., 0] = 16.0
    k[:, :, 4 * page:, 0] = -16.0
    cache = ob.empty_cache_e2m1(5, 1, page, D)
    ob.cache_write_e2m1(k, v, cache, _i32([5 * page]), table=_i32([[0, 1, 2, 3, 4]]))
    table = torch.full((1, width), 4, dtype=torch.int32, device="cuda")
    for i, at in enumerate((0, 1, width // 2, width - 1)):
        table[0, at] = i
    q = _tensor((1, H, 1, D), "heads", BF16, 173)
    q[..., 0] = 8.0
    held = _i32([2**30])
    out = torch.full(q.shape, KEPT, dtype=F32, device="cuda")

    def call():
        return ob.attention_window_e2m1(q, cache, held, table=table, out=out)

    assert _names(call, tmp_path) == LIST
    _check(out, q, _stored(k)[:, :, :4 * page], _stored(v)[:, :, :4 * page], [4 * page], [1])
    ob.library().sync_check()
