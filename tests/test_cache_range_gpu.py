"""attention_window_e2m1 at the ends of its ranges: as many keys as the entry point takes."""

import pytest

from tests.test_cache_gpu import BF16, F32, KEPT, _check, _i32, _stored, _tensor, ob  # noqa: F401
from tests.test_cache_paths_gpu import LIST, _names

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


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
