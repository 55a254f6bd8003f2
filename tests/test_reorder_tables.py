"""The table of a search's beams and the array of the pages that they write: one array for both is refused, two that lie in one another are not."""
import numpy as np
import pytest

import juliavision_b200 as jv
from tests.test_decode_host import I32, FakeCtx, arr, cache, refused

AT = 1 << 20


def parts():
    c = cache(k=arr(np.int8, (64, 16, 2, 5), ptr=2 << 20), v=arr(np.int8, (64, 16, 2, 5), ptr=3 << 20))
    return c, arr(I32, (2, 2), ptr=5 << 20), arr(I32, (4,), ptr=6 << 20)


@pytest.mark.parametrize("ld", [3, 4, 7])
@pytest.mark.parametrize("off", ["same", "a number on", "a column on", "the last number", "a number before", "back to the last"])
def test_shared_memory_is_refused(off, ld):
    """(3, 4) numbers in columns ld apart."""
    c, parents, lens = parts()
    at = {"same": 0, "a number on": 1, "a column on": ld, "the last number": 3 * ld + 2, "a number before": -1, "back to the last": -3 * ld - 2}[off]
    t, own = arr(I32, (3, 4), (1, ld), AT), arr(I32, (3, 4), (1, ld), AT + 4 * at)
    refused(1, jv.cachereorder_, c, t, own, parents, lens)
    refused(1, jv.cachereorder_, [c], t, own, parents, lens)


def test_other_leading_dimensions():
    c, parents, lens = parts()
    refused(1, jv.cachereorder_, c, arr(I32, (3, 4), (1, 6), AT), arr(I32, (3, 4), (1, 5), AT), parents, lens)
    one = arr(I32, (1, 1), ptr=5 << 20)
    refused(1, jv.cachereorder_, c, arr(I32, (3, 1), ptr=AT), arr(I32, (3, 1), ptr=AT + 8), one, arr(I32, (1,), ptr=6 << 20))


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["behind", "before", "side by side", "columns apart", "between the last"])
def test_apart_in_one_buffer(ctx, where):
    """Two beams that change places: their tables and own pages in one buffer, whose other numbers stay."""
    from tests.test_gpu_beams import Cached, ints
    host = np.full(64, 77, np.int32)
    t0, o0, ld = {"behind": (20, 26, 3), "before": (26, 20, 3), "side by side": (20, 24, 8), "columns apart": (20, 36, 8), "between the last": (20, 31, 8)}[where]
    pages = np.array([[4, 0, 2], [1, 5, 3]])
    for s in range(2):
        host[t0 + s * ld:][:3] = host[o0 + s * ld:][:3] = pages[s]
    buf = ctx.toback(host)
    t, own = (jv.DeviceArray(ctx, buf.ptr + 4 * at, np.int32, (3, 2), (1, ld), owner=buf) for at in (t0, o0))
    c = Cached(ctx, np.random.default_rng(12), 64, 16, 2, [96], "int8", spare=0)
    old = c.host()
    jv.cachereorder_(ctx, c.cache, t, own, ints(ctx, [[1, 0]]), ints(ctx, [21, 21]))
    ctx.synchronize()
    for s in range(2):
        host[t0 + s * ld] = pages[1 - s][0]
    assert np.array_equal(buf.to_host(), host)
    want = old[0].copy()
    want[0, :, :5], want[5, :, :5] = old[0][5, :, :5], old[0][0, :, :5]
    assert np.array_equal(c.host()[0], want)
