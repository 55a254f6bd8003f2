"""How much of the workspace attention of packed sequences takes, against what the header promises."""
import os
import re

import numpy as np
import pytest

import juliavision_b200 as jv
from tests.test_gpu_decode import F16, ints

pytestmark = pytest.mark.gpu


def promised():
    with open(os.path.join(os.path.dirname(jv.__file__), "..", "include", "b200dnn.h")) as f:
        text = f.read()
    text = text[text.index("Scratch comes from", text.index("attention of packed sequences")):]
    found = re.search(r"(\d+) MB,? (?:and )?(\d+) bytes a row(?: and (\d+) bytes a sequence)?", text.replace("\n *", "").replace("  ", " "))
    return [int(n or 0) for n in found.groups()]


@pytest.mark.parametrize("E, Hq, N, B", [(128, 128, 60000, 60000), (128, 128, 60000, 100), (64, 1, 3, 4000000), (8, 1, 500000, 500000), (128, 2, 70000, 1024)])
def test_no_more_than_is_promised(ctx, E, Hq, N, B):
    """All heads on one key head, so that a tile has few tokens; a row a sequence; far more sequences than rows."""
    fixed, row, sequence = promised()
    q, out = (ctx.allocate(F16, E, Hq, N) for _ in range(2))
    kv = ctx.allocate(F16, E, 1, 1)
    for a in (q, kv):
        ctx.fill_bytes(a, 0)
    ctx.fill_bytes(out, 0xFF)
    starts, kstarts = np.minimum(np.arange(B + 1) * max(N // B, 1), N), np.zeros(B + 1, np.int64)
    starts[-1], kstarts[-1] = N, 1
    ctx.ws.reset()
    before = ctx.ws.stats()[0]
    jv.packedsdpa_(ctx, out.permute((0, 2, 1)), q.permute((0, 2, 1)), kv.permute((0, 2, 1)), kv.permute((0, 2, 1)), ints(ctx, starts), ints(ctx, kstarts))
    used = ctx.ws.stats()[0] - before
    ctx.synchronize()
    assert used <= fixed * 10 ** 6 + row * N + sequence * B, (used, fixed * 10 ** 6 + row * N + sequence * B)
    last = jv.DeviceArray(ctx, out.ptr + 2 * E * Hq * (N - 1), F16, (E, Hq), owner=out)
    assert not last.to_host().any()
