"""Adapters on the GPU where a tile's workgroups take several adapters one after the other, popular ones (through LDS)
and ones of a few tokens in turn, with K in parts that rounding leaves fewer of (k 5120, 4608, 4104) and in full ones:
against 64 bits, and bit for bit against a few of the tokens alone."""
import numpy as np
import pytest

from atomflow_amd import kv
from test_gpu_lora import Case, say

pytestmark = pytest.mark.gpu


def mixed_ids(m, count, rng):
    """Each tile of 64 tokens: 30 of one adapter, the others two to an adapter; the popular one comes first in
    even tiles and behind 17 others in odd ones."""
    ids = np.zeros(m, np.int32)
    for t, at in enumerate(range(0, m, 64)):
        popular = t % count
        others = (popular + 1 + rng.permutation(count - 1)[:17]) % count
        few, many = np.repeat(others, 2), np.full(30, popular)
        tile = np.concatenate([many, few]) if t % 2 == 0 else np.concatenate([few, many])
        ids[at:at + 64] = tile[:m - at]
    return ids


@pytest.mark.parametrize("m,k,ends,rmax", [
    (300, 5120, [40, 70, 100], 64), (1100, 5120, [60], 16), (2048, 4608, [33, 50], 40), (2000, 4104, [40], 24),
    (1000, 4096, [48], 16), (900, 6656, [20, 30, 40], 32), (700, 14336, [30, 64], 64), (3000, 1304, [20, 40], 128)])
@pytest.mark.parametrize("ranks", [True, False])
def test_tiles_of_many_adapters(gpu, m, k, ends, rmax, ranks):
    say(f"lora, popular adapters and small ones m={m} k={k} ends={ends} rank={rmax} ranks={ranks}")
    r = np.random.default_rng(k + m)
    count = 24
    c = Case(m, k, ends, rmax, count, k, ranks=ranks)
    c.ids[:] = mixed_ids(m, count, r)

    def launch(case):
        case.device()
        if not ranks:
            case.lora = kv.make_lora(case.da, case.db, count, rmax, k, ends, scales=case.ds)
        case.call()
        return case

    launch(c).check()
    got = c.do.get()
    for _ in range(2):  # and again over its own workspace
        c.call()
        assert c.do.get().tobytes() == got.tobytes()
    some = np.concatenate([np.arange(28, 36), r.permutation(m)[:30], [m - 1]])
    part = Case(len(some), k, ends, rmax, count, k, ranks=ranks)
    for name in ("a", "b", "ranks", "scales"):
        setattr(part, name, getattr(c, name))
    part.x, part.y, part.ids = (t[some].copy() for t in (c.x, c.y, c.ids))
    assert launch(part).do.get().tobytes() == got[some].tobytes()
