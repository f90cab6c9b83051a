"""Row counts and bounds up to INT32_MAX on the GPU: a compaction's max_rows, a table's rows, rows that turn."""
import numpy as np
import pytest

from atomflow_amd import AF_ROPE_HALF
from atomflow_amd import device as dev
from atomflow_amd import kv
from inputs import fp16_ulp
from rows_ref import EPS24, assert_compact, table
from test_gpu_compact import Pool, launch, rows_of, say

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("kind", ["window", "half"])
@pytest.mark.parametrize("most", [MOST, MOST - 1, MOST - 300])
def test_compaction_bound(gpu, kind, most):
    """max_rows is any bound: rows that may go in any order, and rows that move in order."""
    say(f"compact {kind}, max_rows {most}")
    r = np.random.default_rng(most % 1000)
    bs, n = 16, 900
    cos, sin = table(n, 64)
    pool = Pool(2, 60, bs, 2, 64, False, 2)
    tables = r.permutation(60)[None, :57].astype(np.int32)
    f = 4 if kind == "window" else 0
    keep = rows_of(kind, n, r)[f:]
    launch(pool, tables, tables, [keep], [f], 64, 0, cos, sin, max_rows=most)
    assert_compact(pool.get(), pool.host, [(tables[0], tables[0], f, keep)], bs, 64, 0, cos, sin)


def test_rows_and_table(gpu):
    """A table of INT32_MAX rows of one pair, and as many rows of one head that turn by it."""
    say("table and rows, INT32_MAX of them")
    cos, sin, x = (dev.DeviceBuffer(4 * MOST) for _ in range(3))
    kv.build_rope_table_scaled(cos, sin, 0, MOST, 2, np.ones(1))
    x.fill_u32(0x3c00)  # (1, 0)
    kv.launch_rope_rows(x, 2, x, 2, 1, None, 0, None, 0, 0, MOST, 2, 2, AF_ROPE_HALF, cos, sin, MOST)
    for at in (0, 2 ** 24 - 50, 2 ** 30, 2 ** 31 - 101):
        angle = np.arange(at, at + 100, dtype=np.longdouble)
        exact = np.stack([np.cos(angle), np.sin(angle)], 1).astype(np.float64)
        got = np.stack([t.download(np.float32, offset=4 * at, count=100) for t in (cos, sin)], 1)
        # half a step of fp32, the series' end, and the turns' rounding
        off = EPS24 * np.abs(exact) + 1e-11 + at * 2.0 ** -51
        assert np.all(np.abs(got - exact) <= off)
        turned = x.download(np.float16, (100, 2), offset=4 * at).astype(np.float64)
        assert np.all(np.abs(turned - got) <= 0.5 * fp16_ulp(np.abs(got)))  # 1 and 0 times the table
