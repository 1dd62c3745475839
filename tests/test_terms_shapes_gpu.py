"""Head counts that are no power of two, with the workspace that the library asks for and no more (see also tests/terms_workspace.cu)."""
import pytest
import torch as th

from helpers import random_graph
from test_terms_gpu import Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("diff,buckets,h,d", [(False, 1, 63, 8), (False, 1, 55, 8), (False, 1, 47, 8), (False, 1, 126, 4), (False, 1, 94, 4),
                                              (True, 0, 63, 4), (True, 0, 47, 4), (True, 2, 63, 4)])
@pytest.mark.parametrize("planned", [False, True])
def test_double_precision_rows_of_many_heads(diff, buckets, h, d, planned):
    g = random_graph(700, 700, [2] * 700, 41)
    layer = Layer(g, diff, buckets, h, d, th.float64, th.int64, seed=41)
    layer.check(layer.step(layer.plans() if planned else None))


@pytest.mark.parametrize("dt,d", [(th.float32, 16), (th.bfloat16, 32)], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("h", [7, 13, 23, 31, 62])
def test_other_types(dt, d, h):
    if h * d * (4 if dt == th.float32 else 2) > 4096:
        d //= 2
    for diff, buckets in ((False, 3), (True, 0)):
        g = random_graph(300, 300, [3] * 300, 42)
        layer = Layer(g, diff, buckets, h if not diff else h // 2, d, dt, seed=42)
        layer.check(layer.step())


def test_the_gathering_walker_at_its_largest_records():
    """A source side whose tables are too large for the summing walker, walked a tile at a time in 63 blocks of heads."""
    g = random_graph(20000, 20000, [1] * 20000, 43)
    layer = Layer(g, False, 1, 63, 8, th.float64, th.int64, seed=43)
    layer.check(layer.step())
