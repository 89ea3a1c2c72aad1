"""Long rows at every place relative to the cuts: matrices of up to 2^20 edges are cut at
multiples of 64 in the order of their nonzeros; rows of up to 512 edges are a
workgroup's where the longest row is known, else, and beyond, they are in pieces."""
import numpy as np
import pytest

from test_gpu_attention import Case, env  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("edges", [63, 64, 65, 127, 128, 129, 511, 512, 513, 576, 577])
@pytest.mark.parametrize("before", [0, 1, 63, 64, 65, 127])
def test_places(env, edges, before):  # noqa: F811
    rng = np.random.RandomState(edges * 3 + before)
    row = np.concatenate([rng.randint(0, 3, before), np.full(edges, 3), rng.randint(4, 9, 130)]).astype(np.int32)
    col = rng.randint(0, 50, len(row)).astype(np.int32)
    for r, c in ((row, col), (col, row)):
        shape = (9, 50) if r is row else (50, 9)
        for case in (Case(env, r, c, shape, 2, 1, 12, "float32", seed=edges), Case(env, r, c, shape, 2, 2, 16, "float16", seed=edges)):
            case.check()
            case.a._max_row = 0
            case.a.transpose()._max_row = 0
            case.check()


def test_several_long_rows_side_by_side(env):  # noqa: F811
    """Rows that end and begin at a cut, one after the other."""
    lengths = [64, 64, 65, 63, 128, 1, 127, 512, 64, 513, 448, 0, 66, 700]
    row = np.repeat(np.arange(len(lengths)), lengths).astype(np.int32)
    col = np.random.RandomState(5).randint(0, 40, len(row)).astype(np.int32)
    for dtype in ("float32", "bfloat16"):
        case = Case(env, row, col, (len(lengths), 40), 4, 2, 8, dtype)
        case.check()
        case.a._max_row = 0
        case.a.transpose()._max_row = 0
        case.check()
