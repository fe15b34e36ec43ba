"""The dense feed-forward operators at their edges on a real MI355X, against 64-bit forms (dense_support.py)."""
import pytest

torch = pytest.importorskip("torch")

import numkong_amd as nk  # noqa: E402
from tests import dense_support as ds  # noqa: E402
from tests.dense_support import normal  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_more_short_rows_than_one_launch_has_tiles_of_64():
    """2^30 rows of 64 values, a window of one vector each (17 GB of results): tiles of 128 rows."""
    rows, width, depth = 1 << 30, 8, 64
    vector = torch.empty(2 * rows + depth, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(1))
    a, w = vector.as_strided((rows, depth), (2, 1)), normal(width, depth, torch.bfloat16, 2).to(DEV)
    y = nk.linear(a, w, activation="relu")
    some = torch.cat([torch.arange(300, device=DEV), rows - 1 - torch.arange(300, device=DEV), torch.randint(0, rows, (4000,), device=DEV, generator=torch.Generator(DEV).manual_seed(3))])
    ds.Linear(a[some].double().cpu(), w.double().cpu(), activation="relu").check(y[some])
