"""The gated recurrence and the norms between two blocks at numbers and sizes where a result can be lost: rows that there are not, gates that are open, calls of no
rows, numbers that are none."""

import pytest

from test_recurrent import BF, F32, FP, NORMS, check_norm, norm_case


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 7])
@pytest.mark.parametrize("width", [512, 513, 520, 1000, 1024, 1030])
@pytest.mark.parametrize("kind", range(len(NORMS)))
def test_norms_without_an_eps(pkg, dev, kind, width, rows):
    """A group of lanes behind the last row has nothing to add to the parameters' gradients, whatever a norm makes of it."""
    check_norm(pkg, dev, *norm_case(rows, width, [BF, F32, FP][(kind + rows) % 3], seed=rows, **NORMS[kind]), eps=0.0, **NORMS[kind])
