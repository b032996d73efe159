"""The gated recurrence and the norms between two blocks at numbers and sizes where a result can be lost: rows that there are not, gates that are open, calls of no
rows, numbers that are none."""

import ctypes

import pytest
import torch

from test_recurrent import BF, F32, FP, NORMS, abi, check_norm, norm_case


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 7])
@pytest.mark.parametrize("width", [512, 513, 520, 1000, 1024, 1030])
@pytest.mark.parametrize("kind", range(len(NORMS)))
def test_norms_without_an_eps(pkg, dev, kind, width, rows):
    """A group of lanes behind the last row has nothing to add to the parameters' gradients, whatever a norm makes of it."""
    check_norm(pkg, dev, *norm_case(rows, width, [BF, F32, FP][(kind + rows) % 3], seed=rows, **NORMS[kind]), eps=0.0, **NORMS[kind])


def test_an_eps_that_is_none_c_abi():
    """An eps that is negative or not finite is refused before a device is touched; 0 is one."""
    L, made = abi()
    ref, at = ctypes.byref, 1 << 20
    norm = lambda **kw: made["HstuResidualNormArgs"](**dict(dict(x=at, y=at, x_row_stride=64, y_row_stride=64, out=at, rows=100, width=64, dtype=0), **kw))  # noqa: E731
    grads = made["HstuResidualNormGrads"](d_out=at, d_x=at, d_out_row_stride=64)
    for eps in (-1e-6, float("inf"), -float("inf"), float("nan")):
        assert L.hstu_recurrent_residual_norm(ref(norm(eps=eps)), None) == -5, eps
        assert L.hstu_recurrent_residual_norm_bwd(ref(norm(eps=eps)), ref(grads), None) == -5, eps
    assert L.hstu_recurrent_residual_norm(ref(norm(eps=0.0, rows=0)), None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [-1e-6, float("inf"), 1e300, float("nan")])
def test_an_eps_that_is_none(pkg, dev, eps):
    for rows in (5, 0):
        x, w = torch.zeros((rows, 64), device=dev), torch.ones(64, device=dev)
        for more in ({}, dict(dropout_ratio=0.5, training=True)):
            before = torch.cuda.default_generators[0].get_offset()
            with pytest.raises(AssertionError):
                pkg.gated_residual_norm(x, x, post_weight=w, eps=eps, **more)
            assert torch.cuda.default_generators[0].get_offset() == before
