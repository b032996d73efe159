"""What lies beside the rows and states of the gated recurrence stays as it was, and numbers that the kernels do not take are refused."""

import ctypes

import pytest
import torch

from test_recurrent import abi


def test_rates_that_are_none_c_abi():
    """A rate that is no finite number larger than 0 is refused before a device is touched."""
    L, made = abi()
    ref, at = ctypes.byref, 1 << 20
    both = dict(x=at, decay_gate=at, input_gate=at, x_row_stride=64, decay_gate_row_stride=64, input_gate_row_stride=64, out=at, decay=at, decay_f32=1, rows=100, width=64)
    for rate in (float("inf"), float("nan"), -1.0, 0.0):
        scan = made["HstuRecurrenceArgs"](rate=rate, seq_offsets=at, batch=2, **both)
        assert L.hstu_recurrent_scan(ref(scan), None) == -5, rate
        step = made["HstuRecurrenceStepArgs"](rate=rate, states=at, state_rows=100, state_row_stride=64, **both)
        assert L.hstu_recurrent_step(ref(step), None) == -5, rate


@pytest.mark.gpu
@pytest.mark.parametrize("rate", [float("inf"), 1e300, float("nan"), 1e-60, -8.0])
def test_rates_that_are_none(pkg, dev, rate):
    x = torch.zeros(5, 64, device=dev)
    decay, offsets = torch.zeros(64, device=dev), torch.tensor([0, 5], device=dev)
    with pytest.raises(AssertionError):
        pkg.gated_recurrence(x, x, x, decay, offsets, rate=rate)
    with pytest.raises(AssertionError):
        pkg.gated_recurrence_step(torch.zeros(5, 64, device=dev), x, x, x, decay, rate=rate)
