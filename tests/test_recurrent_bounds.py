"""What lies beside the rows and states of the gated recurrence stays as it was, and numbers that the kernels do not take are refused."""

import ctypes

import pytest
import torch

from test_recurrent import BF, F32, FP, abi, scan_case


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


class Fenced:
    """A tensor of ``shape`` in the middle of a larger one of a fixed value, whose rows outside it have to stay as they are."""

    FENCE, MARK = 64, 7.0  # more rows than a wave has

    def __init__(self, shape, dtype, dev, inner=None):
        rows, width = shape
        self.whole = torch.full((rows + 2 * self.FENCE, width), self.MARK, dtype=dtype, device=dev)
        self.inner = self.whole[self.FENCE : self.FENCE + rows]

    def check(self, what):
        torch.cuda.synchronize()
        assert bool((self.whole[: self.FENCE] == self.MARK).all()), f"rows in front of {what} were written"
        assert bool((self.whole[self.FENCE + self.inner.shape[0] :] == self.MARK).all()), f"rows behind {what} were written"


def among_nan(t, dev):
    """``t`` as a column slice of a wider tensor that is NaN everywhere else, with rows of it in front and behind."""
    whole = torch.full((t.shape[0] + 128, t.shape[1] + 24), float("nan"), dtype=t.dtype, device=dev)
    inner = whole[64 : 64 + t.shape[0], 8 : 8 + t.shape[1]]
    inner.copy_(t)
    return inner


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("width", [1, 33, 64, 130])
@pytest.mark.parametrize("lengths, behind", [([1], 0), ([15], 0), ([17], 1), ([63, 2], 0), ([600, 0, 1, 577], 3), ([513, 530, 49], 0)], ids=lambda v: str(v))
def test_nothing_beside_the_rows(pkg, dev, dtype, width, lengths, behind):
    """Tiles with fewer rows than they have room for, blocks with fewer columns: their other rows and columns are neither read nor written."""
    L, made = abi()
    case, dout, dfinal = scan_case(lengths, width, dtype, seed=5, behind=behind)
    rows, batch = case["x"].shape[0], len(lengths)
    x, r, i, d = (among_nan(t, dev) for t in (case["x"], case["decay_gate"], case["input_gate"], dout))
    decay, offsets, initial, dfinal = (t.to(dev).contiguous() for t in (case["decay"], case["offsets"], case["initial"], dfinal))
    like = lambda n=rows, t=dtype: Fenced((n, width), t, dev)  # noqa: E731
    out, final = like(), like(batch, F32)
    a = made["HstuRecurrenceArgs"](x=x.data_ptr(), decay_gate=r.data_ptr(), input_gate=i.data_ptr(), x_row_stride=x.stride(0), decay_gate_row_stride=r.stride(0),
                                   input_gate_row_stride=i.stride(0), out=out.inner.data_ptr(), decay=decay.data_ptr(), decay_f32=1, rate=8.0,
                                   seq_offsets=offsets.data_ptr(), seq_offsets_i64=int(offsets.dtype == torch.int64), batch=batch, rows=rows, width=width,
                                   dtype={BF: 0, FP: 1, F32: 3}[dtype], initial_state=initial.data_ptr(), final_state=final.inner.data_ptr(), saved=1 << 20)
    ref, stream = ctypes.byref, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    saved = Fenced((L.hstu_recurrent_scan_saved_bytes(ref(a)) // 4, 1), F32, dev)
    scratch = Fenced((L.hstu_recurrent_scan_workspace_bytes(ref(a)), 1), torch.uint8, dev)
    a.saved, a.workspace, a.workspace_bytes = saved.inner.data_ptr(), scratch.inner.data_ptr(), scratch.inner.numel()
    print("forward", dtype, width, lengths, behind, flush=True)
    assert L.hstu_recurrent_scan(ref(a), stream) == 0
    for name, t in (("out", out), ("the states", final), ("what is saved", saved), ("the workspace", scratch)):
        t.check(name)
    more = Fenced((L.hstu_recurrent_scan_bwd_workspace_bytes(ref(a)), 1), torch.uint8, dev)
    dx, dr, di, dinitial, ddecay = like(), like(), like(), like(batch, F32), like(1, F32)
    g = made["HstuRecurrenceGrads"](d_out=d.data_ptr(), d_out_row_stride=d.stride(0), d_final_state=dfinal.data_ptr(), d_x=dx.inner.data_ptr(), d_decay_gate=dr.inner.data_ptr(),
                                    d_input_gate=di.inner.data_ptr(), d_decay=ddecay.inner.data_ptr(), d_initial_state=dinitial.inner.data_ptr(),
                                    workspace=more.inner.data_ptr(), workspace_bytes=more.inner.numel())
    print("backward", flush=True)
    assert L.hstu_recurrent_scan_bwd(ref(a), ref(g), stream) == 0
    for name, t in (("dx", dx), ("dr", dr), ("di", di), ("the states' gradient", dinitial), ("the decays' gradient", ddecay), ("the backward's workspace", more)):
        t.check(name)
    leaves = [t.to(dev).clone().requires_grad_() for t in (case["x"], case["decay_gate"], case["input_gate"], case["decay"], case["initial"])]
    want = pkg.gated_recurrence(*leaves[:4], offsets, leaves[4], return_state=True)
    grads = torch.autograd.grad(want, leaves, [dout.to(dev), dfinal])
    for name, got, t in zip(("out", "state", "dx", "dr", "di", "d decay", "d initial"), (out, final, dx, dr, di, ddecay, dinitial), tuple(want) + grads):
        assert bool(torch.isfinite(got.inner).all()), f"{name} took up something that is beside the rows"
        assert torch.equal(got.inner.reshape(t.shape), t.detach()), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths", [[1], [3], [70], [600, 5, 513]], ids=lambda v: str(v))
def test_rows_that_are_one_row(pkg, dev, dtype, lengths):
    """One row alone, and rows that are all the same memory (inputs and incoming gradients that were broadcast), give what copies of them give."""
    width = 96
    case, dout, dfinal = scan_case(lengths, width, dtype, seed=9)
    offsets, decay, initial, dfinal = (t.to(dev) for t in (case["offsets"], case["decay"], case["initial"], dfinal))
    rows = case["x"].shape[0]
    broadcast = [t[:1].to(dev).expand(rows, width) for t in (case["x"], case["decay_gate"], case["input_gate"], dout)]

    def gradients(copy):
        x, r, i, d = (torch.cat([t, t])[: t.shape[0]].contiguous() if copy else t for t in broadcast)
        if copy and rows == 1:  # a row's distance from the next that is not zero
            x, r, i, d = (torch.cat([t, torch.zeros_like(t)]).as_strided((1, width), (width, 1)) for t in (x, r, i, d))
        leaves = [t.detach().requires_grad_() for t in (x, r, i, decay, initial)]
        out, state = pkg.gated_recurrence(*leaves[:4], offsets, leaves[4], return_state=True)
        return [out, state] + list(torch.autograd.grad((out, state), leaves, (d, dfinal)))

    a = gradients(False)
    b = gradients(True)
    for name, x, y in zip(("out", "state", "dx", "dr", "di", "d decay", "d initial"), a, b):
        assert torch.equal(x, y), name
    # the decays' gradient in 64 bits: it is the sum over rows of the gates', dr / (rate softplus(decay) (1 - s)), times rate sigmoid(decay)
    leaf = decay.double().cpu().requires_grad_()
    x, r, i, d = (t.double().cpu() for t in broadcast)
    z = 8.0 * torch.nn.functional.softplus(leaf) * torch.sigmoid(r)
    keep, into = torch.exp(-z), torch.sqrt(-torch.expm1(-2 * z)) * torch.sigmoid(i) * x
    total, begin = 0.0, 0
    for b_, n in enumerate(lengths):
        h = initial[b_].double().cpu()
        for t in range(begin, begin + n):
            h = keep[t] * h + into[t]
            total = total + (h * d[t]).sum()
        begin += n
        total = total + (h * dfinal[b_].double().cpu()).sum()
    want = torch.autograd.grad(total, leaf)[0]
    # rounding aside (a few hundred half steps of fp32 of what is summed up), not a multiple of a row's share too much
    assert (a[5].cpu().double() - want).abs().max() <= 2e-3 * want.abs().max(), "d decay"


@pytest.mark.gpu
def test_widths_past_32_bits(pkg, dev):
    """A row of 2^32 + 64 columns is refused, not taken for one of 64."""
    width = (1 << 32) + 64
    x = torch.empty((1, width), dtype=BF, device=dev)
    offsets = torch.tensor([0, 1], device=dev)
    with pytest.raises(NotImplementedError):
        pkg.gated_recurrence(x, x, x, x[0], offsets)
    states = torch.empty((1, 1), device=dev).expand(1, width)
    with pytest.raises((NotImplementedError, AssertionError)):
        pkg.gated_recurrence_step(states, x, x, x, x[0])


@pytest.mark.gpu
def test_a_step_in_inference_mode(pkg, dev):
    x, w = torch.randn((3, 32), device=dev), torch.zeros(32, device=dev)
    want = torch.zeros((3, 32), device=dev)
    out = pkg.gated_recurrence_step(want, x, x, x, w)
    with torch.inference_mode():
        states = torch.zeros((3, 32), device=dev)
        assert torch.equal(pkg.gated_recurrence_step(states, x, x, x, w), out) and torch.equal(states, want)
