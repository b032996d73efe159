"""A gated linear recurrence in the attention's place, and what stands between two layers.

``gated_recurrence`` mixes the rows of jagged sequences as ``hstu_mha`` does, at a cost that grows with their length and not its
square: it takes the column slices that the producer (``hstu_compute_uqvk``) leaves, v as its input and q and k as its gates, and its
output goes to the consumer (``hstu_compute_output``).  ``gated_recurrence_step`` is its cached form, one row for each sequence; what it keeps of a
sequence is one state, not a row per position.  ``gated_residual_norm`` joins a block's output to the residual stream (norm, gate, dropout, scale) and
norms the sum for the next block.  The reference has none of them: its layers are attention, and their norms and residuals steps of their own
(``generative_recommenders/ops/pytorch/pt_hstu_linear.py:24-124``, ``pt_layer_norm.py:24-39``).

Device tensors only; hand-written gfx950 kernels behind ``include/hstu_recurrent.h`` (``csrc/hstu_recurrence_kernel.h``,
``csrc/hstu_residual_norm_kernel.h``), called through the native front.  The functions below check what it leaves: tensors
that need a copy first, and calls that are refused.
"""

from typing import Optional, Tuple

import torch

from . import hip_backend, native
from .hstu_attention import _check_forward_only, _require_device
from .hstu_compute import MUL_U_ACTIVATIONS, _WORD64, _dropout_state
from .paged_cache import _check_no_tangents, _index

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _served(out, name: str):
    if out is None:
        raise RuntimeError(f"hstu_recurrent: {name} has no kernel for this call")
    return out


def _rows_like(name: str, t: torch.Tensor, x: torch.Tensor, of: str = "x") -> None:
    _require_device(t, name)
    torch._assert(t.shape == x.shape, f"{name} must have the shape of {of}")
    torch._assert(t.dtype == x.dtype and t.device == x.device, f"{name} must have the type and device of {of}")


def _check_rows(x: torch.Tensor, what: str) -> int:
    """Checks of the tensor that the others are like; the columns of a row."""
    _require_device(x, "x")
    torch._assert(x.dim() in (2, 3), "x must be [rows, width] or [rows, heads, dim]")
    torch._assert(x.dtype in _TYPES, f"{what} takes bf16, fp16 and fp32")
    return x.shape[1] if x.dim() == 2 else x.shape[1] * x.shape[2]


def _flat(x: torch.Tensor) -> torch.Tensor:
    """``x`` with the columns of a row side by side; a copy that gradients flow through where it needs one."""
    dense = (x.shape[-1] == 1 or x.stride(-1) == 1) and (x.dim() == 2 or x.shape[1] == 1 or x.stride(1) == x.shape[2])
    return x if dense and (x.shape[0] == 1 or 0 <= x.stride(0) <= 1 << 24) else x.clone(memory_format=torch.contiguous_format)


def _check_recurrence(x, decay_gate, input_gate, decay, rate: float, what: str) -> int:
    width = _check_rows(x, what)
    _rows_like("decay_gate", decay_gate, x)
    _rows_like("input_gate", input_gate, x)
    _require_device(decay, "decay")
    torch._assert(decay.dim() == 1 and decay.shape[0] == width, "decay must hold one value per column")
    torch._assert(decay.dtype in (x.dtype, torch.float32) and decay.device == x.device, "decay must be float32 or of x's type, on x's device")
    torch._assert(0.0 < torch.tensor(rate, dtype=torch.float32).item() < float("inf"), "rate must be finite and larger than 0")
    return width


def _check_offsets(offsets: torch.Tensor, rows: int) -> None:
    if int(offsets[0]) != 0 or bool((offsets[1:] < offsets[:-1]).any()) or int(offsets[-1]) > rows:
        raise ValueError("hstu_recurrent: seq_offsets decrease, do not begin at 0 or end behind the rows")


def gated_recurrence(
    x: torch.Tensor,
    decay_gate: torch.Tensor,
    input_gate: torch.Tensor,
    decay: torch.Tensor,
    seq_offsets: torch.Tensor,
    initial_state: Optional[torch.Tensor] = None,
    rate: float = 8.0,
    return_state: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(input_gate_t) x_t`` with ``a_t = exp(-rate softplus(decay) sigmoid(decay_gate_t))``
    along each sequence, for every column by itself; returns ``h`` in the shape and type of ``x``, and the last ``h`` of every sequence.

    ``x``, ``decay_gate``, ``input_gate``: ``[L, width]`` or ``[L, H, D]``, bf16, fp16 or fp32, at most 4194240 columns, any distance between rows (the column
    slices of ``hstu_compute_uqvk`` are read in place); ``decay``: ``[width]``, float32 or of x's type.  Rows ``seq_offsets[b]`` up to
    ``seq_offsets[b + 1]`` are sequence ``b``; it begins with ``initial_state[b]`` (``[B, width]``, float32) or with zeros.  ``return_state``: the second
    result is ``[B, width]``, float32, what ``initial_state`` or ``gated_recurrence_step`` goes on from (a sequence without rows keeps its
    own); else None.  h is fp32 throughout and rounded once for each row.  A row of finite ``x`` whose ``decay_gate`` is as low as its type goes leaves
    the state as it is.  Rows behind the last sequence are zero.  Gradients for ``x``, both gates, ``decay`` and ``initial_state``; the backward computes h again, from a state
    for every 64 rows that the forward keeps.

    Caller contract: ``seq_offsets`` begin at 0, do not decrease and do not end behind the rows (``HSTU_HIP_CHECK_CONTRACT=1`` raises where they
    do).  Tensors with forward-mode tangents are refused.
    """
    out = native.front.gated_recurrence(x, decay_gate, input_gate, decay, seq_offsets, initial_state, rate, return_state, False)
    if out is not None:
        return out
    width = _check_recurrence(x, decay_gate, input_gate, decay, rate, "gated_recurrence")
    torch._assert(seq_offsets.dim() == 1 and seq_offsets.numel() >= 2, "seq_offsets must hold one value more than there are sequences")
    batch = seq_offsets.numel() - 1
    seq_offsets = _index(seq_offsets, "seq_offsets", batch + 1, x.device)
    if initial_state is not None:
        _require_device(initial_state, "initial_state")
        torch._assert(initial_state.shape == (batch, width), "initial_state must be [batch, width]")
        torch._assert(initial_state.dtype == torch.float32 and initial_state.device == x.device, "initial_state must be float32, on x's device")
    _check_no_tangents(x, decay_gate, input_gate, decay, initial_state)
    if hip_backend.contract_checks_enabled():
        _check_offsets(seq_offsets, x.shape[0])
    if x.numel() == 0:
        # No rows, or none with columns; the graph, if there is one, goes on, from every input to both results: gradients of zero, and the states' own.
        out = x * decay_gate * input_gate * decay.to(x.dtype).view((1,) + tuple(x.shape[1:]))
        if initial_state is not None:
            out = torch.cat([out, initial_state[:0].to(x.dtype).view((0,) + tuple(x.shape[1:]))])
        if not return_state:
            return out, None
        state = x.new_zeros((batch, width), dtype=torch.float32) if initial_state is None else initial_state
        return out, torch.cat([state, out.flatten(1)[:0].float()])
    initial_state = None if initial_state is None else initial_state.contiguous()
    return _served(native.front.gated_recurrence(_flat(x), _flat(decay_gate), _flat(input_gate), decay.contiguous(), seq_offsets, initial_state, rate, return_state,
                                                 True), "gated_recurrence")


def gated_recurrence_step(
    states: torch.Tensor,
    x: torch.Tensor,
    decay_gate: torch.Tensor,
    input_gate: torch.Tensor,
    decay: torch.Tensor,
    slots: Optional[torch.Tensor] = None,
    new_slots: Optional[torch.Tensor] = None,
    rate: float = 8.0,
) -> torch.Tensor:
    """One row of ``gated_recurrence`` for each of some sequences whose states lie in ``states`` ``[S, width]`` (float32, changed in place).

    Row ``r`` of ``x`` and of the gates goes on from state ``slots[r]`` -- -1: from zeros, a sequence that begins -- and the state after it is put into
    ``new_slots[r]`` (-1: into none, as for a candidate that is only scored).  Without ``slots`` row ``r`` has state ``r``, without ``new_slots`` each goes
    back to where it was read.  Returns the rows, as ``gated_recurrence`` gives them.  A row whose slot is neither -1 nor one of the states comes back NaN
    and is not kept; a state whose new slot is not one of the states is not kept either.  No gradients.

    Caller contract: no state is put twice in a call, and none that another row reads (``HSTU_HIP_CHECK_CONTRACT=1`` raises, and where a slot
    is none of the above); the states' memory is none of the other tensors'.
    """
    out = native.front.gated_recurrence_step(states, x, decay_gate, input_gate, decay, slots, new_slots, rate, False)
    if out is not None:
        return out
    width, rows = _check_recurrence(x, decay_gate, input_gate, decay, rate, "gated_recurrence_step"), x.shape[0]
    _require_device(states, "states")
    torch._assert(states.dim() == 2 and states.shape[1] == width, "states must be [states, width]")
    torch._assert(states.dtype == torch.float32 and states.device == x.device, "states must be float32, on x's device")
    torch._assert((width <= 1 or states.stride(1) == 1) and (states.shape[0] <= 1 or states.stride(0) >= width),
                  "states must lie row by row, their columns side by side: they are changed in place")
    torch._assert(slots is not None or states.shape[0] == rows, "without slots there is one state for each row")
    slots = None if slots is None else _index(slots, "slots", rows, x.device)
    new_slots = None if new_slots is None else _index(new_slots, "new_slots", rows, x.device)
    _check_forward_only(states, x, decay_gate, input_gate, decay)
    _check_no_tangents(states, x, decay_gate, input_gate, decay)
    if x.numel() == 0:
        return torch.empty_like(x)
    if hip_backend.contract_checks_enabled():
        _check_slots(states.shape[0], rows, slots, new_slots, x.device)
    return _served(native.front.gated_recurrence_step(states, _flat(x), _flat(decay_gate), _flat(input_gate), decay.contiguous(), slots, new_slots, rate, True),
                   "gated_recurrence_step")


def _check_slots(count: int, rows: int, slots: Optional[torch.Tensor], new_slots: Optional[torch.Tensor], device: torch.device) -> None:
    """The caller contract of a step's slots (synchronises)."""
    read = torch.arange(rows, device=device) if slots is None else slots.long()
    put = read if new_slots is None else new_slots.long()
    for s in (read, put):
        if bool(((s < -1) | (s >= count)).any()):
            raise ValueError("hstu_recurrent: a slot is neither -1 nor one of the states")
    kept = put[put >= 0]
    if kept.unique().numel() != kept.numel():
        raise ValueError("hstu_recurrent: a state is put twice")
    owner = torch.full((count,), -1, dtype=torch.long, device=device)
    owner[kept] = torch.arange(rows, device=device)[put >= 0]
    at = read.clamp(min=0)
    if count and bool(((read >= 0) & (owner[at] >= 0) & (owner[at] != torch.arange(rows, device=device))).any()):
        raise ValueError("hstu_recurrent: a state is put that another row reads")


def gated_residual_norm(
    x: torch.Tensor,
    y: torch.Tensor,
    gate: Optional[torch.Tensor] = None,
    post_weight: Optional[torch.Tensor] = None,
    post_bias: Optional[torch.Tensor] = None,
    scale: Optional[torch.Tensor] = None,
    pre_weight: Optional[torch.Tensor] = None,
    pre_bias: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    layer_norm: bool = False,
    gate_activation: str = "sigmoid",
    dropout_ratio: float = 0.0,
    training: bool = False,
    seed: Optional[Tuple[int, int]] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``out = x + scale * dropout(act(gate) * norm(y))`` and ``norm(out)`` for the block that comes next; returns both.

    ``x`` (the residual stream), ``y`` (a block's output), ``gate``: ``[L, width]`` or ``[L, H, D]``, bf16, fp16 or fp32, any distance between rows;
    parameters ``[width]`` of the same type, shared by the rows.  ``norm(v)`` is ``v / sqrt(mean(v^2) + eps) * weight + bias`` over a whole row, with
    ``layer_norm`` of ``v`` less its mean; ``eps`` may be 0 (a row whose mean square is 0 in fp32 is NaN then).  ``post_*`` are those of the norm behind the block
    (left out without ``post_weight``), ``pre_*`` those of the one in front of the next (without ``pre_weight`` the second result is None).  ``act`` is ``gate_activation``: ``"none"``, ``"sigmoid"`` or ``"silu"``;
    without ``gate`` and ``scale`` both are 1.  Everything in fp32, each result rounded once: the second norm takes the sum as it is, not rounded.
    Dropout runs when ``training`` and ``dropout_ratio > 0``, from the Philox stream of ``seed = (seed, offset)`` or of the device's default generator, as in
    ``norm_mul_dropout``; its mask is not stored but computed again for the backward.  (A captured call drops the same elements at every replay.)
    Gradients for all tensors; nothing but the inputs is saved.  Tensors with forward-mode tangents are refused.
    """
    params = (post_weight, post_bias, scale, pre_weight, pre_bias)
    drops = training and dropout_ratio != 0.0
    ratio = word_seed = word_offset = 0
    if drops:
        _check_residual(x, y, gate, params, eps, gate_activation, dropout_ratio)  # before the generator moves on
        ratio, word_seed, word_offset = _dropout_state(dropout_ratio, training, x.numel(), x.device, seed)
        word_seed, word_offset = word_seed & _WORD64, word_offset & _WORD64
    act = MUL_U_ACTIVATIONS.get(gate_activation, -1)
    out = native.front.gated_residual_norm(x, y, gate, post_weight, post_bias, scale, pre_weight, pre_bias, eps, layer_norm, act, ratio, word_seed, word_offset)
    if out is not None:
        return out
    if not drops:
        _check_residual(x, y, gate, params, eps, gate_activation, dropout_ratio)
    if x.numel() == 0:
        out = x + (y if gate is None else y * gate)  # nothing in them; the graph, if there is one, goes on, to gradients of zero for the parameters too
        for p in (p for p in params if p is not None):
            out = out * p.view((1,) + tuple(x.shape[1:]))
        return out, None if pre_weight is None else out * 1
    params = tuple(None if p is None else p.contiguous() for p in params)
    return _served(native.front.gated_residual_norm(_flat(x), _flat(y), None if gate is None else _flat(gate), *params, eps, layer_norm, act, ratio, word_seed,
                                                    word_offset), "gated_residual_norm")


def _check_residual(x, y, gate, params, eps: float, gate_activation: str, dropout_ratio: float) -> None:
    width = _check_rows(x, "gated_residual_norm")
    _rows_like("y", y, x)
    if gate is not None:
        _rows_like("gate", gate, x)
    torch._assert(gate_activation in MUL_U_ACTIVATIONS, "gate_activation must be none, sigmoid or silu")
    torch._assert(0.0 <= torch.tensor(eps, dtype=torch.float32).item() < float("inf"), "eps must be finite and not negative")
    torch._assert(0.0 <= dropout_ratio < 1.0, "dropout_ratio must be below 1")
    for p, name in zip(params, ("post_weight", "post_bias", "scale", "pre_weight", "pre_bias")):
        if p is not None:
            _require_device(p, name)
            torch._assert(p.dim() == 1 and p.shape[0] == width, f"{name} must hold one value per column")
            torch._assert(p.dtype == x.dtype and p.device == x.device, f"{name} must have the type and device of x")
    torch._assert(params[0] is not None or params[1] is None, "post_bias without post_weight")
    torch._assert(params[3] is not None or params[4] is None, "pre_bias without pre_weight")
    _check_no_tangents(x, y, gate, *params)
    if width > 8192:
        raise NotImplementedError("rows are at most 8192 columns wide")
