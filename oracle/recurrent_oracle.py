"""Oracle of the gated recurrence, its step, and what stands between two blocks, in 64 bits on the CPU.  TEST INFRASTRUCTURE ONLY.

Written from the definitions in ``include/hstu_recurrent.h``, row after row.  The gradients written out here are pinned against differences
of the forwards.  Beside each result stands the bound that a kernel's roundings give, from the operations it is known to do.
"""

import numpy as np
import torch

from . import output_oracle

F32 = 2.0**-24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(dtype, value):
    """What one rounding of ``value`` to ``dtype`` is off by."""
    return half_step(dtype) * 1.01 * value.abs() + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2


def flat(x):
    return x.detach().flatten(1).double()


def gates(x, decay_gate, input_gate, decay, rate):
    r, i = torch.sigmoid(flat(decay_gate)), torch.sigmoid(flat(input_gate))
    strength = rate * torch.nn.functional.softplus(decay.detach().double(), threshold=50.0)
    z = strength * r
    return strength, r, z, torch.exp(-z), torch.sqrt(-torch.expm1(-2 * z)), i, i * flat(x)


# How far the kernel's gates may be off, in halves of a unit in fp32's last place.  strength: softplus by exp, log1p, one sum, one product (two
# units each for the functions); a sigmoid: product, exponential, sum, reciprocal, a unit each for the instructions.  So z is off by Z of itself, and
# a by Z z + A of itself.  1 - a comes from a series of six terms at most, or, where z is over 1/16, from 1 - a with a's error over 1 - exp(-1/16)
# > 0.06: M of itself, by its root half that in m, and the gated input adds a sigmoid and two products.
Z, A, B = 18, 6, 100


def scan(x, decay_gate, input_gate, decay, offsets, initial=None, rate=8.0):
    """(h [rows, width], final [batch, width], error of h before it is rounded, h in front of every row, its error, sizes of the terms that h in front is
    a sum of).  Every product and sum of the recurrence rounds once more in whatever order the rows are joined: two roundings for each row that a
    term goes through."""
    strength, r, z, a, m, _, u = gates(x, decay_gate, input_gate, decay, rate)
    h, err, before, before_err, before_size = (torch.zeros_like(a) for _ in range(5))
    final = torch.zeros((offsets.numel() - 1, a.shape[1]), dtype=torch.float64) if initial is None else initial.detach().double().clone()
    for b in range(offsets.numel() - 1):
        now = final[b].clone()
        size, e = now.abs(), torch.zeros_like(now)
        for t in range(int(offsets[b]), int(offsets[b + 1])):
            before[t], before_err[t], before_size[t] = now, e, size
            e = a[t] * e + F32 * a[t] * size * (Z * z[t] + A + 2)
            now = a[t] * now + m[t] * u[t]
            size = a[t] * size + (m[t] * u[t]).abs()
            e = e + F32 * (B * (m[t] * u[t]).abs() + size)
            h[t], err[t] = now, e
        final[b] = now
    return h, final, err, before, before_err, before_size


def scan_grad(x, decay_gate, input_gate, decay, offsets, dout=None, dfinal=None, initial=None, rate=8.0):
    """Gradients of x, both gates, decay and initial, each with its bound before the last rounding, as pairs in a dict."""
    strength, s, z, a, m, i, u = gates(x, decay_gate, input_gate, decay, rate)
    _, _, _, before, before_err, before_size = scan(x, decay_gate, input_gate, decay, offsets, initial, rate)
    g = torch.zeros_like(a) if dout is None else flat(dout)
    total, total_err, total_size = (torch.zeros_like(a) for _ in range(3))
    d0, d0_err = (torch.zeros((offsets.numel() - 1, a.shape[1]), dtype=torch.float64) for _ in range(2))
    for b in range(offsets.numel() - 1):
        later = torch.zeros_like(a[0]) if dfinal is None else dfinal[b].double().clone()
        size, e = later.abs(), torch.zeros_like(later)
        for t in range(int(offsets[b + 1]) - 1, int(offsets[b]) - 1, -1):
            total[t], total_size[t] = g[t] + later, g[t].abs() + size
            total_err[t] = e + 2 * F32 * total_size[t]
            later, size = a[t] * total[t], a[t] * total_size[t]
            e = a[t] * total_err[t] + F32 * (Z * z[t] + A + 2) * size
        d0[b], d0_err[b] = later, e
    share = torch.where(m > 0, s / m, torch.zeros_like(m))
    let_in, kept = u * a * a * share, a * s * before
    q = total * (let_in - kept)
    sizes = total_size * (let_in.abs() + a * s * before_size)
    q_err = total_err * (let_in.abs() + kept.abs()) + total.abs() * a * s * before_err + F32 * (3 * Z * z + 2 * B) * sizes
    out = {
        "x": (total * m * i, total_err * m * i + 2 * B * F32 * total_size * m * i),
        "decay_gate": (strength * (1 - s) * q, strength * ((1 - s) * q_err + 2 * Z * F32 * sizes)),  # (s's error for 1 - s: more than its own)
        "input_gate": (total * m * u * (1 - i), m * u.abs() * (total_err + 2 * B * F32 * total_size)),
        "initial": (d0, d0_err),
    }
    # a lane's fp32 sum over at most 64 rows, eight partial sums, and what the terms are off by
    slope = rate * torch.sigmoid(decay.detach().double())
    out["decay"] = (slope * q.sum(0), slope * (q_err.sum(0) + 80 * F32 * sizes.sum(0)))
    return out


def step(states, x, decay_gate, input_gate, decay, slots=None, new_slots=None, rate=8.0):
    """(rows, states, error of both before the rounding of the rows)"""
    rows = x.shape[0]
    slots = torch.arange(rows) if slots is None else slots
    new_slots = slots if new_slots is None else new_slots
    _, _, z, a, m, _, u = gates(x, decay_gate, input_gate, decay, rate)
    h, err, put, put_err = torch.empty_like(a), torch.empty_like(a), states.double().clone(), torch.zeros_like(states, dtype=torch.float64)
    for t in range(rows):
        k = int(slots[t])
        if k < -1 or k >= states.shape[0]:
            h[t] = float("nan")
            continue
        old = states[k].double() if k >= 0 else torch.zeros_like(a[0])
        h[t] = a[t] * old + m[t] * u[t]
        err[t] = F32 * ((Z * z[t] + A + 2) * a[t] * old.abs() + (B + 2) * (m[t] * u[t]).abs())
        if 0 <= int(new_slots[t]) < states.shape[0]:
            put[int(new_slots[t])], put_err[int(new_slots[t])] = h[t], err[t]
    return h, put, err, put_err


ACT = {"none": lambda g: g, "sigmoid": torch.sigmoid, "silu": lambda g: g * torch.sigmoid(g)}


def norm(v, weight, bias, eps, layer_norm):
    if layer_norm:
        v = v - v.mean(-1, keepdim=True)
    v = v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * weight
    return v if bias is None else v + bias


def residual_norm(x, y, gate=None, post_weight=None, post_bias=None, scale=None, pre_weight=None, pre_bias=None, eps=1e-6, layer_norm=False,
                  gate_activation="sigmoid", keep=None):
    """(out, normed), differentiable, in the inputs' type; ``keep``: what dropout leaves of each element, 0 or 1 / (1 - p)."""
    branch = y if post_weight is None else norm(y, post_weight, post_bias, eps, layer_norm)
    if gate is not None:
        branch = ACT[gate_activation](gate) * branch
    if keep is not None:
        branch = branch * keep
    out = x + (branch if scale is None else scale * branch)
    return out, None if pre_weight is None else norm(out, pre_weight, pre_bias, eps, layer_norm)


def kept(ratio, seed, offset, rows, width):
    """Element (row, column): word element % 4 of the generator at counter element / 4."""
    group = np.arange(-(-rows * width // 4), dtype=np.uint64)
    m32 = np.uint64(0xFFFFFFFF)
    ctr = np.stack([group & m32, group >> np.uint64(32), np.full_like(group, offset & 0xFFFFFFFF), np.full_like(group, offset >> 32)], axis=1)
    words = output_oracle.philox4x32_10(ctr, np.array([seed & 0xFFFFFFFF, seed >> 32]))
    keep = words.reshape(-1)[: rows * width].reshape(rows, width) >= np.uint32(int(ratio * 2.0**32))
    return torch.from_numpy(keep).double() / (1 - ratio)


def residual_norm_grad(x, y, gate, post_weight, post_bias, scale, pre_weight, pre_bias, eps, layer_norm, gate_activation, keep, dout, dnormed):
    """(out, normed, gradients by name, bounds by name), all in 64 bits; the bounds before a result's last rounding.

    The bounds count roundings against sizes that stand for a whole row.  A row's norm: v less its mean is off by no more than 24 halves of a unit of the row's largest
    value (sums of 8, over 6 exchanges of lanes and 16 waves, one subtraction), r and the products by 40 of the result; so
    a normed value is off by N = 64 units of r times the row's largest size.  What is computed from it adds the roundings of its own products and of the
    activation (E = 12), all against the largest size in the row."""
    names = ("x", "y", "gate", "post_weight", "post_bias", "scale", "pre_weight", "pre_bias")
    given = dict(zip(names, (x, y, gate, post_weight, post_bias, scale, pre_weight, pre_bias)))
    t = {k: None if v is None else v.detach().double().requires_grad_(True) for k, v in given.items()}
    out, normed = residual_norm(**t, eps=eps, layer_norm=layer_norm, gate_activation=gate_activation, keep=keep)
    n_, e_ = 64 * F32, 12 * F32

    def row(v):
        return v.abs().amax(-1, keepdim=True)

    def inverse(v):
        v = v - v.mean(-1, keepdim=True) if layer_norm else v
        return (v.square().mean(-1, keepdim=True) + eps) ** -0.5

    with torch.no_grad():
        d = {k: None if v is None else v.detach() for k, v in t.items()}
        one = torch.ones((), dtype=torch.float64)
        ry = inverse(d["y"])
        unit_size = row(d["y"]) * ry * (2 if layer_norm else 1)
        n_size = unit_size * row(d["post_weight"]) + (0 if d["post_bias"] is None else row(d["post_bias"])) if post_weight is not None else row(d["y"])
        act = one if gate is None else row(ACT[gate_activation](d["gate"]))
        slope = one if gate is None else one * 1.1 if gate_activation != "sigmoid" else one * 0.25
        keeps = one if keep is None else keep.max() if keep.numel() else one
        scales = one if scale is None else row(d["scale"])
        branch = n_size * act * keeps * scales
        s_err = (n_ + e_) * branch + e_ * row(out)
        bounds = {"out": s_err}
        if pre_weight is not None:
            rs = inverse(out)
            s_unit = row(out) * rs * (2 if layer_norm else 1)
            # an error e of every value of a row moves its norm by 4 e r at most: once the value, and with mean and r all of them
            unit_err = n_ * s_unit + 4 * rs * s_err
            bounds["normed"] = unit_err * row(d["pre_weight"]) + e_ * row(normed)
    got = {}
    if dout is not None or dnormed is not None:
        wanted = [k for k in names if t[k] is not None]
        pairs = [(o, g) for o, g in ((out, dout), (normed, dnormed)) if o is not None and g is not None]
        grads = torch.autograd.grad([o for o, _ in pairs], [t[k] for k in wanted], [g.double() for _, g in pairs], allow_unused=True)
        got = {k: torch.zeros_like(t[k]) if g is None else g for k, g in zip(wanted, grads)}
        with torch.no_grad():
            ds = row(dout.double()) if dout is not None else one * 0
            ds_err = e_ * ds
            if dnormed is not None:
                g = row(dnormed.double()) * row(d["pre_weight"])
                # r (g - unit mean(g unit) - mean g): three terms, none over g max(1, unit^2)
                big = rs * g * (2 + s_unit.square())
                ds = ds + big
                # r is off by unit_err of itself at most as unit is; mean(g unit) twice
                ds_err = ds_err + 3 * n_ * big + rs * g * unit_err * (2 + 4 * s_unit)
                bounds["pre_weight"] = (row(dnormed.double()) * (unit_err + n_ * s_unit)).sum(0)
                bounds["pre_bias"] = n_ * row(dnormed.double()).sum(0)
            elif pre_weight is not None:
                bounds["pre_weight"] = bounds["pre_bias"] = torch.zeros((), dtype=torch.float64)
            bounds["x"] = ds_err
            inner = n_size * act * keeps
            bounds["scale"] = (ds_err * inner + 2 * (n_ + e_) * ds * inner).sum(0)
            dd, dd_err = ds * scales * keeps, ds_err * scales * keeps + e_ * ds * scales * keeps
            bounds["gate"] = (dd_err + 2 * (n_ + e_) * dd) * n_size * slope * 4
            dn, dn_err = dd * act, dd_err * act + e_ * dd * act
            if post_weight is not None:
                bounds["post_weight"] = ((dn_err + 2 * n_ * dn) * unit_size).sum(0)
                bounds["post_bias"] = (dn_err + n_ * dn).sum(0)
                g, g_err = dn * row(d["post_weight"]), dn_err * row(d["post_weight"])
                bounds["y"] = ry * (2 + unit_size.square()) * (g_err + 8 * n_ * g)
            else:
                bounds["y"] = dn_err
    return out.detach(), None if normed is None else normed.detach(), got, bounds
