"""A recurrent layer beside the attention's, and what stands between two layers, as cases that can be timed.

A case is a dict of plain values; ``op`` says which call of the user's it is:

* ``scan``        the gated linear recurrence over jagged sequences, as a prefill; with ``states`` it goes on from states and returns them
* ``scan_train``  the same forward and backward: its output, the gradients of its three inputs, of the decays and, with ``states``,
                  of the states that it went on from
* ``step``        one row for each sequence: states read from their slots, the new ones put into others
* ``norm``        norm of a block's output, gate, dropout, scale, residual, and the norm in front of the next block
* ``norm_train``  the same forward and backward: both outputs, the gradients of its three inputs and of every parameter

Where ``own`` is false the operators are computed in their plain form.  The shape of a case (lengths) depends on the case
alone, through ``shape_seed``; values on the seed that ``prepare`` gets.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
RATE = 8.0
# Every field that not all cases name, with the value that stands for "not used".
DEFAULTS = {
    "dtype": "bf16", "batch": 1, "lo": 1, "hi": 1, "heads": 4, "dim": 128, "fused": False, "states": False, "slots": 0, "decay32": True,
    "gate": "sigmoid", "post": True, "pre": True, "scaled": False, "layer_norm": False, "biases": False, "dropout": 0.0, "shape_seed": 0,
}


def _full(case):
    return dict(DEFAULTS, **case)


def listed():
    return [
        # One step of generation for a small batch, the states of 256 sequences at hand.  Latency and nothing else.
        dict(name="step", op="step", batch=32, slots=256, shape_seed=1),
        # Candidates of a serving micro-batch, each a row behind a history of its own: eight heads, the second type.
        dict(name="step_many", op="step", dtype="fp16", batch=2000, heads=8, slots=6000, shape_seed=2),
        # A few new rows for each of 32 sequences, from their states to the next ones.
        dict(name="scan_chunk", op="scan", batch=32, lo=1, hi=9, states=True, shape_seed=3),
        # A ragged prefill as the producer leaves it: input and gates column slices of one buffer, the second type, decays of that type.
        dict(name="scan_prefill_fp16", op="scan", dtype="fp16", batch=96, lo=20, hi=1023, heads=8, dim=64, fused=True, decay32=False, shape_seed=4),
        # A few heavy users with very long histories: little to do in parallel but the columns and the history itself.
        dict(name="scan_long", op="scan", batch=5, lo=8000, hi=16000, heads=8, states=True, shape_seed=5),
        # A training batch of ordinary histories.
        dict(name="scan_train", op="scan_train", batch=48, lo=200, hi=2048, shape_seed=6),
        # The largest: long histories, eight heads.
        dict(name="scan_train_long", op="scan_train", batch=32, lo=1024, hi=8192, heads=8, shape_seed=1006),
        # ... and the operator tests' third type on a small odd batch of odd width, with states and their gradients.
        dict(name="scan_train_fp32", op="scan_train", dtype="fp32", batch=16, lo=1, hi=257, heads=1, dim=100, states=True, shape_seed=7),
        # One step of generation between two layers.
        dict(name="norm_step", op="norm", batch=32, lo=1, hi=1, shape_seed=8),
        # A prefill in the second type: layer norms with biases, a SiLU gate, block output and gate column slices of one buffer.
        dict(name="norm_prefill_fp16", op="norm", dtype="fp16", batch=96, lo=20, hi=1023, gate="silu", layer_norm=True, biases=True, fused=True,
             shape_seed=9),
        # A training batch with dropout and a learned scale of the residual branch.
        dict(name="norm_train", op="norm_train", batch=48, lo=200, hi=2048, scaled=True, dropout=0.1, shape_seed=6),
        # The largest: long histories, eight heads, layer norms with biases.
        dict(name="norm_train_long", op="norm_train", batch=32, lo=1024, hi=8192, heads=8, layer_norm=True, biases=True, shape_seed=1006),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    while True:
        op = rng.choice(["scan", "scan", "scan_train", "scan_train", "scan_train", "step", "norm", "norm_train", "norm_train"])
        c = dict(op=op, shape_seed=rng.randrange(1 << 20), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        c["heads"] = rng.choice([1, 2, 3, 4, 4, 8])
        c["dim"] = rng.choice([128, 128, 64, 32, 100, 33])
        if op == "step":
            c["batch"] = _log_int(rng, 1, 4096)
            c["slots"] = 2 * c["batch"] + rng.randrange(100)
        else:
            c["batch"] = _log_int(rng, 1, 256)
            c["hi"] = _log_int(rng, 1, 16384)
            c["lo"] = max(1, int(c["hi"] * rng.choice([0.0, 0.06, 0.5, 1.0])))
            c["fused"] = not op.endswith("train") and rng.random() < 0.5
        if op.startswith("norm"):
            c["gate"] = rng.choice(["sigmoid", "silu", "none", ""])
            c["post"] = rng.random() < 0.8
            c["pre"] = rng.random() < 0.8
            c["scaled"] = rng.random() < 0.5
            c["layer_norm"] = rng.random() < 0.5
            c["biases"] = rng.random() < 0.5
            c["dropout"] = rng.choice([0.0, 0.0, 0.1, 0.3])
        else:
            c["states"] = rng.random() < 0.5
            c["decay32"] = rng.random() < 0.7
        values = int(_lengths(_full(c)).sum()) * c["heads"] * c["dim"] * (2 if c["dtype"] == "fp32" else 1)
        if values <= (3.2e7 if c.get("dropout") else 1.5e8):
            return c


# ---- shapes and work ----------------------------------------------------------------------------------------------------


def _lengths(c):
    """Lengths of the sequences."""
    rng = np.random.RandomState(c["shape_seed"])
    return rng.randint(c["lo"], c["hi"] + 1, size=c["batch"]).astype(np.int64)


def work(case):
    c = _full(case)
    es = 4 if c["dtype"] == "fp32" else 2
    width = c["heads"] * c["dim"]
    values = (c["batch"] if c["op"] == "step" else int(_lengths(c).sum())) * width
    held = 4 * c["batch"] * width
    if c["op"] == "step":
        return {"bytes": 4.0 * es * values + 2.0 * held + 4 * width, "flops": 25.0 * values}
    if c["op"] == "scan":
        return {"bytes": 4.0 * es * values + (2.0 * held if c["states"] else 0.0), "flops": 25.0 * values}
    if c["op"] == "scan_train":
        return {"bytes": 8.0 * es * values + (2.0 * held if c["states"] else 0.0), "flops": 70.0 * values}
    ins, outs = 2 + (c["gate"] != ""), 1 + c["pre"]
    if c["op"] == "norm":
        return {"bytes": float(es * values * (ins + outs)), "flops": 20.0 * values}
    return {"bytes": float(es * values * 2 * (ins + outs)), "flops": 60.0 * values}


# ---- inputs -------------------------------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(c, rows, count, dtype, g):
    """``count`` tensors [rows, heads, dim]; ``fused``: column slices of one wider buffer, as the producer of u, v, q, k leaves them."""
    h, d = c["heads"], c["dim"]
    if c["fused"]:
        buf = torch.randn((rows, (count + 1) * h * d), generator=g, device="cuda").to(dtype)
        return [t.view(rows, h, d) for t in torch.split(buf, h * d, dim=1)[1:]]
    return [torch.randn((rows, h, d), generator=g, device="cuda").to(dtype) for _ in range(count)]


def prepare(case, seed):
    c = _full(case)
    g = _generator(seed)
    dt = DTYPES[c["dtype"]]
    n = _lengths(c)
    width = c["heads"] * c["dim"]
    rows = c["batch"] if c["op"] == "step" else int(n.sum())
    s = {"case": c}
    if c["op"] in ("scan", "scan_train", "step"):
        s["x"], s["decay_gate"], s["input_gate"] = _rows(c, rows, 3, dt, g)
        # decays as such layers are begun with: a row with an open gate keeps 0.9 to 0.999 of the state
        keep = 0.9 + 0.099 * torch.rand(width, generator=g, device="cuda", dtype=torch.float64)
        decay = torch.log(torch.expm1(-torch.log(keep) / RATE))
        s["decay"] = decay.float() if c["decay32"] else decay.to(dt)
        if c["op"] == "step":
            s["states"] = torch.randn((c["slots"], width), generator=g, device="cuda")
            order = torch.randperm(c["slots"], generator=g, device="cuda")
            s["slots"], s["new_slots"] = order[:rows].contiguous(), order[rows : 2 * rows].contiguous()
            return s
        s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(n)])).cuda()
        s["longest"] = int(n.max())
        s["initial"] = torch.randn((c["batch"], width), generator=g, device="cuda") if c["states"] else None
        if c["op"] == "scan_train":
            s["dout"] = torch.randn((rows, c["heads"], c["dim"]), generator=g, device="cuda").to(dt)
            s["dfinal"] = torch.randn((c["batch"], width), generator=g, device="cuda") if c["states"] else None
            s["leaves"] = [s[k].requires_grad_() for k in ("x", "decay_gate", "input_gate", "decay", "initial") if s[k] is not None]
        return s
    y = _rows(c, rows, 2, dt, g)
    s["y"] = y[0].flatten(1)
    s["gate"] = y[1].flatten(1) if c["gate"] != "" else None
    s["x"] = torch.randn((rows, width), generator=g, device="cuda").to(dt)
    for name, there in (("post", c["post"]), ("pre", c["pre"])):
        s[name + "_weight"] = (1 + 0.1 * torch.randn(width, generator=g, device="cuda")).to(dt) if there else None
        s[name + "_bias"] = (0.1 * torch.randn(width, generator=g, device="cuda")).to(dt) if there and c["biases"] else None
    s["scale"] = (0.5 + 0.1 * torch.randn(width, generator=g, device="cuda")).to(dt) if c["scaled"] else None
    s["dropout_seed"] = (int(seed) * 7919 + 17, int(seed) % 1000)
    if c["op"] == "norm_train":
        s["dout"] = torch.randn((rows, width), generator=g, device="cuda").to(dt)
        s["dnormed"] = torch.randn((rows, width), generator=g, device="cuda").to(dt) if c["pre"] else None
        s["leaves"] = [s[k].requires_grad_() for k in NORM_LEAVES if s[k] is not None]
    return s


NORM_LEAVES = ("x", "y", "gate", "post_weight", "post_bias", "scale", "pre_weight", "pre_bias")


# ---- plain form ---------------------------------------------------------------------------------------------------------


def _gates(s):
    """Everything of a row that does not depend on the rows in front of it, in 32 bits: sigmoid of the decay gate, kept share,
    square root of what is let in, sigmoid of the input gate, and the gated input."""
    x, r, i = (s[k].detach().flatten(1).float() for k in ("x", "decay_gate", "input_gate"))
    decay = s["decay"].detach().double()
    strength = (RATE * torch.log1p(torch.exp(decay))).float()
    sr, si = 1 / (1 + torch.exp(-r)), 1 / (1 + torch.exp(-i))
    z = strength * sr
    return strength, sr, torch.exp(-z), torch.sqrt(-torch.expm1(-2 * z)), si, si * x


def _places(s):
    """Place of every row in its sequence, and how many rows come after it there."""
    offsets, rows = s["offsets"], s["x"].shape[0]
    of = torch.repeat_interleave(torch.arange(offsets.numel() - 1, device=offsets.device), offsets[1:] - offsets[:-1], output_size=rows)
    at = torch.arange(rows, device=offsets.device)
    return of, at - offsets[of], offsets[of + 1] - 1 - at


def _scan(a, b, place, longest):
    """h_t = a_t h_{t-1} + b_t from nothing in front of place 0, by doubling; and the products of the a's up to each row."""
    step = 1
    while step < longest:
        there = (place[step:] >= step).view(-1, 1)
        more_b = torch.where(there, a[step:] * b[:-step], torch.zeros_like(b[step:]))
        more_a = torch.where(there, a[:-step], torch.ones_like(a[step:]))
        b, a = torch.cat([b[:step], b[step:] + more_b]), torch.cat([a[:step], a[step:] * more_a])
        step *= 2
    return b, a


def _plain_scan(s):
    c, dtype, shape = s["case"], s["x"].dtype, s["x"].shape
    train = c["op"] == "scan_train"
    strength, sr, a, m, si, u = _gates(s)
    of, place, left = _places(s)
    h, kept = _scan(a, m * u, place, s["longest"])
    if c["states"]:
        h = h + kept * s["initial"].detach()[of]
    out = {"out": h.view(shape).to(dtype)}
    if c["states"]:
        out["final"] = h[s["offsets"][1:] - 1]
    if not train:
        return out
    first = (place == 0).view(-1, 1)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    before = torch.where(first, s["initial"].detach()[of] if c["states"] else torch.zeros_like(h), before)
    g = s["dout"].flatten(1).float()
    if c["states"]:
        g = g + torch.where((left == 0).view(-1, 1), s["dfinal"][of], torch.zeros_like(g))
    ahead = torch.cat([a[1:], torch.zeros_like(a[:1])])
    g = _scan(ahead.flip(0), g.flip(0), left.flip(0), s["longest"])[0].flip(0)
    share = torch.where(m > 0, sr / m, torch.zeros_like(m))
    q = g * (u * a * a * share - a * sr * before)
    out["dx"] = (g * m * si).view(shape).to(dtype)
    out["ddecay_gate"] = (strength * (1 - sr) * q).view(shape).to(dtype)
    out["dinput_gate"] = (g * m * u * (1 - si)).view(shape).to(dtype)
    decay = s["decay"].detach()
    out["ddecay"] = (RATE / (1 + torch.exp(-decay.double())) * q.sum(dim=0, dtype=torch.float64)).to(decay.dtype)
    if c["states"]:
        out["dinitial"] = (a * g)[s["offsets"][:-1]]
    return out


def _plain_step(s):
    _, _, a, m, _, u = _gates(s)
    h = a * s["states"][s["slots"]] + m * u
    s["states"][s["new_slots"]] = h
    return {"out": h.view(s["x"].shape).to(s["x"].dtype), "states": s["states"]}


def _kept(s):
    """What dropout leaves of each element, 0 or 1 / (1 - p): word c % 4 of Philox4x32-10 of (element / 4, offset) under the seed."""
    rows, width = s["x"].shape
    p = s["case"]["dropout"]
    low = 0xFFFFFFFF
    seed, offset = s["dropout_seed"]
    group = torch.arange(-(-rows * width // 4), device="cuda")
    c0, c1, c2, c3 = group & low, group >> 32, torch.full_like(group, offset & low), torch.full_like(group, offset >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], dim=1).flatten()[: rows * width].view(rows, width)
    return (words >= int(p * 2.0**32)).float() / (1 - p)


def _norm(c, x):
    """x with mean 0 (layer norm) and mean square 1, and the factor that did the latter."""
    if c["layer_norm"]:
        x = x - x.mean(dim=-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
    return x * r, r


def _norm_grad(c, d, unit, r):
    d = d - unit * (d * unit).mean(dim=-1, keepdim=True)
    if c["layer_norm"]:
        d = d - d.mean(dim=-1, keepdim=True)
    return d * r


def _plain_norm(s):
    c, dtype = s["case"], s["x"].dtype
    f = {k: s[k].detach().float() if s[k] is not None else None for k in NORM_LEAVES}
    n, y_unit, y_r = f["y"], None, None
    if c["post"]:
        y_unit, y_r = _norm(c, f["y"])
        n = y_unit * f["post_weight"] + (f["post_bias"] if c["biases"] else 0)
    sigma = 1 / (1 + torch.exp(-f["gate"])) if c["gate"] in ("sigmoid", "silu") else None
    act = {"": lambda: 1.0, "none": lambda: f["gate"], "sigmoid": lambda: sigma, "silu": lambda: f["gate"] * sigma}[c["gate"]]()
    kept = _kept(s) if c["dropout"] > 0 else 1.0
    branch = n * act * kept
    total = f["x"] + (branch * f["scale"] if c["scaled"] else branch)
    out = {"out": total.to(dtype)}
    if c["pre"]:
        t_unit, t_r = _norm(c, total)
        out["normed"] = (t_unit * f["pre_weight"] + (f["pre_bias"] if c["biases"] else 0)).to(dtype)
    if c["op"] != "norm_train":
        return out

    def column(x):
        return x.sum(dim=0, dtype=torch.float64).to(dtype)

    d = s["dout"].float()
    if c["pre"]:
        dn = s["dnormed"].float()
        out["dpre_weight"] = column(dn * t_unit)
        if c["biases"]:
            out["dpre_bias"] = column(dn)
        d = d + _norm_grad(c, dn * f["pre_weight"], t_unit, t_r)
    out["dx"] = d.to(dtype)
    if c["scaled"]:
        out["dscale"] = column(d * branch)
        d = d * f["scale"]
    d = d * kept
    if c["gate"] != "":
        slope = {"none": lambda: 1.0, "sigmoid": lambda: sigma * (1 - sigma), "silu": lambda: sigma * (1 + f["gate"] * (1 - sigma))}[c["gate"]]()
        out["dgate"] = (d * n * slope).to(dtype)
        d = d * act
    if c["post"]:
        out["dpost_weight"] = column(d * y_unit)
        if c["biases"]:
            out["dpost_bias"] = column(d)
        d = _norm_grad(c, d * f["post_weight"], y_unit, y_r)
    out["dy"] = d.to(dtype)
    return out


def _plain(s):
    op = s["case"]["op"]
    return _plain_step(s) if op == "step" else _plain_scan(s) if op.startswith("scan") else _plain_norm(s)


# ---- the framework's calls ----------------------------------------------------------------------------------------------


def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _own(s):
    c, pkg = s["case"], _package()
    if c["op"] == "step":
        out = pkg.gated_recurrence_step(s["states"], s["x"], s["decay_gate"], s["input_gate"], s["decay"], slots=s["slots"], new_slots=s["new_slots"], rate=RATE)
        return {"out": out, "states": s["states"]}
    if c["op"].startswith("scan"):
        h, final = pkg.gated_recurrence(s["x"], s["decay_gate"], s["input_gate"], s["decay"], s["offsets"], initial_state=s["initial"], rate=RATE,
                                        return_state=c["states"])
        out = {"out": h.detach()}
        if c["states"]:
            out["final"] = final.detach()
        if c["op"] == "scan_train":
            got = torch.autograd.grad((h, final) if c["states"] else (h,), s["leaves"], (s["dout"], s["dfinal"]) if c["states"] else (s["dout"],))
            out.update(zip(("dx", "ddecay_gate", "dinput_gate", "ddecay", "dinitial"), got))
        return out
    o, normed = pkg.gated_residual_norm(s["x"], s["y"], s["gate"], post_weight=s["post_weight"], post_bias=s["post_bias"], scale=s["scale"],
                                        pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], eps=EPS, layer_norm=c["layer_norm"],
                                        gate_activation=c["gate"] or "none", dropout_ratio=c["dropout"], training=c["dropout"] > 0, seed=s["dropout_seed"])
    out = {"out": o.detach()}
    if c["pre"]:
        out["normed"] = normed.detach()
    if c["op"] == "norm_train":
        got = torch.autograd.grad((o, normed) if c["pre"] else (o,), s["leaves"], (s["dout"], s["dnormed"]) if c["pre"] else (s["dout"],))
        out.update(zip(["d" + k for k in NORM_LEAVES if s[k] is not None], got))
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------


def _exact_gates(s):
    x, r, i = (s[k].detach().double().flatten(1) for k in ("x", "decay_gate", "input_gate"))
    decay = s["decay"].detach().double()
    strength = RATE * torch.nn.functional.softplus(decay, threshold=40.0)
    open_ = torch.sigmoid(r)
    a = torch.exp(-strength * open_)
    return x, torch.sigmoid(i), open_, strength, a, torch.sqrt(-torch.expm1(-2 * strength * open_))


def _exact_scan(s):
    """Row after row, all sequences side by side."""
    c = s["case"]
    x, gi, gr, strength, a, m = _exact_gates(s)
    rows, width = x.shape
    n = (s["offsets"][1:] - s["offsets"][:-1])
    order = torch.argsort(n, descending=True)
    counts = torch.bincount(n.cpu(), minlength=s["longest"] + 1)
    going = (c["batch"] - torch.cumsum(counts, 0)).tolist()  # sequences longer than t
    first = s["offsets"][:-1][order]
    initial = s["initial"].detach().double()[order] if c["states"] else torch.zeros((c["batch"], width), dtype=torch.float64, device="cuda")
    h, before = torch.empty_like(x), torch.empty_like(x)
    b = m * gi * x
    now = initial.clone()
    for t in range(s["longest"]):
        k = going[t]
        at = first[:k] + t
        before[at] = now[:k]
        now[:k] = now[:k] * a[at] + b[at]
        h[at] = now[:k]
    back = torch.empty_like(order)
    back[order] = torch.arange(c["batch"], device="cuda")
    out = {"out": h.view(s["x"].shape)}
    if c["states"]:
        out["final"] = now[back]
    if c["op"] != "scan_train":
        return out
    g = s["dout"].double().flatten(1)
    later = s["dfinal"].double()[order].clone() if c["states"] else torch.zeros_like(initial)
    total = torch.empty_like(g)
    for t in range(s["longest"] - 1, -1, -1):
        k = going[t]
        at = first[:k] + t
        now = g[at] + later[:k]
        total[at] = now
        later[:k] = a[at] * now
    dm = total * gi * x
    # 1 - a^2 = m^2, so dm / da = -a / m; a falls by a * strength for each unit that the gate opens
    da = total * before - torch.where(m > 0, dm * a / m, torch.zeros_like(m))
    out["dx"] = (total * m * gi).view(s["x"].shape)
    out["ddecay_gate"] = (-da * a * strength * gr * (1 - gr)).view(s["x"].shape)
    out["dinput_gate"] = (total * m * x * gi * (1 - gi)).view(s["x"].shape)
    out["ddecay"] = -(da * a * gr).sum(0) * RATE * torch.sigmoid(s["decay"].detach().double())
    if c["states"]:
        out["dinitial"] = later[back]
    return out


def _exact_step(s):
    x, gi, _, _, a, m = _exact_gates(s)
    h = a * s["states"].double()[s["slots"]] + m * gi * x
    states = s["states"].double().clone()
    states[s["new_slots"]] = h
    return {"out": h.view(s["x"].shape), "states": states}


def _exact_kept(s):
    """The generator in unsigned 64-bit integers on the host."""
    rows, width = s["x"].shape
    seed, offset = s["dropout_seed"]
    n = -(-rows * width // 4)
    words = np.empty((n, 4), dtype=np.uint32)
    m32 = np.uint64(0xFFFFFFFF)
    for start in range(0, n, 1 << 20):
        group = np.arange(start, min(n, start + (1 << 20)), dtype=np.uint64)
        ctr = [group & m32, group >> np.uint64(32), np.full_like(group, offset & 0xFFFFFFFF), np.full_like(group, offset >> 32)]
        key = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
            ctr = [(b >> np.uint64(32)) ^ ctr[1] ^ np.uint64(key[0]), b & m32, (a >> np.uint64(32)) ^ ctr[3] ^ np.uint64(key[1]), a & m32]
            key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
        for k in range(4):
            words[start : start + len(group), k] = ctr[k]
    p = s["case"]["dropout"]
    keep = words.reshape(-1)[: rows * width].reshape(rows, width) >= np.uint32(int(p * 2.0**32))
    return torch.from_numpy(keep).cuda().double() / (1 - p)


def _exact_norm(s):
    """Forward from the definition; gradients by automatic differentiation of it in 64 bits."""
    c = s["case"]
    train = c["op"] == "norm_train"
    t = {k: s[k].detach().double().requires_grad_(train) if s[k] is not None else None for k in NORM_LEAVES}

    def norm(v, weight, bias):
        if c["layer_norm"]:
            v = v - v.sum(-1, keepdim=True) / v.shape[-1]
        v = v / torch.sqrt(v.square().sum(-1, keepdim=True) / v.shape[-1] + EPS) * weight
        return v if bias is None else v + bias

    branch = norm(t["y"], t["post_weight"], t["post_bias"]) if c["post"] else t["y"]
    if c["gate"]:
        branch = branch * {"none": lambda v: v, "sigmoid": torch.sigmoid, "silu": lambda v: v * torch.sigmoid(v)}[c["gate"]](t["gate"])
    if c["dropout"] > 0:
        branch = branch * _exact_kept(s)
    total = t["x"] + (branch if t["scale"] is None else branch * t["scale"])
    normed = norm(total, t["pre_weight"], t["pre_bias"]) if c["pre"] else None
    out = {"out": total.detach()}
    if c["pre"]:
        out["normed"] = normed.detach()
    if train:
        names = [k for k in NORM_LEAVES if t[k] is not None]
        got = torch.autograd.grad((total, normed) if c["pre"] else (total,), [t[k] for k in names],
                                  (s["dout"].double(), s["dnormed"].double()) if c["pre"] else (s["dout"].double(),))
        out.update(zip(["d" + k for k in names], got))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = s["case"]["op"]
    return _exact_step(s) if op == "step" else _exact_scan(s) if op.startswith("scan") else _exact_norm(s)
