"""The gated recurrence, its step, and what stands between two blocks, against their definitions in 64 bits."""

import ctypes
import os
import re
import subprocess

import pytest
import torch

from oracle import recurrent_oracle as oracle
from oracle.recurrent_oracle import rounded

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def offsets_of(lengths, dtype=torch.int64):
    return torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=dtype)


def scan_case(lengths, width, dtype, seed=0, states=True, behind=0, decay_dtype=F32, spread=1.0, heads=None):
    """x, gates, decay, offsets, initial, and gradients of both results; ``behind``: rows behind the last sequence."""
    g = torch.Generator().manual_seed(seed)
    offs = offsets_of(lengths)
    rows = int(offs[-1]) + behind
    shape = (rows, width) if heads is None else (rows, heads, width // heads)
    x, r, i, dout = ((torch.randn(shape, generator=g) * spread).to(dtype) for _ in range(4))
    keep = 0.5 + 0.4999 * torch.rand(width, generator=g, dtype=torch.float64) ** 0.25  # from quick to very slow columns
    decay = torch.log(torch.expm1(-torch.log(keep) / 8.0)).to(decay_dtype)
    initial, dfinal = (torch.randn((len(lengths), width), generator=g) if states else None for _ in range(2))
    return dict(x=x, decay_gate=r, input_gate=i, decay=decay, offsets=offs, initial=initial), dout, dfinal


def within(got, want, bound, what, dtype=F32):
    got = got.detach().cpu().double().flatten(1) if got.dim() > 1 else got.detach().cpu().double()
    off = (got - want).abs()
    limit = bound + rounded(dtype, want)
    bad = ~(off <= limit)
    assert not bad.any(), f"{what}: off by {float((off / limit).nan_to_num(1e9)[bad].max()):.3g} of the bound at {bad.nonzero()[0].tolist()}"


# ---- on the host --------------------------------------------------------------------------------------------------------


def lib():
    from generative_recommenders_amd import build

    if not os.path.exists(build.RECURRENT_LIB_PATH):
        import __graft_entry__

        __graft_entry__.build()
    return ctypes.CDLL(build.RECURRENT_LIB_PATH), build


def abi():
    """The library and its argument structures, read from the header."""
    L, build = lib()
    header = re.sub(r"/\*.*?\*/", "", open(os.path.join(build.INCLUDE, "hstu_recurrent.h")).read(), flags=re.S)
    types = {"int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32, "float": ctypes.c_float, "double": ctypes.c_double, "uint64_t": ctypes.c_uint64}
    made = {}
    for body, name in re.findall(r"typedef struct \w+ \{(.*?)\} (\w+);", header, flags=re.S):
        fields = []
        for line in body.split(";"):
            if line.strip():
                kind, names = line.strip().removeprefix("const ").split(None, 1)
                for n in names.split(","):
                    fields.append((n.strip().lstrip("* "), ctypes.c_void_p if "*" in line else types[kind]))
        made[name] = type(name, (ctypes.Structure,), {"_fields_": fields})
    for name in re.findall(r"size_t (\w+)\(", header):
        getattr(L, name).restype = ctypes.c_size_t
    return L, made


def test_exports_are_the_headers():
    L, build = lib()
    header = open(os.path.join(build.INCLUDE, "hstu_recurrent.h")).read()
    declared = set(re.findall(r"\b(hstu_recurrent_\w+)\s*\(", header))
    exported = set(re.findall(r" T (hstu_recurrent_\w+)", subprocess.run(["nm", "-D", build.RECURRENT_LIB_PATH], capture_output=True, text=True, check=True).stdout))
    assert declared == exported and L.hstu_recurrent_version() >= 100
    L.hstu_recurrent_last_error.restype = ctypes.c_char_p
    assert L.hstu_recurrent_last_error() == b""


def test_statuses_of_the_c_abi():
    """Calls that the library refuses before it touches a device; pointers are looked at, never followed."""
    L, made = abi()
    ref, at = ctypes.byref, 1 << 20
    for name in ("scan", "step", "residual_norm"):
        assert getattr(L, f"hstu_recurrent_{name}")(None, None) == -1
    assert L.hstu_recurrent_scan_bwd(None, None, None) == -1 and L.hstu_recurrent_residual_norm_bwd(None, None, None) == -1
    good = dict(x=at, decay_gate=at, input_gate=at, x_row_stride=64, decay_gate_row_stride=64, input_gate_row_stride=64, out=at, decay=at, decay_f32=1, rate=8.0,
                seq_offsets=at, batch=2, rows=100, width=64, dtype=0)
    scan = lambda **kw: made["HstuRecurrenceArgs"](**dict(good, **kw))  # noqa: E731
    for status, change in ((-1, dict(x=0)), (-1, dict(out=0)), (-1, dict(decay=0)), (-1, dict(seq_offsets=0)), (-2, dict(dtype=2)), (-4, dict(x=at + 1)), (-4, dict(decay=at + 2)),
                           (-5, dict(batch=0)), (-5, dict(width=0)), (-5, dict(rows=-1)), (-5, dict(rate=0.0)), (-5, dict(x_row_stride=-64))):
        assert L.hstu_recurrent_scan(ref(scan(**change)), None) == status, change
    grads = made["HstuRecurrenceGrads"](d_out=at, d_out_row_stride=64, d_x=at, workspace=at, workspace_bytes=1 << 40)
    assert L.hstu_recurrent_scan_bwd(ref(scan()), None, None) == -1
    grads.d_out_row_stride = -1
    assert L.hstu_recurrent_scan_bwd(ref(scan()), ref(grads), None) == -5
    step_good = dict(x=at, decay_gate=at, input_gate=at, x_row_stride=64, decay_gate_row_stride=64, input_gate_row_stride=64, out=at, decay=at, decay_f32=1, rate=8.0,
                     states=at, state_rows=10, state_row_stride=64, rows=10, width=64, dtype=0)
    step = lambda **kw: made["HstuRecurrenceStepArgs"](**dict(step_good, **kw))  # noqa: E731
    for status, change in ((-1, dict(x=0)), (-1, dict(states=0)), (-2, dict(dtype=9)), (-4, dict(states=at + 2)), (-5, dict(width=-1)), (-5, dict(state_rows=-1)), (0, dict(rows=0))):
        assert L.hstu_recurrent_step(ref(step(**change)), None) == status, change
    norm_good = dict(x=at, y=at, x_row_stride=64, y_row_stride=64, out=at, eps=1e-6, rows=100, width=64, dtype=0)
    norm = lambda **kw: made["HstuResidualNormArgs"](**dict(norm_good, **kw))  # noqa: E731
    for status, change in ((-1, dict(y=0)), (-1, dict(out=0)), (-1, dict(pre_weight=at)), (-1, dict(post_bias=at)), (-2, dict(dtype=7)), (-4, dict(y=at + 1)), (-5, dict(width=0)),
                           (-5, dict(dropout_ratio=1.0)), (-5, dict(dropout_ratio=float("nan"))), (-5, dict(gate_activation=3)), (-6, dict(width=8193)), (0, dict(rows=0))):
        assert L.hstu_recurrent_residual_norm(ref(norm(**change)), None) == status, change
    g = made["HstuResidualNormGrads"](d_out=at, d_x=at, d_out_row_stride=64, d_post_weight=at)
    assert L.hstu_recurrent_residual_norm_bwd(ref(norm(post_weight=at)), ref(g), None) == -1  # no workspace
    g.workspace, g.workspace_bytes = at, 16
    assert L.hstu_recurrent_residual_norm_bwd(ref(norm(post_weight=at)), ref(g), None) == -5
    assert L.hstu_recurrent_residual_norm_bwd(ref(norm(rows=0)), ref(g), None) == -5


def test_python_refusals_on_the_host(pkg):
    x, w = torch.zeros(4, 8), torch.zeros(8)
    offs = torch.tensor([0, 4])
    with pytest.raises(AssertionError):
        pkg.gated_recurrence(x, x, x, w, offs)
    with pytest.raises(AssertionError):
        pkg.gated_recurrence_step(x, x, x, x, w)
    with pytest.raises(AssertionError):
        pkg.gated_residual_norm(x, x)
    with pytest.raises(AssertionError):
        pkg.gated_residual_norm(x, x, dropout_ratio=0.5, training=True)


@pytest.mark.parametrize("states", [False, True])
def test_oracle_gradients_against_differences(states):
    case, dout, dfinal = scan_case([3, 0, 5, 1], 4, torch.float64, seed=3, states=states, decay_dtype=torch.float64)
    if states:
        case["initial"], dfinal = case["initial"].double(), dfinal.double()
    got = oracle.scan_grad(**case, dout=dout, dfinal=dfinal)

    def loss(name, at, by):
        c = dict(case)
        c[name] = case[name].clone()
        c[name].view(-1)[at] += by
        h, final, *_ = oracle.scan(**c)
        return (h * dout).sum() + ((final * dfinal).sum() if states else 0.0)

    for name in ("x", "decay_gate", "input_gate", "decay") + (("initial",) if states else ()):
        for at in range(case[name].numel()):
            d = (loss(name, at, 1e-5) - loss(name, at, -1e-5)) / 2e-5
            # differences of third order: (1e-5)^2 times third derivatives of order one
            assert abs(float(d - got[name][0].reshape(-1)[at])) < 1e-7, (name, at)


@pytest.mark.parametrize("layer_norm", [False, True])
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
def test_oracle_norm_against_differences(layer_norm, act):
    g = torch.Generator().manual_seed(5)
    t = [torch.randn(3, 6, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(3)]
    p = [torch.randn(6, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(5)]
    keep = oracle.kept(0.3, 7, 2, 3, 6)
    assert 0 < int((keep == 0).sum()) < 18
    torch.autograd.gradcheck(lambda *a: oracle.residual_norm(*a, eps=1e-3, layer_norm=layer_norm, gate_activation=act, keep=keep), (*t, *p))


# ---- on the GPU ---------------------------------------------------------------------------------------------------------


def run_scan(pkg, dev, case, dout=None, dfinal=None, grads=True, change=lambda k, t: t):
    """Results and gradients of the framework's call, by name."""
    t = {k: None if v is None else change(k, v.to(dev)) for k, v in case.items()}
    leaves = {k: t[k].detach().requires_grad_(True) for k in ("x", "decay_gate", "input_gate", "decay", "initial") if grads and t[k] is not None}
    t.update(leaves)
    want_state = dfinal is not None or not grads
    out, final = pkg.gated_recurrence(t["x"], t["decay_gate"], t["input_gate"], t["decay"], t["offsets"], initial_state=t["initial"], return_state=want_state)
    got = {}
    if grads:
        pairs = [(o, g.to(dev)) for o, g in ((out, dout), (final, dfinal)) if g is not None]
        got = dict(zip(leaves, torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [g for _, g in pairs])))
    torch.cuda.synchronize()
    return out, final, got


def check_scan(pkg, dev, case, dout, dfinal, grads=True, **kw):
    out, final, got = run_scan(pkg, dev, case, dout, dfinal, grads, **kw)
    dtype, end = case["x"].dtype, int(case["offsets"][-1])
    h, last, err, *_ = oracle.scan(**case)
    within(out, h, err, "out", dtype)
    assert out.shape == case["x"].shape and out.dtype == dtype and bool((out[end:] == 0).all())
    if final is not None:
        last_err = torch.stack([err[e - 1] if e > s else torch.zeros_like(err[0]) for s, e in zip(case["offsets"][:-1].tolist(), case["offsets"][1:].tolist())])
        within(final, last, last_err, "final")
    if not grads:
        return
    want = oracle.scan_grad(**case, dout=dout, dfinal=dfinal)
    for name in ("x", "decay_gate", "input_gate"):
        within(got[name], *want[name], "d" + name, dtype)
        assert bool((got[name][end:] == 0).all())
    within(got["decay"], *want["decay"], "ddecay", case["decay"].dtype)
    if case["initial"] is not None:
        within(got["initial"], *want["initial"], "dinitial")


LENGTHS = [[1], [5, 0, 3], [0, 0, 7, 0], [64], [65, 1, 63, 128], [200, 3, 0, 300, 17], [1] * 40, [127, 129, 255, 257], [700]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: "-".join(map(str, v[:5])))
def test_scan(pkg, dev, dtype, lengths):
    case, dout, dfinal = scan_case(lengths, 72, dtype, seed=len(lengths), behind=3)
    check_scan(pkg, dev, case, dout, dfinal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("width", [1, 2, 3, 33, 64, 127, 128, 130, 200, 257, 512])
def test_scan_widths(pkg, dev, dtype, width):
    case, dout, dfinal = scan_case([70, 3, 150], width, dtype, seed=width, states=width % 2 == 0, decay_dtype=dtype if width % 3 == 0 else F32)
    check_scan(pkg, dev, case, dout, dfinal)
    check_scan(pkg, dev, case, None, None, grads=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths", [[4700], [2047, 0, 2050, 3, 4500], [64] * 70, [5, 0, 9, 1, 0, 0, 2] * 300, [0] * 1500 + [3000] + [0] * 1500],
                         ids=["one", "some", "whole-tiles", "many", "many-without-rows"])
def test_scan_over_many_tiles(pkg, dev, dtype, lengths):
    """Tiles that go back over groups of others, sequences that begin and end at their borders, more sequences than a workgroup has threads."""
    case, dout, dfinal = scan_case(lengths, 6, dtype, seed=21, behind=200)
    check_scan(pkg, dev, case, dout, dfinal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_scan_reads_slices_in_place(pkg, dev, dtype):
    """Column slices of one buffer, odd distances between rows, addresses off every boundary, heads, rows that repeat, int32 offsets."""
    case, dout, dfinal = scan_case([90, 40, 1], 96, dtype, seed=9, heads=3)

    def slices(pad):
        def change(k, t):
            if k == "offsets":
                return t.int()
            if k not in ("x", "decay_gate", "input_gate"):
                return t
            buf = torch.full((t.shape[0], 96 + 2 * pad), float("nan"), dtype=dtype, device=t.device)
            buf[:, pad : pad + 96] = t.flatten(1)
            return buf[:, pad : pad + 96].view(t.shape)

        return change

    for pad in (8, 4, 3, 1):
        check_scan(pkg, dev, case, dout, dfinal, change=slices(pad))
    check_scan(pkg, dev, case, dout, dfinal, change=lambda k, t: t if k == "offsets" or t.dim() < 3 else t.transpose(1, 2).contiguous().transpose(1, 2))
    case["x"] = case["x"][:1].expand(131, 3, 32)
    check_scan(pkg, dev, case, dout.contiguous(), None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_gates_at_their_ends(pkg, dev, dtype):
    """Lowest and highest values, infinities of both signs: a shut decay gate with a shut input gate leaves the state, bit by bit."""
    case, dout, dfinal = scan_case([30, 20], 40, dtype, seed=2)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    case["decay_gate"][3:9], case["input_gate"][3:9] = low, low
    case["decay_gate"][10], case["input_gate"][11] = high, high
    case["decay_gate"][32], case["input_gate"][33] = float("inf"), float("inf")
    case["decay_gate"][34:36], case["input_gate"][36] = -float("inf"), -float("inf")
    check_scan(pkg, dev, case, dout, dfinal)
    out, final, _ = run_scan(pkg, dev, case, grads=False)
    assert all(torch.equal(out[2], out[t]) for t in range(3, 9))
    case["decay_gate"][:], case["input_gate"][:] = low, low
    out, final, _ = run_scan(pkg, dev, case, grads=False)
    assert torch.equal(final.cpu(), case["initial"])


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[9, 12, 7], [300, 200, 700]], ids=["short", "long"])
def test_what_is_not_finite_stays_where_it_is(pkg, dev, lengths):
    case, dout, dfinal = scan_case(lengths, 70, BF, seed=4)
    clean, clean_state, clean_grad = run_scan(pkg, dev, case, dout, dfinal)
    at = lengths[0] + 3
    case["x"][at, 5], case["x"][at + 1, 8], case["decay_gate"][at + 2, 11] = float("inf"), float("nan"), float("nan")
    out, state, grad = run_scan(pkg, dev, case, dout, dfinal)
    hurt = torch.zeros(sum(lengths), 70, dtype=torch.bool)
    for k, c in enumerate((5, 8, 11)):
        hurt[at + k : lengths[0] + lengths[1], c] = True
    assert torch.equal(~torch.isfinite(out.cpu()), hurt)
    assert torch.equal(out.cpu()[~hurt], clean.cpu()[~hurt])
    others = torch.ones(70, dtype=torch.bool)
    others[[5, 8, 11]] = False
    second = slice(lengths[0], lengths[0] + lengths[1])
    for name in ("x", "decay_gate", "input_gate"):
        got, want = grad[name].cpu(), clean_grad[name].cpu()
        assert torch.equal(got[:, others], want[:, others])
        assert torch.equal(got[: lengths[0]], want[: lengths[0]]) and torch.equal(got[second.stop :], want[second.stop :])
    assert torch.equal(state.cpu()[[0, 2]], clean_state.cpu()[[0, 2]])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_step(pkg, dev, dtype):
    case, *_ = scan_case([23], 72, dtype, seed=6, heads=2)
    g = torch.Generator().manual_seed(1)
    states = torch.randn((40, 72), generator=g)
    order = torch.randperm(40, generator=g)
    slots, new = order[:23].clone(), order[23:40].repeat(2)[:23].clone()
    slots[[3, 7]], new[17:], new[5] = -1, -1, -1
    slots[9], new[2] = 40, 1000
    args = {k: case[k].to(dev) for k in ("x", "decay_gate", "input_gate", "decay")}
    for s, n in ((slots, new), (slots.int(), new), (slots[:23], None), (None, None)):
        held = states if s is not None else states[:23]
        here = held.clone().to(dev)
        out = pkg.gated_recurrence_step(here, **args, slots=None if s is None else s.to(dev), new_slots=None if n is None else n.to(dev))
        h, put, err, put_err = oracle.step(held, *[case[k] for k in ("x", "decay_gate", "input_gate", "decay")], slots=s, new_slots=n)
        torch.cuda.synchronize()
        unknown = torch.isnan(h)
        assert torch.equal(torch.isnan(out.cpu()).flatten(1), unknown) and out.shape == case["x"].shape
        within(out.cpu().flatten(1)[~unknown[:, 0]], h[~unknown[:, 0]], err[~unknown[:, 0]], "step", dtype)
        within(here, put, put_err, "states")
        untouched = put_err.sum(1) == 0
        assert torch.equal(here.cpu()[untouched], held[untouched])


@pytest.mark.gpu
def test_results_are_the_same_from_call_to_call(pkg, dev):
    """Whichever tile comes first, and whatever was in the scratch memory."""
    case, dout, dfinal = scan_case([9000, 40, 3000], 256, BF, seed=22)
    first = run_scan(pkg, dev, case, dout, dfinal)
    for _ in range(5):
        junk = torch.full((1 << 22,), 0x7FC00001, dtype=torch.int32, device=dev)
        del junk
        again = run_scan(pkg, dev, case, dout, dfinal)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1]) and all(torch.equal(first[2][k], again[2][k]) for k in first[2])


@pytest.mark.gpu
def test_a_prefill_and_steps_are_the_whole(pkg, dev):
    """Rows one at a time from the states of a prefill, and a chunk of them at once, give what the whole sequences give."""
    lengths, tail = [30, 1, 77], 9
    case, *_ = scan_case([n + tail for n in lengths], 64, F32, seed=8)
    t = {k: v.to(dev) for k, v in case.items()}
    offs = case["offsets"]
    whole, end = pkg.gated_recurrence(t["x"], t["decay_gate"], t["input_gate"], t["decay"], t["offsets"], t["initial"], return_state=True)
    first = torch.cat([torch.arange(int(offs[b]), int(offs[b]) + n) for b, n in enumerate(lengths)]).to(dev)
    rest = torch.cat([torch.arange(int(offs[b]) + n, int(offs[b + 1])) for b, n in enumerate(lengths)]).to(dev)
    rows = lambda at: (t["x"][at], t["decay_gate"][at], t["input_gate"][at], t["decay"])  # noqa: E731
    a, state = pkg.gated_recurrence(*rows(first), offsets_of(lengths).to(dev), t["initial"], return_state=True)
    b, state_b = pkg.gated_recurrence(*rows(rest), offsets_of([tail] * 3).to(dev), state, return_state=True)
    stepped = state.clone()
    c = torch.stack([pkg.gated_recurrence_step(stepped, *rows(rest.view(3, tail)[:, k])) for k in range(tail)], dim=1).flatten(0, 1)
    h, last, err, *_ = oracle.scan(**case)
    for got, at in ((whole, torch.arange(int(offs[-1]))), (a, first.cpu()), (b, rest.cpu()), (c, rest.cpu())):
        within(got, h[at], 2 * err[at], "rows", F32)
    for got in (end, state_b, stepped):
        within(got, last, 2 * err[offs[1:] - 1], "states")


NORMS = [
    dict(gate="sigmoid", params="00000"), dict(gate="sigmoid", params="10010"), dict(gate="silu", params="11011", layer_norm=True), dict(gate=None, params="00111"),
    dict(gate="none", params="11111"), dict(gate="silu", params="10110", dropout=0.25), dict(gate=None, params="00000", dropout=0.5),
    dict(gate="sigmoid", params="11111", layer_norm=True, dropout=0.1),
]


def norm_case(rows, width, dtype, gate="sigmoid", params="10010", seed=0, heads=None, **_):
    g = torch.Generator().manual_seed(seed)
    shape = (rows, width) if heads is None else (rows, heads, width // heads)
    x, y, z, dout, dnormed = ((torch.randn(shape, generator=g) * s + m).to(dtype) for s, m in ((1, 0), (2, 0.5), (1, 0), (1, 0), (1, 0)))
    made = [(1 + 0.2 * torch.randn(width, generator=g)).to(dtype) if p == "1" else None for p in params]
    names = ("post_weight", "post_bias", "scale", "pre_weight", "pre_bias")
    return dict(x=x, y=y, gate=z if gate else None, **dict(zip(names, made))), dout, dnormed if made[3] is not None else None


def check_norm(pkg, dev, case, dout, dnormed, gate="sigmoid", layer_norm=False, dropout=0.0, eps=1e-6, change=lambda k, t: t, **_):
    dtype = case["x"].dtype
    rows, width = case["x"].flatten(1).shape
    t = {k: None if v is None else change(k, v.to(dev)).detach().requires_grad_(True) for k, v in case.items()}
    seed = (0x123456789ABCDEF, 0x100000007)
    out, normed = pkg.gated_residual_norm(**t, eps=eps, layer_norm=layer_norm, gate_activation=gate or "none", dropout_ratio=dropout, training=True, seed=seed)
    leaves = {k: v for k, v in t.items() if v is not None}
    pairs = [(o, g.to(dev)) for o, g in ((out, dout), (normed, dnormed)) if g is not None]
    got = dict(zip(leaves, torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [g for _, g in pairs])))
    with torch.no_grad():
        again = pkg.gated_residual_norm(**t, eps=eps, layer_norm=layer_norm, gate_activation=gate or "none", dropout_ratio=dropout, training=True, seed=seed)
    torch.cuda.synchronize()
    assert torch.equal(again[0], out) and (normed is None or torch.equal(again[1], normed))
    flat = {k: None if v is None else v.flatten(1) if v.dim() == 3 else v for k, v in case.items()}
    keep = oracle.kept(dropout, *seed, rows, width) if dropout else None
    want, want_normed, grads, bounds = oracle.residual_norm_grad(**flat, eps=eps, layer_norm=layer_norm, gate_activation=gate or "none", keep=keep,
                                                                 dout=dout.flatten(1) if dout is not None else None, dnormed=dnormed.flatten(1) if dnormed is not None else None)
    assert out.shape == case["x"].shape and out.dtype == dtype
    within(out, want, bounds["out"], "out", dtype)
    if normed is not None:
        within(normed, want_normed, bounds["normed"], "normed", dtype)
    else:
        assert want_normed is None
    for k in leaves:
        assert got[k].shape == case[k].shape and got[k].dtype == dtype
        within(got[k], grads[k], bounds[k], "d" + k, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("kind", range(len(NORMS)))
def test_norm(pkg, dev, dtype, kind):
    check_norm(pkg, dev, *norm_case(37, 128, dtype, seed=kind, **NORMS[kind]), **NORMS[kind])


@pytest.mark.gpu
@pytest.mark.parametrize("width", [1, 2, 7, 8, 33, 64, 72, 100, 136, 256, 264, 511, 512, 520, 1000, 1024, 2048, 2056, 4096, 4104, 8191, 8192])
def test_norm_widths(pkg, dev, width):
    kind = NORMS[[2, 5, 7][width % 3]]
    dtype = [BF, F32, FP][width % 5 % 3]
    check_norm(pkg, dev, *norm_case(5 if width > 600 else 150, width, dtype, seed=width, **kind), **kind)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_norm_reads_slices_in_place(pkg, dev, dtype):
    kind = NORMS[7]
    case, dout, dnormed = norm_case(50, 96, dtype, seed=3, heads=3, **kind)

    def slices(pad):
        def change(k, t):
            if t.dim() == 1:
                buf = torch.full((96 + 2 * pad,), float("nan"), dtype=dtype, device=t.device)
                buf[pad : pad + 96] = t
                return buf[pad : pad + 96]
            buf = torch.full((t.shape[0], 96 + 2 * pad), float("nan"), dtype=dtype, device=t.device)
            buf[:, pad : pad + 96] = t.flatten(1)
            return buf[:, pad : pad + 96].view(t.shape)

        return change

    for pad in (8, 4, 1):
        check_norm(pkg, dev, case, dout, dnormed, change=slices(pad), **kind)
    check_norm(pkg, dev, case, dout, dnormed, change=lambda k, t: t if t.dim() < 3 else t.transpose(1, 2).contiguous().transpose(1, 2), **kind)


@pytest.mark.gpu
def test_gradients_of_one_result_alone(pkg, dev):
    case, dout, dnormed = norm_case(20, 64, F32, seed=5, **NORMS[4])
    check_norm(pkg, dev, case, dout, None, **NORMS[4])
    check_norm(pkg, dev, case, None, dnormed, **NORMS[4])
    case, dout, dfinal = scan_case([20, 90], 64, F32, seed=5)
    check_scan(pkg, dev, case, dout, None)
    check_scan(pkg, dev, case, None, dfinal)


@pytest.mark.gpu
def test_rows_at_the_ends_of_a_type(pkg, dev):
    """Rows of zeros, of one value (a variance of nothing), of the smallest and the largest numbers; an infinity or NaN stays in its row."""
    case, dout, dnormed = norm_case(12, 128, F32, params="11011", seed=6)
    case["y"][1], case["x"][2], case["y"][3] = 0, 0, 7.0
    case["y"][4] *= 1e-30
    case["x"][5] *= 1e15
    for layer_norm in (False, True):
        check_norm(pkg, dev, case, dout, dnormed, layer_norm=layer_norm)
    t = {k: None if v is None else v.to(dev) for k, v in case.items()}
    clean = pkg.gated_residual_norm(**t)
    t["y"][2, 5], t["x"][7, 3], t["gate"][9, 0] = float("inf"), float("nan"), float("nan")
    out, normed = pkg.gated_residual_norm(**t)
    fine = torch.ones(12, dtype=torch.bool)
    fine[[2, 7, 9]] = False
    assert torch.equal(out[fine], clean[0][fine]) and torch.equal(normed[fine], clean[1][fine])
    assert all(not torch.isfinite(normed[r]).all() for r in (2, 7, 9))


@pytest.mark.gpu
def test_nothing_in_them(pkg, dev):
    w = torch.ones(16, device=dev, requires_grad=True)
    x = torch.empty((0, 16), device=dev, requires_grad=True)
    offs = torch.zeros(4, dtype=torch.int64, device=dev)
    initial = torch.randn((3, 16), device=dev)
    out, state = pkg.gated_recurrence(x, x, x, w, offs, initial, return_state=True)
    assert out.shape == (0, 16) and torch.equal(state, initial)
    out.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w))
    out, normed = pkg.gated_residual_norm(x, x, pre_weight=w)
    (out.sum() + normed.sum()).backward()
    assert out.shape == normed.shape == (0, 16) and torch.equal(w.grad, torch.zeros_like(w))
    assert pkg.gated_recurrence_step(initial, x.detach()[:0], x.detach()[:0], x.detach()[:0], w.detach(), slots=offs[:0]).shape == (0, 16)
    rows = torch.randn((5, 16), device=dev)
    out, state = pkg.gated_recurrence(rows, rows, rows, w.detach(), offs, initial, return_state=True)  # all rows behind the last sequence
    assert torch.equal(out, torch.zeros_like(out)) and torch.equal(state, initial)


@pytest.mark.gpu
def test_refusals(pkg, dev, monkeypatch):
    x, w, offs = torch.randn((6, 8), device=dev), torch.ones(8, device=dev), torch.tensor([0, 2, 6], device=dev)
    bad = [
        (AssertionError, lambda: pkg.gated_recurrence(x, x[:5], x, w, offs)),
        (AssertionError, lambda: pkg.gated_recurrence(x, x.half(), x, w, offs)),
        (AssertionError, lambda: pkg.gated_recurrence(x, x, x, w[:7], offs)),
        (AssertionError, lambda: pkg.gated_recurrence(x, x, x, w.half(), offs)),
        (AssertionError, lambda: pkg.gated_recurrence(x, x, x, w, offs.float())),
        (AssertionError, lambda: pkg.gated_recurrence(x, x, x, w, offs[:1])),
        (AssertionError, lambda: pkg.gated_recurrence(x, x, x, w, offs.cpu())),
        (AssertionError, lambda: pkg.gated_recurrence(x, x, x, w, offs, torch.zeros((3, 8), device=dev))),
        (AssertionError, lambda: pkg.gated_recurrence(x, x, x, w, offs, torch.zeros((2, 8), device=dev).half())),
        (AssertionError, lambda: pkg.gated_recurrence(x, x, x, w, offs, rate=0.0)),
        (AssertionError, lambda: pkg.gated_recurrence(x, x, x, w, offs, rate=float("nan"))),
        (AssertionError, lambda: pkg.gated_recurrence(x.double(), x.double(), x.double(), w, offs)),
        (AssertionError, lambda: pkg.gated_recurrence_step(torch.zeros((5, 8), device=dev), x, x, x, w)),
        (AssertionError, lambda: pkg.gated_recurrence_step(torch.zeros((8, 6), device=dev).t(), x, x, x, w)),
        (AssertionError, lambda: pkg.gated_recurrence_step(torch.zeros((1, 8), device=dev).expand(6, 8), x, x, x, w)),
        (AssertionError, lambda: pkg.gated_recurrence_step(torch.zeros((6, 8), device=dev), x, x, x, w, slots=offs)),
        (NotImplementedError, lambda: pkg.gated_recurrence_step(torch.zeros((6, 8), device=dev), x, x, x, w.clone().requires_grad_(True))),
        (AssertionError, lambda: pkg.gated_residual_norm(x, x[:, :7])),
        (AssertionError, lambda: pkg.gated_residual_norm(x, x, post_bias=w)),
        (AssertionError, lambda: pkg.gated_residual_norm(x, x, pre_weight=w.half())),
        (AssertionError, lambda: pkg.gated_residual_norm(x, x, gate_activation="tanh")),
        (AssertionError, lambda: pkg.gated_residual_norm(x, x, dropout_ratio=1.0, training=True)),
        (AssertionError, lambda: pkg.gated_residual_norm(x, x, dropout_ratio=-0.5, training=True)),
        (NotImplementedError, lambda: pkg.gated_residual_norm(torch.zeros((2, 8200), device=dev), torch.zeros((2, 8200), device=dev))),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        for call in (lambda: pkg.gated_recurrence(dual, x, x, w, offs), lambda: pkg.gated_residual_norm(x, dual),
                     lambda: pkg.gated_recurrence_step(torch.zeros((6, 8), device=dev), dual, x, x, w)):
            with pytest.raises(NotImplementedError):
                call()
    monkeypatch.setenv("HSTU_HIP_CHECK_CONTRACT", "1")
    pkg.gated_recurrence(x, x, x, w, offs)
    for o in ([1, 2, 6], [0, 4, 2], [0, 2, 7]):
        with pytest.raises(ValueError):
            pkg.gated_recurrence(x, x, x, w, torch.tensor(o, device=dev))
    states = torch.zeros((9, 8), device=dev)
    slot = lambda *v: torch.tensor(v, device=dev)  # noqa: E731
    for s, n in ((slot(0, 1, 2, 3, 4, 9), None), (slot(0, 1, 2, 3, 4, -2), None), (slot(0, 1, 2, 3, 4, 4), None), (slot(0, 1, 2, 3, 4, 5), slot(6, 6, -1, -1, -1, -1)),
                 (slot(0, 1, 2, 3, 4, 5), slot(1, -1, -1, -1, -1, -1)), (None, None)):
        with pytest.raises((ValueError, AssertionError)):
            pkg.gated_recurrence_step(states, x, x, x, w, slots=s, new_slots=n)
    pkg.gated_recurrence_step(states, x, x, x, w, slots=slot(0, 0, 0, -1, 4, 5), new_slots=slot(6, 7, 8, -1, 4, 5))


@pytest.mark.gpu
def test_dropout_from_the_generator(pkg, dev):
    """Without a seed the device's generator gives one and moves on by the words that the call takes; the same state gives the same mask."""
    x, y = torch.zeros((50, 96), device=dev), torch.ones((50, 96), device=dev)
    torch.manual_seed(11)
    a, _ = pkg.gated_residual_norm(x, y, dropout_ratio=0.5, training=True)
    b, _ = pkg.gated_residual_norm(x, y, dropout_ratio=0.5, training=True)
    torch.manual_seed(11)
    c, _ = pkg.gated_residual_norm(x, y, dropout_ratio=0.5, training=True)
    assert torch.equal(a, c) and not torch.equal(a, b)
    assert set(a.unique().tolist()) == {0.0, 2.0}
    assert torch.equal(pkg.gated_residual_norm(x, y, dropout_ratio=0.5, training=False)[0], y)
    assert torch.equal(pkg.gated_residual_norm(x, y, dropout_ratio=0.5, training=True, seed=(3, 4))[0].cpu().double(), oracle.kept(0.5, 3, 4, 50, 96))


@pytest.mark.gpu
def test_a_layer_of_them(pkg, dev):
    """Producer, recurrence, consumer, and the norms between two layers: forward and backward against the oracles one after another."""
    from oracle import output_oracle, uqvk_oracle

    g = torch.Generator().manual_seed(12)
    H, D, dm, lengths = 2, 64, 128, [70, 3, 140]
    rows, width = sum(lengths), H * D
    offs = offsets_of(lengths)
    rnd = lambda *s, by=1.0, add=0.0: (add + by * torch.randn(s, generator=g)).to(BF)  # noqa: E731
    p = dict(x=rnd(rows, dm), nw=rnd(dm, by=0.1, add=1.0), nb=rnd(dm, by=0.1), w=rnd(dm, 4 * width, by=dm**-0.5), b=rnd(4 * width, by=0.1), ow=rnd(width, by=0.1, add=1.0),
             ob=rnd(width, by=0.1), wo=rnd(3 * width, dm, by=(3 * width) ** -0.5), post=rnd(dm, by=0.1, add=1.0), pre=rnd(dm, by=0.1, add=1.0), scale=rnd(dm, by=0.1, add=0.5))
    decay = torch.log(torch.expm1(-torch.log(0.9 + 0.099 * torch.rand(width, generator=g)) / 8.0))
    dout, dnormed = rnd(rows, dm), rnd(rows, dm)

    def layer(q, decay, double):
        if double:
            u, r, i, v = uqvk_oracle.compute_uqvk(q["x"], q["nw"], q["nb"], 1e-6, H, D, D, q["w"], q["b"])
            sr, si = torch.sigmoid(r.flatten(1)), torch.sigmoid(i.flatten(1))
            z = 8.0 * torch.nn.functional.softplus(decay) * sr
            bx, a = torch.sqrt(-torch.expm1(-2 * z)) * si * v.flatten(1), torch.exp(-z)
            hs = []
            for b in range(len(lengths)):
                h = torch.zeros_like(bx[0])
                for t in range(int(offs[b]), int(offs[b + 1])):
                    h = a[t] * h + bx[t]
                    hs.append(h)
            y = output_oracle.compute_output(torch.stack(hs), u, torch.zeros_like(q["x"]), q["ow"], q["ob"], q["wo"], 1e-6, concat_u=True, concat_x=True)
            return oracle.residual_norm(q["x"], y.to(q["x"].dtype), None, q["post"], None, q["scale"], q["pre"], None, eps=1e-6)
        u, r, i, v = pkg.hstu_compute_uqvk(q["x"], q["nw"], q["nb"], 1e-6, H, D, D, q["w"], q["b"])
        h, _ = pkg.gated_recurrence(v, r, i, decay, offs.to(dev))
        y = pkg.hstu_compute_output(h.flatten(1), u, torch.zeros_like(q["x"]), q["ow"], q["ob"], 1e-6, q["wo"], H, D, 0.0, False, True, True, "none", False, False)
        return pkg.gated_residual_norm(q["x"], y, None, q["post"], None, q["scale"], q["pre"])

    results = []
    for double in (False, True):
        q = {k: (v.double() if double else v.to(dev)).requires_grad_(True) for k, v in p.items()}
        d = (decay.double() if double else decay.to(dev)).requires_grad_(True)
        out, normed = layer(q, d, double)
        like = lambda t: t.to(out.device).to(out.dtype)  # noqa: E731
        got = torch.autograd.grad((out, normed), [d, *q.values()], (like(dout), like(dnormed)))
        results.append(dict(zip(["out", "normed", "decay", *q], [out, normed, *got])))
    for name, want in results[1].items():
        got = results[0][name].detach().cpu().double()
        # roundings to bf16 (2^-8 each) of q, k, v, u, h, the consumer's operand and its result, y, and of their gradients on the way back: sixteen
        # at most one behind another, added up as if all pointed one way, and the sums over a row mix them
        assert float((got - want.detach().double()).norm() / want.detach().double().norm()) < 16 * 2.0**-8, name
