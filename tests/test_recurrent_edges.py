"""The gated recurrence and the norms between two blocks where calls differ from the ordinary: streams, graphs, hooks, sizes past 32 bits, one long
history, hundreds of segments, gates and rows that leave nothing."""

import pytest
import torch

from oracle import recurrent_oracle as oracle
from test_recurrent import BF, F32, FP, NORMS, check_norm, check_scan, norm_case, offsets_of, run_scan, scan_case, within

pytestmark = pytest.mark.gpu
LEAVES = ("x", "decay_gate", "input_gate", "decay", "initial")


def to_dev(case, dev):
    return {k: None if v is None else v.to(dev) for k, v in case.items()}


def scan(pkg, t, **kw):
    return pkg.gated_recurrence(t["x"], t["decay_gate"], t["input_gate"], t["decay"], t["offsets"], t["initial"], return_state=True, **kw)


def doubled(a, b, place):
    """h_t = a_t h_{t-1} + b_t from nothing at place 0, in 64 bits, by doubling."""
    step = 1
    while step <= int(place.max()):
        there = (place[step:] >= step).view(-1, 1)
        more_b, more_a = torch.where(there, a[step:] * b[:-step], 0.0), torch.where(there, a[:-step], 1.0)
        b, a = torch.cat([b[:step], b[step:] + more_b]), torch.cat([a[:step], a[step:] * more_a])
        step *= 2
    return b


def check_long(pkg, t, got=None):
    """Every row and its bound, as the oracle has them, by doubling on the device; ``got``: gradients with dout of ones, too."""
    offs = t["offsets"]
    n = offs[1:] - offs[:-1]
    of = torch.repeat_interleave(torch.arange(len(n), device=offs.device), n)
    rows = of.numel()
    place = torch.arange(rows, device=offs.device) - offs[of]
    strength, s, z, a, m, i, u = oracle.gates(t["x"][:rows], t["decay_gate"][:rows], t["input_gate"][:rows], t["decay"], 8.0)
    h = doubled(a, m * u, place)
    size = doubled(a, (m * u).abs(), place)
    in_front = torch.cat([torch.zeros_like(size[:1]), size[:-1]]) * (place > 0).view(-1, 1)
    err = doubled(a, oracle.F32 * (a * in_front * (oracle.Z * z + oracle.A + 2) + oracle.B * (m * u).abs() + size), place)
    out, _ = pkg.gated_recurrence(t["x"], t["decay_gate"], t["input_gate"], t["decay"], offs)
    within(out[:rows], h.cpu(), err.cpu(), "out", t["x"].dtype)
    if got is None:
        return
    left = (n[of] - 1 - place).flip(0)
    ahead = torch.cat([a[1:], torch.zeros_like(a[:1])]).flip(0)
    ones = torch.ones_like(a)
    total = doubled(ahead, ones, left).flip(0)
    z_ahead = torch.cat([z[1:], torch.zeros_like(z[:1])]).flip(0)
    behind = torch.cat([torch.zeros_like(total[:1]), total.flip(0)[:-1]]) * (left > 0).view(-1, 1)
    total_err = doubled(ahead, oracle.F32 * (ahead * behind * (oracle.Z * z_ahead + oracle.A + 2) + 2 * total.flip(0)), left).flip(0)
    want = total * m * i
    within(got["x"][:rows], want.cpu(), (total_err * m * i + 2 * oracle.B * oracle.F32 * want).cpu(), "dx", t["x"].dtype)


@pytest.mark.parametrize("lengths", [[70000], [40000, 1, 30001], [64 * 16 * 9, 64 * 16]], ids=["one", "two", "whole-groups"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_long_histories(pkg, dev, dtype, lengths):
    """Hundreds of tiles of one sequence under way at once, more groups of them than are gone back over."""
    case, *_ = scan_case(lengths, 24, dtype, seed=31, states=False)
    t = to_dev(case, dev)
    leaf = t["x"].clone().requires_grad_(True)
    out, _ = pkg.gated_recurrence(leaf, t["decay_gate"], t["input_gate"], t["decay"], t["offsets"])
    out.backward(torch.ones_like(out))
    check_long(pkg, t, {"x": leaf.grad})


def test_hundreds_of_segments(pkg, dev):
    """A sequence's bits do not depend on the others: each by itself, and among 300 that are planned in five parts."""
    lengths = [600 + (37 * k) % 500 for k in range(300)]
    case, dout, _ = scan_case(lengths, 40, BF, seed=32, states=False)
    t = to_dev(case, dev)
    whole = run_scan(pkg, dev, case, dout)
    for b in (0, 1, 63, 64, 65, 128, 255, 299):
        rows = slice(int(case["offsets"][b]), int(case["offsets"][b + 1]))
        one = dict(case, offsets=offsets_of([lengths[b]]), **{k: case[k][rows] for k in ("x", "decay_gate", "input_gate")})
        alone = run_scan(pkg, dev, one, dout[rows])
        assert torch.equal(whole[0][rows], alone[0])
        assert all(torch.equal(whole[2][k][rows], alone[2][k]) for k in ("x", "decay_gate", "input_gate"))
    check_long(pkg, t)


@pytest.mark.parametrize("rows_more", [0, 1])
@pytest.mark.parametrize("batch", [1, 7, 200])
def test_where_short_sequences_end(pkg, dev, batch, rows_more):
    """On both sides of the rule for a workgroup per sequence: 16 rows to a sequence and 48; and past 4096 rows in all."""
    rows = min(16 * batch + 48, 4096) + rows_more
    lengths = [rows // batch] * batch
    lengths[-1] += rows - sum(lengths)
    case, *_ = scan_case(lengths, 40, BF, seed=batch, behind=5)
    check_scan(pkg, dev, case, None, None, grads=False)


def test_streams(pkg, dev):
    """Calls on other streams than the default one, two at once, forward and backward."""
    cases = [scan_case([3000, 50, 700], 256, BF, seed=k) for k in range(2)]
    norms = [norm_case(3000, 512, BF, seed=k, **NORMS[7]) for k in range(2)]
    want = [run_scan(pkg, dev, *c) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ts = [to_dev(c[0], dev) for c in cases]
    ns = [to_dev(n[0], dev) for n in norms]
    normed = [pkg.gated_residual_norm(**n, dropout_ratio=0.1, training=True, seed=(1, 2)) for n in ns]
    torch.cuda.synchronize()
    for _ in range(3):
        got = [[], []]
        for _ in range(4):
            for k in range(2):
                with torch.cuda.stream(streams[k]):
                    leaf = ts[k]["x"].clone().requires_grad_(True)
                    out, state = scan(pkg, dict(ts[k], x=leaf))
                    grad = torch.autograd.grad((out, state), leaf, (cases[k][1].to(dev), cases[k][2].to(dev)))[0]
                    got[k].append((out, state, grad, *pkg.gated_residual_norm(**ns[k], dropout_ratio=0.1, training=True, seed=(1, 2))))
        torch.cuda.synchronize()
        for k in range(2):
            for out, state, grad, a, b in got[k]:
                assert torch.equal(out, want[k][0]) and torch.equal(state, want[k][1]) and torch.equal(grad, want[k][2]["x"])
                assert torch.equal(a, normed[k][0]) and torch.equal(b, normed[k][1])


def test_captured_and_replayed(pkg, dev):
    """A prefill, a step in place and a norm in one graph; every replay against the eager calls, which go on in between, on inputs that change."""
    case, *_ = scan_case([900, 3, 400], 128, BF, seed=40)
    t = to_dev(case, dev)
    states, w = torch.randn((3, 128), device=dev), torch.ones(128, device=dev, dtype=BF)
    row = t["x"][:3].clone()

    def calls(states):
        out, final = scan(pkg, t)
        stepped = pkg.gated_recurrence_step(states, row, row, row, t["decay"])
        return [out, final, stepped, *pkg.gated_residual_norm(out, t["x"], t["input_gate"], pre_weight=w, dropout_ratio=0.2, training=True, seed=(5, 6))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls(states.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    kept = states.clone()
    with torch.cuda.graph(graph):
        got = calls(kept)
    eager = states.clone()
    kept.copy_(states)
    for k in range(4):
        graph.replay()
        want = calls(eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(kept, eager)
        t["x"].add_(0.125 * (k + 1))
        row.mul_(0.5)


def test_captured_training_step(pkg, dev):
    """Forward and backward in one graph, replayed on other inputs, with eager steps of the same leaves in between."""
    case, dout, dfinal = scan_case([500, 130], 64, BF, seed=41)
    t = to_dev(case, dev)
    leaves = [t[k].requires_grad_(True) for k in LEAVES]
    w = torch.ones(64, device=dev, dtype=BF, requires_grad=True)
    d, f = dout.to(dev), dfinal.to(dev)

    def step():
        out, final = scan(pkg, t)
        y, normed = pkg.gated_residual_norm(t["x"], out, pre_weight=w, dropout_ratio=0.3, training=True, seed=(7, 8))
        return torch.autograd.grad((y, normed, final), [*leaves, w], (d, d, f))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with torch.no_grad():
            t["input_gate"].add_(0.25)
            d.mul_(-1.5)


def test_a_graph_of_gradients_used_twice_and_in_part(pkg, dev):
    case, dout, dfinal = scan_case([300, 20], 64, BF, seed=42)
    t = to_dev(case, dev)
    all_of = run_scan(pkg, dev, case, dout, dfinal)[2]
    for only in LEAVES:
        one = dict(t, **{only: t[only].clone().requires_grad_(True)})
        out, final = scan(pkg, one)
        for _ in range(2):
            got = torch.autograd.grad((out, final), one[only], (dout.to(dev), dfinal.to(dev)), retain_graph=True)[0]
            assert torch.equal(got, all_of[only]), only
    case, dout, dnormed = norm_case(60, 128, BF, seed=3, **NORMS[4])
    names = [k for k in case if case[k] is not None]
    every = {k: case[k].to(dev).requires_grad_(True) for k in names}
    o = pkg.gated_residual_norm(**every, gate_activation="none")
    want = dict(zip(names, torch.autograd.grad(o, list(every.values()), (dout.to(dev), dnormed.to(dev)), retain_graph=True)))
    for only in names:
        one = {k: case[k].to(dev) for k in names}
        one[only].requires_grad_(True)
        got = torch.autograd.grad(pkg.gated_residual_norm(**one, gate_activation="none"), one[only], (dout.to(dev), dnormed.to(dev)))[0]
        assert torch.equal(got, want[only]), only


def test_gradients_that_come_in_otherwise(pkg, dev):
    """Expanded, transposed, of another type; saved tensors that went to the host and back; autocast."""
    case, dout, dfinal = scan_case([100, 28], 64, BF, seed=43, states=False)
    t = to_dev(case, dev)
    t["x"].requires_grad_(True)
    out, _ = scan(pkg, t)
    a = torch.autograd.grad(out.sum(), t["x"], retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(out, t["x"], torch.ones_like(out), retain_graph=True)[0])
    d = dout.to(dev)
    want = torch.autograd.grad(out, t["x"], d, retain_graph=True)[0]
    assert torch.equal(want, torch.autograd.grad(out, t["x"], d.t().contiguous().t(), retain_graph=True)[0])
    with torch.autograd.graph.save_on_cpu():
        out, _ = scan(pkg, t)
    assert torch.equal(want, torch.autograd.grad(out, t["x"], d)[0])
    with torch.autocast("cuda", dtype=torch.float16):
        out, _ = scan(pkg, t)
        y, normed = pkg.gated_residual_norm(t["x"], out, pre_weight=torch.ones(64, device=dev, dtype=BF))
    assert out.dtype == y.dtype == normed.dtype == BF
    assert torch.equal(want, torch.autograd.grad(out, t["x"], d)[0])
    with torch.inference_mode():
        states = torch.zeros((128, 64), device=dev)
        pkg.gated_recurrence_step(states, t["x"], t["decay_gate"], t["input_gate"], t["decay"])
        assert bool((states != 0).any())


def test_a_state_changed_under_a_graph_is_noticed(pkg, dev):
    """The step changes its states in place, and says so to a graph that saved them."""
    states = torch.randn((4, 8), device=dev)
    w = torch.ones(8, device=dev, requires_grad=True)
    y = (states * w).sum()
    x = torch.randn((4, 8), device=dev)
    pkg.gated_recurrence_step(states, x, x, x, w.detach())
    with pytest.raises(RuntimeError):
        y.backward()


def test_elements_past_2_to_the_31(pkg, dev):
    """Sequences and rows that lie behind the first 2^31 elements and 2^32 bytes of their tensors."""
    width, rows = 2048, (1 << 20) + 700
    x = torch.zeros((rows, width), dtype=BF, device=dev)
    tail = 650
    g = torch.Generator().manual_seed(3)
    last = torch.randn((tail, width), generator=g).to(BF)
    x[-tail:] = last.to(dev)
    decay = torch.full((width,), -4.0)
    offs = torch.tensor([0, 1 << 19, rows - tail, rows])
    leaf = x.requires_grad_(True)
    out, _ = pkg.gated_recurrence(leaf, leaf, leaf, decay.to(dev), offs.to(dev))
    at = dict(x=last, decay_gate=last, input_gate=last, decay=decay, offsets=offsets_of([tail]))
    h, _, err, *_ = oracle.scan(**at)
    within(out[-tail:], h, err, "out", BF)
    assert bool((out[: rows - tail] == 0).all())
    d = torch.zeros_like(out)
    d[-tail:] = 1
    got = torch.autograd.grad(out, leaf, d)[0]  # (three gradients of one leaf, added up in bf16)
    want = oracle.scan_grad(**at, dout=torch.ones_like(last))
    parts = [want[k] for k in ("x", "decay_gate", "input_gate")]
    sizes = sum(p[0].abs() for p in parts)
    # each is rounded, then their sum twice, each time no more than half a step of all their sizes
    within(got[-tail:], sum(p[0] for p in parts), sum(p[1] for p in parts) + 5 * 2.0**-8 * sizes, "grad", BF)
    del out, got, d
    x = x.detach()
    w = torch.ones(width, dtype=BF, device=dev)
    o, normed = pkg.gated_residual_norm(x, x, x, pre_weight=w)
    ref, ref_normed, _, bounds = oracle.residual_norm_grad(last, last, last, None, None, None, torch.ones(width, dtype=BF), None, 1e-6, False, "sigmoid", None, None, None)
    within(o[-tail:], ref, bounds["out"], "out", BF)
    within(normed[-tail:], ref_normed, bounds["normed"], "normed", BF)


def test_rows_further_apart_than_the_kernels_take(pkg, dev):
    """Strides past 2^24 elements go through a copy."""
    big = torch.randn(((1 << 24) * 3 + 200,), device=dev, dtype=BF)
    x = big.as_strided((3, 64), ((1 << 24) + 64, 1))
    offs = torch.tensor([0, 3], device=dev)
    w = torch.zeros(64, device=dev)
    assert torch.equal(pkg.gated_recurrence(x, x, x, w, offs)[0], pkg.gated_recurrence(x.contiguous(), x.contiguous(), x.contiguous(), w, offs)[0])
    assert torch.equal(pkg.gated_residual_norm(x, x)[0], pkg.gated_residual_norm(x.contiguous(), x.contiguous())[0])


@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_norm_gates_at_their_ends(pkg, dev, dtype, act):
    """Gates at the ends of what a sigmoid tells apart and far beyond; dropped elements that are infinite leave nothing behind."""
    kind = dict(gate=act, params="10010")
    case, dout, dnormed = norm_case(9, 64, dtype, seed=2, **kind)
    case["gate"][1], case["gate"][2], case["gate"][3] = 80.0, -80.0, 0.0
    check_norm(pkg, dev, case, dout, dnormed, **kind)
    t = to_dev(case, dev)
    t["gate"][4] = torch.finfo(dtype).min
    if act != "none":
        out, normed = pkg.gated_residual_norm(**t, gate_activation=act)
        assert torch.equal(out[4], t["x"][4]) and torch.isfinite(normed).all()
    drop = dict(dropout_ratio=0.5, training=True, seed=(9, 9))
    keep = oracle.kept(0.5, 9, 9, 9, 64)
    y = torch.where(keep == 0, float("inf"), 1.0).to(dtype).to(dev)
    out, _ = pkg.gated_residual_norm(torch.zeros_like(y), y, **drop)
    assert torch.equal(out.cpu().double(), keep)


@pytest.mark.parametrize("ratio", [2.0**-31, 0.999, 1 - 2.0**-33])
def test_dropout_ratios_at_their_ends(pkg, dev, ratio):
    x = torch.ones((64, 96), device=dev)
    out, _ = pkg.gated_residual_norm(torch.zeros_like(x), x, dropout_ratio=ratio, training=True, seed=(1, 1))
    want = oracle.kept(ratio, 1, 1, 64, 96)
    assert torch.equal(out.cpu() != 0, want != 0)
    within(out, want, 2 * oracle.F32 * want, "kept", F32)


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 17])
@pytest.mark.parametrize("width", [24, 512, 1024, 2900])
def test_fewer_rows_than_groups(pkg, dev, rows, width):
    """Groups of lanes, and workgroups, that have no row; an infinity in the last row is no other's."""
    check_norm(pkg, dev, *norm_case(rows, width, BF, seed=rows, **NORMS[7]), **NORMS[7])
    t = {k: v.to(dev).requires_grad_(True) for k, v in norm_case(rows, width, F32, params="00100", gate=None, seed=rows)[0].items() if v is not None}
    with torch.no_grad():
        t["y"][-1, 3] = float("inf")
    out, _ = pkg.gated_residual_norm(**t)
    grad = torch.autograd.grad(out, t["scale"], torch.ones_like(out))[0]
    assert grad[3] == float("inf") and torch.isfinite(grad[:3]).all() and torch.isfinite(grad[4:]).all()


def test_the_steps_of_a_padded_batch(pkg, dev):
    """Rows of padding carry -1 both ways: nothing is read for them and nothing kept; many rows may read one state that none puts."""
    states = torch.randn((6, 32), device=dev)
    before = states.clone()
    x = torch.randn((5, 32), device=dev)
    w = torch.zeros(32, device=dev)
    slots = torch.tensor([2, -1, 2, -1, 4], device=dev)
    out = pkg.gated_recurrence_step(states, x, x, x, w, slots=slots, new_slots=torch.tensor([-1, -1, 5, -1, 4], device=dev))
    assert torch.equal(states[:4], before[:4])
    first = pkg.gated_recurrence_step(before[[2, 2, 4]].clone(), x[[0, 2, 4]], x[[0, 2, 4]], x[[0, 2, 4]], w)
    assert torch.equal(out[[0, 2, 4]], first) and torch.equal(states[5], first[1]) and torch.equal(states[4], first[2])
    fresh = pkg.gated_recurrence_step(torch.zeros((2, 32), device=dev), x[[1, 3]], x[[1, 3]], x[[1, 3]], w)
    assert torch.equal(out[[1, 3]], fresh)
    wide = torch.randn((6, 64), device=dev)
    part = wide[:, 16:48]  # states with columns of others between them
    keep = wide.clone()
    pkg.gated_recurrence_step(part, x, x, x, w, slots=torch.arange(5, device=dev, dtype=torch.int32))
    assert torch.equal(wide[:, :16], keep[:, :16]) and torch.equal(wide[:, 48:], keep[:, 48:]) and torch.equal(wide[5], keep[5])
    assert not torch.equal(part[:5], keep[:5, 16:48])
