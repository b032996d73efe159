"""The gated recurrence and the norms between two blocks at numbers and sizes where a result can be lost: rows that there are not, gates that are open, calls of no
rows, numbers that are none."""

import ctypes

import pytest
import torch

from oracle import recurrent_oracle as oracle
from test_recurrent import BF, F32, FP, NORMS, abi, check_norm, check_scan, norm_case, offsets_of, scan_case, within


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


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 16), (0, 2, 8), (3, 0)], ids=str)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_graphs_of_no_rows(pkg, dev, dtype, shape):
    """Every input of a call with nothing in it is in the graph of both results, as with rows: gradients of zeros, and the states' own."""
    width = 16 if shape[0] == 0 else 0
    offsets = torch.zeros(4, dtype=torch.int64, device=dev)
    for given in (True, False):
        leaves = [torch.zeros(shape, dtype=dtype, device=dev).requires_grad_() for _ in range(3)] + [torch.ones(width, device=dev).requires_grad_()]
        if given:
            leaves.append(torch.randn((3, width), device=dev).requires_grad_())
        initial = leaves[4] if given else None
        out, none = pkg.gated_recurrence(*leaves[:4], offsets, initial)
        assert none is None and out.shape == shape and out.dtype == dtype
        for got, leaf in zip(torch.autograd.grad(out, leaves, torch.zeros_like(out)), leaves):
            assert torch.equal(got, torch.zeros_like(leaf))
        out, state = pkg.gated_recurrence(*leaves[:4], offsets, initial, return_state=True)
        assert torch.equal(state, initial if given else torch.zeros((3, width), device=dev)) and state.dtype == F32
        d = torch.randn((3, width), device=dev)
        for only_state in (True, False):
            results, grads = ((state,), (d,)) if only_state else ((out, state), (torch.zeros_like(out), d))
            got = torch.autograd.grad(results, leaves, grads, retain_graph=True)
            assert all(torch.equal(g, torch.zeros_like(leaf)) for g, leaf in zip(got[:4], leaves))
            assert not given or torch.equal(got[4], d)
    with torch.no_grad():
        out, state = pkg.gated_recurrence(*leaves[:4], offsets, return_state=True)
    assert not out.requires_grad and not state.requires_grad


@pytest.mark.gpu
def test_a_refused_call_leaves_the_generator(pkg, dev):
    x, wide = torch.zeros((2, 64), device=dev), torch.zeros((2, 8200), device=dev)
    before = torch.cuda.default_generators[0].get_offset()
    with pytest.raises(NotImplementedError):
        pkg.gated_residual_norm(wide, wide, dropout_ratio=0.5, training=True)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            pkg.gated_residual_norm(x, torch.autograd.forward_ad.make_dual(x, x), dropout_ratio=0.5, training=True)
    assert torch.cuda.default_generators[0].get_offset() == before
    pkg.gated_residual_norm(x, x, dropout_ratio=0.5, training=True)
    assert torch.cuda.default_generators[0].get_offset() > before


@pytest.mark.gpu
@pytest.mark.parametrize("length", [1, 2, 16, 20, 40, 63, 70])
def test_a_state_that_is_too_large(pkg, dev, length):
    """A last state past fp32 is an infinity; the decays' gradient, to which rows behind it have nothing to add, is finite."""
    width = 8
    x = torch.zeros((length, width))
    x[-1] = 3.2e38
    r, i = torch.full_like(x, -1e30), torch.full_like(x, 20.0)
    r[-1] = 0.0  # the rows in front of the last leave the state as it is
    decay = torch.full((width,), -3.0)
    initial = torch.full((1, width), 3.2e38)
    case = dict(x=x, decay_gate=r, input_gate=i, decay=decay, offsets=offsets_of([length]), initial=initial)
    dout = torch.zeros_like(x)
    dout[-1] = 1e-30
    h, _, *_ = oracle.scan(**case)
    leaves = [case[k].to(dev).requires_grad_() for k in ("x", "decay_gate", "input_gate", "decay", "initial")]
    out, _ = pkg.gated_recurrence(*leaves[:4], case["offsets"].to(dev), leaves[4])
    assert bool(torch.isinf(out[-1]).all()) and bool((h[-1] > torch.finfo(F32).max).all())
    got = torch.autograd.grad(out, leaves, dout.to(dev))
    want = oracle.scan_grad(**case, dout=dout)
    within(got[3], *want["decay"], "d decay")


# Halves of a unit in fp32's last place that a sigmoid and what it leaves of 1 may be off by, each of itself: -x log2(e) is rounded, and so is its log2(e) (to a
# quarter of a half), which an exponential makes |x| times as much of; exponential and reciprocal two each, sum and product one each, 1 - s (where s is the smaller) one and s's own.
def sigmoid_steps(x):
    return 1.25 * x.abs() + 10


OPEN = [0.0, 0.3, 1.0, 2.5, 5.0, 8.0, 9.5, 11.0, 12.0, 13.5, 15.0, 16.0, 17.0, 17.5, 20.0, 30.0, 50.0, 80.0]


def ends(dtype, width, seed):
    """Gates from -80 to 80, a value to a row."""
    values = torch.tensor(OPEN + [-v for v in OPEN[1:]], dtype=torch.float64)
    g = torch.Generator().manual_seed(seed)
    return (values.view(-1, 1) + 0.25 * torch.rand((len(values), width), generator=g, dtype=torch.float64)).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("width", [64, 100, 1024])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_norm_gates_that_are_open(pkg, dev, dtype, width, act):
    """The gate's gradient is dout y act'(gate), good to its own last places where act' is far below 1."""
    gate = ends(dtype, width, 3)
    g = torch.Generator().manual_seed(4)
    y, dout = ((torch.randn(gate.shape, generator=g)).to(dtype) for _ in range(2))
    leaf = gate.to(dev).requires_grad_()
    out, _ = pkg.gated_residual_norm(torch.zeros_like(leaf.detach()), y.to(dev), leaf, gate_activation=act)
    got = torch.autograd.grad(out, leaf, dout.to(dev))[0]
    z = gate.double()
    s, rest = torch.sigmoid(z), torch.sigmoid(-z)
    slope, size = (s * rest, s * rest) if act == "sigmoid" else (s * (1 + z * rest), s * (1 + z.abs() * rest))
    by = dout.double() * y.double()
    # both factors' steps, the products of the slope (SiLU: one more sum) and the two with dout and y: six roundings
    within(got, by * slope, oracle.F32 * (2 * sigmoid_steps(z) + 6) * (by.abs() * size) + 2.0**-122, "dgate", dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 72])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_recurrence_gates_that_are_open(pkg, dev, dtype, width):
    """Both gates' gradients have a factor 1 - s, good to its own last places where s is close to 1.  Sequences of one row that begin with nothing: no sums."""
    gate = ends(dtype, width, 5)
    other = gate.roll(7, 0)
    rows = gate.shape[0]
    g = torch.Generator().manual_seed(6)
    x, dout = ((torch.randn(gate.shape, generator=g)).to(dtype) for _ in range(2))
    decay = torch.log(torch.expm1(-torch.log(0.5 + 0.45 * torch.rand(width, generator=g, dtype=torch.float64)) / 8.0)).float()
    case = dict(x=x, decay_gate=gate, input_gate=other, decay=decay, offsets=offsets_of([1] * rows))
    leaves = [case[k].to(dev).requires_grad_() for k in ("x", "decay_gate", "input_gate", "decay")]
    out, _ = pkg.gated_recurrence(*leaves, case["offsets"].to(dev))
    got = torch.autograd.grad(out, leaves, dout.to(dev))
    strength, s, z, a, m, i, u = oracle.gates(x, gate, other, decay, 8.0)
    r_rest, i_rest, d = torch.sigmoid(-gate.double()), torch.sigmoid(-other.double()), dout.double()
    want_r, want_i = strength * r_rest * d * u * a * a * s / m, d * m * u * i_rest
    # as the oracle counts them: a^2 and m by Z z and B of themselves, a product each; then the two gates' own
    steps = 3 * oracle.Z * z + 2 * oracle.B + 2 * sigmoid_steps(gate.double()) + 2 * sigmoid_steps(other.double())
    within(got[1], want_r, oracle.F32 * steps * want_r.abs() + 2.0**-122, "d decay_gate", dtype)
    within(got[2], want_i, oracle.F32 * steps * want_i.abs() + 2.0**-122, "d input_gate", dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_columns_that_hardly_forget(pkg, dev, dtype):
    """1 - a^2 down to nothing at all: results and gradients are numbers, and what a row lets in is lost only where its square is below fp32's normal numbers."""
    gate = ends(dtype, 72, 7)
    rows = gate.shape[0]
    g = torch.Generator().manual_seed(8)
    x, dout = ((torch.randn(gate.shape, generator=g)).to(dtype) for _ in range(2))
    initial = torch.randn((3, 72), generator=g)
    case = dict(x=x, decay_gate=gate, input_gate=gate.roll(5, 0), decay=torch.linspace(-110, -10, 72), offsets=offsets_of([9, 1, rows - 10]), initial=initial)
    leaves = [case[k].to(dev).requires_grad_() for k in ("x", "decay_gate", "input_gate", "decay", "initial")]
    out, _ = pkg.gated_recurrence(*leaves[:4], case["offsets"].to(dev), leaves[4])
    got = dict(zip(("x", "decay_gate", "input_gate", "decay", "initial"), torch.autograd.grad(out, leaves, dout.to(dev))))
    h, _, err, *_ = oracle.scan(**case)
    want = oracle.scan_grad(**case, dout=dout)
    # a row's m is below 2^-63 where its square is lost: of h each row's m u, of the gradients m, m u and, s / m being m / (2 strength) there, half of that
    most = float(x.double().abs().max())
    total = float(dout.double().abs().sum(0).max())
    within(out, h, err + rows * most * 2.0**-63, "out", dtype)
    for k, (value, bound) in want.items():
        within(got[k], value, bound + (rows if k == "decay" else 1) * total * (most + rows * most) * 2.0**-63 + 2.0**-122, "d " + k, F32 if k in ("decay", "initial") else dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("batch, width", [(64, 4096), (64, 4100), (65, 4096), (512, 512), (513, 512), (4096, 64), (4097, 64), (1100, 200)])
def test_where_many_short_sequences_end(pkg, dev, batch, width):
    """On both sides of the rule for a workgroup per sequence and 64 columns: 4096 of them."""
    lengths = [(k * 7) % 3 for k in range(batch)]
    lengths[-1] = 5
    case, *_ = scan_case(lengths, width, BF, seed=batch, behind=2)
    check_scan(pkg, dev, case, None, None, grads=False)
