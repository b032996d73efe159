"""Rotated positions and the 4-bit paged cache: kernels against the 64-bit oracle at the sizes and masks where they can go wrong, what
is refused, and a run of them together.  Every tolerance is a bound from the roundings that the definition has (oracle)."""

import pytest
import torch

from oracle import hstu_oracle, paged_oracle as O

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rand(seed, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _within(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = off > bound
    assert not over.any(), f"{what}: {int(over.sum())} of {over.numel()} over the bound, worst {float((off / bound.clamp(min=1e-300)).max()):.3g} times"


# ---- the oracle ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_oracles_gradient_against_differences(interleaved):
    x, dy = _rand(1, (5, 2, 32), torch.float64), _rand(2, (5, 2, 32), torch.float64)
    w, pos = 1 + 0.3 * _rand(3, (32,), torch.float64), torch.tensor([0, 9, 3, 77, 2])
    half = 8
    angle = torch.arange(100).double().view(-1, 1) * 0.7 ** torch.arange(half)
    table = torch.cat([angle.cos(), angle.sin()], 1)
    args = (1e-3, table, pos, interleaved)
    dx, dw, _ = O.norm_rope_grad(x, dy, w, *args)
    step = 1e-6  # differences of the second order: step^2 off, and 2^-53 / step
    for seed in range(4):
        v, vw = _rand(10 + seed, x.shape, torch.float64), _rand(20 + seed, w.shape, torch.float64)
        up, down = ((O.norm_rope(x + s * v, w + s * vw, *args) * dy).sum() for s in (step, -step))
        assert abs(float((up - down) / (2 * step) - (dx * v).sum() - (dw * vw).sum())) < 1e-7


def test_the_oracles_attention_is_the_cached_form():
    lengths = torch.tensor([70, 33, 128])
    table, pages = O.page_table(3, lengths, 16)
    cache = O.fill_cache(4, pages, 2, 16, 32, 64, BF16)
    q = _rand(5, (3 * 9, 2, 32), BF16)
    rows = [[sum((lambda c, s, lo: lo + s * c)(*O.sequence_rows(cache, table[b], int(n), i)) for _ in (0,)) for b, n in enumerate(lengths)] for i in (0, 1)]
    k, v = (torch.cat(r) for r in rows)
    offs = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)])
    t = torch.tensor([9, 0, 20])
    want = hstu_oracle.cached_hstu_mha_per_sequence(128, 0.2, q, k, v, offs, num_targets=t, max_attn_len=40, contextual_seq_len=3, compute_dtype=torch.float64)
    got, _ = O.attention(128, 0.2, q, cache, table, lengths, t, 40, 3)
    assert (got - want).abs().max() < 1e-14


# ---- refusals (no kernel is launched) -----------------------------------------------------------------------------------


def test_statuses_of_the_c_abi():
    """Calls that the library refuses before it touches a device; pointers are looked at, never followed."""
    import ctypes
    import os
    import re
    import subprocess

    from generative_recommenders_amd import build

    if not os.path.exists(build.CACHE_LIB_PATH):
        import __graft_entry__

        __graft_entry__.build()
    lib = ctypes.CDLL(build.CACHE_LIB_PATH)
    header = open(os.path.join(build.INCLUDE, "hstu_cache.h")).read()
    declared = set(re.findall(r"\b(hstu_cache_\w+)\s*\(", header))
    exported = set(re.findall(r" T (hstu_cache_\w+)", subprocess.run(["nm", "-D", build.CACHE_LIB_PATH], capture_output=True, text=True, check=True).stdout))
    assert declared == exported and lib.hstu_cache_version() >= 100
    assert lib.hstu_cache_norm_rope(None, None) == -1 and lib.hstu_cache_append(None, None, None) == -1 and lib.hstu_cache_attention(None, None, None) == -1
    lib.hstu_cache_last_error.restype = ctypes.c_char_p
    assert lib.hstu_cache_last_error() == b""


def _abi():
    """The library and its argument structures, read from the header."""
    import ctypes
    import os
    import re

    from generative_recommenders_amd import build

    lib = ctypes.CDLL(build.CACHE_LIB_PATH)
    header = re.sub(r"/\*.*?\*/", "", open(os.path.join(build.INCLUDE, "hstu_cache.h")).read(), flags=re.S)
    types = {"int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32, "float": ctypes.c_float}
    made = {}
    for body, name in re.findall(r"typedef struct \w+ \{(.*?)\} (\w+);", header, flags=re.S):
        fields = []
        for line in body.split(";"):
            if line.strip():
                kind, names = line.strip().removeprefix("const ").split(None, 1)
                for n in names.split(","):
                    fields.append((n.strip().lstrip("* "), ctypes.c_void_p if "*" in line else types[kind]))
        made[name] = type(name, (ctypes.Structure,), {"_fields_": fields})
    for name in ("attention", "norm_rope_bwd"):
        getattr(lib, f"hstu_cache_{name}_workspace_bytes").restype = ctypes.c_size_t
    return lib, ctypes.byref, made


def test_sizes_past_32_bits_in_the_c_abi():
    """Scratch memory of more than 2^31 values is asked for in full, and what no launch can number is refused (pointers are never followed)."""
    lib, ref, made = _abi()
    at = 1 << 20
    cache = made["HstuPagedCache"](k_codes=at, k_scales=at, v_codes=at, v_scales=at, pages=1 << 20, heads=1, page_size=1024, dqk=128, dv=128, dtype=0, page_table=at,
                                   table_row_stride=1024, table_columns=1024, batch=256)
    call = made["HstuPagedAttentionArgs"](q=at, q_row_stride=1024, q_head_stride=128, out=at, seq_lengths=at, q_heads=8, delta_size=512, max_seq_len=1 << 20, alpha=1.0, kv_splits=4096,
                                          workspace=at)
    need = lib.hstu_cache_attention_workspace_bytes(ref(cache), ref(call))
    assert need == 4096 * 256 * 512 * 8 * 128 * 4
    call.workspace_bytes = need - 1
    assert lib.hstu_cache_attention(ref(cache), ref(call), None) == -5
    call.workspace_bytes = need
    assert lib.hstu_cache_attention(ref(cache), ref(call), None) == -6
    call.kv_splits = 1
    assert lib.hstu_cache_attention_workspace_bytes(ref(cache), ref(call)) == 0
    rows = 1 << 28
    for name, start in (("append", made["HstuAppendArgs"](k=at, v=at, rows=rows, k_row_stride=128, k_head_stride=128, v_row_stride=128, v_head_stride=128, start=at)),):
        assert getattr(lib, f"hstu_cache_{name}")(ref(cache), ref(start), None) == -6
    import ctypes

    assert lib.hstu_cache_read(ref(cache), ctypes.c_int64(rows), ctypes.c_void_p(at), 0, None, 0, ctypes.c_void_p(at), ctypes.c_void_p(at), None) == -6
    turn = made["HstuNormRopeArgs"](q=at, q_row_stride=128, q_head_stride=128, q_out=at, q_weight=at, rows=rows, q_heads=1, dim=128, dtype=0)
    assert lib.hstu_cache_norm_rope(ref(turn), None) == -6
    turn.rows = 1 << 40
    assert 0 < lib.hstu_cache_norm_rope_bwd_workspace_bytes(ref(turn)) <= 2048 * 2 * 128 * 4


def test_no_vector_instruction_reads_a_matrix_result_too_early(tmp_path):
    import os
    import shutil
    import subprocess

    from generative_recommenders_amd import build
    from test_matrix_hazards import early_reads

    objdump = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
    if not os.path.exists(objdump) or not os.path.exists(build.CACHE_LIB_PATH):
        pytest.skip("needs llvm-objdump and the built library")
    shutil.copy(build.CACHE_LIB_PATH, tmp_path / "lib.so")
    subprocess.run([objdump, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    total = 0
    for name in sorted(p for p in os.listdir(tmp_path) if p.endswith("gfx950")):
        text = subprocess.run([objdump, "-d", name], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        products, early = early_reads(text)
        total += products
        assert not early, early[:10]
    assert total > 1000


def test_python_refusals_on_the_host(pkg):
    with pytest.raises(NotImplementedError):
        pkg.allocate_paged_kv_cache(4, 24, 1, 64, 64, device="cpu")
    with pytest.raises(NotImplementedError):
        pkg.allocate_paged_kv_cache(4, 16, 1, 96, 64, device="cpu")
    with pytest.raises(AssertionError):
        pkg.allocate_paged_kv_cache(4, 16, 1, 64, 64, dtype=F32, device="cpu")
    with pytest.raises(AssertionError):
        pkg.make_rotary_table(8, 7, device="cpu")
    x = torch.zeros(2, 1, 32)
    with pytest.raises(AssertionError, match="CUDA"):
        pkg.qk_norm_rope(x, None, torch.zeros(2, dtype=torch.int64), torch.zeros(4, 16))
    cache = pkg.allocate_paged_kv_cache(4, 16, 1, 32, 32, device="cpu")
    table, start = torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(AssertionError, match="CUDA"):
        pkg.append_paged_kv(cache, x.bfloat16(), x.bfloat16(), table, start)
    with pytest.raises(AssertionError, match="CUDA"):
        pkg.delta_hstu_mha_paged(16, 1.0, x.bfloat16(), cache, table, start)
    with pytest.raises(AssertionError, match="CUDA"):
        pkg.read_paged_kv(cache, 2, table, start)


def test_the_rotary_tables_angles(pkg):
    """Angles in 64 bits: a far position's cosine is that of the angle, half an fp32 step off."""
    table = pkg.make_rotary_table(200001, 16, device="cpu")
    angle = 200000 * 10000.0 ** (-torch.arange(8).double() / 8)
    assert (table[-1, :8].double() - angle.cos()).abs().max() <= 2.0**-24 * 1.01 and (table[-1, 8:].double() - angle.sin()).abs().max() <= 2.0**-24 * 1.01


# ---- norms and rotation -------------------------------------------------------------------------------------------------

NORM_ROPE = [
    # rows, q heads, k heads, dim, rotary, interleaved, norm, type
    (1, 1, 1, 128, 128, False, True, BF16),
    (37, 4, 2, 128, 64, False, True, BF16),
    (300, 3, 3, 64, 64, True, True, F16),
    (65, 8, 1, 32, 16, False, False, F16),
    (129, 2, 2, 80, 32, False, True, F32),
    (50, 5, 1, 8, 8, True, True, F32),
    (33, 2, 1, 256, 256, False, True, BF16),
    (9, 1, 2, 512, 48, True, True, F16),
    (1000, 1, 1, 16, 16, False, True, BF16),
    (77, 2, 3, 104, 0, False, True, BF16),
    (20, 20, 10, 64, 32, False, True, F32),
]


def _norm_rope_inputs(case, seed=0):
    rows, hq, hk, dim, rotary, interleaved, norm, dtype = case
    q, k = _rand(seed + 1, (rows, hq, dim), dtype), _rand(seed + 2, (rows, hk, dim), dtype, 3.0)
    qw, kw = ((1 + 0.2 * _rand(seed + s, (dim,), F32)).to(dtype) if norm else None for s in (3, 4))
    table = torch.randn((500, rotary), generator=torch.Generator().manual_seed(seed + 5)).tanh() if rotary else None
    pos = torch.randint(0, 500, (rows,), generator=torch.Generator().manual_seed(seed + 6)) if rotary else None
    return q, k, pos, table, qw, kw, interleaved


def _to(dev, *ts):
    return [t.to(dev) if isinstance(t, torch.Tensor) else t for t in ts]


@pytest.mark.gpu
@pytest.mark.parametrize("case", NORM_ROPE, ids=str)
def test_norm_rope_and_its_gradients(pkg, dev, case):
    print(f"[case] norm and rotation {case}", flush=True)
    dtype = case[-1]
    q, k, pos, table, qw, kw, inter = _norm_rope_inputs(case)
    dq, dk = _rand(8, q.shape, dtype), _rand(9, k.shape, dtype)
    on = _to(dev, q, k, pos, table, qw, kw)
    leaves = [t.requires_grad_() for t in (on[0], on[1], on[4], on[5]) if t is not None]
    got = pkg.qk_norm_rope(*on, eps=1e-3, interleaved=inter)
    grads = torch.autograd.grad(got, leaves, (dq.to(dev), dk.to(dev)))
    with torch.no_grad():
        again = pkg.qk_norm_rope(*on, eps=1e-3, interleaved=inter)
    torch.cuda.synchronize()
    for i, (x, w, dy) in enumerate(((q, qw, dq), (k, kw, dk))):
        args = (w, 1e-3, table, pos, inter)
        assert got[i].dtype == dtype and got[i].is_contiguous() and torch.equal(got[i], again[i])
        _within(got[i], O.norm_rope(x, *args), O.norm_rope_bound(x, dtype, *args), "qk"[i])
        dx, dw, _ = O.norm_rope_grad(x, dy, *args)
        dx_bound, dw_bound = O.norm_rope_grad_bounds(x, dy, dtype, *args)
        _within(grads[i], dx, dx_bound, "d" + "qk"[i])
        if w is not None:
            _within(grads[2 + i], dw, dw_bound, "dw of " + "qk"[i])


@pytest.mark.gpu
def test_norm_rope_takes_views_and_copies_the_rest(pkg, dev):
    """Column slices in place; rows that do not lie on 16 bytes, negative or expanded strides, a single row of any stride by a copy; q alone;
    int32 positions; gradients through all of them."""
    print("[case] norm and rotation: layouts", flush=True)
    case = (41, 2, 2, 64, 32, False, True, BF16)
    q, k, pos, table, qw, kw, _ = _norm_rope_inputs(case)
    args = (1e-6, table, pos)
    wide = torch.zeros((41, 5, 64), dtype=BF16)
    wide[:, 1:3], wide[:, 3:] = q, k
    odd = torch.zeros((41, 2 * 64 + 3), dtype=BF16)
    odd[:, 3:] = q.flatten(1)
    wide, odd, qd, kd, posd, tabled, qwd, kwd = _to(dev, wide, odd, q, k, pos, table, qw, kw)
    forms = {
        "slices": (wide[:, 1:3], wide[:, 3:]),
        "odd": (odd[:, 3:].view(41, 2, 64), kd),
        "transposed": (qd.transpose(0, 1).contiguous().transpose(0, 1), kd.flip(1).flip(1)),
        "inner": (qd.transpose(1, 2).contiguous().transpose(1, 2), kd),
    }
    for name, (a, b) in forms.items():
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        y = pkg.qk_norm_rope(a, b, posd.int(), tabled, qwd, kwd)
        ga, gb = torch.autograd.grad(y, (a, b), (torch.ones_like(y[0]).transpose(0, 1).contiguous().transpose(0, 1), y[1].new_ones(()).expand_as(y[1])))
        for i, (x, w, g) in enumerate(((q, qw, ga), (k, kw, gb))):
            _within(y[i], O.norm_rope(x, w, *args), O.norm_rope_bound(x, BF16, w, *args), name)
            one = torch.ones_like(x)
            _within(g, O.norm_rope_grad(x, one, w, *args)[0], O.norm_rope_grad_bounds(x, one, BF16, w, *args)[0], name + " gradient")
    alone, none = pkg.qk_norm_rope(qd, None, posd, tabled)
    assert none is None
    _within(alone, O.norm_rope(q, None, *args), O.norm_rope_bound(q, BF16, None, *args), "q alone")
    row = torch.as_strided(qd, (1, 2, 64), (7, 64, 1))
    _within(pkg.qk_norm_rope(row, None, posd[:1], tabled)[0], O.norm_rope(q[:1], None, 1e-6, table, pos[:1]),
            O.norm_rope_bound(q[:1], BF16, None, 1e-6, table, pos[:1]), "one row")
    empty = pkg.qk_norm_rope(qd[:0], kd[:0], posd[:0], tabled)
    assert empty[0].shape == (0, 2, 64) and empty[1].shape == (0, 2, 64)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_norm_rope_positions_outside_of_the_table_and_partial_gradients(pkg, dev, monkeypatch):
    print("[case] norm and rotation: positions outside, one output's gradient", flush=True)
    q, k, pos, table, qw, kw, _ = _norm_rope_inputs((12, 2, 1, 32, 32, False, True, BF16))
    q, k, pos, table, qw, kw = _to(dev, q, k, pos, table, qw, kw)
    want = pkg.qk_norm_rope(q, k, pos, table, qw, kw)
    pos2 = pos.clone()
    pos2[3], pos2[7] = -1, 500
    got = pkg.qk_norm_rope(q, k, pos2, table, qw, kw)
    for a, b in zip(got, want):
        assert torch.isnan(a[[3, 7]]).all() and torch.equal(a[[0, 1, 2, 4, 5, 6, 8, 9, 10, 11]], b[[0, 1, 2, 4, 5, 6, 8, 9, 10, 11]])
    monkeypatch.setenv("HSTU_HIP_CHECK_CONTRACT", "1")
    with pytest.raises(ValueError, match="positions"):
        pkg.qk_norm_rope(q, k, pos2, table, qw, kw)
    assert torch.equal(pkg.qk_norm_rope(q, k, pos, table, qw, kw)[0], want[0])
    monkeypatch.delenv("HSTU_HIP_CHECK_CONTRACT")
    leaves = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
    y = pkg.qk_norm_rope(leaves[0], leaves[1], pos, table, leaves[2], leaves[3])
    dk = torch.randn_like(y[1])
    only = torch.autograd.grad(y[1], leaves, dk, allow_unused=True, retain_graph=True)
    both = torch.autograd.grad(y, leaves, (torch.zeros_like(y[0]), dk))
    assert only[0] is None and only[2] is None and torch.equal(only[1], both[1]) and torch.equal(only[3], both[3])
    frozen = pkg.qk_norm_rope(q, leaves[1], pos, table, qw, leaves[3])
    assert torch.equal(torch.autograd.grad(frozen[1], leaves[3], dk)[0], both[3])
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope_leaves_an_infinity_where_it_is(pkg, dev, interleaved):
    """Columns that do not turn are what they were, infinities too; those that turn with one are not numbers or infinite."""
    print(f"[case] norm and rotation: an infinity {interleaved}", flush=True)
    q, _, pos, table, *_ = _norm_rope_inputs((6, 2, 1, 64, 32, interleaved, False, BF16))
    q[2, 1, 40], q[3, 0, 4] = float("inf"), float("-inf")
    got = pkg.qk_norm_rope(q.to(dev), None, pos.to(dev), table.to(dev), interleaved=interleaved)[0].cpu()
    assert torch.equal(got[..., 32:], q[..., 32:])
    pair = [4, 5 if interleaved else 20]
    rest = [i for i in range(32) if i not in pair]
    assert not torch.isfinite(got[3, 0, pair]).any() and torch.isfinite(got[3, 0, rest]).all() and torch.isfinite(got[2, 1, :32]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_rope_of_odd_rows(pkg, dev, dtype):
    """Rows of zeros, tiny and huge rows, a NaN: what the formula gives in fp32, rounded once, and the row's neighbours as they are without it."""
    print(f"[case] norm and rotation: odd rows {dtype}", flush=True)
    x = _rand(1, (8, 2, 64), dtype)
    x[0] = 0
    x[1] = x[1] * 1e-30  # squares below all numbers
    x[2] = x[2] * 1e25  # squares above all numbers
    x[3, 0, 7] = float("nan")
    x[4] = x[4] * 1e12
    w = 1 + 0.1 * _rand(2, (64,), dtype)
    for eps in (1e-6, 0.0):
        got = pkg.qk_norm_rope(x.to(dev), None, None, None, w.to(dev), eps=eps)[0].float().cpu()
        f = x.float()
        mean = (f * f).mean(-1, keepdim=True) + eps
        want = f * mean.rsqrt() * w.float()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        # the mean of 64 squares: 7 additions and 2 products; its root twice half of that; two products; the rounding to the type
        bound = (4.5 + 2 + 2) * 2.0**-24 + torch.finfo(dtype).eps / 2
        near = torch.isfinite(want)
        assert ((got - want).abs()[near] <= 1.01 * bound * want.abs()[near] + 1e-37).all()
        assert torch.equal(got[~near & ~torch.isnan(want)], want[~near & ~torch.isnan(want)])


@pytest.mark.gpu
def test_norm_rope_gradients_against_differences_of_the_kernel(pkg, dev):
    """<gradient, direction> against central differences of the kernel's own results, fp32.  With h = 2^-6 and directions of size one: the third
    derivative leaves h^2 / 6 of some units, 2^-12 of the sum's size; the roundings 2^-22 / 2h of it, less."""
    print("[case] norm and rotation: differences", flush=True)
    rows, dim, h = 23, 48, 2.0**-6
    q, k, qw, kw = (_rand(i, shape, F32).to(dev) for i, shape in enumerate(((rows, 3, dim), (rows, 1, dim), (dim,), (dim,))))
    turns, at = pkg.make_rotary_table(50, 32, device=dev), torch.arange(rows, device=dev) * 2
    up = [_rand(9 + i, x.shape, F32).to(dev) for i, x in enumerate((q, k))]
    leaves = [x.clone().requires_grad_() for x in (q, k, qw, kw)]

    def value(q, k, qw, kw):
        a, b = pkg.qk_norm_rope(q, k, at, turns, qw, kw, interleaved=True)
        return (a.double() * up[0]).sum() + (b.double() * up[1]).sum()

    grads = torch.autograd.grad(value(*leaves), leaves)
    for i, g in enumerate(grads):
        way = _rand(20 + i, g.shape, F32).to(dev)
        moved = [[x + s * h * way if j == i else x for j, x in enumerate((q, k, qw, kw))] for s in (1, -1)]
        slope = (value(*moved[0]) - value(*moved[1])) / (2 * h)
        size = (g.double() * way).abs().sum()
        assert abs(float(slope - (g.double() * way).sum())) <= 2.0**-10 * float(size), i


@pytest.mark.gpu
def test_rows_past_32_bit_offsets(pkg, dev):
    """More than 2^31 values in q and in K: the last rows are those that a call on them alone gives, forward, backward and in the cache."""
    print("[case] rows past 2^31 values", flush=True)
    heads, dim, page, tail = 8, 128, 1024, 300
    rows = 2**31 // (heads * dim) + 77
    x = torch.empty((rows, heads, dim), dtype=BF16, device=dev)
    x[: rows - tail] = 1
    x[rows - tail :] = _rand(1, (tail, heads, dim), BF16).to(dev)
    w, turns = (1 + 0.1 * _rand(2, (dim,), BF16)).to(dev), pkg.make_rotary_table(4096, dim, device=dev)
    at = torch.arange(rows, device=dev) % 4096
    got = []
    for q, pos in ((x, at), (x[rows - tail :].clone(), at[rows - tail :].clone())):
        q = q.detach().requires_grad_()
        y = pkg.qk_norm_rope(q, None, pos, turns, w)[0]
        dq = torch.autograd.grad(y, q, q.detach())[0]
        got.append((y.detach()[-tail:].clone(), dq[-tail:].clone()))
        del y, dq, q
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    pages = -(-rows // page)
    cache = pkg.allocate_paged_kv_cache(pages, page, heads, dim, 32, BF16, dev)
    v = x[:, :, 32:64]
    table, zero = torch.arange(pages, dtype=torch.int32, device=dev).view(1, -1), torch.zeros(1, dtype=torch.int64, device=dev)
    pkg.append_paged_kv(cache, x, v, table, zero, None, turns, at, w)
    k_all, v_all = pkg.read_paged_kv(cache, rows, table, zero)
    few = pkg.allocate_paged_kv_cache(1, page, heads, dim, 32, BF16, dev)
    pkg.append_paged_kv(few, x[rows - tail :], v[rows - tail :], zero.int().view(1, 1), zero, None, turns, at[rows - tail :].clone(), w)
    k_few, v_few = pkg.read_paged_kv(few, tail, zero.int().view(1, 1), zero)
    torch.cuda.synchronize()
    assert torch.equal(k_all[-tail:], k_few) and torch.equal(v_all[-tail:], v_few)


@pytest.mark.gpu
def test_norm_rope_refusals(pkg, dev):
    q, k, pos, table, qw, kw, _ = _norm_rope_inputs((12, 2, 1, 32, 32, False, True, BF16))
    q, k, pos, table, qw, kw = _to(dev, q, k, pos, table, qw, kw)
    for bad in ((q[0], k, pos, table), (q, k[:5], pos, table), (q, k, None, table), (q, k, pos[:3], table), (q, k, pos.float(), table), (q, k, pos, table.double()),
                (q, k, pos, table, qw[:5]), (q, k, pos, table, qw.float()), (q, None, pos, table, qw, kw), (q, k), (q, k.half(), pos, table), (q.double(), None, pos, table),
                (q, k, pos, torch.cat([table, table], 1))):
        with pytest.raises(AssertionError):
            pkg.qk_norm_rope(*bad)
    with pytest.raises(NotImplementedError):
        pkg.qk_norm_rope(q, k, pos, table[:, :24])
    with pytest.raises(NotImplementedError):
        pkg.qk_norm_rope(q, k, pos, table.clone().requires_grad_())
    with pytest.raises(NotImplementedError):
        pkg.qk_norm_rope(torch.zeros(2, 1, 12, device=dev), None, pos[:2], table[:, :8], interleaved=True)


# ---- rows into and out of the cache -------------------------------------------------------------------------------------

APPEND = [
    # new rows of each sequence, rows already there, heads, dqk, dv, page, type
    ([1], [0], 1, 128, 128, 16, BF16),
    ([5, 0, 33, 1, 0, 0], [3, 9, 15, 40, 0, 5], 3, 64, 128, 16, F16),
    ([100, 17, 64, 200], [0, 0, 0, 0], 2, 128, 32, 64, BF16),
    ([1] * 70, list(range(70)), 4, 32, 32, 32, BF16),
    ([3, 300, 2], [600, 1, 127], 1, 256, 256, 128, F16),
]


def _append_inputs(case, seed=0):
    new, held, heads, dqk, dv, page, dtype = case
    lengths = [a + b for a, b in zip(new, held)]
    table, pages = O.page_table(seed + 1, lengths, page)
    rows = sum(new)
    k, v = _rand(seed + 2, (rows, heads, dqk), dtype), _rand(seed + 3, (rows, heads, dv), dtype, 0.4)
    offs = torch.tensor([0] + new).cumsum(0)
    cache = O.fill_cache(seed + 4, pages, heads, page, dqk, dv, dtype)
    of = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
    place = torch.tensor(held)[of] + torch.arange(rows) - offs[of]
    return k, v, table, torch.tensor(held), offs, cache, of, place


@pytest.mark.gpu
@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{len(c[0])}x{c[2]}x{c[3]}x{c[4]}p{c[5]}")
def test_rows_are_stored_and_read_exactly(pkg, dev, case):
    """Without norm and rotation the codes, steps and lowest values are the definition's, bit by bit, ties included; every other byte of the
    cache is left as it was; reading gives their values, rounded once."""
    print(f"[case] cache rows {case}", flush=True)
    k, v, table, start, offs, cache, of, place = _append_inputs(case)
    page, dtype = case[5], case[-1]
    k[:, :, : 16] = torch.arange(16).to(dtype) / 2  # rows with ties between codes
    at = (table.long()[of, place // page], slice(None), place % page)
    want = [c.clone() for c in cache]
    for i, x in ((0, k), (2, v)):
        code, step, low = O.four_bits(x)
        want[i][at], want[i + 1][at] = O.pack(code), torch.cat([step, low], -1).to(dtype)
    for i64 in (False, True):
        on = [c.to(dev) for c in cache]
        index = (lambda t: t.to(dev)) if i64 else (lambda t: t.int().to(dev))
        args = (index(table), index(start))
        pkg.append_paged_kv(tuple(on), k.to(dev), v.to(dev), *args, seq_offsets=index(offs))
        kk, vv = pkg.read_paged_kv(pkg.PagedKVCache(*on), k.shape[0], *args, seq_offsets=index(offs))
        torch.cuda.synchronize()
        for got, ref in zip(on, want):
            assert torch.equal(got.cpu().view(torch.uint8), ref.view(torch.uint8))
        assert torch.equal(kk.cpu(), O.values(want[0][at], want[1][at]).to(dtype)) and torch.equal(vv.cpu(), O.values(want[2][at], want[3][at]).to(dtype))


def _held_bound(x, y, dtype, *args):
    """How far a row is from ``y``, norm and rotation of ``x``, once it is held: half a step, 16 roundings of the step to the type (15 at the
    far end), those of the row itself and of its extremes, and the one of the value that is read."""
    u = O.half_step(dtype)
    step = (y.amax(-1, keepdim=True) - y.amin(-1, keepdim=True)) / 15
    row = O.norm_rope_bound(x, dtype, *args).amax(-1, keepdim=True)
    return (0.5 + 16 * u) * step * (1 + 4 * u) + 2 * row + 2 * u * y.abs().amax(-1, keepdim=True)


@pytest.mark.gpu
@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{len(c[0])}x{c[2]}x{c[3]}x{c[4]}p{c[5]}")
@pytest.mark.parametrize("interleaved,norm,given", [(False, True, False), (True, False, True)])
def test_rows_are_normed_and_rotated_on_the_way(pkg, dev, case, interleaved, norm, given):
    """K as it is held against the 64-bit row: half a step (and the step's rounding: 15 steps of it at the far end), the rounding to the
    type, fp32's."""
    print(f"[case] cache rows with rotation {case} {interleaved} {norm} {given}", flush=True)
    k, v, table, start, offs, cache, of, place = _append_inputs(case, 50)
    dtype, dqk = case[-1], case[3]
    turns = torch.randn((900, dqk if interleaved else dqk // 2), generator=torch.Generator().manual_seed(7)).tanh()
    w = (1 + 0.2 * _rand(8, (dqk,), F32)).to(dtype) if norm else None
    pos = torch.randint(0, 900, (k.shape[0],), generator=torch.Generator().manual_seed(9)) if given else None
    on = [c.to(dev) for c in cache]
    kd, vd, tab, st, of_, turns_d, wd, posd = _to(dev, k, v, table, start, offs, turns, w, pos)
    pkg.append_paged_kv(on, kd, vd, tab, st, of_, turns_d, posd, wd, eps=1e-3, interleaved=interleaved)
    kk, vv = pkg.read_paged_kv(on, k.shape[0], tab, st, of_)
    torch.cuda.synchronize()
    args = (w, 1e-3, turns, place if pos is None else pos, interleaved)
    y = O.norm_rope(k, *args)
    _within(kk, y, _held_bound(k, y, dtype, *args), "k")
    code, st_, low = O.four_bits(v)
    assert torch.equal(vv.cpu(), (low + st_ * code).to(dtype))


@pytest.mark.gpu
def test_rows_without_a_place(pkg, dev, monkeypatch):
    """Rows behind the last sequence, places past the page table and pages that are none store nothing; reading gives zeros and NaN.
    Rows with a NaN or an infinity become NaN, constant rows are exact, a range as wide as the type is held, the rest is untouched."""
    print("[case] cache rows without a place, odd values", flush=True)
    heads, dim, page = 2, 64, 16
    table = torch.tensor([[4, 99], [2, -1], [0, 1]], dtype=torch.int32)
    offs, start = torch.tensor([0, 20, 22, 40]), torch.tensor([0, 15, 20])  # 0: second page is none; 1: the same; 2: past its two pages
    k, v = _rand(1, (45, heads, dim), BF16), _rand(2, (45, heads, dim), BF16)
    k[3, 0, 5], k[4, 1, 0], k[5, 0] = float("nan"), float("inf"), 3.0
    v[6, 1, :2], v[7, 0, :2] = torch.tensor([-3e38, 3e38]), torch.tensor([1e-38, 1e-40])
    v[8], v[9], k[10], k[11] = v[8] * 1e-38, v[9] * 1e-30, k[10] * 1e30, 1 + k[11] / 300  # steps below the normal numbers, far ones, few of them
    cache = O.fill_cache(3, 5, heads, page, dim, dim, BF16)
    on = [c.to(dev) for c in cache]
    args = _to(dev, table, start)
    pkg.append_paged_kv(on, k.to(dev), v.to(dev), *args, seq_offsets=offs.to(dev))
    kk, vv = pkg.read_paged_kv(on, 45, *args, seq_offsets=offs.to(dev))
    torch.cuda.synchronize()
    stored = [(i, 4, i) for i in range(16)] + [(20, 2, 15)] + [(22 + i, 1, 4 + i) for i in range(12)]
    want = [c.clone() for c in cache]
    for i, p, at in stored:
        for j, x in ((0, k), (2, v)):
            code, step, low = O.four_bits(x[i])
            want[j][p, :, at], want[j + 1][p, :, at] = O.pack(code), torch.cat([step, low], -1).to(BF16)
    has = [i for i, _, _ in stored]
    none = [i for i in range(40) if i not in has]
    for i, (got, w) in enumerate(zip(on, want)):
        got = got.cpu()
        nan = torch.isnan(want[i | 1][..., :1].float())  # rows that are NaN: their codes say nothing
        assert ((got == w) | nan).all() and (i % 2 == 0 or torch.equal(torch.isnan(got), torch.isnan(w))), i
    assert torch.isnan(kk[none]).all() and torch.isnan(vv[none]).all() and (kk[40:] == 0).all() and (vv[40:] == 0).all()
    assert torch.isnan(kk[3, 0]).all() and torch.isnan(kk[4, 1]).all() and (kk[5, 0] == 3).all() and torch.isfinite(vv[6, 1]).all()
    assert torch.isfinite(kk[3, 1]).all() and torch.isfinite(kk[4, 0]).all()
    monkeypatch.setenv("HSTU_HIP_CHECK_CONTRACT", "1")
    with pytest.raises(ValueError):
        pkg.append_paged_kv(on, k.to(dev), v.to(dev), *args, seq_offsets=offs.to(dev))
    with pytest.raises(ValueError):
        pkg.read_paged_kv(on, 45, *args, seq_offsets=offs.to(dev))
    good = (on, k[:3].to(dev), v[:3].to(dev), table[:, :1].contiguous().to(dev), torch.tensor([0, 1, 2], device=dev))
    pkg.append_paged_kv(*good)
    turns = torch.ones((2, 16), device=dev)
    with pytest.raises(ValueError):
        pkg.append_paged_kv(*good, rotary_table=turns)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_cache_refusals(pkg, dev):
    cache = pkg.allocate_paged_kv_cache(4, 16, 2, 64, 32, device=dev)
    k, v = torch.zeros((6, 2, 64), dtype=BF16, device=dev), torch.zeros((6, 2, 32), dtype=BF16, device=dev)
    table, start = torch.zeros((3, 2), dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    pkg.append_paged_kv(cache, k[:0], v[:0], table, start)
    assert pkg.read_paged_kv(cache, 0, table, start)[1].shape == (0, 2, 32)
    for bad in ((cache, v, v, table, start), (cache, k, v[:5], table, start), (cache, k.half(), v.half(), table, start), (cache, k[:5], v[:5], table, start),
                (cache, k, v, table.float(), start), (cache, k, v, table[0], start), (cache, k, v, table, start[:2]), (cache[:3], k, v, table, start),
                (cache, k, v, table, start, start), ((cache[0],) * 4, k, v, table, start), (cache, k, v, table[:0], start[:0])):
        with pytest.raises((AssertionError, TypeError, RuntimeError)):
            pkg.append_paged_kv(*bad)
    with pytest.raises(NotImplementedError):
        pkg.append_paged_kv(cache, k.clone().requires_grad_(), v, table, start)
    with pytest.raises(AssertionError):
        pkg.read_paged_kv(cache, 7, table, start)
    q = torch.zeros((6, 4, 64), dtype=BF16, device=dev)
    lengths = start + 5
    for bad in ((16, 1.0, q[:, :3], cache, table, lengths), (16, 1.0, q[:5], cache, table, lengths), (0, 1.0, q, cache, table, lengths), (16, 1.0, q.half(), cache, table, lengths),
                (16, 1.0, q, cache, table, lengths[:2]), (16, 1.0, q, cache, table, lengths, start[:1]), (16, 1.0, q, cache, table, lengths, None, -1)):
        with pytest.raises(AssertionError):
            pkg.delta_hstu_mha_paged(*bad)
    with pytest.raises(NotImplementedError):
        pkg.delta_hstu_mha_paged(16, 1.0, q.clone().requires_grad_(), cache, table, lengths)
    assert pkg.delta_hstu_mha_paged(16, 1.0, q[:0], cache, table, lengths).shape == (0, 4, 32)
    torch.cuda.synchronize()


# ---- attention over the cache -------------------------------------------------------------------------------------------

ATTENTION = [
    # lengths, delta, targets, window, contextual, q heads, heads, dqk, dv, page, type
    ([1], 1, None, 0, 0, 1, 1, 128, 128, 16, BF16),
    ([400], 1, None, 0, 0, 4, 4, 128, 128, 16, BF16),
    ([33, 0, 1, 64, 700], 1, None, 0, 0, 2, 2, 64, 64, 32, F16),
    ([300, 17, 5, 0, 96], 7, [7, 7, 3, 0, 1], 0, 0, 3, 3, 128, 128, 64, BF16),
    ([300, 20, 65], 16, [16, 10, 0], 50, 0, 2, 1, 32, 128, 16, BF16),
    ([512, 90, 40], 33, [33, 33, 20], 64, 6, 8, 2, 64, 32, 32, F16),
    ([1500, 260], 130, [130, 130], 0, 4, 2, 2, 128, 128, 128, BF16),
    ([1500, 260], 130, [100, 0], 300, 4, 4, 2, 128, 64, 64, F16),
    ([90, 700], 40, None, 0, 8, 2, 2, 256, 256, 16, BF16),
    ([90, 700, 10], 3, [2, 3, 1], 100, 2, 2, 2, 256, 256, 1024, F16),
    ([40, 61, 35], 35, [5, 0, 12], 0, 10, 1, 1, 32, 32, 16, BF16),  # contextual rows among the newest
    ([3000, 2900, 31], 20, [20, 0, 20], 7, 0, 1, 1, 64, 128, 256, BF16),
    ([2100] * 3, 300, [300] * 3, 0, 0, 1, 1, 64, 64, 64, BF16),
    ([700, 90, 333], 132, [0, 90, 132], 200, 5, 1, 1, 64, 128, 32, F16),
    ([400, 97], 24, None, 90, 0, 1, 1, 128, 128, 16, BF16),
    ([513, 512, 511, 1], 4, [4, 4, 0, 0], 0, 0, 4, 2, 128, 128, 64, F16),
    ([2000, 33], 2, None, 0, 0, 4, 2, 128, 64, 16, BF16),
]


def _attention_inputs(case, seed=0):
    lengths, delta, targets, w, c, hq, heads, dqk, dv, page, dtype = case
    table, pages = O.page_table(seed + 1, lengths, page)
    cache = O.fill_cache(seed + 2, pages, heads, page, dqk, dv, dtype)
    q = _rand(seed + 3, (len(lengths) * delta, hq, dqk), dtype)
    return q, cache, table, torch.tensor(lengths), None if targets is None else torch.tensor(targets)


@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTENTION, ids=str)
def test_attention_over_the_cache(pkg, dev, case):
    print(f"[case] attention over the cache {case}", flush=True)
    q, cache, table, lengths, targets = _attention_inputs(case)
    w, c, dqk, dtype = case[3], case[4], case[7], case[-1]
    N, alpha = max(case[0]), dqk**-0.5
    want, bound = O.attention(N, alpha, q, cache, table, lengths, targets, w, c, dtype)
    for splits, i64 in ((0, False), (1, True), (5, False)):
        index = (lambda t: None if t is None else t.to(dev) if i64 else t.int().to(dev))
        args = (N, alpha, q.to(dev), tuple(x.to(dev) for x in cache), index(table), index(lengths), index(targets), w, c)
        got = pkg.delta_hstu_mha_paged(*args, kv_splits=splits)
        again = pkg.delta_hstu_mha_paged(*args, kv_splits=splits)
        torch.cuda.synchronize()
        assert torch.equal(got, again), "two runs differ"
        _within(got, want, bound, f"splits {splits}")


@pytest.mark.gpu
@pytest.mark.parametrize("dqk,dv,dtype", [(128, 128, BF16), (64, 128, F16), (32, 64, BF16), (128, 32, F16), (256, 256, BF16), (64, 64, F16)])
def test_attention_around_the_kernels_numbers_of_rows(pkg, dev, dqk, dv, dtype):
    """Every number of rows at which another kernel, or another tile of one, takes over; ragged lengths around chunks and pages."""
    for i, rows in enumerate((2, 3, 4, 5, 8, 9, 12, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 193)):
        print(f"[case] attention, {rows} rows {dqk} {dv} {dtype}", flush=True)
        group = 2 if rows % 2 == 0 and i % 3 else 1
        delta = rows // group
        lengths = [delta + 31 * i, delta, 1100 + 7 * i, delta + 512 - 32 * (i % 3)]
        targets, w, c = ([delta, 0, delta // 2, 1], 0, 0) if i % 2 else (None, 150 + i, 3 if delta < 60 else 0)
        case = (lengths, delta, targets, w, c, group, 1, dqk, dv, 16 << (i % 4), dtype)
        q, cache, table, n, t = _attention_inputs(case, seed=10 * i)
        if c and targets is None:
            n = n.clamp(min=c)
        N = max(lengths)
        want, bound = O.attention(N, dqk**-0.5, q, cache, table, n, t, w, c, dtype)
        args = (N, dqk**-0.5, q.to(dev), tuple(x.to(dev) for x in cache), table.to(dev), n.to(dev), None if t is None else t.to(dev), w, c)
        for splits in (0, 2):
            got = pkg.delta_hstu_mha_paged(*args, kv_splits=splits)
            torch.cuda.synchronize()
            _within(got, want, bound, f"{rows} rows, splits {splits}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_masked_places_and_bad_pages(pkg, dev, dtype, monkeypatch):
    """NaN rows that nobody sees (behind the sequence, outside of the window, other targets) change nothing; those that are seen, a page that is
    none and a sequence without room give NaN in their own sequence only; q with rows anywhere."""
    print(f"[case] attention: masked places {dtype}", flush=True)
    case = ([300, 150, 77], 5, [5, 2, 5], 60, 2, 2, 2, 64, 64, 16, dtype)
    q, cache, table, lengths, targets = _attention_inputs(case)
    cache = [c.clone() for c in cache]
    for b, n in enumerate(lengths.tolist()):
        seen = hstu_oracle._seq_mask_rows(n, n - 5, n, int(targets[b]), 60, 2, 0).any(0)
        for place in range(int(table.shape[1]) * 16):
            if place >= n and table[b, place // 16] >= 0 or place < n and not seen[place]:
                for i in (1, 3):
                    cache[i][int(table[b, place // 16]), :, place % 16] = float("nan")
    want, bound = O.attention(300, 0.125, q, cache, table, lengths, targets, 60, 2, dtype)
    buf = torch.zeros((15, 7, 64), dtype=dtype, device=dev)
    buf[:, 2:4] = q.to(dev)
    on = tuple(c.to(dev) for c in cache)
    args = (on, table.to(dev), lengths.to(dev), targets.to(dev), 60, 2)
    good = pkg.delta_hstu_mha_paged(300, 0.125, buf[:, 2:4], *args)
    _within(good, want, bound, "masked NaN")
    # targets see themselves but not each other: a NaN in one's own row is one's own
    own = [c.clone() for c in cache]
    own[3][int(table[0, 297 // 16]), :, 297 % 16] = float("nan")
    got = pkg.delta_hstu_mha_paged(300, 0.125, q.to(dev), tuple(c.to(dev) for c in own), *args[1:])
    assert torch.isnan(got[2]).all() and torch.equal(got[[0, 1, 3, 4] + list(range(5, 15))], good[[0, 1, 3, 4] + list(range(5, 15))])
    bad = table.clone()
    bad[1, 8] = 10**6
    longer = lengths.clone()
    longer[0] = 16 * table.shape[1] + 1
    for splits in (0, 3):
        good_s = pkg.delta_hstu_mha_paged(300, 0.125, q.to(dev), *args, kv_splits=splits)
        got = pkg.delta_hstu_mha_paged(300, 0.125, q.to(dev), on, bad.to(dev), *args[2:], kv_splits=splits)
        assert torch.isnan(got[5:10]).all() and torch.equal(got[:5], good_s[:5]) and torch.equal(got[10:], good_s[10:])
        got = pkg.delta_hstu_mha_paged(300, 0.125, q.to(dev), on, table.to(dev), longer.to(dev), *args[3:], kv_splits=splits)
        assert torch.isnan(got[:5]).all() and torch.equal(got[5:], good_s[5:])
    monkeypatch.setenv("HSTU_HIP_CHECK_CONTRACT", "1")
    for a in ((on, bad.to(dev), *args[2:]), (on, table.to(dev), longer.to(dev), *args[3:])):
        with pytest.raises(ValueError):
            pkg.delta_hstu_mha_paged(300, 0.125, q.to(dev), *a)
    assert torch.equal(pkg.delta_hstu_mha_paged(300, 0.125, q.to(dev), *args), good)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_attention_of_sequences_shorter_than_the_newest_rows(pkg, dev):
    print("[case] attention: short sequences", flush=True)
    for delta, hq in ((40, 2), (4, 1)):
        case = ([3, 0, 50], delta, [1, 0, 2], 0, 1, hq, 1, 64, 32, 16, BF16)
        q, cache, table, lengths, targets = _attention_inputs(case)
        want, bound = O.attention(50, 0.3, q, cache, table, lengths, targets, 0, 1)
        got = pkg.delta_hstu_mha_paged(50, 0.3, q.to(dev), tuple(c.to(dev) for c in cache), *_to(dev, table, lengths, targets), 0, 1)
        torch.cuda.synchronize()
        _within(got, want, bound, f"delta {delta}")
        assert (got[: delta - 3] == 0).all() and (got[delta : 2 * delta] == 0).all()


@pytest.mark.gpu
def test_padded_batches_pass_the_contract_checks(pkg, dev, monkeypatch):
    """Sequences without new rows, of no length at all, or shorter than the newest rows are allowed calls; checks on, they give the same."""
    print("[case] padded batches", flush=True)
    heads, dim, page = 1, 32, 16
    cache = pkg.allocate_paged_kv_cache(6, page, heads, dim, dim, BF16, dev)
    table = torch.tensor([[0, 1], [2, 3], [4, -1], [-1, -1]], dtype=torch.int32, device=dev)
    k, v = _rand(1, (34, heads, dim), BF16).to(dev), _rand(2, (34, heads, dim), BF16).to(dev)
    turns = pkg.make_rotary_table(20, 16, device=dev)
    offs, zero = torch.tensor([0, 20, 20, 34, 34], device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    lengths, targets = torch.tensor([20, 0, 14, 0], device=dev), torch.tensor([3, 0, 3, 0], device=dev)
    q = _rand(3, (4 * 16, 2, dim), BF16).to(dev)
    got = []
    for check in ("0", "1"):
        monkeypatch.setenv("HSTU_HIP_CHECK_CONTRACT", check)
        pkg.append_paged_kv(cache, k, v, table, zero, offs, turns)
        got.append([*pkg.read_paged_kv(cache, 34, table, zero, offs), pkg.delta_hstu_mha_paged(20, 0.2, q, cache, table, lengths, targets, 0, 2)])
    torch.cuda.synchronize()
    for a, b in zip(*got):
        assert torch.equal(a, b) and torch.isfinite(a).all()
    assert (got[0][2][16:32] == 0).all() and (got[0][2][32:34] == 0).all() and (got[0][2][48:] == 0).all()


@pytest.mark.gpu
def test_attention_of_large_scores(pkg, dev):
    """Scores far on both sides of silu: what vanishes is zero, what is large is large, nothing overflows on the way in either type."""
    print("[case] attention: large scores", flush=True)
    for dtype in (BF16, F16):
        case = ([200, 90], 3, None, 0, 0, 2, 2, 64, 64, 16, dtype)
        q, cache, table, lengths, _ = _attention_inputs(case)
        q = q * 40
        want, bound = O.attention(200, 2.0, q, cache, table, lengths, dtype=dtype)
        got = pkg.delta_hstu_mha_paged(200, 2.0, q.to(dev), tuple(c.to(dev) for c in cache), *_to(dev, table, lengths))
        torch.cuda.synchronize()
        _within(got, want, bound, str(dtype))


@pytest.mark.gpu
def test_a_cache_beyond_32_bit_offsets(pkg, dev):
    """Pages that lie past 2^32 bytes of codes: appended, read and attended to as in a small cache."""
    print("[case] a long cache", flush=True)
    heads, dqk, dv, page, N = 1, 128, 64, 1024, 2048
    pages = 70000  # 4.6 GB of K codes
    big = (torch.empty((pages, heads, page, dqk // 2), dtype=torch.uint8, device=dev), torch.empty((pages, heads, page, 2), dtype=BF16, device=dev),
           torch.empty((pages, heads, page, dv // 2), dtype=torch.uint8, device=dev), torch.empty((pages, heads, page, 2), dtype=BF16, device=dev))
    small = pkg.allocate_paged_kv_cache(6, page, heads, dqk, dv, BF16, dev)
    near = torch.tensor([[3, 0], [5, 1], [2, 4]], dtype=torch.int32)
    far = near + (pages - 6)
    lengths = torch.tensor([2048, 1500, 40])
    offs = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]).to(dev)
    k, v = _rand(1, (int(lengths.sum()), heads, dqk), BF16).to(dev), _rand(2, (int(lengths.sum()), heads, dv), BF16).to(dev)
    zero = torch.zeros(3, dtype=torch.int64, device=dev)
    got = []
    for cache, table in ((small, near), (big, far)):
        table = table.to(dev)
        pkg.append_paged_kv(cache, k, v, table, zero, offs)
        out = list(pkg.read_paged_kv(cache, k.shape[0], table, zero, offs))
        for delta in (1, 12, 100):
            q = _rand(10 + delta, (3 * delta, 2, dqk), BF16).to(dev)
            out.append(pkg.delta_hstu_mha_paged(N, 0.1, q, cache, table, lengths.to(dev)))
        got.append(out)
    torch.cuda.synchronize()
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert torch.isfinite(got[0][-1]).all()


@pytest.mark.gpu
def test_attention_of_many_sequences_and_tables_of_any_layout(pkg, dev):
    """More sequences than a workgroup ranks, tables that are columns of a wider one, calls on two streams at once."""
    print("[case] attention: many sequences", flush=True)
    rng = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 90, (300,), generator=rng).tolist()
    for delta, hq in ((1, 1), (17, 1), (40, 2)):
        case = (lengths, delta, None, 0, 0, hq, 1, 32, 32, 16, BF16)
        q, cache, table, n, _ = _attention_inputs(case)
        want, bound = O.attention(90, 0.2, q, cache, table, n)
        wide = torch.full((300, 3 * table.shape[1]), 10**6, dtype=torch.int32)
        wide[:, 2 : 2 + table.shape[1]] = table
        wide, spread = wide.to(dev), torch.full((300, table.shape[1], 2), 10**6, dtype=torch.int64)
        spread[:, :, 0] = table
        on = tuple(c.to(dev) for c in cache)
        first = pkg.delta_hstu_mha_paged(90, 0.2, q.to(dev), on, wide[:, 2 : 2 + table.shape[1]], n.to(dev))
        second = pkg.delta_hstu_mha_paged(90, 0.2, q.to(dev), on, spread.to(dev)[:, :, 0], n.to(dev))
        _within(first, want, bound, f"delta {delta}")
        assert torch.equal(first, second)
        streams = [torch.cuda.Stream() for _ in range(2)]
        args = (90, 0.2, q.to(dev), on, table.to(dev), n.to(dev))
        torch.cuda.synchronize()
        beside = []
        for _ in range(3):
            for st in streams:
                with torch.cuda.stream(st):
                    beside.append(pkg.delta_hstu_mha_paged(*args, kv_splits=3))
        torch.cuda.synchronize()
        assert all(torch.equal(b, beside[0]) for b in beside)


# ---- together -----------------------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prefill_steps_and_candidates_through_one_cache(pkg, dev, dtype):
    """Histories appended with rotation, then steps of one row, then candidates put over the same places: after each the attention over
    the cache against the 64-bit one on what the cache holds, and against the 16-bit operator on the rows read back."""
    print(f"[case] a cache in use {dtype}", flush=True)
    heads, dim, page, N = 2, 64, 16, 128
    held = torch.tensor([40, 0, 77])
    cache = pkg.allocate_paged_kv_cache(3 * (N // page), page, heads, dim, dim, dtype, dev)
    table = torch.randperm(3 * (N // page), generator=torch.Generator().manual_seed(1)).view(3, -1).to(dev)
    turns = pkg.make_rotary_table(N, dim, device=dev)
    w = (1 + 0.1 * _rand(2, (dim,), F32)).to(dtype).to(dev)
    offs = torch.cat([torch.zeros(1, dtype=torch.int64), held.cumsum(0)]).to(dev)
    rows = int(held.sum())
    x = _rand(3, (rows, 2 * heads, dim), dtype).to(dev)
    pkg.append_paged_kv(cache, x[:, :heads], x[:, heads:], table, torch.zeros(3, dtype=torch.int64, device=dev), offs, turns, None, w)
    lengths = held.to(dev)
    for step, delta in enumerate((1, 1, 9, 9)):
        candidates = delta > 1
        q, k, v = (_rand(10 + 3 * step + i, (3 * delta, heads, dim), dtype).to(dev) for i in range(3))
        pos = (lengths.view(-1, 1) + (0 if candidates else torch.arange(delta, device=dev))).expand(3, delta).reshape(-1)
        q, _ = pkg.qk_norm_rope(q, None, pos, turns, w)
        pkg.append_paged_kv(cache, k, v, table, lengths, None, turns, pos, w)
        now = lengths + delta
        targets = torch.full((3,), delta, device=dev) if candidates else None
        out = pkg.delta_hstu_mha_paged(N, dim**-0.5, q, cache, table, now, targets, 0, 0)
        host = tuple(c.cpu() for c in cache)
        want, bound = O.attention(N, dim**-0.5, q.cpu(), host, table.cpu(), now.cpu(), None if targets is None else targets.cpu(), dtype=dtype)
        _within(out, want, bound, f"step {step}")
        all_offs = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), now.cumsum(0)])
        kk, vv = pkg.read_paged_kv(cache, int(now.sum()), table, torch.zeros_like(now), all_offs)
        plain = pkg.delta_hstu_mha(N, dim**-0.5, q, kk, vv, all_offs, targets)
        torch.cuda.synchronize()
        assert float((plain.float() - out.float()).norm() / out.float().norm()) < 1e-2  # (values and P rounded to the type there)
        if not candidates:
            lengths = now
    # the second step's rows are still what they were, under the candidates that came after them
    args = (w.cpu(), 1e-6, turns.cpu(), held + 1)
    fresh = O.norm_rope(_rand(14, (3, heads, dim), dtype), *args)
    row, _ = pkg.read_paged_kv(cache, 3, table, held.to(dev) + 1)
    _within(row, fresh, _held_bound(_rand(14, (3, heads, dim), dtype), fresh, dtype, *args), "the second step's K")


@pytest.mark.gpu
def test_steps_replayed_from_a_graph_and_on_another_stream(pkg, dev):
    """A step captured once and replayed for new rows and lengths, two graphs that share nothing but the cache, eager work between; the same
    on a stream of its own."""
    print("[case] a step in a graph", flush=True)
    heads, dim, page, N, B = 4, 128, 64, 2048, 3
    table, pages = O.page_table(5, [N] * B, page)
    cache = tuple(c.to(dev) for c in O.fill_cache(6, pages, heads, page, dim, dim, BF16))
    table = table.to(dev)
    turns = pkg.make_rotary_table(N, dim, device=dev)
    w = (1 + 0.1 * _rand(7, (dim,), F32)).bfloat16().to(dev)
    q, k, v = (torch.zeros((B, heads, dim), dtype=BF16, device=dev) for _ in range(3))
    start = torch.zeros(B, dtype=torch.int64, device=dev)

    def step():
        r, _ = pkg.qk_norm_rope(q, None, start, turns, w)
        pkg.append_paged_kv(cache, k, v, table, start, None, turns, None, w)
        return pkg.delta_hstu_mha_paged(N, dim**-0.5, r, cache, table, start + 1)

    def inputs(seed):
        for t, s in ((q, 0), (k, 1), (v, 2)):
            t.copy_(_rand(100 * seed + s, t.shape, BF16))
        start.copy_(torch.tensor([seed * 7, 900 + seed, 2000 - seed]))

    inputs(1)
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    other = torch.cuda.Stream()
    for seed in range(2, 7):
        inputs(seed)
        torch.cuda.synchronize()
        eager = step().clone()
        g, out = graphs[seed % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), f"replay {seed}"
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            beside = step()
        other.synchronize()
        assert torch.equal(beside, eager), f"another stream {seed}"


@pytest.mark.gpu
def test_a_training_step_replayed_from_a_graph(pkg, dev):
    print("[case] norm and rotation forward and backward in a graph", flush=True)
    q, k, pos, table, qw, kw, _ = _norm_rope_inputs((200, 4, 2, 128, 128, False, True, BF16))
    leaves = [t.to(dev).requires_grad_() for t in (q, k, qw, kw)]
    pos, table = pos.to(dev), table.to(dev)
    dy = [torch.zeros_like(t) for t in leaves[:2]]

    def step():
        y = pkg.qk_norm_rope(leaves[0], leaves[1], pos, table, leaves[2], leaves[3])
        grads = torch.autograd.grad(y, leaves, dy)
        return [t.detach() for t in y] + list(grads)  # (no graph of these leaves outlives a step)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in range(4):
        for t, s in zip(dy, (1, 2)):
            t.copy_(_rand(50 * seed + s, t.shape, BF16))
        eager = [t.clone() for t in step()]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)
