"""Calls of the rotated positions and the 4-bit paged cache that their documentation allows and that lie off the ordinary path: tables smaller
than the divisor, pages behind a window, empty batches, forward-mode tensors, rows no one owns, and every rule by which the attention cuts a
call into workgroups.  Tolerances are the oracle's bounds, or none where two ways have to give the same bits."""

import pytest
import torch

from oracle import hstu_oracle, paged_oracle as O
from test_paged_cache import _abi, _append_inputs, _norm_rope_inputs, _rand, _to, _within

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# ---- a divisor larger than the table's room -----------------------------------------------------------------------------


def test_scratch_goes_by_the_tables_room():
    """``max_seq_len`` divides the result; no sequence has more positions than its row of the page table has room for.  Scratch memory does not
    grow with a divisor past that room, whichever kernel the number of rows takes (pointers are never followed)."""
    lib, ref, made = _abi()
    at = 1 << 20
    for batch, heads, columns, page in ((64, 8, 128, 64), (32, 4, 8, 64), (1, 1, 1000, 16), (300, 2, 1, 1024)):
        for delta in (1, 8, 12, 24, 64, 257):
            need = []
            for divisor in (columns * page, columns * page + 1, 1 << 20, 2**31 - 1):
                cache = made["HstuPagedCache"](k_codes=at, k_scales=at, v_codes=at, v_scales=at, pages=1 << 16, heads=heads, page_size=page, dqk=128, dv=128, dtype=0, page_table=at,
                                               table_row_stride=columns, table_columns=columns, batch=batch)
                call = made["HstuPagedAttentionArgs"](q=at, q_row_stride=128 * heads, q_head_stride=128, out=at, seq_lengths=at, q_heads=heads, delta_size=delta, max_seq_len=divisor,
                                                      alpha=1.0)
                need.append(lib.hstu_cache_attention_workspace_bytes(ref(cache), ref(call)))
            assert len(set(need)) == 1, (batch, heads, columns, page, delta, need)


@pytest.mark.gpu
def test_any_divisor_is_served(pkg, dev):
    """Divisors of 2^20 and 2^31 - 1 (2^31 in fp32) with a table of 512 positions: the result is that of the divisor 512, scaled by a power of two, in
    the same order of the sums."""
    print("[case] attention: divisors past the table's room", flush=True)
    batch, heads, dim, page, columns = 32, 4, 64, 64, 8
    for delta, hq in ((1, 4), (3, 8), (12, 4), (40, 4)):
        lengths = [delta + (37 * b) % (513 - delta) for b in range(batch)]
        table, pages = O.page_table(delta, lengths, page, columns)
        cache = tuple(c.to(dev) for c in O.fill_cache(delta + 1, pages, heads, page, dim, dim, BF16))
        q, table, n = _to(dev, _rand(delta + 2, (batch * delta, hq, dim), BF16), table, torch.tensor(lengths))
        want = pkg.delta_hstu_mha_paged(512, 0.125, q, cache, table, n)
        for divisor, power in ((1 << 20, 20 - 9), (2**31 - 1, 31 - 9)):
            got = pkg.delta_hstu_mha_paged(divisor, 0.125, q, cache, table, n)
            torch.cuda.synchronize()
            assert torch.equal(got.double(), want.double() * 2.0**-power), (delta, divisor)


# ---- pages that are none ------------------------------------------------------------------------------------------------


def _first_seen(n, delta, targets, w, c):
    """First position that any of the newest ``delta`` rows of a sequence of ``n`` sees."""
    seen = hstu_oracle._seq_mask_rows(n, max(n - delta, 0), n, targets, w, c, 0)
    return int(seen.any(0).nonzero()[0]) if n else 0


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [1, 3, 12, 24, 40, 150])
@pytest.mark.parametrize("page,dtype", [(16, BF16), (64, F16)])
def test_pages_in_front_of_the_window_may_be_gone(pkg, dev, delta, page, dtype, monkeypatch):
    """Pages that lie whole in front of the first position a row sees are not looked at: the table may name anything there, with the contract checks
    on too.  Windows that end anywhere in a chunk of 32 positions."""
    print(f"[case] attention: pages in front of the window {delta} {page} {dtype}", flush=True)
    dim = 32
    for c, w, t in ((0, 41, None), (0, 56, 1), (3, 63, 0), (2, 77, delta)):
        lengths = [700 + 17 * b for b in range(9)] + [delta + c + 20, 0]
        targets = None if t is None else torch.tensor([min(t, n) for n in lengths])
        table, pages = O.page_table(delta, lengths, page)
        cache = tuple(x.to(dev) for x in O.fill_cache(delta + 1, pages, 1, page, dim, dim, dtype))
        q = _rand(delta + 2, (len(lengths) * delta, 1, dim), dtype).to(dev)
        n, tg = torch.tensor(lengths).to(dev), None if targets is None else targets.to(dev)
        gone = table.clone()
        for b, length in enumerate(lengths):
            first = _first_seen(length, delta, None if t is None else int(targets[b]), w, c)
            gone[b, : first // page] = torch.tensor([-1, 10**6, pages], dtype=torch.int32).repeat(100)[: first // page]
        assert int((gone != table).sum()) > 5
        want, bound = O.attention(900, 0.2, q.cpu(), tuple(x.cpu() for x in cache), table, n.cpu(), targets, w, c, dtype)
        for splits in (0, 3):
            for check in ("0", "1"):
                monkeypatch.setenv("HSTU_HIP_CHECK_CONTRACT", check)
                whole = pkg.delta_hstu_mha_paged(900, 0.2, q, cache, table.to(dev), n, tg, w, c, kv_splits=splits)
                got = pkg.delta_hstu_mha_paged(900, 0.2, q, cache, gone.to(dev), n, tg, w, c, kv_splits=splits)
                torch.cuda.synchronize()
                assert torch.equal(got, whole), (c, w, t, splits, check)
                _within(got, want, bound, f"{c} {w} {t}")
        # one page further on is one that a row sees
        b = 4
        first = _first_seen(lengths[b], delta, None if t is None else int(targets[b]), w, c)
        gone[b, first // page] = -1
        monkeypatch.setenv("HSTU_HIP_CHECK_CONTRACT", "1")
        with pytest.raises(ValueError, match="page"):
            pkg.delta_hstu_mha_paged(900, 0.2, q, cache, gone.to(dev), n, tg, w, c)


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [5, 20, 300])
def test_rows_that_see_a_bad_page_are_nan(pkg, dev, delta):
    """A page that is none, among the history or among the targets: every row that sees a position on it is NaN, whatever block it is in, and the
    other sequences are what they were."""
    print(f"[case] attention: bad pages, {delta} rows", flush=True)
    lengths = [delta + 500, delta + 333, delta + 64]
    table, pages = O.page_table(1, lengths, 32)
    cache = tuple(x.to(dev) for x in O.fill_cache(2, pages, 2, 32, 64, 64, BF16))
    q = _rand(3, (3 * delta, 2, 64), BF16).to(dev)
    for t in (0, delta):
        n, tg = torch.tensor(lengths).to(dev), torch.tensor([t] * 3).to(dev)
        good = pkg.delta_hstu_mha_paged(900, 0.2, q, cache, table.to(dev), n, tg)
        for place in (100, lengths[1] - delta, lengths[1] - 1):
            bad = table.clone()
            bad[1, place // 32] = -7
            got = pkg.delta_hstu_mha_paged(900, 0.2, q, cache, bad.to(dev), n, tg)
            torch.cuda.synchronize()
            seen = hstu_oracle._seq_mask_rows(lengths[1], lengths[1] - delta, lengths[1], t, 0, 0, 0)
            on_page = seen[:, place // 32 * 32 : place // 32 * 32 + 32].any(1).to(dev)
            assert torch.isnan(got[delta : 2 * delta][on_page]).all() and bool(on_page.any())
            assert torch.equal(got[:delta], good[:delta]) and torch.equal(got[2 * delta :], good[2 * delta :])


# ---- two ways to one cache ----------------------------------------------------------------------------------------------


def _two_ways(pkg, dev, dqk, dv):
    """K normed and turned on its way into the cache, and by ``qk_norm_rope`` before: the same bytes."""
    print(f"[case] two ways to one cache {dqk} {dv}", flush=True)
    rows, heads, page = 20000, 2, 64
    pages = -(-rows // page)
    turns, zero = pkg.make_rotary_table(rows, dqk, device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    table, at = torch.arange(pages, dtype=torch.int32, device=dev).view(1, -1), torch.arange(rows, device=dev)
    for dtype in (BF16, F16):
        k, v, w = (x.to(dev) for x in (_rand(1, (rows, heads, dqk), dtype), _rand(2, (rows, heads, dv), dtype), (1 + 0.1 * _rand(3, (dqk,), F32)).to(dtype)))
        one, two = (pkg.allocate_paged_kv_cache(pages, page, heads, dqk, dv, dtype, dev) for _ in range(2))
        for table_of, weight, interleaved in ((turns, w, False), (turns, w, True), (None, w, False), (turns, None, False)):
            pkg.append_paged_kv(one, k, v, table, zero, None, table_of, None, weight, interleaved=interleaved)
            ready, _ = pkg.qk_norm_rope(k, None, at, table_of, weight, interleaved=interleaved)
            pkg.append_paged_kv(two, ready, v, table, zero)
            torch.cuda.synchronize()
            for a, b in zip(one, two):
                differ = int((a.view(torch.uint8) != b.view(torch.uint8)).sum())
                assert differ == 0, (dtype, table_of is None, weight is None, interleaved, differ)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_codes_do_not_depend_on_who_normed_and_turned(pkg, dev, dim):
    _two_ways(pkg, dev, dim, dim)


@pytest.mark.gpu
@pytest.mark.parametrize("dqk,dv", [(32, 64), (32, 128), (32, 256), (64, 128), (64, 256), (128, 32), (128, 256), (256, 128)])
def test_codes_do_not_depend_on_the_width_of_v(pkg, dev, dqk, dv):
    _two_ways(pkg, dev, dqk, dv)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_norms_of_a_caches_widths_are_those_of_plain_operators(pkg, dev, dim):
    """At the widths a cache has, the norm in fp32 is bit by bit that of PyTorch's mean, reciprocal root and products, as this image has them (at
    48, 80, 104 or 512 columns it is not: other orders of the sum)."""
    print(f"[case] norm beside plain operators {dim}", flush=True)
    x, w = _rand(1, (20000, 2, dim), F32).to(dev), (1 + 0.1 * _rand(2, (dim,), F32)).to(dev)
    want = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    assert torch.equal(pkg.qk_norm_rope(x, None, None, None, w)[0], want)


# ---- an empty batch, forward mode ---------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_an_empty_batch_gives_gradients_of_zero(pkg, dev):
    """No rows: outputs without rows, and gradients of zero, of the inputs' shapes, for everything that wants one."""
    print("[case] norm and rotation of no rows, backward", flush=True)
    turns = pkg.make_rotary_table(8, 32, device=dev)
    for dtype in (BF16, F32):
        q, k = (torch.empty((0, h, 32), dtype=dtype, device=dev, requires_grad=True) for h in (4, 2))
        qw, kw = (torch.ones(32, dtype=dtype, device=dev, requires_grad=True) for _ in range(2))
        at = torch.empty(0, dtype=torch.int64, device=dev)
        for args, leaves in (((q, k, at, turns, qw, kw), (q, k, qw, kw)), ((q, None, None, None, qw), (q, qw)), ((q, k, None, None, None, kw), (q, k, kw)),
                             ((q.detach(), k.detach(), at, turns, qw, kw), (qw, kw)), ((q, k, at, turns), (q, k))):
            out = pkg.qk_norm_rope(*args)
            assert [None if y is None else (y.shape, y.dtype) for y in out] == [None if x is None else (x.shape, x.dtype) for x in args[:2]]
            grads = torch.autograd.grad([y.sum() for y in out if y is not None and y.requires_grad], leaves)
            for x, g in zip(leaves, grads):
                assert g.shape == x.shape and g.dtype == x.dtype and bool((g == 0).all())


@pytest.mark.gpu
def test_forward_mode_is_refused(pkg, dev):
    """There is no forward derivative: a tensor with a tangent is refused by each operator, with and without grad mode, not answered without it."""
    import torch.autograd.forward_ad as fwd

    print("[case] tensors with tangents", flush=True)
    q, k, pos, table, qw, kw, _ = _norm_rope_inputs((12, 2, 1, 32, 32, False, True, BF16))
    q, k, pos, table, qw, kw = _to(dev, q, k, pos, table, qw, kw)
    cache = pkg.allocate_paged_kv_cache(1, 16, 1, 32, 32, device=dev)
    pages, zero = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    v, n = torch.zeros_like(k), zero + 12
    pkg.append_paged_kv(cache, k, v, pages, zero)
    held = [x.clone() for x in cache]
    want = pkg.qk_norm_rope(q, k, pos, table, qw, kw)
    for grad in (False, True):
        with torch.set_grad_enabled(grad), fwd.dual_level():
            assert torch.equal(pkg.qk_norm_rope(q, k, pos, table, qw, kw)[0], want[0])  # (no tangents: served)
            calls = [(pkg.qk_norm_rope, [q, k, pos, table, qw, kw], i) for i in (0, 1, 3, 4, 5)]
            calls += [(pkg.append_paged_kv, [cache, k, v, pages, zero, None, table, pos, kw], i) for i in (1, 2, 6, 8)]
            calls += [(pkg.delta_hstu_mha_paged, [16, 0.2, q, cache, pages, n], 2)]
            for f, args, i in calls:
                args = list(args)
                args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError):
                    f(*args)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, cache))


# ---- contract checks ----------------------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_positions_of_rows_behind_the_last_sequence_are_no_ones(pkg, dev, monkeypatch):
    """With the contract checks on, positions outside of the table are refused for rows of a sequence and for those alone."""
    print("[case] positions behind the last sequence", flush=True)
    cache = pkg.allocate_paged_kv_cache(4, 16, 1, 32, 32, device=dev)
    k, v = _rand(1, (20, 1, 32), BF16).to(dev), _rand(2, (20, 1, 32), BF16).to(dev)
    pages, zero = torch.tensor([[0, 1], [2, 3]], device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
    offs, turns = torch.tensor([0, 7, 15], device=dev), pkg.make_rotary_table(16, 32, device=dev)
    pos = torch.arange(20, device=dev) % 8
    pos[15:] = torch.tensor([-1, 16, 10**9, 99, -5], device=dev)
    held = []
    for check in ("0", "1"):
        monkeypatch.setenv("HSTU_HIP_CHECK_CONTRACT", check)
        pkg.append_paged_kv(cache, k, v, pages, zero, offs, turns, pos)
        held.append([x.clone() for x in cache])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*held))
    pos[14] = 16
    with pytest.raises(ValueError, match="positions"):
        pkg.append_paged_kv(cache, k, v, pages, zero, offs, turns, pos)


@pytest.mark.gpu
def test_two_rows_for_one_place_are_refused_by_the_checks(pkg, dev, monkeypatch):
    """No two rows of a call may have one place: two sequences that share a page, or one page twice in a sequence.  A shared page that only one of
    them writes to is allowed."""
    print("[case] two rows for one place", flush=True)
    cache = pkg.allocate_paged_kv_cache(6, 16, 1, 32, 32, device=dev)
    k, v = _rand(1, (24, 1, 32), BF16).to(dev), _rand(2, (24, 1, 32), BF16).to(dev)
    monkeypatch.setenv("HSTU_HIP_CHECK_CONTRACT", "1")
    index = lambda *x: torch.tensor(x, device=dev)  # noqa: E731
    for pages, start, offs in ((index([0, 1], [0, 2]), index(0, 0), None), (index([3, 3], [4, 5]), index(0, 0), index(0, 24, 24)), (index([1, 2], [4, 2]), index(16, 20), index(0, 6, 12))):
        with pytest.raises(ValueError, match="one place"):
            pkg.append_paged_kv(cache, k, v, pages, start, offs)
    for pages, start, offs in ((index([0, 1], [0, 2]), index(16, 16), index(0, 10, 20)), (index([0, 1], [0, 2]), index(0, 3), index(0, 3, 8)), (index([5, 1], [5, 2]), index(0, 4), index(0, 4, 9))):
        pkg.append_paged_kv(cache, k, v, pages, start, offs)
    torch.cuda.synchronize()


# ---- how a call is cut into workgroups ----------------------------------------------------------------------------------


def _attend(pkg, dev, lengths, delta, hq, heads, dqk, dv, page, dtype, seed, targets=None, w=0, c=0, splits=(0,), N=None):
    """The attention of random rows against the oracle; results' memory holds NaN before, so that what is not written shows."""
    table, pages = O.page_table(seed, lengths, page)
    cache = O.fill_cache(seed + 1, pages, heads, page, dqk, dv, dtype)
    q, n = _rand(seed + 2, (len(lengths) * delta, hq, dqk), dtype), torch.tensor(lengths)
    t = None if targets is None else torch.tensor(targets)
    N = N or max(lengths)
    want, bound = O.attention(N, dqk**-0.5, q, cache, table, n, t, w, c, dtype)
    on = _to(dev, q, table, n, t)
    cache = tuple(x.to(dev) for x in cache)
    for s in splits:
        for big in (1 << 20, 1 << 26):  # (what the allocator hands out next, for results and for scratch)
            del_me = torch.full((big,), float("nan"), device=dev)
            del del_me
        poison = torch.full((q.shape[0], hq, dv), float("nan"), dtype=dtype, device=dev)
        del poison
        got = pkg.delta_hstu_mha_paged(N, dqk**-0.5, on[0], cache, on[1], on[2], on[3], w, c, kv_splits=s)
        again = pkg.delta_hstu_mha_paged(N, dqk**-0.5, on[0], cache, on[1], on[2], on[3], w, c, kv_splits=s)
        torch.cuda.synchronize()
        _within(got, want, bound, f"splits {s}")
        assert torch.equal(got, again)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 4])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_few_rows_against_long_sequences(pkg, dev, rows, dtype):
    """One to four rows of a head, where a wave goes over several groups of chunks: whole groups that every row sees, the last one short by any
    number of chunks, the next group's loads ahead; with and without a window, a prefix and targets."""
    print(f"[case] attention: {rows} rows, long sequences {dtype}", flush=True)
    group, delta = (2, rows // 2) if rows > 1 else (1, 1)
    for i, (w, c, t) in enumerate(((0, 0, 0), (0, 0, delta), (4700, 0, 0), (2500, 5, delta))):
        # around whole numbers of groups for four waves (16, 8 or 4 chunks of 32 positions each), and anywhere
        lengths = [8192, 8192 + 1, 8192 - 31, 6144 + 32, 5000 + 13 * i, 9000 - i]
        _attend(pkg, dev, lengths, delta, group, 1, 64, 32, 64, dtype, 100 * i + rows, [t] * 6, w, c, (1, 0, 2))
    _attend(pkg, dev, [5120, 7001], delta, group, 1, 128, 128, 16, dtype, 7 + rows, None, 0, 0, (1, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [12, 24])
def test_nine_to_32_rows_against_long_sequences(pkg, dev, delta):
    """Runs in which each of the four waves looks its pages up three times over (32 of its chunks at a time, 4096 positions of the run)."""
    print(f"[case] attention: {delta} rows, long sequences", flush=True)
    for dqk, dv, page, dtype in ((64, 64, 16, F16), (128, 128, 64, BF16)):
        _attend(pkg, dev, [9000, 8193, 8500], delta, 1, 1, dqk, dv, page, dtype, delta + dqk, [delta, 0, 3], 0, 0, (1, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 8])
def test_a_wave_for_each_of_many_short_sequences(pkg, dev, rows):
    """More than 1024 (sequence, head) pairs of at most 17 chunks: a wave each, the last workgroup not full, some sequences empty."""
    print(f"[case] attention: {rows} rows of many short sequences", flush=True)
    lengths = [0 if b % 11 == 3 else 1 + (b * 97) % 500 for b in range(257)]
    for dtype, targets in ((BF16, None), (F16, [min(n, 2) for n in lengths])):
        _attend(pkg, dev, lengths, rows, 5, 5, 32, 32, 16, dtype, rows, targets)


@pytest.mark.gpu
def test_automatic_runs_of_many_long_sequences(pkg, dev):
    """One row each: runs held to 96 chunks, runs of 40, and runs made longer so that no short one is left over."""
    for batch, heads, top in ((48, 4, 9000), (16, 4, 9000), (64, 4, 3080)):
        print(f"[case] attention: runs of {batch} x {heads} up to {top}", flush=True)
        lengths = [top] + [1 + (b * 7919) % top for b in range(1, batch)]
        _attend(pkg, dev, lengths, 1, heads, heads, 32, 32, 64, BF16, batch, N=top)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,heads", [(86, 3), (73, 7), (128, 4), (171, 3), (200, 5), (256, 1), (256, 2), (2, 255)])
def test_blocks_of_every_number_of_workgroups(pkg, dev, batch, heads):
    """More than 32 rows: sequences ranked by length, ties among them, and the second 256 workgroups in reverse where at most 512 run."""
    print(f"[case] attention: {batch * heads} workgroups", flush=True)
    lengths = [40 + (b * 53) % 90 if b % 5 else 77 for b in range(batch)]
    if batch > 2:
        lengths[3], lengths[batch - 1] = 0, 33
    _attend(pkg, dev, lengths, 33, heads, heads, 32, 32, 16, BF16, batch, [min(n, 20) for n in lengths] if heads % 2 else None, splits=(1,))


# ---- the smallest numbers, one weight -----------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_of_the_smallest_numbers(pkg, dev, dtype):
    """Rows whose values, or whose steps, are below the type's normal numbers or at the border: codes, steps and lowest values are the definition's,
    bit by bit, codes above 15 held there, and reading them rounds once."""
    print(f"[case] rows of the smallest numbers {dtype}", flush=True)
    rows, heads, dim, page = 640, 2, 64, 64
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the smallest number there is
    g = torch.Generator().manual_seed(1)
    whole = torch.randint(0, 40, (rows, heads, dim), generator=g).double() * torch.logspace(0, 9, rows, 2, dtype=torch.float64).floor().view(-1, 1, 1)
    k = (whole * tiny).to(dtype)
    v = k - k[:, :, :1] + (torch.randn((rows, heads, 1), generator=g) * 300 * tiny).to(dtype)
    pages = rows // page
    table, zero = torch.randperm(pages, generator=g).to(torch.int32).view(1, -1), torch.zeros(1, dtype=torch.int64, device=dev)
    cache = pkg.allocate_paged_kv_cache(pages, page, heads, dim, dim, dtype, dev)
    pkg.append_paged_kv(cache, k.to(dev), v.to(dev), table.to(dev), zero)
    got = pkg.read_paged_kv(cache, rows, table.to(dev), zero)
    torch.cuda.synchronize()
    places = torch.arange(rows)
    at = (table[0].long()[places // page], slice(None), places % page)
    for i, x in ((0, k), (2, v)):
        code, step, low = O.four_bits(x)
        assert 0 < int((step < torch.finfo(dtype).smallest_normal).sum()) and 0 < int((step > torch.finfo(dtype).smallest_normal).sum())
        scales = torch.cat([step, low], -1).to(dtype)
        assert torch.equal(cache[i].cpu()[at], O.pack(code)) and torch.equal(cache[i + 1].cpu()[at], scales)
        assert torch.equal(got[i // 2].cpu(), O.values(O.pack(code), scales).to(dtype))


@pytest.mark.gpu
def test_one_norm_weight_of_two(pkg, dev):
    """A norm of k alone or of q alone, with and without the rotation: the gradients of what there is."""
    print("[case] norm and rotation: one weight", flush=True)
    q, k, pos, table, qw, kw, _ = _norm_rope_inputs((50, 3, 2, 64, 32, False, True, BF16))
    up = _rand(8, q.shape, BF16), _rand(9, k.shape, BF16)
    for a, b in ((None, kw), (qw, None)):
        for turned in (False, True):
            at, tab = (pos, table) if turned else (None, None)
            on = _to(dev, q, k, at, tab, a, b)
            leaves = [t.requires_grad_() for t in (on[0], on[1], on[4], on[5]) if t is not None]
            y = pkg.qk_norm_rope(*on)
            grads = torch.autograd.grad(y, leaves, _to(dev, *up))
            torch.cuda.synchronize()
            for i, (x, w, dy) in enumerate(((q, a, up[0]), (k, b, up[1]))):
                args = (w, 1e-6, tab, at, False)
                _within(y[i], O.norm_rope(x, *args), O.norm_rope_bound(x, BF16, *args), "qk"[i])
                (dx, dw, _), (dx_bound, dw_bound) = O.norm_rope_grad(x, dy, *args), O.norm_rope_grad_bounds(x, dy, BF16, *args)
                _within(grads[i], dx, dx_bound, "d" + "qk"[i])
                if w is not None:
                    _within(grads[2], dw, dw_bound, "dw of " + "qk"[i])


@pytest.mark.gpu
def test_norm_weights_gradients_keep_their_bits_in_fp32(pkg, dev):
    """A weight's gradient in fp32, 5679 terms a column, relative to its size over the columns.  A term goes through some nine roundings (the mean,
    its root, their product, the turn's three operations, the product, the sum of six in a lane, the partial sum), each off by 0.3 to 0.6 of
    2^-24 in the mean square, independently: three times 0.42, 1.3 of 2^-24 together; sums of hundreds in 32 bits would add three more."""
    print("[case] norm weights' gradients in fp32", flush=True)
    q, k, pos, table, qw, kw, _ = _norm_rope_inputs((1893, 3, 3, 32, 32, False, True, F32), 40)
    up = _rand(8, q.shape, F32), _rand(9, k.shape, F32)
    on = _to(dev, q, k, pos, table, qw, kw)
    leaves = [on[4].requires_grad_(), on[5].requires_grad_()]
    grads = torch.autograd.grad(pkg.qk_norm_rope(*on), leaves, _to(dev, *up))
    torch.cuda.synchronize()
    for x, w, dy, got in ((q, qw, up[0], grads[0]), (k, kw, up[1], grads[1])):
        _, want, _ = O.norm_rope_grad(x, dy, w, 1e-6, table, pos)
        assert float((got.double().cpu() - want).norm() / want.norm()) <= 2 * 2.0**-24


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hq", [(1, 1), (2, 1), (1, 3), (4, 1), (5, 1), (4, 2)])
@pytest.mark.parametrize("dqk,dv", [(128, 128), (32, 64), (64, 32), (256, 256)])
def test_few_rows_are_as_exact_as_their_type(pkg, dev, rows, hq, dqk, dv):
    """Up to eight rows of a head in bf16: P times the step is kept to 16 bits, so that nothing but the result's own rounding is left of bf16."""
    print(f"[case] attention: {rows} x {hq} rows of {dqk} and {dv}, exact", flush=True)
    lengths = [777, 31, 1500, 512, rows]
    table, pages = O.page_table(rows, lengths, 32)
    cache = O.fill_cache(rows + 1, pages, 1, 32, dqk, dv, BF16)
    q, n = _rand(rows + 2, (5 * rows, hq, dqk), BF16), torch.tensor(lengths)
    for targets, w, c in ((None, 0, 0), ([min(m, rows) for m in lengths], 200, 0)):
        t = None if targets is None else torch.tensor(targets)
        want, bound = O.attention(1500, dqk**-0.5, q, cache, table, n, t, w, c, BF16, p_words=2)
        on = _to(dev, q, table, n, t)
        for splits in (0, 1):
            got = pkg.delta_hstu_mha_paged(1500, dqk**-0.5, on[0], tuple(x.to(dev) for x in cache), on[1], on[2], on[3], w, c, kv_splits=splits)
            torch.cuda.synchronize()
            _within(got, want, bound, f"window {w}, splits {splits}")
