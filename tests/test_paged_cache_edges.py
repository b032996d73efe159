"""Calls of the rotated positions and the 4-bit paged cache that their documentation allows and that lie off the ordinary path: tables smaller
than the divisor, pages behind a window, empty batches, forward-mode tensors, rows no one owns, and every rule by which the attention cuts a
call into workgroups.  Tolerances are the oracle's bounds, or none where two ways have to give the same bits."""

import pytest
import torch

from oracle import hstu_oracle, paged_oracle as O
from test_paged_cache import _abi, _append_inputs, _norm_rope_inputs, _rand, _to, _within

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


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
