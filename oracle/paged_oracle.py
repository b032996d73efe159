"""Oracle of the rotated positions and the 4-bit paged cache, in 64 bits on the CPU.  TEST INFRASTRUCTURE ONLY.

Written from the definitions in ``include/hstu_cache.h``; the rotation by complex multiplication, the attention by the cached
form of ``hstu_oracle`` (pinned there) on rows taken out of the pages.  ``norm_rope_grad`` is pinned against differences of
``norm_rope``.  Beside each result stands the bound that a kernel's roundings give, from the operations it is known to do.
"""

import numpy as np
import torch

from . import hstu_oracle

F32 = 2.0**-24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rotate(x, table_rows, interleaved, back=False):
    """``x`` ``[rows, heads, dim]`` turned by ``table_rows`` ``[rows, width]`` (cosines | sines)."""
    half = table_rows.shape[1] // 2
    z = (table_rows[:, :half].double() + 1j * table_rows[:, half:].double()).unsqueeze(1)
    z = z.conj() if back else z
    y = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    turned = torch.complex(x[..., a], x[..., b]) * z
    y[..., a], y[..., b] = turned.real, turned.imag
    return y


def norm_rope(x, weight=None, eps=1e-6, table=None, positions=None, interleaved=False):
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    return y if table is None else rotate(y, table[positions.long()], interleaved)


def norm_rope_bound(x, dtype, weight=None, eps=1e-6, table=None, positions=None, interleaved=False):
    """One rounding to ``dtype``, and in fp32: the mean of squares and its root (dim + 4 roundings relative to the row), two
    products, the turn's two products and sum -- of columns no larger than the row's largest pair."""
    y = norm_rope(x, weight, eps, table, positions, interleaved)
    n = norm_rope(x, weight, eps)
    return half_step(dtype) * 1.01 * y.abs() + (x.shape[-1] / 8 + 16) * F32 * 2 * n.abs().amax(-1, keepdim=True) + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2


def norm_rope_grad(x, dy, weight=None, eps=1e-6, table=None, positions=None, interleaved=False):
    """(dx, dweight, sum of the sizes of dweight's terms)"""
    g = dy.double()
    if table is not None:
        g = rotate(g, table[positions.long()], interleaved, back=True)
    if weight is None:
        return g, None, None
    x64 = x.double()
    r = 1 / (x64.square().mean(-1, keepdim=True) + eps).sqrt()
    unit, gw = x64 * r, g * weight.double()
    return r * (gw - unit * (gw * unit).mean(-1, keepdim=True)), (g * unit).sum((0, 1)), (g * unit).abs().sum((0, 1))


def norm_rope_grad_bounds(x, dy, dtype, weight=None, eps=1e-6, table=None, positions=None, interleaved=False, chain=512):
    """dx: one rounding, and fp32's in the turn, the dot product (dim / 8 + lanes' exchanges) and what follows, relative to the largest
    terms of the row.  dweight: one rounding, and ``chain`` additions in a row of terms that are themselves some fp32 roundings off."""
    dx, dw, size = norm_rope_grad(x, dy, weight, eps, table, positions, interleaved)
    tiny = torch.finfo(dtype).smallest_normal * half_step(dtype) * 2
    if weight is None:
        return half_step(dtype) * 1.01 * dx.abs() + 16 * F32 * dy.double().abs().amax(-1, keepdim=True) * 2 + tiny, None
    x64, w = x.double(), weight.double()
    r = 1 / (x64.square().mean(-1, keepdim=True) + eps).sqrt()
    big = 2 * dy.double().abs().amax(-1, keepdim=True) * w.abs().max()
    terms = r * big * (1 + (x64 * r).abs().amax(-1, keepdim=True) ** 2)
    bound = half_step(dtype) * 1.01 * dx.abs() + (x.shape[-1] / 8 + 32) * F32 * terms + tiny
    per_term = 2 * dy.double().abs().amax(-1, keepdim=True) * (x64 * r).abs()
    return bound, half_step(dtype) * 1.01 * dw.abs() + chain * F32 * size + (x.shape[-1] / 8 + 32) * F32 * per_term.sum((0, 1)) + tiny


def four_bits(x):
    """(codes, step, lowest) of rows ``x`` in the type they are kept for, step and lowest rounded to it; all in 64 bits."""
    x64 = x.double()
    low, high = x64.amin(-1, keepdim=True), x64.amax(-1, keepdim=True)
    step = ((high - low) / 15).to(x.dtype).double()
    code = torch.where(step > 0, ((x64 - low) / step.where(step > 0, torch.ones_like(step))).round().clamp(0, 15), torch.zeros_like(x64))
    bad = ~torch.isfinite(x64).all(-1, keepdim=True) | ~torch.isfinite(step)
    nan = torch.full_like(step, float("nan"))
    return code, torch.where(bad, nan, step), torch.where(bad, nan, low)


def pack(code):
    code = code.to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4)


def unpack(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()


def values(codes, scales):
    return scales[..., 1:].double() + scales[..., :1].double() * unpack(codes)


def sequence_rows(cache, table_row, n, which):
    """Rows 0 .. n - 1 of a sequence: codes ``[n, heads, dim]``, step and lowest ``[n, heads, 1]``, in 64 bits."""
    codes, scales = cache[2 * which], cache[2 * which + 1]
    page = codes.shape[2]
    places = torch.arange(n)
    pages = table_row.long()[places // page]
    c = unpack(codes[pages, :, places % page])
    s = scales[pages, :, places % page].double()
    return c, s[..., :1], s[..., 1:]


def attention(max_seq_len, alpha, q, cache, page_table, lengths, targets=None, max_attn_len=0, contextual_seq_len=0, dtype=torch.bfloat16, p_words=None):
    """(out, bound) of the cached form on CPU copies of a cache, ``[batch * delta, q heads, dv]``.  ``p_words``: bf16 words that P times the step is
    kept in (by default one for bf16, two for fp16)."""
    batch = page_table.shape[0]
    delta, hq, heads = q.shape[0] // batch, q.shape[1], cache[0].shape[1]
    group = hq // heads
    dv = 2 * cache[2].shape[3]
    out = torch.zeros((q.shape[0], hq, dv), dtype=torch.float64)
    bound = torch.zeros_like(out)
    # a code enters a product as 128 + code or 16 + code (fp16's scores: 64 + code)
    off_k, off_v = (128.0 if dtype == torch.bfloat16 else 64.0), 128.0
    # P times the step is rounded to bf16: 8 bits of significand, neighbours 2^-7 2^e apart around values of 2^e and more, so off by at most
    # half of that, 2^-8 of the value (2^-9 holds just below 2^(e+1) alone).  Two words: 2^-8 of what the first left out, 2^-16.
    p_round = 2.0**-8 if (p_words or (1 if dtype == torch.bfloat16 else 2)) == 1 else 2.0**-16
    for b in range(batch):
        n = int(lengths[b])
        if n <= 0:
            continue
        kc, ks, kl = sequence_rows(cache, page_table[b], n, 0)
        vc, vs, vl = sequence_rows(cache, page_table[b], n, 1)
        first = max(0, n - delta)
        rows = q[b * delta + (first - (n - delta)) : (b + 1) * delta].double()  # the rows that have a position
        t = 0 if targets is None else int(targets[b])
        seen = hstu_oracle._seq_mask_rows(n, first, n, t, max_attn_len, contextual_seq_len, 0)
        for h in range(hq):
            kh = h // group
            k, v = kl[:, kh] + ks[:, kh] * kc[:, kh], vl[:, kh] + vs[:, kh] * vc[:, kh]
            k, v = torch.nan_to_num(k), torch.nan_to_num(v)
            qh = rows[:, h]
            s = alpha * (qh @ k.T)
            p = torch.where(seen, s * torch.sigmoid(s), torch.zeros_like(s))
            got = p @ v / max_seq_len
            at = slice(b * delta + (first - (n - delta)), (b + 1) * delta)
            out[at, h] = got
            # the score: fp32 sums of products with offset codes, eight roundings of the whole; silu's slope is at most 1.1, its own roundings
            # (exp2, reciprocal, products) some 2^-21 of it
            size_q = qh.abs().sum(-1, keepdim=True)
            ds = abs(alpha) * 8 * F32 * size_q * (ks[:, kh].T * (off_k + 15) * 2 + kl[:, kh].T.abs()).abs()
            dp = torch.where(seen, 1.1 * ds + 2.0**-21 * p.abs() + 2.0**-21 * s.abs() * torch.sigmoid(s) * (1 + s.abs()), torch.zeros_like(s))
            mid = vl[:, kh] + 7.5 * vs[:, kh]
            from_center = (vs[:, kh] * (vc[:, kh] - 7.5)).abs()
            ps = p.abs() @ vs[:, kh].abs()
            err = dp @ torch.nan_to_num(vl[:, kh].abs() + vs[:, kh] * 15) + p_round * (p.abs() @ torch.nan_to_num(from_center))
            adds = n / 32 + 64
            err = err + adds * F32 * (2 * (off_v + 15) * torch.nan_to_num(ps) + p.abs() @ torch.nan_to_num(mid.abs())) + p_round * F32 * torch.nan_to_num(ps)
            bound[at, h] = err / max_seq_len + half_step(dtype) * 1.01 * got.abs() + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2
    return out, bound


def fill_cache(seed, pages, heads, page, dqk, dv, dtype, spread=(1.0, 0.5)):
    """A cache (CPU) of random rows, every page of it."""
    g = torch.Generator().manual_seed(seed)
    parts = []
    for dim, s in ((dqk, spread[0]), (dv, spread[1])):
        x = (torch.randn((pages, heads, page, dim), generator=g) * s + 0.2 * torch.randn((pages, heads, 1, 1), generator=g)).to(dtype)
        code, step, low = four_bits(x)
        parts += [pack(code), torch.cat([step, low], -1).to(dtype)]
    return tuple(parts)


def page_table(seed, lengths, page, columns=None, spare=3):
    """Pages in random order for sequences of these lengths; unused entries of the table are no pages.  (table, pages)"""
    rng = np.random.default_rng(seed)
    each = [-(-int(n) // page) for n in lengths]
    total = sum(each) + spare
    order = rng.permutation(total)
    columns = max(max(each), 1) if columns is None else columns
    table = torch.full((len(each), columns), -1, dtype=torch.int32)
    at = 0
    for b, count in enumerate(each):
        table[b, :count] = torch.from_numpy(order[at : at + count].astype(np.int32))
        at += count
    return table, total
