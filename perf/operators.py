"""The serving path with rotated positions and a cache in 4 bits, and its training step, as cases that can be timed.

A case is a dict of plain values; ``op`` says which call of the user's it is:

* ``rope``        norms of q and k for each head with the position rotation, as the step between producer and attention
* ``rope_train``  the same step forward and backward: its outputs, the gradients of q, k and of both norm weights
* ``append``      new K and V rows rounded to 4 bits into the pages of a cache, K normed and rotated on the way; what is
                  returned is what the cache then holds for these rows, read back from its pages as values
* ``attention``   the newest ``delta`` positions of every sequence against the whole of it in such a cache

Where ``own`` is false the operators are computed in their plain form.  The shape of a case (lengths) depends on the case
alone, through ``shape_seed``; values and the order of pages on the seed that ``prepare`` gets.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
# Every field that not all cases name, with the value that stands for "not used".
DEFAULTS = {
    "dtype": "bf16", "batch": 1, "lo": 1, "hi": 1, "heads": 4, "kv_heads": 0, "dqk": 128, "dv": 128, "norm": True, "rotary": 0,
    "interleaved": False, "fused": False, "page": 64, "new": 0, "delta": 1, "targets": False, "window": 0, "contextual": 0, "shape_seed": 0,
}


def _full(case):
    c = dict(DEFAULTS, **case)
    c["kv_heads"] = c["kv_heads"] or c["heads"]
    return c


def listed():
    return [
        # One step of generation for a small batch: one new row for each of 32 sequences.  Latency and nothing else.
        dict(name="rope_step", op="rope", batch=32, lo=1, hi=1, rotary=128),
        # A ragged prefill as the producer leaves it: q and k column slices of one buffer, half of each head rotated in
        # neighbouring pairs, no norms, the second data type and the smaller head.
        dict(name="rope_prefill_fp16", op="rope", dtype="fp16", batch=96, lo=20, hi=1023, heads=8, dqk=64, norm=False, rotary=32, interleaved=True,
             fused=True, shape_seed=2),
        # A training batch of ordinary histories, both norms learned.
        dict(name="rope_train", op="rope_train", batch=48, lo=200, hi=2048, rotary=128, shape_seed=6),
        # The largest: long histories, twice the heads for q as for k.
        dict(name="rope_train_long", op="rope_train", batch=32, lo=1024, hi=8192, heads=8, kv_heads=4, rotary=64, shape_seed=1006),
        # ... and the operator tests' third type on a small odd batch with the smallest head.
        dict(name="rope_train_fp32", op="rope_train", dtype="fp32", batch=16, lo=1, hi=257, heads=3, dqk=32, rotary=32, shape_seed=7),
        # One step of generation: a new row for each of 64 sequences into caches of any length so far.
        dict(name="append_step", op="append", batch=64, lo=1, hi=4096, new=1, rotary=128, page=64, shape_seed=8),
        # The second baseline batch as a prefill: whole histories into an empty cache.
        dict(name="append_prefill", op="append", batch=256, lo=64, hi=1024, rotary=128, page=64, shape_seed=1002),
        # Long histories of eight heads, values as column slices of the producer's buffer, fp16, larger pages, no norm.
        dict(name="append_prefill_fp16", op="append", dtype="fp16", batch=16, lo=4096, hi=16384, heads=8, norm=False, rotary=64, interleaved=True,
             fused=True, page=128, shape_seed=1005),
        # One user's next row against a short history: launches and the host's work.
        dict(name="attention_one_user", op="attention", batch=1, lo=401, hi=401, page=16, shape_seed=1),
        # One step of generation for many long histories: the cache's bytes and nothing else.
        dict(name="attention_step", op="attention", batch=128, lo=4096, hi=16384, heads=8, page=64, shape_seed=9),
        # A serving micro-batch: 32 users, 256 candidates each, which see the history and themselves.
        dict(name="attention_candidates", op="attention", batch=32, lo=1280, hi=4352, delta=256, targets=True, page=64, shape_seed=1004),
        # A few heavy users in the second type: an odd number of candidates, a window, a contextual prefix, four heads of q to one of k.
        dict(name="attention_long_fp16", op="attention", dtype="fp16", batch=5, lo=8000, hi=16000, heads=8, kv_heads=2, dqk=64, dv=128, delta=33,
             targets=True, window=4096, contextual=6, page=32, shape_seed=3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    while True:
        op = rng.choice(["rope", "rope_train", "rope_train", "append", "append", "attention", "attention", "attention"])
        c = dict(op=op, shape_seed=rng.randrange(1 << 20), batch=_log_int(rng, 1, 256))
        c["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
        c["dqk"] = rng.choice([128, 128, 64, 32])
        c["kv_heads"] = rng.choice([1, 2, 3, 4, 8])
        c["heads"] = c["kv_heads"] if op == "append" else c["kv_heads"] * rng.choice([1, 1, 2, 4])
        c["hi"] = _log_int(rng, 1, 8192 if op.startswith("rope") else 16384)
        c["lo"] = max(1, int(c["hi"] * rng.choice([0.0, 0.06, 0.5, 1.0])))
        if op != "attention":
            c["rotary"] = rng.choice([0, c["dqk"] // 2, c["dqk"], c["dqk"]])
            c["norm"] = c["rotary"] == 0 or rng.random() < 0.6
            c["interleaved"] = rng.random() < 0.3
            c["fused"] = op != "rope_train" and rng.random() < 0.5
        if op.startswith("rope") and rng.random() < 0.2:
            c["dtype"] = "fp32"
        if op in ("append", "attention"):
            c["dv"] = c["dqk"] if rng.random() < 0.7 else rng.choice([32, 64, 128])
            c["page"] = rng.choice([16, 32, 64, 64, 128])
        if op == "append":
            c["new"] = rng.choice([0, 1, 7, 100])
        if op == "attention":
            c["delta"] = rng.choice([1, 1, 2, 5, 16, _log_int(rng, 1, 512)])
            c["targets"] = rng.random() < 0.5
            c["contextual"] = rng.choice([0, 0, 6])
            c["lo"] = max(c["lo"], c["delta"] + c["contextual"])
            c["hi"] = max(c["hi"], c["lo"])
            c["window"] = rng.choice([0, 0, max(1, c["hi"] // 4)])
        w, f = work(c), _full(c)
        padded = f["batch"] * f["hi"] * (f["kv_heads"] * (f["dqk"] + f["dv"]) + f["heads"] * f["delta"])  # values of the plain attention
        if w["bytes"] <= 1.0e9 and w["flops"] <= 5.0e10 and (op != "attention" or padded <= 4.0e9):
            return c


# ---- shapes and work ----------------------------------------------------------------------------------------------------


def _lengths(c):
    """Lengths of the sequences in the cache, or of the new rows where those are all that there is."""
    rng = np.random.RandomState(c["shape_seed"])
    return rng.randint(c["lo"], c["hi"] + 1, size=c["batch"]).astype(np.int64)


def _pairs(c, n):
    """(query, key) pairs of the newest ``delta`` positions of sequences of these lengths, and the keys that any of them sees."""
    pairs = keys = 0
    for length in n.tolist():
        at = np.arange(max(0, length - c["delta"]), length)
        u = length - (c["delta"] if c["targets"] else 0)
        ctx, w = c["contextual"], c["window"] or (1 << 40)
        ids = np.minimum(np.maximum(at - ctx + 1, 0) if ctx else at, u - ctx + 1 if ctx else u)
        seen = np.minimum(ids, w) + 1 if not ctx else np.where(ids == 0, u, np.minimum(w, ids - 1) + np.where(ids <= w, ctx, 0) + 1)
        pairs += int(seen.sum())
        keys += int(min(length, (w if c["window"] else length) + c["delta"] + ctx))
    return pairs, keys


def work(case):
    c = _full(case)
    n = _lengths(c)
    es = 4 if c["dtype"] == "fp32" else 2
    dq, dv = c["dqk"], c["dv"]
    if c["op"] in ("rope", "rope_train"):
        rows = int(n.sum())
        values = rows * (c["heads"] + c["kv_heads"]) * dq
        table = 4 * c["rotary"] * int(n.max()) + 8 * rows
        if c["op"] == "rope":
            return {"bytes": 2.0 * es * values + table, "flops": 7.0 * values}
        return {"bytes": 4.0 * es * values + table, "flops": 21.0 * values}
    held = c["kv_heads"] * (dq / 2 + dv / 2 + 8)  # bytes of a position: codes, and step and lowest value of each K and V row
    if c["op"] == "append":
        rows = c["batch"] * c["new"] if c["new"] else int(n.sum())
        values = rows * c["kv_heads"] * (dq + dv)
        return {"bytes": 2.0 * es * values + 2.0 * held * rows + 4 * c["rotary"] * min(rows, c["hi"]), "flops": 12.0 * values}
    pairs, keys = _pairs(c, n)
    rows = c["batch"] * c["delta"]
    return {"bytes": held * keys + es * rows * c["heads"] * (dq + dv), "flops": 2.0 * (dq + dv) * c["heads"] * pairs}


# ---- inputs -------------------------------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rotary_table(positions, width):
    """cos | sin of position * 10000 ** (-2 i / width), angles in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, width, 2, dtype=torch.float64, device="cuda") / width)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda").view(-1, 1) * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _fused_columns(rows, widths, dtype, g):
    """Column slices of one buffer, as the producer of u, v, q, k leaves them."""
    buf = torch.randn((rows, sum(widths)), generator=g, device="cuda").to(dtype)
    return list(torch.split(buf, widths, dim=1))


def _pages_for(c, n, g):
    """A table with the pages of every sequence in some order, and how many pages the cache has."""
    each = -(-n // c["page"])
    total = int(each.sum())
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.zeros((c["batch"], int(each.max())), dtype=torch.int32)
    at = 0
    for b, count in enumerate(each.tolist()):
        table[b, :count] = order[at : at + count]
        at += count
    return table.cuda(), total


def _cache_of(c, pages, g):
    """Pages of rows of ordinary spread, K rows with a mean of their own as normed and rotated keys have it."""
    dt = DTYPES[c["dtype"]]
    parts = []
    for width, spread in ((c["dqk"], 1.0), (c["dv"], 0.5)):
        codes = torch.empty((pages, c["kv_heads"], c["page"], width // 2), dtype=torch.uint8, device="cuda")
        scales = torch.empty((pages, c["kv_heads"], c["page"], 2), dtype=dt, device="cuda")
        step = max(1, (1 << 26) // (c["kv_heads"] * c["page"] * width))
        for p in range(0, pages, step):
            x = torch.randn(codes[p : p + step].shape[:3] + (width,), generator=g, device="cuda") * spread
            codes[p : p + step], scales[p : p + step] = _to_four_bits(x.to(dt))
        parts += [codes, scales]
    return tuple(parts)


def prepare(case, seed):
    c = _full(case)
    g = _generator(seed)
    dt = DTYPES[c["dtype"]]
    n = _lengths(c)
    h, hk, d, dv = c["heads"], c["kv_heads"], c["dqk"], c["dv"]
    s = {"case": c}
    if c["norm"] and c["op"] != "attention":
        s["q_weight"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt)
        s["k_weight"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt)
    if c["rotary"]:
        s["table"] = _rotary_table(int(n.max()), c["rotary"])
    if c["op"] in ("rope", "rope_train"):
        rows = int(n.sum())
        if c["hi"] == 1:  # a step of generation: every sequence at a place of its own
            s["table"] = _rotary_table(4096, c["rotary"]) if c["rotary"] else None
            s["positions"] = torch.randint(0, 4096, (rows,), generator=g, device="cuda")
        else:
            s["positions"] = torch.cat([torch.arange(int(x)) for x in n]).cuda()
        if c["fused"]:
            _, _, q, k = _fused_columns(rows, [hk * dv, hk * dv, h * d, hk * d], dt, g)
        else:
            q, k = (torch.randn((rows, x * d), generator=g, device="cuda").to(dt) for x in (h, hk))
        s["q"], s["k"] = q.view(rows, h, d), k.view(rows, hk, d)
        if c["op"] == "rope_train":
            s["dq"], s["dk"] = (torch.randn((rows, x, d), generator=g, device="cuda").to(dt) for x in (h, hk))
            s["leaves"] = [s[name].requires_grad_() for name in ("q", "k", "q_weight", "k_weight") if name in s]
        return s
    s["pages"], total = _pages_for(c, n, g)
    if c["op"] == "append":
        new = np.minimum(n, c["new"]) if c["new"] else n
        rows, start = int(new.sum()), n - new
        k, v = _fused_columns(rows, [hk * d, hk * dv], dt, g) if c["fused"] else [torch.randn((rows, hk * w), generator=g, device="cuda").to(dt) for w in (d, dv)]
        s["k"], s["v"] = k.view(rows, hk, d), v.view(rows, hk, dv)
        s["start"] = torch.from_numpy(start).cuda()
        s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(new)])).cuda()
        s["cache"] = tuple(
            x for w in (d, dv) for x in (torch.zeros((total, hk, c["page"], w // 2), dtype=torch.uint8, device="cuda"),
                                         torch.zeros((total, hk, c["page"], 2), dtype=dt, device="cuda")))
        return s
    s["cache"] = _cache_of(c, total, g)
    s["lengths"] = torch.from_numpy(n).cuda()
    s["targets"] = torch.full((c["batch"],), c["delta"], dtype=torch.int64, device="cuda") if c["targets"] else None
    s["q"] = torch.randn((c["batch"] * c["delta"], h, d), generator=g, device="cuda").to(dt)
    s["alpha"] = 1.0 / math.sqrt(d)
    s["max_seq_len"] = c["hi"]
    return s


# ---- plain form ---------------------------------------------------------------------------------------------------------


def _rotate(x, cos, sin, interleaved):
    """The first 2 * cos.shape[-1] columns of x [rows, heads, width] turned, in x's precision."""
    half = cos.shape[-1]
    cos, sin = cos.to(x.dtype).unsqueeze(1), sin.to(x.dtype).unsqueeze(1)
    if interleaved:
        a, b = x[..., 0 : 2 * half : 2], x[..., 1 : 2 * half : 2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half : 2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., 2 * half :]], dim=-1)


def _turns(s, positions):
    half = s["case"]["rotary"] // 2
    rows = s["table"][positions]
    return rows[:, :half], rows[:, half:]


def _norm_rope(s, x, weight, positions):
    """Norm and rotation of x's rows in 32 bits, not rounded at the end."""
    x = x.detach().float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight.detach().float()
    if s["case"]["rotary"]:
        x = _rotate(x, *_turns(s, positions), s["case"]["interleaved"])
    return x


def _norm_rope_grad(s, x, weight, positions, dy):
    """Gradients of x and of the norm weight from dy."""
    dtype, x, dy = x.dtype, x.detach().float(), dy.float()
    if s["case"]["rotary"]:
        cos, sin = _turns(s, positions)
        dy = _rotate(dy, cos, -sin, s["case"]["interleaved"])
    if weight is None:
        return dy.to(dtype), None
    r = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
    unit = x * r
    by_unit = dy * weight.detach().float()
    dx = r * (by_unit - unit * (by_unit * unit).mean(dim=-1, keepdim=True))
    return dx.to(dtype), (dy * unit).sum(dim=(0, 1), dtype=torch.float64).to(dtype)


def _to_four_bits(x):
    """Codes, two to a byte, and (step, lowest value) of every row; x in the type that step and lowest value are kept in."""
    dtype, x = x.dtype, x.float()
    low, high = x.amin(dim=-1, keepdim=True), x.amax(dim=-1, keepdim=True)
    step = ((high - low) / 15).to(dtype).float()
    code = torch.where(step > 0, ((x - low) / step).round().clamp(0, 15), torch.zeros_like(x)).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat([step, low], dim=-1).to(dtype)


def _from_four_bits(codes, scales):
    code = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).float()
    return code * scales[..., :1].float() + scales[..., 1:].float()


def _places(s):
    """Sequence and place in it of every new row."""
    offsets, rows = s["offsets"], s["k"].shape[0]
    of = torch.repeat_interleave(torch.arange(offsets.numel() - 1, device=offsets.device), offsets[1:] - offsets[:-1], output_size=rows)
    return of, s["start"][of] + torch.arange(rows, device=offsets.device) - offsets[of]


def _plain_append(s):
    c, cache, dtype = s["case"], s["cache"], s["k"].dtype
    of, place = _places(s)
    page, at = s["pages"][of, place // c["page"]].long(), place % c["page"]
    k = _norm_rope(s, s["k"], s.get("k_weight"), place).to(dtype)
    cache[0][page, :, at], cache[1][page, :, at] = _to_four_bits(k)
    cache[2][page, :, at], cache[3][page, :, at] = _to_four_bits(s["v"])
    return {"k": _from_four_bits(cache[0][page, :, at], cache[1][page, :, at]).to(dtype),
            "v": _from_four_bits(cache[2][page, :, at], cache[3][page, :, at]).to(dtype)}


def _seen(c, lengths, targets, positions):
    """Whether each of the newest ``delta`` positions sees each position: [batch, delta, positions]."""
    at = (lengths.view(-1, 1) - c["delta"] + torch.arange(c["delta"], device=lengths.device)).unsqueeze(2)
    col = torch.arange(positions, device=lengths.device).view(1, 1, -1)
    ctx = c["contextual"]
    last = lengths.view(-1, 1, 1) - (targets.view(-1, 1, 1) if targets is not None else 0)
    if ctx:
        last = last - ctx + 1
    row_id, col_id = ((x - ctx + 1).clamp(min=0) if ctx else x for x in (at, col))
    if targets is not None:
        row_id, col_id = torch.minimum(row_id, last), torch.minimum(col_id, last)
    far = row_id - col_id
    seen = (at == col) | (far > 0)
    if c["window"]:
        seen = seen & (far <= c["window"])
    if ctx:
        seen = seen | ((row_id == 0) & (col_id < last))
    return seen & (col < lengths.view(-1, 1, 1)) & (at >= 0)


def _plain_attention(s):
    c = s["case"]
    batch, delta, h, hk = c["batch"], c["delta"], c["heads"], c["kv_heads"]
    pages = s["pages"].long()

    def rows_of(codes, scales):
        x = _from_four_bits(codes[pages], scales[pages])  # [batch, pages, heads, page, width]
        return x.transpose(1, 2).flatten(2, 3)

    k, v = rows_of(*s["cache"][:2]), rows_of(*s["cache"][2:])
    q = s["q"].float().view(batch, delta, hk, h // hk, -1).permute(0, 2, 1, 3, 4).flatten(2, 3)  # rows of one K head side by side
    score = torch.matmul(q, k.transpose(2, 3)) * s["alpha"]
    seen = _seen(c, s["lengths"], s["targets"], k.shape[2]).repeat_interleave(h // hk, dim=1).unsqueeze(1)
    p = torch.where(seen, score / (1 + torch.exp(-score)) / s["max_seq_len"], torch.zeros_like(score))
    v = torch.where((torch.arange(v.shape[2], device=v.device) < s["lengths"].view(-1, 1)).view(batch, 1, -1, 1), v, torch.zeros_like(v))
    out = torch.matmul(p, v)
    return out.view(batch, hk, delta, h // hk, -1).permute(0, 2, 1, 3, 4).reshape(batch * delta, h, -1).to(s["q"].dtype)


def _plain(s):
    op = s["case"]["op"]
    if op == "append":
        return _plain_append(s)
    if op == "attention":
        return {"out": _plain_attention(s)}
    out = {}
    for x, weight in (("q", s.get("q_weight")), ("k", s.get("k_weight"))):
        out[x] = _norm_rope(s, s[x], weight, s["positions"]).to(s[x].dtype)
        if op == "rope_train":
            out["d" + x], dw = _norm_rope_grad(s, s[x], weight, s["positions"], s["d" + x])
            if dw is not None:
                out["d" + x + "_weight"] = dw
    return out


# ---- the framework's calls ----------------------------------------------------------------------------------------------


def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _own(s):
    c, pkg = s["case"], _package()
    if c["op"] == "append":
        pkg.append_paged_kv(s["cache"], s["k"], s["v"], s["pages"], s["start"], seq_offsets=s["offsets"], rotary_table=s.get("table"),
                            k_weight=s.get("k_weight"), eps=EPS, interleaved=c["interleaved"])
        k, v = pkg.read_paged_kv(s["cache"], s["k"].shape[0], s["pages"], s["start"], seq_offsets=s["offsets"])
        return {"k": k, "v": v}
    if c["op"] == "attention":
        return {"out": pkg.delta_hstu_mha_paged(s["max_seq_len"], s["alpha"], s["q"], s["cache"], s["pages"], s["lengths"], num_targets=s["targets"],
                                                max_attn_len=c["window"], contextual_seq_len=c["contextual"])}
    q, k = pkg.qk_norm_rope(s["q"], s["k"], s["positions"], s.get("table"), s.get("q_weight"), s.get("k_weight"), eps=EPS, interleaved=c["interleaved"])
    out = {"q": q.detach(), "k": k.detach()}
    if c["op"] == "rope_train":
        got = torch.autograd.grad((q, k), s["leaves"], (s["dq"], s["dk"]))
        out.update(zip(("dq", "dk", "dq_weight", "dk_weight"), got))
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------


def _exact_turn(x, angle_rows, interleaved, back=False):
    """x [rows, heads, width] as complex numbers times e^(i angle), cos | sin given for each row."""
    half = angle_rows.shape[1] // 2
    z = torch.complex(angle_rows[:, :half].double(), angle_rows[:, half:].double()).unsqueeze(1)
    z = z.conj() if back else z
    head, rest = x[..., : 2 * half], x[..., 2 * half :]
    pairs = head.unflatten(-1, (half, 2)) if interleaved else head.unflatten(-1, (2, half)).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
    turned = turned.flatten(-2) if interleaved else turned.transpose(-1, -2).flatten(-2)
    return torch.cat([turned, rest], dim=-1)


def _exact_norm_rope(s, x, weight, positions):
    y = x.detach().double()
    if weight is not None:
        y = weight.detach().double() * y / (y.square().mean(-1, keepdim=True) + EPS).sqrt()
    return _exact_turn(y, s["table"][positions], s["case"]["interleaved"]) if s["case"]["rotary"] else y


def _exact_rows(x):
    """What rows held in 4 bits stand for: lowest value + step * code, both kept in x's type."""
    rows = x.double()
    low, high = rows.min(-1, keepdim=True).values, rows.max(-1, keepdim=True).values
    step = ((high - low) / 15).to(x.dtype).double()
    code = torch.clamp(torch.round((rows - low) / torch.where(step > 0, step, torch.ones_like(step))), 0, 15)
    return low + step * code


def _exact_attention(s):
    c = s["case"]
    delta, h, hk, page = c["delta"], c["heads"], c["kv_heads"], c["page"]
    out = torch.zeros((c["batch"], delta, h, c["dv"]), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        pages = s["pages"][b, : -(-n // page)].long()

        def rows(codes, scales):
            low4, high4 = codes[pages].long() % 16, codes[pages].long() // 16
            code = torch.stack((low4, high4), -1).reshape(low4.shape[:3] + (-1,)).double()
            x = scales[pages][..., 1:].double() + code * scales[pages][..., :1].double()
            return x.permute(1, 0, 2, 3).reshape(hk, -1, x.shape[-1])[:, :n]

        k, v = rows(*s["cache"][:2]), rows(*s["cache"][2:])
        u = n - (delta if c["targets"] else 0)
        at = torch.arange(n - delta, n, device="cuda").view(-1, 1)
        col = torch.arange(n, device="cuda").view(1, -1)
        ctx, w = c["contextual"], c["window"]
        # by the kind of position: history rows see what is before them, targets see the history and themselves, contextual rows
        # all that is no target
        step = torch.minimum(at, torch.full_like(at, u)) if not ctx else torch.minimum((at - ctx + 1).clamp(min=0), torch.full_like(at, u - ctx + 1))
        age = step - (col if not ctx else (col - ctx + 1).clamp(min=0))
        seen = (col < at) & (col < u) & (age > 0) & ((age <= w) if w else torch.ones_like(age, dtype=torch.bool)) | (col == at)
        if ctx:
            seen = seen | ((at < ctx) & (col < u))
        for head in range(h):
            score = s["alpha"] * (s["q"].view(c["batch"], delta, h, -1)[b, :, head].double() @ k[head * hk // h].T)
            out[b, :, head] = torch.where(seen, score * torch.sigmoid(score), torch.zeros_like(score)) @ v[head * hk // h] / s["max_seq_len"]
    return out.view(c["batch"] * delta, h, -1)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "attention":
        return {"out": _exact_attention(s)}
    if c["op"] == "append":
        _, place = _places(s)
        k = _exact_norm_rope(s, s["k"], s.get("k_weight"), place).to(s["k"].dtype)
        return {"k": _exact_rows(k), "v": _exact_rows(s["v"])}
    out = {}
    for x, weight in (("q", s.get("q_weight")), ("k", s.get("k_weight"))):
        out[x] = _exact_norm_rope(s, s[x], weight, s["positions"])
        if c["op"] == "rope_train":
            dy, y = s["d" + x].double(), s[x].detach().double()
            if c["rotary"]:
                dy = _exact_turn(dy, s["table"][s["positions"]], c["interleaved"], back=True)
            if weight is None:
                out["d" + x] = dy
                continue
            size = (y.square().mean(-1, keepdim=True) + EPS).sqrt()
            g = dy * weight.detach().double()
            out["d" + x] = g / size - y * (g * y).mean(-1, keepdim=True) / size**3
            out["d" + x + "_weight"] = (dy * y / size).sum((0, 1))
    return out
