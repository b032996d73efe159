"""Blocks of a user's own one behind another: the second norm of ``gated_residual_norm`` is what the next block's products read."""

import pytest
import torch

from oracle import recurrent_oracle as oracle
from test_recurrent import offsets_of


def block_weights(width, d):
    g = torch.Generator().manual_seed(17)
    rnd = lambda *s, by=1.0, add=0.0: add + by * torch.randn(s, generator=g)  # noqa: E731
    p = {}
    for k in range(2):
        p.update({f"in{k}": rnd(d, 3 * width + d, by=d**-0.5), f"out{k}": rnd(width, d, by=width**-0.5), f"post{k}": rnd(d, by=0.1, add=1.0), f"scale{k}": rnd(d, by=0.1, add=0.5),
                  f"pre{k}": rnd(d, by=0.1, add=1.0), f"decay{k}": torch.log(torch.expm1(-torch.log(0.9 + 0.099 * torch.rand(width, generator=g)) / 8.0))})
    return p


def recurrence_in_64_bits(v, r, i, decay, offs):
    z = 8.0 * torch.nn.functional.softplus(decay) * torch.sigmoid(r)
    a, b = torch.exp(-z), torch.sqrt(-torch.expm1(-2 * z)) * torch.sigmoid(i) * v
    rows = []
    for begin, end in zip(offs[:-1].tolist(), offs[1:].tolist()):
        h = torch.zeros_like(b[0])
        for t in range(begin, end):
            h = a[t] * h + b[t]
            rows.append(h)
    return torch.stack(rows)


@pytest.mark.gpu
def test_two_blocks(pkg, dev):
    width, d, lengths = 96, 128, [40, 1, 90]
    offs = offsets_of(lengths)
    p = dict(block_weights(width, d), x=torch.randn(sum(lengths), d, generator=torch.Generator().manual_seed(18)))
    g = torch.Generator().manual_seed(19)
    dx, dnormed = torch.randn(sum(lengths), d, generator=g), torch.randn(sum(lengths), d, generator=g)

    def run(q, own):
        x, normed = q["x"], q["x"]
        for k in range(2):
            v, r, i, gate = (normed @ q[f"in{k}"]).split([width, width, width, d], 1)
            if own:
                h, _ = pkg.gated_recurrence(v, r, i, q[f"decay{k}"], offs.to(dev))
                x, normed = pkg.gated_residual_norm(x, h @ q[f"out{k}"], gate, post_weight=q[f"post{k}"], scale=q[f"scale{k}"], pre_weight=q[f"pre{k}"])
            else:
                h = recurrence_in_64_bits(v, r, i, q[f"decay{k}"], offs)
                x, normed = oracle.residual_norm(x, h @ q[f"out{k}"], gate, q[f"post{k}"], None, q[f"scale{k}"], q[f"pre{k}"], None, eps=1e-6)
        return x, normed

    results = []
    for own in (True, False):
        q = {k: (t.to(dev) if own else t.double()).requires_grad_() for k, t in p.items()}
        x, normed = run(q, own)
        grads = torch.autograd.grad((x, normed), list(q.values()), (dx.to(x), dnormed.to(x)))
        results.append(dict(zip(["out", "normed", *("d " + k for k in q)], [x, normed, *grads])))
    for name, want in results[1].items():
        got, want = results[0][name].detach().cpu().double(), want.detach()
        # In halves of a unit of fp32: four products of 128 terms at most forward and eight backward, two recurrences and two boundaries each way at 100 and 64, all of
        # them one behind another: 2200; four times that for what sums lose against the sizes of their terms.
        assert float((got - want).norm() / want.norm()) < 4 * 2200 * 2.0**-24, name
