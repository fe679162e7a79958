"""m3_window_attention against a float64 formula: outputs, log sums, gradients, strides, values that are not finite, graphs.

Tolerances, with h half a step of the type relative to the value (``finfo.eps / 2``) and u = 2^-24:

* a logit is a sum of D products in fp32 and a product with the scale: off by e = (D + 8) u scale sum |q||k|, and a weight
  by 2 e + 8 u of itself (its own logit, the maximum's, exp and sum), in the gradients by one more rounding of the
  log sum (u |lse|);
* weights enter the second product rounded once (h in 16 bits, 0 in fp32), so out is off by (h + 2 e + (n + 8) u)
  sum p|v|, n keys, then by h of itself;
* delta = dO . out takes the out of the forward in 2 h^2, its weights' rounding (h) included;
* ds = p (dp - delta) is off by p (D u sum |dO||v| + that of delta) and its weight's error of |ds|, and is rounded once;
* each gradient is a sum of products of these, off by the sum of their errors' magnitudes, then by h of itself.

What falls below the type's range is off by its smallest step.
"""

from __future__ import annotations

import pytest
import torch

import msa_triton_amd as msa
from tests.helpers import cu_tensor

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def visible(n, window, sinks, device):
    i = torch.arange(n, device=device)
    back = i[:, None] - i
    return (back >= 0) & ((back < (window or n + 1)) | (i < sinks))


def reference(q, k, v, lengths, window, sinks, scale, do=None):
    """float64 results and how far a kernel may be off, by name."""
    total, hq, d = q.shape
    g = k.shape[1]
    ratio = hq // g
    h = half_step(q.dtype)
    h_in = 0.0 if q.dtype == torch.float32 else h  # of a weight or a ds on its way into a product
    res = {x: torch.zeros(total, hq, d, dtype=torch.float64, device=q.device) for x in ("out", "dq")}
    res |= {x: torch.zeros(total, g, d, dtype=torch.float64, device=q.device) for x in ("dk", "dv")}
    res["lse"] = torch.zeros(total, hq, dtype=torch.float64, device=q.device)
    off = {x: torch.zeros_like(y) for x, y in res.items()}
    at = 0
    for n in lengths:
        rows = slice(at, at + n)
        at += n
        if n == 0:
            continue
        seen = visible(n, window, sinks, q.device)
        for head in range(hq):
            a, kk, vv = q[rows, head].double(), k[rows, head // ratio].double(), v[rows, head // ratio].double()
            x = (a @ kk.T * scale).masked_fill(~seen, float("-inf"))
            lse = torch.logsumexp(x, 1, keepdim=True)
            p = torch.exp(x - lse)
            e = (d + 8) * U * abs(scale) * ((a.abs() @ kk.abs().T) * seen).amax(1, keepdim=True)
            w = 2 * e + 8 * U  # of a weight, relative
            res["out"][rows, head], res["lse"][rows, head] = p @ vv, lse[:, 0]
            size = p @ vv.abs()
            off["out"][rows, head] = (h_in + w + (n + 8) * U) * size
            off["lse"][rows, head] = (e + (n + 8) * U + 2 * U * lse.abs())[:, 0]
            if do is None:
                continue
            w = w + U * (lse.abs() + (n + 8))
            y = do[rows, head].double()
            dp, delta = y @ vv.T, (y * (p @ vv)).sum(1, keepdim=True)
            ds = p * (dp - delta)
            e_delta = (y.abs() * (off["out"][rows, head] + (2 * h_in * h_in + (d + 8) * U) * size)).sum(1, keepdim=True)
            e_ds = p * ((d + 8) * U * (y.abs() @ vv.abs().T) + e_delta) + (h_in + w) * (ds.abs() + 4 * U * p * delta.abs())
            few = (n * ratio + 8) * U  # of a sum
            res["dq"][rows, head] = ds @ kk * scale
            off["dq"][rows, head] = (e_ds + few * ds.abs()) @ kk.abs() * abs(scale)
            res["dk"][rows, head // ratio] += ds.T @ a * scale
            off["dk"][rows, head // ratio] += (e_ds + few * ds.abs()).T @ a.abs() * abs(scale)
            res["dv"][rows, head // ratio] += p.T @ y
            off["dv"][rows, head // ratio] += ((h_in + w + few) * p).T @ y.abs()
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    for x, y in res.items():
        own = 4 * U if x == "lse" else h
        off[x] = off[x] * (1 + own) + own * y.abs() + (1e-30 if x == "lse" else tiny)
    return res, off


def check(got, want, off, what):
    assert torch.isfinite(got).all(), what
    part = ((got.double() - want).abs() / off).max().item() if got.numel() else 0.0
    assert part <= 1.0, f"{what}: {part:.2f} of the bound"


def inputs(lengths, hq, g, d, dtype, seed=5, device="cuda"):
    gen = torch.Generator().manual_seed(seed)
    total = sum(lengths)

    def rand(n):
        return (torch.randn(total, n, d, generator=gen) * (0.5 + torch.rand(n, 1, generator=gen))).to(dtype).to(device)

    return rand(hq), rand(g), rand(g), rand(hq)


CASES = [  # lengths, hq, g, d, window, sinks, dtype
    ([1], 1, 1, 64, 1, 0, torch.bfloat16),
    ([1], 8, 1, 128, None, 0, torch.float16),
    ([2, 0, 1, 3], 4, 2, 64, 2, 1, torch.float32),
    ([130, 0, 1, 257], 8, 2, 64, 33, 4, torch.bfloat16),
    ([300], 32, 4, 128, 128, 4, torch.bfloat16),
    ([300], 32, 4, 128, 128, 4, torch.float16),
    ([300], 16, 4, 128, 100, 3, torch.float32),
    ([511], 5, 1, 128, None, 0, torch.bfloat16),         # a ratio of 5: tokens across tiles
    ([511], 4, 4, 128, 64, 0, torch.float16),            # a ratio of 1
    ([200, 333], 6, 2, 96, 77, 130, torch.bfloat16),     # sinks over several tiles
    ([200, 333], 6, 2, 96, 77, 130, torch.float32),
    ([700], 3, 1, 72, 5, 300, torch.float16),            # more sinks than window
    ([257, 64], 4, 2, 192, 50, 2, torch.bfloat16),
    ([257, 64], 4, 2, 256, 50, 2, torch.float16),
    ([129], 2, 1, 256, 40, 65, torch.float32),
    ([65], 3, 3, 8, 16, 1, torch.bfloat16),              # one fragment's dims
    ([65], 3, 3, 4, 16, 1, torch.float32),
    ([2500], 2, 1, 64, 300, 4, torch.bfloat16),          # three chunks of rows behind the window
    ([2500], 2, 1, 64, 1, 70, torch.float16),
    ([2100, 1, 1030], 2, 1, 64, 1024, 16, torch.float32),
    ([64] * 40, 2, 2, 64, 8, 2, torch.bfloat16),
    ([3] * 200 + [90], 8, 2, 64, 2, 1, torch.bfloat16),  # more sequences than a wave has lanes
    ([400], 64, 1, 64, 31, 4, torch.bfloat16),           # one token a tile of rows
    ([37], 200, 1, 64, 10, 0, torch.float16),            # less than one
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in (len(c[0]), max(c[0]), *c[1:6], c[6]))[:60])
def test_against_the_formula(case):
    lengths, hq, g, d, window, sinks, dtype = case
    q, k, v, do = inputs(lengths, hq, g, d, dtype)
    for x in (q, k, v):
        x.requires_grad_()
    out, lse = msa.m3_window_attention(q, k, v, cu_tensor(lengths, "cuda"), max(lengths), window_size=window, sink_tokens=sinks,
                                       return_lse=True)
    assert not lse.requires_grad and lse.dtype == torch.float32 and out.dtype == dtype
    grads = torch.autograd.grad(out, (q, k, v), do)
    with torch.no_grad():
        res, off = reference(q, k, v, lengths, window, sinks, d ** -0.5, do)
        plain = msa.m3_window_attention(q, k, v, cu_tensor(lengths, "cuda"), max(lengths), window_size=window, sink_tokens=sinks)
    assert torch.equal(plain, out)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out.detach(), lse, *grads)):
        check(got, res[name], off[name], name)
