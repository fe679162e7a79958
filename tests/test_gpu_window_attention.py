"""m3_window_attention against a float64 formula: outputs, log sums, gradients, strides, values that are not finite, graphs.

Tolerances, with h half a step of the type relative to the value (``finfo.eps / 2``) and u = 2^-24:

* a logit is a sum of D products in fp32 and a product with the scale: off by e = (D + 8) u scale sum |q||k|, and a weight
  by 2 e + 8 u of itself (its own logit, the maximum's, exp and sum), in the gradients by one more rounding of the
  log sum (u |lse|);
* weights enter the second product rounded once (h in 16 bits, 0 in fp32), or, for a backward pass, as two terms (h^2 left
  out), so out is off by (h + 2 e + (n + 8) u) sum p|v|, n keys, then by h of itself;
* delta = dO . out takes the latter out, to 2 h^2;
* ds = p (dp - delta) is off by p (D u sum |dO||v| + that of delta) and its weight's error of |ds|, and is two terms (h^2);
* each gradient is a sum of products of these, off by the sum of their errors' magnitudes, then by h of itself.

What falls below the type's range is off by its smallest step.
"""

from __future__ import annotations

import pytest
import torch
import torch.utils.checkpoint

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
    off["trained"] = torch.zeros_like(res["out"])  # out for a backward pass
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
            off["trained"][rows, head] = (h_in * h_in + w + (n + 8) * U) * size
            off["lse"][rows, head] = (e + (n + 8) * U + 2 * U * lse.abs())[:, 0]
            if do is None:
                continue
            w = w + U * (lse.abs() + (n + 8))
            y = do[rows, head].double()
            dp, delta = y @ vv.T, (y * (p @ vv)).sum(1, keepdim=True)
            ds = p * (dp - delta)
            e_delta = (y.abs() * (off["trained"][rows, head] + (2 * h_in * h_in + (d + 8) * U) * size)).sum(1, keepdim=True)
            e_ds = p * ((d + 8) * U * (y.abs() @ vv.abs().T) + e_delta) + (h_in * h_in + w) * (ds.abs() + 4 * U * p * delta.abs())
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
    off["trained"] = off["trained"] * (1 + h) + h * res["out"].abs() + tiny
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
    ([65], 3, 3, 8, 16, 1, torch.float32),
    ([2500], 2, 1, 64, 300, 4, torch.bfloat16),          # three chunks of rows behind the window
    ([2500], 2, 1, 64, 1, 70, torch.float16),
    ([2100, 1, 1030], 2, 1, 64, 1024, 16, torch.float32),
    ([6000, 700], 2, 1, 64, 5, 900, torch.bfloat16),     # tiles of first tokens that go through all rows
    ([2, 65] * 150, 2, 1, 256, 5, 64, torch.float16),    # the same: many short sequences
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
    check(plain, res["out"], off["out"], "out without gradients")
    off["out"] = off["trained"]
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out.detach(), lse, *grads)):
        check(got, res[name], off[name], name)


def run(q, k, v, lengths, do=None, window=40, sinks=3, **kw):
    """out, lse and, with do, the gradients."""
    leaves = [x.detach().requires_grad_(do is not None) for x in (q, k, v)]
    out, lse = msa.m3_window_attention(*leaves, cu_tensor(lengths, "cuda"), max(lengths), window_size=window, sink_tokens=sinks,
                                       return_lse=True, **kw)
    return (out.detach(), lse, *(torch.autograd.grad(out, leaves, do) if do is not None else ()))


def against(got, q, k, v, lengths, window, sinks, scale, do):
    res, off = reference(q, k, v, lengths, window, sinks, scale, do)
    if do is not None:
        off["out"] = off["trained"]
    for name, x in zip(("out", "lse", "dq", "dk", "dv"), got):
        check(x, res[name], off[name], name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_strides(dtype):
    """Slices of one projection, heads in front, a shared key head, odd addresses; gradients that are views."""
    lengths, hq, g, d = [70, 130], 4, 2, 64
    q, k, v, do = inputs(lengths, hq, g, d, dtype)
    want = run(q, k, v, lengths, do)
    against(want, q, k, v, lengths, 40, 3, d ** -0.5, do)
    fused = torch.cat([q, k, v], 1)
    cases = [tuple(fused.split([hq, g, g], 1)), tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)),
             tuple(torch.nn.functional.pad(x, (1, 7))[..., 1:d + 1] for x in (q, k, v)),  # rows off 16 bytes
             tuple(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v))]    # no unit stride
    grads = [do, do.transpose(0, 1).contiguous().transpose(0, 1), torch.nn.functional.pad(do, (1, 7))[..., 1:d + 1], do]
    for (a, b, c), y in zip(cases, grads):
        assert all(torch.equal(x, z) for x, z in zip(run(a, b, c, lengths, y), want))
    shared = k[:, :1].expand(-1, g, -1)  # stride 0
    got = run(q, shared, shared, lengths, do)
    assert all(torch.equal(x, z) for x, z in zip(got, run(q, shared.contiguous(), shared.contiguous(), lengths, do)))
    ones = torch.ones((), dtype=dtype, device="cuda").expand_as(do)
    assert all(torch.equal(x, z) for x, z in zip(run(q, k, v, lengths, ones), run(q, k, v, lengths, ones.contiguous())))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.5, 1e-9])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_scales(dtype, scale):
    lengths = [90, 33]
    q, k, v, do = inputs(lengths, 4, 2, 64, dtype)
    against(run(q, k, v, lengths, do, scale=scale), q, k, v, lengths, 40, 3, scale, do)


def test_rows_that_see_one_key_have_gradients_of_zero():
    """Their softmax is 1 whatever the key: ds = dp - delta vanishes, not only to rounding."""
    for dtype, d in ((torch.bfloat16, 128), (torch.float16, 80), (torch.float32, 64), (torch.bfloat16, 192)):
        q, k, v, do = inputs([300, 1], 8, 2, d, dtype)
        out, _, dq, dk, dv = run(q, k, v, [300, 1], do, 1, 0)
        assert torch.equal(out, v.repeat_interleave(4, 1)) and not dq.any() and not dk.any()


def test_each_gradient_alone():
    lengths = [150]
    q, k, v, do = inputs(lengths, 8, 2, 128, torch.bfloat16)
    want = run(q, k, v, lengths, do)[2:]
    for keep in range(1, 8):
        leaves = [x.detach().requires_grad_(bool(keep >> i & 1)) for i, x in enumerate((q, k, v))]
        out = msa.m3_window_attention(*leaves, cu_tensor(lengths, "cuda"), 150, window_size=40, sink_tokens=3)
        out.backward(do)
        for i, x in enumerate(leaves):
            assert torch.equal(x.grad, want[i]) if keep >> i & 1 else x.grad is None


def test_gradients_against_differences():
    """fp32: (f(x + s y) - f(x - s y)) / 2 s for f = <out, do>, along random y. The difference of third order is s^2 / 6 times
    the third derivative; with logits of size 1 that is below s^2 sum |do| |out| 10, and the two f are off by their bounds over s."""
    lengths, scale = [37, 20], 16 ** -0.5
    q, k, v, do = (x * 0.5 for x in inputs(lengths, 4, 2, 16, torch.float32))
    window, sinks, s = 9, 2, 2.0 ** -6
    grads = run(q, k, v, lengths, do, window, sinks)[2:]
    gen = torch.Generator().manual_seed(8)
    for i in range(3):
        y = torch.randn((q, k, v)[i].shape, generator=gen).cuda()
        y /= y.norm() / 4
        f = []
        room = 0.0
        for sign in (1, -1):
            x = [a.clone() for a in (q, k, v)]
            x[i] += sign * s * y
            f.append((run(*x, lengths, None, window, sinks)[0].double() * do.double()).sum().item())
            res, off = reference(*x, lengths, window, sinks, scale)
            room += (off["out"] * do.abs().double()).sum().item() / (2 * s)
        bound = room + 10 * s * s * (do.abs().double() * res["out"].abs()).sum().item()
        assert abs((f[0] - f[1]) / (2 * s) - (grads[i].double() * y.double()).sum().item()) <= bound


def test_fp16_gradients_of_any_size():
    """Incoming gradients of 2^-20 and of 2^10, as without and with loss scaling: what fp16 holds of the results is theirs."""
    lengths = [300]
    q, k, v, do = inputs(lengths, 4, 2, 64, torch.float16)
    for power in (-20, -12, 10):
        y = (do.double() * 2.0 ** power).half()
        against(run(q, k, v, lengths, y, 100, 4), q, k, v, lengths, 100, 4, 64 ** -0.5, y)
    rows = torch.randint(-22, 9, (300, 4, 1), generator=torch.Generator().manual_seed(2)).double().exp2().cuda()
    y = (do.double() * rows).half()  # rows of different size
    against(run(q, k, v, lengths, y, 100, 4), q, k, v, lengths, 100, 4, 64 ** -0.5, y)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64), (torch.bfloat16, 256)])
def test_what_is_not_finite_stays_with_the_rows_that_see_it(dtype, d):
    lengths, window, sinks = [200, 90], 32, 2
    q, k, v, do = inputs(lengths, 4, 2, d, dtype)
    plain = run(q, k, v, lengths, do, window, sinks)
    res, off = reference(q, k, v, lengths, window, sinks, d ** -0.5, do)
    for what, value in ((0, float("nan")), (1, float("nan")), (1, float("inf")), (2, float("nan")), (2, float("inf")), (3, float("nan")),
                        (3, float("-inf"))):
        for at in (0, 1, 100, 199, 230):  # a first token, a later one, the last of a sequence, one of the second
            x = [y.clone() for y in (q, k, v, do)]
            x[what][at, 0, 3] = value
            got = run(*x[:3], lengths, x[3], window, sinks)
            start, end = (0, 200) if at < 200 else (200, 290)
            sees = torch.zeros(290, dtype=torch.bool, device="cuda")  # rows that see token `at`
            sees[at:end] = True if at - start < sinks else False
            sees[at:min(end, at + window)] = True
            keys = torch.zeros(290, dtype=torch.bool, device="cuda")  # keys that token `at` sees
            keys[max(start, at - window + 1):at + 1] = True
            keys[start:min(start + sinks, at + 1)] = True
            heads = [0, 1] if what in (1, 2) else [0]
            if what in (1, 2):  # a key's or value's: its rows, and the keys that those see
                far = torch.zeros_like(keys)
                for i in sees.nonzero().flatten().tolist():
                    far[max(start, i - window + 1):i + 1] = True
                    far[start:min(start + sinks, i + 1)] = True
            else:
                sees, far = torch.zeros_like(sees), keys
                sees[at] = True
            for name, a in zip(("out", "lse", "dq", "dk", "dv"), got):
                other = torch.ones_like(a, dtype=torch.bool)
                if name in ("out", "lse", "dq"):
                    for h in heads:
                        other[:, h] &= (~sees).view(-1, *[1] * (a.ndim - 2))
                else:
                    other[:, 0] &= (~far)[:, None]
                # (tiles that met the value are formed again, key by key: within the same bound, not the same bits)
                check(a[other], res[name][other], off[name][other], (what, value, at, name))
            if what == 2:  # the value's dim alone, as the formula has it
                out = got[0][sees][:, :2]
                assert (torch.isnan(out[..., 3]).all() if value != value else (out[..., 3] == value).all())
                keep = [i for i in range(d) if i != 3]
                check(out[..., keep], res["out"][sees][:, :2][..., keep], off["out"][sees][:, :2][..., keep], (value, at))
                assert torch.equal(got[1], plain[1])
            if what == 3:
                assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])


def test_an_infinity_counts_whatever_its_weight():
    """A key so far from the row's best that its weight is 0 in fp32."""
    q, k, v, _ = inputs([64], 1, 1, 64, torch.bfloat16)
    k[5] = -200.0 * q[63, 0].sign()
    v[5, 0, 7] = float("inf")
    out = run(q, k, v, [64], None, 64, 0)[0]
    assert out[63, 0, 7] == float("inf") and torch.isfinite(out[63, 0, :7]).all() and torch.isfinite(out[:5]).all()


def test_all_of_a_batch_not_finite_ends():
    q, k, v, do = inputs([600], 8, 2, 128, torch.bfloat16)
    for i in range(4):
        x = [y.clone() for y in (q, k, v, do)]
        x[i].fill_(float("nan"))
        got = run(*x[:3], [600], x[3], 256, 4)
        assert torch.isnan(got[0]).all() == (i < 3) and torch.isnan(got[2]).all() and torch.isnan(got[3]).all()


def test_larger_calls():
    """Enough keys for tiles of keys that no workgroups share, with first tokens seen from behind the window."""
    lengths, hq, g, d, window, sinks = [5000, 3001, 1], 16, 16, 64, 130, 5
    q, k, v, do = inputs(lengths, hq, g, d, torch.bfloat16)
    against(run(q, k, v, lengths, do, window, sinks), q, k, v, lengths, window, sinks, d ** -0.5, do)


def test_streams_and_determinism():
    q, k, v, do = inputs([700, 129], 8, 2, 128, torch.float16)
    want = run(q, k, v, [700, 129], do, 200, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(q, k, v, [700, 129], do, 200, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_captured_step_replays():
    lengths = [300, 1, 77]
    seqs = msa.prepare_sequences(cu_tensor(lengths, "cuda"))
    q, k, v, do = inputs(lengths, 8, 2, 64, torch.bfloat16)
    leaves = [x.requires_grad_() for x in (q, k, v)]

    def step():
        out, lse = msa.m3_window_attention(*leaves, seqs, 300, window_size=50, sink_tokens=4, return_lse=True)
        return (out.detach(), lse, *torch.autograd.grad(out, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(3):
        gen = torch.Generator(device="cuda").manual_seed(turn)
        with torch.no_grad():
            for x in (*leaves, do):
                x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        graph.replay()
        want = run(q, k, v, lengths, do, 50, 4)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_checkpointing_and_offloaded_saved_tensors():
    lengths = [140]
    q, k, v, do = inputs(lengths, 4, 2, 64, torch.bfloat16)
    want = run(q, k, v, lengths, do)[2:]
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    f = lambda *x: msa.m3_window_attention(*x, cu_tensor(lengths, "cuda"), 140, window_size=40, sink_tokens=3)  # noqa: E731
    torch.utils.checkpoint.checkpoint(f, *leaves, use_reentrant=False).backward(do)
    assert all(torch.equal(x.grad, y) for x, y in zip(leaves, want))
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    with torch.autograd.graph.save_on_cpu():
        out = f(*leaves)
    out.backward(do)
    assert all(torch.equal(x.grad, y) for x, y in zip(leaves, want))


def test_an_input_changed_before_its_backward_pass_is_noticed():
    q, k, v, do = inputs([30], 2, 1, 64, torch.bfloat16)
    q.requires_grad_()
    out = msa.m3_window_attention(q, k, v, cu_tensor([30], "cuda"), 30, window_size=None)
    k.zero_()
    with pytest.raises(RuntimeError, match="inplace operation"):
        out.backward(do)


def test_no_tokens():
    for dtype in (torch.bfloat16, torch.float32):
        q, k = torch.zeros(0, 4, 64, dtype=dtype, device="cuda"), torch.zeros(0, 2, 64, dtype=dtype, device="cuda")
        q.requires_grad_()
        out, lse = msa.m3_window_attention(q, k, k, cu_tensor([0, 0], "cuda"), 1, window_size=3, return_lse=True)
        out.sum().backward()
        assert out.shape == q.shape and lse.shape == (0, 4) and q.grad.shape == q.shape


def test_offsets_past_32_bits():
    """2.3e9 values a tensor, checked at their ends and in between."""
    tokens, hq, d, window = 140_000, 64, 256, 3
    q = torch.empty(tokens, hq, d, dtype=torch.bfloat16, device="cuda")
    assert q.numel() > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(1)
    q.normal_(generator=gen)
    k, v = (torch.randn(tokens, 1, d, generator=gen, device="cuda").bfloat16() for _ in range(2))
    q.requires_grad_(), k.requires_grad_(), v.requires_grad_()
    out = msa.m3_window_attention(q, k, v, cu_tensor([tokens], "cuda"), tokens, window_size=window)
    do = torch.empty_like(out).normal_(generator=gen)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    for a, b in ((0, 40), (69_000, 69_040), (tokens - 40, tokens)):
        front = min(a, window - 1)  # (rows in front complete the windows of the checked ones)
        back = min(tokens - b, window - 1)
        rows = slice(a - front, b + back)
        res, off = reference(*(x.detach()[rows] for x in (q, k, v)), [b - a + front + back], window, 0, d ** -0.5, do[rows])
        mine = slice(front, front + b - a)
        for name, got in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
            check(got.detach()[a:b], res[name][mine], off[name][mine], name)


def test_calls_of_more_than_2_to_the_23_workgroups():
    """Sequences of one token, in one call: out is v, with the gradients of that. dq = (dO . v - dO . out) k is nothing but the
    errors of two sums of 8 products, each off by at most 16 u sum |dO||v|."""
    from msa_triton_amd.window_attention import _backward, _forward

    n = (1 << 23) + 77
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v, do = (torch.randn(n, 1, 8, generator=gen, device="cuda").bfloat16() for _ in range(4))
    out, lse, lo = _forward(q, k, v, cu, n, 5, 0, 1.0, True, True)
    dq, dk, dv = _backward(q, k, v, cu, n, 1, 5, 0, 1.0, out, lo, lse, do, True, True, True)
    assert torch.equal(out, v) and torch.equal(dv, do)
    most = 2 * 16 * U * (do.double().abs() * v.double().abs()).sum(2, keepdim=True) * (1 + 2.0 ** -7)
    assert (dq.double().abs() <= most * k.double().abs()).all() and (dk.double().abs() <= most * q.double().abs()).all()


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 72)])
def test_several_values_that_are_not_finite(dtype, d):
    """Infinities that meet, beside NaN, under a logit of -inf, and in more than one dim: NaN, +inf and -inf stand where the
    formula over the visible tokens has them, and the rest is within the bound."""
    n, window, sinks, scale = 150, 20, 2, d ** -0.5
    q, k, v, do = inputs([n], 2, 1, d, dtype)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    res, off = reference(q, k, v, [n], window, sinks, scale, do)
    inf = float("inf")
    x = [y.clone() for y in (q, k, v, do)]
    x[2][60, 0, 5], x[2][62, 0, 5], x[2][64, 0, 6], x[2][64, 0, 7] = inf, -inf, float("nan"), inf
    x[2][100, 0, 9], x[1][100, 0, 0] = inf, -inf  # a weight of 0 under an infinity
    out = run(*x[:3], [n], None, window, sinks)[0]
    for i in range(n):
        seen = [j for j in range(i + 1) if i - j < window or j < sinks]
        for h in range(2):
            p = torch.softmax(x[0][i, h].double() @ x[1][seen, 0].double().T * scale, -1)
            want = (p[:, None] * x[2][seen, 0].double()).sum(0)
            for name in (torch.isnan, torch.isposinf, torch.isneginf):
                assert torch.equal(name(out[i, h]), name(want)), (i, h, name)
    far = torch.ones(n, dtype=torch.bool, device="cuda")
    far[60:120] = False
    check(out[far], res["out"][far], off["out"][far], "out")
    x = [y.clone() for y in (q, k, v, do)]
    x[3][60, 0, 5], x[3][62, 0, 5], x[3][64, 1, 6], x[3][64, 1, 7] = inf, -inf, float("nan"), inf
    _, _, dq, dk, dv = run(*x[:3], [n], x[3], window, sinks)
    lse = res["lse"]
    for j in range(n):
        rows = [i for i in range(j, n) if i - j < window or j < sinks]
        p = torch.exp(x[0][rows].double() @ x[1][j, 0].double() * scale - lse[rows])
        want = (p[..., None] * x[3][rows].double()).sum((0, 1))
        for name in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(name(dv[j, 0]), name(want)), (j, name)
        clean = torch.isfinite(want)
        check(dv[j, 0][clean], res["dv"][j, 0][clean], off["dv"][j, 0][clean], ("dv", j))
    other = [i for i in range(n) if i not in (60, 62, 64)]
    check(dq[other], res["dq"][other], off["dq"][other], "dq")
    x = [y.clone() for y in (q, k, v, do)]
    x[2].fill_(float("nan"))
    out, lse, dq, dk, dv = run(*x[:3], [n], x[3], window, sinks)
    assert all(torch.isnan(y).all() for y in (out, dq, dk))
    check(lse, res["lse"], off["lse"], "lse")
    check(dv, res["dv"], off["dv"], "dv")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_row_whose_logits_are_all_minus_infinity(dtype):
    q, k, v, do = inputs([70], 2, 1, 64, dtype)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    k[0, 0, 0] = float("-inf")  # the first token's only key; the others' weight of 0
    out, lse, dq, dk, dv = run(q, k, v, [70], do, window=8, sinks=0)
    assert not out[0].any() and (lse[0] == float("-inf")).all()
    assert torch.isfinite(out).all() and torch.isfinite(lse[1:]).all() and torch.isfinite(dk).all() and torch.isfinite(dv).all()
    assert not dk[0].any() and not dv[0].any() and torch.isfinite(dq[8:]).all()
    other, _ = run(q, k, v, [70], None, window=8, sinks=0)
    assert not other[0].any()
