"""The norm, the append and the window and tree attention as a server uses them, against the packed operators over the whole
sequences: a prompt and single tokens, a drafted tree, the tokens of it that were accepted, and one more.

Both sides' keys and queries have the same bits (the append writes what the norm gives), so both are within their own bounds of
one float64 result, and within the sum of these of each other.
"""

from __future__ import annotations

import pytest
import torch

import msa_triton_amd as msa
from tests.helpers import cu_tensor
from tests.test_gpu_window_attention import reference
from tests.test_gpu_window_paged import oracle, paths

pytestmark = pytest.mark.gpu

HQ, G, D, PAGE = 16, 2, 64, 16
PROMPT = [70, 1, 129]
PARENTS = [[-1, 0, 0, 1, 2, -1, 5], [-1], [-1, -1, 0, 1, 3]]


def _layer(dtype, seed=6):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    most = 200
    raw = [dict(q=rand(most, HQ, D), k=rand(most, G, D), v=rand(most, G, D)) for _ in PROMPT]
    weights = [1 + 0.2 * rand(D) for _ in range(2)]
    table = msa.rope_table(most, 32, base=1e4, device="cuda")
    pages = torch.randperm(64, generator=torch.Generator().manual_seed(1))[:39].view(3, 13).to(torch.int32).cuda()
    kc, vc = (torch.full((64, G, PAGE, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    return raw, weights, table, pages, kc, vc


def _packed(raw, rows, weights, table, window, sinks):
    """The packed operators over one sequence of the given tokens: out of its last token, and how far it may be off."""
    x = [raw[n][rows] for n in ("q", "k", "v")]
    cu, n = cu_tensor([len(rows)], "cuda"), len(rows)
    q, k = msa.m3_qk_norm_rope(x[0], x[1], *weights, table, cu)
    out = msa.m3_window_attention(q, k, x[2], cu, n, window_size=window, sink_tokens=sinks)
    _, off = reference(q, k, x[2], [n], window, sinks, D ** -0.5)
    return out[-1], off["out"][-1]


@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@torch.no_grad()
def test_prompt_decoding_and_a_tree(dtype, window, sinks):
    raw, weights, table, pages, kc, vc = _layer(dtype)
    x = dict(kc=kc, vc=vc, ks=None, vs=None, table=pages, parents=None)

    def part(name, spans):
        return torch.cat([raw[s][name][span] for s, span in enumerate(spans)])

    # the prompts, then four tokens of each request
    length = [0, 0, 0]
    tokens = [list(range(n)) for n in PROMPT]
    for step in range(5):
        spans = [slice(a, a + (n if step == 0 else 1)) for a, n in zip(length, PROMPT)]
        new = [s.stop - s.start for s in spans]
        seqs = msa.prepare_sequences(cu_tensor(new, "cuda"))
        context = torch.tensor(length, dtype=torch.int32, device="cuda")
        q, _ = msa.m3_qk_norm_rope(part("q", spans), None, weights[0], None, table, seqs, context_lens=context)
        msa.m3_cache_append(part("k", spans), part("v", spans), kc, vc, pages, seqs, context, k_weight=weights[1], cos_sin=table)
        out = msa.m3_window_attention_paged(q, kc, vc, pages, seqs, context, window_size=window, sink_tokens=sinks)
        _, _, tol, _ = oracle(dict(x, q=q), new, length, window or 0, sinks, D ** -0.5)
        length = [s.stop for s in spans]
        for s in range(3):
            want, off = _packed(raw[s], list(range(length[s])), weights, table, window, sinks)
            last = sum(new[:s + 1]) - 1
            assert ((out[last].double() - want.double()).abs() <= tol[last] + off).all(), (step, s)
    tokens = [list(range(n)) for n in length]

    # a tree behind each: positions by depth, slots by place
    nodes = [[150 + i for i in range(len(p))] for p in PARENTS]  # (tokens that no request has used)
    new = [len(p) for p in PARENTS]
    seqs = msa.prepare_sequences(cu_tensor(new, "cuda"))
    context = torch.tensor(length, dtype=torch.int32, device="cuda")
    ways = [paths(p, len(p)) for p in PARENTS]
    place = torch.tensor([length[s] + len(w) - 1 for s in range(3) for w in ways[s]], device="cuda")
    one = cu_tensor([sum(new)], "cuda")
    q, k = msa.m3_qk_norm_rope(part("q", nodes), part("k", nodes), *weights, table[place], one)
    msa.m3_cache_append(k, part("v", nodes), kc, vc, pages, seqs, context)
    parents = torch.tensor(sum(PARENTS, []), dtype=torch.int32, device="cuda")
    out = msa.m3_tree_attention_paged(q, kc, vc, pages, seqs, context, parents, window_size=window, sink_tokens=sinks)
    _, _, tol, _ = oracle(dict(x, q=q, parents=parents), new, length, window or 0, sinks, D ** -0.5)
    at = 0
    for s in range(3):
        for way in ways[s]:
            want, off = _packed(raw[s], tokens[s] + [nodes[s][i] for i in way], weights, table, window, sinks)
            assert ((out[at].double() - want.double()).abs() <= tol[at] + off).all(), (s, way)
            at += 1

    # the accepted path of each takes the slots behind the context; then one more token
    kept = [ways[0][4], ways[1][0], ways[2][4]]
    first = [0, *torch.tensor(new).cumsum(0).tolist()]
    rows = torch.tensor([first[s] + i for s in range(3) for i in kept[s]], device="cuda")
    taken = [len(w) for w in kept]
    seqs = msa.prepare_sequences(cu_tensor(taken, "cuda"))
    msa.m3_cache_append(k[rows], part("v", nodes)[rows], kc, vc, pages, seqs, context)
    tokens = [t + [nodes[s][i] for i in kept[s]] + [199] for s, t in enumerate(tokens)]
    context += torch.tensor(taken, dtype=torch.int32, device="cuda")
    seqs = msa.prepare_sequences(cu_tensor([1, 1, 1], "cuda"))
    spans = [[199]] * 3
    q, _ = msa.m3_qk_norm_rope(part("q", spans), None, weights[0], None, table, seqs, context_lens=context)
    msa.m3_cache_append(part("k", spans), part("v", spans), kc, vc, pages, seqs, context, k_weight=weights[1], cos_sin=table)
    out = msa.m3_window_attention_paged(q, kc, vc, pages, seqs, context, window_size=window, sink_tokens=sinks)
    _, _, tol, _ = oracle(dict(x, q=q), [1, 1, 1], context.tolist(), window or 0, sinks, D ** -0.5)
    for s in range(3):
        want, off = _packed(raw[s], tokens[s], weights, table, window, sinks)
        assert ((out[s].double() - want.double()).abs() <= tol[s] + off).all(), s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_layer_trains(dtype):
    """Norm and window attention in one graph: the projections' gradients against those of the formula in float64."""
    lengths = [33, 50]
    raw, weights, table, *_ = _layer(dtype)
    x = [torch.cat([raw[s][n][:m] for s, m in enumerate(lengths)]).requires_grad_() for n in ("q", "k", "v")]
    cu = cu_tensor(lengths, "cuda")
    q, k = msa.m3_qk_norm_rope(x[0], x[1], *weights, table, cu)
    out = msa.m3_window_attention(q, k, x[2], cu, 50, window_size=11, sink_tokens=2)
    do = torch.randn_like(out)
    mids = torch.autograd.grad(out, (q, k, x[2]), do, retain_graph=True)
    grads = torch.autograd.grad(out, x, do, retain_graph=True)
    through = torch.autograd.grad((q, k), x[:2], mids[:2])
    assert torch.equal(grads[0], through[0]) and torch.equal(grads[1], through[1]) and torch.equal(grads[2], mids[2])
    with torch.no_grad():
        res, off = reference(q, k, x[2], lengths, 11, 2, D ** -0.5, do)
    for name, got in zip(("dq", "dk", "dv"), mids):
        assert ((got.double() - res[name]).abs() <= off[name]).all(), name
