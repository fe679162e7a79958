"""Timed cases of the window and tree attention operators.

Three operators for the layers that stand beside the block-sparse ones:

* ``window``  causal attention of packed sequences with a sliding window and a few first tokens that stay
              visible, forward alone (prompts) or forward and backward (training): ``m3_window_attention``;
* ``serve``   the same attention of new tokens against a paged cache of 16-bit or 8-bit entries:
              ``m3_window_attention_paged``;
* ``tree``    attention of a tree of drafted tokens over a paged cache, each node seeing the cached tokens and its
              ancestors: ``m3_tree_attention_paged``.

``run`` computes them in elementary torch operations, or with the package's operators where
``own`` is true; ``exact`` restates them in float64.
"""

from __future__ import annotations

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8 = torch.float8_e4m3fn
DEVICE = "cuda"
BUDGET = 1 << 27  # logits held at once by the plain and the float64 forms


def _spread(n, low, high):
    """`n` lengths between `low` and `high`, spread evenly over their logarithm and mixed."""
    out = [int(round(low * (high / low) ** (((7 * i + 3) % n + 0.5) / n))) for i in range(n)]
    return ",".join(str(x) for x in out)


def _ones(n):
    return ",".join(["1"] * n)


def listed():
    # (a window of 0 stands for none: plain causal attention)
    return [
        # The smallest training configuration (c1): two short sequences, heads of 64, a window inside them.
        dict(name="window_train_small", op="window", dtype="bf16", new="512,768", hq=8, g=2, d=64, window=256, sinks=4,
             grad=True),
        # fp32, as used to check a model before it goes to 16 bits; no power of two anywhere.
        dict(name="window_train_fp32", op="window", dtype="fp32", new="701,1347", hq=16, g=2, d=128, window=500,
             sinks=3, grad=True),
        # Packed training sequences of uneven length in fp16, heads of 96.
        dict(name="window_train_ragged", op="window", dtype="fp16", new="2047,3001,5003,6151,97,1", hq=16, g=4, d=96,
             window=1024, sinks=16, grad=True),
        # The headline training length (c4's 32K tokens and heads) in a local layer.
        dict(name="window_train_32k", op="window", dtype="bf16", new="32768", hq=32, g=4, d=128, window=4096, sinks=4,
             grad=True),
        # Prompts of a serving batch through a layer without a window.
        dict(name="window_prompts", op="window", dtype="bf16", new="8192,1837,411,4001,96,733", hq=32, g=4, d=128,
             window=0, sinks=0, grad=False),
        # One request at a time: latency.
        dict(name="serve_single", op="serve", dtype="bf16", cache="16", new="1", context="20011", hq=32, g=4, d=128,
             page=128, window=4096, sinks=4),
        # A decoding step of 64 requests over an 8-bit cache, a local layer.
        dict(name="serve_decode_fp8", op="serve", dtype="bf16", cache="fp8", new=_ones(64),
             context=_spread(64, 60, 30000), hq=32, g=4, d=128, page=64, window=4096, sinks=4),
        # The same step in a layer without a window: lengths differ by orders.
        dict(name="serve_decode_full", op="serve", dtype="bf16", cache="16", new=_ones(64),
             context=_spread(64, 60, 30000), hq=32, g=4, d=128, page=128, window=0, sinks=0),
        # Later parts of long prompts behind what the cache holds of them.
        dict(name="serve_chunk_fp16", op="serve", dtype="fp16", cache="16", new="512,300,1", context="8192,1000,5000",
             hq=32, g=4, d=128, page=64, window=2048, sinks=64),
        # A small tree behind one request: latency.
        dict(name="tree_single", op="tree", dtype="bf16", cache="16", new="15", context="1999", hq=32, g=4, d=128,
             page=128, window=0, sinks=0),
        # Trees of up to 64 nodes for a batch over an 8-bit cache.
        dict(name="tree_batch_fp8", op="tree", dtype="bf16", cache="fp8", new="64,48,64,33,64,17,64,64,1,64,60,64,64,5,64,64",
             context=_spread(16, 500, 30000), hq=32, g=4, d=128, page=64, window=0, sinks=0),
        # One wide tree behind a very long context, c5's heads, in a local layer.
        dict(name="tree_long_fp16", op="tree", dtype="fp16", cache="16", new="127", context="130000", hq=64, g=8, d=128,
             page=128, window=16000, sinks=4),
    ]


def _log_uniform(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def _split(rng, tokens, most):
    """`tokens` tokens in 1 to `most` sequences of uneven length."""
    n = min(rng.choice([1, 1, 2, 3, 5, 8, 13, 24]), most, tokens)
    cuts = sorted(rng.sample(range(1, tokens), n - 1)) if n > 1 else []
    return [b - a for a, b in zip([0, *cuts], [*cuts, tokens])]


def _text(values):
    return ",".join(str(v) for v in values)


def draw(rng):
    op = rng.choice(["window", "window", "window", "serve", "serve", "tree", "tree"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    g = rng.choice([1, 2, 4, 8])
    case = dict(op=op, dtype=dtype, g=g, window=rng.choice([0, _log_uniform(rng, 1, 8000), _log_uniform(rng, 64, 8000)]),
                sinks=rng.choice([0, 0, 1, 4, 4, 16, 130]))
    if op == "window":
        case["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        case["d"] = rng.choice([64, 72, 80, 96, 128, 128, 128, 192, 256])
        case["hq"] = g * rng.choice([1, 4, 5, 8])
        case["grad"] = rng.random() < 0.6
        most = 24000 if case["dtype"] != "fp32" else 6000
        while most > 64 and _flops(most, case) > (5e12 if case["dtype"] != "fp32" else 5e11):
            most //= 2
        return dict(case, new=_text(_split(rng, _log_uniform(rng, 1, most), 24)))
    case["page"] = rng.choice([16, 64, 128])
    case["cache"] = rng.choice(["fp8", "16"])
    case["hq"] = g * rng.choice([1, 4, 8, 8, 16])
    case["d"] = rng.choice([64, 96, 128, 128, 128, 256])
    if op == "tree":
        new = [rng.choice([1, _log_uniform(rng, 2, 150)]) for _ in range(_log_uniform(rng, 1, 16))]
    elif rng.random() < 0.7:
        new = [rng.choice([1, 1, 1, 1, 2, 5]) for _ in range(_log_uniform(rng, 1, 64))]
    else:
        new = [_log_uniform(rng, 1, 600) for _ in range(_log_uniform(rng, 1, 4))]
    most = max(2000, min(100_000, 400_000 // len(new), int(4e9) // (sum(new) * case["hq"])))
    return dict(case, new=_text(new), context=_text(rng.choice([0, *[_log_uniform(rng, 20, most)] * 7]) for _ in new))


def _flops(tokens, case):
    """Of a case with its tokens in one sequence, roughly."""
    seen = min(tokens / 2, case["window"] + case["sinks"]) if case["window"] else tokens / 2
    return (14.0 if case["grad"] else 4.0) * tokens * seen * case["hq"] * case["d"]


# ---------------------------------------------------------------------------- inputs


def _ints(text):
    return [int(x) for x in text.split(",")]


def _bounds(case):
    bounds = [0]
    for n in _ints(case["new"]):
        bounds.append(bounds[-1] + n)
    return bounds


def _contexts(case):
    return _ints(case["context"]) if "context" in case else [0] * len(_ints(case["new"]))


def _cached(case):
    """Tokens that the cache holds of each sequence, the new ones among them."""
    return [n + c for n, c in zip(_ints(case["new"]), _contexts(case))]


def _pages(case, gen):
    """Page table [N, M] of a cache that other requests have used: pages in no order, -1 behind each sequence."""
    need = [-(-n // case["page"]) for n in _cached(case)]
    order = torch.randperm(sum(need) + 3, generator=gen, device=DEVICE, dtype=torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, order.numel()


def _cache(case, pages, gen):
    """A filled cache [P, G, page, D], with its scales [P, G] where it is held in 8 bits."""
    x = torch.randn(pages, case["g"], case["page"], case["d"], generator=gen, device=DEVICE, dtype=torch.float32)
    if case["cache"] != "fp8":
        return x.to(DTYPES[case["dtype"]]), None
    scale = torch.exp2(torch.randint(-6, -4, (pages, case["g"]), generator=gen, device=DEVICE).float())
    return (x / scale[:, :, None, None]).to(FP8), scale


def _parents(case, gen):
    """Each node's parent, by its place among its sequence's new tokens: -1 behind the context itself, otherwise one
    of the last few nodes in front of it, as a drafter that widens and deepens a tree in turn lists them."""
    out = []
    for n in _ints(case["new"]):
        i = torch.arange(n, device=DEVICE)
        back = (torch.rand(n, generator=gen, device=DEVICE) ** 2 * (i + 1).clamp(max=9)).long()
        out.append(torch.where(i < 3, -1, i - 1 - back).clamp(min=-1))
    return torch.cat(out).to(torch.int32)


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(1000003 * int(seed) + 31)
    dtype = DTYPES[case["dtype"]]
    total = _bounds(case)[-1]

    def heads(n):  # normed and rotated heads: some attend sharply, some evenly
        size = 0.5 + 1.5 * torch.rand(n, 1, generator=gen, device=DEVICE)
        return (size * torch.randn(total, n, case["d"], generator=gen, device=DEVICE)).to(dtype)

    x = {"q": heads(case["hq"])}
    if case["op"] == "window":
        x["k"], x["v"] = heads(case["g"]), heads(case["g"])
        if case["grad"]:
            x["do"] = torch.randn(total, case["hq"], case["d"], generator=gen, device=DEVICE).to(dtype)
        return x
    x["pages"], count = _pages(case, gen)
    x["kc"], x["ks"] = _cache(case, count, gen)
    x["vc"], x["vs"] = _cache(case, count, gen)
    if case["op"] == "tree":
        x["parents"] = _parents(case, gen)
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    x["case"] = case
    x["cu"] = torch.tensor(_bounds(case), dtype=torch.int32, device=DEVICE)
    x["context"] = torch.tensor(_contexts(case), dtype=torch.int32, device=DEVICE)
    x["most"] = max(_ints(case["new"]))
    if own:  # the metadata of a packed batch, kept beside it
        import msa_triton_amd as msa

        x["seqs"] = msa.prepare_sequences(x["cu"])
    if case["op"] == "window" and case["grad"]:
        for name in ("q", "k", "v"):
            x[name].requires_grad_()
    return x


# ---------------------------------------------------------------------------- one pass


def run(x):
    return _own(x) if own else _PLAIN[x["case"]["op"]](x)


def _own(x):
    import msa_triton_amd as msa

    case = x["case"]
    window = case["window"] or None
    if case["op"] == "window":
        out, lse = msa.m3_window_attention(x["q"], x["k"], x["v"], x["seqs"], x["most"], window_size=window,
                                           sink_tokens=case["sinks"], return_lse=True)
        if not case["grad"]:
            return out, lse
        return out.detach(), lse, *torch.autograd.grad(out, (x["q"], x["k"], x["v"]), x["do"])
    if case["op"] == "serve":
        return msa.m3_window_attention_paged(x["q"], x["kc"], x["vc"], x["pages"], x["seqs"], x["context"],
                                             window_size=window, sink_tokens=case["sinks"], k_scale=x["ks"],
                                             v_scale=x["vs"], return_lse=True)
    return msa.m3_tree_attention_paged(x["q"], x["kc"], x["vc"], x["pages"], x["seqs"], x["context"], x["parents"],
                                       window_size=window, sink_tokens=case["sinks"], k_scale=x["ks"],
                                       v_scale=x["vs"], return_lse=True)


def _seen(query, key, case):
    """Which keys a query sees, from the positions of both: [queries, keys]."""
    back = query[:, None] - key
    seen = back >= 0
    if case["window"]:
        seen &= (back < case["window"]) | (key < case["sinks"])
    return seen


def _softmax_parts(q, k, seen):
    """Weights and log sums of rows q [G, R, D] (scaled) over k [G, L, D]; seen [R, L]."""
    logit = torch.matmul(q, k.transpose(1, 2)).masked_fill_(~seen, float("-inf"))
    most = logit.amax(2, keepdim=True)
    p = torch.exp_(logit.sub_(most))
    mass = p.sum(2, keepdim=True)
    return p.div_(mass), (most + torch.log(mass)).squeeze(2)


def _grouped(x, g):
    """[n, G * ratio, D] as [G, n * ratio, D] in 32 bits: the rows that share a key head."""
    n, hq, d = x.shape
    return x.float().view(n, g, hq // g, d).transpose(0, 1).reshape(g, n * hq // g, d)


def _ungrouped(x, n):
    g, rows, d = x.shape
    return x.view(g, n, rows // n, d).transpose(0, 1).reshape(n, g * rows // n, d)


def _plain_window(x):
    case = x["case"]
    g, ratio, scale = case["g"], case["hq"] // case["g"], case["d"] ** -0.5
    with torch.no_grad():
        q, k, v = x["q"], x["k"], x["v"]
        out = torch.empty_like(q)
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
        if case["grad"]:
            dq = torch.empty_like(q)
            dk, dv = torch.zeros_like(k, dtype=torch.float32), torch.zeros_like(v, dtype=torch.float32)
        bounds = _bounds(case)
        for a, b in zip(bounds, bounds[1:]):
            rows = max(1, BUDGET // (case["hq"] * min(b - a, case["window"] + case["sinks"] or b - a) + 1))
            for at in range(0, b - a, rows):
                end = min(at + rows, b - a)
                low = max(0, at - case["window"] + 1) if case["window"] else 0
                keys = torch.arange(low, end, device=DEVICE)
                if low:
                    keys = torch.cat([torch.arange(min(low, case["sinks"]), device=DEVICE), keys])
                kk, vv = k[a + keys].float().transpose(0, 1), v[a + keys].float().transpose(0, 1)
                query = torch.arange(at, end, device=DEVICE).repeat_interleave(ratio)
                qq = _grouped(q[a + at:a + end], g) * scale
                p, sums = _softmax_parts(qq, kk, _seen(query, keys, case))
                o = torch.matmul(p, vv)
                out[a + at:a + end] = _ungrouped(o, end - at).to(q.dtype)
                lse[a + at:a + end] = _ungrouped(sums[..., None], end - at)[..., 0]
                if case["grad"]:
                    do = _grouped(x["do"][a + at:a + end], g)
                    ds = torch.matmul(do, vv.transpose(1, 2)).sub_((do * o).sum(2, keepdim=True)).mul_(p)
                    dv.index_add_(0, a + keys, torch.matmul(p.transpose(1, 2), do).transpose(0, 1))
                    dk.index_add_(0, a + keys, torch.matmul(ds.transpose(1, 2), qq).transpose(0, 1))
                    dq[a + at:a + end] = _ungrouped(torch.matmul(ds, kk) * scale, end - at).to(q.dtype)
        if case["grad"]:
            return out, lse, dq, dk.to(k.dtype), dv.to(v.dtype)
        return out, lse


def _gather(x, s, keys):
    """Keys and values of positions `keys` of sequence s in 32 bits: [G, L, D] each."""
    case = x["case"]
    page, slot = x["pages"][s, keys // case["page"]].long(), keys % case["page"]
    k, v = x["kc"][page, :, slot].float(), x["vc"][page, :, slot].float()
    if x["ks"] is not None:
        k, v = k * x["ks"][page][..., None], v * x["vs"][page][..., None]
    return k.transpose(0, 1), v.transpose(0, 1)


def _plain_paged(x, nodes):
    """`nodes(s, a, b)`: depth of each new token and which new tokens each one sees (lower triangle without a tree)."""
    case = x["case"]
    g, ratio, scale = case["g"], case["hq"] // case["g"], case["d"] ** -0.5
    out = torch.empty_like(x["q"])
    lse = torch.empty(x["q"].shape[:2], dtype=torch.float32, device=DEVICE)
    bounds = _bounds(case)
    for s, (a, b, c) in enumerate(zip(bounds, bounds[1:], _contexts(case))):
        depth, among = nodes(a, b)
        rows = max(1, BUDGET // (case["hq"] * (c + b - a)))
        for at in range(0, b - a, rows):
            end = min(at + rows, b - a)
            low = max(0, c - case["window"] + 1) if case["window"] else 0
            keys = torch.arange(low, c + b - a, device=DEVICE)
            if low:
                keys = torch.cat([torch.arange(min(low, case["sinks"]), device=DEVICE), keys])
            position = torch.where(keys < c, keys, c + depth[(keys - c).clamp(min=0)])
            seen = _seen(c + depth[at:end], position, case)
            seen &= (keys < c) | among[at:end][:, (keys - c).clamp(min=0)]
            k, v = _gather(x, s, keys)
            p, sums = _softmax_parts(_grouped(x["q"][a + at:a + end], g) * scale, k,
                                     seen.repeat_interleave(ratio, 0))
            out[a + at:a + end] = _ungrouped(torch.matmul(p, v), end - at).to(out.dtype)
            lse[a + at:a + end] = _ungrouped(sums[..., None], end - at)[..., 0]
    return out, lse


def _plain_serve(x):
    def nodes(a, b):
        i = torch.arange(b - a, device=DEVICE)
        return i, i[:, None] >= i

    return _plain_paged(x, nodes)


def _plain_tree(x):
    def nodes(a, b):
        i = torch.arange(b - a, device=DEVICE)
        parent = x["parents"][a:b].long()
        reach = ((i == parent[:, None]) | (i == i[:, None])).float()
        for _ in range((b - a).bit_length()):  # twice as far each time
            reach = (torch.matmul(reach, reach) > 0).float()
        return reach.sum(1).long() - 1, reach > 0

    return _plain_paged(x, nodes)


_PLAIN = {"window": _plain_window, "serve": _plain_serve, "tree": _plain_tree}


# ---------------------------------------------------------------------------- work


def _pairs(n, context, case):
    """(query, key) pairs that a sequence of n new tokens behind `context` sees, and keys that any of them sees, without
    a tree."""
    w = case["window"] or n + context
    first = min(context + 1, w)  # keys of the first row's window; one more a row until the window is full
    rising = min(n, w - first)
    pairs = rising * first + rising * (rising - 1) // 2 + (n - rising) * w
    low = max(0, context + 1 - w)
    sinks = min(case["sinks"], context + n)
    for i in range(n):  # sinks in front of each row's window
        gap = context + i + 1 - w
        if gap >= sinks:
            pairs += (n - i) * sinks
            break
        pairs += max(0, gap)
    return pairs, context + n - low + min(low, sinks)


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    total, hq, d, g = _bounds(case)[-1], case["hq"], case["d"], case["g"]
    seen = [_pairs(n, c, case) for n, c in zip(_ints(case["new"]), _contexts(case))]
    pairs, keys = float(sum(p for p, _ in seen)), float(sum(k for _, k in seen))
    rows = float(total * hq)
    if case["op"] == "window":
        # forward: q, k, v in, out and log sums out; backward: those and the incoming gradient in, three gradients out
        moved = size * d * (2 * rows + 2 * total * g) + 4 * rows
        if case["grad"]:
            return {"bytes": 2 * moved + size * d * (2 * rows + 2 * total * g), "flops": 14.0 * pairs * hq * d}
        return {"bytes": moved, "flops": 4.0 * pairs * hq * d}
    held = 1 if case["cache"] == "fp8" else size
    if case["op"] == "tree":  # a row sees cached keys and a path
        pairs = 0.0
        for n, c in zip(_ints(case["new"]), _contexts(case)):
            near = min(c + n.bit_length(), case["window"] or c + n)
            pairs += n * (near + min(case["sinks"], c + n - near))
    return {"bytes": 2 * keys * g * d * held + rows * (2 * d * size + 4), "flops": 4.0 * pairs * hq * d}


# ---------------------------------------------------------------------------- float64


def exact(case, seed):
    x = _inputs(case, seed)
    return _exact_window(case, x) if case["op"] == "window" else _exact_paged(case, x)


def _attend(q, k, v, hidden, scale):
    """One key head's attention in float64: q [n, ratio, D], k and v [L, D], hidden [n, L]."""
    logit = (q @ k.T * scale).masked_fill(hidden[:, None], float("-inf"))
    return torch.softmax(logit, 2) @ v, torch.logsumexp(logit, 2)


def _exact_window(case, x):
    ratio, d, g = case["hq"] // case["g"], case["d"], case["g"]
    n_all = x["q"].shape[0]
    res = {name: torch.zeros(*x[name].shape, dtype=torch.float64, device=DEVICE) for name in ("q", "k", "v")}
    out = torch.zeros_like(res["q"])
    lse = torch.zeros(n_all, case["hq"], dtype=torch.float64, device=DEVICE)
    bounds = _bounds(case)
    w = case["window"] or n_all
    for a, b in zip(bounds, bounds[1:]):
        step = max(1, BUDGET // 4 // (ratio * min(b - a, w + case["sinks"])))
        for h in range(g):
            heads = slice(h * ratio, (h + 1) * ratio)
            for i in range(a, b, step):
                e = min(i + step, b)
                lo = max(a, i - w + 1)
                front = min(a + case["sinks"], lo)  # tokens a .. front are seen as well
                rows = torch.arange(i, e, device=DEVICE)[:, None]
                cols = torch.cat([torch.arange(a, front, device=DEVICE), torch.arange(lo, e, device=DEVICE)])
                hidden = (cols > rows) | ((rows - cols >= w) & (cols >= a + case["sinks"]))
                leaves = [x["q"][i:e, heads].double(), x["k"][cols, h].double(), x["v"][cols, h].double()]
                if case["grad"]:
                    leaves = [t.requires_grad_() for t in leaves]
                o, s = _attend(*leaves, hidden, d ** -0.5)
                out[i:e, heads], lse[i:e, heads] = o.detach(), s.detach()
                if case["grad"]:
                    dq, dk, dv = torch.autograd.grad(o, leaves, x["do"][i:e, heads].double())
                    res["q"][i:e, heads] = dq
                    res["k"][:, h].index_add_(0, cols, dk)
                    res["v"][:, h].index_add_(0, cols, dv)
                del o, s, leaves
    return (out, lse, res["q"], res["k"], res["v"]) if case["grad"] else (out, lse)


def _exact_paged(case, x):
    ratio, d, size = case["hq"] // case["g"], case["d"], case["page"]
    out = torch.zeros(*x["q"].shape, dtype=torch.float64, device=DEVICE)
    lse = torch.zeros(*x["q"].shape[:2], dtype=torch.float64, device=DEVICE)
    bounds = _bounds(case)
    parents = x["parents"].tolist() if case["op"] == "tree" else None
    for s, (a, b, c) in enumerate(zip(bounds, bounds[1:], _contexts(case))):
        n, total = b - a, c + b - a
        paths = []  # of each new token: the new tokens that it sees, the last one itself
        for i in range(n):
            if parents is None:
                paths.append(range(i + 1))
            else:
                paths.append([*(paths[parents[a + i]] if parents[a + i] >= 0 else []), i])
        pages = x["pages"][s, :-(-total // size)].long()
        for h in range(case["g"]):
            k, v = x["kc"][pages, h].double(), x["vc"][pages, h].double()
            if x["ks"] is not None:
                k, v = k * x["ks"][pages, h, None, None].double(), v * x["vs"][pages, h, None, None].double()
            k, v = k.reshape(-1, d)[:total], v.reshape(-1, d)[:total]
            step = max(1, BUDGET // 4 // (ratio * total))
            for i in range(0, n, step):
                e = min(i + step, n)
                shown = torch.zeros(e - i, total, dtype=torch.bool)
                for r, path in enumerate(paths[i:e]):
                    place = c + len(path) - 1
                    low = max(0, place - case["window"] + 1) if case["window"] else 0
                    shown[r, :min(case["sinks"], c)] = True
                    shown[r, low:c] = True
                    for deep, j in enumerate(path):
                        shown[r, c + j] = c + deep >= low or c + deep < case["sinks"]
                o, sums = _attend(x["q"][a + i:a + e, h * ratio:(h + 1) * ratio].double(), k, v,
                                  ~shown.to(DEVICE), d ** -0.5)
                out[a + i:a + e, h * ratio:(h + 1) * ratio] = o
                lse[a + i:a + e, h * ratio:(h + 1) * ratio] = sums
    return out, lse
