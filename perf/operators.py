"""Timed cases of the serving operators and of the query / key preparation.

Four operators that stand around the sparse attention path of a decoder layer:

* ``norm``    per-head RMS norm of queries and keys with the position rotation, forward alone
              (serving) or forward and backward (training): ``m3_qk_norm_rope``;
* ``append``  new keys, values and index keys written into a paged cache of 16-bit or 8-bit
              entries, keys normed and rotated on the way: ``m3_cache_append``;
* ``select``  indexer scores and causal top-k of new tokens against the paged index keys:
              ``m3_index_score_topk_paged``;
* ``attend``  sparse attention of new tokens over the selected blocks of the paged cache:
              ``m3_sparse_attention_paged``.

``run`` computes them in elementary torch operations, or with the package's operators where
``own`` is true; ``exact`` restates them in float64.
"""

from __future__ import annotations

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8 = torch.float8_e4m3fn
FP8_MOST = 448.0
EPS = 1e-6
DEVICE = "cuda"

# A serving batch: many requests of uneven length.
REQUESTS = ("1837,96,411,733,1290,57,208,1544,367,905,129,640,1021,288,77,1466,512,353,842,190,"
            "1127,33,675,1713,246,401,989,150,1358,568,301,784")


def _spread(n, low, high):
    """`n` lengths between `low` and `high`, spread evenly over their logarithm and mixed."""
    out = [int(round(low * (high / low) ** (((7 * i + 3) % n + 0.5) / n))) for i in range(n)]
    return ",".join(str(x) for x in out)


def _ones(n):
    return ",".join(["1"] * n)


def listed():
    return [
        # One decoding step of 64 requests: queries and keys of one token each. Launches count.
        dict(name="norm_decode", op="norm", dtype="bf16", new=_ones(64), context=_spread(64, 60, 30000), hq=32, g=4,
             d=128, rot=64, grad=False),
        # The smallest training configuration (c1): two short sequences, heads of 64, all dims rotated.
        dict(name="norm_train_small", op="norm", dtype="bf16", new="512,768", context="0,0", hq=8, g=2, d=64, rot=64,
             grad=True),
        # fp32, as used to check a model before it goes to 16 bits.
        dict(name="norm_train_fp32", op="norm", dtype="fp32", new="701,1347", context="0,0", hq=16, g=2, d=128,
             rot=128, grad=True),
        # The headline training configuration (c4): 32K tokens.
        dict(name="norm_train_32k", op="norm", dtype="bf16", new="32768", context="0", hq=32, g=4, d=128, rot=64,
             grad=True),
        # One decoding step of 64 requests into an 8-bit cache.
        dict(name="append_decode_fp8", op="append", dtype="bf16", cache="fp8", new=_ones(64),
             context=_spread(64, 60, 30000), g=4, d=128, di=128, rot=64, page=64),
        # Prompts of a serving batch into an 8-bit cache, some of them behind a cached prefix that ends in a page.
        dict(name="append_prompts_fp8", op="append", dtype="bf16", cache="fp8", new=REQUESTS,
             context="0,0,1000,0,37," + ",".join(["0"] * 27), g=4, d=128, di=128, rot=64, page=128),
        # Prompts of c3's size (odd lengths) into a 16-bit cache.
        dict(name="append_prompts", op="append", dtype="bf16", cache="16", new="2047,3071,5003,6151",
             context="0,0,0,0", g=4, d=128, di=128, rot=64, page=128),
        # Block selection in a decoding step of 32 requests.
        dict(name="select_decode", op="select", dtype="bf16", new=_ones(32), context=_spread(32, 500, 30000), g=4,
             di=128, block=128, page=64, topk=16, local=1),
        # Block selection for a drafted run of 5 tokens behind one very long context.
        dict(name="select_long_fp16", op="select", dtype="fp16", new="5", context="130000", g=4, di=128, block=128,
             page=128, topk=16, local=1),
        # One request at a time: latency.
        dict(name="attend_single", op="attend", dtype="bf16", cache="16", new="1", context="20011", hq=32, g=4, d=128,
             block=128, page=128, topk=16, local=1),
        # A decoding step of 64 requests over an 8-bit cache.
        dict(name="attend_decode_fp8", op="attend", dtype="bf16", cache="fp8", new=_ones(64),
             context=_spread(64, 60, 30000), hq=32, g=4, d=128, block=128, page=64, topk=16, local=1),
        # A decoding step of c5's heads, with a few drafted tokens for some requests.
        dict(name="attend_draft", op="attend", dtype="bf16", cache="16",
             new="1,1,4,1,1,4,1,1,2,1,4,1,1,1,1,3,1,1,4,1,1,1,1,1", context=_spread(24, 900, 30000), hq=64, g=8, d=128,
             block=128, page=128, topk=32, local=2),
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
    op = rng.choice(["norm", "norm", "append", "append", "select", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    g = rng.choice([1, 2, 4, 8])
    case = dict(op=op, dtype=dtype, g=g)
    if op == "norm":
        case["dtype"] = dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        case["d"] = rng.choice([64, 80, 96, 128, 128, 192, 256])
        case["rot"] = rng.choice([r for r in (32, 64, 64, 96, 128) if r <= case["d"]])
        case["hq"] = case["g"] * rng.choice([4, 8])
        case["grad"] = rng.random() < 0.6
        row = (case["hq"] + g) * case["d"] * DTYPES[dtype].itemsize
        new = _split(rng, _log_uniform(rng, 1, min(20000, 200_000_000 // row)), 24)
        context = [0] * len(new) if case["grad"] else [rng.choice([0, _log_uniform(rng, 1, 30000)]) for _ in new]
        return dict(case, new=_text(new), context=_text(context))
    if op == "append":
        case["cache"] = rng.choice(["fp8", "16"])
        case["d"] = rng.choice([64, 96, 128, 128, 256])
        case["di"] = rng.choice([64, 128])
        case["rot"] = rng.choice([32, 64])
        case["page"] = rng.choice([16, 64, 128])
        if rng.random() < 0.5:
            new = [rng.choice([1, 1, 1, 2, 4]) for _ in range(_log_uniform(rng, 1, 96))]
        else:
            new = _split(rng, _log_uniform(rng, 100, 12000), 24)
        most = max(200, 40000 // len(new))
        return dict(case, new=_text(new), context=_text(rng.choice([0, _log_uniform(rng, 1, most)]) for _ in new))
    case["page"] = rng.choice([16, 64, 128])
    case["block"] = rng.choice([64, 128, 128])
    case["topk"] = rng.choice([4, 8, 16, 16])
    case["local"] = rng.choice([1, 1, 2])
    new = [rng.choice([1, 1, 1, 1, 2, 5]) for _ in range(_log_uniform(rng, 1, 40))]
    most = max(2000, min(60000, 500_000 // len(new)))
    context = [_log_uniform(rng, 20, most) for _ in new]
    if op == "select":
        case["di"] = rng.choice([64, 96, 128, 128])
    else:
        case["cache"] = rng.choice(["fp8", "16"])
        case["hq"] = g * rng.choice([4, 8, 8, 16])
        case["d"] = rng.choice([64, 96, 128, 128, 256])
    return dict(case, new=_text(new), context=_text(context))


# ---------------------------------------------------------------------------- inputs


def _ints(text):
    return [int(x) for x in text.split(",")]


def _bounds(case):
    bounds = [0]
    for n in _ints(case["new"]):
        bounds.append(bounds[-1] + n)
    return bounds


def _totals(case):
    """Length of each sequence with its new tokens."""
    return [n + c for n, c in zip(_ints(case["new"]), _ints(case["context"]))]


def _pages(case, gen):
    """Page table [N, M] of a cache that other requests have used: pages in no order, -1 behind each sequence."""
    need = [-(-n // case["page"]) for n in _totals(case)]
    order = torch.randperm(sum(need) + 3, generator=gen, device=DEVICE, dtype=torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, order.numel()


def _cache(case, pages, heads, dim, gen, kind):
    """A filled cache [P, H, page, D], with its scales [P, H] where it is held in 8 bits."""
    x = torch.randn(pages, heads, case["page"], dim, generator=gen, device=DEVICE, dtype=torch.float32)
    if kind != "fp8":
        return x.to(DTYPES[case["dtype"]]), None
    scale = torch.exp2(torch.randint(-6, -4, (pages, heads), generator=gen, device=DEVICE).float())
    return (x / scale[:, :, None, None]).to(FP8), scale


def _selection(case, gen):
    """Distinct causal blocks of every (token, group): the local ones first, then by random score; -1 behind."""
    pos = _positions(case)
    nb = -(-max(_totals(case)) // case["block"])
    own_block = (pos // case["block"])[:, None, None]
    b = torch.arange(nb, device=DEVICE)[None, None]
    score = torch.rand(pos.numel(), case["g"], nb, generator=gen, device=DEVICE)
    score = score.masked_fill((b <= own_block) & (b > own_block - case["local"]), 2.0)
    score = score.masked_fill(b > own_block, -1.0)
    value, ids = torch.topk(score, min(case["topk"], nb), dim=2)
    ids = torch.where(value < 0, -1, ids).to(torch.int32)
    pad = torch.full((*ids.shape[:2], case["topk"] - ids.shape[2]), -1, dtype=torch.int32, device=DEVICE)
    return torch.cat([ids, pad], dim=2).contiguous()


def _positions(case):
    """Position of each new token in its sequence."""
    pos = [torch.arange(c, c + n) for n, c in zip(_ints(case["new"]), _ints(case["context"]))]
    return torch.cat(pos).to(DEVICE)


def _table(case, rows):
    """cos and sin of the first `rows` positions, fp32 [rows, rot]: the cosines, then the sines."""
    half = case["rot"] // 2
    freq = 5e6 ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half)
    angle = torch.arange(rows, dtype=torch.float64, device=DEVICE)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float().contiguous()


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(1000003 * int(seed) + 29)
    dtype = DTYPES[case["dtype"]]
    total = _bounds(case)[-1]

    def heads(n, dim):  # a projection's output: heads of different size
        size = 0.5 + 1.5 * torch.rand(n, 1, generator=gen, device=DEVICE)
        return (size * torch.randn(total, n, dim, generator=gen, device=DEVICE)).to(dtype)

    def weight(dim):
        return (1 + 0.2 * torch.randn(dim, generator=gen, device=DEVICE)).to(dtype)

    x = {}
    op = case["op"]
    if op in ("norm", "append"):
        x["table"] = _table(case, max(_totals(case)) + 1)
    if op == "norm":
        x["q"], x["k"] = heads(case["hq"], case["d"]), heads(case["g"], case["d"])
        x["wq"], x["wk"] = weight(case["d"]), weight(case["d"])
        if case["grad"]:
            x["dq"] = torch.randn(total, case["hq"], case["d"], generator=gen, device=DEVICE).to(dtype)
            x["dk"] = torch.randn(total, case["g"], case["d"], generator=gen, device=DEVICE).to(dtype)
        return x
    x["pages"], count = _pages(case, gen)
    if op == "append":
        x["k"], x["v"], x["ik"] = heads(case["g"], case["d"]), heads(case["g"], case["d"]), heads(1, case["di"])
        x["wk"], x["wi"] = weight(case["d"]), weight(case["di"])
        x["kc"], x["ks"] = _cache(case, count, case["g"], case["d"], gen, case["cache"])
        x["vc"], x["vs"] = _cache(case, count, case["g"], case["d"], gen, case["cache"])
        x["ic"], _ = _cache(case, count, 1, case["di"], gen, "16")
    if op == "select":
        x["iq"] = heads(case["g"], case["di"])
        x["ic"], _ = _cache(case, count, 1, case["di"], gen, "16")
    if op == "attend":
        x["q"] = heads(case["hq"], case["d"])
        x["kc"], x["ks"] = _cache(case, count, case["g"], case["d"], gen, case["cache"])
        x["vc"], x["vs"] = _cache(case, count, case["g"], case["d"], gen, case["cache"])
        x["ids"] = _selection(case, gen)
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    x["case"] = case
    x["cu"] = torch.tensor(_bounds(case), dtype=torch.int32, device=DEVICE)
    x["context"] = torch.tensor(_ints(case["context"]), dtype=torch.int32, device=DEVICE)
    x["most"] = max(_totals(case))
    if own:  # the metadata of a packed batch, kept beside it
        import msa_triton_amd as msa

        x["seqs"] = msa.prepare_sequences(x["cu"], block_size=case.get("block", 128))
    if case["op"] == "norm" and case["grad"]:
        for name in ("q", "k", "wq", "wk"):
            x[name].requires_grad_()
    return x


# ---------------------------------------------------------------------------- one pass


def run(x):
    return _own(x) if own else _PLAIN[x["case"]["op"]](x)


def _own(x):
    import msa_triton_amd as msa

    case = x["case"]
    op = case["op"]
    if op == "norm":
        if not case["grad"]:
            with torch.no_grad():
                return msa.m3_qk_norm_rope(x["q"], x["k"], x["wq"], x["wk"], x["table"], x["seqs"], eps=EPS,
                                           context_lens=x["context"])
        q, k = msa.m3_qk_norm_rope(x["q"], x["k"], x["wq"], x["wk"], x["table"], x["seqs"], eps=EPS)
        grads = torch.autograd.grad((q, k), (x["q"], x["k"], x["wq"], x["wk"]), (x["dq"], x["dk"]))
        return q.detach(), k.detach(), *grads
    if op == "append":
        msa.m3_cache_append(x["k"], x["v"], x["kc"], x["vc"], x["pages"], x["seqs"], x["context"],
                            index_k=x["ik"], index_cache=x["ic"], k_scale=x["ks"], v_scale=x["vs"], k_weight=x["wk"],
                            index_weight=x["wi"], cos_sin=x["table"], eps=EPS)
        return x["kc"], x["vc"], x["ic"], x["ks"], x["vs"]
    if op == "select":
        return msa.m3_index_score_topk_paged(x["iq"], x["ic"], x["pages"], x["seqs"], x["context"], x["most"],
                                             block_size=case["block"], topk_blocks=case["topk"],
                                             local_blocks=case["local"])
    return msa.m3_sparse_attention_paged(x["q"], x["kc"], x["vc"], x["ids"], x["pages"], x["seqs"], x["context"],
                                         block_size=case["block"], k_scale=x["ks"], v_scale=x["vs"], return_lse=True)


def _tokens(x, total):
    """Sequence and position of every new token, as the cache's lengths say."""
    t = torch.arange(total, device=DEVICE)
    seq = torch.searchsorted(x["cu"].long(), t, right=True) - 1
    return seq, x["context"].long()[seq] + t - x["cu"].long()[seq]


def _rotate(y, cos, sin):
    half = cos.shape[-1]
    a, b = y[..., :half], y[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]], dim=-1)


def _norm_rope(v, w, cos, sin, wide):
    v = v.to(wide)
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return _rotate(v * r * w.to(wide), cos.to(wide), sin.to(wide))


def _norm_rope_grad(v, w, cos, sin, dy):
    v, w, dy = v.float(), w.float(), dy.float()
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    dn = _rotate(dy, cos, -sin)
    n = v * r
    dv = r * (dn * w - n * (dn * w * n).mean(-1, keepdim=True))
    return dv, (dn * n).double().sum((0, 1))  # a long sum: 64 bits


def _plain_norm(x):
    case = x["case"]
    with torch.no_grad():
        q, k, wq, wk = x["q"], x["k"], x["wq"], x["wk"]
        _, pos = _tokens(x, q.shape[0])
        cs = x["table"][pos][:, None]
        half = case["rot"] // 2
        cos, sin = cs[..., :half], cs[..., half:]
        out = [_norm_rope(v, w, cos, sin, torch.float32).to(v.dtype) for v, w in ((q, wq), (k, wk))]
        if case["grad"]:
            dq, dwq = _norm_rope_grad(q, wq, cos, sin, x["dq"])
            dk, dwk = _norm_rope_grad(k, wk, cos, sin, x["dk"])
            out += [dq.to(q.dtype), dk.to(k.dtype), dwq.to(wq.dtype), dwk.to(wk.dtype)]
        return tuple(out)


def _round_fp8(y):
    """float64 values of at most 448 in magnitude, rounded once to e4m3 (to even); infinities become NaN."""
    y = torch.where(y.isfinite(), y, float("nan"))
    exponent = torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 1
    step = torch.exp2((exponent - 3).double())
    return (torch.round(y / step) * step).to(FP8)


def _scale_for(amax):
    """The smallest power of two s >= 2^-100 with 448 s >= amax; 0 for 0."""
    m, e = torch.frexp(amax / FP8_MOST)
    s = torch.exp2(torch.where(m == 0.5, e - 1, e).double().clamp(min=-100.0))
    return torch.where(amax == 0, 0.0, s)


def _put_fp8(rows, cache, scale, page_of, slot, pos, seq, x):
    """Rows [T, H, D] (float64) into an 8-bit cache, over the pages that they reach. A page's scale never shrinks while
    it holds earlier tokens; where it grows, they are rounded again."""
    page, at = torch.unique(page_of, return_inverse=True)
    _, heads, size, dim = cache.shape
    new = torch.zeros((page.numel(), heads, size, dim), dtype=torch.float64, device=DEVICE)
    new[at, :, slot] = rows
    fresh = torch.zeros((page.numel(), size), dtype=torch.bool, device=DEVICE)
    fresh[at, slot] = True
    kept = torch.zeros(page.numel(), dtype=torch.long, device=DEVICE)  # tokens of the page in front of the new ones
    kept[at] = (x["context"].long()[seq] - (pos - slot)).clamp(min=0)
    held, had = cache[page], scale[page].double()
    amax = torch.where(new.isfinite(), new, 0.0).abs().amax((2, 3))
    before = torch.where(kept[:, None] > 0, had, 0.0)
    after = torch.maximum(before, _scale_for(amax))
    safe = torch.where(after == 0, 1.0, after)[:, :, None, None]
    again = _round_fp8(held.double() * before[:, :, None, None] / safe)
    old = torch.arange(size, device=DEVICE)[None] < kept[:, None]
    moved = old[:, None, :, None] & (after != before)[:, :, None, None]
    held = torch.where(moved, again.float(), held.float())
    cache[page] = torch.where(fresh[:, None, :, None], _round_fp8(new / safe).float(), held).to(FP8)
    scale[page] = after.float()


def _plain_append(x):
    case = x["case"]
    size, half = case["page"], case["rot"] // 2
    seq, pos = _tokens(x, x["k"].shape[0])
    page_of, slot = x["pages"][seq, pos // size].long(), pos % size
    cs = x["table"][pos][:, None]
    cos, sin = cs[..., :half], cs[..., half:]
    k = _norm_rope(x["k"], x["wk"], cos, sin, torch.float64)
    x["ic"][page_of, :, slot] = _norm_rope(x["ik"], x["wi"], cos, sin, torch.float32).to(x["ic"].dtype)
    if case["cache"] == "fp8":
        _put_fp8(k, x["kc"], x["ks"], page_of, slot, pos, seq, x)
        _put_fp8(x["v"].double(), x["vc"], x["vs"], page_of, slot, pos, seq, x)
    else:
        x["kc"][page_of, :, slot] = k.to(x["kc"].dtype)
        x["vc"][page_of, :, slot] = x["v"]
    return x["kc"], x["vc"], x["ic"], x["ks"], x["vs"]


def _plain_select(x):
    case = x["case"]
    block, size = case["block"], case["page"]
    total, g, di = x["iq"].shape
    seq, pos = _tokens(x, total)
    nb = -(-x["most"] // block)
    keys = torch.arange(nb * block, device=DEVICE)
    page = x["pages"][:, (keys // size).clamp(max=x["pages"].shape[1] - 1)].long().clamp(min=0)
    k = x["ic"][page, 0, keys % size].double()  # [N, NB * block, Di]
    s = torch.empty(total, g, nb, dtype=torch.float32, device=DEVICE)
    n = max(1, (1 << 28) // (nb * block * max(g, di)))  # tokens at a time
    parts = []
    for q, w, p in zip(x["iq"].split(n), seq.split(n), pos.split(n)):
        dots = torch.matmul(q.double(), k[w].transpose(1, 2))
        dots = dots.masked_fill((keys[None] > p[:, None])[:, None], float("-inf"))
        parts.append(dots.view(len(p), g, nb, block).amax(3).float())
    s = torch.cat(parts)
    b = torch.arange(nb, device=DEVICE)
    own_block = (pos // block)[:, None]
    local = ((b <= own_block) & (b > own_block - case["local"]))[:, None]
    value, ids = torch.sort(s.masked_fill(local, float("inf")), dim=2, descending=True, stable=True)
    ids = torch.where(value == float("-inf"), -1, ids)[..., :case["topk"]].to(torch.int32)
    pad = torch.full((total, g, case["topk"] - ids.shape[2]), -1, dtype=torch.int32, device=DEVICE)
    return s, torch.cat([ids, pad], dim=2)


def _plain_attend(x):
    case = x["case"]
    block, size = case["block"], case["page"]
    total, hq, d = x["q"].shape
    g = case["g"]
    seq, pos = _tokens(x, total)
    keys = (x["ids"][..., None].long() * block + torch.arange(block, device=DEVICE)).flatten(2)  # [T, G, K * block]
    seen = (keys >= 0) & (keys <= pos[:, None, None]) & (x["ids"] >= 0).repeat_interleave(block, 2)
    keys = torch.where(seen, keys, 0)
    page = x["pages"][seq[:, None, None], keys // size].long()
    head = torch.arange(g, device=DEVICE)[None, :, None]
    k = x["kc"][page, head, keys % size].float()  # [T, G, K * block, D]
    v = x["vc"][page, head, keys % size].float()
    if x["ks"] is not None:
        k = k * x["ks"][page, head][..., None]
        v = v * x["vs"][page, head][..., None]
    q = x["q"].view(total, g, hq // g, d).float() * d ** -0.5
    logit = torch.matmul(q, k.transpose(2, 3)).masked_fill(~seen[:, :, None], float("-inf"))
    most = logit.amax(3, keepdim=True)
    most = torch.where(most == float("-inf"), 0.0, most)
    p = torch.exp(logit - most)
    mass = p.sum(3, keepdim=True)
    out = torch.matmul(p, torch.where(seen[..., None], v, 0.0)) / torch.where(mass == 0, 1.0, mass)
    lse = most + torch.log(mass)
    return out.reshape(total, hq, d).to(x["q"].dtype), lse.reshape(total, hq)


_PLAIN = {"norm": _plain_norm, "append": _plain_append, "select": _plain_select, "attend": _plain_attend}


# ---------------------------------------------------------------------------- work


def work(case):
    total = _bounds(case)[-1]
    size = DTYPES[case["dtype"]].itemsize
    op, g = case["op"], case["g"]
    if op == "norm":
        values = total * (case["hq"] + g) * case["d"]
        table = total * case["rot"] * 4
        if case["grad"]:  # forward: in and out; backward: in, incoming gradient and gradient
            return {"bytes": 5.0 * values * size + 2 * table, "flops": 25.0 * values}
        return {"bytes": 2.0 * values * size + table, "flops": 8.0 * values}
    if op == "append":
        held = 1 if case["cache"] == "fp8" else size
        kv, index = 2 * total * g * case["d"], total * case["di"]
        return {"bytes": float(kv * (size + held) + index * 2 * size + total * case["rot"] * 4),
                "flops": 8.0 * (kv + index)}
    new, totals = _ints(case["new"]), _totals(case)
    if op == "select":
        nb = -(-max(totals) // case["block"])
        keys = float(sum(n * t for n, t in zip(new, totals)))
        return {"bytes": float(sum(totals) * case["di"] * size + total * g * (case["di"] * size + 4 * nb + 4 * case["topk"])),
                "flops": 2.0 * case["di"] * g * keys}
    held = 1 if case["cache"] == "fp8" else size
    read = sum(min(t, n * case["topk"] * case["block"]) for n, t in zip(new, totals))
    seen = sum(n * min(t, case["topk"] * case["block"]) for n, t in zip(new, totals))
    return {"bytes": float(2 * read * g * case["d"] * held + total * case["hq"] * (2 * case["d"] * size + 4)),
            "flops": 4.0 * seen * case["hq"] * case["d"]}


# ---------------------------------------------------------------------------- float64


def exact(case, seed):
    x = _inputs(case, seed)
    return _EXACT[case["op"]](case, x)


def _exact_turn(case, v, w, pos, table):
    """Norm and rotation by complex products."""
    v = v.double()
    n = v / torch.sqrt(v.pow(2).sum(-1, keepdim=True) / v.shape[-1] + EPS) * w.double()
    half = case["rot"] // 2
    turn = torch.complex(table[pos, :half].double(), table[pos, half:].double())[:, None]
    z = torch.complex(n[..., :half], n[..., half:case["rot"]]) * turn
    return torch.cat([z.real, z.imag, n[..., case["rot"]:]], dim=-1)


def _exact_norm(case, x):
    pos = _positions(case)
    out, grads = [], []
    for v, w, dy in (("q", "wq", "dq"), ("k", "wk", "dk")):
        a, b = x[v].double(), x[w].double()
        if case["grad"]:
            a.requires_grad_()
            b.requires_grad_()
        y = _exact_turn(case, a, b, pos, x["table"])
        out.append(y.detach())
        if case["grad"]:
            grads.append(torch.autograd.grad(y, (a, b), x[dy].double()))
        del y
    if not case["grad"]:
        return tuple(out)
    return (*out, grads[0][0], grads[1][0], grads[0][1], grads[1][1])


def _exact_fp8(y):
    """The nearest e4m3 value, ties to the even code, by search in the list of all of them."""
    grid = torch.arange(127, dtype=torch.uint8, device=DEVICE).view(FP8).double()
    m = y.abs()
    hi = torch.searchsorted(grid, m.contiguous()).clamp(1, 126)
    lo = hi - 1
    below, above = m - grid[lo], grid[hi] - m
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return torch.where(up, grid[hi], grid[lo]).copysign(y)


def _exact_put(case, x, rows, cache, scale):
    """The cache's values and scales after the append, page by page."""
    held, scale, size = cache.double(), scale.double(), case["page"]
    bounds = _bounds(case)
    table = x["pages"].tolist()
    for s, (a, b) in enumerate(zip(bounds, bounds[1:])):
        c = _ints(case["context"])[s]
        for p in range(c // size, -(-(c + b - a) // size)):
            lo, hi = max(c, p * size), min(c + b - a, (p + 1) * size)
            page, kept = table[s][p], lo - p * size
            new = rows[a + lo - c:a + hi - c].transpose(0, 1)  # [H, n, D]
            top = new.abs().amax((1, 2)).cpu()
            for h in range(cache.shape[1]):
                need = 0.0
                if float(top[h]) > 0:
                    need = 2.0 ** -100
                    while 448.0 * need < float(top[h]):
                        need *= 2.0
                before = float(scale[page, h]) if kept else 0.0
                after = max(before, need)
                if after > 0 and after != before:
                    held[page, h, :kept] = _exact_fp8(held[page, h, :kept] * (before / after))
                held[page, h, kept:kept + hi - lo] = _exact_fp8(new[h] / after) if after > 0 else 0.0
                scale[page, h] = after
    return held, scale


def _exact_append(case, x):
    pos = _positions(case)
    size = case["page"]
    seq = torch.repeat_interleave(torch.arange(len(_ints(case["new"])), device=DEVICE),
                                  torch.tensor(_ints(case["new"]), device=DEVICE))
    k = _exact_turn(case, x["k"], x["wk"], pos, x["table"])
    ik = _exact_turn(case, x["ik"], x["wi"], pos, x["table"])
    ic = x["ic"].double()
    where = x["pages"][seq, pos // size].long() * size + pos % size
    ic.view(-1, case["di"])[where] = ik[:, 0]
    if case["cache"] == "fp8":
        pages = sum(n // size + 2 for n in _ints(case["new"])) * case["g"]
        if pages > 12000:  # too many to go through one by one
            return None, None, ic
        kc, ks = _exact_put(case, x, k, x["kc"], x["ks"])
        vc, vs = _exact_put(case, x, x["v"].double(), x["vc"], x["vs"])
        return kc, vc, ic, ks, vs
    caches = []
    for cache, rows in ((x["kc"], k), (x["vc"], x["v"].double())):
        flat = cache.double().transpose(1, 2).reshape(-1, case["g"], case["d"])
        flat[where] = rows
        caches.append(flat.view(-1, size, case["g"], case["d"]).transpose(1, 2).contiguous())
    return caches[0], caches[1], ic


def _exact_select(case, x):
    bounds, size, block = _bounds(case), case["page"], case["block"]
    nb = -(-max(_totals(case)) // block)
    out = torch.full((bounds[-1], case["g"], nb), float("-inf"), dtype=torch.float64, device=DEVICE)
    for s, (a, b) in enumerate(zip(bounds, bounds[1:])):
        c = _ints(case["context"])[s]
        pages = x["pages"][s, :-(-(c + b - a) // size)].long()
        keys = x["ic"][pages, 0].reshape(-1, case["di"]).double()
        for t in range(a, b):
            n = c + t - a + 1
            dots = x["iq"][t].double() @ keys[:n].T
            dots = torch.nn.functional.pad(dots, (0, -n % block), value=float("-inf"))
            out[t, :, :-(-n // block)] = dots.view(case["g"], -1, block).amax(2)
    return out, None


def _exact_attend(case, x):
    bounds, size, block = _bounds(case), case["page"], case["block"]
    total, hq, d = x["q"].shape
    ratio = hq // case["g"]
    out = torch.zeros(total, hq, d, dtype=torch.float64, device=DEVICE)
    lse = torch.full((total, hq), float("-inf"), dtype=torch.float64, device=DEVICE)
    ids, tables = x["ids"].tolist(), x["pages"].tolist()
    for s, (a, b) in enumerate(zip(bounds, bounds[1:])):
        for t in range(a, b):
            n = _ints(case["context"])[s] + t - a + 1
            for h in range(case["g"]):
                keys = [j for i in ids[t][h] if i >= 0 for j in range(i * block, min((i + 1) * block, n))]
                if not keys:
                    continue
                page = torch.tensor([tables[s][j // size] for j in keys], device=DEVICE)
                at = torch.tensor([j % size for j in keys], device=DEVICE)
                k, v = x["kc"][page, h, at].double(), x["vc"][page, h, at].double()
                if x["ks"] is not None:
                    k, v = k * x["ks"][page, h, None].double(), v * x["vs"][page, h, None].double()
                logit = x["q"][t, h * ratio:(h + 1) * ratio].double() @ k.T / d ** 0.5
                lse[t, h * ratio:(h + 1) * ratio] = torch.logsumexp(logit, 1)
                out[t, h * ratio:(h + 1) * ratio] = torch.softmax(logit, 1) @ v
    return out, lse


_EXACT = {"norm": _exact_norm, "append": _exact_append, "select": _exact_select, "attend": _exact_attend}
