"""The operators around an 8-bit paged cache and the end of a speculative verify step, and the sizes they are
measured at:

* ``append``: rotary positions on queries and keys, keys and values stored in a paged cache of 8 bits
  (e4m3) with a power-of-two scale for each block of tokens and head;
* ``attention``: attention of drafted token trees over that cache;
* ``probs``: the probabilities that temperature, top-k, top-p and min-p leave of logits;
* ``verify``: verification of drafted tokens against the target's probabilities, from given random numbers;
* ``compact``: the accepted nodes' keys and values moved behind the context, in all layers.

``run`` computes a case in its plain form (elementary torch operations) or, where ``own`` is set, with the
package's operators.
"""

import math
import random

import torch

own = False

ONE = 1 << 40  # the weight of a row's most likely token, in the fixed point in which weights are summed
UNIT = float(1 << 52)  # probability one, in the fixed point in which residuals are summed
LARGEST = 448.0  # of e4m3
LOWEST = -40  # exponent of the smallest scale: blocks of zeros have it

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------------------- cases


def listed():
    app = dict(op="append")
    att = dict(op="attention")
    prb = dict(op="probs")
    ver = dict(op="verify")
    cmp = dict(op="compact")
    return [
        # the nodes of one request's tree, a quarter of each head rotated
        dict(app, name="append tree 8", batch=1, tokens=8, q_heads=16, kv_heads=2, dim=256, rotated=64,
             interleaved=False, page=64, block=64, type="bf16"),
        # a prompt chunk of an odd length, neighbouring elements paired
        dict(app, name="append prompt 4097", batch=1, tokens=4097, q_heads=32, kv_heads=8, dim=128, rotated=64,
             interleaved=True, page=16, block=16, type="fp16"),
        # one token, short chat: latency
        dict(att, name="attention decode 1k", batch=1, nodes=1, context=1000, q_heads=16, kv_heads=2,
             dim=256, page=64, block=64, type="bf16"),
        # one request, a 16-node tree, mid-length context: the verify step of single-stream decoding
        dict(att, name="attention tree 16 32k", batch=1, nodes=16, context=32768, q_heads=16, kv_heads=2,
             dim=256, page=64, block=32, type="bf16"),
        # a served batch with uneven contexts and trees
        dict(att, name="attention batch 24 ragged", batch=24, nodes=9, context=6001, q_heads=32,
             kv_heads=8, dim=128, page=16, block=16, type="fp16"),
        # long contexts under the widest trees
        dict(att, name="attention tree 64 128k", batch=4, nodes=64, context=131072, q_heads=32,
             kv_heads=8, dim=128, page=64, block=64, type="bf16"),
        # every node of a 16-node tree
        dict(prb, name="probs 16 rows", rows=16, vocab=151936, type="bf16", masked=False),
        # a served batch over the widest vocabulary, tokens banned by a grammar
        dict(prb, name="probs 128 rows", rows=128, vocab=248320, type="fp32", masked=True),
        # one request's chain of five drafted tokens behind its last one
        dict(ver, name="verify chain 6", batch=1, nodes=6, vocab=151936, drafts=True, chain=True),
        # a served batch of drafted trees
        dict(ver, name="verify batch 32 trees", batch=32, nodes=16, vocab=151936, drafts=True, chain=False),
        # one request, all layers of a 16-bit cache
        dict(cmp, name="compact one request", batch=1, nodes=16, layers=48, kv_heads=2, dim=256, page=64, block=0,
             type="bf16"),
        # a served batch, all layers of an 8-bit cache
        dict(cmp, name="compact batch 24 8-bit", batch=24, nodes=33, layers=48, kv_heads=8, dim=128, page=16,
             block=16, type="e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(16, 2), (32, 8), (12, 12), (16, 1), (64, 8), (24, 4)]
PAGES = [(16, 16), (32, 16), (48, 16), (64, 16), (64, 32), (64, 64), (96, 32), (256, 64)]


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "probs", "verify", "compact"])
    heads, dim = rng.choice(HEADS), rng.choice([64, 128, 256])
    page, block = rng.choice(PAGES)
    if op == "append":
        batch = _log(rng, 1, 32)
        most = min(4097, 4097 * 32 * 128 // (max(32, heads[0] + 2 * heads[1]) * dim * batch))
        return dict(op=op, batch=batch, tokens=_log(rng, 1, max(2, most)), q_heads=heads[0], kv_heads=heads[1],
                    dim=dim, rotated=rng.choice([dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5,
                    page=page, block=block, type=rng.choice(["bf16", "fp16"]))
    if op == "attention":
        nodes, batch = _log(rng, 1, 64), _log(rng, 1, 32)
        # no more cached bytes, nor products, than the largest listed case
        most = min(131072, 4 * 131072 * 8 * 128 // (batch * heads[1] * dim),
                   4 * 131072 * 64 * 32 * 128 // (batch * nodes * heads[0] * dim))
        return dict(op=op, batch=batch, nodes=nodes, context=_log(rng, 1, max(2, most)), q_heads=heads[0],
                    kv_heads=heads[1], dim=dim, page=page, block=block, type=rng.choice(["bf16", "fp16"]))
    vocab = rng.choice([49152, 151936, 248320, _log(rng, 1000, 248320)])
    if op == "probs":
        return dict(op=op, rows=_log(rng, 1, 128), vocab=vocab, type=rng.choice(["bf16", "fp16", "fp32"]),
                    masked=rng.random() < 0.5)
    if op == "verify":
        batch = _log(rng, 1, 32)
        # no more rows of probabilities than the largest listed case
        nodes = _log(rng, 1, min(64, 32 * 16 * 151936 // (batch * vocab)))
        return dict(op=op, batch=batch, nodes=nodes, vocab=vocab, drafts=rng.random() < 0.6, chain=rng.random() < 0.3)
    batch, wide = _log(rng, 1, 24), rng.random() < 0.5
    nodes = _log(rng, 1, 64)
    most = 24 * 33 * 48 * 8 * 128 // (batch * max(page, nodes) * heads[1] * dim)
    return dict(op=op, batch=batch, nodes=nodes, layers=_log(rng, 1, max(1, min(64, most))), kv_heads=heads[1],
                dim=dim, page=page, block=0 if wide else block, type=rng.choice(["bf16", "fp16"]) if wide else "e4m3")


def _lengths(case):
    """(context, nodes) of each request: the longest first, the others spread below it."""
    B, T, L = case["batch"], case["nodes"], case["context"]
    return [(L - (L * 5 * b) // (6 * B), 1 + (T - 1 + 5 * b) % T) for b in range(B)]


def _counts(case, key):
    """New tokens of each request."""
    B, T = case["batch"], case[key]
    return [1 + (T - 1 + 5 * b) % T for b in range(B)]


def work(case):
    if case["op"] == "append":
        H, K, D, size = case["q_heads"], case["kv_heads"], case["dim"], SIZE[case["type"]]
        T = sum(_counts(case, "tokens"))
        moved = T * ((2 * H + 2 * K) * D * size + 2 * K * D + case["rotated"] * 4 + 8)
        return {"bytes": moved + 8 * K * (T // case["block"] + case["batch"]), "flops": T * (3 * (H + K) * case["rotated"] + 4 * K * D)}
    if case["op"] == "attention":
        H, K, D, size = case["q_heads"], case["kv_heads"], case["dim"], SIZE[case["type"]]
        per = _lengths(case)
        keys = sum(c + t for c, t in per)
        nodes = sum(t for _, t in per)
        blocks = sum(-(-(c + t) // case["block"]) for c, t in per)
        return {"bytes": (keys * D * 2 + blocks * 8) * K + nodes * H * (2 * D * size + 4) + nodes * 8 + blocks * 4,
                "flops": sum(4 * (c + t) * t for c, t in per) * H * D}
    if case["op"] == "probs":
        return {"bytes": case["rows"] * (case["vocab"] * (SIZE[case["type"]] + 4) + 16),
                "flops": 5 * case["rows"] * case["vocab"]}
    if case["op"] == "verify":  # the rows at the path's end; the others are read at a few places
        rows = 2 if case["drafts"] and case["nodes"] > 1 else 1
        return {"bytes": case["batch"] * (rows * case["vocab"] * 4 + case["nodes"] * 24 + 16),
                "flops": 3 * case["batch"] * rows * case["vocab"]}
    # nodes whose place is not theirs yet are read and written once
    size = 1 if case["block"] else SIZE[case["type"]]
    paths = [_path(t, b) for b, t in enumerate(_counts(case, "nodes"))]
    moved = sum(n != d for path in paths for d, n in enumerate(path))
    return {"bytes": 2 * 2 * case["layers"] * moved * case["kv_heads"] * case["dim"] * size + 4 * sum(map(len, paths)) + 64,
            "flops": 0}


# --------------------------------------------------------------------------------------- inputs


def _generator(case, seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * seed + 29)


def _exponent(amax):
    """The exponent of the smallest power of two, 2^LOWEST at least, by which amax divided is at most LARGEST."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1); LARGEST = 7/8 2^9
    return torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), LOWEST).clamp(min=LOWEST)


def _scale(amax):
    """The power of two itself."""
    return ((_exponent(amax) + 127) << 23).view(torch.float32)


def _blocks(x, block):
    """[..., page, K, D] as [..., page / block, block, K, D]."""
    return x.unflatten(-3, (-1, block))


def _quantized(x, block):
    """(e4m3 tensor, scales [..., page / block, K]) of x [..., page, K, D] in 32 bits."""
    y = _blocks(x, block)
    scale = _scale(y.abs().amax((-3, -1)))
    return (y / scale[..., None, :, None]).flatten(-4, -3).to(E4M3), scale


def _page_table(need, pages, g):
    """int32 [B, max(need)]: page numbers in random order, -1 behind a request's own."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    used = torch.arange(max(need), device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device="cuda")
    table[used] = order[: sum(need)]
    return table


def _offsets(counts):
    return torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], dtype=torch.int32, device="cuda")


def _cache8(pages, page, K, D, block, g):
    """A cache whose blocks and heads have sizes of their own, as text gives them."""
    size = torch.exp2(torch.randn(pages, page // block, 1, K, 1, generator=g, device="cuda"))
    x = torch.randn(pages, page // block, block, K, D, generator=g, device="cuda") * size
    return _quantized(x.flatten(1, 2), block)


def _prepare_append(case, seed):
    g = _generator(case, seed)
    H, K, D, R, page, block = (case[k] for k in ("q_heads", "kv_heads", "dim", "rotated", "page", "block"))
    dtype, counts = TYPES[case["type"]], _counts(case, "tokens")
    T = sum(counts)
    qkv = torch.randn(T, (H + 2 * K) * D, generator=g, device="cuda").to(dtype)  # one projection's rows
    q, k, v = (x.view(T, -1, D) for x in qkv.split([H * D, K * D, K * D], dim=1))
    positions = 8192
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * _frequencies(case)
    # contexts that end inside a block, at its start, and none at all
    lens = [random.Random(1009 * seed + b).choice([0, block, page, 3, page + 7, 2 * page - 1, block + 5])
            for b in range(len(counts))]
    need = [-(-(2 * page + 7 + t) // page) for t in counts]  # whatever the context
    pages = sum(need) + 1
    first = torch.randint(0, positions - case["tokens"] + 1, (len(counts),), generator=g, device="cuda")
    offsets = _offsets(counts)
    request = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), offsets.diff().long(), output_size=T)
    place = torch.arange(T, device="cuda") - offsets.long()[request]
    k_cache, k_scale = _cache8(pages, page, K, D, block, g)
    v_cache, v_scale = _cache8(pages, page, K, D, block, g)
    return dict(case=case, q=q, k=k, v=v, positions=first[request] + place,
                context_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), node_offsets=offsets,
                page_table=_page_table(need, pages, g), table=torch.cat([angle.cos(), angle.sin()], 1).float(),
                k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale)


def _frequencies(case):
    half = case["rotated"] // 2
    return 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)


def _parents(t, b, chain=False):
    """Each node's parent, an earlier node; node 0 is the request's last token."""
    rng = random.Random(7919 * t + b)
    return [-1] + [i - 1 if chain else rng.randrange(max(0, i - 6), i) for i in range(1, t)]


def _path(t, b):
    """A path from node 0 on, through about half of the nodes, as a verification accepts it."""
    rng, path = random.Random(104729 * t + b), [0]
    while path[-1] < t - 3:
        path.append(path[-1] + rng.randrange(1, 4))
    return path


def _prepare_attention(case, seed):
    g = _generator(case, seed)
    H, K, D, page, block = (case[k] for k in ("q_heads", "kv_heads", "dim", "page", "block"))
    per = _lengths(case)
    need = [-(-(c + t) // page) for c, t in per]
    pages = sum(need) + 1
    k_cache, k_scale = _cache8(pages, page, K, D, block, g)
    v_cache, v_scale = _cache8(pages, page, K, D, block, g)
    masks = []
    for b, (_, t) in enumerate(per):  # a node sees itself and its ancestors
        seen = []
        for i, p in enumerate(_parents(t, b + seed)):
            seen.append((seen[p] if i else 0) | 1 << i)
        masks += seen
    masks = [m - (1 << 64) if m >> 63 else m for m in masks]
    offsets = _offsets([t for _, t in per])
    # keys have sizes around one: scores a little wider than a unit normal's
    q = torch.randn(len(masks), H, D, generator=g, device="cuda")
    return dict(case=case, q=q.to(TYPES[case["type"]]), k_cache=k_cache, v_cache=v_cache, k_scale=k_scale,
                v_scale=v_scale, page_table=_page_table(need, pages, g),
                context_lens=torch.tensor([c for c, _ in per], dtype=torch.int32, device="cuda"),
                node_offsets=offsets, tree_mask=torch.tensor(masks, dtype=torch.int64, device="cuda"),
                max_nodes=case["nodes"], max_context=case["context"])


def _logits(M, V, g):
    x = torch.randn(M, V, generator=g, device="cuda") * 2.2
    some = torch.randint(0, V, (M, 64), generator=g, device="cuda")  # the tokens the text makes likely
    return x.scatter_add_(1, some, torch.rand(M, 64, generator=g, device="cuda") * 12)


def _prepare_probs(case, seed):
    g = _generator(case, seed)
    M, V = case["rows"], case["vocab"]
    logits = _logits(M, V, g)
    if case["masked"]:  # tokens a grammar bans
        logits.masked_fill_(torch.rand(M, V, generator=g, device="cuda") < 0.3, -math.inf)
    row = torch.arange(M, device="cuda")
    pick = lambda *v: torch.tensor(v, device="cuda")[(row + seed) % len(v)]  # noqa: E731
    return dict(case=case, logits=logits.to(TYPES[case["type"]]),
                temperature=pick(0.7, 1.0, 0.6, 1.0, 0.0, 0.8, 1.2),
                top_k=pick(20, 50, 0, 0, 40, 1000).to(torch.int32),
                top_p=pick(0.95, 1.0, 0.8, 0.9, 0.95), min_p=pick(0.0, 0.0, 0.05, 0.02))


def _prepare_verify(case, seed):
    g = _generator(case, seed)
    counts = _counts(case, "nodes")
    N, V = sum(counts), case["vocab"]
    x = _logits(N, V, g)
    target = torch.softmax(x, -1)
    # the drafter sees nearly what the target sees
    draft = torch.softmax(x.add_(torch.randn(N, V, generator=g, device="cuda"), alpha=0.7), -1)
    parents = torch.tensor([p for b, t in enumerate(counts) for p in _parents(t, b + seed, case["chain"])],
                           dtype=torch.int32, device="cuda")
    offsets = _offsets(counts)
    request = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), offsets.diff().long(), output_size=N)
    row = offsets.long()[request] + parents.clamp(min=0)
    # a drafted token is drawn from its parent's row, or is one of its likeliest
    if case["drafts"]:
        tokens = torch.multinomial(draft[row], 1, generator=g)[:, 0]
    else:
        likely = torch.topk(draft, min(4, V), -1).indices
        tokens = likely[row, (torch.arange(N, device="cuda") - row) % likely.shape[1]]
    return dict(case=case, target_probs=target, draft_probs=draft if case["drafts"] else None, tokens=tokens,
                parents=parents, node_offsets=offsets, node_uniforms=torch.rand(N, generator=g, device="cuda"),
                draw_uniforms=torch.rand(len(counts), generator=g, device="cuda"), max_nodes=case["nodes"])


def _prepare_compact(case, seed):
    g = _generator(case, seed)
    L, K, D, page, block = (case[k] for k in ("layers", "kv_heads", "dim", "page", "block"))
    counts = _counts(case, "nodes")
    lens = [random.Random(1013 * seed + b).choice([0, 16, page, 3, page + 7, 2 * page - 1, 21]) for b in range(len(counts))]
    need = [-(-(2 * page + 7 + t) // page) for t in counts]  # whatever the context
    pages = sum(need) + 1
    paths = [_path(t, b) for b, t in enumerate(counts)]
    path = torch.full((len(counts), case["nodes"]), -1, dtype=torch.int32)
    for b, p in enumerate(paths):
        path[b, : len(p)] = torch.tensor(p, dtype=torch.int32)
    s = dict(case=case, page_table=_page_table(need, pages, g),
             context_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), path=path.cuda(),
             accepted=torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda"), k_scale=None,
             v_scale=None)
    for name in ("k", "v"):
        if block:
            x, scale = _cache8(L * pages, page, K, D, block, g)
            s[name + "_scale"] = scale.view(L, pages, -1, K)
        else:
            x = torch.randn(L * pages, page, K, D, generator=g, device="cuda").to(TYPES[case["type"]])
        s[name + "_cache"] = x.view(L, pages, page, K, D)
    return s


def prepare(case, seed):
    return {"append": _prepare_append, "attention": _prepare_attention, "probs": _prepare_probs,
            "verify": _prepare_verify, "compact": _prepare_compact}[case["op"]](case, seed)


# --------------------------------------------------------------------------------- the operators


def _rotate(x, cos, sin, interleaved):
    """x [T, H, D] in 32 bits, with its first 2 * cos.shape[1] elements of each head rotated."""
    R = 2 * cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., : R // 2], x[..., R // 2 : R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _append(s):
    case = s["case"]
    half, page, block = case["rotated"] // 2, case["page"], case["block"]
    at = s["table"][s["positions"]]
    cos, sin = at[:, :half], at[:, half:]
    q = _rotate(s["q"].float(), cos, sin, case["interleaved"]).to(s["q"].dtype)
    T = q.shape[0]
    request = torch.searchsorted(s["node_offsets"].long(), torch.arange(T, device="cuda"), right=True) - 1
    context = s["context_lens"].long()[request]
    place = context + torch.arange(T, device="cuda") - s["node_offsets"].long()[request]
    slot = s["page_table"].long()[request, place // page] * page + place % page
    leads = (place == context) | (place % block == 0)  # the first new token of its block
    number = leads.long().cumsum(0) - 1
    at = slot[leads] // block
    kept = (context - place // block * block).clamp(min=0)[leads]  # tokens that were there before
    stays = (torch.arange(block, device="cuda") < kept[:, None])[:, :, None, None]
    new = (("k", _rotate(s["k"].float(), cos, sin, case["interleaved"])), ("v", s["v"].float()))
    for name, x in new:
        K, D = x.shape[1:]
        rows, scale = s[name + "_cache"].view(torch.uint8).view(-1, K, D), s[name + "_scale"].view(-1, K)
        old, blocks = scale[at], rows.view(-1, block, K, D)[at]
        need = _scale(torch.zeros_like(old).index_reduce_(0, number, x.abs().amax(-1), "amax"))
        now = torch.where((kept > 0)[:, None], torch.maximum(need, old), need)
        again = (blocks.view(E4M3).float() * (old / now)[:, None, :, None]).to(E4M3).view(torch.uint8)
        rows.view(-1, block, K, D)[at] = torch.where(stays, again, blocks)  # what was there takes the new scale
        rows[slot] = (x / now[number][..., None]).to(E4M3).view(torch.uint8)
        scale[at] = now
    return {"q": q, **{k: s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale")}}


def _attention(s):
    case = s["case"]
    H, K, D, page, block = (case[k] for k in ("q_heads", "kv_heads", "dim", "page", "block"))
    T, G = s["max_nodes"], H // K
    table = s["page_table"].long().clamp(min=0)
    B, L = table.shape[0], table.shape[1] * page

    def gathered(cache, scale):
        x = cache.view(torch.uint8)[table].view(E4M3).float()
        x = _blocks(x, block) * scale[table][..., None, :, None]
        return x.view(B, L, K, D).transpose(1, 2)

    keys, values = gathered(s["k_cache"], s["k_scale"]), gathered(s["v_cache"], s["v_scale"])
    first, count = s["node_offsets"][:-1].long(), s["node_offsets"].diff().long()
    node = torch.arange(T, device=table.device)
    there = node < count[:, None]
    at = (first[:, None] + node).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[at].view(B, T, K, G, D).permute(0, 2, 1, 3, 4).reshape(B, K, T * G, D)
    scores = (q @ keys.transpose(-1, -2)) * D**-0.5
    # the context is seen by all nodes, drafted token j by the nodes whose mask has bit j
    drafted = torch.arange(L, device=table.device) - s["context_lens"].long()[:, None]
    bit = (s["tree_mask"][at][..., None] >> drafted.clamp(0, 63)[:, None]) & 1
    seen = (drafted < 0)[:, None] | ((drafted < count[:, None])[:, None] & (bit == 1))
    seen = seen[:, None, :, None].expand(B, 1, T, G, L).reshape(B, 1, T * G, L)
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weight = torch.exp(scores - top)
    total = weight.sum(-1, keepdim=True)
    out = (weight @ values) / torch.where(total == 0, 1.0, total)
    lse = torch.log(total) + top
    out = out.view(B, K, T, G, D).permute(0, 2, 1, 3, 4).reshape(B, T, H, D)
    lse = lse.view(B, K, T, G).permute(0, 2, 1, 3).reshape(B, T, H)
    return {"out": out[there].to(s["q"].dtype), "lse": lse[there]}


def _probs(s):
    x = s["logits"].float()
    x = torch.where(x.isnan(), -math.inf, x)
    V = x.shape[1]
    temperature, top_p, min_p = (s[k].float()[:, None] for k in ("temperature", "top_p", "min_p"))
    greedy = ~(temperature > 0)
    top_k = s["top_k"].long()[:, None]
    top_k = torch.where(greedy, 1, torch.where(top_k > 0, top_k, V))
    top = x.amax(-1, keepdim=True)
    weight = torch.exp((x - top) / torch.where(greedy, 1.0, temperature))
    weight = torch.where(x == top, 1.0, torch.where(x == -math.inf, 0.0, weight))
    weight = torch.where(top == -math.inf, 0.0, weight)
    fixed = (weight * ONE).long()  # sums of whole numbers do not depend on their order
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    mass = fixed.gather(1, order)
    mass = torch.where(torch.arange(V, device=x.device) < top_k, mass, 0)
    sums = mass.cumsum(-1)
    before = (sums - mass).double()
    inside = (before < top_p.double() * sums[:, -1:].double()) | (top_p >= 1)
    inside[:, 0] = True
    inside &= weight.gather(1, order) >= min_p
    mass = torch.where(inside, mass, 0)
    total = mass.sum(-1, keepdim=True)
    share = (mass.double() / torch.where(total == 0, 1, total).double()).float()
    return {"probs": torch.zeros_like(x).scatter_(1, order, share)}


def _verify(s):
    B, T = s["node_offsets"].shape[0] - 1, s["max_nodes"]
    offsets = s["node_offsets"].long()
    first, count, b = offsets[:-1], offsets.diff(), torch.arange(B, device="cuda")
    target, draft = s["target_probs"], s["draft_probs"]
    current = torch.zeros(B, dtype=torch.int64, device="cuda")
    path = torch.full((B, T), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    accepted = torch.ones(B, dtype=torch.int64, device="cuda")
    # what is left of the target's row at the path's end, and its sum
    left, total = target[first].double(), torch.ones(B, dtype=torch.float64, device="cuda")
    for i in range(1, T):  # a node's parent and elder siblings come before it
        at = (first + i).clamp(max=target.shape[0] - 1)
        asked = (i < count) & (s["parents"][at] == current)
        token, uniform = s["tokens"][at], s["node_uniforms"][at].double()
        chance = left[b, token]
        if draft is None:
            accept = asked & (uniform * total < chance)
        else:
            row = draft[first + current].double()
            accept = asked & (uniform * row[b, token] < chance * (1.0 / total))
        reject = asked & ~accept
        if draft is None:
            total = torch.where(reject, (total - chance).clamp(min=0), total)
            left[b, token] = torch.where(reject, 0.0, chance)
        else:
            rest = (left * (1.0 / total)[:, None] - row).clamp(min=0)
            whole = (rest * UNIT).long().sum(-1)
            reject &= whole > 0  # nothing left: what was before stays
            left = torch.where(reject[:, None], rest, left)
            total = torch.where(reject, whole.double() / UNIT, total)
        path[b, accepted.clamp(max=T - 1)] = torch.where(accept, i, path[b, accepted.clamp(max=T - 1)])
        accepted += accept
        current = torch.where(accept, i, current)
        left = torch.where(accept[:, None], target[first + current].double(), left)
        total = torch.where(accept, 1.0, total)
    sums = (left * UNIT).long().cumsum(-1)
    whole = sums[:, -1:]
    aim = torch.minimum((s["draw_uniforms"][:, None].double() * whole.double()).long(), whole - 1)
    token = (sums > aim).long().argmax(-1)
    return {"path": path, "accepted": accepted.int(), "tokens": torch.where(whole[:, 0] > 0, token, -1)}


def _compact(s):
    case = s["case"]
    page, block = case["page"], case["block"]
    place = torch.arange(s["path"].shape[1], device="cuda")
    moved = place < s["accepted"][:, None]
    context = s["context_lens"].long()[:, None]
    to, source = context + place, context + s["path"].long().clamp(min=0)
    table, last = s["page_table"].long(), s["page_table"].shape[1] - 1
    slot = lambda x: (table.gather(1, (x // page).clamp(max=last)) * page + x % page)[moved]  # noqa: E731
    dst, src = slot(to), slot(source)
    if block:
        leads = ((place == 0) | (to % block == 0))[moved]  # the first of its block
        number = leads.long().cumsum(0) - 1
        at = dst[leads] // block
        kept = (context - to // block * block).clamp(min=0)[moved][leads]  # tokens of the context in the block
        stays = (torch.arange(block, device="cuda") < kept[:, None])[:, :, None, None]
    for name in ("k", "v"):
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        L, K, D = cache.shape[0], *cache.shape[3:]
        if scale is None:
            rows = cache.view(L, -1, K, D)
            rows[:, dst] = rows[:, src]
            continue
        rows, scale = cache.view(torch.uint8).view(L, -1, K, D), scale.view(L, -1, K)
        # a block's scale is the largest of what stays in it and what comes to it
        old, came, whose = scale[:, at], rows[:, src], scale[:, src // block]
        now = torch.where((kept > 0)[:, None], old, 0.0).index_reduce_(1, number, whose, "amax")
        blocks = rows.view(L, -1, block, K, D)[:, at]
        again = (blocks.view(E4M3).float() * (old / now)[:, :, None, :, None]).to(E4M3).view(torch.uint8)
        rows.view(L, -1, block, K, D)[:, at] = torch.where(stays, again, blocks)
        rows[:, dst] = (came.view(E4M3).float() * (whose / now[:, number])[..., None]).to(E4M3).view(torch.uint8)
        scale[:, at] = now
    out = {k: s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale") if s[k] is not None}
    return {**out, "context_lens": s["context_lens"] + s["accepted"]}


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"append": _append, "attention": _attention, "probs": _probs, "verify": _verify,
                "compact": _compact}[case["op"]](s)
    import flash_next_rtxpro6000_b200 as fx

    if case["op"] == "append":
        q = fx.rotary_append8(s["q"], s["k"], s["v"], s["positions"], s["context_lens"], s["node_offsets"],
                              s["page_table"], s["table"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                              interleaved=case["interleaved"])
        return {"q": q, **{k: s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale")}}
    if case["op"] == "attention":
        out, lse = fx.tree_attention8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                                      s["page_table"], s["context_lens"], s["node_offsets"], s["tree_mask"],
                                      max_nodes=s["max_nodes"], max_context=s["max_context"])
        return {"out": out, "lse": lse}
    if case["op"] == "probs":
        return {"probs": fx.token_probs(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])}
    if case["op"] == "verify":
        path, accepted, tokens = fx.verify_tokens(s["target_probs"], s["draft_probs"], s["tokens"], s["parents"],
                                                  s["node_offsets"], s["node_uniforms"], s["draw_uniforms"],
                                                  max_nodes=s["max_nodes"])
        return {"path": path, "accepted": accepted, "tokens": tokens}
    lens = fx.compact_nodes(s["k_cache"], s["v_cache"], s["page_table"], s["context_lens"], s["path"],
                            s["accepted"], s["k_scale"], s["v_scale"])
    out = {k: s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale") if s[k] is not None}
    return {**out, "context_lens": lens}


# ------------------------------------------------------------------------------ in 64 bits


def _power(amax):
    """The smallest power of two by which amax divided is at most LARGEST, as a number."""
    return max(2.0**LOWEST, 2.0 ** math.ceil(math.log2(amax / LARGEST))) if amax > 0 else 2.0**LOWEST


def _exact_append(case, s):
    page, block, R = case["page"], case["block"], case["rotated"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * _frequencies(case))[:, None]  # a pair is a complex number

    def turned(x):
        y = x.double()
        z = y[..., :R]
        if case["interleaved"]:
            z = torch.view_as_real(torch.complex(z[..., 0::2].contiguous(), z[..., 1::2].contiguous()) * turn).flatten(-2)
        else:
            z = torch.complex(z[..., : R // 2].contiguous(), z[..., R // 2 :].contiguous()) * turn
            z = torch.cat([z.real, z.imag], -1)
        return torch.cat([z, y[..., R:]], -1)

    out = {"q": turned(s["q"])}
    offsets, lens, table = s["node_offsets"].tolist(), s["context_lens"].tolist(), s["page_table"].tolist()
    for name, x in (("k", turned(s["k"])), ("v", s["v"].double())):
        cache, scale = s[name + "_cache"].double(), s[name + "_scale"].double()
        for b, c in enumerate(lens):
            n = offsets[b + 1] - offsets[b]
            for j in range(c // block, (c + n - 1) // block + 1):  # the block's tokens lo .. hi - 1 are new
                lo, hi = max(c, j * block), min(c + n, (j + 1) * block)
                number, p = table[b][j * block // page], j * block % page
                new = x[offsets[b] + lo - c : offsets[b] + hi - c]
                amax = new.abs().amax((0, 2))
                need = torch.tensor([_power(v) for v in amax.tolist()], dtype=torch.float64, device="cuda")
                old = scale[number, p // block].clone()
                if lo > j * block:
                    need = torch.maximum(need, old)
                    cache[number, p : p + lo - j * block] *= (old / need)[:, None]
                scale[number, p // block] = need
                cache[number, p + lo - j * block : p + hi - j * block] = new / need[:, None]
        out[name + "_cache"], out[name + "_scale"] = cache, scale
    return out


def _exact_attention(case, s):
    H, K, D, page, block = (case[k] for k in ("q_heads", "kv_heads", "dim", "page", "block"))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    n = 0
    for b, (c, t) in enumerate(_lengths(case)):
        at = torch.arange(c + t, device="cuda")
        number, place = s["page_table"][b].long()[at // page], at % page
        bits = torch.tensor([[int(m) >> j & 1 for j in range(t)] for m in s["tree_mask"][n : n + t].tolist()],
                            device="cuda", dtype=torch.bool)
        hidden = torch.cat([torch.zeros(t, c, dtype=torch.bool, device="cuda"), ~bits], 1)
        for h in range(K):
            one = lambda x, z: x.view(torch.uint8)[number, place, h].view(E4M3).double() * z[number, place // block, h].double()[:, None]  # noqa: E731
            keys, values = one(s["k_cache"], s["k_scale"]), one(s["v_cache"], s["v_scale"])
            for j in range(h * (H // K), (h + 1) * (H // K)):
                scores = (s["q"][n : n + t, j].double() @ keys.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
                lse[n : n + t, j] = torch.logsumexp(scores, 1)
                out[n : n + t, j] = torch.softmax(scores, 1) @ values
        n += t
    return {"out": out, "lse": lse}


def _exact_probs(case, s):
    out = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
    for i in range(case["rows"]):
        x = s["logits"][i].double()
        t, k = float(s["temperature"][i]), int(s["top_k"][i])
        if t <= 0:
            out[i, x.argmax()] = 1.0
            continue
        p = torch.softmax(x / t, 0)
        index = torch.sort(x, descending=True, stable=True).indices
        q = p[index]
        if k > 0:
            q[k:] = 0.0
        q = q / q.sum()
        if float(s["top_p"][i]) < 1:
            ahead = torch.cat([q.new_zeros(1), q.cumsum(0)[:-1]])
            q = torch.where(ahead < float(s["top_p"][i]), q, 0.0)
        q = torch.where(p[index] >= float(s["min_p"][i]) * p.max(), q, 0.0)
        out[i, index] = q / q.sum()
    return {"probs": out}


def _exact_verify(case, s):
    offsets, parents, tokens = (s[k].tolist() for k in ("node_offsets", "parents", "tokens"))
    uniforms = s["node_uniforms"].double().tolist()
    paths, counts = [], []
    for b in range(case["batch"]):
        n0, n1 = offsets[b], offsets[b + 1]
        path = [0]
        children = lambda at: [i for i in range(n0 + 1, n1) if parents[i] == at]  # noqa: E731
        todo = children(0)
        p = s["target_probs"][n0].double()
        while todo:
            i = todo.pop(0)
            if s["draft_probs"] is None:
                q = torch.zeros_like(p)
                q[tokens[i]] = 1.0
            else:
                q = s["draft_probs"][n0 + path[-1]].double()
            if uniforms[i] * float(q[tokens[i]]) < float(p[tokens[i]]):
                path.append(i - n0)
                todo, p = children(i - n0), s["target_probs"][i].double()
                continue
            rest = (p - q).clamp(min=0)
            p = rest / rest.sum() if float(rest.sum()) > 0 else p
        paths.append(path + [-1] * (case["nodes"] - len(path)))
        counts.append(len(path))
    return {"path": torch.tensor(paths, dtype=torch.int32), "accepted": torch.tensor(counts, dtype=torch.int32), "tokens": None}


def _exact_compact(case, s):
    page, block = case["page"], case["block"]
    out = {"context_lens": s["context_lens"] + s["accepted"]}
    lens, accepted, table, paths = (s[k].tolist() for k in ("context_lens", "accepted", "page_table", "path"))
    for name in ("k", "v"):
        cache = s[name + "_cache"].double()
        was = cache.clone()
        if block:
            scale = s[name + "_scale"].double()
            old = scale.clone()
            out[name + "_scale"] = scale
        out[name + "_cache"] = cache
        for b, c in enumerate(lens):
            where = lambda x: (table[b][x // page], x % page)  # noqa: E731
            for j in range(c // (block or page), (c + accepted[b] - 1) // (block or page) + 1):
                size = block or page
                here = [d for d in range(accepted[b]) if (c + d) // size == j]
                if block:
                    number, p = where(j * block)
                    z = [old[:, where(c + paths[b][d])[0], where(c + paths[b][d])[1] // block] for d in here]
                    if c > j * block:
                        z.append(old[:, number, p // block])
                    z = torch.stack(z).amax(0)
                    if c > j * block:
                        cache[:, number, p : p + c - j * block] *= (old[:, number, p // block] / z)[:, None, :, None]
                    scale[:, number, p // block] = z
                for d in here:
                    (n1, p1), (n0, p0) = where(c + d), where(c + paths[b][d])
                    cache[:, n1, p1] = was[:, n0, p0]
                    if block:
                        cache[:, n1, p1] *= (old[:, n0, p0 // block] / z)[..., None]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "probs": _exact_probs, "verify": _exact_verify,
            "compact": _exact_compact}[case["op"]](case, s)
