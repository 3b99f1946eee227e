"""The operators of a speculative verify step that follow the drafted tokens through the model, and the
sizes they are measured at:

* ``rotary``: rotary positions on queries and keys, keys and values stored in a paged cache;
* ``attention``: attention of drafted token trees over a paged cache;
* ``sampling``: tokens drawn from logits with temperature, top-k, top-p and min-p, from given
  random numbers.

``run`` computes a case in its plain form (elementary torch operations in 32 bits) or, where ``own``
is set, with the package's operators.
"""

import math
import random

import torch

own = False

ONE = 1 << 40  # the weight of a row's most likely token, in the fixed point in which weights are summed

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------------------- cases


def listed():
    rot = dict(op="rotary")
    att = dict(op="attention")
    smp = dict(op="sampling")
    return [
        # one request's next token: a quarter of each head rotated, long-context table
        dict(rot, name="rotary decode", tokens=1, q_heads=16, kv_heads=2, dim=256, rotated=64,
             interleaved=False, page=64, positions=262144, scaled=True, type="bf16"),
        # the widest verify pass of the GEMV operators
        dict(rot, name="rotary verify 16", tokens=16, q_heads=32, kv_heads=8, dim=128, rotated=128,
             interleaved=False, page=16, positions=40960, scaled=False, type="bf16"),
        # a prompt chunk of an odd length, neighbouring elements paired
        dict(rot, name="rotary prompt 4097", tokens=4097, q_heads=32, kv_heads=8, dim=128, rotated=64,
             interleaved=True, page=16, positions=8192, scaled=False, type="fp16"),
        # one token, short chat: latency
        dict(att, name="attention decode 1k", batch=1, nodes=1, context=1000, q_heads=16, kv_heads=2,
             dim=256, page=64, type="bf16"),
        # one request, a 16-node tree, mid-length context: the verify step of single-stream decoding
        dict(att, name="attention tree 16 32k", batch=1, nodes=16, context=32768, q_heads=16, kv_heads=2,
             dim=256, page=64, type="bf16"),
        # a served batch with uneven contexts and trees
        dict(att, name="attention batch 24 ragged", batch=24, nodes=9, context=6001, q_heads=32,
             kv_heads=8, dim=128, page=16, type="fp16"),
        # small heads without sharing, pages that divide nothing
        dict(att, name="attention heads 64", batch=5, nodes=33, context=2777, q_heads=12, kv_heads=12,
             dim=64, page=24, type="bf16"),
        # long contexts under the widest trees
        dict(att, name="attention tree 64 128k", batch=4, nodes=64, context=131072, q_heads=32,
             kv_heads=8, dim=128, page=64, type="bf16"),
        # one request's token from the lm_head's logits
        dict(smp, name="sampling 1 row", rows=1, vocab=151936, type="bf16", masked=False),
        # every node of a 16-node tree
        dict(smp, name="sampling 16 rows", rows=16, vocab=151936, type="fp32", masked=False),
        # the reduced draft vocabulary, tokens banned by a grammar
        dict(smp, name="sampling draft vocab", rows=4, vocab=49152, type="bf16", masked=True),
        # a served batch over the widest vocabulary
        dict(smp, name="sampling 128 rows", rows=128, vocab=248320, type="fp32", masked=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "attention", "attention", "sampling"])
    if op == "rotary":
        heads = rng.choice([(16, 2), (32, 8), (8, 8), (24, 4), (64, 8), (7, 1)])
        dim = rng.choice([64, 128, 256])
        return dict(op=op, tokens=_log(rng, 1, 4097 if heads[0] * dim <= 4096 else 1024), q_heads=heads[0],
                    kv_heads=heads[1], dim=dim, rotated=rng.choice([dim, dim // 2, dim // 4]),
                    interleaved=rng.random() < 0.5, page=rng.choice([1, 16, 24, 64]),
                    positions=_log(rng, 8192, 262144), scaled=rng.random() < 0.5,
                    type=rng.choice(["bf16", "fp16"]))
    if op == "attention":
        heads = rng.choice([(16, 2), (32, 8), (12, 12), (16, 1), (64, 8), (24, 4)])
        dim = rng.choice([64, 128, 256])
        nodes = _log(rng, 1, 64)
        batch = _log(rng, 1, 32)
        # no more cached bytes, nor products, than the largest listed case
        most = min(131072, 4 * 131072 * 8 * 128 // (batch * heads[1] * dim),
                   4 * 131072 * 64 * 32 * 128 // (batch * nodes * heads[0] * dim))
        return dict(op=op, batch=batch, nodes=nodes, context=_log(rng, 1, max(2, most)), q_heads=heads[0],
                    kv_heads=heads[1], dim=dim, page=rng.choice([1, 16, 24, 64, 256]),
                    type=rng.choice(["bf16", "fp16"]))
    vocab = rng.choice([49152, 151936, 248320, _log(rng, 1000, 248320)])
    return dict(op=op, rows=_log(rng, 1, 128), vocab=vocab, type=rng.choice(["bf16", "fp16", "fp32"]),
                masked=rng.random() < 0.5)


def _lengths(case):
    """(context, nodes) of each request: the longest first, the others spread below it."""
    B, T, L = case["batch"], case["nodes"], case["context"]
    return [(L - (L * 5 * b) // (6 * B), 1 + (T - 1 + 5 * b) % T) for b in range(B)]


def work(case):
    if case["op"] == "rotary":
        T, H, K, D, R = (case[k] for k in ("tokens", "q_heads", "kv_heads", "dim", "rotated"))
        moved = 2 * T * (H + 2 * K) * D * SIZE[case["type"]] + T * (R * 4 + 12)
        return {"bytes": moved, "flops": 3 * T * (H + K) * R}
    if case["op"] == "attention":
        H, K, D, size = case["q_heads"], case["kv_heads"], case["dim"], SIZE[case["type"]]
        per = _lengths(case)
        keys = sum(c + t for c, t in per)
        nodes = sum(t for _, t in per)
        pages = sum(-(-(c + t) // case["page"]) for c, t in per)
        return {"bytes": keys * K * D * 2 * size + nodes * H * (2 * D * size + 4) + nodes * 8 + pages * 4,
                "flops": sum(4 * (c + t) * t for c, t in per) * H * D}
    return {"bytes": case["rows"] * (case["vocab"] * SIZE[case["type"]] + 32),
            "flops": 4 * case["rows"] * case["vocab"]}


# --------------------------------------------------------------------------------------- inputs


def _generator(case, seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)


def _frequencies(case):
    """The rotation's angle per position for each pair, and the factor on its cosine and sine. Scaled
    contexts: slow pairs are slowed down 8 times, fast ones kept, with a ramp between."""
    half = case["rotated"] // 2
    base, factor, original = 1000000.0, 8.0, 32768.0
    freq = base ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    if not case["scaled"]:
        return freq, 1.0
    turns = original * freq / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
    return freq * keep + freq / factor * (1 - keep), 0.1 * math.log(factor) + 1.0


def _prepare_rotary(case, seed):
    g = _generator(case, seed)
    T, H, K, D, page = (case[k] for k in ("tokens", "q_heads", "kv_heads", "dim", "page"))
    dtype = TYPES[case["type"]]
    qkv = torch.randn(T, (H + 2 * K) * D, generator=g, device="cuda").to(dtype)  # one projection's rows
    q, k, v = (x.view(T, -1, D) for x in qkv.split([H * D, K * D, K * D], dim=1))
    freq, factor = _frequencies(case)
    angle = torch.arange(case["positions"], dtype=torch.float64, device="cuda")[:, None] * freq
    table = torch.cat([angle.cos() * factor, angle.sin() * factor], 1).float()
    first = int(torch.randint(0, case["positions"] - T + 1, (1,), generator=g, device="cuda"))
    positions = torch.arange(first, first + T, device="cuda")
    pages = T // page + 2
    slots = torch.randperm(pages, generator=g, device="cuda")[:, None] * page + torch.arange(page, device="cuda")
    slots = slots.reshape(-1)[:T].clone()
    cache = [torch.zeros(pages, page, K, D, dtype=dtype, device="cuda") for _ in range(2)]
    return dict(case=case, q=q, k=k, v=v, table=table, positions=positions, slots=slots, k_cache=cache[0],
                v_cache=cache[1])


def _prepare_attention(case, seed):
    g = _generator(case, seed)
    H, K, D, page, dtype = case["q_heads"], case["kv_heads"], case["dim"], case["page"], TYPES[case["type"]]
    per = _lengths(case)
    need = [-(-(c + t) // page) for c, t in per]
    width = max(need)
    pages = sum(need) + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    used = torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    page_table = torch.full((len(per), width), -1, dtype=torch.int32, device="cuda")
    page_table[used] = order[: sum(need)]
    k_cache = torch.randn(pages, page, K, D, generator=g, device="cuda", dtype=dtype)
    v_cache = torch.randn(pages, page, K, D, generator=g, device="cuda", dtype=dtype)
    rng = random.Random(seed)
    masks = []
    for _, t in per:  # each node's parent is an earlier node; a node sees itself and its ancestors
        seen = []
        for i in range(t):
            seen.append((seen[rng.randrange(max(0, i - 6), i)] if i else 0) | 1 << i)
        masks += seen
    masks = [m - (1 << 64) if m >> 63 else m for m in masks]
    offsets = [0]
    for _, t in per:
        offsets.append(offsets[-1] + t)
    # scores a little wider than a unit normal's, so that some keys weigh far more than others
    q = torch.randn(offsets[-1], H, D, generator=g, device="cuda") * 1.5
    return dict(case=case, q=q.to(dtype), k_cache=k_cache, v_cache=v_cache, page_table=page_table,
                context_lens=torch.tensor([c for c, _ in per], dtype=torch.int32, device="cuda"),
                node_offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"),
                tree_mask=torch.tensor(masks, dtype=torch.int64, device="cuda"),
                max_nodes=case["nodes"], max_context=case["context"])


def _prepare_sampling(case, seed):
    g = _generator(case, seed)
    M, V = case["rows"], case["vocab"]
    logits = torch.randn(M, V, generator=g, device="cuda") * 2.2
    some = torch.randint(0, V, (M, 64), generator=g, device="cuda")  # the tokens the text makes likely
    logits.scatter_add_(1, some, torch.rand(M, 64, generator=g, device="cuda") * 12)
    if case["masked"]:  # tokens a grammar bans
        logits.masked_fill_(torch.rand(M, V, generator=g, device="cuda") < 0.3, -math.inf)
    row = torch.arange(M, device="cuda")
    pick = lambda *v: torch.tensor(v, device="cuda")[(row + seed) % len(v)]  # noqa: E731
    return dict(case=case, logits=logits.to(TYPES[case["type"]]),
                uniforms=torch.rand(M, generator=g, device="cuda"),
                temperature=pick(0.7, 1.0, 0.6, 1.0, 0.0, 0.8, 1.2),
                top_k=pick(20, 50, 0, 0, 40, 1000).to(torch.int32),
                top_p=pick(0.95, 1.0, 0.8, 0.9, 0.95),
                min_p=pick(0.0, 0.0, 0.05, 0.02))


def prepare(case, seed):
    return {"rotary": _prepare_rotary, "attention": _prepare_attention,
            "sampling": _prepare_sampling}[case["op"]](case, seed)


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


def _rotary(s):
    case = s["case"]
    half = case["rotated"] // 2
    at = s["table"][s["positions"]]
    cos, sin = at[:, :half], at[:, half:]
    q = _rotate(s["q"].float(), cos, sin, case["interleaved"]).to(s["q"].dtype)
    k = _rotate(s["k"].float(), cos, sin, case["interleaved"]).to(s["k_cache"].dtype)
    s["k_cache"].view(-1, *k.shape[1:])[s["slots"]] = k
    s["v_cache"].view(-1, *k.shape[1:])[s["slots"]] = s["v"].to(s["v_cache"].dtype)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attention(s):
    case = s["case"]
    H, K, D, page = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    T, G = s["max_nodes"], H // K
    table = s["page_table"].long().clamp(min=0)
    B, L = table.shape[0], table.shape[1] * page
    keys = s["k_cache"][table].view(B, L, K, D).transpose(1, 2).float()
    values = s["v_cache"][table].view(B, L, K, D).transpose(1, 2).float()
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


def _sampling(s):
    x = s["logits"].float()
    x = torch.where(x.isnan(), -math.inf, x)
    M, V = x.shape
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
    # the token at the random share of what is kept, from the most likely token on
    sums = mass.cumsum(-1)
    total = sums[:, -1:]
    target = (s["uniforms"][:, None].double() * total.double()).long()
    target = torch.minimum(target, total - 1)
    at = (sums > target).long().argmax(-1, keepdim=True)
    token = order.gather(1, at)
    prob = (mass.gather(1, at).double() / total.double()).float()
    none = total == 0
    return {"tokens": torch.where(none, -1, token)[:, 0], "probs": torch.where(none, 0.0, prob)[:, 0]}


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"rotary": _rotary, "attention": _attention, "sampling": _sampling}[case["op"]](s)
    import flash_next_rtxpro6000_b200 as fx

    if case["op"] == "rotary":
        q = fx.rotary_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["table"], s["k_cache"],
                             s["v_cache"], interleaved=case["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["op"] == "attention":
        out, lse = fx.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"],
                                     s["context_lens"], s["node_offsets"], s["tree_mask"],
                                     max_nodes=s["max_nodes"], max_context=s["max_context"])
        return {"out": out, "lse": lse}
    tokens, probs = fx.sample_tokens(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"],
                                     s["min_p"])
    return {"tokens": tokens, "probs": probs}


# ------------------------------------------------------------------------------ in 64 bits


def _exact_rotary(case, s):
    freq, factor = _frequencies(case)
    turn = torch.polar(torch.full((1,), factor, dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * freq)[:, None]  # a pair is a complex number

    def turned(x):
        x = x.double()
        R = case["rotated"]
        y = x[..., :R]
        if case["interleaved"]:
            z = torch.complex(y[..., 0::2].contiguous(), y[..., 1::2].contiguous()) * turn
            y = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(y[..., : R // 2].contiguous(), y[..., R // 2 :].contiguous()) * turn
            y = torch.cat([z.real, z.imag], -1)
        return torch.cat([y, x[..., R:]], -1)

    caches = []
    for old, new in ((s["k_cache"], turned(s["k"])), (s["v_cache"], s["v"].double())):
        c = old.double().view(-1, *old.shape[2:])
        c[s["slots"]] = new
        caches.append(c.view(old.shape))
    return {"q": turned(s["q"]), "k_cache": caches[0], "v_cache": caches[1]}


def _exact_attention(case, s):
    H, K, D, page = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    n = 0
    for b, (c, t) in enumerate(_lengths(case)):
        at = torch.arange(c + t, device="cuda")
        rows = (s["page_table"][b].long()[at // page] * page) + at % page
        bits = torch.tensor([[int(m) >> j & 1 for j in range(t)] for m in s["tree_mask"][n : n + t].tolist()],
                            device="cuda", dtype=torch.bool)
        hidden = torch.cat([torch.zeros(t, c, dtype=torch.bool, device="cuda"), ~bits], 1)
        for h in range(K):
            keys = s["k_cache"].view(-1, K, D)[rows, h].double()
            values = s["v_cache"].view(-1, K, D)[rows, h].double()
            for j in range(h * (H // K), (h + 1) * (H // K)):
                scores = (s["q"][n : n + t, j].double() @ keys.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
                lse[n : n + t, j] = torch.logsumexp(scores, 1)
                out[n : n + t, j] = torch.softmax(scores, 1) @ values
        n += t
    return {"out": out, "lse": lse}


def _exact_sampling(case, s):
    probs = []
    for i in range(case["rows"]):
        x = s["logits"][i].double()
        t, k = float(s["temperature"][i]), int(s["top_k"][i])
        p = torch.softmax(x / t, 0) if t > 0 else torch.nn.functional.one_hot(x.argmax(), len(x)).double()
        value, index = torch.sort(x, descending=True, stable=True)
        q = p[index]
        if k > 0:
            q = torch.where(torch.arange(len(x), device="cuda") < k, q, 0.0)
        q = q / q.sum()
        if float(s["top_p"][i]) < 1:
            ahead = torch.cat([q.new_zeros(1), q.cumsum(0)[:-1]])
            q = torch.where(ahead < float(s["top_p"][i]), q, 0.0)
        q = torch.where(p[index] >= float(s["min_p"][i]) * p.max(), q, 0.0)
        q = q / q.sum()
        token = int(torch.searchsorted(q.cumsum(0), float(s["uniforms"][i]), right=True))
        probs.append(q[min(token, len(x) - 1)])
    return {"tokens": None, "probs": torch.stack(probs)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "attention": _exact_attention,
            "sampling": _exact_sampling}[case["op"]](case, s)
