"""The operators of speculative decoding with sampling, draft trees and an 8-bit cache: cases, plain forms, exact values.

Five kinds of case, one operator each:

  attn    `ops.tree_attention`: attention of a tree of drafted tokens (or of single tokens) over a paged cache
  cache   `ops.qkv_rope_append_fp8` then `ops.kv_read_fp8`: K/V rotated, quantised to e4m3 as they are written, read back
  chain   `ops.sample_accept`: a chain of drafts verified against the target's probabilities from given random numbers
  tree    `ops.tree_sample_accept`: the same for a tree of drafts
  commit  `ops.kv_commit_path`: the accepted path's cache rows moved together, in every layer

`own` false computes the plain form with elementary torch operations; true calls the framework.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
# (query heads, kv heads, head_dim): this repository's model shapes, then two common ones.
HEADS = [(14, 2, 64), (16, 2, 128), (4, 2, 64), (2, 1, 128), (32, 8, 128), (8, 8, 64)]
VOCABS = [1024, 32000, 50257, 151936]


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # One request of the fp32 configuration verifying a small tree: launch latency.
        dict(name="attn fp32 one request", kind="attn", dtype="fp32", cache="same", heads=14, kv_heads=2, head_dim=64,
             batch=1, nodes=9, ctx=131, block=16, tree=True, ragged=False),
        # The 3B target verifying 16-node trees for a batch of 64 requests: an ordinary step.
        dict(name="attn bf16 batch", kind="attn", dtype="bf16", cache="same", heads=16, kv_heads=2, head_dim=128,
             batch=64, nodes=16, ctx=700, block=16, tree=True, ragged=True),
        # Wide trees over long contexts: the most arithmetic a verify step meets.
        dict(name="attn bf16 wide trees", kind="attn", dtype="bf16", cache="same", heads=16, kv_heads=2, head_dim=128,
             batch=32, nodes=64, ctx=4500, block=16, tree=True, ragged=False),
        # Single tokens over long 8-bit caches: the cache's bytes are all there is.
        dict(name="attn fp8 long decode", kind="attn", dtype="bf16", cache="fp8", heads=16, kv_heads=2, head_dim=128,
             batch=64, nodes=1, ctx=9000, block=16, tree=False, ragged=True),
        # A decode step's new rows (64 requests, the 0.5B shape) written to the 8-bit cache.
        dict(name="cache decode step", kind="cache", dtype="bf16", heads=14, kv_heads=2, head_dim=64, tokens=64,
             block=16),
        # A batch of prompts of the 3B shape written to it.
        dict(name="cache prompts", kind="cache", dtype="bf16", heads=16, kv_heads=2, head_dim=128, tokens=16384,
             block=16),
        # One request with greedily drafted tokens (no draft distribution): latency of a single stream.
        dict(name="chain bf16 one request", kind="chain", dtype="bf16", batch=1, k=4, vocab=151936, draft=False,
             filtered=False, greedy=False),
        # A large batch with sampled drafts and their logits.
        dict(name="chain fp32 batch", kind="chain", dtype="fp32", batch=128, k=4, vocab=151936, draft=True,
             filtered=False, greedy=False),
        # A small vocabulary, two requests, one of them greedy.
        dict(name="tree fp32 small", kind="tree", dtype="fp32", batch=2, nodes=7, vocab=1024, filtered=False,
             greedy=True),
        # The verify step of 64 requests with 16-node trees.
        dict(name="tree bf16 batch", kind="tree", dtype="bf16", batch=64, nodes=16, vocab=151936, filtered=False,
             greedy=False),
        # One request of the 0.5B shape on an 8-bit cache.
        dict(name="commit fp8 one request", kind="commit", dtype="bf16", cache="fp8", kv_heads=2, head_dim=64, layers=24,
             batch=1, nodes=9, block=16),
        # The whole batch of the 3B shape.
        dict(name="commit bf16 batch", kind="commit", dtype="bf16", cache="same", kv_heads=2, head_dim=128, layers=36,
             batch=64, nodes=16, block=16),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "cache", "chain", "tree", "commit"])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    block = rng.choice([16, 16, 16, 1, 7, 32, 64])
    if kind == "attn":
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        cache = rng.choice(["same", "fp8"]) if dtype == "bf16" else "same"
        nodes = rng.choice([1, _log_int(rng, 2, 64)])
        batch = _log_int(rng, 1, 64)
        # at most the largest listed case's arithmetic, and the long decode's bytes; fp32 an eighth of them
        work = 32 * 64 * 4500 * 16 * 128 // (8 if dtype == "fp32" else 1)
        rows = 64 * 9000 * 2 * 128 // (8 if dtype == "fp32" else 2 if cache == "same" else 1)
        most = min(16000, work // (batch * nodes * heads * head_dim), rows // (batch * kv_heads * head_dim))
        return dict(kind="attn", dtype=dtype, cache=cache, heads=heads, kv_heads=kv_heads, head_dim=head_dim, batch=batch,
                    nodes=nodes, ctx=_log_int(rng, 1, max(1, most)), block=block, tree=nodes > 1 and rng.random() < 0.8,
                    ragged=rng.random() < 0.7)
    if kind == "cache":
        most = 16384 * 20 * 128 // ((heads + 2 * kv_heads) * head_dim)
        return dict(kind="cache", dtype=rng.choice(["bf16", "bf16", "fp32"]), heads=heads, kv_heads=kv_heads,
                    head_dim=head_dim, tokens=_log_int(rng, 1, most // 2), block=block)
    vocab = rng.choice(VOCABS)
    if kind == "chain":
        k, draft = rng.randint(1, 8), rng.random() < 0.6
        most = 128 * 9 * 151936 // ((2 * k + 1) * vocab)
        return dict(kind="chain", dtype=rng.choice(["bf16", "fp32"]), batch=_log_int(rng, 1, min(256, most)), k=k,
                    vocab=vocab, draft=draft, filtered=rng.random() < 0.3, greedy=rng.random() < 0.3)
    if kind == "tree":
        nodes = _log_int(rng, 2, 64)
        most = 64 * 16 * 151936 // (nodes * vocab)
        return dict(kind="tree", dtype=rng.choice(["bf16", "fp32"]), batch=_log_int(rng, 1, min(256, most)), nodes=nodes,
                    vocab=vocab, filtered=rng.random() < 0.3, greedy=rng.random() < 0.3)
    return dict(kind="commit", dtype=rng.choice(["bf16", "fp32"]), cache=rng.choice(["same", "fp8"]), kv_heads=kv_heads,
                head_dim=head_dim, layers=rng.randint(1, 36), batch=_log_int(rng, 1, 64 // (kv_heads // 2 or 1)),
                nodes=_log_int(rng, 2, 16), block=block)


def _own_rng(case):
    """What belongs to the case whatever the seed: lengths and trees."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _trees(case, rng):
    """A random tree per sequence: parents in ascending order, node 0 the root, a few children each."""
    trees = []
    for _ in range(case["batch"]):
        n = case["nodes"]
        if case.get("ragged"):
            n = rng.randint(max(1, n // 2), n)
        trees.append([-1] + [rng.randint(max(0, i - 6), i - 1) for i in range(1, n)])
    return trees


def _lengths(case):
    """(history length, new tokens, parents) of every sequence."""
    rng = _own_rng(case)
    trees = _trees(case, rng)
    hist = [rng.randint(max(1, case["ctx"] // 4), case["ctx"]) if case.get("ragged") else case["ctx"] for _ in trees]
    return hist, [len(t) for t in trees], trees


def _work_attn(case):
    hist, nodes, _ = _lengths(case)
    hd, nq, nkv = case["head_dim"], case["heads"], case["kv_heads"]
    elem = 4 if case["dtype"] == "fp32" else 2
    keys = sum(h + n for h, n in zip(hist, nodes))
    row = hd + 1 if case["cache"] == "fp8" else hd * elem
    visible = sum(n * h + (n * (n + 1) // 2) for h, n in zip(hist, nodes))
    return {"bytes": 2 * keys * nkv * row + 2 * sum(nodes) * nq * hd * elem, "flops": 4 * visible * nq * hd}


def work(case):
    kind = case["kind"]
    if kind == "attn":
        return _work_attn(case)
    if kind == "cache":
        elem = 4 if case["dtype"] == "fp32" else 2
        t, nq, nkv, hd = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        # qkv in, q out, the cache rows written and read, K and V out
        bytes_ = t * hd * elem * (nq + 2 * nkv) + t * hd * elem * nq + 2 * 2 * t * nkv * (hd + 1) + 2 * t * nkv * hd * elem
        return {"bytes": bytes_ + t * hd * 4, "flops": 3 * t * (nq + nkv) * hd + 4 * t * nkv * hd}
    if kind in ("chain", "tree"):
        elem = 4 if case["dtype"] == "fp32" else 2
        rows = case["nodes"] if kind == "tree" else case["k"] * (2 if case["draft"] else 1) + 1
        values = case["batch"] * rows * case["vocab"]
        return {"bytes": values * elem + case["batch"] * case["vocab"] * 4, "flops": 3 * values}
    hist, nodes, trees = _commit_lengths(case)
    moved = sum(len(p) - 1 for p in _paths(case, trees))
    row = case["head_dim"] + 1 if case["cache"] == "fp8" else case["head_dim"] * (4 if case["dtype"] == "fp32" else 2)
    return {"bytes": 2 * 2 * moved * case["layers"] * case["kv_heads"] * row, "flops": 0}


# ---------------------------------------------------------------------------- inputs
def _pages(case, lens, rng, device):
    """Shuffled block tables [batch, width] int32 and the number of blocks of the pool."""
    bs = case["block"]
    need = [-(-n // bs) for n in lens]
    blocks = list(range(sum(need) + 3))
    rng.shuffle(blocks)
    width = max(need)
    flat, at = [], 0
    for n in need:
        flat.append(blocks[at:at + n] + [0] * (width - n))
        at += n
    return torch.tensor(flat, dtype=torch.int32, device=device), len(blocks)


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _generator(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


def _ancestors(trees, words, device):
    """Mask words [rows, words]: bit j of a node's row is set for itself and its ancestors."""
    rows = []
    for t in trees:
        bits = []
        for i, p in enumerate(t):
            bits.append((bits[p] if p >= 0 else 0) | 1 << i)
        for b in bits:
            rows.append([(b >> 32 * w & 0xFFFFFFFF) for w in range(words)])
    return torch.tensor(rows, dtype=torch.int64).to(torch.int32).to(device)


def _random_cache(shape, case, g, device):
    """A cache with contents: (values, None), or e4m3 values and their scale bytes (exponent + 127)."""
    if case["cache"] != "fp8":
        return torch.randn(shape, generator=g, device=device).to(DTYPES[case["dtype"]]), None
    values = (torch.randn(shape, generator=g, device=device) * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)
    return values, torch.randint(119, 123, shape[:-1], generator=g, device=device).to(torch.uint8)


def _prepare_attn(case, seed, device):
    g, rng = _generator(seed, device), random.Random(seed)
    hist, nodes, trees = _lengths(case)
    ctx = [h + n for h, n in zip(hist, nodes)]
    tables, num_blocks = _pages(case, ctx, rng, device)
    shape = (num_blocks, case["block"], case["kv_heads"], case["head_dim"])
    s = {"case": case, "tables": tables, "ctx": _i32(ctx, device), "q_lens": _i32(nodes, device), "max_q": max(nodes),
         "max_ctx": max(ctx), "scale": case["head_dim"] ** -0.5}
    offsets = [0]
    for n in nodes:
        offsets.append(offsets[-1] + n)
    s["q_offsets"] = _i32(offsets, device)
    s["q"] = torch.randn(offsets[-1], case["heads"], case["head_dim"], generator=g, device=device).to(
        DTYPES[case["dtype"]])
    s["mask"] = _ancestors(trees, -(-max(nodes) // 32), device) if case["tree"] else None
    for x in "kv":
        s[x], s[x + "_scale"] = _random_cache(shape, case, g, device)
    # where a row of the padded [batch, max_q] layout lies in the packed one
    at = torch.arange(max(nodes), device=device)[None] + s["q_offsets"][:-1, None]
    s["padded"] = at.clamp_(max=offsets[-1] - 1).long()
    s["packed"] = torch.tensor([b * max(nodes) + i for b, n in enumerate(nodes) for i in range(n)], device=device)
    return s


def _prepare_cache(case, seed, device):
    g, rng = _generator(seed, device), random.Random(seed)
    nq, nkv, hd, n, bs = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"], case["block"]
    num_blocks = -(-n // bs) + 5
    # rows of prompts or of many sequences' single tokens: any distinct slots, any positions
    slots = torch.randperm(num_blocks * bs, generator=g, device=device)[:n]
    longest = 32768
    inv = 1e6 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    angle = torch.arange(longest, dtype=torch.float64)[:, None].to(device) * inv[None].to(device)
    shape = (num_blocks, bs, nkv, hd)
    # activations: unit rows with the few large channels that keys have
    spread = 1 + 7 * (torch.rand((nq + 2 * nkv) * hd, generator=g, device=device) < 0.02)
    qkv = torch.randn(n, (nq + 2 * nkv) * hd, generator=g, device=device) * spread
    s = {"case": case, "qkv": qkv.to(DTYPES[case["dtype"]]), "slots": slots, "slots32": slots.to(torch.int32),
         "positions": torch.randint(0, longest, (n,), generator=g, device=device).to(torch.int32),
         "cos": angle.cos().float(), "sin": angle.sin().float()}
    s["q_out"] = torch.empty(n, nq, hd, dtype=DTYPES[case["dtype"]], device=device)
    for x in "kv":
        s[x] = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        s[x + "_scale"] = torch.full(shape[:-1], 127, dtype=torch.uint8, device=device)
    return s


def _temperatures(case, g, device):
    t = 0.5 + 0.8 * torch.rand(case["batch"], generator=g, device=device)
    if case["greedy"]:
        t[::2] = 0
    return t


def _filter(x, keep):
    """What a top-k filter leaves: everything below a row's threshold is minus infinity."""
    return x.masked_fill_(x < keep, -math.inf)


def _gumbel(shape, g, device):
    return -torch.empty(shape, device=device).exponential_(generator=g).log()


def _prepare_chain(case, seed, device):
    g = _generator(seed, device)
    b, k, vocab, dtype = case["batch"], case["k"], case["vocab"], DTYPES[case["dtype"]]
    t = _temperatures(case, g, device)
    target = torch.randn(b, k + 1, vocab, generator=g, device=device) * 2.5
    # the draft model agrees with the target up to some noise
    draft = target[:, :k] * 0.9 + torch.randn(b, k, vocab, generator=g, device=device)
    if case["filtered"]:
        _filter(target, 2.0)
        _filter(draft, 2.0)
    target, draft = target.to(dtype), draft.to(dtype)
    # drafts drawn from the draft's distribution, or its largest logits where it is greedy
    noise = _gumbel((b, 1, vocab), g, device) * (t[:, None, None] if case["draft"] else 0)
    drafts = torch.stack([(draft[:, j].float() + noise[:, 0]).argmax(-1) for j in range(k)], 1)
    u = torch.rand(b, k, generator=g, device=device)
    s = {"case": case, "logits": target, "draft_logits": draft if case["draft"] else None, "t": t,
         "drafts": drafts.to(torch.int32), "u": u, "gumbel": _gumbel((b, vocab), g, device)}
    return s


def _prepare_tree(case, seed, device):
    g = _generator(seed, device)
    b, vocab = case["batch"], case["vocab"]
    _, nodes, trees = _lengths(dict(case, ctx=1))
    n = sum(nodes)
    logits = torch.randn(n, vocab, generator=g, device=device) * 2.5
    # siblings draft their parent's likeliest tokens by a noisy guess: the rank-th largest
    parents = [p for t in trees for p in t]
    base = [off for off, m in zip([sum(nodes[:i]) for i in range(b)], nodes) for _ in range(m)]
    rank = [sum(q == p for q in t[:i]) for t in trees for i, p in enumerate(t)]
    guess = torch.cat([(rows + 0.7 * torch.randn(rows.shape, generator=g, device=device)).topk(min(vocab, 64)).indices
                       for rows in logits.split(64)])
    from_row = torch.tensor([o + max(p, 0) for o, p in zip(base, parents)], device=device)
    tokens = guess[from_row, torch.tensor(rank, device=device)].to(torch.int32)
    if case["filtered"]:
        _filter(logits, 2.0)
    anc = torch.zeros(b, case["nodes"], case["nodes"], dtype=torch.bool)
    sib = torch.zeros(b, case["nodes"], case["nodes"], dtype=torch.bool)
    for i, t in enumerate(trees):
        for j, p in enumerate(t):
            if p >= 0:
                anc[i, j] = anc[i, p]
                sib[i, j, :j] = torch.tensor(t[:j]) == p
            anc[i, j, j] = True
    return {"case": case, "logits": logits.to(DTYPES[case["dtype"]]), "tokens": tokens, "parents": _i32(parents, device),
            "q_lens": _i32(nodes, device), "q_offsets": _i32([sum(nodes[:i]) for i in range(b + 1)], device),
            "max_q": max(nodes), "u": torch.rand(n, generator=g, device=device), "gumbel": _gumbel((b, vocab), g, device),
            "t": _temperatures(case, g, device), "ancestors": anc.to(device), "siblings": sib.to(device)}


def _commit_lengths(case):
    return _lengths(dict(case, ctx=400, ragged=True))


def _paths(case, trees):
    """An accepted path per tree: node 0, then a child at a time, some stopping early."""
    rng, paths = random.Random(len(trees)), []
    for t in trees:
        path = [0]
        while rng.random() < 0.8:
            kids = [i for i, p in enumerate(t) if p == path[-1]]
            if not kids:
                break
            path.append(rng.choice(kids))
        paths.append(path)
    return paths


def _prepare_commit(case, seed, device):
    g, rng = _generator(seed, device), random.Random(seed)
    hist, nodes, trees = _commit_lengths(case)
    tables, num_blocks = _pages(case, [h + n for h, n in zip(hist, nodes)], rng, device)
    paths = _paths(case, trees)
    width = max(nodes)
    shape = (case["layers"], num_blocks, case["block"], case["kv_heads"], case["head_dim"])
    s = {"case": case, "tables": tables, "start": _i32(hist, device),
         "path": _i32([p + [-1] * (width - len(p)) for p in paths], device),
         "accepted": _i32([len(p) - 1 for p in paths], device)}
    for x in "kv":
        s[x], s[x + "_scale"] = _random_cache(shape, case, g, device)
    return s


def prepare(case, seed):
    device = torch.device("cuda")
    return globals()["_prepare_" + case["kind"]](case, seed, device)


# ---------------------------------------------------------------------------- plain forms
def _dequantised(rows, scales, dtype=torch.float32):
    """e4m3 rows [..., hd] and scale bytes [...] to the values they stand for."""
    if scales is None:
        return rows.to(dtype)
    return torch.ldexp(rows.to(dtype), scales.int()[..., None] - 127)


def _slots(tables, positions, block):
    """Flat slots of positions [batch, n]."""
    return torch.gather(tables.long(), 1, positions // block) * block + positions % block


def _plain_attn(s):
    case = s["case"]
    b, nq, nkv, hd = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
    key = torch.arange(s["max_ctx"], device=s["q"].device)
    inside = key[None] < s["ctx"][:, None]
    at = _slots(s["tables"], torch.where(inside, key[None], 0), case["block"])
    rows = {x: s[x].view(-1, nkv, hd) for x in "kv"}
    scales = {x: None if s[x + "_scale"] is None else s[x + "_scale"].view(-1, nkv)[at] for x in "kv"}
    # float8 rows are indexed as bytes
    k, v = (_dequantised(rows[x].view(torch.uint8)[at].view(torch.float8_e4m3fn) if scales[x] is not None
                         else rows[x][at], scales[x]) for x in "kv")
    q = s["q"][s["padded"]].float().view(b, s["max_q"], nkv, nq // nkv, hd)
    scores = torch.einsum("bqhgd,bkhd->bhgqk", q * s["scale"], k)
    node = key[None] - (s["ctx"] - s["q_lens"])[:, None]  # below 0: history
    row = torch.arange(s["max_q"], device=q.device)
    if s["mask"] is None:
        seen = node[:, None] <= row[None, :, None]
    else:
        words = s["mask"][s["padded"]]  # [batch, max_q, words]
        bit = node.clamp(min=0, max=s["max_q"] - 1)
        word = torch.gather(words, 2, (bit // 32)[:, None].expand(-1, s["max_q"], -1))
        seen = (node < 0)[:, None] | ((word >> (bit % 32).to(torch.int32)[:, None]) & 1).bool()
    seen = (seen & inside[:, None])[:, None, None]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1)
    out = torch.einsum("bhgqk,bkhd->bqhgd", p, v)
    total = total.permute(0, 3, 1, 2)[..., None]
    out = torch.where(total > 0, out / total, 0.0)
    return out.reshape(b * s["max_q"], nq, hd)[s["packed"]].to(s["q"].dtype)


def _rotate(x, cos, sin):
    """Rotate-half rotation of [tokens, heads, head_dim] by [tokens, head_dim / 2] tables."""
    half = x.shape[-1] // 2
    a, b, cos, sin = x[..., :half], x[..., half:], cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _exponent(x):
    """The least e >= -126 with |x| <= 448 * 2^e in every row; 0 for a zero row."""
    top = x.abs().amax(-1)
    f, e = torch.frexp(top)
    e = (e - 9 + (f > 0.875)).clamp(min=-126)
    return torch.where(top == 0, 0, e)


def _plain_cache(s):
    case = s["case"]
    nq, nkv, hd, n = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"]
    qkv = s["qkv"].float().view(n, nq + 2 * nkv, hd)
    pos = s["positions"].long()
    rotated = _rotate(qkv[:, :nq + nkv], s["cos"][pos], s["sin"][pos])
    got = [rotated[:, :nq].to(s["qkv"].dtype)]
    for x, rows in (("k", rotated[:, nq:]), ("v", qkv[:, nq + nkv:])):
        e = _exponent(rows)
        s[x].view(torch.uint8).view(-1, nkv, hd)[s["slots"]] = torch.ldexp(rows, -e[..., None]).to(
            torch.float8_e4m3fn).view(torch.uint8)
        s[x + "_scale"].view(-1, nkv)[s["slots"]] = (e + 127).to(torch.uint8)
        back = s[x].view(torch.uint8).view(-1, nkv, hd)[s["slots"]].view(torch.float8_e4m3fn)
        got.append(_dequantised(back, s[x + "_scale"].view(-1, nkv)[s["slots"]]).to(s["qkv"].dtype))
    return got


def _lowest_argmax(x):
    index = torch.arange(x.shape[-1], device=x.device)
    return torch.where(x == x.amax(-1, keepdim=True), index, x.shape[-1]).amin(-1)


def _probabilities(x, t):
    """softmax(x / t) of rows [..., vocab] in 64 bits (tokens are chosen next to borders); one-hot at the largest where t is 0."""
    greedy = (t == 0)[:, None]
    x = x.double()
    z = x / torch.where(greedy, 1.0, t.double()[:, None])
    z = torch.exp(z - z.amax(-1, keepdim=True))
    index = torch.arange(x.shape[-1], device=x.device)
    hot = (index == _lowest_argmax(x)[:, None]).double()
    return torch.where(greedy, hot, z / z.sum(-1, keepdim=True))


def _final(w, p, gumbel):
    """The token drawn from weights w (from p where none is left) by the given noise."""
    w = torch.where((w > 0).any(-1, keepdim=True), w, p)
    return _lowest_argmax(torch.log(w) + gumbel.double())


def _plain_chain(s):
    b, k, vocab = s["case"]["batch"], s["case"]["k"], s["case"]["vocab"]
    p = _probabilities(s["logits"].view(-1, vocab), s["t"].repeat_interleave(k + 1)).view(b, k + 1, vocab)
    drafts = s["drafts"].long()
    pd = torch.gather(p[:, :k], 2, drafts[..., None])[..., 0]
    if s["draft_logits"] is not None:
        q = _probabilities(s["draft_logits"].view(-1, vocab), s["t"].repeat_interleave(k)).view(b, k, vocab)
    else:
        q = torch.zeros_like(p[:, :k]).scatter_(2, drafts[..., None], 1.0)
    qd = torch.gather(q, 2, drafts[..., None])[..., 0]
    n = (s["u"].double() * qd < pd).long().cumprod(1).sum(1)
    last = torch.gather(p, 1, n[:, None, None].expand(-1, -1, vocab))[:, 0]
    q = torch.cat([q, torch.zeros_like(q[:, :1])], 1)
    rest = torch.gather(q, 1, n[:, None, None].expand(-1, -1, vocab))[:, 0]
    token = _final((last - rest).clamp(min=0), last, s["gumbel"])
    j = torch.arange(k + 1, device=p.device)[None]
    emitted = torch.cat([drafts, drafts[:, :1]], 1)
    emitted = torch.where(j < n[:, None], emitted, torch.where(j == n[:, None], token[:, None], -1))
    logp = torch.log(torch.gather(p, 2, emitted.clamp(min=0)[..., None])[..., 0])
    logp = torch.where(j <= n[:, None], logp, 0.0)
    return n.to(torch.int32), emitted.to(torch.int32), logp.float()


def _plain_tree(s):
    b, vocab = s["case"]["batch"], s["case"]["vocab"]
    n, wide = s["q_lens"].long(), s["max_q"]
    index = torch.arange(wide, device=n.device)
    inside = index[None] < n[:, None]
    at = (s["q_offsets"][:-1, None] + torch.where(inside, index[None], 0)).long()
    p = _probabilities(s["logits"], s["t"].repeat_interleave(s["case"]["nodes"]))
    tokens, parent = s["tokens"].long()[at], s["parents"].long()[at]
    row = (s["q_offsets"][:-1, None] + parent.clamp(min=0)).long()
    pt = p[row, tokens]  # a node's token at its parent
    sib = s["siblings"][:, :wide, :wide]
    again = (sib & (tokens[:, :, None] == tokens[:, None])).any(-1)  # an earlier sibling had the same token
    pt = torch.where(again, 0.0, pt)
    left = 1 - (sib.double() @ pt[..., None])[..., 0]
    yes = (s["u"].double()[at] * left < pt) & (parent >= 0) & inside
    first = yes & ~(sib & yes[:, None]).any(-1) | (parent < 0)
    reached = (first[:, None] | ~s["ancestors"][:, :wide, :wide]).all(-1) & inside
    count = reached.sum(-1) - 1
    path = torch.where(reached, index[None], wide).sort(-1).values
    last = torch.gather(path, 1, count[:, None])[:, 0]
    here = p[(s["q_offsets"][:-1] + last).long()]
    kids = (parent == last[:, None]) & inside & (parent >= 0)
    w = here.clone().scatter_reduce_(1, tokens, torch.where(kids, 0.0, math.inf).double(), "amin")
    token = _final(w, here, s["gumbel"])
    path = torch.where(index[None] <= count[:, None], path, -1)
    nxt = torch.cat([path[:, 1:], path[:, :1]], 1).clamp(min=0)
    emitted = torch.where(index[None] < count[:, None], torch.gather(tokens, 1, nxt), -1)
    emitted = torch.where(index[None] == count[:, None], token[:, None], emitted)
    logp = torch.log(p[at.gather(1, path.clamp(min=0)), emitted.clamp(min=0)])
    logp = torch.where(index[None] <= count[:, None], logp, 0.0)
    return count.to(torch.int32), path.to(torch.int32), emitted.to(torch.int32), logp.float()


def _plain_commit(s):
    case = s["case"]
    j = torch.arange(s["path"].shape[1], device=s["path"].device)[None]
    moved = j <= s["accepted"][:, None]
    to = (s["start"][:, None] + torch.where(moved, j, 0)).long()
    frm = (s["start"][:, None] + torch.where(moved, s["path"], 0)).long()
    to, frm = (_slots(s["tables"], x, case["block"]).view(-1) for x in (to, frm))
    got = []
    for x in ("k", "v", "k_scale", "v_scale"):
        if s[x] is not None:
            bits = s[x].view(torch.uint8) if case["cache"] == "fp8" else s[x]
            flat = bits.view(case["layers"], -1, *bits.shape[3:])
            flat[:, to] = flat[:, frm]
            got.append(s[x])
    return got


# ---------------------------------------------------------------------------- the framework
def _own_run(s):
    from kvengine_b200 import ops

    case = s["case"]
    if case["kind"] != "cache" and "ws" not in s:
        s["ws"] = ops.Workspace(s["t"].device if "t" in s else s["tables"].device)
    if case["kind"] == "attn":
        return ops.tree_attention(s["q"], s["k"], s["v"], s["tables"], s["ctx"], s["q_lens"], s["q_offsets"], s["max_q"],
                                  s["max_ctx"], s["scale"], tree_mask=s["mask"], k_scale=s["k_scale"],
                                  v_scale=s["v_scale"], workspace=s["ws"])
    if case["kind"] == "cache":
        ops.qkv_rope_append_fp8(s["qkv"], s["positions"], s["slots32"], s["cos"], s["sin"], s["q_out"], s["k"], s["v"],
                                s["k_scale"], s["v_scale"], case["heads"], case["kv_heads"], case["head_dim"])
        k, v = ops.kv_read_fp8(s["k"], s["v"], s["k_scale"], s["v_scale"], s["slots"], dtype=s["qkv"].dtype)
        return [s["q_out"], k, v]
    if case["kind"] == "chain":
        return ops.sample_accept(s["logits"], s["drafts"], s["u"], s["gumbel"], s["t"], draft_logits=s["draft_logits"],
                                 workspace=s["ws"])
    if case["kind"] == "tree":
        return ops.tree_sample_accept(s["logits"], s["tokens"], s["parents"], s["q_lens"], s["q_offsets"], s["max_q"],
                                      s["u"], s["gumbel"], s["t"], workspace=s["ws"])
    ops.kv_commit_path(s["k"], s["v"], s["tables"], s["start"], s["path"], s["accepted"], k_scale=s["k_scale"],
                       v_scale=s["v_scale"])
    return [s[x] for x in ("k", "v", "k_scale", "v_scale") if s[x] is not None]


def run(s):
    if own:
        return _own_run(s)
    return globals()["_plain_" + s["case"]["kind"]](s)


# ---------------------------------------------------------------------------- exact values
def _value(byte, scale):
    """The real number of e4m3 bytes with scale bytes, from the format's definition."""
    byte = byte.to(torch.int64)
    e, m = byte >> 3 & 15, (byte & 7).double()
    size = torch.where(e == 0, m * 2.0 ** -9, torch.ldexp(8 + m, e - 10))
    return torch.ldexp(torch.where(byte >= 128, -size, size), scale.int()[..., None] - 127)


def _exact_attn(s):
    case, out = s["case"], torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    nkv, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    for b, (ctx, n, off) in enumerate(zip(s["ctx"].tolist(), s["q_lens"].tolist(), s["q_offsets"].tolist())):
        blocks = s["tables"][b, :-(-ctx // case["block"])].long()
        if case["cache"] == "fp8":
            k, v = (_value(s[x].view(torch.uint8)[blocks], s[x + "_scale"][blocks]) for x in "kv")
        else:
            k, v = s["k"][blocks].double(), s["v"][blocks].double()
        k, v = (x.flatten(0, 1)[:ctx].transpose(0, 1) for x in (k, v))  # [kv heads, ctx, head_dim]
        seen = torch.ones(n, ctx, dtype=torch.bool, device=out.device)
        if s["mask"] is None:
            seen[:, ctx - n:] = torch.ones(n, n, device=out.device).tril().bool()
        else:
            words = s["mask"][off:off + n].long() & 0xFFFFFFFF
            for t in range(n):
                seen[:, ctx - n + t] = (words[:, t // 32] >> t % 32 & 1).bool()
        for h in range(nkv):
            q = s["q"][off:off + n, h * group:(h + 1) * group].double()
            w = (q.reshape(n * group, -1) @ k[h].T) * s["scale"]
            w = w.masked_fill(~seen.repeat_interleave(group, 0), -math.inf).softmax(-1).nan_to_num(0.0)
            out[off:off + n, h * group:(h + 1) * group] = (w @ v[h]).view(n, group, -1)
    return out


def _nearest_e4m3(x):
    """x (at most 448 in size) to the nearest e4m3 number, ties to the even one, by arithmetic."""
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x.abs().clamp(min=2.0 ** -6)).exponent - 4)
    return torch.round(x / step) * step


def _exact_cache(s):
    case = s["case"]
    nq, nkv, hd, n = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"]
    x = s["qkv"].double().view(n, nq + 2 * nkv, 2, hd // 2)
    c, i = (s[t].double()[s["positions"].long()][:, None] for t in ("cos", "sin"))
    turned = torch.complex(x[..., 0, :], x[..., 1, :]) * torch.complex(c, i)
    turned = torch.stack([turned.real, turned.imag], 2).reshape(n, nq + 2 * nkv, hd)
    got = [turned[:, :nq]]
    for rows in (turned[:, nq:nq + nkv], s["qkv"].double().view(n, -1, hd)[:, nq + nkv:]):
        part, power = torch.frexp(rows.abs().amax(-1, keepdim=True) / 448)
        unit = torch.ldexp(torch.ones_like(part), (power - (part == 0.5).int()).clamp(min=-126))
        got.append(_nearest_e4m3(rows / unit) * unit)
    return got


def _row(x, t):
    """Probabilities of one row of logits at temperature t, in 64 bits."""
    if t > 0:
        return (x.double() / t).softmax(-1)
    p = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    p[(x == x.max()).nonzero()[0, 0]] = 1
    return p


def _exact_chain(s):
    """Draft by draft, as the method is usually told."""
    b, k = s["drafts"].shape
    drafts, u, gumbel = s["drafts"].tolist(), s["u"].tolist(), s["gumbel"].double()
    counts, tokens, logps = [], [], []
    for i, t in enumerate(s["t"].tolist()):
        tok, logp = [], []
        for j in range(k + 1):
            p = _row(s["logits"][i, j], t)
            if j == k:
                w = p
                break
            d = drafts[i][j]
            q = torch.zeros_like(p)
            if s["draft_logits"] is None:
                q[d] = 1
            else:
                q = _row(s["draft_logits"][i, j], t)
            if u[i][j] >= float(p[d] / q[d]):
                w = torch.relu(p - q)
                break
            tok.append(d)
            logp.append(math.log(p[d]))
        w = w if float(w.max()) > 0 else p
        last = int((w.log() + gumbel[i]).argmax())
        counts.append(len(tok))
        tokens.append(tok + [last] + [-1] * (k - len(tok)))
        logps.append(logp + [math.log(p[last])] + [0.0] * (k - len(logp)))
    return torch.tensor(counts), torch.tensor(tokens), torch.tensor(logps, dtype=torch.float64)


def _exact_tree(s):
    u, tokens, parents = s["u"].tolist(), s["tokens"].tolist(), s["parents"].tolist()
    wide, got = s["max_q"], ([], [], [], [])
    for i, (t, off, n) in enumerate(zip(s["t"].tolist(), s["q_offsets"].tolist(), s["q_lens"].tolist())):
        path, tok, logp = [0], [], []
        while True:
            p = _row(s["logits"][off + path[-1]], t)
            w = p.clone()
            for c in (c for c in range(n) if parents[off + c] == path[-1]):
                d = tokens[off + c]
                if u[off + c] * (1 - float((p - w).sum())) < float(w[d]):
                    path.append(c)
                    tok.append(d)
                    logp.append(math.log(p[d]))
                    break
                w[d] = 0
            else:
                break
        w = w if float(w.max()) > 0 else p
        tok.append(int((w.log() + s["gumbel"][i].double()).argmax()))
        logp.append(math.log(p[tok[-1]]))
        for x, row, pad in zip(got[1:], (path, tok, logp), (-1, -1, 0.0)):
            x.append(row + [pad] * (wide - len(row)))
        got[0].append(len(path) - 1)
    return tuple(torch.tensor(x, dtype=torch.float64 if x is got[3] else torch.int64) for x in got)


def exact(case, seed):
    if case["kind"] == "commit":
        return None  # copies: nothing is computed
    return globals()["_exact_" + case["kind"]](prepare(case, seed))
