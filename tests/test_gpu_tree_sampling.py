"""Sampling, draft trees and the 8-bit cache on the GPU, against plain 64-bit implementations.

Tolerances count roundings, per output element. A rounding is off by at most half a step: bf16 numbers
in [1, 2) are 2^-7 apart, so u16 = 2^-8 of the value at the binade's lower end (and not 2^-9, which holds
at its upper end only); fp32's are 2^-23 apart: u32 = 2^-24.

attention, with p the exact weights, A = sum_j p_j |v_j| and s = scale * sum_d |q_d| |k_d| (its largest
over the row's keys):
  * a score is a sum of head_dim products in fp32: off by at most d = (head_dim + 4) u32 s, plus
    2^-21 for the scaling, the running base and the exponential (ex2.approx: 2^-22); a
    change of d in the scores changes a weight's share by at most 2 d, so the output by 2 (d + 2^-21) A;
  * bf16 rounds p (u16 A) and the output (u16 |o|); fp32 splits p and v to 2^-22 each (2^-21 A, the
    same again for q and k: 2^-21 s in d) and rounds the output (u32 |o|);
  * sums of up to n terms in fp32: n u32 A, n < 2^12 here, in chains far shorter: 2^-14 A is generous for
    bf16 (a sixty-fourth of u16 A; where more than eight rows share a kv head, a quarter of the
    exponentials come from a polynomial off by 2.6e-6 of the value, 2^-18, well inside it); fp32
    sums its n terms in order within a stream: n u32 A.
log-probabilities: (x - m) / T - log z with z from ex2.approx (2^-22 relative, arguments in fp32 off by
2 u32 |x - m| / T) and sums of a few dozen fp32 additions (64 u32): in absolute terms
2^-22 + 2 u32 R + 64 u32, R the range of (x - m) / T that carries weight (below 40), then one rounding.
"""

import math
import random

import pytest
import torch

from kvengine_b200 import PagedKVCache, ops
from kvengine_b200 import _lib as L

pytestmark = pytest.mark.gpu
U16, U32 = torch.finfo(torch.bfloat16).eps / 2, torch.finfo(torch.float32).eps / 2
E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------- attention
def cache_of(case, num_blocks, bs, nkv, hd, g, dev):
    shape = (num_blocks, bs, nkv, hd)
    if case == "fp8":
        mk = lambda: (torch.randn(shape, generator=g) * 90).clamp(-448, 448).to(E4M3)  # noqa: E731
        sc = lambda: torch.randint(117, 124, shape[:-1], generator=g).to(torch.uint8)  # noqa: E731
        return [x.to(dev) for x in (mk(), mk(), sc(), sc())]
    dt = torch.float32 if case == "fp32" else torch.bfloat16
    return [torch.randn(shape, generator=g).to(dt).to(dev) for _ in range(2)] + [None, None]


def values(pool, scale):
    x = pool.double()
    return x if scale is None else x * torch.pow(2.0, scale.double() - 127)[..., None]


def reference(q, k, v, ks, vs, tables, ctx, ql, off, mask, scale):
    """Exact outputs, and per element the bound on |got - exact| as the module's text derives it."""
    kd, vd = values(k.cpu(), None if ks is None else ks.cpu()), values(v.cpu(), None if vs is None else vs.cpu())
    bs, nkv, hd = k.shape[1:]
    q64 = q.cpu().double()
    out, tol = torch.zeros_like(q64), torch.zeros_like(q64)
    group = q.shape[1] // nkv
    for b, (c, n, o) in enumerate(zip(ctx, ql, off)):
        pos = torch.arange(c)
        t = tables[b].cpu().long()
        keys, vals = kd[t[pos // bs], pos % bs], vd[t[pos // bs], pos % bs]  # [c, nkv, hd]
        for i in range(n):
            seen = torch.zeros(c, dtype=torch.bool)
            seen[:c - n] = True
            for j in range(n):
                seen[c - n + j] = j <= i if mask is None else bool(int(mask[o + i, j // 32]) >> j % 32 & 1)
            if not bool(seen.any()):
                continue
            for h in range(q.shape[1]):
                kk, vv = keys[seen, h // group], vals[seen, h // group]
                p = (kk @ q64[o + i, h] * scale).softmax(0)
                r = p @ vv
                a = p @ vv.abs()
                s = float((kk.abs() @ q64[o + i, h].abs()).max()) * scale
                d = (hd + 4) * U32 * s + 2.0 ** -21
                if q.dtype == torch.float32:
                    e = 2 * (d + 2.0 ** -21 * s) * a + (2.0 ** -21 + int(seen.sum()) * U32) * a + U32 * r.abs()
                else:
                    e = 2 * d * a + (U16 + 2.0 ** -14) * a + U16 * r.abs()
                out[o + i, h], tol[o + i, h] = r, e * 1.01 + 1e-30
    return out, tol


def attention_case(cache, heads, nodes, hists, bs, kind, seed, dev, scale=None):
    """(arguments of ops.tree_attention, lengths) of shuffled pages and random trees."""
    nq, nkv, hd = heads
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    ctx = [h + n for h, n in zip(hists, nodes)]
    need = [-(-c // bs) for c in ctx]
    ids = list(range(sum(need) + 2))
    rng.shuffle(ids)
    width = max(max(need), 1)
    table = torch.zeros(len(ctx), width, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    off = [sum(nodes[:b]) for b in range(len(nodes) + 1)]
    k, v, ks, vs = cache_of(cache, sum(need) + 2, bs, nkv, hd, g, dev)
    q = torch.randn(off[-1], nq, hd, generator=g).to(torch.float32 if cache == "fp32" else torch.bfloat16).to(dev)
    trees = [[-1] + [rng.randint(0, i - 1) for i in range(1, n)] if n else [] for n in nodes]
    if kind == "tree":
        mask = ops.tree_mask_words(trees, max(nodes))
    elif kind == "random":  # any bits, those past a tree's nodes and past max_q_len too; some rows without one
        mask = torch.randint(-2 ** 31, 2 ** 31, (off[-1], -(-max(nodes) // 32) + 1), generator=g, dtype=torch.int64).int()
        mask[::3] = 0
    else:
        mask = None
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    args = dict(q=q, pool_k_layer=k, pool_v_layer=v, block_tables=table.to(dev), ctx_lens=i32(ctx), q_lens=i32(nodes),
                q_offsets=i32(off), max_q_len=max(nodes), max_ctx=max(ctx), scale=scale or hd ** -0.5,
                tree_mask=None if mask is None else mask.to(dev), k_scale=ks, v_scale=vs)
    return args, ctx, nodes, off


def check_attention(args, ctx, nodes, off, got):
    want, tol = reference(args["q"], args["pool_k_layer"], args["pool_v_layer"], args["k_scale"], args["v_scale"],
                          args["block_tables"], ctx, nodes, off, None if args["tree_mask"] is None else args["tree_mask"].cpu(),
                          args["scale"])
    err = (got.cpu().double() - want).abs()
    assert got.dtype == args["q"].dtype and torch.isfinite(got.float()).all()
    bad = err > tol
    assert not bool(bad.any()), (int(bad.sum()), float((err / tol).max()))


HEADS = [(14, 2, 64), (16, 2, 128), (4, 4, 64), (2, 1, 128), (48, 1, 64)]


@pytest.mark.parametrize("cache", ["bf16", "fp32", "fp8"])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("nodes, hists, bs, kind", [
    ([1], [0], 16, "none"),                                   # one token, no history
    ([1, 1, 1], [1, 15, 16], 16, "none"),                     # pages that end at, before and behind a tile
    ([5, 1, 9, 2], [40, 0, 300, 129], 16, "tree"),
    ([13, 33], [7, 150], 7, "tree"),                          # odd pages, masks of two words
    ([3, 0, 6], [20, 5, 0], 1, "random"),                     # a sequence without new tokens, rows without keys
    ([40, 8], [0, 61], 64, "random"),
    ([4, 17], [90, 31], 32, "none"),                          # chains
])
def test_tree_attention(cuda_device, cache, heads, nodes, hists, bs, kind):
    args, *lens = attention_case(cache, heads, nodes, hists, bs, kind, 11, cuda_device)
    status = ops.status_tensor(cuda_device)
    check_attention(args, *lens, ops.tree_attention(**args, status=status))
    assert int(status) == 0


@pytest.mark.parametrize("cache", ["bf16", "fp32", "fp8"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (16, 2, 128)])
@pytest.mark.parametrize("nodes, hists, bs", [([1], [2300], 16), ([7], [1800], 16), ([2, 5], [1000, 3000], 5)])
def test_tree_attention_long_histories_are_split_and_joined(cuda_device, cache, heads, nodes, hists, bs):
    args, *lens = attention_case(cache, heads, nodes, hists, bs, "tree", 5, cuda_device)
    ws = ops.Workspace(cuda_device)
    got = ops.tree_attention(**args, workspace=ws)
    check_attention(args, *lens, got)
    assert ws.buf.numel() > 65536 and int(ws.buf[:65536].view(torch.int32).abs().sum()) == 0  # counters left at zero
    assert torch.equal(ops.tree_attention(**args, workspace=ws), got)


@pytest.mark.parametrize("cache, heads", [("bf16", (14, 2, 64)), ("bf16", (16, 2, 128)), ("bf16", (3, 3, 64)),
                                          ("bf16", (64, 1, 128)), ("fp8", (14, 2, 64)), ("fp8", (16, 2, 128)),
                                          ("fp8", (3, 3, 64))])
@pytest.mark.parametrize("nodes, hists, bs, kind", [
    ([45], [0], 16, "tree"),                     # the tree alone
    ([50, 64, 7], [300, 129, 128], 16, "tree"),  # histories around a key tile's end
    ([130, 1, 40], [33, 700, 0], 32, "random"),  # rows without keys, masks of five words
    ([64, 64], [63, 1000], 48, "none"),          # chains
    ([33, 0, 35], [2500, 5, 90], 16, "tree"),    # split into chunks, a sequence without new tokens
])
def test_tree_attention_many_rows(cuda_device, cache, heads, nodes, hists, bs, kind):
    """Trees of more rows than one tensor-core tile, in every arrangement of tiles and chunks."""
    args, *lens = attention_case(cache, heads, nodes, hists, bs, kind, 17, cuda_device)
    status = ops.status_tensor(cuda_device)
    ws = ops.Workspace(cuda_device)
    got = ops.tree_attention(**args, workspace=ws, status=status)
    check_attention(args, *lens, got)
    assert int(status) == 0 and int(ws.buf[:65536].view(torch.int32).abs().sum()) == 0
    assert torch.equal(ops.tree_attention(**args, workspace=ws), got)
    check_attention(dict(args, scale=-0.05), *lens, ops.tree_attention(**dict(args, scale=-0.05)))


@pytest.mark.parametrize("heads, nodes", [((8, 4, 64), 8), ((16, 4, 128), 40)])
@pytest.mark.parametrize("cache", ["bf16", "fp8"])
def test_tree_attention_long_chunks(cuda_device, cache, heads, nodes):
    """More sequences than the grid needs: a block's keys go round its ring several times."""
    hists = [1400 + 13 * i % 200 for i in range(40)]
    args, *lens = attention_case(cache, heads, [nodes] * 40, hists, 16, "tree", 29, cuda_device)
    status = ops.status_tensor(cuda_device)
    check_attention(args, *lens, ops.tree_attention(**args, status=status))
    assert int(status) == 0


@pytest.mark.parametrize("bs", [16, 7])
@pytest.mark.parametrize("exponent", [30, 127, 134, 135, 150])
@pytest.mark.parametrize("group", [1, 16])
def test_tree_attention_over_one_8_bit_key_is_its_value(cuda_device, group, exponent, bs):
    """One key: p = 1, and every finite e4m3 times 2^(exponent - 127) is a bf16: the output is V exactly, NaN bytes NaN."""
    pool_k = torch.zeros(4, bs, 2, 128, dtype=torch.uint8, device=cuda_device)
    pool_v = (torch.arange(4 * bs * 2 * 128, device=cuda_device) * 37 % 256).to(torch.uint8).view(4, bs, 2, 128)
    scale = torch.full((4, bs, 2), exponent, dtype=torch.uint8, device=cuda_device)
    for history in (False, True):  # the key is the new token, or of the history (and the new token unseen)
        ctx = 2 if history else 1
        mask = torch.ones(2, 1, dtype=torch.int32, device=cuda_device) * (0 if history else 1)
        if history:
            pool_v[2, 1] = 0
        out = ops.tree_attention(
            torch.ones(1, 2 * group, 128, dtype=torch.bfloat16, device=cuda_device), pool_k.view(torch.float8_e4m3fn),
            pool_v.view(torch.float8_e4m3fn), torch.tensor([[2]], dtype=torch.int32, device=cuda_device),
            *[torch.tensor([x], dtype=torch.int32, device=cuda_device) for x in (ctx, 1, 0)], 1, ctx, 0.1,
            tree_mask=mask[:1], k_scale=scale, v_scale=scale)
        want = pool_v[2, 0].view(torch.float8_e4m3fn).float() * 2.0 ** (exponent - 127)
        assert bool(want.isnan().any())
        got = out.float().view(2, group, 128)
        assert torch.equal(got.nan_to_num(7e30), want.nan_to_num(7e30)[:, None].expand(2, group, 128)), (group, exponent, history)


def test_tree_attention_joins_with_extreme_scores(cuda_device):
    """Scores hundreds apart between chunks and streams: shares of exactly 0 and 1, no overflow."""
    for cache in ("bf16", "fp32", "fp8"):
        args, *lens = attention_case(cache, (4, 2, 64), [3], [1500], 16, "tree", 8, cuda_device, scale=20.0)
        check_attention(args, *lens, ops.tree_attention(**args))


def test_tree_attention_same_rows_as_paged_attention_on_chains(cuda_device):
    """Without a mask it is the verify attention: the two kernels agree within both bounds."""
    args, ctx, nodes, off = attention_case("bf16", (16, 2, 128), [5, 5, 5], [100, 640, 33], 16, "none", 2, cuda_device)
    a = ops.tree_attention(**args)
    b = ops.paged_attention(*[args[x] for x in ("q", "pool_k_layer", "pool_v_layer", "block_tables", "ctx_lens", "q_lens",
                                                "q_offsets", "max_q_len", "max_ctx", "scale")])
    _, tol = reference(args["q"], args["pool_k_layer"], args["pool_v_layer"], None, None, args["block_tables"], ctx, nodes,
                       off, None, args["scale"])
    assert bool(((a.double() - b.double()).abs().cpu() <= 2 * tol).all())


@pytest.mark.parametrize("heads", [(2, 1, 128), (4, 4, 64), (8, 2, 64), (16, 2, 128)])
@pytest.mark.parametrize("nodes, hists, bs, kind", [
    ([1], [0], 16, "none"), ([1] * 5, [1, 15, 16, 31, 700], 16, "none"), ([2, 1, 2, 0, 1], [40, 0, 2100, 9, 32], 32, "tree"),
    ([2, 2, 1], [14, 300, 95], 16, "random"), ([2, 1], [5000, 60], 48, "none")])
@pytest.mark.parametrize("cache", ["bf16", "fp8"])
def test_tree_attention_few_rows(cuda_device, cache, heads, nodes, hists, bs, kind):
    """Single tokens and pairs: at most eight rows per kv head (sixteen in the last layout)."""
    args, *lens = attention_case(cache, heads, nodes, hists, bs, kind, 23, cuda_device)
    status = ops.status_tensor(cuda_device)
    ws = ops.Workspace(cuda_device)
    got = ops.tree_attention(**args, workspace=ws, status=status)
    check_attention(args, *lens, got)
    assert int(status) == 0 and int(ws.buf[:65536 if ws.buf.numel() > 65536 else 0].sum()) == 0
    assert torch.equal(ops.tree_attention(**args, workspace=ws), got)


def test_tree_attention_few_rows_bad_block(cuda_device):
    """A block id outside the pool reads as zeros, its exponents too."""
    for cache in ("bf16", "fp8"):
        args, ctx, nodes, off = attention_case(cache, (8, 2, 64), [1, 1], [40, 70], 16, "none", 3, cuda_device)
        want = ops.tree_attention(**args)
        tables = args["block_tables"].clone()
        tables[1, 1] = -1
        status = ops.status_tensor(cuda_device)
        got = ops.tree_attention(**dict(args, block_tables=tables), status=status)
        assert int(status) == -7 and torch.equal(got[0], want[0]) and torch.isfinite(got.float()).all()
        zero = dict(args)
        for x in ("pool_k_layer", "pool_v_layer"):
            zero[x] = args[x].clone()
            zero[x].view(torch.uint8)[args["block_tables"][1, 1].long()] = 0
        check_attention(zero, ctx, nodes, off, got)


@pytest.mark.parametrize("heads", [(4, 2, 64), (4, 4, 64), (2, 2, 128), (16, 2, 128)])
@pytest.mark.parametrize("cache", ["bf16", "fp32", "fp8"])
def test_tree_attention_garbage_in_unseen_places(cuda_device, cache, heads):
    """Infinities and NaN in unused slots, in a partial page's tail and in nodes a row does not see
    reach no row that does not see them; a row that sees a NaN gets one."""
    args, ctx, nodes, off = attention_case(cache, heads, [6, 4], [35, 3], 16, "tree", 21, cuda_device)
    clean = ops.tree_attention(**args)
    mask = ops.tree_mask_words([[-1, 0, 0, 1, 2, 2], [-1, -1, 0, 0]], 6)
    args["tree_mask"] = mask.to(cuda_device)
    want = ops.tree_attention(**args)
    check_attention(args, ctx, nodes, off, want)
    used = torch.zeros(args["pool_k_layer"].shape[:2], dtype=torch.bool)
    for b, c in enumerate(ctx):
        for p in range(c):
            used[args["block_tables"][b, p // 16], p % 16] = True
    for x, s in (("pool_k_layer", "k_scale"), ("pool_v_layer", "v_scale")):
        if cache == "fp8":
            args[x].view(torch.uint8)[~used] = 0x7f
            args[s][~used] = 255
        else:
            args[x][~used] = float("nan")
    assert torch.equal(ops.tree_attention(**args), want)
    # node 2 of sequence 0 (seen by itself, 4 and 5) and node 1 of sequence 1 (by itself alone)
    for b, node in ((0, 2), (1, 1)):
        p = ctx[b] - nodes[b] + node
        at = (int(args["block_tables"][b, p // 16]), p % 16)
        if cache == "fp8":
            args["pool_v_layer"].view(torch.uint8)[at] = 0x7f
            args["pool_k_layer"].view(torch.uint8)[at] = 0xff
        else:
            args["pool_v_layer"][at] = float("inf")
            args["pool_k_layer"][at] = float("nan")
    got = ops.tree_attention(**args)
    touched = [2, 4, 5, 6 + 1]
    rest = [i for i in range(10) if i not in touched]
    assert bool(torch.isnan(got[touched]).all())
    # rows of the same tile are summed in another order and, in bf16, with p unrounded
    _, tol = reference(args["q"], *[torch.nan_to_num(args[x].float(), 0.0, 0.0, 0.0) for x in ("pool_k_layer", "pool_v_layer")],
                       args["k_scale"], args["v_scale"], args["block_tables"], ctx, nodes, off, mask, args["scale"])
    assert bool(((got - want).double().abs().cpu()[rest] <= 2 * tol[rest]).all())
    assert torch.isfinite(clean.float()).all()


@pytest.mark.parametrize("cache", ["bf16", "fp8"])
def test_tree_attention_value_seen_with_an_infinity(cuda_device, cache):
    """A node whose V holds one infinity: rows that see it are infinite there and right elsewhere."""
    if cache == "fp8":
        pytest.skip("e4m3 has no infinity")
    args, ctx, nodes, off = attention_case(cache, (2, 1, 64), [3], [20], 16, "tree", 4, cuda_device)
    args["tree_mask"] = ops.tree_mask_words([[-1, 0, 0]]).to(cuda_device)
    p = ctx[0] - 1
    at = (int(args["block_tables"][0, p // 16]), p % 16, 0, 10)
    args["pool_v_layer"][at] = 0
    want, tol = reference(args["q"], args["pool_k_layer"], args["pool_v_layer"], None, None, args["block_tables"], ctx, nodes,
                          off, args["tree_mask"].cpu(), args["scale"])
    args["pool_v_layer"][at] = float("inf")
    got = ops.tree_attention(**args).cpu().double()
    assert bool((got[2, :, 10] == math.inf).all())
    got[2, :, 10] = want[2, :, 10]
    assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("nodes", [1, 9, 40])
@pytest.mark.parametrize("cache", ["bf16", "fp32", "fp8"])
def test_tree_attention_nan_and_infinite_scores_in_the_history(cuda_device, cache, nodes):
    """Every row sees the history: a NaN there, or an infinite score, makes its kv head's rows NaN, whichever key
    of a tile it is, and no other's."""
    args, *_ = attention_case(cache, (8, 2, 64), [nodes], [330], 16, "tree", 37, cuda_device)
    want = ops.tree_attention(**args)[:nodes]
    bits = {"bf16": torch.int16, "fp32": torch.int32, "fp8": torch.uint8}[cache]
    nan = torch.tensor(math.nan).to(args["pool_k_layer"].dtype).view(bits).to(cuda_device)
    table = args["block_tables"][0].tolist()
    for which in ("pool_k_layer", "pool_v_layer"):
        for pos in list(range(8)) + [62, 63, 64, 127, 190, 319]:
            pool = args[which].view(bits).clone()
            pool[table[pos // 16], pos % 16, 0, :] = nan
            got = ops.tree_attention(**dict(args, **{which: pool.view(args[which].dtype)}))[:nodes]
            assert bool(got[:, :4].isnan().all()), (which, pos)
            assert torch.equal(got[:, 4:], want[:, 4:]), (which, pos)
    if cache == "bf16":  # q.k overflows fp32 for one key
        for pos in (6, 7, 70, 200):
            pool = args["pool_k_layer"].clone()
            pool[table[pos // 16], pos % 16, 0, :] = 3e38 * args["q"][0, 0].sign()
            got = ops.tree_attention(**dict(args, q=args["q"][:1].expand(nodes, -1, -1)[:, :1].expand(-1, 8, -1).contiguous(),
                                            tree_mask=args["tree_mask"][:nodes], pool_k_layer=pool))
            assert bool(got[:, :4].isnan().all()) and bool(got[:, 4:].isfinite().all()), pos


@pytest.mark.parametrize("nodes", [1, 9, 40])
@pytest.mark.parametrize("cache", ["bf16", "fp32", "fp8"])
def test_tree_attention_with_scale_zero_is_the_mean(cuda_device, cache, nodes):
    args, *lens = attention_case(cache, (8, 2, 64), [nodes, nodes], [100, 0], 16, "random", 41, cuda_device)
    args["scale"] = 0.0
    check_attention(args, *lens, ops.tree_attention(**args))


def test_tree_attention_leaves_other_rows_and_reports_bad_inputs(cuda_device):
    dev = cuda_device
    args, ctx, nodes, off = attention_case("bf16", (4, 2, 64), [3, 2, 4], [30, 17, 9], 16, "tree", 9, dev)
    q = torch.cat([args["q"], args["q"][:5]])
    args["q"] = q
    args["tree_mask"] = torch.cat([args["tree_mask"], args["tree_mask"][:5]])
    out = torch.full_like(q, 7.0)
    want = ops.tree_attention(**args, out=out).clone()
    assert bool((out[9:] == 7).all())
    # lengths that do not fit: that sequence is skipped, the others are right
    for change in (dict(ctx_lens=[ctx[0], 1, ctx[2]]), dict(q_lens=[3, 5, 4]), dict(q_lens=[3, -1, 4]),
                   dict(ctx_lens=[ctx[0], 16 * args["block_tables"].shape[1] + 1, ctx[2]])):
        name, vals = next(iter(change.items()))
        status = ops.status_tensor(dev)
        out = torch.full_like(q, 7.0)
        ops.tree_attention(**dict(args, **{name: torch.tensor(vals, dtype=torch.int32, device=dev)}), out=out, status=status)
        assert int(status) == -7, change
        assert bool((out[3:5] == 7).all()) and torch.equal(out[:3], want[:3]) and torch.equal(out[5:9], want[5:9])
    # a block id outside the pool reads as zeros
    status = ops.status_tensor(dev)
    tables = args["block_tables"].clone()
    tables[2, 0] = 1 << 20
    got = ops.tree_attention(**dict(args, block_tables=tables), status=status)
    assert int(status) == -7 and torch.equal(got[:5], want[:5]) and torch.isfinite(got[:9].float()).all()


@pytest.mark.parametrize("cache, heads, nodes", [("bf16", (4, 2, 64), [2, 2, 1]), ("fp8", (4, 2, 64), [2, 2, 1]),
                                                 ("bf16", (8, 2, 128), [9, 9, 4]), ("fp8", (8, 2, 128), [9, 9, 4]),
                                                 ("fp32", (4, 2, 64), [5, 5, 3])])
def test_tree_attention_rows_past_the_end_are_refused(cuda_device, cache, heads, nodes):
    """An offset that would put a sequence's rows past q's: skipped and reported; the others are right."""
    args, *_ = attention_case(cache, heads, nodes, [50, 20, 90], 16, "tree", 31, cuda_device)
    rows = sum(nodes)
    for key, short in (("q", rows), ("tree_mask", rows)):
        args[key] = args[key][:short].contiguous()
    want = ops.tree_attention(**args)
    for bad in (rows - nodes[1] + 1, rows, 2 ** 31 - 1, -1):
        status = ops.status_tensor(cuda_device)
        off = args["q_offsets"].clone()
        off[1] = bad
        out = torch.full_like(want, 7.0)
        ops.tree_attention(**dict(args, q_offsets=off), out=out, status=status)
        assert int(status) == -7, bad
        a, b = nodes[0], nodes[0] + nodes[1]
        assert torch.equal(out[:a], want[:a]) and torch.equal(out[b:], want[b:]) and bool((out[a:b] == 7).all()), bad


def test_tree_attention_far_offsets(cuda_device):
    """Blocks past 2^31 elements and 2^32 bytes of the layer."""
    dev = cuda_device
    for cache, dt in (("bf16", torch.bfloat16), ("fp8", torch.uint8)):
        blocks = (5 << 30) // (16 * 8 * 128)
        args, ctx, nodes, off = attention_case(cache, (8, 8, 128), [3], [40], 16, "tree", 3, dev)
        far = torch.tensor([[blocks - 1, blocks - 3, blocks - 2]], dtype=torch.int32, device=dev)
        big = dict(args, block_tables=far)
        for x in ("pool_k_layer", "pool_v_layer"):
            pool = torch.empty(blocks, 16, 8, 128, dtype=dt, device=dev).view(args[x].dtype)
            pool.view(dt)[far[0].long()] = args[x].view(dt)[args["block_tables"][0].long()]
            big[x] = pool
        if cache == "fp8":
            for x in ("k_scale", "v_scale"):
                s = torch.empty(blocks, 16, 8, dtype=torch.uint8, device=dev)
                s[far[0].long()] = args[x][args["block_tables"][0].long()]
                big[x] = s
        assert torch.equal(ops.tree_attention(**big), ops.tree_attention(**args))
        del big, pool


def test_tree_attention_in_graphs_and_on_other_streams(cuda_device):
    """Two captured graphs that share a workspace, replayed in turn with new inputs, on a side stream."""
    dev = cuda_device
    a, *la = attention_case("bf16", (14, 2, 64), [4, 4], [900, 40], 16, "tree", 1, dev)
    b, *lb = attention_case("fp8", (16, 2, 128), [1], [2500], 16, "none", 2, dev)
    ws = ops.Workspace(dev)
    ws.get(8 << 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs, graphs = [], []
    with torch.cuda.stream(side):
        for args in (a, b):
            ops.tree_attention(**args, workspace=ws)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(ops.tree_attention(**args, workspace=ws))
            graphs.append(graph)
        a["q"].copy_(a["q"].flip(0))
        for _ in range(3):
            for graph in graphs:
                graph.replay()
    side.synchronize()
    check_attention(a, *la, outs[0])
    check_attention(b, *lb, outs[1])


def test_tree_attention_wrapper_refusals(cuda_device):
    args, *_ = attention_case("bf16", (4, 2, 64), [3], [30], 16, "tree", 9, cuda_device)
    for change in (dict(q=args["q"].transpose(0, 1)), dict(q=args["q"].half()), dict(tree_mask=args["tree_mask"].long()),
                   dict(tree_mask=args["tree_mask"][:2]), dict(ctx_lens=args["ctx_lens"].cpu()),
                   dict(k_scale=torch.zeros(1, dtype=torch.uint8, device=cuda_device)),
                   dict(pool_v_layer=args["pool_v_layer"][:1]), dict(block_tables=args["block_tables"][0]),
                   dict(out=torch.empty_like(args["q"]).float()), dict(q=args["q"].float())):
        with pytest.raises((ValueError, TypeError)):
            ops.tree_attention(**dict(args, **change))


# ---------------------------------------------------------------- the 8-bit cache
def quantised(x):
    """(values, e + 127) of rows x [..., hd] (float64) by the definition, element by element."""
    fin = torch.where(torch.isfinite(x), x, 0.0)
    top = fin.abs().amax(-1)
    f, e = torch.frexp(top / 448)
    e = torch.where(top == 0, 0, (e - (f == 0.5).int()).clamp(min=-126))
    y = torch.ldexp(fin, -e[..., None])
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 4)
    y = torch.ldexp(torch.round(y / step) * step, e[..., None])
    return torch.where(torch.isfinite(x), y, math.nan), (e + 127).to(torch.uint8)


def hard_rows(n, nkv, hd, dt, g):
    x = torch.randn(n, nkv, hd, generator=g) * torch.exp(torch.randn(n, nkv, 1, generator=g) * 3)
    x[0] = 0
    x[1, 0, 3], x[1, 0, 7] = math.inf, math.nan
    x[2, 0] = math.nan
    x[3, 0] *= 2.0 ** -120        # rows whose scale ends at 2^-126
    x[4, 0] = 0
    x[4, 0, 5] = 2.0 ** -133      # the least bf16
    x[5, 0, 0] = 448 * 2.0 ** 6 * torch.sign(x[5, 0, 0]); x[5, 0, 1:] = x[5, 0, 1:].clamp(-448, 448)  # noqa: E702
    x[6, 0] *= 2.0 ** 120
    x[7, 0] = torch.arange(hd) - hd / 2.0  # ties
    return x.to(dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nkv, hd, bs", [(2, 64, 16), (2, 128, 16), (1, 64, 5), (8, 128, 3)])
@pytest.mark.parametrize("n", [8, 67])
def test_kv_append_and_read_fp8(cuda_device, dt, nkv, hd, bs, n):
    g = torch.Generator().manual_seed(n + hd)
    k, v = hard_rows(n, nkv, hd, dt, g), hard_rows(n, nkv, hd, dt, g).flip(0)
    blocks = n // bs + 3
    slots = torch.randperm(blocks * bs, generator=g)[:n]
    pools = [torch.full((blocks, bs, nkv, hd), 0x35, dtype=torch.uint8, device=cuda_device).view(E4M3) for _ in range(2)]
    scales = [torch.full((blocks, bs, nkv), 9, dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    status = ops.status_tensor(cuda_device)
    ops.kv_append_fp8(k.to(cuda_device), v.to(cuda_device), slots.to(cuda_device), *pools, *scales, status=status)
    for odt in (torch.float32, torch.bfloat16):
        back = ops.kv_read_fp8(*pools, *scales, slots.to(cuda_device), dtype=odt, status=status)
        for x, got, scale in zip((k, v), back, scales):
            want, byte = quantised(x.double())
            assert torch.equal(scale.view(-1, nkv)[slots.to(cuda_device)].cpu(), byte)
            assert torch.equal(got.cpu().double().nan_to_num(1e300), want.to(odt).double().nan_to_num(1e300))
    untouched = torch.ones(blocks * bs, dtype=torch.bool)
    untouched[slots] = False
    for p, s in zip(pools, scales):
        assert bool((p.view(torch.uint8).view(-1, nkv, hd).cpu()[untouched] == 0x35).all())
        assert bool((s.view(-1, nkv).cpu()[untouched] == 9).all())
    assert int(status) == 0


def test_fp8_cache_out_of_range_slots(cuda_device):
    g = torch.Generator().manual_seed(1)
    k = torch.randn(4, 2, 64, generator=g).to(cuda_device)
    pools = [torch.zeros(2, 16, 2, 64, dtype=torch.uint8, device=cuda_device).view(E4M3) for _ in range(2)]
    scales = [torch.full((2, 16, 2), 127, dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    slots = torch.tensor([5, -1, 32, 9], device=cuda_device)
    status = ops.status_tensor(cuda_device)
    ops.kv_append_fp8(k, k, slots, *pools, *scales, status=status)
    assert int(status) == -7
    status.zero_()
    a, b = ops.kv_read_fp8(*pools, *scales, slots, dtype=torch.float32, status=status)
    assert int(status) == -7 and torch.equal(a, b)
    assert bool((a[1:3] == 0).all()) and torch.equal(a[[0, 3]].cpu().double(), quantised(k[[0, 3]].cpu().double())[0])
    assert int((pools[0].view(torch.uint8).view(32, -1) != 0).any(1).sum()) == 2
    empty = torch.empty(0, dtype=torch.int64, device=cuda_device)
    assert ops.kv_read_fp8(*pools, *scales, empty)[0].shape == (0, 2, 64)
    ops.kv_append_fp8(k[:0], k[:0], empty, *pools, *scales)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq, nkv, hd, n", [(14, 2, 64, 5), (16, 2, 128, 33), (1, 1, 64, 1), (8, 8, 128, 7)])
def test_qkv_rope_append_fp8(cuda_device, dt, nq, nkv, hd, n):
    dev = cuda_device
    g = torch.Generator().manual_seed(nq)
    qkv = torch.randn(n, (nq + 2 * nkv) * hd, generator=g).to(dt).to(dev)
    slots = torch.randperm(64, generator=g)[:n].to(torch.int32).to(dev)
    pos = torch.randint(0, 500, (n,), generator=g).to(torch.int32)
    angle = torch.arange(500.0)[:, None] * 1e4 ** (-torch.arange(0, hd, 2) / hd)
    cos, sin = angle.cos().to(dev), angle.sin().to(dev)
    pools = [torch.zeros(4, 16, nkv, hd, dtype=torch.uint8, device=dev).view(E4M3) for _ in range(2)]
    scales = [torch.full((4, 16, nkv), 127, dtype=torch.uint8, device=dev) for _ in range(2)]
    q_out = torch.empty(n, nq, hd, dtype=dt, device=dev)
    ops.qkv_rope_append_fp8(qkv, pos.to(dev), slots, cos, sin, q_out, *pools, *scales, nq, nkv, hd)
    x = qkv.view(n, nq + 2 * nkv, hd)
    a, b = x[:, :nq + nkv].float().chunk(2, -1)
    c, s = cos[pos.long()][:, None], sin[pos.long()][:, None]
    turned = torch.cat([a * c - b * s, b * c + a * s], -1)  # the fp32 operations in the documented order
    assert torch.equal(q_out, turned[:, :nq].to(dt))
    k, v = ops.kv_read_fp8(*pools, *scales, slots.long(), dtype=torch.float32)
    assert torch.equal(k.cpu().double(), quantised(turned[:, nq:].cpu().double())[0])
    assert torch.equal(v.cpu().double(), quantised(x[:, nq + nkv:].cpu().double())[0])
    # against the angles themselves: q within fp32's error of the tables and one rounding
    ex = torch.polar(torch.ones_like(angle.double()), angle.double())[pos.long()][:, None]
    z = torch.complex(*x[:, :nq].cpu().double().chunk(2, -1)) * ex
    z = torch.cat([z.real, z.imag], -1)
    size = torch.hypot(*x[:, :nq].cpu().double().chunk(2, -1)).repeat(1, 1, 2)
    assert bool(((q_out.cpu().double() - z).abs() <= size * 8 * U32 + z.abs() * (U16 if dt == torch.bfloat16 else U32)).all())
    # bad positions and slots are reported; a token with a bad slot still gets its q
    status = ops.status_tensor(dev)
    bad = slots.clone()
    bad[0] = 64
    before = pools[0].view(torch.uint8).clone()
    q2 = torch.zeros_like(q_out)
    ops.qkv_rope_append_fp8(qkv, pos.to(dev), bad, cos, sin, q2, *pools, *scales, nq, nkv, hd, status=status)
    assert int(status) == -7 and torch.equal(q2, q_out) and torch.equal(pools[0].view(torch.uint8), before)
    status.zero_()
    ops.qkv_rope_append_fp8(qkv, torch.full_like(pos, 500).to(dev), slots, cos, sin, q2, *pools, *scales, nq, nkv, hd,
                            status=status)
    assert int(status) == -7


def test_fp8_pool_write_returns_what_it_holds(cuda_device):
    pool = PagedKVCache(2, 2, 64, 8, 16, E4M3, cuda_device)
    seq = pool.new_sequence("s")
    g = torch.Generator().manual_seed(0)
    rows = []
    for n in (20, 1, 5):
        k = torch.randn(1, 2, n, 64, generator=g).to(torch.bfloat16).to(cuda_device)
        rows.append(k)
        start = seq.length
        seq.reserve(n)
        for layer in range(2):
            k_all, v_all = seq.write(layer, k, -k, start)
        seq.commit(n)
        want = quantised(torch.cat(rows, 2).cpu().double())[0]
        assert k_all.shape == (1, 2, start + n, 64) and k_all.dtype == torch.bfloat16
        assert torch.equal(k_all.cpu().double(), want) and torch.equal(v_all, -k_all)


# ---------------------------------------------------------------- sampled verification
def clean(x):
    return torch.where(torch.isnan(x), -math.inf, x.double())


def probs(x, t):
    x = clean(x)
    top = x.max()
    p = torch.zeros_like(x)
    if not t > 0:
        p[int((x == top).nonzero()[0])] = 1
    elif top == math.inf:
        p[x == math.inf] = 1.0 / int((x == math.inf).sum())
    elif top > -math.inf:
        p = (x / t).softmax(0)
    return p


def pick(w, p, gumbel):
    w = w if bool((w > 0).any()) else p
    if not bool((w > 0).any()):
        return 0
    key = w.log() + gumbel.double()
    return int((key == key.max()).nonzero()[0])


def plain_chain(logits, drafts, u, gumbel, t, draft_logits=None):
    B, k = drafts.shape
    ns, em, lp = [], [], []
    for b in range(B):
        tok, ll, temp = [], [], float(t[b])
        for j in range(k + 1):
            p = probs(logits[b, j], temp)
            w = p
            if j == k:
                break
            d = int(drafts[b, j])
            q = torch.zeros_like(p)
            if draft_logits is None:
                q[d] = 1
            else:
                q = probs(draft_logits[b, j], temp)
            if not 0 <= d < p.numel() or not float(u[b, j]) * float(q[d]) < float(p[d]):
                w = (p - q).clamp(min=0)
                break
            tok.append(d)
            ll.append(math.log(p[d]) if temp > 0 else 0.0)
        last = pick(w, p, gumbel[b])
        ll.append(0.0 if not temp > 0 else math.log(p[last]) if p[last] > 0 else -math.inf)
        ns.append(len(tok))
        em.append(tok + [last] + [-1] * (k - len(tok)))
        lp.append(ll + [0.0] * (k + 1 - len(ll)))
    return ns, em, lp


LOGP = 2.0 ** -22 + 2 * U32 * 40 + 64 * U32  # as derived above


def same_logprobs(got, want):
    got, want = got.cpu().double(), torch.tensor(want, dtype=torch.float64)
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin], want[~fin])
    assert bool(((got - want)[fin].abs() <= LOGP + U32 * want[fin].abs()).all()), float((got - want)[fin].abs().max())


def chain_inputs(B, k, V, dt, g, spread=2.5):
    target = torch.randn(B, k + 1, V, generator=g) * spread
    draft = (target[:, :k] * 0.9 + torch.randn(B, k, V, generator=g)).to(dt)
    t = 0.5 + torch.rand(B, generator=g)
    gum = lambda *s: -torch.empty(*s).exponential_(generator=g).log()  # noqa: E731
    drafts = (draft.float() / t[:, None, None] + gum(B, k, V)).argmax(-1).int()
    return target.to(dt), draft, drafts, torch.rand(B, k, generator=g), gum(B, V), t


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B, k, V", [(1, 1, 1), (3, 2, 7), (5, 4, 1000), (9, 3, 50257), (2, 31, 333), (1, 4, 151936)])
@pytest.mark.parametrize("with_draft", [False, True])
def test_sample_accept(cuda_device, dt, B, k, V, with_draft):
    g = torch.Generator().manual_seed(B * 100 + k)
    target, draft, drafts, u, gumbel, t = chain_inputs(B, k, V, dt, g)
    t[B // 2:: 3] = 0
    if V > 20:  # what a top-k filter leaves, in one row and the whole of one sequence
        target[0, 0, target[0, 0] < 1] = -math.inf
        draft[-1][draft[-1] < 1] = -math.inf
    want = plain_chain(target, drafts, u, gumbel, t, draft if with_draft else None)
    dev = [x.to(cuda_device) for x in (target, drafts, u, gumbel, t)]
    ws = ops.Workspace(cuda_device)
    status = ops.status_tensor(cuda_device)
    got = ops.sample_accept(*dev, draft_logits=draft.to(cuda_device) if with_draft else None, workspace=ws, status=status)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    same_logprobs(got[2], want[2])
    assert int(status) == 0 and int(ws.buf[:65536].sum()) == 0
    # the same from strided inputs: rows of a wider buffer from an odd column on, drafts and their logits transposed
    wide = torch.full((B * (k + 1), V + 13), math.nan, dtype=dt, device=cuda_device)
    wide[:, 5:5 + V] = dev[0].view(-1, V)
    strided = wide[:, 5:5 + V].unflatten(0, (B, k + 1))
    dl = draft.to(cuda_device).transpose(0, 1).contiguous().transpose(0, 1) if with_draft else None
    gw = torch.full((B, V + 3), math.nan, device=cuda_device)
    gw[:, 1:V + 1] = dev[3]
    again = ops.sample_accept(strided, dev[1].t().contiguous().t(), dev[2], gw[:, 1:V + 1], dev[4], draft_logits=dl)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
    same_logprobs(again[2], want[2])


def test_sample_accept_odd_logits(cuda_device):
    """NaN, infinities, rows without probability, equal distributions, drafts out of range."""
    g = torch.Generator().manual_seed(7)
    B, k, V = 8, 2, 900
    target, draft, drafts, u, gumbel, t = chain_inputs(B, k, V, torch.float32, g)
    t[:] = 0.8
    target[0, :, 5] = math.nan
    draft[0, :, 9] = math.nan
    drafts[0, 0] = 5                       # a draft whose logit is NaN
    target[1, 0, [3, 8]] = math.inf        # two infinities share the probability
    drafts[1, 0] = 8
    target[2] = -math.inf                  # no probability at all
    draft[3] = target[3, :k]               # p = q: always accepted
    target[4] = target[4] + 3e4            # large logits
    target[5, :, 1:] = -math.inf           # one token
    drafts[6] = torch.tensor([-1, V])      # not tokens
    target[7, 0] = torch.finfo(torch.float32).min
    target[7, 0, 4] = 0
    for dl in (draft, None):
        want = plain_chain(target, drafts.clamp(0, V - 1) if dl is not None else drafts.clamp(0, V - 1), u, gumbel, t, dl)
        status = ops.status_tensor(cuda_device)
        got = ops.sample_accept(*[x.to(cuda_device) for x in (target, drafts, u, gumbel, t)],
                                draft_logits=None if dl is None else dl.to(cuda_device), status=status)
        rows = [0, 1, 2, 3, 4, 5, 7]
        assert [got[0].tolist()[i] for i in rows] == [want[0][i] for i in rows]
        assert [got[1].tolist()[i] for i in rows] == [want[1][i] for i in rows]
        same_logprobs(got[2][rows], [want[2][i] for i in rows])
        assert int(status) == -7 and int(got[0][6]) == 0 and 0 <= int(got[1][6, 0]) < V
    assert got[1][2].tolist() == [0, -1, -1] and float(got[2][2, 0]) == -math.inf


@pytest.mark.parametrize("with_draft", [False, True])
def test_sample_accept_neighbouring_columns_that_fp32_cannot_tell_apart(cuda_device, with_draft):
    """Two neighbours whose keys differ by 1e-7 at a key of 40: the greater wins, wherever it lies; equal ones: the lower."""
    B, V = 64, 4096
    target = torch.full((B, 2, V), -5.0)
    target[:, :, 7] = 30.0
    draft = torch.full((B, 1, V), -5.0)
    draft[:, :, 5] = 60.0
    gumbel = torch.zeros(B, V)
    drafts = torch.full((B, 1), 5, dtype=torch.int32)
    want = []
    for b in range(B):
        c = 8 + 61 * b
        gumbel[b, c:c + 2] = 60.0
        target[b, :, c] = 0.0
        target[b, :, c + 1] = (b % 3 - 1) * 1.2e-7  # below, the same, above
        want.append(c + 1 if b % 3 == 2 else c)
    u, t = torch.full((B, 1), 0.5), torch.ones(B)  # rejected: q(5) is 1, p(5) e^-35
    got = ops.sample_accept(*[x.to(cuda_device) for x in (target, drafts, u, gumbel, t)],
                            draft_logits=draft.to(cuda_device) if with_draft else None)
    assert got[0].tolist() == [0] * B and got[1][:, 0].tolist() == want
    assert plain_chain(target, drafts, u, gumbel, t, draft if with_draft else None)[1] == got[1].tolist()


def test_sample_accept_draws_from_the_target(cuda_device):
    """Whatever the draft, the first emitted token is distributed as the target's: counts within five
    standard deviations (fixed seed), with a draft distribution, and with drafts that have none."""
    B, V = 40000, 6
    g = torch.Generator().manual_seed(3)
    row, guess = torch.randn(V, generator=g) * 1.5, torch.randn(V, generator=g) * 1.5
    gum = lambda: -torch.empty(B, V).exponential_(generator=g).log()  # noqa: E731
    t = torch.full((B,), 0.7)
    p = (row.double() / 0.7).softmax(0)
    for dl in (guess, None):
        if dl is None:
            drafts = torch.full((B, 1), int(guess.argmax()), dtype=torch.int32)
        else:
            drafts = (guess / 0.7 + gum()).argmax(1, keepdim=True).int()
        _, emitted, _ = ops.sample_accept(
            row.expand(B, 2, V).contiguous().to(cuda_device), drafts.to(cuda_device),
            torch.rand(B, 1, generator=g).to(cuda_device), gum().to(cuda_device), t.to(cuda_device),
            draft_logits=None if dl is None else dl.expand(B, 1, V).contiguous().to(cuda_device))
        share = torch.bincount(emitted[:, 0].cpu().long(), minlength=V) / B
        assert bool(((share - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all()), (share, p)


def plain_tree(logits, tokens, parents, u, gumbel, t, wide):
    """One tree, walked node by node."""
    n, temp = len(parents), float(t)
    path, tok, lp = [0], [], []
    while True:
        p = probs(logits[path[-1]], temp)
        w, left, nxt = p.clone(), 1.0, None
        for c in range(1, n):
            if parents[c] != path[-1]:
                continue
            d = int(tokens[c])
            if float(u[c]) * left < float(w[d]):
                nxt = c
                break
            left -= float(w[d])
            w[d] = 0
        if nxt is None:
            break
        path.append(nxt)
        tok.append(int(tokens[nxt]))
        lp.append(math.log(p[tok[-1]]) if temp > 0 else 0.0)
    tok.append(pick(w, p, gumbel))
    lp.append(0.0 if not temp > 0 else math.log(p[tok[-1]]) if p[tok[-1]] > 0 else -math.inf)
    pad = lambda x, v: x + [v] * (wide - len(x))  # noqa: E731
    return len(path) - 1, pad(path, -1), pad(tok, -1), pad(lp, 0.0)


def tree_inputs(trees, V, dt, g, rng, spread=3.0):
    n = sum(len(t) for t in trees)
    logits = (torch.randn(n, V, generator=g) * spread).to(dt)
    tokens, row = [], 0
    for t in trees:
        for i, p in enumerate(t):
            if i == 0:
                tokens.append(-5)  # not read
            else:  # a likely token of the parent, siblings may repeat one
                tokens.append(int(logits[row + p].float().topk(min(V, 4)).indices[rng.randrange(min(V, 4))]))
        row += len(t)
    return logits, torch.tensor(tokens, dtype=torch.int32), torch.rand(n, generator=g)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V, shapes", [(1, [1, 2]), (17, [5, 1, 9]), (1024, [7, 33, 0, 2]), (50257, [16] * 5),
                                       (151936, [9]), (600, [64, 3, 40])])
def test_tree_sample_accept(cuda_device, dt, V, shapes):
    g, rng = torch.Generator().manual_seed(V), random.Random(V)
    trees = [[-1] + [rng.randint(max(0, i - 4), i - 1) for i in range(1, n)] if n else [] for n in shapes]
    logits, tokens, u = tree_inputs(trees, V, dt, g, rng)
    B, wide = len(trees), max(shapes)
    t = 0.5 + torch.rand(B, generator=g)
    t[1::2] = 0
    gumbel = -torch.empty(B, V).exponential_(generator=g).log()
    off = [sum(shapes[:b]) for b in range(B + 1)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    status = ops.status_tensor(cuda_device)
    got = ops.tree_sample_accept(logits.to(cuda_device), tokens.to(cuda_device), i32([p for x in trees for p in x]),
                                 i32(shapes), i32(off), wide, u.to(cuda_device), gumbel.to(cuda_device), t.to(cuda_device),
                                 status=status)
    assert int(status) == 0
    for b, x in enumerate(trees):
        if not x:
            assert int(got[0][b]) == -1
            continue
        s = slice(off[b], off[b + 1])
        want = plain_tree(logits[s], tokens[s], x, u[s], gumbel[b], t[b], wide)
        assert (int(got[0][b]), got[1][b].tolist(), got[2][b].tolist()) == want[:3], b
        same_logprobs(got[3][b:b + 1], [want[3]])


def test_tree_sample_accept_largest_tree(cuda_device):
    """1024 nodes: a chain that is accepted to its end, and a random tree beside it."""
    g, rng = torch.Generator().manual_seed(47), random.Random(47)
    trees = [[i - 1 for i in range(1024)], [-1] + [rng.randint(0, i - 1) for i in range(1, 1024)]]
    V = 1500
    logits, tokens, u = tree_inputs(trees, V, torch.float32, g, rng)
    u[:1024] = 0.0
    gumbel = -torch.empty(2, V).exponential_(generator=g).log()
    t = torch.tensor([0.9, 1.1])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    got = ops.tree_sample_accept(logits.to(cuda_device), tokens.to(cuda_device), i32(trees[0] + trees[1]), i32([1024, 1024]),
                                 i32([0, 1024, 2048]), 1024, u.to(cuda_device), gumbel.to(cuda_device), t.to(cuda_device))
    want = [plain_tree(logits[o:o + 1024], tokens[o:o + 1024], trees[b], u[o:o + 1024], gumbel[b], t[b], 1024)
            for b, o in ((0, 0), (1, 1024))]
    assert got[0].tolist() == [w[0] for w in want] and got[0].tolist()[0] == 1023
    assert got[1].tolist() == [w[1] for w in want] and got[2].tolist() == [w[2] for w in want]


def test_tree_sample_accept_stars_chains_and_bad_nodes(cuda_device):
    g, rng = torch.Generator().manual_seed(2), random.Random(2)
    V, wide = 300, 1024
    trees = [[-1] + [0] * 1023, [-1] + list(range(1023)), [-1, 0, 0, 0]]
    logits, tokens, u = tree_inputs(trees, V, torch.float32, g, rng)
    u[1024:2048] = 0                                  # the chain is accepted to its end
    tokens[1:1024] = torch.arange(1023) % V           # the star: every token, some again and again
    u[:1024] = 0.9999
    t, gumbel = torch.tensor([1.0, 0.6, 0.9]), -torch.empty(3, V).exponential_(generator=g).log()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    args = [x.to(cuda_device) for x in (logits, tokens)] + [i32([p for x in trees for p in x]), i32([1024, 1024, 4]),
                                                            i32([0, 1024, 2048]), wide, u.to(cuda_device),
                                                            gumbel.to(cuda_device), t.to(cuda_device)]
    got = ops.tree_sample_accept(*args)
    for b, x in enumerate(trees):
        s = slice(1024 * b, 1024 * b + len(x))
        want = plain_tree(logits[s], tokens[s], x, u[s], gumbel[b], t[b], wide)
        assert (int(got[0][b]), got[1][b].tolist(), got[2][b].tolist()) == want[:3], b
    assert int(got[0][1]) == 1023
    # nodes with a parent or token out of range are nobody's children
    status = ops.status_tensor(cuda_device)
    par = [p for x in trees for p in x]
    par[2049], tok = 7, tokens.clone()
    tok[2050] = V
    res = ops.tree_sample_accept(args[0], tok.to(cuda_device), i32(par), *args[3:], status=status)
    s = slice(2048, 2052)
    want = plain_tree(logits[s], torch.where(tokens[s] < 0, 0, tokens[s]), [-1, -1, -1, 0], u[s], gumbel[2], t[2], wide)
    assert int(status) == -7 and (int(res[0][2]), res[1][2].tolist(), res[2][2].tolist()) == want[:3]
    # lengths that do not fit the rows
    for lens, offs in (([1024, 1024, 5], [0, 1024, 2048]), ([1024, 1024, 4], [0, 1024, -1]), ([1024, -2, 4], [0, 1024, 2048])):
        status.zero_()
        res = ops.tree_sample_accept(*args[:3], i32(lens), i32(offs), *args[5:], status=status)
        assert int(status) == -7 and -1 in res[0].tolist()


def test_tree_sample_accept_draws_from_the_target(cuda_device):
    B, V = 40000, 6
    g = torch.Generator().manual_seed(5)
    row = torch.randn(V, generator=g) * 1.5
    p = (row.double() / 0.8).softmax(0)
    trees = torch.tensor([-1, 0, 0, 0], dtype=torch.int32).repeat(B)   # three candidates, one of them twice
    tokens = torch.tensor([0, 2, 4, 2], dtype=torch.int32).repeat(B)
    gumbel = -torch.empty(B, V).exponential_(generator=g).log()
    n, path, emitted, _ = ops.tree_sample_accept(
        row.expand(4 * B, V).contiguous().to(cuda_device), tokens.to(cuda_device), trees.to(cuda_device),
        torch.full((B,), 4, dtype=torch.int32, device=cuda_device),
        (torch.arange(B + 1, dtype=torch.int32) * 4).to(cuda_device), 4, torch.rand(4 * B, generator=g).to(cuda_device),
        gumbel.to(cuda_device), torch.full((B,), 0.8, device=cuda_device))
    share = torch.bincount(emitted[:, 0].cpu().long(), minlength=V) / B
    assert bool(((share - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all()), (share, p)
    assert not bool((path == 3).any())  # the repeated token is never accepted the second time


def test_sampling_wrapper_refusals(cuda_device):
    g = torch.Generator().manual_seed(1)
    target, draft, drafts, u, gumbel, t = [x.to(cuda_device) for x in chain_inputs(2, 3, 40, torch.float32, g)]
    ok = dict(logits=target, drafts=drafts, uniforms=u, gumbel=gumbel, temperature=t, draft_logits=draft)
    ops.sample_accept(**ok)
    for change in (dict(logits=target.transpose(0, 1)), dict(drafts=drafts.long()), dict(uniforms=u[:, :2]),
                   dict(gumbel=gumbel.double()), dict(gumbel=gumbel.t().contiguous().t()), dict(temperature=t[:1]),
                   dict(draft_logits=draft.bfloat16()), dict(draft_logits=draft[:, :2]), dict(temperature=t.cpu()),
                   dict(logits=target.half()), dict(out=(t, t, t))):
        with pytest.raises((ValueError, TypeError)):
            ops.sample_accept(**dict(ok, **change))


def test_sampling_in_a_graph_with_new_inputs(cuda_device):
    g = torch.Generator().manual_seed(9)
    first = [x.to(cuda_device) for x in chain_inputs(3, 4, 2000, torch.bfloat16, g)]
    ws = ops.Workspace(cuda_device)
    run = lambda: ops.sample_accept(first[0], first[2], first[3], first[4], first[5], draft_logits=first[1], workspace=ws)  # noqa: E731
    ws.get(1 << 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = run()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        new = chain_inputs(3, 4, 2000, torch.bfloat16, g)
        for x, y in zip(first, new):
            x.copy_(y)
        graph.replay()
        want = plain_chain(new[0], new[2], new[3], new[4], new[5], new[1])
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1]


# ---------------------------------------------------------------- the accepted path
@pytest.mark.parametrize("cache", ["bf16", "fp32", "fp8"])
@pytest.mark.parametrize("nkv, hd, bs, layers", [(2, 64, 16, 3), (2, 128, 16, 2), (1, 64, 1, 2), (3, 32, 5, 1)])
def test_kv_commit_path(cuda_device, cache, nkv, hd, bs, layers):
    g, rng = torch.Generator().manual_seed(bs), random.Random(bs)
    starts, width = [0, 37, 15, 4, 80], 20
    paths = [[0, 2, 3, 9, 17], [0], [0, 1, 2], [0, 1, 5, 6, 7, 8, 9, 10, 11, 12, 13, 19], [0] + list(range(2, 20))]
    need = [-(-(s + 20) // bs) for s in starts]
    ids = list(range(sum(need)))
    rng.shuffle(ids)
    table = torch.zeros(5, max(need), dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([ids.pop() for _ in range(n)])
    k, v, ks, vs = zip(*[cache_of(cache, sum(need), bs, nkv, hd, g, cuda_device) for _ in range(layers)])
    stack = lambda xs: None if xs[0] is None else torch.stack([x.view(torch.uint8) for x in xs]).view(xs[0].dtype)  # noqa: E731
    got = [stack(x) for x in (k, v, ks, vs)]
    want = [None if x is None else x.view(torch.uint8).clone().cpu().flatten(1, 2) for x in got]
    for b, (s, path) in enumerate(zip(starts, paths)):
        slot = lambda p: int(table[b, p // bs]) * bs + p % bs  # noqa: E731
        for x in want:
            if x is not None:
                rows = [x[:, slot(s + node)].clone() for node in path]
                for j, r in enumerate(rows):
                    x[:, slot(s + j)] = r
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    status = ops.status_tensor(cuda_device)
    ops.kv_commit_path(got[0], got[1], table.to(cuda_device), i32(starts), i32([p + [-1] * (width - len(p)) for p in paths]),
                       i32([len(p) - 1 for p in paths]), k_scale=got[2], v_scale=got[3], status=status)
    assert int(status) == 0
    for x, y in zip(got, want):
        assert x is None or torch.equal(x.view(torch.uint8).cpu().flatten(1, 2), y)


def test_kv_commit_path_skips_bad_paths(cuda_device):
    g = torch.Generator().manual_seed(0)
    pool = torch.randn(1, 4, 16, 1, 64, generator=g).to(cuda_device)
    other = pool.clone()
    table = torch.tensor([[0], [1], [2], [3]], dtype=torch.int32, device=cuda_device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    good = pool.clone()
    good[0, 3, 5] = pool[0, 3, 6]
    for starts, paths, n, tab in (
            ([4, 4, 4, 4], [[0, 3, 2], [0, 0, 1], [0, 5, 12], [0, 2, -1]], [2, 1, 2, 1], table),  # not ascending, past the table
            ([4, -1, 4, 4], [[0, 2, 3], [0, 2, 3], [0, 2, 3], [0, 2, 3]], [3, 1, -2, 1], table),  # counts and starts
            ([4, 4, 4, 4], [[0, 2, 3], [0, 2, 3], [0, 2, 3], [0, 2, 3]], [0, -1, 1, 1], i32([[0], [1], [9], [3]]))):  # a block
        a, b = pool.clone(), other.clone()
        status = ops.status_tensor(cuda_device)
        ops.kv_commit_path(a, b, tab, i32(starts), i32(paths), i32(n), status=status)
        assert int(status) == -7 and torch.equal(a, good) and torch.equal(b, good)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("cache", ["bf16", "fp8"])
def test_a_tree_step_then_a_decode_step(cuda_device, cache):
    """Trees written behind two sequences' histories, attended, verified, their accepted paths moved
    together: the next single-token attention equals one over a cache that only ever held the
    accepted tokens."""
    dev = cuda_device
    nq, nkv, hd, bs, L, V = 4, 2, 64, 16, 2, 500
    g, rng = torch.Generator().manual_seed(6), random.Random(6)
    trees = [[-1, 0, 0, 1, 1, 3, 5], [-1, 0, 1, 1, 2]]
    hist = [33, 14]
    B, nodes = 2, [len(t) for t in trees]
    off = [0, 7, 12]
    dt = torch.bfloat16
    pool = PagedKVCache(L, nkv, hd, 16, bs, E4M3 if cache == "fp8" else dt, dev)
    seqs = [pool.new_sequence(b) for b in range(B)]
    angle = torch.arange(64.0)[:, None] * 1e4 ** (-torch.arange(0, hd, 2) / hd)
    cos, sin = angle.cos().to(dev), angle.sin().to(dev)

    def append(pool, layer, qkv, pos, slots):
        q = torch.empty(qkv.shape[0], nq, hd, dtype=dt, device=dev)
        pos, slots = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (pos, slots))
        if cache == "fp8":
            ops.qkv_rope_append_fp8(qkv, pos, slots, cos, sin, q, pool.k[layer], pool.v[layer], pool.k_scale[layer],
                                    pool.v_scale[layer], nq, nkv, hd)
        else:
            ops.qkv_rope_append(qkv, pos, slots, cos, sin, q, pool.k[layer], pool.v[layer], nq, nkv, hd)
        return q

    def attend(pool, layer, q, seqs, ctx, lens, mask):
        width = max(len(s.blocks) for s in seqs)
        tables = torch.stack([s.block_table_tensor(width) for s in seqs])
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        scales = {} if cache != "fp8" else dict(k_scale=pool.k_scale[layer], v_scale=pool.v_scale[layer])
        return tables, ops.tree_attention(q, pool.k[layer], pool.v[layer], tables, i32(ctx), i32(lens),
                                          i32([sum(lens[:b]) for b in range(len(lens) + 1)]), max(lens), max(ctx), hd ** -0.5,
                                          tree_mask=mask, **scales)

    width = (nq + 2 * nkv) * hd
    history = [[torch.randn(h, width, generator=g).to(dt).to(dev) for h in hist] for _ in range(L)]
    fresh = [torch.randn(12, width, generator=g).to(dt).to(dev) for _ in range(L)]
    for s, h in zip(seqs, hist):
        s.reserve(h)
    for layer in range(L):
        for s, h, x in zip(seqs, hist, history[layer]):
            append(pool, layer, x, list(range(h)), s.slot_list(0, h))
    for s, h, n in zip(seqs, hist, nodes):
        s.commit(h)
        s.reserve(n)
    # the trees: a node's position is its depth, its slot its index
    depth = []
    for t, h in zip(trees, hist):
        d = []
        for p in t:
            d.append(d[p] + 1 if p >= 0 else h)
        depth.append(d)
    mask = ops.tree_mask_words(trees).to(dev)
    for layer in range(L):
        q = append(pool, layer, fresh[layer], depth[0] + depth[1],
                   seqs[0].slot_list(hist[0], 7) + seqs[1].slot_list(hist[1], 5))
        tables, out = attend(pool, layer, q, seqs, [h + n for h, n in zip(hist, nodes)], nodes, mask)
    # verification, with numbers that accept a path of each tree
    logits, tokens, u = tree_inputs(trees, V, dt, g, rng)
    u *= 0.05
    gumbel = -torch.empty(B, V).exponential_(generator=g).log()
    t = torch.tensor([0.7, 0.7])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    n_acc, path, emitted, _ = ops.tree_sample_accept(
        logits.to(dev), tokens.to(dev), i32(trees[0] + trees[1]), i32(nodes), i32(off), 7, u.to(dev), gumbel.to(dev), t.to(dev))
    want = [plain_tree(logits[off[b]:off[b + 1]], tokens[off[b]:off[b + 1]], trees[b], u[off[b]:off[b + 1]], gumbel[b], t[b], 7)
            for b in range(B)]
    assert n_acc.tolist() == [w[0] for w in want] and path.tolist() == [w[1] for w in want]
    assert max(n_acc.tolist()) >= 2
    ops.kv_commit_path(pool.k, pool.v, tables, i32(hist), path, n_acc, k_scale=pool.k_scale, v_scale=pool.v_scale)
    kept = [h + n + 1 for h, n in zip(hist, n_acc.tolist())]
    for s, n, keep in zip(seqs, nodes, kept):
        s.commit_and_keep(n, keep)
        s.reserve(1)
    # the same tokens alone
    pool2 = PagedKVCache(L, nkv, hd, 16, bs, pool.dtype, dev)
    seqs2 = [pool2.new_sequence(b) for b in range(B)]
    for s, keep in zip(seqs2, kept):
        s.reserve(keep + 1)
    step = [torch.randn(2, width, generator=g).to(dt).to(dev) for _ in range(L)]
    for layer in range(L):
        for b, (s, h) in enumerate(zip(seqs2, hist)):
            rows = [off[b] + x for x in want[b][1] if x >= 0]
            append(pool2, layer, torch.cat([history[layer][b], fresh[layer][rows]]), list(range(kept[b])),
                   s.slot_list(0, kept[b]))
        outs = []
        for p, ss in ((pool, seqs), (pool2, seqs2)):
            q = append(p, layer, step[layer], kept, [s.slot_list(keep, 1)[0] for s, keep in zip(ss, kept)])
            outs.append(attend(p, layer, q, ss, [keep + 1 for keep in kept], [1, 1], None)[1])
        assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("cache", ["bf16", "fp8"])
def test_calls_without_the_cpp_binding(cuda_device, monkeypatch, cache):
    """The same calls through Python and ctypes: results, checks and refusals."""
    monkeypatch.setattr(L, "_fast", L._NoFast())
    test_tree_attention_many_rows(cuda_device, cache, (16, 2, 128), [8, 3], [100, 700], 16, "tree")
    test_tree_attention_wrapper_refusals(cuda_device)
    test_kv_append_and_read_fp8(cuda_device, torch.bfloat16, 2, 64, 16, 67)
    test_qkv_rope_append_fp8(cuda_device, torch.float32, 14, 2, 64, 5)
    test_sample_accept(cuda_device, torch.bfloat16, 5, 4, 1000, True)
    test_tree_sample_accept(cuda_device, torch.float32, 1024, [7, 33, 0, 2])
    test_sampling_wrapper_refusals(cuda_device)
    test_kv_commit_path(cuda_device, cache, 2, 64, 16, 3)
    test_a_tree_step_then_a_decode_step(cuda_device, cache)
