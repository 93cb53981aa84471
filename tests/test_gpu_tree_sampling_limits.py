"""Sampling, draft trees and the 8-bit cache at their limits: temperatures and logits of every size,
drafts whose distribution is nearly the target's.

Tolerances as in test_gpu_tree_sampling.py, which derives them.
"""

import math
import random

import pytest
import torch

from kvengine_b200 import PagedKVCache, ops
from test_gpu_tree_sampling import (U16, U32, attention_case, check_attention, plain_chain, plain_tree, same_logprobs,
                                    tree_inputs, values)

pytestmark = pytest.mark.gpu


def gumbels(*shape, g):
    return -torch.empty(*shape).exponential_(generator=g).log()


# ---------------------------------------------------------------- temperatures and logits of every size
def extreme_rows(n, V, dt, g, kind):
    """Rows of logits, some with two equal largest ones."""
    x = torch.randn(n, V, generator=g) * 3
    if kind == "large":
        x = x * 1e10
    elif kind == "largest":
        x[:, :: 2] = -torch.finfo(dt).max
        x[:, 1] = torch.finfo(dt).max
    else:
        x[:, 7] = 30.0
    x[::3, 5] = x[::3].max(-1).values
    x[1::4, 3] = -math.inf
    return x.to(dt)


EXTREMES = [("usual", t) for t in (1e-2, 1e-4, 1e-6, 1e-7, 1e-8, 1e-9, 1e-12, 1e-20, 1e-30, 1e-37, 1e-38, 1e-41, 1e10, 1e30,
                                   3e38)] + [("large", 1.0), ("large", 1e-3), ("large", 1e10), ("largest", 1.0),
                                                 ("largest", 1e-6), ("largest", 1e20)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [40, 9000])
@pytest.mark.parametrize("kind, temperature", EXTREMES)
def test_sample_accept_at_any_temperature(cuda_device, dt, V, kind, temperature):
    """Down to the least temperatures and up to the largest logits the probabilities are the definition's: near zero
    the equal largest logits share everything."""
    g = torch.Generator().manual_seed(V + 1)
    B, k = 6, 3
    target = extreme_rows(B * (k + 1), V, dt, g, kind).view(B, k + 1, V)
    draft = extreme_rows(B * k, V, dt, g, kind).view(B, k, V)
    drafts = target[:, :k].float().argmax(-1).int()
    drafts[1::2, 1] = 11
    u, t, gumbel = torch.rand(B, k, generator=g), torch.full((B,), temperature), gumbels(B, V, g=g)
    for dl in (None, draft):
        want = plain_chain(target, drafts, u, gumbel, t, dl)
        got = ops.sample_accept(*[x.to(cuda_device) for x in (target, drafts, u, gumbel, t)],
                                draft_logits=None if dl is None else dl.to(cuda_device))
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
        same_logprobs(got[2], want[2])


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind, temperature", EXTREMES)
def test_tree_sample_accept_at_any_temperature(cuda_device, dt, kind, temperature):
    g = torch.Generator().manual_seed(5)
    V, tree = 9000, [-1, 0, 0, 1, 1, 2, 3]
    B, n = 5, len(tree)
    logits = extreme_rows(B * n, V, dt, g, kind)
    top = logits.float().topk(2).indices
    tokens = torch.tensor([0 if p < 0 else int(top[b * n + p, i % 2]) for b in range(B) for i, p in enumerate(tree)],
                          dtype=torch.int32)
    u, t, gumbel = torch.rand(B * n, generator=g), torch.full((B,), temperature), gumbels(B, V, g=g)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    got = ops.tree_sample_accept(logits.to(cuda_device), tokens.to(cuda_device), i32(tree * B), i32([n] * B),
                                 i32([n * b for b in range(B + 1)]), n, u.to(cuda_device), gumbel.to(cuda_device),
                                 t.to(cuda_device))
    for b in range(B):
        s = slice(b * n, b * n + n)
        want = plain_tree(logits[s], tokens[s], tree, u[s], gumbel[b], t[b], n)
        assert (int(got[0][b]), got[1][b].tolist(), got[2][b].tolist()) == want[:3], b
        same_logprobs(got[3][b:b + 1], [want[3]])


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [3e3, 1e5, -1e6, 1.5e6, 2.9e6, 6e6])
@pytest.mark.parametrize("V", [5, 2000, 30000])
def test_sampling_with_logits_far_from_zero(cuda_device, dt, shift, V):
    """The probabilities are those of the logits' differences, wherever they lie: x c has an ulp of up to 1/2 here, which
    a thread whose largest logit changes on the way must not lose."""
    g = torch.Generator().manual_seed(V)
    B, k = 8, 3
    target = torch.sort(torch.randn(B, k + 1, V, generator=g) * 3, -1).values if V == 2000 else torch.randn(B, k + 1, V, generator=g) * 3
    draft = target[:, :k] + torch.randn(B, k, V, generator=g)
    target, draft = (target + shift).to(dt), (draft + shift).to(dt)
    t = torch.tensor([0.7, 1.0, 0.99, 1.3, 3.0, 0.5, 0.31, 2.0])
    drafts = (draft.float() / t[:, None, None] + gumbels(B, k, V, g=g)).argmax(-1).int()
    u, gumbel = torch.rand(B, k, generator=g), gumbels(B, V, g=g)
    for dl in (None, draft):
        want = plain_chain(target, drafts, u, gumbel, t, dl)
        got = ops.sample_accept(*[x.to(cuda_device) for x in (target, drafts, u, gumbel, t)],
                                draft_logits=None if dl is None else dl.to(cuda_device))
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
        same_logprobs(got[2], want[2])


def test_sampling_at_an_infinite_temperature(cuda_device):
    """All tokens but those of minus infinity have the same probability."""
    g = torch.Generator().manual_seed(3)
    B, k, V = 4, 1, 5000
    x = torch.randn(B, k + 1, V, generator=g) * 3
    x[:, :, ::3] = -math.inf
    x[0, :, 1] = 3e38
    x[1, :, 1] = -3e38
    gumbel, t = gumbels(B, V, g=g), torch.full((B,), math.inf)
    drafts = torch.zeros(B, k, dtype=torch.int32)  # a token without probability: rejected
    n, emitted, logp = ops.sample_accept(*[y.to(cuda_device) for y in (x, drafts, torch.full((B, k), 0.5), gumbel, t)])
    live = (x[0, 0] > -math.inf)
    want = torch.where(live, gumbel, -math.inf).argmax(-1)
    assert n.tolist() == [0] * B and emitted[:, 0].tolist() == want.tolist()
    assert bool(((logp[:, 0].cpu() + math.log(int(live.sum()))).abs() <= 1e-5).all())


@pytest.mark.parametrize("dt, V", [(torch.bfloat16, (1 << 28) + 3), (torch.float32, (1 << 27) + 1), (torch.bfloat16, (1 << 30))])
def test_sample_accept_over_long_rows(cuda_device, dt, V):
    """Sums of 2^30 terms, each below half an ulp of what a thread has summed: the log-probability is that of the
    count. And tokens beyond 2^29 are drawn by their keys."""
    x = torch.full((1, 2, V), -0.357, dtype=dt, device=cuda_device)
    x[:, :, ::1021] = 0.0  # some in every thread's share
    gumbel = torch.zeros(1, V, device=cuda_device)
    gumbel[0, V - 2] = 3.0
    n, emitted, logp = ops.sample_accept(x, torch.full((1, 1), 7, dtype=torch.int32, device=cuda_device),
                                         torch.full((1, 1), 0.999, device=cuda_device), gumbel,
                                         torch.ones(1, device=cuda_device))
    e, tops = float(x[0, 0, 1]), -(-V // 1021)
    want = float(x[0, 0, V - 2]) - math.log(tops + (V - tops) * math.exp(e))
    assert n.tolist() == [0] and emitted[:, 0].tolist() == [V - 2]
    assert abs(float(logp[0, 0]) - want) <= 2.0 ** -22 + 3 * U32 + 64 * U32 + U32 * abs(want)


def test_tree_sample_accept_refuses_rows_of_another_temperature(cuda_device):
    """Offsets that do not ascend, or rows that two sequences share, would give a row the sums of another
    sequence's temperature: such a sequence is reported and left out, the others are right, and where the
    temperatures are the same nothing is wrong."""
    g = torch.Generator().manual_seed(2)
    V, n, tree = 700, 5, [-1, 0, 0, 1, 1]
    logits = torch.randn(3 * n, V, generator=g) * 3
    tokens = torch.randint(0, V, (3 * n,), generator=g, dtype=torch.int32)
    for b in range(3):
        tokens[b * n + 1] = int(logits[b * n].argmax())
    u, gumbel = torch.rand(3 * n, generator=g) * 0.5, gumbels(4, V, g=g)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    for offsets, lens, temps, good in (
            ([0, 5, 10, 15], [5, 5, 5, 0], [0.7, 0.0, 1.3, 0.4], [0, 1, 2]),   # as documented, one without nodes
            ([0, 5, 10, 0], [5, 5, 5, 0], [0.7, 0.0, 1.3, 0.4], None),         # the padding's offset does not ascend
            ([10, 0, 5, 15], [5, 5, 5, 0], [0.7, 0.0, 1.3, 0.4], None),
            ([0, 0, 5, 10], [5, 5, 5, 5], [0.7, 0.9, 1.3, 0.4], [1, 2, 3]),    # shared rows, of two temperatures
            ([0, 0, 5, 10], [5, 5, 5, 5], [0.7, 0.7, 0.0, 0.4], [0, 1, 2, 3]),  # of one
            ([0, 3, 5, 10], [5, 5, 5, 5], [0.7, 0.9, 1.3, 0.4], [2, 3])):
        status = ops.status_tensor(cuda_device)
        t = torch.tensor(temps)
        got = ops.tree_sample_accept(logits.to(cuda_device), tokens.to(cuda_device), i32(tree * 3), i32(lens), i32(offsets), n,
                                     u.to(cuda_device), gumbel.to(cuda_device), t.to(cuda_device), status=status)
        live = [b for b in range(4) if lens[b]]
        right = []
        for b in live:
            s = slice(offsets[b], offsets[b] + n)
            want = plain_tree(logits[s], tokens[s], tree, u[s], gumbel[b], t[b], n)
            if int(got[0][b]) != -1:
                assert (int(got[0][b]), got[1][b].tolist(), got[2][b].tolist()) == want[:3], (offsets, b)
                same_logprobs(got[3][b:b + 1], [want[3]])
                right.append(b)
        assert good is None or right == good, (offsets, right)
        assert (int(status) == -7) == (right != live), offsets


# ---------------------------------------------------------------- drafts whose distribution is nearly the target's
def near_chain(B, V, g, eps, bump):
    """One draft a sequence, its logits eps away from the target's, its own raised by `bump`: it is rejected."""
    target = torch.randn(B, 2, V, generator=g) * 2
    draft = (target[:, :1] + eps * torch.randn(B, 1, V, generator=g)).float()
    p = target[:, 0].double().softmax(-1)
    drafts = (p - 1e-5).abs().argmin(-1)  # a token of about 1e-5: little of the residual is its doing
    draft[torch.arange(B), 0, drafts] += bump
    return target, draft, drafts[:, None].int(), torch.full((B, 1), 0.9999), gumbels(B, V, g=g), torch.ones(B)


@pytest.mark.parametrize("V", [2000, 32000])
@pytest.mark.parametrize("bump", [0.2, 1.0, 3.0])
def test_residual_of_equal_distributions_but_for_one_token(cuda_device, V, bump):
    """p - q is a small share of p, the same for every other token (their logits are equal): the draw is that from
    p without the draft, whatever the share. p and q are good to 2^-20 together, the share here is above
    1e-5 (e^bump - 1): its sign is certain, and the order is that of log p + gumbel, which 64 bits tell apart."""
    g = torch.Generator().manual_seed(V)
    target, draft, drafts, u, gumbel, t = near_chain(400, V, g, 0.0, bump)
    got = ops.sample_accept(*[x.to(cuda_device) for x in (target, drafts, u, gumbel, t)], draft_logits=draft.to(cuda_device))
    key = target[:, 0].double() + gumbel.double()
    key.scatter_(1, drafts.long(), -math.inf)
    assert got[0].tolist() == [0] * 400 and got[1][:, 0].tolist() == key.argmax(-1).tolist()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("eps", [1e-2, 1e-3, 1e-4, 1e-5, 1e-6])
def test_residual_of_nearly_equal_distributions(cuda_device, dt, eps):
    """The token drawn is the argmax of log(p - q) + gumbel for some p and q within their error: with both off
    by at most r of themselves (2^-21 for the exponentials and sums, the exponents' 2^-22 times their
    mean size under p), its greatest key reaches every other token's least."""
    g = torch.Generator().manual_seed(11)
    B, V = 400, 32000
    target, draft, drafts, u, gumbel, t = near_chain(B, V, g, eps, 2.0)
    target, draft = target.to(dt), draft.to(dt)
    n, emitted, _ = ops.sample_accept(*[x.to(cuda_device) for x in (target, drafts, u, gumbel, t)],
                                      draft_logits=draft.to(cuda_device))
    p, q = target[:, 0].double().softmax(-1), draft[:, 0].double().softmax(-1)
    rejected = 0.9999 * q.gather(1, drafts.long()) >= p.gather(1, drafts.long())
    assert bool(rejected.all()) and n.tolist() == [0] * B
    top = target[:, 0].double()
    r = 2.0 ** -21 + 2.0 ** -22 * 1.4427 * float((p * (top.amax(-1, keepdim=True) - top)).sum(-1).max())
    greatest = ((p - q) + r * (p + q)).clamp(min=0).log() + gumbel.double()
    least = ((p - q) - r * (p + q)).clamp(min=0).log() + gumbel.double()
    assert bool((least.amax(-1) > -math.inf).all())
    bar = least.amax(-1)
    chosen = greatest.gather(1, emitted[:, :1].long().cpu())[:, 0]
    assert bool((chosen >= bar).all()), int((chosen < bar).sum())


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 300, 30000])
@pytest.mark.parametrize("temperature", [0.3, 0.1, 0.04, 0.02])
def test_residual_where_one_token_has_nearly_all(cuda_device, dt, V, temperature):
    """p and q both give nearly all to the same token, and a draft of the little rest is rejected: that rest decides. The
    sums hold the largest token's 1 apart, so what p and q are off by, relative to themselves, is that of the others' terms: 2^-21 of
    their share, and 2^-22 times the exponents' mean size (the largest's is 0). The exponents x / T here, of 64 bits, are off by half
    an ulp of up to s = max |x| / T each, at x and at the largest: 2^-52 s of p, and 2^-51 for the other roundings. The token
    drawn is the argmax for some p and q within that; one of no weight to speak of never is."""
    g = torch.Generator().manual_seed(V)
    B = 300
    target = torch.randn(B, 2, V, generator=g)
    target[:, :, 1] += 5.0
    draft = target[:, :1] + 0.1 * torch.randn(B, 1, V, generator=g)
    drafts = 2 + torch.randint(0, V - 2, (B,), generator=g)
    draft[torch.arange(B), 0, drafts] += 3 * temperature
    draft[:, 0, 1] += 0.3 * (torch.arange(B) % 3 - 1) * temperature
    target, draft = target.to(dt), draft.to(dt)
    u, gumbel, t = torch.full((B, 1), 0.9999), gumbels(B, V, g=g), torch.full((B,), temperature)
    n, emitted, _ = ops.sample_accept(*[x.to(cuda_device) for x in (target, drafts[:, None].int(), u, gumbel, t)],
                                      draft_logits=draft.to(cuda_device))
    temp = float(t[0])
    p, q = (target[:, 0].double() / temp).softmax(-1), (draft[:, 0].double() / temp).softmax(-1)
    rejected = (0.9999 * q.gather(1, drafts[:, None]) > 1.001 * p.gather(1, drafts[:, None]))[:, 0]
    assert int(rejected.sum()) >= B // 2 and bool((n.cpu()[rejected] == 0).all())

    def error(w, x):
        x = x.double() / temp
        size = (w * (x.amax(-1, keepdim=True) - x)).sum(-1, keepdim=True) * 1.4427
        return w * (2.0 ** -21 * (1 - w.amax(-1, keepdim=True)) + 2.0 ** -22 * size + 2.0 ** -51 + 2.0 ** -52 * float(x.abs().max()))

    off = error(p, target[:, 0]) + error(q, draft[:, 0])
    greatest = ((p - q) + off).clamp(min=0).log() + gumbel.double()
    bar = (((p - q) - off).clamp(min=0).log() + gumbel.double()).amax(-1)
    chosen = greatest.gather(1, emitted[:, :1].long().cpu())[:, 0]
    sure = rejected & (bar > -math.inf)
    assert int(sure.sum()) >= B // 3 and bool((chosen >= bar)[sure].all()), int((chosen < bar)[sure].sum())

# ---------------------------------------------------------------- the 8-bit cache's scales
@pytest.mark.parametrize("heads, nodes, bs", [((3, 3, 64), [2, 1], 1), ((4, 1, 128), [2, 1], 7), ((3, 3, 64), [5, 9], 1),
                                              ((6, 1, 128), [9, 4], 7), ((6, 3, 64), [1, 2], 16)])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_scales_that_start_and_end_anywhere(cuda_device, heads, nodes, bs, shift):
    """Scales that are a slice of a larger buffer, at any byte, and end inside an aligned word."""
    args, *lens = attention_case("fp8", heads, nodes, [37, 90], bs, "tree", 12, cuda_device)
    want = ops.tree_attention(**args)
    check_attention(args, *lens, want)
    for name in ("k_scale", "v_scale"):
        n = args[name].numel()
        buf = torch.full((n + 8,), 255, dtype=torch.uint8, device=cuda_device)
        args[name] = buf[shift:shift + n].view(args[name].shape).copy_(args[name])
    status = ops.status_tensor(cuda_device)
    got = ops.tree_attention(**args, status=status)
    check_attention(args, *lens, got)
    assert int(status) == 0


# ---------------------------------------------------------------- infinities in the history
def exact_rows(args, ctx, nodes, off):
    """The formula in 64 bits, a score of minus infinity being a weight of 0 (a row of nothing else: zeros), and the
    bound on the error of the outputs: that of test_gpu_tree_sampling.py over the keys with finite scores."""
    q, mask = args["q"].cpu().double(), args["tree_mask"].cpu()
    k, v = values(args["pool_k_layer"].cpu(), None if args["k_scale"] is None else args["k_scale"].cpu()), \
        values(args["pool_v_layer"].cpu(), None if args["v_scale"] is None else args["v_scale"].cpu())
    bs, nkv, hd = k.shape[1:]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for b, (c, n, o) in enumerate(zip(ctx, nodes, off)):
        t, pos = args["block_tables"][b].cpu().long(), torch.arange(c)
        kk, vv = k[t[pos // bs], pos % bs], v[t[pos // bs], pos % bs]
        bits = torch.tensor([[bool(int(mask[o + i, j // 32]) >> j % 32 & 1) for j in range(n)] for i in range(n)])
        seen = torch.cat([torch.ones(n, c - n, dtype=torch.bool), bits], 1)
        for h in range(q.shape[1]):
            kh, vh, qh = kk[:, h // (q.shape[1] // nkv)], vv[:, h // (q.shape[1] // nkv)], q[o:o + n, h]
            s = (qh[:, None] * kh[None]).sum(-1) * args["scale"]
            live = seen & (s > -math.inf)
            s = torch.where(live, s, -math.inf)
            top = s.amax(-1, keepdim=True)
            w = torch.where(live, (s - torch.where(top == -math.inf, 0.0, top)).exp(), 0.0)
            w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
            terms = torch.where(live[..., None], w[..., None] * vh[None], 0.0)
            r, a = terms.sum(1), terms.abs().sum(1)
            size = torch.where(live, (qh.abs()[:, None] * kh.abs()[None]).sum(-1), 0.0).amax(-1)[:, None] * args["scale"]
            d = (hd + 4) * U32 * size + 2.0 ** -21
            if args["q"].dtype == torch.float32:
                e = 2 * (d + 2.0 ** -21 * size) * a + (2.0 ** -21 + c * U32) * a + U32 * r.abs()
            else:
                e = 2 * d * a + (U16 + 2.0 ** -14) * a + U16 * r.abs()
            out[o:o + n, h], tol[o:o + n, h] = r, e * 1.01 + 1e-30
    return out, tol


def compare(got, want, tol):
    got, fin = got.cpu().double(), torch.isfinite(want)
    assert torch.equal(got[~fin].nan_to_num(7e300), want[~fin].nan_to_num(7e300))
    assert bool(((got - want).abs() <= tol)[fin].all()), float(((got - want).abs() / tol)[fin].max())


SHAPES = [((8, 2, 64), [1, 2]), ((8, 2, 64), [9, 4]), ((16, 2, 128), [40, 3])]


@pytest.mark.parametrize("heads, nodes", SHAPES)
@pytest.mark.parametrize("cache, share, nodes_seen", [("bf16", 0.5, False), ("bf16", 0.5, True), ("bf16", 1.0, False),
                                                      ("bf16", 1.0, True), ("fp8", 1.0, False), ("fp32", 0.5, False),
                                                      ("fp32", 0.5, True), ("fp32", 1.0, False), ("fp32", 1.0, True)])
def test_scores_of_minus_infinity_in_the_history(cuda_device, cache, heads, nodes, share, nodes_seen):
    """A key whose score is minus infinity has no weight; a row with no other key gets zeros. In e4m3, which has no
    infinity, it is q that makes the scores infinite, all of them."""
    args, ctx, nodes, off = attention_case(cache, heads, nodes, [700, 130], 16, "tree", 3, cuda_device)
    if not nodes_seen:
        args["tree_mask"].zero_()
    k = args["pool_k_layer"]
    if cache == "fp8":
        k.view(torch.uint8)[..., 0] = 0x38  # 1
        args["q"][..., 0] = -math.inf
    else:
        spare = torch.rand(k.shape[:-1], generator=torch.Generator().manual_seed(1)).to(cuda_device) >= share
        k[..., 0] = torch.where(spare, 1.0, -math.inf)
        args["q"][..., 0] = 1.0
    compare(ops.tree_attention(**args), *exact_rows(args, ctx, nodes, off))


@pytest.mark.parametrize("heads, nodes", SHAPES)
@pytest.mark.parametrize("cache", ["bf16", "fp32"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_infinite_values_in_the_history(cuda_device, cache, heads, nodes, value):
    """Infinite elements of the history's V make their dims infinite in every row, opposite ones NaN, and leave
    the others right."""
    args, ctx, nodes, off = attention_case(cache, heads, nodes, [700, 130], 16, "tree", 6, cuda_device)
    v, table = args["pool_v_layer"], args["block_tables"].tolist()
    for b, pos, h, d in ((0, 0, 0, 5), (0, 399, 1, 17), (0, 650, 1, 63), (1, 64, 0, 0), (1, 100, 0, 1)):
        v[table[b][pos // 16], pos % 16, h, d] = value
    v[table[1][5], 3, 0, 0] = math.inf   # sequence 1, kv head 0, dim 0: infinity of either sign, or a NaN
    compare(ops.tree_attention(**args), *exact_rows(args, ctx, nodes, off))


@pytest.mark.parametrize("heads", [(8, 2, 64), (2, 2, 128)])
def test_fp32_values_next_to_the_largest(cuda_device, heads):
    """One key: its V comes back as it is, the largest numbers too."""
    args, ctx, nodes, off = attention_case("fp32", heads, [1, 1], [0, 0], 16, "tree", 6, cuda_device)
    args["pool_v_layer"][..., ::3] = torch.finfo(torch.float32).max
    args["pool_v_layer"][..., 1::3] = -3.4e38
    want, tol = exact_rows(args, ctx, nodes, off)
    compare(ops.tree_attention(**args), want, tol)


# ---------------------------------------------------------------- the largest calls
def check_on_device(args, ctx, nodes, off, got):
    """check_attention for many rows: the same formula and bound, in 64 bits on the device."""
    q, mask = args["q"].double(), args["tree_mask"]
    k, v = values(args["pool_k_layer"], args["k_scale"]), values(args["pool_v_layer"], args["v_scale"])
    bs, nkv, hd = k.shape[1:]
    group = q.shape[1] // nkv
    for b, (c, n, o) in enumerate(zip(ctx, nodes, off)):
        pos = torch.arange(c, device=q.device)
        t = args["block_tables"][b].long()
        kk, vv = k[t[pos // bs], pos % bs], v[t[pos // bs], pos % bs]
        j = torch.arange(n, device=q.device)
        if mask is None:
            bits = j[None] <= j[:, None]
        else:
            bits = (mask[o:o + n][:, j // 32] >> (j % 32)[None] & 1).bool()
        seen = torch.cat([torch.ones(n, c - n, dtype=torch.bool, device=q.device), bits], 1)
        for h in range(q.shape[1]):
            qh, kh, vh = q[o:o + n, h], kk[:, h // group], vv[:, h // group]
            s = torch.where(seen, qh @ kh.T * args["scale"], -math.inf)
            w = torch.where(seen.any(1, keepdim=True), s.softmax(-1), 0.0)
            r, a = w @ vh, w @ vh.abs()
            size = torch.where(seen, qh.abs() @ kh.abs().T, 0.0).amax(-1, keepdim=True) * args["scale"]
            d = (hd + 4) * U32 * size + 2.0 ** -21
            if args["q"].dtype == torch.float32:
                tol = 2 * (d + 2.0 ** -21 * size) * a + (2.0 ** -21 + c * U32) * a + U32 * r.abs()
            else:
                tol = 2 * d * a + (U16 + 2.0 ** -14) * a + U16 * r.abs()
            err = (got[o:o + n, h].double() - r).abs()
            assert bool((err <= tol * 1.01 + 1e-30).all()), (b, h, float((err / (tol * 1.01 + 1e-30)).max()))


@pytest.mark.parametrize("cache", ["bf16", "fp32", "fp8"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (16, 2, 128)])
@pytest.mark.parametrize("nodes, hists, kind", [([1024, 1000], [0, 700], "none"), ([1024, 1, 513], [1500, 40, 31], "random"),
                                                ([700, 1024], [64, 3], "tree")])
def test_tree_attention_of_up_to_1024_rows(cuda_device, cache, heads, nodes, hists, kind):
    """The pieces in which a prompt is read, and the largest trees."""
    args, *lens = attention_case(cache, heads, nodes, hists, 16, kind, 51, cuda_device)
    status = ops.status_tensor(cuda_device)
    ws = ops.Workspace(cuda_device)
    got = ops.tree_attention(**args, workspace=ws, status=status)
    check_on_device(args, *lens, got)
    assert int(status) == 0 and int(ws.buf[:65536 if ws.buf.numel() > 65536 else 0].sum()) == 0
    assert torch.equal(ops.tree_attention(**args, workspace=ws), got)


def test_a_prompt_in_pieces_over_the_8_bit_cache(cuda_device):
    """A prompt written and attended in pieces of 1024, 1024 and 500: every piece's rows are those of one causal
    attention over what the cache holds."""
    nq, nkv, hd, bs, n = 8, 2, 64, 16, 2548
    g = torch.Generator().manual_seed(7)
    pools = [torch.zeros(n // bs + 2, bs, nkv, hd, dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.full((n // bs + 2, bs, nkv), 127, dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    table = torch.randperm(n // bs + 2, generator=g)[:-(-n // bs)].to(torch.int32)[None].to(cuda_device)
    angle = torch.arange(float(n))[:, None] * 1e4 ** (-torch.arange(0, hd, 2) / hd)
    cos, sin = angle.cos().to(cuda_device), angle.sin().to(cuda_device)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    ws, start = ops.Workspace(cuda_device), 0
    for m in (1024, 1024, 500):
        qkv = torch.randn(m, (nq + 2 * nkv) * hd, generator=g).to(torch.bfloat16).to(cuda_device)
        pos = torch.arange(start, start + m, dtype=torch.int32, device=cuda_device)
        slots = table[0][(pos // bs).long()] * bs + pos % bs
        q = torch.empty(m, nq, hd, dtype=torch.bfloat16, device=cuda_device)
        ops.qkv_rope_append_fp8(qkv, pos, slots.to(torch.int32), cos, sin, q, *pools, *scales, nq, nkv, hd)
        args = dict(q=q, pool_k_layer=pools[0], pool_v_layer=pools[1], block_tables=table, ctx_lens=i32(start + m),
                    q_lens=i32(m), q_offsets=i32(0), max_q_len=m, max_ctx=start + m, scale=hd ** -0.5, tree_mask=None,
                    k_scale=scales[0], v_scale=scales[1])
        check_on_device(args, [start + m], [m], [0], ops.tree_attention(**args, workspace=ws))
        start += m


# ---------------------------------------------------------------- a captured step
@pytest.mark.parametrize("cache", ["bf16", "fp8"])
def test_a_whole_step_captured_and_replayed(cuda_device, cache):
    """Rows written, attended, verified and moved together in one graph on a side stream, with one workspace for all: replays
    with new inputs leave what the same calls leave outside a graph."""
    dev, nq, nkv, hd, bs, layers, V = cuda_device, 14, 2, 64, 16, 3, 3000
    g, rng = torch.Generator().manual_seed(4), random.Random(4)
    trees = [[-1, 0, 0, 1, 1, 3, 5], [-1, 0, 1, 1, 2], [-1]]
    nodes, hist, off = [7, 5, 1], [900, 30, 77], [0, 7, 12, 13]
    fp8, dt, n = cache == "fp8", torch.bfloat16, 13
    pools = []
    for _ in range(2):
        pool = PagedKVCache(layers, nkv, hd, 70, bs, torch.float8_e4m3fn if fp8 else dt, dev)
        for x in (pool.k, pool.v):
            x.copy_((torch.randn(x.shape, generator=torch.Generator().manual_seed(8)) * 2).to(x.dtype))
        pools.append(pool)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    ids = list(range(70))
    rng.shuffle(ids)
    table = torch.zeros(3, 57, dtype=torch.int32)
    for b, (h, m) in enumerate(zip(hist, nodes)):
        k = -(-(h + m) // bs)
        table[b, :k] = torch.tensor([ids.pop() for _ in range(k)])
    slots = i32([int(table[b, p // bs]) * bs + p % bs for b in range(3) for p in range(hist[b], hist[b] + nodes[b])])
    pos = i32([h + i for h, m in zip(hist, nodes) for i in range(m)])
    angle = torch.arange(1000.0)[:, None] * 1e4 ** (-torch.arange(0, hd, 2) / hd)
    cos, sin, mask = angle.cos().to(dev), angle.sin().to(dev), ops.tree_mask_words(trees).to(dev)
    fixed = [table.to(dev), i32([h + m for h, m in zip(hist, nodes)]), i32(nodes), i32(off), i32(hist), i32(sum(trees, []))]

    def fresh():
        logits, tokens, u = tree_inputs(trees, V, dt, g, rng)
        return [torch.randn(layers, n, (nq + 2 * nkv) * hd, generator=g).to(dt), logits, tokens, u * 0.005, gumbels(3, V, g=g),
                torch.tensor([0.8, 0.0, 1.2])]

    def step(pool, x, ws, q):
        outs = []
        for layer in range(layers):
            into = [pool.k[layer], pool.v[layer]]
            scales = [pool.k_scale[layer], pool.v_scale[layer]] if fp8 else []
            (ops.qkv_rope_append_fp8 if fp8 else ops.qkv_rope_append)(x[0][layer], pos, slots, cos, sin, q, *into, *scales, nq, nkv, hd)
            outs.append(ops.tree_attention(q, *into, *fixed[:4], 7, 907, hd ** -0.5, mask, *scales, workspace=ws))
        res = ops.tree_sample_accept(x[1], x[2], fixed[5], fixed[2], fixed[3], 7, x[3], x[4], x[5], workspace=ws)
        ops.kv_commit_path(pool.k, pool.v, fixed[0], fixed[4], res[1], res[0], pool.k_scale, pool.v_scale)
        return outs + list(res)

    q = torch.empty(n, nq, hd, dtype=dt, device=dev)
    inputs = [x.to(dev) for x in fresh()]
    ws = ops.Workspace(dev)
    ws.get(8 << 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    moved = 0
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(pools[0], inputs, ws, q)
        for _ in range(3):
            new = [x.to(dev) for x in fresh()]
            for x, y in zip(inputs, new):
                x.copy_(y)
            graph.replay()
            want = step(pools[1], new, ops.Workspace(dev), torch.empty_like(q))
            side.synchronize()
            for x, y in zip(got, want):
                assert torch.equal(x, y)
            for a, b in ((pools[0].k, pools[1].k), (pools[0].v, pools[1].v)):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            if fp8:
                assert torch.equal(pools[0].k_scale, pools[1].k_scale) and torch.equal(pools[0].v_scale, pools[1].v_scale)
            moved += sum(want[layers].tolist())
    assert moved >= 3  # the numbers accept paths, so that rows move
    assert int(ws.buf[:65536].sum()) == 0
