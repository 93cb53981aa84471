"""Sampling, draft trees and the 8-bit cache at their limits: temperatures and logits of every size.

Tolerances as in test_gpu_tree_sampling.py, which derives them.
"""

import math

import pytest
import torch

from kvengine_b200 import ops
from test_gpu_tree_sampling import plain_chain, plain_tree, same_logprobs

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
