"""Host side of the sampling, draft-tree and 8-bit-cache operators: every refusal of the C ABI
comes before anything is launched (so it is testable without a GPU), mask words against a
plain construction, and the 8-bit pool's bookkeeping."""

import ctypes as C
import random

import pytest
import torch

from kvengine_b200 import _lib as L
from kvengine_b200 import ops
from kvengine_b200.paged import PagedKVCache

P = 1 << 20  # a stand-in pointer, 16-byte aligned and never read: all calls here are refused


def refused(code, words, rc):
    assert rc == code, (rc, L.load().kve_last_error())
    assert words in L.load().kve_last_error().decode()


ATTN = dict(q=P, dtype=L.KVE_BF16, pool_k=P, pool_v=P, kv_dtype=L.KVE_BF16, k_scale=None, v_scale=None, tables=P, stride=8,
            ctx=P, q_lens=P, q_offsets=P, mask=P, words=1, batch=2, q_rows=18, max_q=9, max_ctx=100, nq=8, nkv=2, hd=64, bs=16,
            blocks=32, scale=0.1, out=P, ws=P, ws_bytes=1 << 30, status=None, stream=None)


@pytest.mark.parametrize("change, code, words", [
    (dict(batch=-1), -1, "bad sizes"), (dict(max_q=-1), -1, "bad sizes"), (dict(q_rows=-1), -1, "bad sizes"), (dict(scale=float("nan")), -1, "scale nan"),
    (dict(scale=float("inf")), -1, "scale inf"), (dict(max_ctx=8), -1, "bad sizes"),
    (dict(nq=7), -1, "bad sizes"), (dict(nkv=0), -1, "bad sizes"), (dict(bs=0), -1, "bad sizes"),
    (dict(stride=0), -1, "bad sizes"), (dict(blocks=0), -1, "bad sizes"),
    (dict(hd=96), -2, "head_dim 96"), (dict(nq=130), -2, "group 65"),
    (dict(max_q=1025, max_ctx=2000, words=33), -2, "max_q_len 1025"),
    (dict(dtype=2), -3, "dtype 2"), (dict(kv_dtype=L.KVE_F32), -3, "cache of dtype 0"),
    (dict(dtype=L.KVE_F32, kv_dtype=L.KVE_FP8_E4M3, k_scale=P, v_scale=P), -3, "cache of dtype 2"),
    (dict(kv_dtype=L.KVE_FP8_E4M3, k_scale=P), -1, "null scales"),
    (dict(q=None), -1, "null pointer"), (dict(out=None), -1, "null pointer"), (dict(tables=None), -1, "null pointer"),
    (dict(max_q=33, words=1), -1, "mask words"), (dict(pool_k=P + 8), -1, "aligned"), (dict(q=P + 4), -1, "aligned"),
    (dict(max_ctx=5000, ws=None), -6, "workspace needs"), (dict(max_ctx=5000, ws_bytes=65536), -6, "workspace needs"),
    (dict(max_ctx=5000, ws=P + 8), -1, "workspace must be"),
])
def test_tree_attention_refusals(change, code, words):
    a = dict(ATTN, **change)
    refused(code, words, L.load().kve_paged_tree_attn(*a.values()))


def test_tree_attention_empty_calls_and_workspace():
    lib = L.load()
    assert lib.kve_paged_tree_attn(*dict(ATTN, batch=0, q=None).values()) == 0
    assert lib.kve_paged_tree_attn(*dict(ATTN, max_q=0, q=None).values()) == 0
    assert lib.kve_tree_attn_workspace_bytes(0, 1, 1, 8, 2, 64) == 0
    assert lib.kve_tree_attn_workspace_bytes(1, 1, 64, 8, 2, 64) == 0  # one chunk: nothing to join
    assert lib.kve_tree_attn_workspace_bytes(1, 1, 5000, 8, 2, 64) > 65536


def test_fp8_cache_refusals():
    lib = L.load()
    rope = dict(qkv=P, dtype=1, n=4, nq=4, nkv=2, hd=64, pos=P, slots=P, cos=P, sin=P, rope_len=10, q_out=P, k=P, v=P, ks=P,
                vs=P, num_slots=64, status=None, stream=None)
    app = dict(k_new=P, v_new=P, dtype=1, slots=P, n=4, nkv=2, hd=64, k=P, v=P, ks=P, vs=P, num_slots=64, status=None,
               stream=None)
    read = dict(k=P, v=P, ks=P, vs=P, slots=P, n=4, nkv=2, hd=64, num_slots=64, dtype=1, k_out=P, v_out=P, status=None,
                stream=None)
    for fn, base in ((lib.kve_qkv_rope_append_fp8, rope), (lib.kve_kv_append_fp8, app), (lib.kve_kv_read_fp8, read)):
        refused(-1, "bad sizes", fn(*dict(base, n=-1).values()))
        refused(-1, "bad sizes", fn(*dict(base, nkv=0).values()))
        refused(-1, "bad sizes", fn(*dict(base, num_slots=0).values()))
        refused(-2, "head_dim 80", fn(*dict(base, hd=80).values()))
        refused(-3, "dtype 2", fn(*dict(base, dtype=2).values()))
        refused(-1, "null pool", fn(*dict(base, ks=None).values()))
        refused(-1, "aligned", fn(*dict(base, v=P + 1).values()))
        refused(-1, "null pointer", fn(*dict(base, slots=None).values()))
        assert fn(*dict(base, n=0, slots=None).values()) == 0
    refused(-1, "bad sizes", lib.kve_qkv_rope_append_fp8(*dict(rope, rope_len=0).values()))
    refused(-1, "aligned", lib.kve_qkv_rope_append_fp8(*dict(rope, cos=P + 4).values()))
    refused(-1, "aligned", lib.kve_kv_append_fp8(*dict(app, k_new=P + 2).values()))
    refused(-1, "aligned", lib.kve_kv_read_fp8(*dict(read, v_out=P + 2).values()))


CHAIN = dict(logits=P, dtype=0, stride=1000, draft=None, dsb=0, dsj=0, drafts=P, tsb=4, tsj=1, u=P, usb=4, gumbel=P, gs=1000,
             t=P, batch=2, k=4, vocab=1000, n=P, emitted=P, logp=P, ws=P, ws_bytes=1 << 20, status=None, stream=None)
TREE = dict(logits=P, dtype=0, stride=1000, tokens=P, parents=P, q_lens=P, q_offsets=P, u=P, gumbel=P, gs=1000, t=P, batch=2,
            rows=12, max_q=7, vocab=1000, n=P, path=P, emitted=P, logp=P, ws=P, ws_bytes=1 << 20, status=None, stream=None)


@pytest.mark.parametrize("change, code, words", [
    (dict(batch=-1), -1, "bad sizes"), (dict(k=0), -1, "bad sizes"), (dict(k=32, usb=32), -1, "bad sizes"),
    (dict(vocab=0), -1, "bad sizes"), (dict(stride=999), -1, "bad sizes"), (dict(gs=999), -1, "bad sizes"),
    (dict(usb=3), -1, "bad sizes"), (dict(draft=P, dsb=-1), -1, "bad sizes"), (dict(dtype=2), -3, "dtype 2"),
    (dict(logits=None), -1, "null pointer"), (dict(t=None), -1, "null pointer"), (dict(ws=None), -6, "workspace needs"),
    (dict(ws_bytes=65536), -6, "workspace needs"), (dict(ws=P + 8), -1, "aligned"),
    (dict(batch=1 << 29), -2, "too many rows"),
    (dict(vocab=(1 << 30) + 1, stride=1 << 31, gs=1 << 31), -2, "vocab 1073741825"),
])
def test_sample_accept_refusals(change, code, words):
    refused(code, words, L.load().kve_sample_accept(*dict(CHAIN, **change).values()))


@pytest.mark.parametrize("change, code, words", [
    (dict(batch=-1), -1, "bad sizes"), (dict(max_q=0), -1, "bad sizes"), (dict(rows=-1), -1, "bad sizes"),
    (dict(rows=0), -1, "no rows"), (dict(max_q=1025), -2, "max_q_len 1025"), (dict(dtype=5), -3, "dtype 5"),
    (dict(parents=None), -1, "null pointer"), (dict(path=None), -1, "null pointer"),
    (dict(ws_bytes=65535), -6, "workspace needs"),
    (dict(vocab=(1 << 30) + 1, stride=1 << 31, gs=1 << 31), -2, "vocab 1073741825"),
])
def test_tree_sample_accept_refusals(change, code, words):
    refused(code, words, L.load().kve_tree_sample_accept(*dict(TREE, **change).values()))


def test_sample_workspaces_stay_clear_of_the_shared_counters():
    lib = L.load()
    assert lib.kve_sample_accept_workspace_bytes(0, 4, 1000, 0) == 0
    assert lib.kve_sample_accept_workspace_bytes(2, 4, 1000, 0) == 65536 + 10 * 8
    assert lib.kve_sample_accept_workspace_bytes(2, 4, 1000, 1) == 65536 + 18 * 8
    assert lib.kve_tree_sample_accept_workspace_bytes(12, 1000) == 65536 + 12 * 8
    assert lib.kve_sample_accept(*dict(CHAIN, batch=0, logits=None).values()) == 0
    assert lib.kve_tree_sample_accept(*dict(TREE, batch=0, logits=None).values()) == 0


COMMIT = dict(k=P, v=P, dtype=1, ks=None, vs=None, layers=2, blocks=8, bs=16, nkv=2, hd=64, tables=P, stride=4, start=P,
              path=P, path_stride=5, n=P, batch=2, status=None, stream=None)


@pytest.mark.parametrize("change, code, words", [
    (dict(layers=0), -1, "bad sizes"), (dict(path_stride=0), -1, "bad sizes"), (dict(dtype=3), -3, "dtype 3"),
    (dict(nkv=1, hd=4), -2, "bytes a row"), (dict(path_stride=1025), -2, "path_stride"), (dict(batch=65536), -2, "batch"),
    (dict(path=None), -1, "null pointer"), (dict(ks=P, vs=P), -1, "scales belong"), (dict(dtype=2), -1, "scales belong"),
    (dict(dtype=2, ks=P), -1, "scales belong"), (dict(k=P + 8), -1, "aligned"),
])
def test_commit_path_refusals(change, code, words):
    refused(code, words, L.load().kve_kv_commit_path(*dict(COMMIT, **change).values()))


def test_ops_refuse_cpu_tensors():
    x = torch.zeros(2, 4, 64)
    with pytest.raises(ValueError):
        ops.tree_attention(x, x, x, x, x, x, x, 1, 1, 1.0)
    with pytest.raises(ValueError):
        ops.sample_accept(x, x, x, x, x)
    with pytest.raises(ValueError):
        ops.tree_sample_accept(x[0], x, x, x, x, 2, x, x, x)
    with pytest.raises(ValueError):
        ops.kv_append_fp8(x, x, x, x, x, x, x)
    with pytest.raises(ValueError):
        ops.kv_read_fp8(x, x, x, x, x)
    with pytest.raises(ValueError):
        ops.qkv_rope_append_fp8(x, x, x, x, x, x, x, x, x, x, 2, 1, 64)
    with pytest.raises(ValueError):
        ops.kv_commit_path(x, x, x, x, x, x)


def test_tree_mask_words():
    rng = random.Random(3)
    trees = [[-1], [-1, 0, 0, 1], [], [-1] + [rng.randint(0, i - 1) for i in range(1, 70)], [-1, -1, 1]]
    words = ops.tree_mask_words(trees)
    assert words.shape == (78, 3) and words.dtype == torch.int32
    row = 0
    for t in trees:
        for i in range(len(t)):
            seen, at = set(), i
            while at >= 0:
                seen.add(at)
                at = t[at]
            got = {j for j in range(96) if int(words[row, j // 32]) >> j % 32 & 1}
            assert got == seen, (t, i)
            row += 1
    assert ops.tree_mask_words([[-1, 0]], max_q_len=40).shape == (2, 2)
    assert ops.tree_mask_words([]).shape == (0, 1)
    for bad in ([0], [-1, 1], [-1, -2]):
        with pytest.raises(ValueError):
            ops.tree_mask_words([bad])


def test_fp8_pool_bookkeeping():
    pool = PagedKVCache(2, 2, 64, 8, 16, torch.float8_e4m3fn, "cpu")
    assert pool.k.dtype == torch.float8_e4m3fn and pool.k_scale.shape == (2, 8, 16, 2)
    assert pool.nbytes() == 2 * (2 * 8 * 16 * 2 * 64 + 2 * 8 * 16 * 2)
    assert int(pool.k_scale.min()) == int(pool.v_scale.max()) == 127
    assert PagedKVCache(2, 2, 64, 8, 16, torch.bfloat16, "cpu").k_scale is None


def test_the_cpp_binding_is_built_and_leaves_other_calls_to_python():
    """Its functions return None, and touch nothing, for what is not a CUDA tensor."""
    fast = L.fast()
    assert not isinstance(fast, L._NoFast)
    q = torch.zeros(1, 2, 64)
    i = torch.zeros(1, dtype=torch.int32)
    assert fast.tree_attention(q, q, q, i, i, i, i, 1, 1, 1.0, None, None, None, None, None, None) is None
    with pytest.raises((ValueError, RuntimeError, TypeError)):
        ops.tree_attention(q, q[None], q[None], i[None], i, i, i, 1, 1, 1.0)
