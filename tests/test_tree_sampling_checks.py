"""Checks of the Python wrappers of sampling, draft trees and the 8-bit cache that no GPU is needed for: tensors on the
CPU stand in for those of a device (their index is -1 throughout), and the library's call is recorded instead of made."""

import pytest
import torch

from kvengine_b200 import _lib as L
from kvengine_b200 import ops

E4M3, U8, I32, BF = torch.float8_e4m3fn, torch.uint8, torch.int32, torch.bfloat16


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(ops, "_device", lambda t: -1)
    monkeypatch.setattr(ops, "_call", lambda fn, index, *args: made.append(args))
    monkeypatch.setattr(L, "_fast", L._NoFast())
    return made


def cache(layers=None):
    shape = (4, 16, 2, 64) if layers is None else (layers, 4, 16, 2, 64)
    return [torch.zeros(shape, dtype=U8).view(E4M3) for _ in range(2)] + [torch.zeros(shape[:-1], dtype=U8) for _ in range(2)]


def i32(*x):
    return torch.tensor(x, dtype=I32)


def public_calls():
    k, v, ks, vs = cache()
    q, qkv = torch.zeros(3, 4, 64, dtype=BF), torch.zeros(3, 8 * 64, dtype=BF)
    rope = torch.zeros(9, 32)
    rows = torch.zeros(3, 2, 64, dtype=BF)
    logits, t1 = torch.zeros(1, 3, 50), torch.zeros(1)
    big = cache(2)
    return {
        "tree_attention": lambda **kw: ops.tree_attention(q, k, v, i32(0, 1, 2, 3)[None], i32(60), i32(3), i32(0), 3, 3000, 0.1,
                                                          k_scale=ks, v_scale=vs, **kw),
        "qkv_rope_append_fp8": lambda **kw: ops.qkv_rope_append_fp8(qkv, i32(0, 1, 2), i32(0, 1, 2), rope, rope, q, k, v, ks, vs,
                                                                    4, 2, 64, **kw),
        "kv_append_fp8": lambda **kw: ops.kv_append_fp8(rows, rows, torch.arange(3), k, v, ks, vs, **kw),
        "kv_read_fp8": lambda **kw: ops.kv_read_fp8(k, v, ks, vs, torch.arange(3), **kw),
        "sample_accept": lambda **kw: ops.sample_accept(logits, i32(1, 2)[None], torch.zeros(1, 2), torch.zeros(1, 50), t1, **kw),
        "tree_sample_accept": lambda **kw: ops.tree_sample_accept(logits[0], i32(0, 1, 2), i32(-1, 0, 0), i32(3), i32(0), 3,
                                                                  torch.zeros(3), torch.zeros(1, 50), t1, **kw),
        "kv_commit_path": lambda **kw: ops.kv_commit_path(big[0], big[1], i32(0, 1)[None], i32(4), i32(0, 2)[None], i32(1),
                                                          big[2], big[3], **kw),
    }


NAMES = ["tree_attention", "qkv_rope_append_fp8", "kv_append_fp8", "kv_read_fp8", "sample_accept", "tree_sample_accept",
         "kv_commit_path"]


@pytest.mark.parametrize("name", NAMES)
def test_status_is_checked(calls, name):
    """A kernel writes there: only int32 of the call's device will do."""
    call = public_calls()[name]
    call()
    call(status=torch.zeros(1, dtype=I32))
    assert len(calls) == 2
    for bad in (torch.zeros(1, dtype=torch.int64), torch.zeros(1), torch.zeros(0, dtype=I32), torch.zeros(4, dtype=I32)[::2]):
        with pytest.raises(ValueError):
            call(status=bad)
    assert len(calls) == 2


@pytest.mark.parametrize("name", ["tree_attention", "sample_accept", "tree_sample_accept"])
def test_workspace_is_checked(calls, name):
    class Other(ops.Workspace):
        def get(self, nbytes):
            return torch.zeros(nbytes, dtype=torch.int8)  # stands for a buffer of another device

    call = public_calls()[name]
    call(workspace=ops.Workspace("cpu"))
    assert len(calls) == 1
    with pytest.raises(ValueError):
        call(workspace=Other("cpu"))
    assert len(calls) == 1
